// Shared parts of the attention kernels for long sequences (attention_long_fwd.hip, attention_long_bwd.hip).
//
// Mathematics (M maps per head: 1 = bucketed-bias attention, 2 = differential attention):
//   score2_m[i, j] = log2(e) * (scale * q_m[i] . k_m[j] + table[bucket(j - qpos_i), h]),  qpos_i = q_start + i
//   P_m = softmax over the keys a query may see, in base 2:  P_m = 2^(score2_m - lse2_m[i]),  lse2 = max + log2(sum)
//   out = P_0 v            (M = 1)          out = P_0 v - lam P_1 v   (M = 2),  lam = e^(l0 . l1) - e^(l2 . l3) + lam_init
//   backward: dP = dout v^T;  D_m[i] = sum_j P_m dP;  dS_m = c_m P_m (dP - D_m),  c = (1, -lam)
//             dq_m = scale dS_m k_m;  dk_m = scale dS_m^T q_m;  dv = (P_0 - lam P_1)^T dout;  dlam = -sum_i D_1
//             dtable[b, h] = sum over the pairs of bucket b of sum_m dS_m
//
// Every product runs on the 32 x 32 matrix instructions.  A lane of a 32 x 32 result holds ONE column (lane & 31) and the 16
// rows 8 (r / 4) + 4 (lane >> 5) + r % 4: with keys as rows and queries as columns the softmax is a loop over registers and one
// exchange between the two half waves, and the probabilities are already laid out as the second operand of the next product
// (the order of the contracted index inside an instruction is free; the transposed first operand is read from LDS in the same
// order: ds_read_b64_tr_b16 for 16-bit elements, plain words for f32).
//
// One code for three element types through 16-byte fragments (uint4): a lane's fragment is 8 (16-bit) or 4 (f32) consecutive
// elements of a row; mma() contracts two half waves' fragments -- one 32x32x16 instruction, or four exact 32x32x2 f32 ones.
#pragma once
#include "lds_dma.h"
#include "ptpp_common.h"

constexpr int LA_EDGES = 64;      // most logarithmic bucket edges
struct LongP {
  const void *q, *k, *v, *dout;
  void *out, *out2;  // out2: the second map's context, kept for backward (M = 2)
  void *dq, *gk, *gv;
  const float *table, *lam;
  const int *k_lengths, *q_lengths, *q_start;
  float *lse, *D;              // (M, B, H, TqP)
  double* lam_part;            // [B][H][query blocks]
  float* tab_part;             // [H][nbuckets][B][key blocks]
  float *part_o, *part_ml;     // few-row forward: [blocks][splits][M][32] rows of DV sums and their (max, sum)
  int64_t sq, sk, sv, so, sdo, sdq, sdk, sdv;  // batch strides, elements
  int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
  int B, Tq, Tk, TqP, H, Hk, dk, nbuckets, bidirectional, causal, lam_heads, max_distance, nexact, nedges;
  int nqt, nkt;         // row blocks of the forward / dq and of the dk, dv launches
  int nh, nrb, splits;  // few-row forward: query heads of a block, row blocks per head, key ranges
  int few_q, few_k;     // backward: blocks of 32 rows
  float scale, lam_init;
  int edges[LA_EDGES];
};

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(4))) short s16x4;

constexpr int LA_TILE = 64;       // rows of a streamed tile (keys in the forward / dq kernels, queries in the dk / dv kernel)
constexpr int LA_OWN = 32;        // rows that a wave owns
constexpr int LA_WAVES = 4;       // waves of a block
constexpr int LA_MAXD = 1024;     // largest max_distance
constexpr int LA_PAD = 2 * LA_OWN - 2;  // distances of a 32 x 32 patch beside a near pair lie within max_distance + 62
constexpr float LA_LOG2E = 1.4426950408889634f;

// ---- element types -----------------------------------------------------------------------------------------------------
template <typename E>
struct LOp;
template <>
struct LOp<bf16_raw> {
  static constexpr int CH = 8;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pk(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bf16x2_t));
  }
  static __device__ __forceinline__ float lo(uint32_t r) { return __uint_as_float(r << 16); }
  static __device__ __forceinline__ float hi(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }
};
template <>
struct LOp<f16_raw> {
  static constexpr int CH = 8;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pk(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, f16x2_t));
  }
  static __device__ __forceinline__ float lo(uint32_t r) { return (float)__builtin_bit_cast(f16x2_t, r)[0]; }
  static __device__ __forceinline__ float hi(uint32_t r) { return (float)__builtin_bit_cast(f16x2_t, r)[1]; }
};
template <>
struct LOp<float> {
  static constexpr int CH = 4;
  static __device__ __forceinline__ f32x16 mma(uint4 a, uint4 b, f32x16 c) {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
};

// CH consecutive registers of a 32 x 32 result -> a fragment.  16-bit: probabilities and dS are rounded to the element type
// (to nearest; dS in f16 scaled: LScale) because the matrix instruction takes both operands in it; their sums (softmax denominator, D)
// use the f32 values.
template <typename E>
__device__ __forceinline__ uint4 la_pack(const f32x16& v, int s) {
  if constexpr (sizeof(E) == 4) {
    return uint4{__float_as_uint(v[4 * s]), __float_as_uint(v[4 * s + 1]), __float_as_uint(v[4 * s + 2]), __float_as_uint(v[4 * s + 3])};
  } else {
    return uint4{LOp<E>::pk(v[8 * s], v[8 * s + 1]), LOp<E>::pk(v[8 * s + 2], v[8 * s + 3]), LOp<E>::pk(v[8 * s + 4], v[8 * s + 5]),
                 LOp<E>::pk(v[8 * s + 6], v[8 * s + 7])};
  }
}
// what la_pack's rounding took from registers [CH s, CH s + CH) of v, in the same layout (16-bit elements)
template <typename E>
__device__ __forceinline__ uint4 la_pack_rest(const f32x16& v, int s, uint4 f) {
  const uint32_t r[4] = {f.x, f.y, f.z, f.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = LOp<E>::pk(v[8 * s + 2 * i] - LOp<E>::lo(r[i]), v[8 * s + 2 * i + 1] - LOp<E>::hi(r[i]));
  return uint4{o[0], o[1], o[2], o[3]};
}
__device__ __forceinline__ float la_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float la_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// f16: dS as an operand.  dS = P (dP - D) is about 1 / keys of the gradient that arrives, and f16 ends at 2^-24 (2^-14 with all its bits) and
// 65504: unscaled, gradients of 1e-4 on 2000 keys kept four bits, smaller ones none.  A column of dS -- one query in dq, one key in dk --
// goes through the product times a power of two, its accumulators with it: the column's largest value so far lies in [2^11, 2^15], so a
// term loses at most 2^-36 of it beside its own rounding.  The scale starts at 2^100 and is lowered when a patch passes 2^15 (the accumulators
// follow, exactly); the other element types have f32's range and take none.  P needs none either: its rows add up to one.
// Price: backward of 24 x 833-1250 of 4 x 64 206 -> 220 us, of 8 x 1333-2000 differential 391 -> 410 us, of 32 x 145-217 of 2 x 128 none.
template <typename E>
struct LScale {
  template <int NT>
  __device__ __forceinline__ void apply(f32x16&, f32x16 (&)[NT]) {}
  __device__ __forceinline__ float undo(float v) const { return v; }
};
template <>
struct LScale<f16_raw> {
  float mul = 0x1p100f;  // (the first value above 2^-85 lowers it)
  template <int NT>
  __device__ __forceinline__ void apply(f32x16& s, f32x16 (&acc)[NT]) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(s[r]));
    m = la_half_max(m);
    const uint32_t old = __float_as_uint(mul) >> 23;  // exponents with their offset of 127
    const bool over = m > __uint_as_float(min(127 + 15 + 127 - old, 254u) << 23);  // 2^15 / mul
    if (__any(over)) {
      const uint32_t now = over ? 127 + 11 + 127 - (__float_as_uint(m) >> 23) : old;  // (at least 10: an infinity's exponent is 255)
      mul = __uint_as_float(now << 23);
      const float ratio = __uint_as_float((uint32_t)max((int)(now - old) + 127, 0) << 23);  // (now <= old)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] *= ratio;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= mul;
  }
  __device__ __forceinline__ float undo(float v) const { return v * __uint_as_float((254u << 23) - __float_as_uint(mul)); }
};

// dot product of two fragments in f32
template <typename E>
__device__ __forceinline__ float la_dot(uint4 a, uint4 b) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(E) == 4) s = fmaf(__uint_as_float(x[i]), __uint_as_float(y[i]), s);
    else s = fmaf(LOp<E>::hi(x[i]), LOp<E>::hi(y[i]), fmaf(LOp<E>::lo(x[i]), LOp<E>::lo(y[i]), s));
  }
  return s;
}
template <typename E>
__device__ __forceinline__ void la_store4(E* p, float a, float b, float c, float d) {
  if constexpr (sizeof(E) == 4) *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d};
  else *reinterpret_cast<uint2*>(p) = uint2{LOp<E>::pk(a, b), LOp<E>::pk(c, d)};
}

// ---- LDS images: [rows][DK] elements, the 16-byte chunks of a row permuted by la_swz(row) --------------------------------
// Chosen so that the 16 rows of a b128 read group fall into 16 different chunk positions, and the 4 x 64-byte blocks of a
// transposing read spread over the banks as evenly as a 16-byte permutation allows.
template <int CPR>
__device__ __forceinline__ int la_swz(int row) {
  if constexpr (CPR == 4) return (row >> 2) & 3;
  else if constexpr (CPR == 8) return ((row << 1) & 4) | ((row >> 1) & 2) | ((row >> 3) & 1);
  else if constexpr (CPR == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return row & 15;
}
// row-major fragment: chunk c of `row`
template <typename E, int DK>
__device__ __forceinline__ uint4 la_frag(const E* img, int row, int c) {
  constexpr int CPR = DK / LOp<E>::CH;
  return *reinterpret_cast<const uint4*>(img + row * DK + (c ^ la_swz<CPR>(row)) * LOp<E>::CH);
}
// transposed fragment: column 32 n + (lane & 31) of the rows that registers [CH s, CH s + CH) of a 32 x 32 result stand for,
// rows counted from row0 of the image
template <typename E, int DK>
__device__ __forceinline__ uint4 la_tfrag(const E* img, int row0, int s, int n, int lane) {
  constexpr int CPR = DK / LOp<E>::CH;
  const int hw = lane >> 5;
  if constexpr (sizeof(E) == 4) {
    const int col = 32 * n + (lane & 31), ch = col >> 2, in = col & 3;
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = row0 + 8 * s + 4 * hw + e;
      r[e] = img[row * DK + ((ch ^ la_swz<CPR>(row)) << 2) + in];
    }
    return uint4{__float_as_uint(r[0]), __float_as_uint(r[1]), __float_as_uint(r[2]), __float_as_uint(r[3])};
  } else {
    // 16 lanes read 4 rows x 16 columns, 8 bytes each; lane i of them receives column i of the 4 rows
    const int ch = 4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), in = (lane & 1) * 4;
    const int ra = row0 + 16 * s + 4 * hw + ((lane & 15) >> 2), rb = ra + 8;
    typedef __attribute__((address_space(3))) s16x4* lp;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(img + ra * DK + ((ch ^ la_swz<CPR>(ra)) << 3) + in));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(img + rb * DK + ((ch ^ la_swz<CPR>(rb)) << 3) + in));
    const uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
    return uint4{x.x, x.y, y.x, y.y};
  }
}

// the same value, but not known to be: LDS addresses derived from it are computed where they are used instead of being kept in
// registers across a loop (the f32 kernels have none to spare, and their matrix instructions leave the vector unit idle)
__device__ __forceinline__ int la_opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// an address that is the same in all lanes, as the scalar it is
__device__ __forceinline__ const void* la_uniform(const void* p) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v), hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const void*)(uintptr_t)(lo | (hi << 32));
}

// A ROWS x DK image fetched by LDS-DMA, by WAVES waves, NI wave instructions each (lane offsets kept in registers; rows >= nrows and
// the channels that pad dk to DK come from the zero page, so nothing behind a sequence is ever read).
template <typename E, int DK, int ROWS = LA_TILE, int WAVES = LA_WAVES, bool KEEP = sizeof(E) == 2>
struct LTile {
  static constexpr int CH = LOp<E>::CH, CPR = DK / CH, NI = ROWS * CPR / 64 / WAVES;
  static_assert(ROWS * CPR % (64 * WAVES) == 0, "whole wave instructions");
  // element offsets inside the tile, -1: padding channels.  !KEEP: computed anew each time -- f32 (twice the instructions, short of
  // registers, its vector unit idle beside the matrix instructions) and the few-row backward
  int off[KEEP ? NI : 1], ld_, dk_;
  bool whole;  // no padding channels, and every byte offset of a tile fits 31 bits
  static __device__ __forceinline__ int offset(int i, int ld, int dk, int lane, int wave) {
    const int x = (wave * NI + i) * 64 + lane, row = x / CPR, c = (x % CPR) ^ la_swz<CPR>(row);
    return c * CH < dk ? row * ld + c * CH : -1;
  }
  __device__ __forceinline__ void init(int ld, int dk, int lane, int wave) {
    ld_ = ld;
    dk_ = dk;
    whole = dk == DK && ld < (1 << 22);
    if constexpr (KEEP) {
#pragma unroll
      for (int i = 0; i < NI; ++i) off[i] = offset(i, ld, dk, lane, wave);
    }
  }
  // whole tiles: one scalar address and the kept lane offsets, no vector work at all (forward of 2 x 6001 219 -> 201 us); the last tile of a
  // sequence: row by row
  __device__ __forceinline__ void issue(const E* tile, int nrows, const E* img, int lane, int wave) const {
    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_addr(img) + wave * (NI * 1024));
    if constexpr (KEEP) {
      if (whole && nrows >= ROWS) {
#pragma unroll
        for (int i = 0; i < NI; ++i) glds16_s(la_uniform(tile), (uint32_t)off[i] * (uint32_t)sizeof(E), dst + i * 1024);
        return;
      }
    }
    lane = la_opaque(lane);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int row = ((wave * NI + i) * 64 + lane) / CPR;
      int o;
      if constexpr (KEEP) o = off[i];
      else o = offset(i, ld_, dk_, lane, wave);
      const void* src = (o >= 0 && row < nrows) ? (const void*)(tile + o) : (const void*)g_conv_zero_page;
      glds16(src, dst + i * 1024);
    }
  }
};

// blocks of few rows: each of W waves streams its own 32-row chunks through its own two buffers (attention_long_fwd.hip)
template <typename E, int DK, int DV, int MAPS>
struct LSplit {
  static constexpr int STAGE = 32 * (MAPS * DK + DV);                     // elements of a chunk's images
  // Chunks of up to 16 KB: two buffers per wave.  f32 with wide heads, 32 KB: one buffer and four waves -- the matrix units of all four SIMDs
  // gain more than the fetch that two waves with two buffers would hide (4 x 333 of 2 x 128: forward 40 -> 23, dq 59 -> 39, dk / dv 83 -> 49 us)
  static constexpr int W = LA_WAVES, NB = STAGE * (int)sizeof(E) > 16384 ? 1 : 2;
  static constexpr int LDS = NB * W * STAGE * (int)sizeof(E);
};

// Blocks use up to 158 KB of dynamic LDS beside at most 2 KB of named arrays.  The limit is raised once per kernel and device: the runtime's
// call costs the host as much as a launch.
constexpr int LA_LDS = 158 * 1024;
inline bool la_lds_limit(const void* kern, size_t bytes, const char* who) {
  if (bytes <= 64 * 1024 || lds_limit_raised(kern)) return true;
  if (!ptpp_lds_limit(kern, LA_LDS, who)) return false;
  lds_limit_mark(kern);
  return true;
}

// every wave's LDS reads are done and every wave is here (the DMA queue is counted separately: glds_wait)
__device__ __forceinline__ void la_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float la_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// wave number, known to be the same in all lanes: what depends on it alone is scalar work and scalar branches
__device__ __forceinline__ int la_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// bucket of a distance d = key position - query position (Raffel et al. 2020: half of the buckets per direction, the first
// nexact distances one each, then logarithmic steps up to max_distance; the steps' first distances come from the host as whole
// numbers, so no logarithm is rounded here)
__device__ __forceinline__ int la_bucket(const LongP& p, int d) {
  const int n = p.bidirectional ? abs(d) : max(-d, 0);
  int b = n;
  if (n >= p.nexact) {
    b = p.nexact;
    for (int t = 0; t < p.nedges; ++t) b += n >= p.edges[t];
  }
  return b + (p.bidirectional && d > 0 ? p.nbuckets / 2 : 0);
}
// bias of every distance in [-D - PAD, D + PAD] of head h, times log2(e); distances outside [-D, D] share the outermost buckets
__device__ __forceinline__ int la_btab_len(const LongP& p) { return 2 * (p.max_distance + LA_PAD) + 1; }
__device__ __forceinline__ void la_fill_btab(const LongP& p, float* bt, int h) {
  const int D = p.max_distance, n = la_btab_len(p);
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int d = min(max(i - D - LA_PAD, -D), D);
    bt[i] = p.table[(int64_t)la_bucket(p, d) * p.H + h] * LA_LOG2E;
  }
}

// block -> (tile, pair), a pair being one (utterance, head) with `tiles` blocks; `pairs` of them.  Tiles of a pair run on one XCD (they share
// keys and values in its L2), and an XCD gets every 8th pair: lengths differ from utterance to utterance, and consecutive pairs are one
// utterance's heads -- with contiguous ranges of pairs the XCD of the longest utterance ran on alone (training of 8 x 1317-2000 differential
// 600 us that way, 545 us this way).
__device__ __forceinline__ void la_block(int tiles, int pairs, int& tile, int& pair) {
  const int t = xcd_remap(blockIdx.x, gridDim.x), pos = t / tiles;
  tile = t - pos * tiles;
  const int q = pairs >> 3, rem = pairs & 7, big = rem * (q + 1);
  pair = pos < big ? pos / (q + 1) + 8 * (pos % (q + 1)) : rem + (pos - big) / max(q, 1) + 8 * ((pos - big) % max(q, 1));
}

// lam of head h (every lane of a wave calls it, all with the same h: lane c takes channel c of that head's vectors; dk <= 64)
__device__ __forceinline__ void la_lambda_parts(const LongP& p, int h, int lane, float& e1, float& e2) {
  const int hh = p.lam_heads > 1 ? h : 0;
  float a = 0.f, b = 0.f;
  if (lane < p.dk) {
    const int64_t n = (int64_t)p.lam_heads * p.dk, o = (int64_t)hh * p.dk + lane;
    a = p.lam[o] * p.lam[n + o];
    b = p.lam[2 * n + o] * p.lam[3 * n + o];
  }
  e1 = expf(wave_sum(a));
  e2 = expf(wave_sum(b));
}
__device__ __forceinline__ float la_lambda(const LongP& p, int h, int lane) {
  float e1, e2;
  la_lambda_parts(p, h, lane, e1, e2);
  return e1 - e2 + p.lam_init;
}

__device__ __forceinline__ int la_klen(const LongP& p, int b) { return p.k_lengths ? min(max(p.k_lengths[b], 0), p.Tk) : p.Tk; }
__device__ __forceinline__ int la_qlen(const LongP& p, int b) { return p.q_lengths ? min(max(p.q_lengths[b], 0), p.Tq) : p.Tq; }
// Blocks of the longest utterance first: utterance in place `slot` of their order by `lengths`.  The rule: more blocks than CUs (one round
// gains nothing and pays about 1.5 us), and at most 64 utterances, one per lane (every wave sorts them anew, some 200 instructions; larger
// batches have many blocks per CU in any order).  dq and dk, dv of 24 x 761-1250 frames 81 -> 78 and 130 -> 122 us, of 8 x 1317-2000
// differential 140 -> 132 and 272 -> 265 us.
__device__ __forceinline__ int la_longest(const LongP& p, const int* lengths, int slot, int lane) {
  if (!lengths || p.B > 64 || gridDim.x <= 256) return slot;
  const int n = lane < p.B ? lengths[lane] : INT_MIN;
  int rank = 0;
  for (int j = 0; j < p.B; ++j) {
    const int o = __builtin_amdgcn_readlane(n, j);
    rank += o > n || (o == n && j < lane);
  }
  return __builtin_ctzll(__ballot(lane < p.B && rank == slot));
}
// position of query 0; held to +-2^30 so that no distance leaves 32 bits
__device__ __forceinline__ int la_qstart(const LongP& p, int b) {
  return p.q_start ? min(max(p.q_start[b], -(1 << 30)), 1 << 30) : 0;
}

}  // namespace

// host side: blocks of 32 rows (their four waves share the streamed side) instead of 128, up to which number of them.  Two rounds of the chip
// where a block's buffers take a CU but its waves four times as long per row (f32), or where two blocks fit a CU (heads of up to 64
// channels in all maps); one round for wide 16-bit heads.  128 -> 32 rows, forward / dq / dk, dv, us:
//   16-bit, 64 channels:     384 blocks (6 x 512)  17 -> 12 / 21 -> 16 / 32 -> 34, 512 (4 x 1024) 25 -> 16 / 31 -> 23 / 49 -> 48,
//                            768 (12 x 512) 17 -> 18 / 21 -> 25 / 33 -> 50
//   f32, 64 channels:        512 (8 x 512) 56 -> 43 / 71 -> 55 / 98 -> 70, 768 (12 x 512) 57 -> 63 / 73 -> 81 / 100 -> 105
//   f32, 128 channels:       512 (4 x 1024) 175 -> 129 / 246 -> 164 / 330 -> 209
//   16-bit, 128 channels:    256 (4 x 512) 19 -> 13 / 27 -> 19 / 41 -> 24, 384 (6 x 512) 20 -> 22 / 28 -> 33 / 42 -> 46
static inline int64_t la_few_blocks(int dtype, int maps, int dk) { return dtype == PTPP_F32 || maps * dk <= 64 ? 512 : 256; }

// host side (attention_long_fwd.hip): argument checks shared by both directions; fills the kernel parameters
int ptpp_attention_long_params(const ptpp_attention_long_args* a, int backward, LongP* out, const char* who);
