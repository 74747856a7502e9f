// Forward of the attention kernels for long sequences (mathematics and layout: attention_long.h), and the argument checks of
// both directions.
#include <stdlib.h>

#include "attention_long.h"

namespace {

// ---- the softmax of one 32 x 32 patch of scores, a lane = one query and 16 of the keys -----------------------------------
// No running maximum yet: far below every score that a matrix instruction of finite operands gives, and still a finite reference.  A table entry
// of -1e30 (-1.44e30 in base 2) stays below it for good: it hides its keys
constexpr float LA_NONE = -1.0e30f;
// The reference is raised only when a score passes it by more than this (base 2): probabilities up to 2^6 are as exact in every
// element type, and the rescaling of the context -- as many operations as there are scores -- almost never happens (with two waves per
// SIMD instead of one, 2 x 6001 of 8 x 64: 305 -> 206 us).
constexpr float LA_RAISE = 6.f;

// scores in base 2 are s * mul + add afterwards.  Patches with a distance inside (-max_distance, max_distance) read the bias of every pair
// (bt: the table at the lane's query and first key), the others share one value: no operation per element.
template <bool BIAS>
__device__ __forceinline__ void la_scores(f32x16& s, float c2, const float* bt, const float* table, int D, int dmin, int dmax, float& mul, float& add) {
  mul = c2;
  add = 0.f;
  if constexpr (BIAS) {
    if (dmin < D && dmax > -D) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, bt[8 * (r >> 2) + (r & 3)]);
      mul = 1.f;
    } else {
      add = table[dmin >= D ? 2 * (D + LA_PAD) : 0];
    }
  }
}
__device__ __forceinline__ void la_mask(f32x16& s, int jend) {  // keys from jend on (counted from the lane's first) are not seen
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) < jend ? s[r] : -INFINITY;
}
__device__ __forceinline__ float la_max16(const f32x16& s) {
  float m = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
  return m;
}
template <int NT>
__device__ __forceinline__ void la_raise(float& mx, float& l, f32x16 (&o)[NT], float tm) {
  if (!__any(tm > mx + LA_RAISE)) return;
  const float mn = fmaxf(mx, tm), al = la_exp2(mx - mn);
  mx = mn;
  l *= al;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[n][r] *= al;
}
// s -> 2^(s * mul + add), and their sum
__device__ __forceinline__ float la_probs(f32x16& s, float mul, float add) {
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int r = 0; r < 16; r += 2) {
    s[r] = la_exp2(fmaf(s[r], mul, add));
    s[r + 1] = la_exp2(fmaf(s[r + 1], mul, add));
    a += s[r];
    b += s[r + 1];
  }
  return a + b;
}

// One block = 128 query rows of one (utterance, head), a wave = 32 of them; keys and values stream through LDS in tiles of 64,
// the next tile's LDS-DMA under the current tile's products.  Bound by the vector unit: about 120 instructions and 16 exponentials (a quarter
// of the rate) per 32 x 32 patch of 64 channels, 617 cycles against 256 of matrix work.  In calls back to
// back 2 x 6001 of 8 x 64 f16 210 us, 700 TFLOP/s; 24 x 761-1250 of 4 x 64 bf16 62 us (800 blocks on 768 places); 8 x 1317-2000
// differential 117 us.
template <typename E, int DK, int DV, int MAPS, bool BIAS>
__global__ __launch_bounds__(256, sizeof(E) == 4 ? 1 : 2) void attn_long_fwd_kernel(const LongP p) {
  constexpr int CH = LOp<E>::CH, KS = DK / (2 * CH), PS = 16 / CH, NT = DV / 32;
  constexpr int KSUB = sizeof(E) == 4 || MAPS * DV == 256 ? 1 : 2;  // 32-key patches taken at once (as registers allow)
  constexpr bool TIGHT = sizeof(E) == 4 || MAPS * DV == 256;  // registers are short: LDS addresses and fragments not far ahead of use
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int KIMG = LA_TILE * DK, VIMG = LA_TILE * DV, BUF = MAPS * KIMG + VIMG;
  E* const img = reinterpret_cast<E*>(smem);
  float* const btab = reinterpret_cast<float*>(smem + 2 * BUF * sizeof(E));
  const int lane = threadIdx.x & 63, wave = la_wave(), lq = lane & 31, hw = lane >> 5;

  int qt, bh;
  la_block(p.nqt, p.B * p.H, qt, bh);
  if (p.causal) qt = p.nqt - 1 - qt;  // (the longest rows first)
  const int h = bh % p.H, b = la_longest(p, p.k_lengths, bh / p.H, lane), hk = h / (p.H / p.Hk);
  const int klen = la_klen(p, b), qlen = la_qlen(p, b), qs = la_qstart(p, b);
  const int ib = qt * (LA_OWN * LA_WAVES), i0 = ib + wave * LA_OWN, iq = i0 + lq;
  const int dv = MAPS * p.dk;

  int kend = ib < qlen ? klen : 0;  // keys that any row of the block may see
  if (p.causal) kend = min(kend, max(0, qs + min(ib + LA_OWN * LA_WAVES, qlen)));
  const int nt = (kend + LA_TILE - 1) / LA_TILE;

  const E* kb = reinterpret_cast<const E*>(p.k) + b * p.sk + (int64_t)hk * MAPS * p.dk;
  const E* vb = reinterpret_cast<const E*>(p.v) + b * p.sv + (int64_t)hk * dv;
  LTile<E, DK> kt;
  LTile<E, DV> vt;
  kt.init(p.ldk, p.dk, lane, wave);
  vt.init(p.ldv, dv, lane, wave);
  constexpr int NDMA = MAPS * LTile<E, DK>::NI + LTile<E, DV>::NI;
  auto issue = [&](int tile, int buf) {
    const int j0 = tile * LA_TILE;
    E* d = img + buf * BUF;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) kt.issue(kb + (int64_t)j0 * p.ldk + m * p.dk, kend - j0, d + m * KIMG, lane, wave);
    vt.issue(vb + (int64_t)j0 * p.ldv, kend - j0, d + MAPS * KIMG, lane, wave);
  };
  if (nt > 0) issue(0, 0);
  if constexpr (BIAS) la_fill_btab(p, btab, h);

  // the wave's queries: lane (query lq, chunk 2 s + hw)
  uint4 qf[MAPS][KS];
  {
    const E* qb = reinterpret_cast<const E*>(p.q) + b * p.sq + (int64_t)h * MAPS * p.dk + (int64_t)iq * p.ldq;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = (2 * s + hw) * CH;
        qf[m][s] = (iq < qlen && c < p.dk) ? *reinterpret_cast<const uint4*>(qb + m * p.dk + c) : uint4{0, 0, 0, 0};
      }
  }
  f32x16 o[MAPS][NT];
  float mx[MAPS], l[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    mx[m] = LA_NONE;
    l[m] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[m][n] = f32x16{};
  }
  const float c2 = p.scale * LA_LOG2E;
  const int q0 = qs + i0;  // position of the wave's first query
  const int D = p.max_distance;

  for (int tile = 0; tile < nt; ++tile) {
    const int buf = tile & 1;
    if (tile + 1 < nt) {
      issue(tile + 1, buf ^ 1);
      glds_wait<NDMA>();
    } else {
      glds_wait<0>();
    }
    la_barrier();
    const E* kimg = img + buf * BUF;
    const E* vimg = kimg + MAPS * KIMG;
#pragma unroll 1
    for (int sub = 0; sub < 2 / KSUB; ++sub) {
      uint4 pf[MAPS][KSUB][PS];
      const int ln = TIGHT ? la_opaque(lane) : lane, lr = ln & 31, hr = ln >> 5;
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        f32x16 s[KSUB];
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
          s[ks] = f32x16{};
#pragma unroll
          for (int kk = 0; kk < KS; ++kk)
            s[ks] = LOp<E>::mma(la_frag<E, DK>(kimg + m * KIMG, 32 * (sub * KSUB + ks) + lr, 2 * kk + hr), qf[m][kk], s[ks]);
        }
        float tm = -INFINITY, mul[KSUB], add[KSUB];
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
          const int j0 = tile * LA_TILE + 32 * (sub * KSUB + ks);
          const float* bt = btab + (j0 - q0 - lq + 4 * hw + D + LA_PAD);
          la_scores<BIAS>(s[ks], c2, bt, btab, D, j0 - (q0 + 31), j0 + 31 - q0, mul[ks], add[ks]);
          if (j0 + 32 > kend || (p.causal && j0 + 31 > q0)) la_mask(s[ks], min(klen, p.causal ? q0 + lq + 1 : klen) - j0 - 4 * hw);
          tm = fmaxf(tm, fmaf(la_max16(s[ks]), mul[ks], add[ks]));
        }
        la_raise<NT>(mx[m], l[m], o[m], la_half_max(tm));
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
          l[m] += la_probs(s[ks], mul[ks], add[ks] - mx[m]);
#pragma unroll
          for (int st = 0; st < PS; ++st) pf[m][ks][st] = la_pack<E>(s[ks], st);
        }
      }
#pragma unroll
      for (int ks = 0; ks < KSUB; ++ks)
#pragma unroll
        for (int st = 0; st < PS; ++st)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 vf = la_tfrag<E, DV>(vimg, 32 * (sub * KSUB + ks), st, n, ln);
#pragma unroll
            for (int m = 0; m < MAPS; ++m) o[m][n] = LOp<E>::mma(vf, pf[m][ks][st], o[m][n]);
            if (TIGHT && n % 2 == 1) __builtin_amdgcn_sched_barrier(0);
          }
    }
    la_barrier();
  }

  // ---- epilogue: lane (query lq) holds channels 32 n + 8 g + 4 hw + (0..3) ----
  float inv[MAPS];
  bool on[MAPS];  // a row that is none, or sees no key, gives zeros by selection: its sums may hold NaN from infinite keys or values
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    l[m] = la_half_sum(l[m]);
    on[m] = iq < qlen && !(l[m] == 0.f);  // (a NaN sum passes: it belongs in the output)
    inv[m] = 1.f / l[m];
    if (p.lse && hw == 0 && iq < p.TqP)
      p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] = on[m] ? mx[m] + log2f(l[m]) : INFINITY;
  }
  float lam = 0.f;
  if constexpr (MAPS == 2) lam = la_lambda(p, h, lane);
  if (iq >= p.Tq) return;
  E* ob = reinterpret_cast<E*>(p.out) + b * p.so + (int64_t)iq * p.ldo + (int64_t)h * dv;
  E* o2 = MAPS == 2 && p.out2 ? reinterpret_cast<E*>(p.out2) + ((int64_t)b * p.Tq + iq) * ((int64_t)p.H * dv) + (int64_t)h * dv : nullptr;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * n + 8 * g + 4 * hw;
      if (c < dv) {
        float v[4], w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = on[0] ? o[0][n][4 * g + e] * inv[0] : 0.f;
          w[e] = on[MAPS - 1] ? o[MAPS - 1][n][4 * g + e] * inv[MAPS - 1] : 0.f;
          if constexpr (MAPS == 2) v[e] = fmaf(-lam, w[e], v[e]);
        }
        la_store4<E>(ob + c, v[0], v[1], v[2], v[3]);
        if constexpr (MAPS == 2) {
          if (o2) la_store4<E>(o2 + c, w[0], w[1], w[2], w[3]);
        }
      }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Few query rows or few tiles: one block = 32 columns -- 32 queries of one head, or all queries of several heads that share their
// keys (a step of one query: Tq = 1) -- and one of `splits` ranges of the keys; its W waves take 32-key chunks of the range in turn,
// each streaming its own chunks through its own two LDS buffers (no block barrier in the loop), and join at the end.  With more
// than one range the blocks leave unnormalised sums and (max, sum) for the join kernel.  A step is HBM-bound: every key and value is
// read once, two chunks per wave on their way (one query on 16 x 4001, differential f16: 51 us with one chunk ahead, 47 us with two;
// on 32 x 8191 of 12 heads on 4 x 64 bf16: 40 us, 5.4 TB/s).
template <typename E, int DK, int DV, int MAPS, bool BIAS, bool REST>
__global__ __launch_bounds__((LSplit<E, DK, DV, MAPS>::W * 64), sizeof(E) == 4 || MAPS * DV == 256 ? 1 : 2) void attn_long_split_kernel(const LongP p) {
  typedef LSplit<E, DK, DV, MAPS> S_;
  constexpr int W = S_::W, NB = S_::NB, STAGE = S_::STAGE, KIMG = 32 * DK;
  // REST: 16-bit probabilities as two operands, the rounded value and what the rounding took: the matrix units wait for memory here, and the
  // context has the accuracy of f32 probabilities (against 64 bits one f16 query on 4001 keys, differential: 3.1e-4 -> 2.1e-4, the output's
  // own rounding) for 50.5 instead of 46.8 us, 40.2 instead of 39.3 us for one bf16 query on 8191 keys.  Not where backward follows, which
  // rounds the same probabilities once.
  constexpr bool TIGHT = sizeof(E) == 4 || MAPS * DV == 256;
  constexpr int CH = LOp<E>::CH, KS = DK / (2 * CH), PS = 16 / CH, NT = DV / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float wml[W][MAPS][2][32];
  const int lane = threadIdx.x & 63, wave = la_wave(), lq = lane & 31, hw = lane >> 5;
  float* const btab = reinterpret_cast<float*>(smem + S_::LDS);
  E* const img = reinterpret_cast<E*>(smem) + wave * NB * STAGE;

  // block -> (range, utterance, key head, head group, row block); ranges of one key head run on the same XCD
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int sp = t % p.splits, tl = t / p.splits;  // tl: number of the 32-column block
  const int rb = tl % p.nrb, G = p.H / p.Hk, hg = (tl / p.nrb) % (G / p.nh), bk = tl / (p.nrb * (G / p.nh));
  const int hk = bk % p.Hk, b = bk / p.Hk, h0 = hk * G + hg * p.nh;
  const int klen = la_klen(p, b), qlen = la_qlen(p, b), qs = la_qstart(p, b);
  const int dv = MAPS * p.dk;

  // the lane's column: query iq of head h
  const int hcol = p.nh > 1 ? min(lq / p.Tq, p.nh - 1) : 0, h = h0 + hcol;
  const int i0 = rb * 32, iq = p.nh > 1 ? (lq < p.nh * p.Tq ? lq % p.Tq : p.Tq) : i0 + lq;  // (Tq: no query)
  const int ilo = i0, ihi = p.nh > 1 ? p.Tq - 1 : i0 + 31;
  int kend = ilo < qlen ? klen : 0;
  if (p.causal) kend = min(kend, max(0, qs + min(ihi + 1, qlen)));
  const int nc = (kend + 31) >> 5, per = (nc + p.splits - 1) / p.splits;
  const int c0 = sp * per, c1 = min(nc, c0 + per);

  const E* kb = reinterpret_cast<const E*>(p.k) + b * p.sk + (int64_t)hk * MAPS * p.dk;
  const E* vb = reinterpret_cast<const E*>(p.v) + b * p.sv + (int64_t)hk * dv;
  LTile<E, DK, 32, 1> kt;
  LTile<E, DV, 32, 1> vt;
  kt.init(p.ldk, p.dk, lane, 0);
  vt.init(p.ldv, dv, lane, 0);
  constexpr int NK = MAPS * LTile<E, DK, 32, 1>::NI, NV = LTile<E, DV, 32, 1>::NI;
  auto issue_k = [&](int c, int buf) {
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
      kt.issue(kb + (int64_t)(32 * c) * p.ldk + m * p.dk, kend - 32 * c, img + buf * STAGE + m * KIMG, lane, 0);
  };
  auto issue_v = [&](int c, int buf) { vt.issue(vb + (int64_t)(32 * c) * p.ldv, kend - 32 * c, img + buf * STAGE + MAPS * KIMG, lane, 0); };
  int c = c0 + wave;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (NB == 2 && c + i * W < c1) {
      issue_k(c + i * W, i);
      issue_v(c + i * W, i);
    }
  const int dist_n = la_btab_len(p);
  if constexpr (BIAS)
    for (int n = 0; n < p.nh; ++n) la_fill_btab(p, btab + n * dist_n, h0 + n);

  uint4 qf[MAPS][KS];
  {
    const E* qb = reinterpret_cast<const E*>(p.q) + b * p.sq + (int64_t)h * MAPS * p.dk + (int64_t)iq * p.ldq;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int ch = (2 * s + hw) * CH;
        qf[m][s] = (iq < qlen && ch < p.dk) ? *reinterpret_cast<const uint4*>(qb + m * p.dk + ch) : uint4{0, 0, 0, 0};
      }
  }
  f32x16 o[MAPS][NT];
  float mx[MAPS], l[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    mx[m] = LA_NONE;
    l[m] = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) o[m][n] = f32x16{};
  }
  const float c2 = p.scale * LA_LOG2E;
  const int D = p.max_distance, qp = qs + min(iq, ihi);  // (a column without a query reads the table within bounds)
  if constexpr (BIAS) la_barrier();

  // Two chunks are on their way ahead of the one in hand: the keys' half of a buffer is refilled as soon as the scores are computed, the
  // values' half after the second product.  The waits count what was asked for later (in order: V, K', V', K'').
  for (int buf = 0; c < c1; c += W, buf ^= NB - 1) {
    const bool one = c + W < c1, two = c + 2 * W < c1;
    if (NB == 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer's last reads are done
      issue_k(c, 0);
      issue_v(c, 0);
      glds_wait<NV>();
    } else if (one) {
      glds_wait<NK + 2 * NV>();
    } else {
      glds_wait<NV>();
    }
    const E* kimg = img + buf * STAGE;
    const E* vimg = kimg + MAPS * KIMG;
    const int j0 = 32 * c;
    const int ln = TIGHT ? la_opaque(lane) : lane, lr = ln & 31, hr = ln >> 5;
    uint4 pf[MAPS][PS], pr[REST ? MAPS : 1][REST ? PS : 1];
    f32x16 s[MAPS];
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      s[m] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        s[m] = LOp<E>::mma(la_frag<E, DK>(kimg + m * KIMG, lr, 2 * kk + hr), qf[m][kk], s[m]);
        if (TIGHT && kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (NB == 2 && two) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the keys' last reads are done
      issue_k(c + 2 * W, buf);
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      float mul, add;
      const float* bt0 = btab + hcol * dist_n;
      la_scores<BIAS>(s[m], c2, bt0 + (j0 - qp + 4 * hw + D + LA_PAD), bt0, D, j0 - (qs + ihi), j0 + 31 - (qs + ilo), mul, add);
      if (j0 + 32 > kend || (p.causal && j0 + 31 > qs + ilo)) la_mask(s[m], min(klen, p.causal ? qp + 1 : klen) - j0 - 4 * hw);
      la_raise<NT>(mx[m], l[m], o[m], la_half_max(fmaf(la_max16(s[m]), mul, add)));
      l[m] += la_probs(s[m], mul, add - mx[m]);
#pragma unroll
      for (int st = 0; st < PS; ++st) {
        pf[m][st] = la_pack<E>(s[m], st);
        if constexpr (REST) pr[m][st] = la_pack_rest<E>(s[m], st, pf[m][st]);
      }
    }
    if (NB == 2 && two) glds_wait<2 * NK + NV>();
    else if (NB == 2 && one) glds_wait<NK + NV>();
    else glds_wait<0>();
#pragma unroll
    for (int st = 0; st < PS; ++st)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 vf = la_tfrag<E, DV>(vimg, 0, st, n, ln);
#pragma unroll
        for (int m = 0; m < MAPS; ++m) o[m][n] = LOp<E>::mma(vf, pf[m][st], o[m][n]);
        if constexpr (REST) {
#pragma unroll
          for (int m = 0; m < MAPS; ++m) o[m][n] = LOp<E>::mma(vf, pr[m][st], o[m][n]);
        }
        if (TIGHT && (!REST || n % 2 == 1)) __builtin_amdgcn_sched_barrier(0);
      }
    if (NB == 2 && two) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the values' last reads are done
      issue_v(c + 2 * W, buf);
    }
  }

  // ---- join the waves: common maximum, then each wave's sums through its own buffers ----
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    l[m] = la_half_sum(l[m]);
    if (hw == 0) {
      wml[wave][m][0][lq] = mx[m];
      wml[wave][m][1][lq] = l[m];
    }
  }
  la_barrier();
  float M[MAPS], L[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    M[m] = LA_NONE;
#pragma unroll
    for (int w = 0; w < W; ++w) M[m] = fmaxf(M[m], wml[w][m][0][lq]);
    L[m] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) L[m] = fmaf(wml[w][m][1][lq], la_exp2(wml[w][m][0][lq] - M[m]), L[m]);
    const float al = la_exp2(mx[m] - M[m]);
    float* mine = reinterpret_cast<float*>(img) + m * NT * 1024 + lane;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[(n * 16 + r) * 64] = o[m][n][r] * al;
  }
  static_assert(MAPS * NT * 1024 * 4 <= NB * STAGE * (int)sizeof(E), "a wave's sums fit its buffers");
  la_barrier();
  const bool row = iq < p.Tq;
  float lam = 0.f;
  if constexpr (MAPS == 2) {
    if (p.splits == 1)  // (with more ranges the join applies it)
      for (int n = 0; n < (p.lam_heads > 1 ? p.nh : 1); ++n) {  // one head after the other: a whole wave computes one value
        const float l = la_lambda(p, h0 + n, lane);
        if (p.lam_heads == 1 || n == hcol) lam = l;
      }
  }
  float inv[MAPS];
  bool on[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    on[m] = iq < qlen && !(L[m] == 0.f);
    inv[m] = 1.f / L[m];
    if (wave == 0 && hw == 0) {
      if (p.splits > 1) {
        if (row) {
          float* ml = p.part_ml + ((((int64_t)tl * p.splits + sp) * MAPS + m) * 32 + lq) * 2;
          ml[0] = M[m];
          ml[1] = L[m];
        }
      } else if (p.lse && iq < p.TqP) {
        p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] = on[m] ? M[m] + log2f(L[m]) : INFINITY;
      }
    }
  }
  const float* all = reinterpret_cast<const float*>(smem) + lane;
  for (int ng = wave; ng < NT * 4; ng += W) {  // registers 4 g .. 4 g + 3 of channel block n: channels 32 n + 8 g + 4 hw + (0..3)
    const int ch = 32 * (ng >> 2) + 8 * (ng & 3) + 4 * hw;
    float v[MAPS][4];
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[m][e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[m][e] += all[w * (NB * STAGE * (int)sizeof(E) / 4) + (m * NT * 16 + ng * 4 + e) * 64];
      }
    if (!row || ch >= dv) continue;
    if (p.splits > 1) {
#pragma unroll
      for (int m = 0; m < MAPS; ++m)
        *reinterpret_cast<f32x4*>(p.part_o + ((((int64_t)tl * p.splits + sp) * MAPS + m) * 32 + lq) * DV + ch) = f32x4{v[m][0], v[m][1], v[m][2], v[m][3]};
    } else {
      E* ob = reinterpret_cast<E*>(p.out) + b * p.so + (int64_t)iq * p.ldo + (int64_t)h * dv + ch;
      float r[4], w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r[e] = on[0] ? v[0][e] * inv[0] : 0.f;
        w[e] = on[MAPS - 1] ? v[MAPS - 1][e] * inv[MAPS - 1] : 0.f;
        if constexpr (MAPS == 2) r[e] = fmaf(-lam, w[e], r[e]);
      }
      la_store4<E>(ob, r[0], r[1], r[2], r[3]);
      if constexpr (MAPS == 2) {
        if (p.out2)
          la_store4<E>(reinterpret_cast<E*>(p.out2) + ((int64_t)b * p.Tq + iq) * ((int64_t)p.H * dv) + (int64_t)h * dv + ch, w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// columns of a block that the join has to look at: its queries (with statistics also the rows that pad them)
__host__ __device__ __forceinline__ int join_cols(const LongP& p) { return p.nh > 1 ? p.nh * p.Tq : p.nrb > 1 || p.lse ? 32 : min(p.Tq, 32); }
// join of the key ranges: one wave per (block, column).  Latency: 4.7 us for 384 columns in 4 ranges, 7 us for 128 of two maps in 16
template <typename E, int DV, int MAPS>
__global__ __launch_bounds__(256) void attn_long_join_kernel(const LongP p, int ncol) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * LA_WAVES + la_wave();
  const int G = p.H / p.Hk, cols = join_cols(p);
  if (w >= (int64_t)ncol) return;
  const int tl = (int)(w / cols), lq = (int)(w % cols);
  const int rb = tl % p.nrb, hg = (tl / p.nrb) % (G / p.nh), bk = tl / (p.nrb * (G / p.nh));
  const int hk = bk % p.Hk, b = bk / p.Hk, h = hk * G + hg * p.nh + (p.nh > 1 ? lq / p.Tq : 0);
  const int iq = p.nh > 1 ? lq % p.Tq : rb * 32 + lq, dv = MAPS * p.dk;
  float lam = 0.f;
  if constexpr (MAPS == 2) lam = la_lambda(p, h, lane);
  constexpr int NC = DV / 64;  // channels per lane
  float r[MAPS][NC];
  const bool row = iq < p.Tq;
  const bool on = iq < la_qlen(p, b);
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const int64_t base = (((int64_t)tl * p.splits) * MAPS + m) * 32 + lq, step = MAPS * 32;
    float mm = LA_NONE, ll = 0.f;
    if (row && lane < p.splits) {  // (splits <= 64)
      mm = p.part_ml[(base + lane * step) * 2];
      ll = p.part_ml[(base + lane * step) * 2 + 1];
    }
    float M = mm;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float f = la_exp2(mm - M);
    const float L = wave_sum(f * ll);
    const bool ok = on && !(L == 0.f);
#pragma unroll
    for (int n = 0; n < NC; ++n) r[m][n] = 0.f;
    if (row)
      for (int s = 0; s < p.splits; ++s) {
        const float fs = __shfl(f, s, 64);
#pragma unroll
        for (int n = 0; n < NC; ++n)
          if (lane + 64 * n < dv) r[m][n] = fmaf(p.part_o[(base + s * step) * DV + lane + 64 * n], fs, r[m][n]);
      }
#pragma unroll
    for (int n = 0; n < NC; ++n) r[m][n] = ok ? r[m][n] * (1.f / L) : 0.f;
    if (p.lse && lane == 0 && iq < p.TqP) p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] = ok ? M + log2f(L) : INFINITY;
  }
  if (!row) return;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int ch = lane + 64 * n;
    if (ch >= dv) continue;
    float v = r[0][n];
    if constexpr (MAPS == 2) {
      v = fmaf(-lam, r[MAPS - 1][n], v);
      if (p.out2) Elem<E>::st(reinterpret_cast<E*>(p.out2) + ((int64_t)b * p.Tq + iq) * ((int64_t)p.H * dv) + (int64_t)h * dv + ch, r[MAPS - 1][n]);
    }
    Elem<E>::st(reinterpret_cast<E*>(p.out) + b * p.so + (int64_t)iq * p.ldo + (int64_t)h * dv + ch, v);
  }
}

// The rule: blocks of 128 rows, unless there are at most 32 rows, or few blocks (la_few_blocks); then as many key ranges as fill the chip
// once -- one or two blocks per CU, as their buffers fit -- at no fewer than four 32-key chunks per wave (f32: two), which is what the join
// of many rows costs: 4 x 512 rows of 4 x 64 channels 10.1 us in one range, 10.5 + 7 us in two; one query against 8000 keys of 8 x 64
// channels 16.3 us this way, 19.3 us from two chunks on.
bool few_rows(const LongP& p, int dtype, int maps) {
  return p.Tq <= 32 || (int64_t)((p.Tq + 31) / 32) * p.B * p.H <= la_few_blocks(dtype, maps, p.dk);
}
// fills nh, nrb, splits; returns the number of 32-column blocks (0: too many to number)
int plan_few(LongP& p, int lds, int dtype) {
  const int G = p.H / p.Hk;
  p.nh = 1;
  if (!p.lse)  // (backward's statistics are padded to whole blocks of one head's rows)
    for (int n = 2; n <= G && n * p.Tq <= 32; ++n)
      if (G % n == 0 && (!p.table || n * (2 * (p.max_distance + LA_PAD) + 1) <= 6144)) p.nh = n;  // (24 KB of bias tables)
  p.nrb = p.nh > 1 ? 1 : (p.lse ? p.TqP : p.Tq + 31) / 32;
  const int64_t blocks = (int64_t)p.B * p.Hk * (G / p.nh) * p.nrb;
  const int64_t range = (dtype == PTPP_F32 ? 2 : 4) * 32 * LA_WAVES, most = (p.Tk + range - 1) / range;
  int64_t s = blocks ? (lds > 72 * 1024 ? 256 : 512) / blocks : 1;  // (72 KB: two blocks per CU with their tables and statistics)
  if (s > most) s = most;
  p.splits = s < 1 ? 1 : s > 64 ? 64 : (int)s;
  return blocks * p.splits < (1ll << 24) ? (int)blocks : 0;  // (a launch holds fewer than 2^32 threads)
}
template <typename E>
int few_lds(int maps, int dk) {
  if (maps == 1) return dk <= 64 ? LSplit<E, 64, 64, 1>::LDS : LSplit<E, 128, 128, 1>::LDS;
  return dk <= 32 ? LSplit<E, 32, 64, 2>::LDS : LSplit<E, 64, 128, 2>::LDS;
}
int few_lds(int dtype, int maps, int dk) { return dtype == PTPP_F32 ? few_lds<float>(maps, dk) : few_lds<bf16_raw>(maps, dk); }  // (f16 as bf16)
int pad_dv(int maps, int dk) { return maps == 1 ? (dk <= 64 ? 64 : 128) : (dk <= 32 ? 64 : 128); }

template <typename E, int DK, int DV, int MAPS, bool BIAS, bool REST>
int launch_split(const LongP& p, unsigned blocks, size_t sm, hipStream_t st) {
  if (!la_lds_limit((const void*)attn_long_split_kernel<E, DK, DV, MAPS, BIAS, REST>, sm, "attention_long_fwd")) return PTPP_ELAUNCH;
  hipLaunchKernelGGL((attn_long_split_kernel<E, DK, DV, MAPS, BIAS, REST>), dim3(blocks), dim3(LSplit<E, DK, DV, MAPS>::W * 64), sm, st, p);
  PTPP_CHECK_LAUNCH("attention_long_fwd (few rows)");
  return PTPP_OK;
}
template <typename E, int DK, int DV, int MAPS, bool BIAS>
int launch_split(const LongP& p, unsigned blocks, size_t sm, hipStream_t st) {
  if constexpr (sizeof(E) == 2)
    if (!p.lse) return launch_split<E, DK, DV, MAPS, BIAS, true>(p, blocks, sm, st);
  return launch_split<E, DK, DV, MAPS, BIAS, false>(p, blocks, sm, st);
}
template <typename E, int DK, int DV, int MAPS>
int launch_fwd(const LongP& p, hipStream_t st) {
  const size_t tab = p.table ? (2 * (p.max_distance + LA_PAD) + 1) * sizeof(float) : 0;
  if (!p.splits) {
    const size_t sm = 2 * (size_t)LA_TILE * (MAPS * DK + DV) * sizeof(E) + tab;
    const dim3 g((unsigned)((int64_t)p.nqt * p.B * p.H));
    const void* kern = p.table ? (const void*)attn_long_fwd_kernel<E, DK, DV, MAPS, true> : (const void*)attn_long_fwd_kernel<E, DK, DV, MAPS, MAPS == 1>;
    if (!la_lds_limit(kern, sm, "attention_long_fwd")) return PTPP_ELAUNCH;
    if (p.table) hipLaunchKernelGGL((attn_long_fwd_kernel<E, DK, DV, MAPS, true>), g, dim3(256), sm, st, p);
    else if constexpr (MAPS == 2) hipLaunchKernelGGL((attn_long_fwd_kernel<E, DK, DV, MAPS, false>), g, dim3(256), sm, st, p);
    PTPP_CHECK_LAUNCH("attention_long_fwd");
    return PTPP_OK;
  }
  typedef LSplit<E, DK, DV, MAPS> S_;
  const size_t sm = S_::LDS + p.nh * tab;
  const int blocks = p.B * p.Hk * (p.H / p.Hk / p.nh) * p.nrb;
  int r = PTPP_OK;
  if (p.table) r = launch_split<E, DK, DV, MAPS, true>(p, (unsigned)(blocks * p.splits), sm, st);
  else if constexpr (MAPS == 2) r = launch_split<E, DK, DV, MAPS, false>(p, (unsigned)(blocks * p.splits), sm, st);
  if (r != PTPP_OK) return r;
  if (p.splits > 1) {
    const int ncol = blocks * join_cols(p);
    hipLaunchKernelGGL((attn_long_join_kernel<E, DV, MAPS>), dim3((ncol + LA_WAVES - 1) / LA_WAVES), dim3(256), 0, st, p, ncol);
    PTPP_CHECK_LAUNCH("attention_long_fwd (join)");
  }
  return PTPP_OK;
}
template <typename E>
int dispatch_fwd(const LongP& p, int maps, hipStream_t st) {
  if (maps == 1) return p.dk <= 64 ? launch_fwd<E, 64, 64, 1>(p, st) : launch_fwd<E, 128, 128, 1>(p, st);
  return p.dk <= 32 ? launch_fwd<E, 32, 64, 2>(p, st) : launch_fwd<E, 64, 128, 2>(p, st);
}

// forward plan: p.splits == 0: tiles.  -> bytes of workspace, < 0: refused
int64_t plan_fwd(LongP& p, const ptpp_attention_long_args* a, int64_t* o_ml, const char* who) {
  *o_ml = 0;
  if (!few_rows(p, a->dtype, a->maps)) return 0;
  const int blocks = plan_few(p, few_lds(a->dtype, a->maps, a->dk), a->dtype);
  if (!blocks) {
    ptpp_set_error("%s: too many tiles", who);
    return -1;
  }
  if (p.splits == 1) return 0;
  const int64_t rows = (int64_t)blocks * p.splits * a->maps * 32;
  *o_ml = rows * pad_dv(a->maps, a->dk);
  return (*o_ml + 2 * rows) * (int64_t)sizeof(float);
}

}  // namespace

int ptpp_attention_long_params(const ptpp_attention_long_args* a, int backward, LongP* o, const char* who) {
  PTPP_CHECK_ARG(a, "%s: null arguments", who);
  PTPP_CHECK_ARG(a->dtype == PTPP_F32 || a->dtype == PTPP_BF16 || a->dtype == PTPP_F16, "%s: bad dtype %d", who, a->dtype);
  PTPP_CHECK_ARG(a->maps == 1 || a->maps == 2, "%s: maps must be 1 or 2, not %d", who, a->maps);
  PTPP_CHECK_ARG(a->B > 0 && a->Tq > 0 && a->Tk > 0 && a->H > 0 && a->Hk > 0, "%s: empty shape (B %d, Tq %d, Tk %d, H %d, Hk %d)", who, a->B,
                 a->Tq, a->Tk, a->H, a->Hk);
  PTPP_CHECK_ARG(a->Tq <= (1 << 28) && a->Tk <= (1 << 28), "%s: sequences of at most 2^28 positions", who);
  PTPP_CHECK_ARG(a->H % a->Hk == 0, "%s: %d key heads do not divide %d query heads", who, a->Hk, a->H);
  PTPP_CHECK_ARG(a->dk > 0 && a->dk % 8 == 0 && a->dk <= (a->maps == 1 ? 128 : 64), "%s: head width %d (a multiple of 8, at most %d)", who, a->dk,
                 a->maps == 1 ? 128 : 64);
  PTPP_CHECK_ARG(a->scale > 0.f && a->scale < 1e30f, "%s: scale must be positive and finite", who);
  PTPP_CHECK_ARG(a->q && a->k && a->v && a->out, "%s: null tensor", who);
  const int es = a->dtype == PTPP_F32 ? 4 : 2, al = 16 / es;
  const int wq = a->H * a->maps * a->dk, wk = a->Hk * a->maps * a->dk;
  PTPP_CHECK_ARG((int64_t)a->H * a->maps * a->dk < (1 << 24), "%s: rows too wide", who);
  struct Row { const void* p; int64_t s; int ld, w, T; const char* n; };
  const Row rows[] = {{a->q, a->sq, a->ldq, wq, a->Tq, "q"},          {a->k, a->sk, a->ldk, wk, a->Tk, "k"},    {a->v, a->sv, a->ldv, wk, a->Tk, "v"},
                      {a->out, a->so, a->ldo, wq, a->Tq, "out"},      {a->dout, a->sdo, a->lddo, wq, a->Tq, "dout"},
                      {a->dq, a->sdq, a->lddq, wq, a->Tq, "dq"},      {a->dk_out, a->sdk, a->lddk, wk, a->Tk, "dk"},
                      {a->dv, a->sdv, a->lddv, wk, a->Tk, "dv"}};
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    const Row& r = rows[i];
    PTPP_CHECK_ARG(r.p, "%s: null %s", who, r.n);
    PTPP_CHECK_ARG((uintptr_t)r.p % 16 == 0 && r.ld % al == 0 && r.s % al == 0, "%s: %s is not 16-byte aligned (pointer, row stride %d, batch stride %lld)",
                   who, r.n, r.ld, (long long)r.s);
    PTPP_CHECK_ARG(r.ld >= r.w && r.ld < (1 << 24), "%s: row stride %d of %s (rows are %d wide)", who, r.ld, r.n, r.w);
    PTPP_CHECK_ARG(r.s >= 0, "%s: negative batch stride of %s", who, r.n);
  }
  PTPP_CHECK_ARG((uintptr_t)a->out2 % 16 == 0, "%s: the second map's context is not 16-byte aligned", who);  // (stored like out)
  const void* words[] = {a->table, a->lam, a->dtable, a->dlam, a->lse, a->k_lengths, a->q_lengths, a->q_start, a->edges};
  for (const void* w : words) PTPP_CHECK_ARG((uintptr_t)w % 4 == 0, "%s: tables, statistics and lengths must be 4-byte aligned", who);
  if (a->maps == 1) PTPP_CHECK_ARG(a->table, "%s: the bucketed form needs a table", who);
  if (a->maps == 2) {
    PTPP_CHECK_ARG(a->lam, "%s: null lam", who);
    PTPP_CHECK_ARG(a->lam_heads == 1 || a->lam_heads == a->H, "%s: lam for %d heads (1 or %d)", who, a->lam_heads, a->H);
  }
  *o = LongP{};
  if (a->table) {
    const int n = a->bidirectional ? a->nbuckets / 2 : a->nbuckets;
    PTPP_CHECK_ARG(a->nbuckets >= 2 && a->nbuckets <= 128 && (!a->bidirectional || a->nbuckets % 2 == 0) && n >= 2,
                   "%s: %d buckets (2 to 128 per table, two or more per direction)", who, a->nbuckets);
    PTPP_CHECK_ARG(a->nexact == n / 2 && a->nedges == n - n / 2 - 1 && a->nedges <= LA_EDGES && (a->edges || !a->nedges), "%s: bucket edges do not fit %d buckets",
                   who, a->nbuckets);
    PTPP_CHECK_ARG(a->max_distance > a->nexact && a->max_distance <= LA_MAXD, "%s: max_distance %d (more than %d, at most %d)", who, a->max_distance,
                   a->nexact, LA_MAXD);
    for (int t = 0; t < a->nedges; ++t) {
      PTPP_CHECK_ARG(a->edges[t] >= (t ? a->edges[t - 1] : a->nexact) && a->edges[t] <= a->max_distance, "%s: bucket edges are not ascending", who);
      o->edges[t] = a->edges[t];
    }
  }
  const int64_t nqt = ((int64_t)a->Tq + 127) / 128, nkt = ((int64_t)a->Tk + 127) / 128;
  // (a launch holds fewer than 2^32 threads: 2^24 blocks of 256)
  PTPP_CHECK_ARG(nqt * a->B * a->H < (1ll << 24) && nkt * a->B * a->Hk < (1ll << 24), "%s: too many tiles", who);
  o->q = a->q; o->k = a->k; o->v = a->v; o->dout = a->dout; o->out = a->out; o->out2 = a->out2; o->dq = a->dq;
  o->gk = a->dk_out; o->gv = a->dv;
  o->table = a->table; o->lam = a->lam; o->k_lengths = a->k_lengths; o->q_lengths = a->q_lengths; o->q_start = a->q_start;
  o->lse = a->lse;
  o->sq = a->sq; o->sk = a->sk; o->sv = a->sv; o->so = a->so; o->sdo = a->sdo; o->sdq = a->sdq; o->sdk = a->sdk; o->sdv = a->sdv;
  o->ldq = a->ldq; o->ldk = a->ldk; o->ldv = a->ldv; o->ldo = a->ldo; o->lddo = a->lddo; o->lddq = a->lddq; o->lddk = a->lddk; o->lddv = a->lddv;
  o->B = a->B; o->Tq = a->Tq; o->Tk = a->Tk; o->TqP = (a->Tq + 63) & ~63; o->H = a->H; o->Hk = a->Hk; o->dk = a->dk;
  o->nbuckets = a->nbuckets; o->bidirectional = a->bidirectional; o->causal = a->causal; o->lam_heads = a->lam_heads;
  o->max_distance = a->max_distance; o->nexact = a->nexact; o->nedges = a->nedges;
  o->nqt = (int)nqt; o->nkt = (int)nkt;
  o->scale = a->scale; o->lam_init = a->lam_init;
  return PTPP_OK;
}

extern "C" int ptpp_attention_long_fwd(const ptpp_attention_long_args* a, void* stream) {
  LongP p;
  const int rc = ptpp_attention_long_params(a, 0, &p, "attention_long_fwd");
  if (rc != PTPP_OK) return rc;
  PTPP_CHECK_ARG(a->maps == 1 || !a->lse == !a->out2, "attention_long_fwd: lse and out2 are kept together");
  int64_t o_ml;
  const int64_t need = plan_fwd(p, a, &o_ml, "attention_long_fwd");
  if (need < 0) return PTPP_EINVAL;
  PTPP_CHECK_ARG(!need || (a->ws && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= (size_t)need),
                 "attention_long_fwd: workspace of %zu bytes, needs %lld (16-byte aligned)", a->ws_bytes, (long long)need);
  p.part_o = reinterpret_cast<float*>(a->ws);
  p.part_ml = p.part_o + o_ml;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->dtype == PTPP_F32) return dispatch_fwd<float>(p, a->maps, st);
  if (a->dtype == PTPP_BF16) return dispatch_fwd<bf16_raw>(p, a->maps, st);
  return dispatch_fwd<f16_raw>(p, a->maps, st);
}

int64_t ptpp_attention_long_ws_bwd(LongP p, int maps, int dtype);
extern "C" int64_t ptpp_attention_long_ws_bytes(const ptpp_attention_long_args* a, int backward) {
  LongP p;
  if (ptpp_attention_long_params(a, backward, &p, "attention_long_ws_bytes") != PTPP_OK) return -1;
  if (backward) return ptpp_attention_long_ws_bwd(p, a->maps, a->dtype);
  int64_t o_ml;
  return plan_fwd(p, a, &o_ml, "attention_long_ws_bytes");
}
