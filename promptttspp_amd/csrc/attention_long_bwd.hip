// Backward of the attention kernels for long sequences (mathematics and layout: attention_long.h).  Two passes that each own what
// they write -- no atomics on memory, the same bits on every run -- and one small launch for the parameter gradients:
//   attn_long_dq_kernel   owns 128 queries, streams keys and values: dq, and D_m[i] = sum_j P_m dP in f32
//   attn_long_dkv_kernel  owns 128 keys, streams queries and dout:   dk, dv, per-block sums of the table's gradient
//   attn_long_fin_kernel  adds the per-block sums of dtable and dlam in a fixed order
// The price of the second pass is 2 of 7 products (4 of 14 units with two maps); one pass would need f32 atomics on dq.
// 24 x 761-1250 of 4 x 64 bf16, calls back to back: dq 78, dk / dv 119 us (385 and 336 TFLOP/s; 800 blocks on 768 and 512 places);
// 8 x 1317-2000 differential: 129 and 253 us (dk / dv: its accumulators leave one wave per SIMD).  Counters of the former dk / dv: vector
// unit 33 %, matrix 18 %, LDS 17 % busy, no bank conflicts, 1.45 waves per SIMD on average -- the second, partly empty round of blocks.
//
// D_m: rows of dout . out_m give it only to the rounding of the kept 16-bit context.  That is enough to centre dS where a row sees many keys (in
// dq the centre's error is multiplied by the mean of their k); where a block's rows see few, up to LA_TWICE, a first sweep corrects it.  The table's
// gradient is a sum with heavy cancellation (every row of dS adds up to zero), so the dq pass also sums P_m (dP - D_m') in f32 and the dk / dv
// pass uses the corrected D_m.  lam's gradient adds the D_1 of all rows (50000 of 8 x 1317-2000, of either sign), and takes that sum as exact as
// its terms are, at no operation per pair (EXACT; error of such a D_1 against 64 bits 1.7e-7 -> 0.9e-7, of dlam 1.8e-4 -> 0.46e-4 where plain
// f32 has 0.9e-4; backward of 8 x 1333-2000 bf16 385 -> 389 us):
//   - D' rounded to the grid of dP's largest values (la_grid): dP - D' is then exact, else it is rounded the same way for all pairs of a row;
//   - P taken against lse - log2(keys) / 2, a whole number, instead of lse (la_half_lse): a row spread over n keys has scores log2(n) below lse,
//     whose rounding would grow with that; the factor is applied to the row's sums;
//   - the patches' sums added with their rounding errors carried along;
//   - 16-bit: dP of every other row as the product with -dout.  The matrix instruction's 16-bit sums are rounded with a bias that does not
//     follow their sign (D_1 came out 1.6e-9 too small on average, with dout and with -dout; f32 has none).
#include <type_traits>

#include "attention_long.h"

namespace {

// FEW: the launch would not fill the chip with blocks of 128 rows.  A block owns 32, its W waves take 32-row chunks of the streamed side
// in turn, each through its own two buffers, and add their sums at the end (the shape of the forward's few-row kernel).
template <typename E, int DK, int DV, int MAPS, bool FEW>
struct LBwd {
  static constexpr int W = FEW ? LSplit<E, DK, DV, MAPS>::W : LA_WAVES;
  static constexpr int ROWS = FEW ? 32 : LA_TILE;  // streamed rows of a buffer
  static constexpr int LOADERS = FEW ? 1 : LA_WAVES;
  static constexpr int PATCHES = ROWS / 32;
  static constexpr int NB = FEW ? LSplit<E, DK, DV, MAPS>::NB : 2;
};

// Most keys of a row, 16-bit, for which the centre is corrected before dq is summed.  Error of dq against 64 bits, in units of its output's
// rounding, without and with: 2-12 keys 1.6-3.4 and 1.4, 16-41 keys 1.5-1.6 and 1.4, 63-128 keys 1.5 and 1.4.  Backward, us: 32 x 64 of
// 2 x 128 27.8 and 29.9, 200 x 64 of 4 x 64 49 and 53; up to 128 keys 200 x 128 of 4 x 64 would go from 74 to 82.
constexpr int LA_TWICE = 64;

// x rounded to the steps that f32 has at `size` (both f32; no excess precision or reassociation in the compiler's defaults)
__device__ __forceinline__ float la_grid(float x, float size) {
  const float c = 1.5f * __uint_as_float((uint32_t)min((int)(__float_as_uint(size) >> 23) + 1, 254) << 23);
  return (x + c) - c;
}
__device__ __forceinline__ float la_half_lse(float lse, int keys) { return rintf(lse - 0.5f * log2f((float)max(keys, 1))); }

template <typename E, int DK, int DV, int MAPS, bool BIAS, bool FEW>
__global__ __launch_bounds__((LBwd<E, DK, DV, MAPS, FEW>::W * 64), sizeof(E) == 4 ? 1 : 2) void attn_long_dq_kernel(const LongP p) {
  typedef LBwd<E, DK, DV, MAPS, FEW> X;
  constexpr int W = X::W, ROWS = X::ROWS, NB = X::NB;
  constexpr int CH = LOp<E>::CH, KS = DK / (2 * CH), VS = DV / (2 * CH), PS = 16 / CH, NT = DK / 32;
  constexpr bool TIGHT = sizeof(E) == 4 || MAPS * DV == 256 || FEW;  // registers are short: LDS addresses not kept across patches
  constexpr bool EXACT = MAPS == 2, FLIP = EXACT && sizeof(E) == 2;  // D_1 as exact as its terms (head of this file)
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ double lred[LA_WAVES];
  __shared__ float weps[W][MAPS][32];
  constexpr int KIMG = ROWS * DK, VIMG = ROWS * DV, BUF = MAPS * KIMG + VIMG;
  const int lane = threadIdx.x & 63, wave = la_wave(), lq = lane & 31, hw = lane >> 5;
  E* const img = reinterpret_cast<E*>(smem) + (FEW ? wave * NB * BUF : 0);
  float* const btab = reinterpret_cast<float*>(smem + (FEW ? W : 1) * NB * BUF * sizeof(E));

  int qt, bh;
  la_block(p.nqt, p.B * p.H, qt, bh);
  if (p.causal) qt = p.nqt - 1 - qt;  // (the longest rows first)
  const int h = bh % p.H, b = FEW ? bh / p.H : la_longest(p, p.k_lengths, bh / p.H, lane), hk = h / (p.H / p.Hk);
  const int klen = la_klen(p, b), qlen = la_qlen(p, b), qs = la_qstart(p, b);
  constexpr int OWN = FEW ? LA_OWN : LA_OWN * LA_WAVES;
  const int ib = qt * OWN, i0 = ib + (FEW ? 0 : wave * LA_OWN), iq = i0 + lq;
  const int dv = MAPS * p.dk;
  int kend = ib < qlen ? klen : 0;
  if (p.causal) kend = min(kend, max(0, qs + min(ib + OWN, qlen)));
  const int nt = (kend + ROWS - 1) / ROWS;

  const E* kb = reinterpret_cast<const E*>(p.k) + b * p.sk + (int64_t)hk * MAPS * p.dk;
  const E* vb = reinterpret_cast<const E*>(p.v) + b * p.sv + (int64_t)hk * dv;
  typedef LTile<E, DK, ROWS, X::LOADERS, sizeof(E) == 2 && !FEW> KT;
  typedef LTile<E, DV, ROWS, X::LOADERS, sizeof(E) == 2 && !FEW> VT;
  const int part = FEW ? 0 : wave;
  KT kt;
  VT vt;
  kt.init(p.ldk, p.dk, lane, part);
  vt.init(p.ldv, dv, lane, part);
  constexpr int NDMA = MAPS * KT::NI + VT::NI;
  auto issue = [&](int tile, int buf) {
    const int j0 = tile * ROWS;
    E* d = img + buf * BUF;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) kt.issue(kb + (int64_t)j0 * p.ldk + m * p.dk, kend - j0, d + m * KIMG, lane, part);
    vt.issue(vb + (int64_t)j0 * p.ldv, kend - j0, d + MAPS * KIMG, lane, part);
  };
  const int first = FEW ? wave : 0;
  constexpr int STEP = FEW ? W : 1;
  if (NB == 2 && first < nt) issue(first, 0);
  if constexpr (BIAS) la_fill_btab(p, btab, h);
  float lam = 0.f;
  if constexpr (MAPS == 2) lam = la_lambda(p, h, lane);

  uint4 qf[MAPS][KS], df[VS];
  float Dm[MAPS], ref[MAPS], eps[MAPS], low = 0.f, size = 0.f;  // ref: lse or its stand-in; eps, low: the sum and what its roundings left
  {
    const bool on = iq < qlen;
    const E* qb = reinterpret_cast<const E*>(p.q) + b * p.sq + (int64_t)h * MAPS * p.dk + (int64_t)iq * p.ldq;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = (2 * s + hw) * CH;
        qf[m][s] = (on && c < p.dk) ? *reinterpret_cast<const uint4*>(qb + m * p.dk + c) : uint4{0, 0, 0, 0};
      }
    const E* db = reinterpret_cast<const E*>(p.dout) + b * p.sdo + (int64_t)h * dv + (int64_t)iq * p.lddo;
    const E* ob = reinterpret_cast<const E*>(p.out) + b * p.so + (int64_t)h * dv + (int64_t)iq * p.ldo;
    const E* o2 = reinterpret_cast<const E*>(p.out2) + ((int64_t)b * p.Tq + iq) * ((int64_t)p.H * dv) + (int64_t)h * dv;
    float d0 = 0.f, d1 = 0.f, dn = 0.f, vn = 0.f;
    uint4 vf[EXACT ? VS : 1];
    if constexpr (EXACT) {  // |v| of the first 32 keys, and |dout|: dP's size
#pragma unroll
      for (int s = 0; s < VS; ++s) {
        const int c = (2 * s + hw) * CH;
        vf[s] = *(lq < kend && c < dv ? reinterpret_cast<const uint4*>(vb + (int64_t)lq * p.ldv + c) : g_conv_zero_page);
      }
    }
#pragma unroll
    for (int s = 0; s < VS; ++s) {
      const int c = (2 * s + hw) * CH;
      df[s] = uint4{0, 0, 0, 0};
      if (on && c < dv) {
        df[s] = *reinterpret_cast<const uint4*>(db + c);
        if constexpr (EXACT) dn += la_dot<E>(df[s], df[s]);
        d0 += la_dot<E>(df[s], *reinterpret_cast<const uint4*>(ob + c));
        if constexpr (MAPS == 2) d1 += la_dot<E>(df[s], *reinterpret_cast<const uint4*>(o2 + c));
      }
    }
    d0 = la_half_sum(d0);
    Dm[0] = d0;
    if constexpr (MAPS == 2) {  // out = out_0 - lam out_1
      d1 = la_half_sum(d1);
      Dm[0] = fmaf(lam, d1, d0);
      Dm[MAPS - 1] = d1;
    }
    if constexpr (EXACT) {
#pragma unroll
      for (int s = 0; s < VS; ++s) vn += la_dot<E>(vf[s], vf[s]);
      vn = la_half_sum(vn);
      float lg = vn > 0.f ? log2f(vn) : 0.f, cnt = vn > 0.f ? 1.f : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {  // (the geometric mean: one key of another size must not coarsen the others' grid)
        lg += __shfl_xor(lg, o, 64);
        cnt += __shfl_xor(cnt, o, 64);
      }
      size = 2.f * sqrtf(la_half_sum(dn)) * exp2f(0.5f * lg / fmaxf(cnt, 1.f));
    }
    if constexpr (FLIP) {
      const uint32_t flip = lq & 1 ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < VS; ++s) df[s] = uint4{df[s].x ^ flip, df[s].y ^ flip, df[s].z ^ flip, df[s].w ^ flip};
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      ref[m] = on ? p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] : INFINITY;
      if (EXACT && m == MAPS - 1) {
        ref[m] = la_half_lse(ref[m], klen);
        Dm[m] = la_grid(Dm[m], size);
      }
      eps[m] = 0.f;
    }
  }
  f32x16 acc[MAPS][NT];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x16{};
  LScale<E> sc[MAPS];
  const float c2 = p.scale * LA_LOG2E, sign = lq & 1 ? -1.f : 1.f;
  const int q0 = qs + i0, D = p.max_distance;

  // one 32 x 32 patch; `sums`: only what corrects D'
  auto patch = [&](auto sums, const E* kimg, const E* vimg, int ks, int j0) __attribute__((always_inline)) {
    const int ln = TIGHT ? la_opaque(lane) : lane, lr = ln & 31, hr = ln >> 5;
    f32x16 dp = f32x16{};
#pragma unroll
    for (int kk = 0; kk < VS; ++kk) {
      dp = LOp<E>::mma(la_frag<E, DV>(vimg, 32 * ks + lr, 2 * kk + hr), df[kk], dp);
      if (TIGHT && kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      f32x16 s = f32x16{};
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) s = LOp<E>::mma(la_frag<E, DK>(kimg + m * KIMG, 32 * ks + lr, 2 * kk + hr), qf[m][kk], s);
      const int dmin = j0 - (q0 + 31), dmax = j0 + 31 - q0;
      if (BIAS && dmin < D && dmax > -D) {
        const float* bt = btab + (j0 - q0 - lr + 4 * hr + D + LA_PAD);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, bt[8 * (r >> 2) + (r & 3)]) - ref[m];
      } else {
        const float bc = (BIAS ? btab[dmin >= D ? 2 * (D + LA_PAD) : 0] : 0.f) - ref[m];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], c2, bc);
      }
      if ((j0 + 32 > kend || (p.causal && j0 + 31 > q0))) {
        const int jend = min(klen, p.causal ? q0 + lr + 1 : klen) - j0 - 4 * hr;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) < jend ? s[r] : -INFINITY;
      }
      float e[4] = {};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = la_exp2(s[r]) * (FLIP ? fmaf(dp[r], sign, -Dm[m]) : dp[r] - Dm[m]);
        e[r & 3] += s[r];
      }
      const float y = (e[0] + e[1]) + (e[2] + e[3]) - (EXACT && m == MAPS - 1 ? low : 0.f), t = eps[m] + y;
      if (EXACT && m == MAPS - 1) low = (t - eps[m]) - y;  // (compensated: what the addition rounded away)
      eps[m] = t;
      if constexpr (!decltype(sums)::value) {
        sc[m].apply(s, acc[m]);
#pragma unroll
        for (int st = 0; st < PS; ++st) {
          const uint4 f = la_pack<E>(s, st);
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[m][n] = LOp<E>::mma(la_tfrag<E, DK>(kimg + m * KIMG, 32 * ks, st, n, ln), f, acc[m][n]);
        }
      }
      if (TIGHT) __builtin_amdgcn_sched_barrier(0);
    }
  };

  auto sweep = [&](auto sums) __attribute__((always_inline)) {
    for (int tile = first, buf = 0; tile < nt; tile += STEP, buf ^= NB - 1) {
      if constexpr (FEW) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the next buffer's last reads are done
      if (NB == 1) {
        issue(tile, 0);
        glds_wait<0>();
      } else if (tile + STEP < nt) {
        issue(tile + STEP, buf ^ 1);
        glds_wait<NDMA>();
      } else {
        glds_wait<0>();
      }
      if constexpr (!FEW) la_barrier();
      const E* kimg = img + buf * BUF;
      const E* vimg = kimg + MAPS * KIMG;
#pragma unroll 1
      for (int ks = 0; ks < X::PATCHES; ++ks) patch(sums, kimg, vimg, ks, tile * ROWS + 32 * ks);
      if constexpr (!FEW) la_barrier();
    }
  };
  if constexpr (FEW && BIAS) la_barrier();  // (the table; the loop itself has no barrier)
  if constexpr (sizeof(E) == 2) {
    if (kend <= LA_TWICE || (p.causal && qs + ib < LA_TWICE)) {  // (the whole block; causal: its first rows see few, and it is a short one)
      sweep(std::true_type{});
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        eps[m] = la_half_sum(eps[m]);
        if (FEW && hw == 0) weps[wave][m][lq] = eps[m];
      }
      if constexpr (FEW) {
        la_barrier();
#pragma unroll
        for (int m = 0; m < MAPS; ++m) {
          eps[m] = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) eps[m] += weps[w][m][lq];
        }
        la_barrier();  // (weps is written again at the end)
      }
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        const float lse = iq < qlen ? p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] : INFINITY;
        const float d = EXACT && m == MAPS - 1 ? eps[m] * la_exp2(ref[m] - lse) : eps[m];
        if (!(lse == INFINITY)) Dm[m] += d;
        if (EXACT && m == MAPS - 1) Dm[m] = la_grid(Dm[m], size);
        eps[m] = 0.f;
      }
      low = 0.f;
      if (NB == 2 && first < nt) issue(first, 0);
    }
  }
  sweep(std::false_type{});

  if constexpr (FEW) {  // the waves' sums of this row
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const float e = la_half_sum(eps[m]);
      if (hw == 0) weps[wave][m][lq] = e;
      float* mine = reinterpret_cast<float*>(img) + m * NT * 1024 + lane;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[(n * 16 + r) * 64] = sc[m].undo(acc[m][n][r]);
    }
    static_assert(MAPS * NT * 1024 * 4 <= NB * BUF * (int)sizeof(E), "a wave's sums fit its buffers");
    la_barrier();
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      eps[m] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) eps[m] += weps[w][m][lq];
    }
  } else {
#pragma unroll
    for (int m = 0; m < MAPS; ++m) eps[m] = la_half_sum(eps[m]);
  }
  const bool stat = hw == 0 && (!FEW || wave == 0);
  float fac[MAPS];  // from the stand-in to lse (read anew: the loop has no register to spare)
  bool live[MAPS];  // rows that are none, or see no key: zeros by selection, as in forward
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const int64_t at = (((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq;
    const float lse = iq < qlen ? p.lse[at] : INFINITY;
    live[m] = iq < qlen && !(lse == INFINITY);
    fac[m] = EXACT && m == MAPS - 1 ? la_exp2(ref[m] - lse) : 1.f;
    if (stat && iq < p.TqP) p.D[at] = live[m] ? fmaf(fac[m], eps[m], Dm[m]) : 0.f;
  }
  if constexpr (MAPS == 2) {  // this block's share of dlam = -sum_i D_1 (64 bits: the rows' terms cancel)
    double s = stat && live[MAPS - 1] ? (double)Dm[MAPS - 1] + (double)fac[MAPS - 1] * (double)eps[MAPS - 1] : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) lred[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0.0;
#pragma unroll
      for (int w = 0; w < W; ++w) t -= lred[w];
      p.lam_part[((int64_t)b * p.H + h) * p.nqt + qt] = t;
    }
  }
  if (iq >= p.Tq) return;
  E* qo = reinterpret_cast<E*>(p.dq) + b * p.sdq + (int64_t)h * MAPS * p.dk + (int64_t)iq * p.lddq;
  if constexpr (FEW) {
    const float* all = reinterpret_cast<const float*>(smem) + lane;
    for (int g = wave; g < MAPS * NT * 4; g += W) {  // 4 registers = 4 channels at a time
      const int m = g / (NT * 4), ch = 32 * ((g >> 2) % NT) + 8 * (g & 3) + 4 * hw;
      const float c = (m == 0 ? p.scale : -lam * p.scale) * (m == 0 ? fac[0] : fac[MAPS - 1]);
      const bool on = m == 0 ? live[0] : live[MAPS - 1];
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[e] += all[w * (NB * BUF * (int)sizeof(E) / 4) + (4 * g + e) * 64];
        v[e] = on ? v[e] * c : 0.f;
      }
      if (ch < p.dk) la_store4<E>(qo + m * p.dk + ch, v[0], v[1], v[2], v[3]);
    }
    return;
  }
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    const float c = (m == 0 ? p.scale : -lam * p.scale) * fac[m];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ch = 32 * n + 8 * g + 4 * hw;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live[m] ? sc[m].undo(acc[m][n][4 * g + e]) * c : 0.f;
        if (ch < p.dk) la_store4<E>(qo + m * p.dk + ch, v[0], v[1], v[2], v[3]);
      }
  }
}

// Sums along the diagonals of a 32 x 32 result x (columns c = lane & 31, rows q): s0: rows 0-15, lane n holds the diagonal
// c - q = n - 15; s1: rows 16-31, c - q = n - 31; lanes >= 47 are zero.  Horner's scheme over the rows, each step one lane further
// (the half waves hold rows 4 apart: both are spread over the whole wave first, the other half zero).
__device__ __forceinline__ void la_diagonals(const f32x16& x, float& s0, float& s1) {
  float acc[2] = {0.f, 0.f};
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float lo[4], hi[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[4 * g + e]), 0u, false, false);
      lo[e] = __uint_as_float(r[0]);
      hi[e] = __uint_as_float(r[1]);
    }
    float& a = acc[g >> 1];
#pragma unroll
    for (int e = 0; e < 4; ++e) a = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a), 0x138, 0xf, 0xf, true)) + lo[e];  // wave_shr:1
#pragma unroll
    for (int e = 0; e < 4; ++e) a = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(a), 0x138, 0xf, 0xf, true)) + hi[e];
  }
  s0 = acc[0];
  s1 = acc[1];
}

// Distances [lo, hi] of bucket bk, clipped to what the sums below hold; false: none
__device__ __forceinline__ bool la_bucket_range(const LongP& p, int bk, int& lo, int& hi) {
  const int far = p.max_distance + LA_PAD, half = p.bidirectional ? p.nbuckets / 2 : p.nbuckets;
  const bool pos = bk >= half;
  const int b = pos ? bk - half : bk;
  const int n0 = b <= p.nexact ? b : p.edges[b - p.nexact - 1];
  const int n1 = b < p.nexact ? b : (b - p.nexact < p.nedges ? p.edges[b - p.nexact] - 1 : far);
  if (pos) {
    lo = max(n0, 1);
    hi = n1;
  } else {
    lo = -n1;
    hi = (!p.bidirectional && b == 0) ? far : -n0;
  }
  return lo <= hi;
}

// One block = 128 keys of one (utterance, key head), a wave = 32 of them; the queries of every head of the group stream through LDS.
// Table gradient: a wave adds dS along its patches' diagonals (la_diagonals) into its own two copies of a distance-indexed array in
// LDS, read and written back by the one lane that holds a distance; patches beyond max_distance go into two registers.  LDS atomics
// instead (ds_add_f32 of every element, no two lanes on one address) took about 330 cycles per wave instruction: 361 us for 24 x 761-1250
// frames of 4 x 64 channels against 123 us this way.
template <typename E, int DK, int DV, int MAPS, bool BIAS, bool FEW>
__global__ __launch_bounds__((LBwd<E, DK, DV, MAPS, FEW>::W * 64), sizeof(E) == 4 || MAPS * DK == 128 ? 1 : 2) void attn_long_dkv_kernel(const LongP p) {
  typedef LBwd<E, DK, DV, MAPS, FEW> X;
  constexpr int W = X::W, ROWS = X::ROWS, NB = X::NB;
  constexpr int CH = LOp<E>::CH, KS = DK / (2 * CH), VS = DV / (2 * CH), PS = 16 / CH, NK = DK / 32, NV = DV / 32;
  constexpr bool AHEAD = sizeof(E) == 2 && !(MAPS == 2 && DK == 32);  // (as registers allow; 64 channels 135 -> 128 us)
  constexpr bool F32 = sizeof(E) == 4;  // (its fragments fill the register file: the scheduler must not fetch further ahead)
  constexpr int NBUF = FEW ? NB : sizeof(E) == 4 ? 1 : 2;  // (f32 tiles twice and the widest distance array would pass 160 KiB)
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int QIMG = ROWS * DK, OIMG = ROWS * DV;
  constexpr int BUFB = (MAPS * QIMG + OIMG) * (int)sizeof(E) + 1024;  // + (lse, D) of every map, ROWS floats each
  float* const btab = reinterpret_cast<float*>(smem + (FEW ? W : 1) * NBUF * BUFB);
  const int lane = threadIdx.x & 63, wave = la_wave(), lk = lane & 31, hw = lane >> 5;
  const int dist_n = la_btab_len(p);
  char* const bufs = smem + (FEW ? wave * NBUF * BUFB : 0);
  float* const hist = btab + ((dist_n + 3) & ~3);  // [2 W][dist_n]
  float* const myhist = hist + 2 * wave * dist_n;

  int kt, bh;
  la_block(p.nkt, p.B * p.Hk, kt, bh);
  const int hk = bh % p.Hk, b = FEW ? bh / p.Hk : la_longest(p, p.q_lengths, bh / p.Hk, lane), G = p.H / p.Hk;
  const int klen = la_klen(p, b), qlen = la_qlen(p, b), qs = la_qstart(p, b);
  constexpr int OWN = FEW ? LA_OWN : LA_OWN * LA_WAVES;
  const int jb = kt * OWN, j0 = jb + (FEW ? 0 : wave * LA_OWN), jk = j0 + lk;
  const int dv = MAPS * p.dk;
  const int t0 = p.causal ? max(0, jb - qs) / ROWS : 0;  // first tile with a query that sees a key of the block
  const int ntq = jb < klen ? max(0, (qlen + ROWS - 1) / ROWS - t0) : 0;
  const int total = ntq * G;

  const E* qb = reinterpret_cast<const E*>(p.q) + b * p.sq;
  const E* ob = reinterpret_cast<const E*>(p.dout) + b * p.sdo;
  typedef LTile<E, DK, ROWS, X::LOADERS, sizeof(E) == 2 && !FEW> QT;
  typedef LTile<E, DV, ROWS, X::LOADERS, sizeof(E) == 2 && !FEW> OT;
  const int part = FEW ? 0 : wave;
  QT qt;
  OT ot;
  qt.init(p.ldq, p.dk, lane, part);
  ot.init(p.lddo, dv, lane, part);
  constexpr int NDMA = MAPS * QT::NI + OT::NI + 1;
  auto issue = [&](int it, int buf) {
    const int h = hk * G + it / ntq, i0 = (t0 + it % ntq) * ROWS;
    char* d = bufs + buf * BUFB;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
      qt.issue(qb + (int64_t)i0 * p.ldq + (h * MAPS + m) * p.dk, qlen - i0, reinterpret_cast<E*>(d) + m * QIMG, lane, part);
    ot.issue(ob + (int64_t)i0 * p.lddo + h * dv, qlen - i0, reinterpret_cast<E*>(d) + MAPS * QIMG, lane, part);
    // statistics: ROWS / 4 lanes per array (lse_0, D_0, lse_1, D_1); every wave issues the same copy so that all count alike
    const int arr = lane / (ROWS / 4), m = arr >> 1;
    const float* src = ((arr & 1) ? p.D : p.lse) + (((int64_t)m * p.B + b) * p.H + h) * p.TqP + i0 + 4 * (lane % (ROWS / 4));
    glds16(m < MAPS ? (const void*)src : (const void*)g_conv_zero_page, __builtin_amdgcn_readfirstlane(lds_addr(d + (MAPS * QIMG + OIMG) * sizeof(E))));
  };
  if (!FEW && NBUF == 2 && total > 0) issue(0, 0);

  // the wave's keys and values: lane (key lk, chunk 2 s + hw)
  uint4 kf[MAPS][KS], vf[VS];
  {
    const bool on = jk < klen;
    const E* kb = reinterpret_cast<const E*>(p.k) + b * p.sk + (int64_t)hk * MAPS * p.dk + (int64_t)jk * p.ldk;
    const E* vb = reinterpret_cast<const E*>(p.v) + b * p.sv + (int64_t)hk * dv + (int64_t)jk * p.ldv;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int c = (2 * s + hw) * CH;
        kf[m][s] = (on && c < p.dk) ? *reinterpret_cast<const uint4*>(kb + m * p.dk + c) : uint4{0, 0, 0, 0};
      }
#pragma unroll
    for (int s = 0; s < VS; ++s) {
      const int c = (2 * s + hw) * CH;
      vf[s] = (on && c < dv) ? *reinterpret_cast<const uint4*>(vb + c) : uint4{0, 0, 0, 0};
    }
  }
  f32x16 ak[MAPS][NK], av[NV];
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int n = 0; n < NK; ++n) ak[m][n] = f32x16{};
#pragma unroll
  for (int n = 0; n < NV; ++n) av[n] = f32x16{};
  LScale<E> sc[MAPS];
  const float c2 = p.scale * LA_LOG2E;
  const int D = p.max_distance;
  float far_lo = 0.f, far_hi = 0.f, lam = 0.f;

  // end of a head: this block's sums per bucket
  auto flush = [&](int h) {
    la_barrier();
    const float lo = wave_sum(far_lo), hi = wave_sum(far_hi);
    if (lane == 0) {  // the two outermost entries, which no near patch reaches
      hist[2 * wave * dist_n] = lo;
      hist[2 * wave * dist_n + dist_n - 1] = hi;
    }
    la_barrier();
    for (int i = threadIdx.x; i < dist_n; i += W * 64) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < 2 * W; ++c) s += hist[c * dist_n + i];
      hist[i] = s;
    }
    la_barrier();
    for (int bk = wave; bk < p.nbuckets; bk += W) {
      int lo_d, hi_d;
      float s = 0.f;
      if (la_bucket_range(p, bk, lo_d, hi_d))
        for (int d = max(lo_d, -D - LA_PAD) + lane; d <= min(hi_d, D + LA_PAD); d += 64) s += hist[d + D + LA_PAD];
      s = wave_sum(s);
      if (lane == 0) p.tab_part[((int64_t)h * p.nbuckets + bk) * ((int64_t)p.B * p.nkt) + b * p.nkt + kt] = s;
    }
    la_barrier();
  };

  // one 32 x 32 patch
  auto patch = [&](const E* qimg, const E* oimg, const float* stat, int sub, int q0) __attribute__((always_inline)) {
    const int ln = F32 || FEW || (MAPS == 2 && DK == 32) ? la_opaque(lane) : lane, lr = ln & 31, hr = ln >> 5;
    const float* st0 = stat + 32 * sub + 4 * hr;  // [m][lse, D][ROWS]; b128 broadcasts: a half wave's rows are the same in all its lanes
    f32x16 dp = f32x16{}, s[MAPS], hsum;
#pragma unroll
    for (int kk = 0; kk < VS; ++kk) {
      dp = LOp<E>::mma(la_frag<E, DV>(oimg, 32 * sub + lr, 2 * kk + hr), vf[kk], dp);
      if (F32 && kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      s[m] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) {
        s[m] = LOp<E>::mma(la_frag<E, DK>(qimg + m * QIMG, 32 * sub + lr, 2 * kk + hr), kf[m][kk], s[m]);
        if (F32 && kk % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
    // the transposed operands of the last products are fetched before the softmax, which hides their way
    uint4 tq[AHEAD ? MAPS : 1][AHEAD ? PS : 1][AHEAD ? NK : 1], to[AHEAD ? PS : 1][AHEAD ? NV : 1];
    if constexpr (AHEAD) {
#pragma unroll
      for (int st = 0; st < PS; ++st) {
#pragma unroll
        for (int m = 0; m < MAPS; ++m)
#pragma unroll
          for (int n = 0; n < NK; ++n) tq[m][st][n] = la_tfrag<E, DK>(qimg + m * QIMG, 32 * sub, st, n, ln);
#pragma unroll
        for (int n = 0; n < NV; ++n) to[st][n] = la_tfrag<E, DV>(oimg, 32 * sub, st, n, ln);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int dmin = j0 - (q0 + 31), dmax = j0 + 31 - q0;
    const bool near = BIAS && dmin < D && dmax > -D;
    if (near) {
      const float* bt = btab + (jk - q0 - 4 * hw + D + LA_PAD);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float bv = bt[-(8 * (r >> 2) + (r & 3))];
#pragma unroll
        for (int m = 0; m < MAPS; ++m) s[m][r] = fmaf(s[m][r], c2, bv);
      }
    } else {
      const float bc = BIAS ? btab[dmin >= D ? dist_n - 1 : 0] : 0.f;
#pragma unroll
      for (int m = 0; m < MAPS; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[m][r] = fmaf(s[m][r], c2, bc);
    }
    if (p.causal && dmax > 0) {
      const int qmin = jk - q0 - 4 * hw;  // register r's query sees the key from this row on
#pragma unroll
      for (int m = 0; m < MAPS; ++m)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[m][r] = 8 * (r >> 2) + (r & 3) >= qmin ? s[m][r] : -INFINITY;
    }
    f32x16 w;
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      const float* ls = st0 + 2 * ROWS * m;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float pr = la_exp2(s[m][r] - ls[8 * (r >> 2) + (r & 3)]);
        if (m == 1) pr *= -lam;
        w[r] = m == 0 ? pr : w[r] + pr;
        s[m][r] = pr * (dp[r] - ls[ROWS + 8 * (r >> 2) + (r & 3)]);
        if constexpr (BIAS) hsum[r] = m == 0 ? s[m][r] : hsum[r] + s[m][r];
      }
    }
#pragma unroll
    for (int m = 0; m < MAPS; ++m) {
      sc[m].apply(s[m], ak[m]);
#pragma unroll
      for (int st = 0; st < PS; ++st) {
        const uint4 f = la_pack<E>(s[m], st);
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          uint4 t;
          if constexpr (AHEAD) t = tq[m][st][n];
          else t = la_tfrag<E, DK>(qimg + m * QIMG, 32 * sub, st, n, ln);
          ak[m][n] = LOp<E>::mma(t, f, ak[m][n]);
          if (F32) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (int st = 0; st < PS; ++st) {
      const uint4 f = la_pack<E>(w, st);
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        uint4 t;
        if constexpr (AHEAD) t = to[st][n];
        else t = la_tfrag<E, DV>(oimg, 32 * sub, st, n, ln);
        av[n] = LOp<E>::mma(t, f, av[n]);
        if (F32) __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (BIAS) {
      if (j0 + 32 > klen) {  // (a column behind the keys holds unmasked values: it must not count; its dk / dv rows are written as zeros)
#pragma unroll
        for (int r = 0; r < 16; ++r) hsum[r] = jk < klen ? hsum[r] : 0.f;
      }
      if (near) {
        float s0, s1;
        la_diagonals(hsum, s0, s1);
        if (lane < 47) {
          float* hp = myhist + (j0 - q0 + D + LA_PAD - 15 + lane);
          hp[0] += s0;
          hp[dist_n - 16] += s1;
        }
      } else {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          s0 += hsum[r];
          s1 += hsum[r + 1];
        }
        if (dmin >= D) far_hi += s0 + s1;
        else far_lo += s0 + s1;
      }
    }
  };

  for (int g = 0; g < G; ++g) {
    const int h = hk * G + g;
    if constexpr (BIAS) {
      la_fill_btab(p, btab, h);
      for (int i = threadIdx.x; i < 2 * W * dist_n; i += W * 64) hist[i] = 0.f;
      far_lo = far_hi = 0.f;
    }
    if constexpr (MAPS == 2) lam = la_lambda(p, h, lane);
    if constexpr (FEW) {
      if (NBUF == 2 && wave < ntq) issue(g * ntq + wave, 0);
      if constexpr (BIAS) la_barrier();  // (the table and the cleared sums; the loop itself has no barrier)
    }
    constexpr int STEP = FEW ? W : 1;
    for (int iq = FEW ? wave : 0, fb = 0; iq < ntq; iq += STEP, fb ^= NBUF - 1) {
      const int it = g * ntq + iq, buf = FEW ? fb : NBUF == 2 ? it & 1 : 0;
      if constexpr (FEW) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the next buffer's last reads are done
      if (NBUF == 1) {
        issue(it, 0);
        glds_wait<0>();
      } else if (FEW ? iq + STEP < ntq : it + 1 < total) {
        issue(it + STEP, buf ^ 1);
        glds_wait<NDMA>();
      } else {
        glds_wait<0>();
      }
      if constexpr (!FEW) la_barrier();
      const E* qimg = reinterpret_cast<const E*>(bufs + buf * BUFB);
      const E* oimg = qimg + MAPS * QIMG;
      const float* stat = reinterpret_cast<const float*>(oimg + OIMG);
      const int q0 = qs + (t0 + iq) * ROWS;
#pragma unroll 1
      for (int sub = 0; sub < X::PATCHES; ++sub) patch(qimg, oimg, stat, sub, q0 + 32 * sub);
      if constexpr (!FEW) la_barrier();
    }
    if constexpr (FEW) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the next head's first chunk goes into buffer 0)
    if constexpr (BIAS) flush(h);
  }

  if constexpr (FEW) {  // every wave's sums into its own buffers
    constexpr int NS = (MAPS * NK + NV) * 1024;
    static_assert(NS * 4 <= NBUF * BUFB, "a wave's sums fit its buffers");
    float* mine = reinterpret_cast<float*>(bufs) + lane;
#pragma unroll
    for (int m = 0; m < MAPS; ++m)
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) mine[((m * NK + n) * 16 + r) * 64] = sc[m].undo(ak[m][n][r]);
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[((MAPS * NK + n) * 16 + r) * 64] = av[n][r];
    la_barrier();
  }
  if (jk >= p.Tk) return;
  const bool on = jk < klen;
  E* ko = reinterpret_cast<E*>(p.gk) + b * p.sdk + (int64_t)hk * MAPS * p.dk + (int64_t)jk * p.lddk;
  E* vo = reinterpret_cast<E*>(p.gv) + b * p.sdv + (int64_t)hk * dv + (int64_t)jk * p.lddv;
  if constexpr (FEW) {
    const float* all = reinterpret_cast<const float*>(smem) + lane;
    for (int g = wave; g < (MAPS * NK + NV) * 4; g += W) {  // 4 registers = 4 channels at a time: dk's, then dv's
      const int n = g >> 2, ch0 = 8 * (g & 3) + 4 * hw;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v[e] += all[w * (NBUF * BUFB / 4) + (4 * g + e) * 64];
        v[e] = on ? (n < MAPS * NK ? v[e] * p.scale : v[e]) : 0.f;
      }
      if (n < MAPS * NK) {
        const int ch = 32 * (n % NK) + ch0;
        if (ch < p.dk) la_store4<E>(ko + (n / NK) * p.dk + ch, v[0], v[1], v[2], v[3]);
      } else {
        const int ch = 32 * (n - MAPS * NK) + ch0;
        if (ch < dv) la_store4<E>(vo + ch, v[0], v[1], v[2], v[3]);
      }
    }
    return;
  }
#pragma unroll
  for (int m = 0; m < MAPS; ++m)
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ch = 32 * n + 8 * g + 4 * hw;
        if (ch < p.dk) {
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = on ? sc[m].undo(ak[m][n][4 * g + e]) * p.scale : 0.f;
          la_store4<E>(ko + m * p.dk + ch, v[0], v[1], v[2], v[3]);
        }
      }
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = 32 * n + 8 * g + 4 * hw;
      if (ch < dv) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = on ? av[n][4 * g + e] : 0.f;
        la_store4<E>(vo + ch, v[0], v[1], v[2], v[3]);
      }
    }
}

// waves [0, H * nbuckets) (with a table): one entry of dtable each; the last blocks: one head's (or the shared) lam vectors
__global__ __launch_bounds__(256) void attn_long_fin_kernel(const LongP p, float* dtable, float* dlam, int accumulate) {
  const int lane = threadIdx.x & 63, wave = la_wave();
  const int ntab = p.table ? (p.H * p.nbuckets + LA_WAVES - 1) / LA_WAVES : 0;
  if ((int)blockIdx.x < ntab) {
    const int w = blockIdx.x * LA_WAVES + wave, h = w / p.nbuckets, bk = w % p.nbuckets, n = p.B * p.nkt;
    if (h >= p.H) return;
    float s = 0.f;
#pragma unroll 8
    for (int i = lane; i < n; i += 64) s += p.tab_part[((int64_t)h * p.nbuckets + bk) * n + i];
    s = wave_sum(s);
    float* d = dtable + (int64_t)bk * p.H + h;
    if (lane == 0) *d = accumulate ? *d + s : s;
    return;
  }
  __shared__ double red[LA_WAVES];
  const int hh = blockIdx.x - ntab, per = p.lam_heads > 1 ? 1 : p.H;  // query heads that share these vectors
  const int64_t n = (int64_t)p.B * per * p.nqt;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const int64_t b = i / (per * p.nqt), r = i % (per * p.nqt);
    s += p.lam_part[(b * p.H + hh) * p.nqt + r];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  if (wave != 0) return;
  const float gl = (float)((red[0] + red[1]) + (red[2] + red[3]));
  float e1, e2;
  la_lambda_parts(p, hh, lane, e1, e2);
  if (lane < p.dk) {
    const int64_t nn = (int64_t)p.lam_heads * p.dk, o = (int64_t)hh * p.dk + lane;
    const float g[4] = {gl * e1 * p.lam[nn + o], gl * e1 * p.lam[o], -gl * e2 * p.lam[3 * nn + o], -gl * e2 * p.lam[2 * nn + o]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* d = dlam + i * nn + o;
      *d = accumulate ? *d + g[i] : g[i];
    }
  }
}

// The rule (as in forward): blocks of 32 rows where that gives few of them (la_few_blocks), else of 128 -- also where the few-row form's
// buffers and the distance sums of a wide table do not fit LDS together.
template <typename E, int DK, int DV, int MAPS>
size_t lds_dq(bool few, int dn) {
  typedef LSplit<E, DK, DV, MAPS> S_;
  return (few ? S_::NB * S_::W * 32 : 2 * LA_TILE) * (size_t)(MAPS * DK + DV) * sizeof(E) + ((dn + 3) & ~3) * sizeof(float);
}
template <typename E, int DK, int DV, int MAPS>
size_t lds_dkv(bool few, int dn) {
  const int W = few ? LSplit<E, DK, DV, MAPS>::W : LA_WAVES;
  const size_t buf = (few ? 32 : LA_TILE) * (size_t)(MAPS * DK + DV) * sizeof(E) + 1024;
  return (few ? LSplit<E, DK, DV, MAPS>::NB * W : sizeof(E) == 4 ? 1 : 2) * buf + (((dn + 3) & ~3) + 2 * W * (size_t)dn) * sizeof(float);
}
// chooses the launch shape and sets the row-block counts
template <typename E, int DK, int DV, int MAPS>
void plan_bwd(LongP& p) {
  const int dn = p.table ? 2 * (p.max_distance + LA_PAD) + 1 : 0;
  const int64_t few = la_few_blocks(sizeof(E) == 4 ? PTPP_F32 : PTPP_BF16, MAPS, p.dk);
  p.few_q = (int64_t)(p.TqP / 32) * p.B * p.H <= few;
  p.few_k = (int64_t)((p.Tk + 31) / 32) * p.B * p.Hk <= few && lds_dkv<E, DK, DV, MAPS>(true, dn) <= LA_LDS;
  if (p.few_q) p.nqt = p.TqP / 32;  // (D is written up to the padding of its rows)
  if (p.few_k) p.nkt = (p.Tk + 31) / 32;
}
template <typename E>
void plan_bwd(LongP& p, int maps) {
  if (maps == 1) p.dk <= 64 ? plan_bwd<E, 64, 64, 1>(p) : plan_bwd<E, 128, 128, 1>(p);
  else p.dk <= 32 ? plan_bwd<E, 32, 64, 2>(p) : plan_bwd<E, 64, 128, 2>(p);
}
void plan_bwd(LongP& p, int maps, int dtype) {
  if (dtype == PTPP_F32) plan_bwd<float>(p, maps);
  else if (dtype == PTPP_BF16) plan_bwd<bf16_raw>(p, maps);
  else plan_bwd<f16_raw>(p, maps);
}

template <typename E, int DK, int DV, int MAPS, bool BIAS, bool FEW>
int launch_dq(const LongP& p, size_t sm, hipStream_t st) {
  if (!la_lds_limit((const void*)attn_long_dq_kernel<E, DK, DV, MAPS, BIAS, FEW>, sm, "attention_long_bwd")) return PTPP_ELAUNCH;
  hipLaunchKernelGGL((attn_long_dq_kernel<E, DK, DV, MAPS, BIAS, FEW>), dim3((unsigned)((int64_t)p.nqt * p.B * p.H)), dim3(LBwd<E, DK, DV, MAPS, FEW>::W * 64), sm,
                     st, p);
  PTPP_CHECK_LAUNCH("attention_long_bwd (dq)");
  return PTPP_OK;
}
template <typename E, int DK, int DV, int MAPS, bool BIAS, bool FEW>
int launch_dkv(const LongP& p, size_t sm, hipStream_t st) {
  if (!la_lds_limit((const void*)attn_long_dkv_kernel<E, DK, DV, MAPS, BIAS, FEW>, sm, "attention_long_bwd")) return PTPP_ELAUNCH;
  hipLaunchKernelGGL((attn_long_dkv_kernel<E, DK, DV, MAPS, BIAS, FEW>), dim3((unsigned)((int64_t)p.nkt * p.B * p.Hk)), dim3(LBwd<E, DK, DV, MAPS, FEW>::W * 64),
                     sm, st, p);
  PTPP_CHECK_LAUNCH("attention_long_bwd (dk, dv)");
  return PTPP_OK;
}
template <typename E, int DK, int DV, int MAPS, bool BIAS>
int launch_bwd(const LongP& p, hipStream_t st) {
  const int dn = BIAS ? 2 * (p.max_distance + LA_PAD) + 1 : 0;
  const size_t s1 = lds_dq<E, DK, DV, MAPS>(p.few_q, dn), s2 = lds_dkv<E, DK, DV, MAPS>(p.few_k, dn);
  const int r = p.few_q ? launch_dq<E, DK, DV, MAPS, BIAS, true>(p, s1, st) : launch_dq<E, DK, DV, MAPS, BIAS, false>(p, s1, st);
  if (r != PTPP_OK) return r;
  return p.few_k ? launch_dkv<E, DK, DV, MAPS, BIAS, true>(p, s2, st) : launch_dkv<E, DK, DV, MAPS, BIAS, false>(p, s2, st);
}
template <typename E, int DK, int DV>
int launch_bwd2(const LongP& p, hipStream_t st) {
  return p.table ? launch_bwd<E, DK, DV, 2, true>(p, st) : launch_bwd<E, DK, DV, 2, false>(p, st);
}
template <typename E>
int dispatch_bwd(const LongP& p, int maps, hipStream_t st) {
  if (maps == 1) return p.dk <= 64 ? launch_bwd<E, 64, 64, 1, true>(p, st) : launch_bwd<E, 128, 128, 1, true>(p, st);
  return p.dk <= 32 ? launch_bwd2<E, 32, 64>(p, st) : launch_bwd2<E, 64, 128>(p, st);
}

int64_t up64(int64_t n) { return (n + 63) & ~(int64_t)63; }
// backward workspace, floats: D | lam_part | tab_part
void bwd_layout(const LongP& p, int maps, int64_t* o_lam, int64_t* o_tab, int64_t* total) {
  *o_lam = up64((int64_t)maps * p.B * p.H * p.TqP);
  *o_tab = *o_lam + (maps == 2 ? up64(2 * (int64_t)p.B * p.H * p.nqt) : 0);  // (64-bit sums)
  *total = *o_tab + (p.table ? up64((int64_t)p.B * p.nkt * p.H * p.nbuckets) : 0);
}

}  // namespace

int64_t ptpp_attention_long_ws_bwd(LongP p, int maps, int dtype) {
  int64_t a, b, n;
  plan_bwd(p, maps, dtype);
  bwd_layout(p, maps, &a, &b, &n);
  return n * (int64_t)sizeof(float);
}

extern "C" int ptpp_attention_long_bwd(const ptpp_attention_long_args* a, void* stream) {
  LongP p;
  const int rc = ptpp_attention_long_params(a, 1, &p, "attention_long_bwd");
  if (rc != PTPP_OK) return rc;
  PTPP_CHECK_ARG(a->lse && (uintptr_t)a->lse % 16 == 0, "attention_long_bwd: needs the statistics of the forward pass (16-byte aligned)");
  PTPP_CHECK_ARG(a->maps == 1 || a->out2, "attention_long_bwd: needs the second map's context");
  PTPP_CHECK_ARG((!a->table || a->dtable) && (a->maps == 1 || a->dlam), "attention_long_bwd: null gradient");
  int64_t o_lam, o_tab, total;
  plan_bwd(p, a->maps, a->dtype);
  bwd_layout(p, a->maps, &o_lam, &o_tab, &total);
  PTPP_CHECK_ARG(a->ws && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= (size_t)total * sizeof(float),
                 "attention_long_bwd: workspace of %zu bytes, needs %lld (16-byte aligned)", a->ws_bytes, (long long)(total * sizeof(float)));
  p.D = reinterpret_cast<float*>(a->ws);
  p.lam_part = reinterpret_cast<double*>(p.D + o_lam);
  p.tab_part = p.D + o_tab;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  int r;
  if (a->dtype == PTPP_F32) r = dispatch_bwd<float>(p, a->maps, st);
  else if (a->dtype == PTPP_BF16) r = dispatch_bwd<bf16_raw>(p, a->maps, st);
  else r = dispatch_bwd<f16_raw>(p, a->maps, st);
  if (r != PTPP_OK) return r;
  const int blocks = (p.table ? (p.H * p.nbuckets + LA_WAVES - 1) / LA_WAVES : 0) + (a->maps == 2 ? p.lam_heads : 0);
  hipLaunchKernelGGL(attn_long_fin_kernel, dim3(blocks), dim3(256), 0, st, p, a->dtable, a->dlam, a->accumulate);
  PTPP_CHECK_LAUNCH("attention_long_bwd (parameters)");
  return PTPP_OK;
}
