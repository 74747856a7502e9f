// The step between two blocks of a deep encoder in one launch each way:
//   u = post norm(f),  y = x + scale * gate * u,  z = pre norm(y)
// (include/ptpp.h "ptpp_residual_norm").  HBM-bound: forward moves f, x, y, z once, backward dy, dz, f, x, df, dx once -- y is
// recomputed from f, x and the kept statistics, which costs the bytes of reading it and none of its rounding, so the parameter
// gradients are sums of f32 values.
//
// A row belongs to LPR lanes (16, 32 or 64 of a wave, or a whole block), each holding NV vectors of 4 columns in registers for the
// whole row: every tensor element is touched once, means and squared deviations are two passes over registers.  In backward a lane
// group walks over rows of one utterance with the column sums in registers; the block adds its groups in a fixed order and writes
// one partial row per sum, a finishing launch adds the partial rows (no atomics: the same bits on every run).  24 x 875-1250 of 256 bf16:
// forward 19 us (2.9 TB/s), backward 30 + 5 us; 8 x 1638-2048 of 1024 f16: forward 30 us (4.2 TB/s), backward 67 + 4.3 us (2.9 TB/s).
#include "ptpp_common.h"

namespace {

struct RnP {
  const void *f, *x, *dy, *dz;
  void *y, *z, *df, *dx;
  const float *gate, *post_g, *post_b, *pre_g, *pre_b;
  float* stats;  // (4, B * T): mean f, rstd f, mean y, rstd y
  const int* lengths;
  float* part;   // [B * chunks][slots][C]
  int B, T, C, rms, gate_rows, chunks, rows_per_chunk, nslots;
  int slot[5];   // pre_g, pre_b, post_g, post_b, gate: position among the wanted sums, -1: not wanted
  float scale, eps, inv_c;
};

template <typename E>
__device__ __forceinline__ void rn_st4(E* p, f32x4 v) {
  if constexpr (sizeof(E) == 4) {
    *reinterpret_cast<f32x4*>(p) = v;
  } else if constexpr (IsBf16<E>::value) {
    typedef __attribute__((ext_vector_type(4))) __bf16 b4;
    *reinterpret_cast<b4*>(p) = __builtin_convertvector(v, b4);
  } else {
    typedef __attribute__((ext_vector_type(4))) _Float16 h4;
    *reinterpret_cast<h4*>(p) = __builtin_convertvector(v, h4);
  }
}

// sum over the lanes of a row; a whole block (LPR > 64) goes through LDS (`red`: one float per wave, two sets used in turn)
template <int LPR>
__device__ __forceinline__ float rn_sum(float v, float* red, int& turn) {
#pragma unroll
  for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    float* r = red + (turn & 1) * W;
    ++turn;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += r[w];
  }
  return v;
}

// mean (0 for rms) and 1 / deviation of the row in v; lanes past the row hold zeros in v and must not count
template <int LPR, int NV>
__device__ __forceinline__ void rn_stats(const f32x4 (&v)[NV], const bool (&on)[NV], const RnP& p, float* red, int& turn, float& mean, float& rstd) {
  mean = 0.f;
  if (!p.rms) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s += (v[i][0] + v[i][1]) + (v[i][2] + v[i][3]);
    mean = rn_sum<LPR>(s, red, turn) * p.inv_c;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (on[i])
#pragma unroll
      for (int e = 0; e < 4; ++e) q = fmaf(v[i][e] - mean, v[i][e] - mean, q);
  rstd = rsqrtf(rn_sum<LPR>(q, red, turn) * p.inv_c + p.eps);
}

template <int NV>
struct RnVec {
  f32x4 v[NV];
  __device__ __forceinline__ void load(const float* src, const bool (&on)[NV], const int (&col)[NV], float none) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = src && on[i] ? *reinterpret_cast<const f32x4*>(src + col[i]) : f32x4{none, none, none, none};
  }
};

template <typename E, int NT, int LPR, int NV>
__global__ __launch_bounds__(NT) void residual_norm_fwd_kernel(const RnP p) {
  __shared__ float red[2 * (LPR > 64 ? LPR / 64 : 1)];
  constexpr int RPB = NT / LPR;  // rows of a block
  const int sub = threadIdx.x / LPR, ln = threadIdx.x % LPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + sub;
  const int64_t rows = (int64_t)p.B * p.T;
  if (row >= rows) return;  // (LPR > 64: the whole block)
  const int b = (int)(row / p.T), t = (int)(row - (int64_t)b * p.T);
  int turn = 0;
  bool on[NV];
  int col[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = 4 * (i * LPR + ln);
    on[i] = col[i] < p.C;
  }
  E* yo = reinterpret_cast<E*>(p.y) + row * p.C;
  E* zo = reinterpret_cast<E*>(p.z) + row * p.C;
  if (p.lengths && t >= p.lengths[b]) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (on[i]) {
        rn_st4<E>(yo + col[i], f32x4{0.f, 0.f, 0.f, 0.f});
        if (p.z) rn_st4<E>(zo + col[i], f32x4{0.f, 0.f, 0.f, 0.f});
      }
    return;
  }
  const E* fi = reinterpret_cast<const E*>(p.f) + row * p.C;
  const E* xi = reinterpret_cast<const E*>(p.x) + row * p.C;
  f32x4 v[NV], y[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = on[i] ? Elem<E>::ld4(fi + col[i]) : f32x4{0.f, 0.f, 0.f, 0.f};
    y[i] = p.x && on[i] ? Elem<E>::ld4(xi + col[i]) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  RnVec<NV> ga;
  ga.load(p.gate ? p.gate + (p.gate_rows > 1 ? (int64_t)b * p.C : 0) : nullptr, on, col, 1.f);
  float mf = 0.f, rf = 1.f, my = 0.f, ry = 1.f;
  if (p.post_g) {
    RnVec<NV> g, be;
    g.load(p.post_g, on, col, 0.f);
    be.load(p.post_b, on, col, 0.f);
    rn_stats<LPR, NV>(v, on, p, red, turn, mf, rf);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = fmaf((v[i][e] - mf) * rf, g.v[i][e], be.v[i][e]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) y[i][e] = on[i] ? fmaf(p.scale * ga.v[i][e], v[i][e], y[i][e]) : 0.f;
    if (on[i]) rn_st4<E>(yo + col[i], y[i]);
  }
  if (p.pre_g) {
    RnVec<NV> g, be;
    g.load(p.pre_g, on, col, 0.f);
    be.load(p.pre_b, on, col, 0.f);
    rn_stats<LPR, NV>(y, on, p, red, turn, my, ry);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (on[i]) {
        f32x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = fmaf((y[i][e] - my) * ry, g.v[i][e], be.v[i][e]);
        rn_st4<E>(zo + col[i], z);
      }
  }
  if (p.stats && ln == 0) {
    p.stats[row] = mf;
    p.stats[rows + row] = rf;
    p.stats[2 * rows + row] = my;
    p.stats[3 * rows + row] = ry;
  }
}

// gradient of v -> (v - mean) * rstd * gamma through h = (v - mean) * rstd and g = gamma * upstream:
// rstd * (g - mean(g) - h * mean(g h)); without the mean term for rms
template <int LPR, int NV>
__device__ __forceinline__ void rn_back(f32x4 (&g)[NV], const f32x4 (&h)[NV], float rstd, const RnP& p, float* red, int& turn) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)  // (lanes past the row hold zero gradients)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s0 += g[i][e];
      s1 = fmaf(g[i][e], h[i][e], s1);
    }
  s1 = rn_sum<LPR>(s1, red, turn) * p.inv_c;
  s0 = p.rms ? 0.f : rn_sum<LPR>(s0, red, turn) * p.inv_c;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) g[i][e] = rstd * (g[i][e] - s0 - h[i][e] * s1);
}

template <typename E, int NT, int LPR, int NV>
__global__ __launch_bounds__(NT) void residual_norm_bwd_kernel(const RnP p) {
  __shared__ float red[2 * (LPR > 64 ? LPR / 64 : 1)];
  extern __shared__ __attribute__((aligned(16))) float tot[];  // [RPB][C]: the groups' column sums, one kind at a time
  constexpr int RPB = NT / LPR;
  const int sub = threadIdx.x / LPR, ln = threadIdx.x % LPR;
  const int b = blockIdx.x / p.chunks, ck = blockIdx.x % p.chunks;
  const int64_t rows = (int64_t)p.B * p.T;
  int turn = 0;
  bool on[NV];
  int col[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    col[i] = 4 * (i * LPR + ln);
    on[i] = col[i] < p.C;
  }
  RnVec<NV> ga, pg, pb, qg;  // gate, post gamma / beta, pre gamma
  ga.load(p.gate ? p.gate + (p.gate_rows > 1 ? (int64_t)b * p.C : 0) : nullptr, on, col, 1.f);
  pg.load(p.post_g, on, col, 1.f);
  pb.load(p.post_b, on, col, 0.f);
  qg.load(p.pre_g, on, col, 0.f);
  f32x4 acc[5][NV];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[k][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int len = p.lengths ? min(p.lengths[b], p.T) : p.T;
  const int t1 = min(p.T, (ck + 1) * p.rows_per_chunk);
  for (int t = ck * p.rows_per_chunk + sub; t < t1; t += RPB) {  // (LPR > 64: RPB == 1, the same trips for the whole block)
    const int64_t row = (int64_t)b * p.T + t, o = row * p.C;
    if (t >= len) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) {
          if (p.df) rn_st4<E>(reinterpret_cast<E*>(p.df) + o + col[i], f32x4{0.f, 0.f, 0.f, 0.f});
          if (p.dx) rn_st4<E>(reinterpret_cast<E*>(p.dx) + o + col[i], f32x4{0.f, 0.f, 0.f, 0.f});
        }
      continue;
    }
    f32x4 h[NV], y[NV], gy[NV], gz[NV];
    const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      h[i] = on[i] ? Elem<E>::ld4(reinterpret_cast<const E*>(p.f) + o + col[i]) : zero;
      y[i] = p.x && on[i] ? Elem<E>::ld4(reinterpret_cast<const E*>(p.x) + o + col[i]) : zero;
      gy[i] = p.dy && on[i] ? Elem<E>::ld4(reinterpret_cast<const E*>(p.dy) + o + col[i]) : zero;
      gz[i] = p.dz && on[i] ? Elem<E>::ld4(reinterpret_cast<const E*>(p.dz) + o + col[i]) : zero;
    }
    const float mf = p.stats[row], rf = p.stats[rows + row], my = p.stats[2 * rows + row], ry = p.stats[3 * rows + row];
    f32x4 u[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[i][e] = (h[i][e] - mf) * rf;                       // normalised f (f itself without a post norm)
        u[i][e] = fmaf(h[i][e], pg.v[i][e], pb.v[i][e]);
        y[i][e] = (fmaf(p.scale * ga.v[i][e], u[i][e], y[i][e]) - my) * ry;  // normalised y
      }
    if (p.dz && p.pre_g) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[0][i][e] = fmaf(gz[i][e], y[i][e], acc[0][i][e]);
          acc[1][i][e] += gz[i][e];
          gz[i][e] *= qg.v[i][e];
        }
      rn_back<LPR, NV>(gz, y, ry, p, red, turn);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) gy[i][e] += gz[i][e];
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (p.dx && on[i]) rn_st4<E>(reinterpret_cast<E*>(p.dx) + o + col[i], gy[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = on[i] ? p.scale * gy[i][e] : 0.f;
        acc[4][i][e] = fmaf(d, u[i][e], acc[4][i][e]);
        const float du = d * ga.v[i][e];
        acc[2][i][e] = fmaf(du, h[i][e], acc[2][i][e]);
        acc[3][i][e] += du;
        gz[i][e] = du * pg.v[i][e];
      }
    }
    if (p.post_g) rn_back<LPR, NV>(gz, h, rf, p, red, turn);
    if (p.df) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) rn_st4<E>(reinterpret_cast<E*>(p.df) + o + col[i], gz[i]);
    }
  }
  float* part = p.part + (int64_t)blockIdx.x * p.nslots * p.C;
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (p.slot[k] < 0) continue;
    float* dst = part + (int64_t)p.slot[k] * p.C;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) *reinterpret_cast<f32x4*>(dst + col[i]) = acc[k][i];
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (on[i]) *reinterpret_cast<f32x4*>(tot + sub * p.C + col[i]) = acc[k][i];
      __syncthreads();
      for (int c = threadIdx.x; c < p.C; c += NT) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < RPB; ++r) s += tot[r * p.C + c];
        dst[c] = s;
      }
    }
  }
}

struct RnDst {
  float* dst[5];
};
// grid: (columns / 32, wanted sums; a per-utterance gate takes one row of blocks per utterance)
__global__ __launch_bounds__(1024) void residual_norm_fin_kernel(const RnP p, const RnDst d, int accumulate) {
  __shared__ float red[32][33];
  const int cl = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  const int plain = p.nslots - (p.slot[4] >= 0 ? 1 : 0);
  const bool gate = (int)blockIdx.y >= plain;
  const int ub = gate ? blockIdx.y - plain : 0;
  int k = 4;
  if (!gate)
    for (int i = 0; i < 4; ++i)
      if (p.slot[i] == (int)blockIdx.y) k = i;
  const bool per_utt = gate && p.gate_rows > 1;
  const int lo = per_utt ? ub * p.chunks : 0, n = per_utt ? p.chunks : p.B * p.chunks;
  float s = 0.f;
  if (c < p.C)
#pragma unroll 8
    for (int i = r; i < n; i += 32) s += p.part[((int64_t)(lo + i) * p.nslots + p.slot[k]) * p.C + c];
  red[r][cl] = s;
  __syncthreads();
  if (r == 0 && c < p.C) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += red[i][cl];
    float* o = d.dst[k] + (per_utt ? (int64_t)ub * p.C : 0) + c;
    *o = accumulate ? *o + v : v;
  }
}

int check(const ptpp_residual_norm_args* a, int backward, RnP* p, const char* who) {
  PTPP_CHECK_ARG(a, "%s: null arguments", who);
  PTPP_CHECK_ARG(a->dtype == PTPP_F32 || a->dtype == PTPP_BF16 || a->dtype == PTPP_F16, "%s: bad dtype %d", who, a->dtype);
  PTPP_CHECK_ARG(a->B > 0 && a->T > 0 && a->C > 0 && a->C % 4 == 0 && a->C <= 4096, "%s: bad shape (B %d, T %d, C %d: a multiple of 4, at most 4096)",
                 who, a->B, a->T, a->C);
  PTPP_CHECK_ARG((int64_t)a->B * a->T < (1ll << 28), "%s: too many rows", who);
  PTPP_CHECK_ARG(a->f && (backward || a->y), "%s: null tensor", who);
  PTPP_CHECK_ARG(backward || !a->pre_g == !a->z, "%s: z and the pre norm come together", who);
  PTPP_CHECK_ARG(!a->gate || a->gate_rows == 1 || a->gate_rows == a->B, "%s: a gate of %d rows (1 or %d)", who, a->gate_rows, a->B);
  PTPP_CHECK_ARG((a->post_g || !a->post_b) && (a->pre_g || !a->pre_b), "%s: a beta without its gamma", who);
  PTPP_CHECK_ARG(!a->rms || (!a->post_b && !a->pre_b), "%s: root-mean-square norms have no beta", who);
  PTPP_CHECK_ARG(a->eps > 0.f, "%s: eps must be positive", who);
  const int al = a->dtype == PTPP_F32 ? 16 : 8;
  const void* ten[] = {a->f, a->x, a->dy, a->dz, a->y, a->z, a->df, a->dx};
  for (const void* q : ten) PTPP_CHECK_ARG((uintptr_t)q % al == 0, "%s: tensors must be %d-byte aligned", who, al);
  const void* words[] = {a->stats, a->lengths, a->dgate, a->dpost_g, a->dpost_b, a->dpre_g, a->dpre_b};
  for (const void* w : words) PTPP_CHECK_ARG((uintptr_t)w % 4 == 0, "%s: statistics, lengths and sums must be 4-byte aligned", who);
  const void* par[] = {a->gate, a->post_g, a->post_b, a->pre_g, a->pre_b};
  for (const void* q : par) PTPP_CHECK_ARG((uintptr_t)q % 16 == 0, "%s: parameters must be 16-byte aligned", who);
  *p = RnP{};
  p->f = a->f; p->x = a->x; p->dy = a->dy; p->dz = a->dz; p->y = a->y; p->z = a->z; p->df = a->df; p->dx = a->dx;
  p->gate = a->gate; p->post_g = a->post_g; p->post_b = a->post_b; p->pre_g = a->pre_g; p->pre_b = a->pre_b;
  p->stats = a->stats; p->lengths = a->lengths;
  p->B = a->B; p->T = a->T; p->C = a->C; p->rms = a->rms; p->gate_rows = a->gate ? a->gate_rows : 1;
  p->scale = a->scale; p->eps = a->eps; p->inv_c = 1.f / (float)a->C;
  if (backward) {
    // about 1024 blocks; a chunk is a whole number of block passes
    const int want = (1024 + a->B - 1) / a->B;
    int rpc = (a->T + want - 1) / want;
    rpc = (rpc + 15) & ~15;
    p->rows_per_chunk = rpc;
    p->chunks = (a->T + rpc - 1) / rpc;
    const float* want_p[] = {a->dpre_g, a->dpre_b, a->dpost_g, a->dpost_b, a->dgate};
    const float* have_p[] = {a->pre_g, a->pre_b, a->post_g, a->post_b, a->gate};
    for (int k = 0; k < 5; ++k) {
      PTPP_CHECK_ARG(!want_p[k] || have_p[k], "%s: the gradient of an absent parameter", who);
      p->slot[k] = want_p[k] ? p->nslots++ : -1;
    }
  }
  return PTPP_OK;
}

template <typename E, int NT, int LPR, int NV>
int launch(const RnP& p, bool bwd, hipStream_t st) {
  constexpr int RPB = NT / LPR;
  const int64_t rows = (int64_t)p.B * p.T, blocks = bwd ? (int64_t)p.B * p.chunks : (rows + RPB - 1) / RPB;
  PTPP_CHECK_ARG(blocks * NT < (1ll << 32), "residual_norm: too many rows");
  if (!bwd) {
    hipLaunchKernelGGL((residual_norm_fwd_kernel<E, NT, LPR, NV>), dim3((unsigned)blocks), dim3(NT), 0, st, p);
    PTPP_CHECK_LAUNCH("residual_norm_fwd");
  } else {
    const size_t sm = RPB > 1 ? (size_t)RPB * p.C * sizeof(float) : 0;
    hipLaunchKernelGGL((residual_norm_bwd_kernel<E, NT, LPR, NV>), dim3((unsigned)blocks), dim3(NT), sm, st, p);
    PTPP_CHECK_LAUNCH("residual_norm_bwd");
  }
  return PTPP_OK;
}
template <typename E>
int dispatch(const RnP& p, bool bwd, hipStream_t st) {
  // lanes per row: as few as hold the row in two vectors each (more leave backward, with five column sums per vector, one wave
  // per SIMD); beyond 512 columns a block
  if (p.C <= 64) return launch<E, 256, 16, 1>(p, bwd, st);
  if (p.C <= 128) return launch<E, 256, 32, 1>(p, bwd, st);
  if (p.C <= 256) return launch<E, 256, 64, 1>(p, bwd, st);
  if (p.C <= 512) return launch<E, 256, 64, 2>(p, bwd, st);
  if (p.C <= 1024) return launch<E, 256, 256, 1>(p, bwd, st);
  if (p.C <= 2048) return launch<E, 256, 256, 2>(p, bwd, st);
  return launch<E, 512, 512, 2>(p, bwd, st);
}
int run(const RnP& p, bool bwd, int dtype, hipStream_t st) {
  if (dtype == PTPP_F32) return dispatch<float>(p, bwd, st);
  if (dtype == PTPP_BF16) return dispatch<bf16_raw>(p, bwd, st);
  return dispatch<f16_raw>(p, bwd, st);
}

}  // namespace

extern "C" int64_t ptpp_residual_norm_ws_bytes(const ptpp_residual_norm_args* a) {
  RnP p;
  if (check(a, 1, &p, "residual_norm_ws_bytes") != PTPP_OK) return -1;
  return (int64_t)p.B * p.chunks * p.nslots * p.C * (int64_t)sizeof(float);
}

extern "C" int ptpp_residual_norm_fwd(const ptpp_residual_norm_args* a, void* stream) {
  RnP p;
  const int rc = check(a, 0, &p, "residual_norm_fwd");
  if (rc != PTPP_OK) return rc;
  return run(p, false, a->dtype, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int ptpp_residual_norm_bwd(const ptpp_residual_norm_args* a, void* stream) {
  RnP p;
  const int rc = check(a, 1, &p, "residual_norm_bwd");
  if (rc != PTPP_OK) return rc;
  PTPP_CHECK_ARG(a->stats, "residual_norm_bwd: needs the statistics of the forward pass");
  const int64_t need = (int64_t)p.B * p.chunks * p.nslots * p.C * (int64_t)sizeof(float);
  PTPP_CHECK_ARG(!need || (a->ws && (uintptr_t)a->ws % 16 == 0 && (int64_t)a->ws_bytes >= need), "residual_norm_bwd: workspace of %zu bytes, needs %lld (16-byte aligned)",
                 a->ws_bytes, (long long)need);
  p.part = reinterpret_cast<float*>(a->ws);
  const int ny = p.nslots - (p.slot[4] >= 0 ? 1 : 0) + (p.slot[4] >= 0 ? p.gate_rows : 0);
  PTPP_CHECK_ARG(ny <= 65535, "residual_norm_bwd: a gate of %d rows", p.gate_rows);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int r = run(p, true, a->dtype, st);
  if (r != PTPP_OK || !p.nslots) return r;
  const RnDst d = {{a->dpre_g, a->dpre_b, a->dpost_g, a->dpost_b, a->dgate}};
  hipLaunchKernelGGL(residual_norm_fin_kernel, dim3((p.C + 31) / 32, ny), dim3(1024), 0, st, p, d, a->accumulate);
  PTPP_CHECK_LAUNCH("residual_norm_bwd (sums)");
  return PTPP_OK;
}
