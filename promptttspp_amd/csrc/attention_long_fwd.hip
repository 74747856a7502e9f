// Forward of the attention kernels for long sequences (mathematics and layout: attention_long.h), and the argument checks of
// both directions.
#include <stdlib.h>

#include "attention_long.h"

namespace {

// One block = 128 query rows of one (utterance, head), a wave = 32 of them; keys and values stream through LDS in tiles of 64,
// the next tile's LDS-DMA under the current tile's products.
template <typename E, int DK, int DV, int MAPS, bool BIAS>
__global__ __launch_bounds__(256) void attn_long_fwd_kernel(const LongP p) {
  constexpr int CH = LOp<E>::CH, KS = DK / (2 * CH), PS = 16 / CH, NT = DV / 32;
  constexpr int KSUB = sizeof(E) == 4 ? 1 : 2;  // 32-key patches taken at once (f32 fragments are twice as many registers)
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int KIMG = LA_TILE * DK, VIMG = LA_TILE * DV, BUF = MAPS * KIMG + VIMG;
  E* const img = reinterpret_cast<E*>(smem);
  float* const btab = reinterpret_cast<float*>(smem + 2 * BUF * sizeof(E));
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lq = lane & 31, hw = lane >> 5;

  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int qt = t % p.nqt, bh = t / p.nqt, h = bh % p.H, b = bh / p.H, hk = h / (p.H / p.Hk);
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
    mx[m] = -INFINITY;
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
#pragma unroll
      for (int m = 0; m < MAPS; ++m) {
        f32x16 s[KSUB];
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
          s[ks] = f32x16{};
#pragma unroll
          for (int kk = 0; kk < KS; ++kk)
            s[ks] = LOp<E>::mma(la_frag<E, DK>(kimg + m * KIMG, 32 * (sub * KSUB + ks) + lq, 2 * kk + hw), qf[m][kk], s[ks]);
        }
        float tm = -INFINITY;
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
          const int j0 = tile * LA_TILE + 32 * (sub * KSUB + ks);
          if constexpr (BIAS) {
            const int dmin = j0 - (q0 + 31), dmax = j0 + 31 - q0;  // distances of this 32 x 32 patch
            if (dmin < D && dmax > -D) {
              const float* bt = btab + (j0 - q0 - lq + 4 * hw + D + LA_PAD);
#pragma unroll
              for (int r = 0; r < 16; ++r) s[ks][r] = fmaf(s[ks][r], c2, bt[8 * (r >> 2) + (r & 3)]);
            } else {
              const float bc = dmin >= D ? btab[2 * (D + LA_PAD)] : btab[0];
#pragma unroll
              for (int r = 0; r < 16; ++r) s[ks][r] = fmaf(s[ks][r], c2, bc);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[ks][r] *= c2;
          }
          if (j0 + 32 > kend || (p.causal && j0 + 31 > q0)) {
            const int jend = min(klen, p.causal ? q0 + lq + 1 : klen) - j0 - 4 * hw;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[ks][r] = 8 * (r >> 2) + (r & 3) < jend ? s[ks][r] : -INFINITY;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) tm = fmaxf(tm, s[ks][r]);
        }
        const float mn = fmaxf(mx[m], la_half_max(tm));
        const float mu = mn == -INFINITY ? 0.f : mn;  // (no key seen yet: every exponent below is -inf)
        const float al = la_exp2(mx[m] - mu);
        mx[m] = mn;
        float sum = 0.f;
#pragma unroll
        for (int ks = 0; ks < KSUB; ++ks) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[ks][r] = la_exp2(s[ks][r] - mu);
            sum += s[ks][r];
          }
#pragma unroll
          for (int st = 0; st < PS; ++st) pf[m][ks][st] = la_pack<E>(s[ks], st);
        }
        l[m] = fmaf(l[m], al, sum);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[m][n][r] *= al;
      }
#pragma unroll
      for (int ks = 0; ks < KSUB; ++ks)
#pragma unroll
        for (int st = 0; st < PS; ++st)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 vf = la_tfrag<E, DV>(vimg, 32 * (sub * KSUB + ks), st, n, lane);
#pragma unroll
            for (int m = 0; m < MAPS; ++m) o[m][n] = LOp<E>::mma(vf, pf[m][ks][st], o[m][n]);
          }
    }
    la_barrier();
  }

  // ---- epilogue: lane (query lq) holds channels 32 n + 8 g + 4 hw + (0..3) ----
  float inv[MAPS];
#pragma unroll
  for (int m = 0; m < MAPS; ++m) {
    l[m] = la_half_sum(l[m]);
    const bool on = iq < qlen && !(l[m] == 0.f);  // (a NaN sum passes: it belongs in the output)
    inv[m] = on ? 1.f / l[m] : 0.f;
    if (p.lse && hw == 0 && iq < p.TqP)
      p.lse[(((int64_t)m * p.B + b) * p.H + h) * p.TqP + iq] = on ? mx[m] + log2f(l[m]) : INFINITY;
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
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = o[0][n][4 * g + e] * inv[0];
          if constexpr (MAPS == 2) v[e] = fmaf(-lam, o[MAPS - 1][n][4 * g + e] * inv[MAPS - 1], v[e]);
        }
        // (a row that sees nothing has all-zero probabilities, and V rows behind the keys are never loaded: v is 0, not NaN)
        la_store4<E>(ob + c, v[0], v[1], v[2], v[3]);
        if constexpr (MAPS == 2) {
          if (o2) {
            const float w = inv[MAPS - 1];
            la_store4<E>(o2 + c, o[MAPS - 1][n][4 * g] * w, o[MAPS - 1][n][4 * g + 1] * w, o[MAPS - 1][n][4 * g + 2] * w, o[MAPS - 1][n][4 * g + 3] * w);
          }
        }
      }
    }
}

template <typename E, int DK, int DV, int MAPS>
int launch_fwd(const LongP& p, hipStream_t st) {
  const size_t sm = 2 * (size_t)LA_TILE * (MAPS * DK + DV) * sizeof(E) + (p.table ? (2 * (p.max_distance + LA_PAD) + 4) * sizeof(float) : 0);
  const dim3 g((unsigned)((int64_t)p.nqt * p.B * p.H));
  const void* kern = p.table ? (const void*)attn_long_fwd_kernel<E, DK, DV, MAPS, true> : (const void*)attn_long_fwd_kernel<E, DK, DV, MAPS, false>;
  if (sm > 64 * 1024 && !ptpp_lds_limit(kern, (int)sm, "attention_long_fwd")) return PTPP_ELAUNCH;
  if (p.table) hipLaunchKernelGGL((attn_long_fwd_kernel<E, DK, DV, MAPS, true>), g, dim3(256), sm, st, p);
  else if constexpr (MAPS == 2) hipLaunchKernelGGL((attn_long_fwd_kernel<E, DK, DV, MAPS, false>), g, dim3(256), sm, st, p);
  PTPP_CHECK_LAUNCH("attention_long_fwd");
  return PTPP_OK;
}
template <typename E>
int dispatch_fwd(const LongP& p, int maps, hipStream_t st) {
  if (maps == 1) return p.dk <= 64 ? launch_fwd<E, 64, 64, 1>(p, st) : launch_fwd<E, 128, 128, 1>(p, st);
  return p.dk <= 32 ? launch_fwd<E, 32, 64, 2>(p, st) : launch_fwd<E, 64, 128, 2>(p, st);
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
  PTPP_CHECK_ARG(nqt * a->B * a->H < (1ll << 31) && nkt * a->B * a->H < (1ll << 31), "%s: too many tiles", who);
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
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->dtype == PTPP_F32) return dispatch_fwd<float>(p, a->maps, st);
  if (a->dtype == PTPP_BF16) return dispatch_fwd<bf16_raw>(p, a->maps, st);
  return dispatch_fwd<f16_raw>(p, a->maps, st);
}

int64_t ptpp_attention_long_ws_bwd(const LongP& p, int maps);
extern "C" int64_t ptpp_attention_long_ws_bytes(const ptpp_attention_long_args* a, int backward) {
  LongP p;
  if (ptpp_attention_long_params(a, backward, &p, "attention_long_ws_bytes") != PTPP_OK) return -1;
  return backward ? ptpp_attention_long_ws_bwd(p, a->maps) : 0;
}
