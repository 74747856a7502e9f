"""Attention over long sequences (learned bucketed position bias, differential) and the norm / gate / residual step against plain
64-bit implementations, with element-wise error bounds from the roundings that the kernels make:

* u = eps / 2 of the element type: outputs are rounded once; in 16-bit types the probabilities and dS are rounded once more as
  operands of the matrix instructions, which moves a sum over keys by at most u * sum |term|;
* rho: the relative error of a probability computed in f32 -- a dot product of dk terms, a fused multiply-add, the statistics and
  an exponential of an argument of size a are off by at most (dk + 16) * 2^-24 * a, which enters as a relative error of p.
"""
import ctypes
import math

import pytest
import torch

from conftest import ROOT  # noqa: F401

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_ulp(dt):
    return torch.finfo(dt).eps / 2


# ---------------------------------------------------------------------------------------------------------------------
# plain forms in 64 bits (CPU)
# ---------------------------------------------------------------------------------------------------------------------
def ref_bucket(dist, n_all, max_distance, bidirectional):
    n = n_all // 2 if bidirectional else n_all
    e = n // 2
    out = torch.empty_like(dist)
    for val in dist.unique().tolist():
        a = abs(val) if bidirectional else max(-val, 0)
        if a < e:
            b = a
        else:
            b = e
            while b < n - 1 and a ** (n - e) * e ** (b + 1 - e) >= max_distance ** (b + 1 - e) * e ** (n - e):
                b += 1
        out[dist == val] = b + (n if bidirectional and val > 0 else 0)
    return out


class RefAttention:
    """Everything of one call in 64 bits, utterance by utterance and head by head, plus the sums that the error bounds need."""

    def __init__(self, q, k, v, table, lam, lam_init, dout, heads, kv_heads, maps, max_distance=128, bidirectional=True, lengths=None,
                 q_lengths=None, q_start=None, causal=False, scale=None, dt=torch.float32):
        B, Tq, Tk = q.shape[0], q.shape[1], k.shape[1]
        dk = q.shape[2] // heads // maps
        dv = maps * dk
        q = q.double().reshape(B, Tq, heads, maps, dk)
        k = k.double().reshape(B, Tk, kv_heads, maps, dk)
        v = v.double().reshape(B, Tk, kv_heads, dv)
        do = dout.double().reshape(B, Tq, heads, dv) if dout is not None else None
        u = half_ulp(dt)
        up = u if dt != torch.float32 else 2.0 ** -24   # probabilities / dS as operands
        f = 2.0 ** -24
        # below 2^-14 the f16 values are 2^-24 apart: a rounding there is off by up to half of that, 2^-25, whatever the value.  It enters
        # once per output and, for the operands P (divided by a sum of at least 1) and dS, once per term of a sum
        tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
        scale = scale if scale is not None else dk ** -0.5
        z = torch.zeros
        self.out, self.out_b = z(B, Tq, heads, dv, dtype=torch.float64), z(B, Tq, heads, dv, dtype=torch.float64)
        self.g = {n: torch.zeros_like(t) for n, t in (("dq", q), ("dk", k), ("dv", v))}
        self.b = {n: torch.zeros_like(t) for n, t in (("dq", q), ("dk", k), ("dv", v))}
        if table is not None:
            self.g["dtable"], self.b["dtable"] = torch.zeros_like(table, dtype=torch.float64), torch.zeros_like(table, dtype=torch.float64)
        dlam, dlam_b = z(heads, dtype=torch.float64), z(heads, dtype=torch.float64)
        for b in range(B):
            nk = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
            nq = Tq if q_lengths is None else min(max(int(q_lengths[b]), 0), Tq)
            if nq == 0 or nk == 0:
                continue
            i = torch.arange(nq) + (int(q_start[b]) if q_start is not None else 0)
            dist = torch.arange(nk)[None] - i[:, None]
            see = torch.ones(nq, nk, dtype=torch.bool) if not causal else dist <= 0
            bk = ref_bucket(dist, table.shape[0], max_distance, bidirectional) if table is not None else None
            for h in range(heads):
                kh = h // (heads // kv_heads)
                ps, rhos = [], []
                L = 0.0
                if maps == 2:
                    lv = lam.double()[:, min(h, lam.shape[1] - 1)]
                    L = float((lv[0] @ lv[1]).exp() - (lv[2] @ lv[3]).exp() + lam_init)
                for m in range(maps):
                    s = q[b, :nq, h, m] @ k[b, :nk, kh, m].T * scale
                    mag = (q[b, :nq, h, m].abs() @ k[b, :nk, kh, m].abs().T * scale).amax()
                    if table is not None:
                        s = s + table.double()[:, h][bk]
                        mag = mag + table.double().abs().max()
                    s = s.masked_fill(~see, -math.inf)
                    mx = s.amax(-1, keepdim=True)
                    e = (s - torch.where(mx.isfinite(), mx, torch.zeros_like(mx))).exp()
                    l = e.sum(-1, keepdim=True)
                    ps.append(e / torch.where(l > 0, l, torch.ones_like(l)))
                    rhos.append(float((dk + 16) * f * (2 * mag + 4)) + nk * f * 0.05)
                c = [1.0, -L]
                vb = v[b, :nk, kh]
                w = sum(c[m] * ps[m] for m in range(maps))
                wa = sum(abs(c[m]) * ps[m] for m in range(maps))
                rho = max(rhos)
                self.out[b, :nq, h] = w @ vb
                self.out_b[b, :nq, h] = (up + rho + 8 * f) * (wa @ vb.abs()) + u * (w @ vb).abs() + tiny * (1 + (1 + abs(L)) * vb.abs().sum(0))
                if do is None:
                    continue
                dob = do[b, :nq, h]
                dp = dob @ vb.T
                dpe = (dob.abs() @ vb.abs().T) * (dv * f)             # dP in f32
                self.g["dv"][b, :nk, kh] += w.T @ dob
                self.b["dv"][b, :nk, kh] += (up + rho + (16 + 0.05 * nq) * f) * (wa.T @ dob.abs()) + tiny * dob.abs().sum(0)
                oe = (u + up + rho) * (wa @ vb.abs())                  # kept contexts: what centres dS in the dq pass
                De1 = (oe * dob.abs()).sum(-1, keepdim=True) * (1 + abs(L))
                for m in range(maps):
                    D = (ps[m] * dp).sum(-1, keepdim=True)
                    ds = c[m] * ps[m] * (dp - D)
                    mag = ps[m] * (dp.abs() + D.abs())
                    De = (rho + 32 * f) * mag.sum(-1, keepdim=True) + (ps[m] * dpe).sum(-1, keepdim=True)   # corrected D, f32
                    # dS in f32 (corrected D): relative error of p, the error of dP and of D
                    dse = abs(c[m]) * (rho * mag + ps[m] * (dpe + De) + 4 * f * mag)
                    kb, qb = k[b, :nk, kh, m], q[b, :nq, h, m]
                    self.g["dq"][b, :nq, h, m] = scale * (ds @ kb)
                    self.b["dq"][b, :nq, h, m] = scale * ((dse + up * (ds.abs() + abs(c[m]) * ps[m] * De1)) @ kb.abs()
                                                          + abs(c[m]) * (ps[m] * De1) @ kb.abs()
                                                          + (16 + 0.05 * nk) * f * ds.abs() @ kb.abs()) + u * scale * (ds @ kb).abs() \
                        + tiny * (1 + scale * max(1.0, abs(L)) * kb.abs().sum(0))
                    self.g["dk"][b, :nk, kh, m] += scale * (ds.T @ qb)
                    self.b["dk"][b, :nk, kh, m] += scale * ((dse + up * ds.abs() + (16 + 0.05 * nq) * f * ds.abs()).T @ qb.abs()) + tiny * scale * qb.abs().sum(0)
                    if table is not None:
                        nb = table.shape[0]
                        add = lambda t: torch.zeros(nb, dtype=torch.float64).index_add_(0, bk.reshape(-1), t.reshape(-1))  # noqa: E731
                        self.g["dtable"][:, h] += add(ds)
                        self.b["dtable"][:, h] += add(dse + 64 * f * ds.abs())
                    if m == 1:
                        dlam[h] -= D.sum()
                        dlam_b[h] += De.sum() + 64 * f * D.abs().sum()
        for n in ("dk", "dv"):  # rounded once, after the heads that share them have been added
            self.b[n] = self.b[n] + u * self.g[n].abs() + tiny
        if maps == 2 and do is not None:
            per = heads // lam.shape[1]
            G = dlam.view(lam.shape[1], per).sum(1)[:, None] if per > 1 else dlam[:, None]
            Gb = dlam_b.view(lam.shape[1], per).sum(1)[:, None] if per > 1 else dlam_b[:, None]
            lv = lam.double()
            e1, e2 = (lv[0] * lv[1]).sum(-1, keepdim=True).exp(), (lv[2] * lv[3]).sum(-1, keepdim=True).exp()
            self.g["dlam"] = torch.stack([G * e1 * lv[1], G * e1 * lv[0], -G * e2 * lv[3], -G * e2 * lv[2]])
            B_ = (Gb + 16 * dk * f * G.abs())
            self.b["dlam"] = torch.stack([B_ * e1 * lv[1].abs(), B_ * e1 * lv[0].abs(), B_ * e2 * lv[3].abs(), B_ * e2 * lv[2].abs()])
        self.out, self.out_b = self.out.flatten(2), self.out_b.flatten(2)
        for n, fl in (("dq", (B, Tq, -1)), ("dk", (B, Tk, -1)), ("dv", (B, Tk, -1))):
            self.g[n], self.b[n] = self.g[n].reshape(fl), self.b[n].reshape(fl)


def within(got, ref, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    bad = (got - ref).abs() - (bound + 1e-30)
    worst = float(bad.max()) if bad.numel() else 0.0
    at = int(bad.argmax()) if bad.numel() else 0
    assert worst <= 0, f"{what}: off by {float((got - ref).abs().flatten()[at]):.3e} where {float(bound.flatten()[at]):.3e} is allowed (value {float(ref.flatten()[at]):.3e})"


def make(maps, dt, B, Tq, Tk, heads, kv_heads, dk, buckets, seed=0, lam_heads=1, fused=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(B, Tq, heads * maps * dk).to(dt), r(B, Tk, kv_heads * maps * dk).to(dt), r(B, Tk, kv_heads * maps * dk).to(dt)
    table = (0.7 * r(buckets, heads)) if buckets else None
    lam = 0.3 * r(4, lam_heads, dk) if maps == 2 else None
    return q, k, v, table, lam, r(B, Tq, heads * maps * dk).to(dt)


def call(maps, q, k, v, table, lam, heads, **kw):
    from promptttspp_amd import functional as PF

    if maps == 2:
        return PF.attention_diff(q, k, v, lam, 0.35, heads, table=table, **kw)
    return PF.attention_bucket(q, k, v, table, heads, **kw)


def check_attention(dev, maps, dtype, B, Tq, Tk, heads, kv_heads, dk, buckets, lam_heads=1, seed=0, fused=False, garbage=False, train=True, **kw):
    dt = DT[dtype]
    q, k, v, table, lam, dout = make(maps, dt, B, Tq, Tk, heads, kv_heads, dk, buckets, seed, lam_heads)
    rkw = dict(kw)
    if fused:
        rkw.setdefault("q_lengths", kw.get("lengths"))
    ref = RefAttention(q, k, v, table, lam, 0.35, dout if train else None, heads, kv_heads, maps, dt=dt, **rkw)
    if garbage:  # whatever lies behind the lengths must not be read
        for t, n in ((k, kw.get("lengths")), (v, kw.get("lengths")), (q, rkw.get("q_lengths")), (dout, rkw.get("q_lengths"))):
            for b in range(B):
                if n is not None:
                    t[b, max(int(n[b]), 0):] = float("nan") if b % 2 else float("inf")
    kwd = {n: (torch.tensor(t, device=dev, dtype=torch.int32) if isinstance(t, (list, tuple)) else t) for n, t in kw.items()}
    if kv_heads != heads:
        kwd["kv_heads"] = kv_heads
    leaf = lambda t: None if t is None else t.to(dev).requires_grad_(train)  # noqa: E731
    table_d, lam_d = leaf(table), leaf(lam)
    if fused:
        qkv = leaf(torch.cat([q, k, v], dim=2))
        out = call(maps, qkv, None, None, table_d, lam_d, heads, **kwd)
        leaves = [qkv]
    else:
        leaves = [leaf(q), leaf(k), leaf(v)]
        out = call(maps, *leaves, table_d, lam_d, heads, **kwd)
    within(out, ref.out, ref.out_b, "out")
    if not train:
        return
    extra = [t for t in (table_d, lam_d) if t is not None]
    grads = torch.autograd.grad(out, leaves + extra, dout.to(dev))
    names = (["dtable"] if table is not None else []) + (["dlam"] if maps == 2 else [])
    for n, t in zip(names, grads[len(leaves):]):
        within(t, ref.g[n], ref.b[n], n)
    parts = grads[0].split([q.shape[2], k.shape[2], v.shape[2]], dim=2) if fused else grads[:3]
    for n, t in zip(("dq", "dk", "dv"), parts):
        within(t, ref.g[n], ref.b[n], n)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("maps,dk", [(1, 64), (1, 128), (2, 32), (2, 64)])
@pytest.mark.parametrize("T", [1, 2, 33, 129, 200])
def test_self_attention_sizes(dev, dtype, maps, dk, T):
    check_attention(dev, maps, dtype, 2, T, T, 2, 2, dk, 32, fused=True, lengths=[T, max(1, T - 37)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("Tq,Tk", [(1, 300), (16, 65), (17, 64), (63, 1), (65, 127), (128, 31), (31, 257), (130, 128)])
def test_cross_attention_sizes(dev, dtype, maps, Tq, Tk):
    check_attention(dev, maps, dtype, 2, Tq, Tk, 2, 1, 32, 16, lam_heads=2, q_start=[5, -3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("maps,dk", [(1, 8), (1, 40), (1, 80), (1, 120), (2, 8), (2, 16), (2, 40), (2, 56)])
def test_odd_head_widths(dev, dtype, maps, dk):
    check_attention(dev, maps, dtype, 2, 70, 90, 3, 3, dk, 8, lengths=[90, 41])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("maps", [1, 2])
def test_rows_without_keys_and_garbage_behind_the_lengths(dev, dtype, maps):
    """lengths of zero and one, NaN and infinities behind them, queries before the first key under the causal rule"""
    check_attention(dev, maps, dtype, 5, 70, 140, 2, 2, 64, 32, garbage=True, lengths=[140, 0, 1, 65, 64], q_lengths=[70, 70, 1, 0, 33],
                    q_start=[-40, 0, 0, 3, 100], causal=True)
    check_attention(dev, maps, dtype, 4, 140, 140, 2, 2, 64, 32, fused=True, garbage=True, lengths=[140, 0, 1, 77])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("B,T", [(2, 70), (2, 600), (70, 140)])
def test_rows_behind_the_queries_stay_zero_beside_infinities(dev, dtype, maps, B, T):
    """infinities and NaN among the valid keys and values reach the rows of valid queries only: outputs and query gradients behind
    ``q_lengths`` are exact zeros, as are those of a row that sees no key (few rows, many, and without gradients)"""
    dt, H, dk = DT[dtype], 2, 32
    q, k, v, table, lam, dout = make(maps, dt, B, T, T, H, H, dk, 16, seed=2)
    v[0, 3], k[1, 5], v[1, 40] = float("inf"), float("nan"), float("nan")
    n = [T - 21, T - 40] + [T] * (B - 2)
    kw = dict(q_lengths=torch.tensor(n, device=dev, dtype=torch.int32))
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table) + ((lam,) if maps == 2 else ())]
    full = leaves + [None] * (5 - len(leaves))
    out = call(maps, *full, H, **kw)
    dq, dk_, dv = torch.autograd.grad(out, leaves[:3], dout.to(dev))
    with torch.no_grad():
        few = call(maps, full[0][:, :24].contiguous(), *full[1:], H, q_lengths=torch.full((B,), 9, device=dev))
    for b in range(2):
        for t in (out, dq):
            assert not t[b, n[b]:].any()
            assert not bool(torch.isfinite(t[b, :n[b]]).all())
        assert not few[b, 9:].any() and not bool(torch.isfinite(few[b, :9]).all())
    assert bool(torch.isfinite(out[2:]).all()) and bool(torch.isfinite(dk_[2:]).all())
    # rows before the first key under the causal rule see nothing
    with torch.no_grad():
        a = call(maps, *full, H, causal=True, q_start=torch.full((B,), -10, device=dev, dtype=torch.int32))
    assert not a[:, :10].any() and not bool(torch.isfinite(a[0, 20:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("bidirectional", [True, False])
def test_causal(dev, dtype, maps, bidirectional):
    check_attention(dev, maps, dtype, 2, 300, 300, 2, 2, 32, 32, fused=True, lengths=[300, 211], causal=True, bidirectional=bidirectional)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("buckets,max_distance,bidirectional", [(2, 1024, False), (4, 2, True), (6, 5, True), (64, 128, True), (128, 1024, True),
                                                                (128, 777, False), (32, 20, False)])
def test_bucket_layouts(dev, maps, buckets, max_distance, bidirectional):
    check_attention(dev, maps, "bf16", 2, 260, 260, 2, 2, 64, buckets, fused=True, lengths=[260, 131], max_distance=max_distance,
                    bidirectional=bidirectional)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("maps,heads,kv_heads,lam_heads", [(1, 4, 1, 1), (1, 6, 2, 1), (2, 4, 2, 4), (2, 3, 1, 1), (2, 12, 4, 1)])
def test_shared_key_heads(dev, dtype, maps, heads, kv_heads, lam_heads):
    check_attention(dev, maps, dtype, 2, 75, 75, heads, kv_heads, 32, 16, fused=True, lam_heads=lam_heads, lengths=[75, 50])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_differential_without_a_table(dev, dtype):
    check_attention(dev, 2, dtype, 3, 150, 150, 2, 2, 64, 0, fused=True, lengths=[150, 64, 1])


@pytest.mark.gpu
def test_positions_far_beyond_the_table_and_large_scores(dev):
    """distances that only fit 32 bits with care, and scores whose exponentials overflow without the running maximum"""
    check_attention(dev, 1, "bf16", 2, 40, 200, 2, 2, 64, 32, q_start=[2 ** 31 - 1, -2 ** 31], lengths=[200, 90])
    check_attention(dev, 1, "f32", 1, 64, 200, 2, 2, 64, 32, scale=3.0)
    check_attention(dev, 2, "bf16", 1, 64, 200, 2, 2, 32, 32, scale=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("dtype,dk", [("bf16", 64), ("f16", 32), ("f32", 64), ("bf16", 40)])
@pytest.mark.parametrize("Tk", [1, 63, 500, 2100])
def test_one_query_against_a_memory(dev, maps, dtype, dk, Tk):
    lens = [Tk, max(1, Tk // 3), max(1, Tk - 64)]
    check_attention(dev, maps, dtype, 3, 1, Tk, 4, 2, dk, 32, train=False, garbage=True, lengths=lens, q_start=[n - 1 for n in lens], causal=True,
                    bidirectional=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dk", [("bf16", 64), ("f16", 32), ("f32", 64)])
@pytest.mark.parametrize("B,Tq,Tk,heads,kv_heads", [(3, 1, 63, 4, 2), (3, 1, 2100, 4, 2), (2, 5, 200, 6, 2), (2, 1, 120, 12, 1), (150, 1, 600, 4, 2)])
def test_lam_per_head_where_a_block_takes_several_heads(dev, dtype, dk, B, Tq, Tk, heads, kv_heads):
    """few queries without gradients: heads that share their keys lie side by side in one block, each with its own lam -- short memories and
    large batches (one range of keys per block) and long memories (ranges joined afterwards)"""
    lens = [max(Tq, Tk - 37 * b % Tk) for b in range(B)]
    check_attention(dev, 2, dtype, B, Tq, Tk, heads, kv_heads, dk, 16, lam_heads=heads, train=False, garbage=True, lengths=lens,
                    q_start=[n - Tq for n in lens], causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("Tq", [2, 5, 16, 24])
def test_few_queries_against_a_long_memory(dev, maps, Tq):
    check_attention(dev, maps, "bf16", 2, Tq, 1500, 4, 1, 64, 32, train=False, lengths=[1500, 777], q_start=[1500 - Tq, 777 - Tq], causal=True)
    check_attention(dev, maps, "f32", 1, Tq, 1500, 2, 2, 32, 32, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("maps,dk", [(1, 64), (1, 128), (2, 32), (2, 64)])
@pytest.mark.parametrize("causal", [False, True])
def test_batches_that_fill_the_chip(dev, dtype, maps, dk, causal):
    """more than 256 blocks of 128 rows: the launch shapes of full batches (few rows take others), lengths of zero and garbage included"""
    B = 66 if dk != 128 else 44
    lens = [(37 * b) % 150 for b in range(B)]
    lens[1] = 149
    check_attention(dev, maps, dtype, B, 149, 149, 6 if dk == 128 else 4, 2, dk, 32, fused=True, garbage=True, lengths=lens, causal=causal, bidirectional=not causal)


@pytest.mark.gpu
@pytest.mark.parametrize("maps,dk", [(1, 64), (1, 128), (2, 32), (2, 64)])
@pytest.mark.parametrize("B,T", [(1, 700), (16, 500)])
@pytest.mark.parametrize("power", [-14, -9, 12])
def test_f16_gradients_of_any_size(dev, maps, dk, B, T, power):
    """Gradients that arrive at 2^-14 (what they are without a loss scale) to 2^12 keep the accuracy of those of order one.  The bounds are those
    of the same gradient times 2^20, divided by it -- dS is an operand whose 2^-25 per term then counts for nothing, since a column of it
    is scaled to 2^11 and more, and its error is 2^-36 of the column's largest term -- and the output's own rounding, 2^-25 below 2^-14."""
    H = 2
    q, k, v, table, lam, dout = make(maps, torch.float16, B, T, T, H, H, dk, 32, seed=4)
    dout = (dout.double() * 2.0 ** power).half()
    lens = [T - 11 * b for b in range(B)]
    up = 2.0 ** 20
    ref = RefAttention(q, k, v, table, lam, 0.35, dout.double() * up, H, H, maps, dt=torch.float16, lengths=lens, q_lengths=lens)
    out_tiny = 2.0 ** -25
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table) + ((lam,) if maps == 2 else ())]
    full = leaves + [None] * (5 - len(leaves))
    rows = torch.tensor(lens, device=dev, dtype=torch.int32)
    out = call(maps, *full, H, lengths=rows, q_lengths=rows)
    grads = torch.autograd.grad(out, leaves, dout.to(dev))
    for n, t in zip(("dq", "dk", "dtable") + (("dlam",) if maps == 2 else ()), grads[:2] + grads[3:]):
        within(t, ref.g[n] / up, ref.b[n] / up + (out_tiny if n in ("dq", "dk") else 0.0), n)
    # P is not scaled: a term of dv is off by half a step of f16, 2^-25, of the gradient that it weighs
    weigh = dout.double().abs().view(B, T, H, -1) * (torch.arange(T)[None] < torch.tensor(lens)[:, None])[:, :, None, None]
    c = 1.0 if maps == 1 else 2.0 * (1.0 + float(((lam.double()[0] * lam.double()[1]).sum(-1).exp() + (lam.double()[2] * lam.double()[3]).sum(-1).exp()).max()))
    within(grads[2], ref.g["dv"] / up, ref.b["dv"] / up + out_tiny * (1 + c * weigh.sum(1, keepdim=True).expand(B, T, H, -1).reshape(B, T, -1)), "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("maps,dk", [(1, 64), (1, 128), (2, 32), (2, 64)])
@pytest.mark.parametrize("B,T,causal", [(3, 2, False), (3, 2, True), (3, 7, False), (3, 7, True), (3, 33, False), (3, 33, True), (3, 64, False), (3, 64, True),
                                        (90, 64, False), (90, 64, True), (2, 300, True), (50, 150, True)])
def test_query_gradients_of_short_rows(dev, dtype, maps, dk, B, T, causal):
    """Where a row sees few keys the centre D of dS must not carry the rounding of the kept 16-bit context: dq is off by the f32 errors (those of
    the f32 form), by dS rounded once as an operand -- half a step of sum |dS| |k| -- and by its own rounding; a row with one key gives next
    to nothing.  Long sequences: the first 64 rows under the causal rule"""
    dt, H = DT[dtype], 2
    u, tiny = half_ulp(dt), 2.0 ** -25 if dtype == "f16" else 0.0
    q, k, v, _, lam, dout = make(maps, dt, B, T, T, H, H, dk, 0, seed=13)
    table = torch.zeros(4, H) if maps == 1 else None
    lens = [max(1, T - 5 * b % T) for b in range(B)]
    kw = dict(lengths=lens, q_lengths=lens, causal=causal)
    ref = RefAttention(q, k, v, table, lam, 0.35, dout, H, H, maps, dt=torch.float32, **kw)
    half = torch.zeros(B, T, H, maps, dk, dtype=torch.float64)
    split = lambda t, *n: t.double().view(B, T, H, *n)  # noqa: E731
    Q, K, V, G = split(q, maps, dk), split(k, maps, dk), split(v, -1), split(dout, -1)
    L = 0.0 if maps == 1 else float((lam.double()[0, 0] @ lam.double()[1, 0]).exp() - (lam.double()[2, 0] @ lam.double()[3, 0]).exp() + 0.35)
    for b, n in enumerate(lens):
        see = torch.ones(n, n, dtype=torch.bool).tril() if causal else torch.ones(n, n, dtype=torch.bool)
        for h in range(H):
            dp = G[b, :n, h] @ V[b, :n, h].T
            for m in range(maps):
                P = (Q[b, :n, h, m] @ K[b, :n, h, m].T * dk ** -0.5).masked_fill(~see, -math.inf).softmax(-1)
                dS = (1.0, -L)[m] * P * (dp - (P * dp).sum(-1, keepdim=True))
                half[b, :n, h, m] = dk ** -0.5 * (u * dS.abs()) @ K[b, :n, h, m].abs()
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    rows = torch.tensor(lens, device=dev, dtype=torch.int32)
    out = call(maps, *leaves, None if table is None else table.to(dev), None if lam is None else lam.to(dev), H, lengths=rows, q_lengths=rows, causal=causal)
    (dq,) = torch.autograd.grad(out, leaves[:1], dout.to(dev))
    bound = ref.b["dq"] + half.reshape(B, T, -1) + u * ref.g["dq"].abs() + tiny
    within(dq[:, :64], ref.g["dq"][:, :64], bound[:, :64], "dq")


@pytest.mark.gpu
@pytest.mark.parametrize("maps,dk", [(1, 64), (2, 32), (2, 64)])
@pytest.mark.parametrize("B,T,at", [(2, 300, 0), (2, 300, 200), (60, 140, 0)])
def test_one_value_of_another_size(dev, maps, dk, B, T, at):
    """a key that next to no query sees, with values 10^4 times the others': nothing of it shows in the others' gradients (f32)"""
    H = 2
    q, k, v, table, lam, dout = make(maps, torch.float32, B, T, T, H, H, dk, 16, seed=21)
    q.view(B, T, H, maps, dk)[..., 0] = 20.0
    k.view(B, T, H, maps, dk)[..., 0] = 0.0
    k.view(B, T, H, maps, dk)[:, at, ..., 0] = -4.0 * dk ** 0.5   # 80 below the others: seen with 10^-34
    v[:, at] *= 1e4
    ref = RefAttention(q, k, v, table, lam, 0.35, dout, H, H, maps)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table) + ((lam,) if maps == 2 else ())]
    full = leaves + [None] * (5 - len(leaves))
    grads = torch.autograd.grad(call(maps, *full, H), leaves, dout.to(dev))
    seen = torch.ones(T, dtype=torch.bool)
    seen[at] = False
    for n, t in zip(("dq", "dk", "dv"), grads):
        rows = slice(None) if n == "dq" else seen
        within(t[:, rows], ref.g[n][:, rows], ref.b[n][:, rows], n)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_table_entries_of_minus_1e30_hide_keys(dev, maps):
    test_table_entries_that_hide_keys(dev, maps, -1e30, 150, 150)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dk", [32, 64])
@pytest.mark.parametrize("B", [4, 12])
def test_lam_gradient_follows_the_sign_of_the_gradient(dev, dtype, dk, B):
    """Every rounding of the gradient of lam has to follow the sign of what arrives: a bias that does not adds up over all rows.  With each query
    given twice (rows 2 i and 2 i + 1) the pairs' roundings are each other's mirror image, whatever the matrix instructions do: the gradient of
    -dout is the negative one up to the order of a sum in 64 bits and one rounding to f32, 2^-24 of it"""
    T, H = 700, 4
    q, k, v, _, lam, dout = make(2, DT[dtype], B, T, T, H, H, dk, 0, seed=11)
    q, dout = (t[:, ::2].repeat_interleave(2, dim=1).to(dev) for t in (q, dout))
    k, v = k.to(dev), v.to(dev)
    lam = lam.to(dev).requires_grad_()
    out = call(2, q, k, v, None, lam, H)
    plus, minus = (torch.autograd.grad(out, lam, g, retain_graph=True)[0] for g in (dout, -dout))
    assert bool(((plus + minus).abs() <= 2.0 ** -22 * plus.abs()).all()), float(((plus + minus) / plus).abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_full_batches_of_unequal_sides(dev, maps):
    """few queries against many keys and the other way round in batches large enough for either launch shape of either pass"""
    check_attention(dev, maps, "bf16", 150, 140, 30, 2, 2, 40, 16, q_start=[b - 70 for b in range(150)])
    check_attention(dev, maps, "bf16", 150, 33, 260, 2, 1, 40, 16, causal=True, q_start=[2 * b for b in range(150)])


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_strided_operands(dev, maps):
    """slices of a wider tensor, batch strides that are no multiple of the rows, a key tensor shared by the whole batch"""
    dk, H, B, T = 32, 2, 3, 70
    q, k, v, table, lam, dout = make(maps, torch.bfloat16, B, T, T, H, H, dk, 16)
    k = k[:1].expand(B, -1, -1).contiguous()
    C = H * maps * dk
    ref = RefAttention(q, k, v, table, lam, 0.35, dout, H, H, maps, dt=torch.bfloat16)
    big = torch.zeros(B, T + 3, C + 24, dtype=torch.bfloat16, device=dev)
    big[:, 1:T + 1, 8:C + 8] = q.to(dev)
    qs = big[:, 1:T + 1, 8:C + 8].detach().requires_grad_()
    k1 = k[:1].to(dev).requires_grad_()
    vs = v.to(dev).requires_grad_()
    out = call(maps, qs, k1.expand(B, -1, -1), vs, table.to(dev), None if lam is None else lam.to(dev), H)
    within(out, ref.out, ref.out_b, "out")
    dq, dk1, dv = torch.autograd.grad(out, [qs, k1, vs], dout.to(dev))
    within(dq, ref.g["dq"], ref.b["dq"], "dq")
    within(dv, ref.g["dv"], ref.b["dv"], "dv")
    # torch adds the utterances' gradients of the shared keys: three bf16 values, rounded after each addition
    s = ref.g["dk"].abs().sum(0, keepdim=True)
    within(dk1, ref.g["dk"].sum(0, keepdim=True), ref.b["dk"].sum(0, keepdim=True) + 3 * 2.0 ** -8 * s, "dk")
    # a gradient that torch hands over as an expanded scalar
    (ones,) = torch.autograd.grad(call(maps, qs, k1.expand(B, -1, -1), vs, table.to(dev), None if lam is None else lam.to(dev), H).sum(), [vs])
    ref1 = RefAttention(q, k, v, table, lam, 0.35, torch.ones_like(dout), H, H, maps, dt=torch.bfloat16)
    within(ones, ref1.g["dv"], ref1.b["dv"], "dv of a sum")


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_attention_gradients_against_differences(dev, maps):
    """(L(w + h d) - L(w - h d)) / 2h along a random direction of all inputs, f32: the third-order term and the f32 rounding of L are
    both below 1e-3 of the value at h = 1e-2"""
    B, T, H, dk = 2, 50, 2, 32
    q, k, v, table, lam, dout = (t if t is None else t.to(dev) for t in make(maps, torch.float32, B, T, T, H, H, dk, 16, seed=3))
    ws = [t for t in (q, k, v, table, lam) if t is not None]
    g = torch.Generator(device=dev).manual_seed(1)
    ds = [torch.randn(t.shape, device=dev, generator=g) for t in ws]

    def loss(step):
        w = [(t.double() + step * d.double()).float() for t, d in zip(ws, ds)]
        w = w + [None] * (5 - len(w))
        return float((call(maps, w[0], w[1], w[2], w[3], w[4], H).double() * dout.double()).sum())

    leaves = [t.clone().requires_grad_() for t in ws]
    full = leaves + [None] * (5 - len(leaves))
    out = call(maps, full[0], full[1], full[2], full[3], full[4], H)
    ana = sum(float((gr.double() * d.double()).sum()) for gr, d in zip(torch.autograd.grad(out, leaves, dout), ds))
    num = (loss(1e-2) - loss(-1e-2)) / 2e-2
    num2 = (loss(5e-3) - loss(-5e-3)) / 1e-2
    num = (4 * num2 - num) / 3  # (the h^2 term cancelled)
    assert abs(ana - num) < 5e-3 * max(1.0, abs(ana)), (ana, num)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
def test_attention_same_bits_every_run_and_on_another_stream(dev, maps):
    q, k, v, table, lam, dout = (t if t is None else t.to(dev) for t in make(maps, torch.bfloat16, 3, 333, 333, 4, 2, 64, 32, seed=5))

    def once():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table, lam) if t is not None]
        full = leaves + [None] * (5 - len(leaves))
        out = call(maps, *full, 4, kv_heads=2, causal=True)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    a = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = once()
    c = once()  # (beside the other stream's call)
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("Tq", [1, 70])
def test_attention_in_captured_graphs(dev, maps, Tq):
    """forward and backward captured, replayed with new inputs between eager calls; two graphs do not share a workspace"""
    B, Tk, H = 2, 900, 4
    sets = [[t if t is None else t.to(dev) for t in make(maps, torch.bfloat16, B, Tq, Tk, H, 2, 64, 32, seed=s)] for s in (1, 2, 3)]

    def step(q, k, v, table, lam, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table, lam) if t is not None]
        full = leaves + [None] * (5 - len(leaves))
        out = call(maps, *full, H, kv_heads=2)
        with torch.no_grad():
            serve = call(maps, q, k, v, table, lam, H, kv_heads=2)
        return [serve, out.detach(), *torch.autograd.grad(out, leaves, dout)]

    graphs = []
    for n in (0, 1):
        static = [None if t is None else t.clone() for t in sets[n]]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(*static)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(*static)
        graphs.append((gr, static, outs))
    for trip in range(3):
        want = []
        for n, (gr, static, outs) in enumerate(graphs):
            src = sets[(trip + n) % 3]
            want.append([t.clone() for t in step(*src)])
            for d, t in zip(static, src):
                if t is not None:
                    d.copy_(t)
        for gr, _, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for (gr, _, outs), w in zip(graphs, want):
            for o, t in zip(outs, w):
                assert torch.equal(o, t)


@pytest.mark.gpu
def test_attention_only_some_inputs_need_gradients(dev):
    from promptttspp_amd import functional as PF

    q, k, v, table, lam, dout = (t if t is None else t.to(dev) for t in make(1, torch.float32, 2, 40, 40, 2, 2, 64, 16))
    table.requires_grad_()
    (dt,) = torch.autograd.grad(PF.attention_bucket(q, k, v, table, 2), [table], dout)
    ref = RefAttention(q.cpu(), k.cpu(), v.cpu(), table.detach().cpu(), None, 0, dout.cpu(), 2, 2, 1)
    within(dt, ref.g["dtable"], ref.b["dtable"], "dtable")


@pytest.mark.gpu
@pytest.mark.parametrize("maps,buckets,lam_heads", [(1, 32, 1), (2, 32, 1), (2, 32, 4), (2, 0, 4), (2, 0, 1)])
@pytest.mark.parametrize("B,T", [(2, 70), (40, 140)])
def test_parameter_gradients_added_in_place(dev, maps, buckets, lam_heads, B, T):
    """with the flat gradient buffer two passes leave exactly twice the gradient of the table and of the lam vectors (the sums have a fixed order,
    and doubling is exact); the inputs' gradients come back as ever, and a parameter that is frozen stays out"""
    from promptttspp_amd import functional as PF
    from promptttspp_amd.parallel import FlatGradReducer

    heads = 4
    q, k, v, table, lam, dout = (t if t is None else t.to(dev) for t in make(maps, torch.float32, B, T, T, heads, 2, 32, buckets, seed=7, lam_heads=lam_heads))
    table, lam = (None if t is None else torch.nn.Parameter(t) for t in (table, lam))
    params = [p for p in (table, lam) if p is not None]
    q.requires_grad_()
    want = torch.autograd.grad(call(maps, q, k, v, table, lam, heads, kv_heads=2, causal=True), [q, *params], dout)
    assert all(bool(g.any()) for g in want)
    try:
        red = FlatGradReducer(params)
        red.zero_grad()
        for _ in range(2):
            q.grad = None
            call(maps, q, k, v, table, lam, heads, kv_heads=2, causal=True).backward(dout)
        red.finish()
        torch.cuda.synchronize()
        assert torch.equal(q.grad, want[0])
        for p, w in zip(params, want[1:]):
            assert torch.equal(p.grad, 2 * w)
        if len(params) == 2:
            red.zero_grad()
            table.requires_grad_(False)
            call(maps, q, k, v, table, lam, heads, kv_heads=2, causal=True).backward(dout)
            red.finish()
            torch.cuda.synchronize()
            assert torch.equal(lam.grad, want[2]) and not table.grad.any()
    finally:
        PF.enable_direct_grads(False)


@pytest.mark.gpu
def test_long_batch_strides_pass_32_bits(dev):
    """the second utterance of a kept memory lies more than 2^31 elements behind the first"""
    from promptttspp_amd import functional as PF

    H, dk, T = 2, 64, 100
    room = 2 ** 31 // (H * dk) + 64  # positions of room per utterance
    mem = torch.empty(2 * room * H * dk, device=dev, dtype=torch.bfloat16).view(2, room, H * dk)
    q, k, v, table, _, _ = make(1, torch.bfloat16, 2, 1, T, H, H, dk, 32)
    vals = torch.zeros(2, T, H * dk, dtype=torch.bfloat16)
    mem[:, :T] = k.to(dev)
    vals = v.to(dev)
    ref = RefAttention(q, k, v, table, None, 0, None, H, H, 1, dt=torch.bfloat16, q_start=[T - 1, T - 1])
    with torch.no_grad():
        out = PF.attention_bucket(q.to(dev), mem[:, :T], vals, table.to(dev), H, q_start=torch.tensor([T - 1, T - 1], device=dev))
    within(out, ref.out, ref.out_b, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("name", ["lengths", "q_lengths", "q_start"])
def test_attention_rows_refilled_before_backward_are_refused(dev, maps, name):
    """lengths and positions that forward read are saved like any other tensor: refilled in place, backward raises; one of another type was
    copied, and one refilled after backward, or restored by a hook at another address, changes nothing"""
    q, k, v, table, lam, dout = (t if t is None else t.to(dev) for t in make(maps, torch.bfloat16, 2, 40, 40, 2, 2, 32, 16, seed=8))
    full = [t if t is None else t.requires_grad_() for t in (q, k, v, table, lam)]
    leaves = [t for t in full if t is not None]

    def run(rows, touch=None):
        out = call(maps, *full, 2, causal=name == "q_start", **{name: rows})
        if touch is not None:
            rows.fill_(touch)
        return torch.autograd.grad(out, leaves, dout)

    i32 = lambda *n: torch.tensor(n, device=dev, dtype=torch.int32)  # noqa: E731
    want = run(i32(30, 17))
    with pytest.raises(RuntimeError, match="inplace"):
        run(i32(30, 17), touch=5)
    for got in (run(i32(30, 17).long(), touch=5), run(torch.tensor([30, 17]), touch=5)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode():
        rows = i32(30, 17)
    assert all(torch.equal(a, b) for a, b in zip(run(rows), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        assert all(torch.equal(a, b) for a, b in zip(run(i32(30, 17)), want))


@pytest.mark.gpu
def test_residual_norm_lengths_refilled_before_backward_are_refused(dev):
    from promptttspp_amd import functional as PF

    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    leaves = [r(2, 30, 64).requires_grad_(), r(2, 30, 64).requires_grad_(), r(64).requires_grad_(), r(64).requires_grad_()]
    dy, dz = r(2, 30, 64), r(2, 30, 64)

    def run(rows, touch=None):
        out = PF.residual_norm(leaves[0], leaves[1], post=(leaves[2], None), pre=(leaves[3], None), lengths=rows)
        if touch is not None:
            rows.fill_(touch)
        return torch.autograd.grad(out, leaves, (dy, dz))

    want = run(torch.tensor([22, 9], device=dev, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="inplace"):
        run(torch.tensor([22, 9], device=dev, dtype=torch.int32), touch=30)
    with torch.inference_mode():
        rows = torch.tensor([22, 9], device=dev, dtype=torch.int32)
    for got in (run(torch.tensor([22, 9], device=dev), touch=30), run(rows)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t.clone()):
        assert all(torch.equal(a, b) for a, b in zip(run(torch.tensor([22, 9], device=dev, dtype=torch.int32)), want))


def _tangent_calls(dev):
    """every operator with one input that carries a tangent and nothing that requires a gradient"""
    from promptttspp_amd import functional as PF

    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    return [lambda: PF.attention_bucket(dual(z(1, 4, 96)), None, None, z(16, 1), 1), lambda: PF.attention_bucket(z(1, 4, 96), None, None, dual(z(16, 1)), 1),
            lambda: PF.attention_diff(z(1, 4, 96), None, None, dual(z(4, 1, 16)), 0.1, 1), lambda: PF.residual_norm(dual(z(1, 4, 32)), pre=(z(32), None)),
            lambda: PF.residual_norm(z(1, 4, 32), gate=dual(z(32)))]


def test_open_forward_levels_and_traces_make_nodes(monkeypatch):
    """(no GPU: where the calls go) a tangent or a trace never meets a launch that passes autograd by"""
    from promptttspp_amd import functional as PF

    class Node(Exception):
        pass

    def node(*a):
        raise Node

    for fn in (PF.AttentionLongFn, PF.ResidualNormFn):
        monkeypatch.setattr(fn, "apply", node)
    with torch.autograd.forward_ad.dual_level():
        for f in _tangent_calls("cpu"):
            with pytest.raises(Node):
                f()
    t = torch.zeros(16, 1)
    for f in (lambda x: PF.attention_bucket(x, None, None, t, 1), lambda x: PF.residual_norm(x)[0]):
        with torch.no_grad(), pytest.raises(Node):
            torch.jit.trace(f, (torch.zeros(1, 4, 96),), check_trace=False)


@pytest.mark.gpu
def test_tangents_are_refused(dev):
    with torch.autograd.forward_ad.dual_level():
        for f in _tangent_calls(dev):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()
    for f in _tangent_calls(dev):  # (no level open: make_dual refuses, nothing else is left behind)
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_run_the_kernels(dev, grad):
    """a traced function computes what the function computes, with other inputs, other lengths and their gradients too"""
    from promptttspp_amd import functional as PF

    g = torch.Generator(device=dev).manual_seed(6)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    ws = [t.requires_grad_(grad) for t in (r(16, 2), 0.2 * r(4, 1, 32), r(2, 128), r(128))]

    def fun(x, lengths, table, lam, gate, w):  # (torch takes nothing that requires a gradient as a constant of a trace)
        a = PF.attention_bucket(x, None, None, table, 2, lengths=lengths)
        b = PF.attention_diff(x, None, None, lam, 0.3, 2, lengths=lengths, causal=True)
        return PF.residual_norm(a, b, gate=gate, post=(w, None), pre=(w, None), kind="rms", lengths=lengths)

    inputs = [(r(2, 50, 384), torch.tensor(n, device=dev, dtype=torch.int32)) for n in ([50, 31], [7, 50], [0, 1])]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(fun, (*inputs[0], *ws), check_trace=False)
        for x, n in inputs:
            got, want = traced(x, n, *ws), fun(x, n, *ws)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
            if grad:
                for a, b in zip(torch.autograd.grad(got[0].sum() + got[1].square().sum(), ws), torch.autograd.grad(want[0].sum() + want[1].square().sum(), ws)):
                    assert torch.equal(a, b)


def test_bucket_edges_are_the_whole_number_solution():
    from promptttspp_amd import ops

    for n, D, bi in ((32, 128, True), (32, 128, False), (64, 128, True), (8, 128, True), (128, 1024, False), (6, 5, True), (2, 1024, False), (4, 2, True)):
        e, edges, cnt = ops.bucket_edges(n, D, bi)
        d = torch.arange(-2 * D, 2 * D + 1)
        want = ref_bucket(d, n, D, bi)
        half = n // 2 if bi else n
        a = d.abs() if bi else (-d).clamp(min=0)
        got = torch.where(a < e, a, torch.full_like(a, e))
        for t in range(cnt):
            got = got + (a >= edges[t])
        got = got + half * ((d > 0) & bi)
        assert torch.equal(got, want), (n, D, bi)
    for bad in ((3, 128, True), (130, 128, True), (2, 128, True), (1, 128, False), (32, 8, True), (32, 1025, True), (0, 10, False)):
        with pytest.raises(ValueError):
            ops.bucket_edges(*bad)


def test_attention_refusals_on_the_host():
    """what the C entry refuses before any launch (no GPU needed: the pointers are never followed)"""
    from promptttspp_amd import _lib, ops

    lib = _lib.load()
    e, edges, cnt = ops.bucket_edges(32, 128, True)

    def args(**kw):
        a = _lib.AttentionLongArgs()
        for n in ("q", "k", "v", "out", "table"):
            setattr(a, n, 4096)
        a.B, a.Tq, a.Tk, a.H, a.Hk, a.dk, a.maps, a.dtype = 2, 10, 10, 2, 2, 64, 1, _lib.BF16
        a.ldq = a.ldk = a.ldv = a.ldo = a.lddo = a.lddq = a.lddk = a.lddv = 128
        a.sq = a.sk = a.sv = a.so = a.sdo = a.sdq = a.sdk = a.sdv = 1280
        a.nbuckets, a.bidirectional, a.max_distance, a.nexact, a.nedges, a.edges = 32, 1, 128, e, cnt, ctypes.addressof(edges)
        a.scale = 0.125
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(args()), 0) >= 0
    back = {n: 4096 for n in ("dout", "dq", "dk_out", "dv", "dtable", "lse")}
    assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(args(**back)), 1) > 0
    descending = (ctypes.c_int32 * 16)(*([20] + [19] * 15))
    bad = [dict(q=None), dict(out=None), dict(dtype=7), dict(maps=3), dict(B=0), dict(Tq=0), dict(Tk=-1), dict(H=3), dict(Hk=0), dict(dk=60), dict(dk=136),
           dict(dk=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=4098), dict(ldq=127), dict(ldk=120),
           dict(sv=1281), dict(sk=-1280), dict(table=None), dict(maps=2, dk=72, lam=4096, lam_heads=1), dict(maps=2, dk=32), dict(maps=2, dk=32, lam=4096, lam_heads=3),
           dict(nbuckets=31), dict(nbuckets=130), dict(nexact=9), dict(nedges=3), dict(edges=None), dict(max_distance=8), dict(max_distance=1025),
           dict(edges=ctypes.addressof(descending)), dict(B=2 ** 30, Tq=2 ** 20)]
    for kw in bad:
        a = args(**kw)
        assert lib.ptpp_attention_long_fwd(ctypes.byref(a), None) == -1, kw
        assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(a), 0) < 0, kw
    assert lib.ptpp_attention_long_fwd(None, None) == -1
    for kw in (dict(back, lse=None), dict(back, lse=4100), dict(back, dtable=None), dict(back, dq=None), dict(back, lddv=64), dict(back, ws=None, ws_bytes=1 << 30),
               dict(back, ws=4096, ws_bytes=16), dict(back, ws=4104, ws_bytes=1 << 30)):
        assert lib.ptpp_attention_long_bwd(ctypes.byref(args(**kw)), None) == -1, kw
    assert b"attention_long" in lib.ptpp_last_error()


def test_misaligned_side_arguments_are_refused():
    """the second map's context is stored in 16-byte pieces like the output; tables, statistics and lengths are words"""
    from promptttspp_amd import _lib

    lib = _lib.load()

    def attention(**kw):
        a = _lib.AttentionLongArgs()
        for n in ("q", "k", "v", "out", "lam", "lse", "out2"):
            setattr(a, n, 4096)
        a.B, a.Tq, a.Tk, a.H, a.Hk, a.dk, a.maps, a.lam_heads, a.dtype, a.scale = 2, 600, 10, 2, 2, 64, 2, 1, _lib.BF16, 0.125
        a.ldq = a.ldk = a.ldv = a.ldo = 256
        a.sq = a.so = 600 * 256
        a.sk = a.sv = 2560
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(attention()), 0) >= 0
    for kw in (dict(out2=4104), dict(lam=4097), dict(lse=4098), dict(k_lengths=4097), dict(q_lengths=4097), dict(q_start=4098), dict(table=4098)):
        assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(attention(**kw)), 0) < 0, kw
        assert lib.ptpp_attention_long_fwd(ctypes.byref(attention(**kw)), None) == -1, kw
    for kw in (dict(stats=4098), dict(lengths=4097)):
        n = _lib.ResidualNormArgs()
        n.f = n.y = 4096
        n.B, n.T, n.C, n.gate_rows, n.dtype, n.scale, n.eps = 2, 3, 64, 1, _lib.F32, 1.0, 1e-5
        for k, x in kw.items():
            setattr(n, k, x)
        assert lib.ptpp_residual_norm_fwd(ctypes.byref(n), None) == -1, kw


def test_launches_beyond_the_grid_are_refused():
    """a launch holds fewer than 2^32 threads: more one-query blocks, or more rows of a norm, are refused before any launch"""
    from promptttspp_amd import _lib, ops

    lib = _lib.load()
    e, edges, cnt = ops.bucket_edges(32, 128, True)
    a = _lib.AttentionLongArgs()
    for n in ("q", "k", "v", "out", "table"):
        setattr(a, n, 4096)
    a.Tq, a.Tk, a.H, a.Hk, a.dk, a.maps, a.dtype = 1, 1, 16, 16, 64, 1, _lib.BF16
    a.ldq = a.ldk = a.ldv = a.ldo = a.sq = a.sk = a.sv = a.so = 1024
    a.nbuckets, a.bidirectional, a.max_distance, a.nexact, a.nedges, a.edges = 32, 1, 128, e, cnt, ctypes.addressof(edges)
    a.scale = 0.125
    a.B = 2 ** 20 - 1
    assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(a), 0) >= 0
    a.B = 2 ** 20
    assert lib.ptpp_attention_long_ws_bytes(ctypes.byref(a), 0) < 0
    assert lib.ptpp_attention_long_fwd(ctypes.byref(a), None) == -1
    n = _lib.ResidualNormArgs()
    n.f = n.y = 4096
    n.B, n.T, n.C, n.gate_rows, n.dtype, n.scale, n.eps = 2 ** 12, 2 ** 13, 1024, 1, _lib.BF16, 1.0, 1e-5
    assert lib.ptpp_residual_norm_fwd(ctypes.byref(n), None) == -1
    # a gate row per utterance: one block of the finishing launch each
    n.B, n.T, n.C, n.gate, n.gate_rows, n.dy, n.stats, n.dgate = 65536, 1, 4, 4096, 65536, 4096, 4096, 4096
    n.ws, n.ws_bytes = 4096, lib.ptpp_residual_norm_ws_bytes(ctypes.byref(n))
    assert lib.ptpp_residual_norm_bwd(ctypes.byref(n), None) == -1


def test_attention_refuses_cpu_tensors():
    from promptttspp_amd import _lib
    from promptttspp_amd import functional as PF

    x = torch.zeros(1, 4, 3 * 64)
    with pytest.raises(_lib.PtppError):
        PF.attention_bucket(x, None, None, torch.zeros(32, 1), 1)
    with pytest.raises(ValueError):
        PF.attention_bucket(x, None, None, None, 1)
    with pytest.raises(ValueError):
        PF.attention_bucket(x, x, None, torch.zeros(32, 1), 1)
    with pytest.raises(ValueError):
        PF.attention_diff(x, None, None, None, 0.1, 1)
    with pytest.raises(_lib.PtppError):
        PF.residual_norm(torch.zeros(1, 4, 8))
    # what is given by value cannot be learned, and is not cut off
    one = torch.ones((), requires_grad=True)
    with pytest.raises(ValueError):
        PF.attention_bucket(x, None, None, torch.zeros(32, 1), 1, scale=one)
    with pytest.raises(ValueError):
        PF.attention_diff(x, None, None, torch.zeros(4, 1, 32), one, 1)
    with pytest.raises(ValueError):
        PF.residual_norm(torch.zeros(1, 4, 8), scale=one)
    with pytest.raises(TypeError):
        PF.attention_bucket(x, None, None, torch.zeros(32, 1), 1, max_distance=128.5)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("Tq,start", [(1, 0), (1, 299), (5, 300), (40, 256)])
def test_memory_behind_the_last_query_is_not_read(dev, maps, Tq, start):
    """a step against a preallocated memory: with ``causal`` what lies behind the last query is not read, lengths or not"""
    B, Tk, heads, dk = 2, 700, 2, 64 // maps
    q, k, v, table, lam, _ = make(maps, torch.bfloat16, B, Tq, Tk, heads, heads, dk, 32, seed=9)
    ref = RefAttention(q, k, v, table, lam, 0.35, None, heads, heads, maps, causal=True, q_start=[start, start], dt=torch.bfloat16)
    k[:, start + Tq:], v[:, start + Tq:] = float("nan"), float("inf")
    d = lambda t: None if t is None else t.to(dev)  # noqa: E731
    out = call(maps, d(q), d(k), d(v), d(table), d(lam), heads, causal=True, q_start=torch.full((B,), start, device=dev, dtype=torch.int32))
    within(out, ref.out, ref.out_b, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("hide", [float("-inf"), -3.4028234663852886e38])
@pytest.mark.parametrize("Tq,Tk", [(150, 150), (3, 200)])
def test_table_entries_that_hide_keys(dev, maps, hide, Tq, Tk):
    """buckets of the lowest values: their keys count for nothing, in every direction; a row that sees only such keys gives zeros"""
    heads, dk, B = 2, 64 // maps, 2
    q, k, v, table, lam, dout = make(maps, torch.bfloat16, B, Tq, Tk, heads, heads, dk, 32, seed=5)
    finite = table.clone()
    table[15, 0] = table[31, 0] = hide      # head 0: everything far away (in either direction)
    table[:, 1] = hide                      # head 1: all keys
    dist = torch.arange(Tk)[None] - torch.arange(Tq)[:, None]
    bk = ref_bucket(dist, 32, 128, True)
    seen = (bk != 15) & (bk != 31)
    f = 2.0 ** -24
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v, table) + ((lam,) if maps == 2 else ())]
    out = call(maps, *leaves[:4], leaves[4] if maps == 2 else None, heads)
    assert not out[:, :, 64:].any()
    qd, kd, vd = (t.double().view(B, -1, heads, 64)[:, :, 0] for t in (q, k, v))
    for b in range(B):
        ps, rhos = [], []
        for m in range(maps):
            s = dk ** -0.5 * qd[b, :, m * dk:(m + 1) * dk] @ kd[b, :, m * dk:(m + 1) * dk].T + finite.double()[bk, 0]
            rhos.append((dk + 16) * f * float(s.abs().max()))
            ps.append(s.masked_fill(~seen, float("-inf")).softmax(-1))
        c = [1.0]
        if maps == 2:
            lv = lam.double()
            c.append(-float((lv[0, 0] @ lv[1, 0]).exp() - (lv[2, 0] @ lv[3, 0]).exp() + 0.35))
        w, wa = sum(x * p for x, p in zip(c, ps)), sum(abs(x) * p for x, p in zip(c, ps))
        u = 2.0 ** -8
        want = w @ vd[b]
        within(out[b, :, :64], want, (u + 2 * max(rhos) + 8 * f) * (wa @ vd[b].abs()) + u * want.abs(), "out")
    grads = torch.autograd.grad(out, leaves, dout.to(dev))
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    dt = grads[3]
    assert not dt[:, 1].any() and not dt[15].any() and not dt[31].any() and dt[:, 0].any()
    for t in grads[:3]:
        assert not t[:, :, 64:].any()


@pytest.mark.gpu
def test_attention_refusals(dev):
    from promptttspp_amd import _lib
    from promptttspp_amd import functional as PF

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device=dev, dtype=dt)  # noqa: E731
    tab = z(32, 2, dt=torch.float32)
    ok = (z(2, 5, 128), z(2, 7, 128), z(2, 7, 128), tab, 2)
    PF.attention_bucket(*ok)
    val = [((z(2, 5, 120), *ok[1:]), {}), ((z(2, 5, 128, dt=torch.float32), *ok[1:]), {}), ((ok[0], z(1, 7, 128), *ok[2:]), {}),
           ((ok[0], z(2, 7, 64), *ok[2:]), {}), ((*ok[:3], z(32, 3, dt=torch.float32), 2), {}), ((*ok[:3], z(33, 2, dt=torch.float32), 2), {}),
           (ok, {"kv_heads": 3}), (ok, {"scale": 0.0}), (ok, {"scale": -1.0}), (ok, {"max_distance": 2000}), (ok, {"max_distance": 4}),
           (ok, {"lengths": torch.ones(3, device=dev, dtype=torch.int32)}), (ok, {"lengths": torch.ones(2, device=dev)}),
           (ok, {"q_start": torch.ones(2, 1, device=dev, dtype=torch.int32)}), ((z(2, 128, 5).transpose(1, 2), *ok[1:]), {}),
           ((z(2, 0, 128), *ok[1:]), {}), ((ok[0], z(2, 0, 128), z(2, 0, 128), tab, 2), {}), ((ok[0], None, ok[2], tab, 2), {}),
           ((z(2, 5, 130), None, None, tab, 2), {})]
    for a, kw in val:
        with pytest.raises(ValueError):
            PF.attention_bucket(*a, **kw)
    with pytest.raises(TypeError):
        PF.attention_bucket(z(2, 5, 128, dt=torch.float64), z(2, 7, 128, dt=torch.float64), z(2, 7, 128, dt=torch.float64), tab, 2)
    with pytest.raises(_lib.PtppError):  # rows that are not 16-byte aligned
        PF.attention_bucket(z(2, 5, 132)[:, :, 2:130], *ok[1:])
    with pytest.raises(_lib.PtppError):
        PF.attention_bucket(*ok[:3], tab.cpu(), 2)
    for lam in (z(4, 3, 32, dt=torch.float32), z(3, 1, 32, dt=torch.float32), z(4, 1, 16, dt=torch.float32)):
        with pytest.raises(ValueError):
            PF.attention_diff(*ok[:3], lam, 0.1, 2)
    with pytest.raises(ValueError):  # a map of 72 channels
        PF.attention_diff(z(1, 5, 144), z(1, 5, 144), z(1, 5, 144), z(4, 1, 72, dt=torch.float32), 0.1, 1)


# ---------------------------------------------------------------------------------------------------------------------
# norm, gate, residual, norm
# ---------------------------------------------------------------------------------------------------------------------
def ref_norm(f, x, gate, post, pre, scale, eps, kind, lengths, dy, dz, dt):
    """values, gradients and bounds in 64 bits.  f32 inside the kernel: a row's mean and deviation are sums of C terms in registers and
    over lanes (depth <= 24), so every intermediate is off by at most ~64 * 2^-24 of the magnitudes that enter it"""
    rms, u, f32 = kind == "rms", half_ulp(dt), 64 * 2.0 ** -24
    B, T, C = f.shape
    d = lambda t: None if t is None else t.double()  # noqa: E731
    rows = torch.ones(B, T, 1, dtype=torch.float64) if lengths is None else \
        (torch.arange(T)[None] < torch.tensor(lengths)[:, None]).double()[:, :, None]
    f = torch.where(rows > 0, f.double(), torch.zeros(())).double()
    x = None if x is None else torch.where(rows > 0, x.double(), torch.zeros(())).double()
    dy, dz = (None if t is None else torch.where(rows > 0, t.double(), torch.zeros(())).double() for t in (dy, dz))
    (pg, pb), (qg, qb), gate = tuple(map(d, post)), tuple(map(d, pre)), d(gate)
    g = 1.0 if gate is None else gate[:, None] if gate.dim() == 2 else gate

    def hat(v):
        mu = 0.0 if rms else v.mean(-1, keepdim=True)
        r = ((v - mu).square().mean(-1, keepdim=True) + eps).rsqrt()
        # |v| + |mean| enters the subtraction, the deviation scales everything by its own relative error
        amp = r * (v.abs() + (0.0 if rms else v.abs().mean(-1, keepdim=True)))
        return (v - mu) * r, r, amp

    def back(gh, h, r):
        t = gh - h * (gh * h).mean(-1, keepdim=True)
        b = gh.abs() + h.abs() * (gh.abs() * h.abs()).mean(-1, keepdim=True) + gh.abs().mean(-1, keepdim=True)
        return r * (t if rms else t - gh.mean(-1, keepdim=True)), r * b

    if pg is not None:
        fh, fr, fa = hat(f)
        fa = fa + fh.abs() * (fa * fh.abs()).mean(-1, keepdim=True)
        uu, ua = fh * pg + (0.0 if pb is None else pb), fa * pg.abs() + (0.0 if pb is None else pb.abs())
    else:
        fh, fr, fa, uu, ua = f, torch.ones(()).double(), f.abs(), f, f.abs()
    y = ((0.0 if x is None else x) + scale * g * uu) * rows
    ya = (0.0 if x is None else x.abs()) + abs(scale) * (g.abs() if torch.is_tensor(g) else g) * ua
    res = {"y": (y, f32 * ya + u * y.abs())}
    yh = None
    if qg is not None:
        yh, yr, ym = hat(y)
        ye = yr * ya + ym                                    # error sources of the normalised y: its own, and y's
        ye = ye + yh.abs() * (ye * yh.abs()).mean(-1, keepdim=True) + ye.mean(-1, keepdim=True)
        z = (yh * qg + (0.0 if qb is None else qb)) * rows
        res["z"] = (z, f32 * (ye * qg.abs() + (0.0 if qb is None else qb.abs())) + u * z.abs())
    if dy is None and dz is None:
        return res
    dx = torch.zeros_like(f) if dy is None else dy.clone()
    dxa = dx.abs()
    if dz is not None:
        t, ta = back(dz * qg, yh, yr)
        te = yr * (dz * qg).abs().mean(-1, keepdim=True) * ye + ta * (1 + (ye * yh.abs()).mean(-1, keepdim=True))
        dx, dxa = dx + t, dxa + ta + te
        res["dpre_g"] = ((dz * yh).sum((0, 1)), f32 * (dz.abs() * (ye + yh.abs())).sum((0, 1)))
        res["dpre_b"] = (dz.sum((0, 1)), f32 * dz.abs().sum((0, 1)))
    dx = dx * rows
    res["dx"] = (dx, f32 * dxa + u * dx.abs())
    du, dua = scale * g * dx, abs(scale) * (g.abs() if torch.is_tensor(g) else g) * dxa
    if pg is not None:
        df, dfa = back(du * pg, fh, fr)
        _, e1 = back(dua * pg.abs(), fh, fr)
        dfa = dfa * (1 + (fa * fh.abs()).mean(-1, keepdim=True)) + e1 + fr * (du * pg).abs().mean(-1, keepdim=True) * fa
        res["dpost_g"] = ((du * fh).sum((0, 1)), f32 * (dua * fh.abs() + du.abs() * fa).sum((0, 1)))
        res["dpost_b"] = (du.sum((0, 1)), f32 * dua.sum((0, 1)))
    else:
        df, dfa = du, dua
    res["df"] = (df * rows, f32 * dfa + u * df.abs())
    if gate is not None:
        dims = (1,) if gate.dim() == 2 else (0, 1)
        res["dgate"] = ((scale * uu * dx).sum(dims), f32 * abs(scale) * (ua * dxa).sum(dims))
    return res


def check_norm(dev, dtype, B, T, C, kind="layer", gate="utt", res=True, post=True, pre=True, beta=True, lengths=None, scale=0.5, use="both", garbage=False,
               train=True, eps=1e-5, seed=0):
    from promptttspp_amd import functional as PF

    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    f, x = (2 * r(B, T, C) + 0.5).to(dt), (3 * r(B, T, C)).to(dt) if res else None
    beta = beta and kind == "layer"
    par = {"gate": {"utt": r(B, C), "chan": r(C), "none": None}[gate], "post_g": 1 + 0.2 * r(C) if post else None, "post_b": 0.2 * r(C) if post and beta else None,
           "pre_g": 1 + 0.2 * r(C) if pre else None, "pre_b": 0.2 * r(C) if pre and beta else None}
    dy, dz = r(B, T, C).to(dt), r(B, T, C).to(dt)
    use_y, use_z = use in ("both", "y"), use in ("both", "z") and pre
    want = ref_norm(f, x, par["gate"], (par["post_g"], par["post_b"]), (par["pre_g"], par["pre_b"]), scale, eps, kind, lengths,
                    dy if train and use_y else None, dz if train and use_z else None, dt)
    if garbage:
        for t in (f, x, dy, dz):
            if t is not None:
                for b in range(B):
                    t[b, lengths[b]:] = float("nan") if b % 2 else float("inf")
    leaves = {n: t.to(dev).requires_grad_(train) for n, t in (("f", f), ("x", x), *par.items()) if t is not None}
    y, z = PF.residual_norm(leaves["f"], leaves.get("x"), gate=leaves.get("gate"), post=(leaves["post_g"], leaves.get("post_b")) if post else None,
                            pre=(leaves["pre_g"], leaves.get("pre_b")) if pre else None, scale=scale, eps=eps, kind=kind,
                            lengths=None if lengths is None else torch.tensor(lengths, device=dev))
    got = {"y": y}
    assert (z is not None) == pre
    if pre:
        got["z"] = z
    if train:
        outs = ([y] if use_y else []) + ([z] if use_z else [])
        gouts = ([dy.to(dev)] if use_y else []) + ([dz.to(dev)] if use_z else [])
        for n, t in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gouts, allow_unused=True)):
            got["d" + n] = t
    for n, t in got.items():
        if n in want:
            within(t, *want[n], n)
        else:
            assert n in ("dpre_g", "dpre_b") and (t is None or float(t.abs().max()) == 0.0), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("C", [4, 60, 64, 68, 128, 132, 256, 260, 512, 516, 1024, 1028, 2048, 2052, 4096])
def test_residual_norm_widths(dev, dtype, C):
    check_norm(dev, dtype, 2, 19, C, lengths=[19, 7])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,T", [(1, 1), (32, 1), (1, 5000), (3, 333), (1100, 3)])
def test_residual_norm_row_counts(dev, dtype, B, T):
    check_norm(dev, dtype, B, T, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["utt", "chan", "none"])
@pytest.mark.parametrize("res,post,pre", [(True, True, True), (True, True, False), (True, False, True), (False, True, False), (False, True, True),
                                          (True, False, False), (False, False, True)])
def test_residual_norm_forms(dev, kind, gate, res, post, pre):
    check_norm(dev, "f32", 3, 21, 192, kind=kind, gate=gate, res=res, post=post, pre=pre, lengths=[21, 1, 0])
    check_norm(dev, "bf16", 3, 21, 576, kind=kind, gate=gate, res=res, post=post, pre=pre, beta=False)


@pytest.mark.gpu
@pytest.mark.parametrize("use", ["y", "z"])
def test_residual_norm_one_output_used(dev, use):
    check_norm(dev, "bf16", 2, 30, 256, use=use, lengths=[30, 11])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_residual_norm_garbage_behind_the_lengths(dev, dtype):
    check_norm(dev, dtype, 4, 40, 256, lengths=[40, 0, 1, 23], garbage=True)
    check_norm(dev, dtype, 4, 40, 1500, kind="rms", lengths=[40, 0, 1, 23], garbage=True)
    check_norm(dev, dtype, 4, 40, 256, lengths=[40, 0, 1, 23], garbage=True, train=False)


@pytest.mark.gpu
def test_residual_norm_inputs_off_the_beaten_path(dev):
    """transposed and expanded inputs, (1, C, 1) parameters, an expanded gradient; parameters of another float type keep it"""
    from promptttspp_amd import functional as PF

    g = torch.Generator().manual_seed(2)
    f = torch.randn(2, 24, 10, generator=g)
    x = torch.randn(1, 1, 24, generator=g)
    pg = (1 + 0.1 * torch.randn(1, 24, 1, generator=g)).to(dev).requires_grad_()
    qg = (1 + 0.1 * torch.randn(24, generator=g)).bfloat16().to(dev).requires_grad_()
    fd, xd = f.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    y, z = PF.residual_norm(fd.transpose(1, 2), xd.expand(2, 10, 24), post=(pg, None), pre=(qg, None), kind="rms", scale=1.0)
    ones = torch.ones(2, 10, 24)
    want = ref_norm(f.transpose(1, 2), x.expand(2, 10, 24), None, (pg.detach().cpu().reshape(-1), None), (qg.detach().cpu().float(), None), 1.0, 1e-5, "rms", None,
                    ones, ones, torch.float32)
    within(y, *want["y"], "y")
    within(z, *want["z"], "z")
    df, dx, dpg, dqg = torch.autograd.grad(y.sum() + z.sum(), [fd, xd, pg, qg])
    within(df.transpose(1, 2), *want["df"], "df")
    within(dx, want["dx"][0].sum((0, 1), keepdim=True), want["dx"][1].sum((0, 1), keepdim=True) + 32 * 2.0 ** -24 * want["dx"][0].abs().sum((0, 1), keepdim=True), "dx")
    assert dpg.shape == pg.shape and dqg.dtype == torch.bfloat16
    within(dpg.reshape(-1), *want["dpost_g"], "dpost_g")
    within(dqg, want["dpre_g"][0], want["dpre_g"][1] + 2.0 ** -8 * want["dpre_g"][0].abs(), "dpre_g")


@pytest.mark.gpu
def test_residual_norm_off_the_16_byte_grid(dev):
    """contiguous operands, parameters and gradients that start anywhere"""
    from promptttspp_amd import functional as PF

    g = torch.Generator().manual_seed(8)
    f, x = torch.randn(2, 2, 7, 12, generator=g).bfloat16()
    pg, dy = 1 + 0.1 * torch.randn(12, generator=g), torch.randn(2, 7, 12, generator=g).bfloat16()
    want = ref_norm(f, x, None, (pg, None), (None, None), 1.0, 1e-5, "rms", None, dy, None, torch.bfloat16)

    def off(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)]).to(dev).requires_grad_()

    fd, xd, pd = off(f), off(x), off(pg)
    y, _ = PF.residual_norm(fd[1:].view(2, 7, 12), xd[1:].view(2, 7, 12), post=(pd[1:], None), kind="rms")
    within(y, *want["y"], "y")
    joined = torch.cat([y.new_zeros(1), y.reshape(-1)])  # (its backward hands a gradient one element off)
    df, dx, dp = torch.autograd.grad(joined, [fd, xd, pd], torch.cat([dy.new_zeros(1), dy.reshape(-1)]).to(dev))
    within(df[1:].view(2, 7, 12), *want["df"], "df")
    within(dx[1:].view(2, 7, 12), *want["dx"], "dx")
    within(dp[1:], *want["dpost_g"], "dpost_g")
    with torch.no_grad():
        y2, _ = PF.residual_norm(fd[1:].view(2, 7, 12), xd[1:].view(2, 7, 12), post=(pd[1:], None), kind="rms")
    assert torch.equal(y, y2)


@pytest.mark.gpu
def test_residual_norm_gradients_against_differences(dev):
    """central differences along a random direction, f32, the h^2 term cancelled"""
    from promptttspp_amd import functional as PF

    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    ws = [r(2, 9, 64), r(2, 9, 64), r(2, 64), 1 + 0.2 * r(64), r(64), 1 + 0.2 * r(64), r(64)]
    ds, dy, dz = [r(*w.shape) for w in ws], r(2, 9, 64).double(), r(2, 9, 64).double()

    def run(w):
        return PF.residual_norm(w[0], w[1], gate=w[2], post=(w[3], w[4]), pre=(w[5], w[6]), scale=0.7)

    def loss(h):
        y, z = run([(w.double() + h * d.double()).float() for w, d in zip(ws, ds)])
        return float((y.double() * dy + z.double() * dz).sum())

    leaves = [w.clone().requires_grad_() for w in ws]
    y, z = run(leaves)
    ana = sum(float((a.double() * d.double()).sum()) for a, d in zip(torch.autograd.grad((y, z), leaves, (dy.float(), dz.float())), ds))
    num = (4 * (loss(5e-3) - loss(-5e-3)) / 1e-2 - (loss(1e-2) - loss(-1e-2)) / 2e-2) / 3
    assert abs(ana - num) < 5e-3 * max(1.0, abs(ana)), (ana, num)


@pytest.mark.gpu
def test_residual_norm_same_bits_and_captured(dev):
    from promptttspp_amd import functional as PF

    g = torch.Generator(device=dev).manual_seed(4)
    r = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    sets = [[r(5, 77, 256), r(5, 77, 256), r(5, 256), r(256), r(256), r(256), r(256), r(5, 77, 256), r(5, 77, 256)] for _ in range(2)]

    def step(ts):
        lv = [t.detach().requires_grad_() for t in ts[:7]]
        y, z = PF.residual_norm(lv[0], lv[1], gate=lv[2], post=(lv[3], lv[4]), pre=(lv[5], lv[6]), scale=0.5)
        return [y.detach(), z.detach(), *torch.autograd.grad((y, z), lv, (ts[7], ts[8]))]

    static = [t.clone() for t in sets[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step(static)
    for trip in range(4):
        for d, t in zip(static, sets[trip % 2]):
            d.copy_(t)
        gr.replay()
        want = step(sets[trip % 2])
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_residual_norm_refusals_on_the_host():
    from promptttspp_amd import _lib

    lib = _lib.load()

    def args(**kw):
        a = _lib.ResidualNormArgs()
        a.f = a.x = a.y = a.z = a.gate = a.post_g = a.post_b = a.pre_g = a.pre_b = 4096
        a.B, a.T, a.C, a.gate_rows, a.dtype, a.scale, a.eps = 2, 3, 64, 2, _lib.F32, 1.0, 1e-5
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    for kw in (dict(f=None), dict(y=None), dict(z=None), dict(pre_g=None), dict(B=0), dict(T=0), dict(C=66), dict(C=4100), dict(C=0), dict(dtype=9), dict(gate_rows=3),
               dict(post_g=None), dict(rms=1), dict(eps=0.0), dict(eps=float("nan")), dict(f=4104), dict(gate=4100), dict(B=2 ** 20, T=2 ** 12)):
        assert lib.ptpp_residual_norm_fwd(ctypes.byref(args(**kw)), None) == -1, kw
    grads = dict(dy=4096, dz=4096, df=4096, dx=4096, stats=4096, dgate=4096, dpost_g=4096)
    n = lib.ptpp_residual_norm_ws_bytes(ctypes.byref(args(**grads)))
    assert n > 0
    for kw in (dict(grads, stats=None, ws=4096, ws_bytes=n), dict(grads, ws=None), dict(grads, ws=4096, ws_bytes=n - 1), dict(grads, ws=4100, ws_bytes=n),
               dict(grads, gate=None, ws=4096, ws_bytes=n), dict(grads, dpre_g=4096, pre_g=None, pre_b=None, z=None, ws=4096, ws_bytes=1 << 20)):
        assert lib.ptpp_residual_norm_bwd(ctypes.byref(args(**kw)), None) == -1, kw


@pytest.mark.gpu
def test_residual_norm_refusals(dev):
    from promptttspp_amd import _lib
    from promptttspp_amd import functional as PF

    z = lambda *s, dt=torch.float32: torch.zeros(*s, device=dev, dtype=dt)  # noqa: E731
    f = z(2, 3, 64)
    for kw in (dict(x=z(2, 3, 60)), dict(x=z(2, 3, 64, dt=torch.bfloat16)), dict(gate=z(3, 64)), dict(gate=z(32)), dict(gate=z(2, 3, 64)), dict(post=(z(60), None)),
               dict(post=(None, z(64))), dict(pre=(z(64), z(64)), kind="rms"), dict(kind="batch"), dict(eps=0.0), dict(lengths=z(2)),
               dict(lengths=torch.ones(3, device=dev, dtype=torch.int64))):
        with pytest.raises(ValueError):
            PF.residual_norm(f, **kw)
    for bad in (z(2, 3, 66), z(2, 3, 4100), z(2, 64), z(0, 3, 64)):
        with pytest.raises(ValueError):
            PF.residual_norm(bad)
    with pytest.raises(TypeError):
        PF.residual_norm(z(2, 3, 64, dt=torch.float64))
    with pytest.raises(_lib.PtppError):
        PF.residual_norm(f, gate=torch.zeros(64))


def test_argument_blocks_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess

    from promptttspp_amd import _lib

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    pairs = [("ptpp_attention_long_args", _lib.AttentionLongArgs), ("ptpp_residual_norm_args", _lib.ResidualNormArgs)]
    src = tmp_path / "sz.c"
    fields = "".join('printf("%%zu\\n", offsetof(%s, %s));' % (n, f[0]) for n, c in pairs for f in c._fields_)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "%s"\nint main(void){%s%s return 0;}\n' % (
        os.path.join(ROOT, "include", "ptpp.h"), "".join('printf("%%zu\\n", sizeof(%s));' % n for n, _ in pairs), fields))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "sz")], check=True)
    vals = [int(v) for v in subprocess.run([str(tmp_path / "sz")], check=True, capture_output=True, text=True).stdout.split()]
    want = [ctypes.sizeof(c) for _, c in pairs] + [getattr(c, f[0]).offset for _, c in pairs for f in c._fields_]
    assert vals == want
