"""Measured cases of the long-sequence encoder-block operators.

Three operators, each in its plain form (elementary torch operations in 32 bits) and through the package's entry points:

* ``bucket``: attention with a learned relative-position bias by buckets,
  ``softmax(scale * q k^T + table[bucket(j - i)]) v``, and its gradients;
* ``diff``: differential attention, ``(softmax(q1 k1^T) - lam * softmax(q2 k2^T)) v`` with
  ``lam = exp(l0 . l1) - exp(l2 . l3) + lam_init``, and its gradients;
* ``norm``: ``y = x + scale * gate * post_norm(f)``, ``z = pre_norm(y)``, and its gradients.

Modes: ``train`` (forward and all gradients), ``infer`` (forward of whole sequences), ``step`` (one query per utterance
against a long memory of keys and values).
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_MAX_DISTANCE = 128
_LAM_INIT = 0.2
_EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attn(name, op, mode, dtype, B, T, heads, dk, kv_heads=0, ragged=0.4, buckets=32, causal=False):
    """dk: channels of one map's query; ``buckets`` 0: no table (diff only); kv_heads 0: as many as heads."""
    return {"name": name, "op": op, "mode": mode, "dtype": dtype, "B": B, "T": T, "heads": heads, "kv_heads": kv_heads or heads, "dk": dk,
            "ragged": ragged, "buckets": buckets, "causal": causal}


def _norm(name, mode, dtype, B, T, C, kind="layer", gate="utt", ragged=0.3):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "B": B, "T": T, "C": C, "kind": kind, "gate": gate, "ragged": ragged}


def listed():
    return [
        # a phoneme-level encoder layer of a training batch: 256 channels in 2 heads, utterances of up to 217 phones
        _attn("bucket_train_phones", "bucket", "train", "bf16", 32, 217, 2, 128),
        # a mel-frame-level layer of a 30 000-token training batch
        _attn("bucket_train_frames", "bucket", "train", "bf16", 24, 1250, 4, 64),
        # the 32-bit mode in which results are compared with other implementations
        _attn("bucket_train_f32", "bucket", "train", "f32", 4, 333, 2, 128, ragged=0.7),
        # one long recording in half precision, no gradients
        _attn("bucket_infer_long", "bucket", "infer", "f16", 2, 6001, 8, 64, ragged=0.0),
        # one new query per utterance against a kept memory with shared key / value heads (causal buckets)
        _attn("bucket_step", "bucket", "step", "bf16", 32, 8191, 12, 64, kv_heads=4, causal=True),
        # the differential form of the phoneme-level layer: 2 heads of 2 x 64 channels
        _attn("diff_train_phones", "diff", "train", "bf16", 32, 217, 2, 64, buckets=0),
        # ... of a long frame-level batch, with the position table
        _attn("diff_train_frames", "diff", "train", "bf16", 8, 2000, 4, 64),
        # odd sizes in 32 bits, forward only, small heads
        _attn("diff_infer_f32", "diff", "infer", "f32", 3, 517, 4, 32, ragged=0.6),
        # one new query per utterance, half precision
        _attn("diff_step", "diff", "step", "f16", 16, 4001, 8, 64, kv_heads=8, causal=True),
        # the norm / gate / residual step of one position of 32 utterances: latency
        _norm("norm_step", "infer", "bf16", 32, 1, 256, ragged=0.0),
        # ... of the 30 000-token training batch, gates from the utterance's style
        _norm("norm_train_frames", "train", "bf16", 24, 1250, 256),
        # ... of a wide model with root-mean-square norms and a learned per-channel gate
        _norm("norm_train_wide", "train", "f16", 8, 2048, 1024, kind="rms", gate="chan", ragged=0.2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("bucket", "diff", "norm"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if op == "norm":
        mode = rng.choice(("train", "infer"))
        C = 4 * _log_int(rng, 16, 512)
        T = _log_int(rng, 1, 2048)
        B = max(1, min(_log_int(rng, 1, 48), 12_000_000 // (T * C)))
        return _norm("", mode, dtype, B, T, C, kind=rng.choice(("layer", "rms")), gate=rng.choice(("utt", "chan", "none")),
                     ragged=rng.uniform(0.0, 0.9))
    mode = rng.choice(("train", "infer", "step"))
    heads = rng.choice((1, 2, 3, 4, 6, 8, 12))
    kv = rng.choice([g for g in (1, 2, 3, 4, 6, 8, 12) if heads % g == 0] + [heads] * 3)
    dk = rng.choice((32, 40, 64, 80, 128) if op == "bucket" else (16, 32, 48, 64))
    buckets = rng.choice((8, 32, 64)) if op == "bucket" or rng.random() < 0.5 else 0
    if mode == "step":
        T, B = _log_int(rng, 1, 8192), _log_int(rng, 1, 32)
        row = kv * dk * (4 if op == "diff" else 2) * _SIZE[dtype]  # bytes of keys and values per position
        B = max(1, min(B, 200_000_000 // (T * row)))
    else:
        T = _log_int(rng, 1, 2000 if mode == "train" else 6001)
        cap = 6.0e8 if mode == "train" else 2.0e9
        if dtype == "f32":
            cap *= 0.25
        B = max(1, min(_log_int(rng, 1, 40), int(cap // (T * T * heads * dk // 16 + 1))))
        while T > 1 and T * T * heads * dk // 16 > cap:
            T = T * 3 // 4
    return _attn("", op, mode, dtype, B, T, heads, dk, kv_heads=kv, ragged=rng.uniform(0.0, 0.95), buckets=buckets,
                 causal=mode == "step" or rng.random() < 0.3)


def _lengths(case):
    """Valid positions of every utterance: the longest has all T, the others spread over the lower ``ragged`` share."""
    B, T = case["B"], case["T"]
    out = [T]
    for b in range(1, B):
        out.append(max(1, T - int(T * case["ragged"] * ((b * 0.6180339887498949) % 1.0))))
    return out


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _spread(case):
    """(maps, width of one value head)"""
    return (2, 2 * case["dk"]) if case["op"] == "diff" else (1, case["dk"])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    lens = _lengths(case)
    st = {"case": case, "lengths": torch.tensor(lens, dtype=torch.int32, device=dev)}

    def rnd(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)

    B, T = case["B"], case["T"]
    if case["op"] == "norm":
        C = case["C"]
        st["f"] = rnd(B, T, C, std=2.0)
        st["x"] = rnd(B, T, C, std=3.0)
        rms = case["kind"] == "rms"
        for n in ("post", "pre"):
            st[n + "_g"] = 1.0 + rnd(C, std=0.2, dtype=torch.float32)
            st[n + "_b"] = None if rms else rnd(C, std=0.2, dtype=torch.float32)
        st["gate"] = {"utt": lambda: rnd(B, C, std=0.5, dtype=torch.float32), "chan": lambda: rnd(C, std=0.5, dtype=torch.float32),
                      "none": lambda: None}[case["gate"]]()
        if case["mode"] == "train":
            st["dy"], st["dz"] = rnd(B, T, C), rnd(B, T, C)
        return st
    maps, dv = _spread(case)
    H, Hk, dk = case["heads"], case["kv_heads"], case["dk"]
    if case["mode"] == "step":  # a fresh query, and the memory that the program keeps
        st["q"] = rnd(B, 1, H * maps * dk)
        st["k"] = rnd(B, T, Hk * maps * dk)
        st["v"] = rnd(B, T, Hk * dv)
        st["q_start"] = st["lengths"] - 1
    else:  # the fused q | k | v projection
        st["qkv"] = rnd(B, T, H * maps * dk + Hk * maps * dk + Hk * dv)
        st["q_start"] = None
    st["table"] = rnd(case["buckets"], H, std=0.7, dtype=torch.float32) if case["buckets"] else None
    if maps == 2:
        st["lam"] = rnd(4, 1, dk, std=0.1, dtype=torch.float32)
    if case["mode"] == "train":
        st["dout"] = rnd(B, T, H * dv)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
_bucket_of = {}  # the plan of the plain form: bucket of every distance in [-D, D]


def _bucket_map(buckets, causal, device):
    """Bucket of j - i for j - i in [-D, D] (clamped outside): half of the buckets for keys behind the query, half for keys before
    it (causal: all of them for keys before it); within a half the first ``e`` distances have their own, the rest share
    logarithmically up to D.  floor(log(n / e) / log(D / e) * L) in whole numbers: n^L e^t >= D^t e^L."""
    key = (buckets, causal, str(device))
    m = _bucket_of.get(key)
    if m is None:
        D, nb = _MAX_DISTANCE, buckets if causal else buckets // 2
        e = nb // 2
        L = nb - e
        out = []
        for r in range(-D, D + 1):
            n = max(-r, 0) if causal else abs(r)
            if n < e:
                b = n
            else:
                t = 0
                while t + 1 < L and n ** L * e ** (t + 1) >= D ** (t + 1) * e ** L:
                    t += 1
                b = e + t
            out.append(b + (nb if r > 0 and not causal else 0))
        m = _bucket_of[key] = torch.tensor(out, device=device)
    return m


def _allowed_and_bias(st, Tq, Tk):
    """(B,1,Tq,Tk) keys that a query may see, and the bias of every pair or None"""
    case, dev = st["case"], st["lengths"].device
    B = case["B"]
    j = torch.arange(Tk, device=dev)
    start = st["q_start"] if st["q_start"] is not None else torch.zeros(B, dtype=torch.int32, device=dev)
    i = start.long()[:, None] + torch.arange(Tq, device=dev)[None, :]  # (B,Tq)
    allowed = (j[None, :] < st["lengths"].long()[:, None])[:, None, None, :]
    if case["causal"]:
        allowed = allowed & (j[None, None, :] <= i[:, :, None])[:, None]

    def bias(table):
        if table is None:
            return None
        bucket = _bucket_map(case["buckets"], case["causal"], dev)
        if table.requires_grad:  # one value per distance, every row one further along its copy (64 bits: the gradient is a long sum)
            r = torch.arange(1 - Tq, Tq, device=dev).clamp(-_MAX_DISTANCE, _MAX_DISTANCE) + _MAX_DISTANCE
            copies = table.double()[bucket[r]].t().repeat(1, Tq)  # (H, Tq (2 Tq - 1)), Tq = Tk
            return copies[:, Tq - 1:Tq - 1 + Tq * (2 * Tq - 2)].view(1, -1, Tq, 2 * Tq - 2)[..., :Tk].float() if Tq > 1 else copies[None, :, None].float()
        i1 = i[:1] if st["q_start"] is None else i  # (without offsets all utterances share the distances)
        d = (j[None, None, :] - i1[:, :, None]).clamp(-_MAX_DISTANCE, _MAX_DISTANCE) + _MAX_DISTANCE
        return table[bucket[d]].permute(0, 3, 1, 2)  # (1 or B, H, Tq, Tk)

    return allowed, bias


def _softmax(s, allowed):
    s = s.masked_fill(~allowed, float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    p = (s - m).exp()
    l = p.sum(dim=-1, keepdim=True)
    return p / torch.where(l > 0, l, torch.ones_like(l))


def _plain_attention(st, q, k, v, table, lam):
    """q (B,Tq,H,maps,dk), k (B,Tk,Hk,maps,dk), v (B,Tk,Hk,dv) in 32 bits -> (B,Tq,H*dv)"""
    case = st["case"]
    B, Tq, H, maps, dk = q.shape
    Tk, Hk, dv = v.shape[1:]
    rep = H // Hk
    allowed, bias_of = _allowed_and_bias(st, Tq, Tk)
    bias = bias_of(table)
    vv = v.permute(0, 2, 1, 3).repeat_interleave(rep, dim=1) if rep > 1 else v.permute(0, 2, 1, 3)
    w = None
    for m in range(maps):
        kk = k[:, :, :, m].permute(0, 2, 3, 1)
        kk = kk.repeat_interleave(rep, dim=1) if rep > 1 else kk
        s = q[:, :, :, m].permute(0, 2, 1, 3) @ kk * (1.0 / math.sqrt(dk))
        if bias is not None:
            s = s + bias
        p = _softmax(s, allowed)
        w = p if m == 0 else w - lam * p
    o = (w @ vv).permute(0, 2, 1, 3).reshape(B, Tq, H * dv)
    if st["q_start"] is None:  # self-attention: rows behind the utterance are zero
        rows = torch.arange(Tq, device=o.device)[None, :] < st["lengths"].long()[:, None]
        o = o * rows[:, :, None]
    return o


def _split(st, qkv):
    case = st["case"]
    maps, dv = _spread(case)
    B, T = qkv.shape[:2]
    H, Hk, dk = case["heads"], case["kv_heads"], case["dk"]
    nq, nk = H * maps * dk, Hk * maps * dk
    return (qkv[:, :, :nq].reshape(B, T, H, maps, dk), qkv[:, :, nq:nq + nk].reshape(B, T, Hk, maps, dk),
            qkv[:, :, nq + nk:].reshape(B, T, Hk, dv))


def _plain_lam(lam):
    return (lam[0] * lam[1]).sum().exp() - (lam[2] * lam[3]).sum().exp() + _LAM_INIT


def _plain_run_attention(st):
    case = st["case"]
    maps, dv = _spread(case)
    dt = _DT[case["dtype"]]
    train = case["mode"] == "train"
    if case["mode"] == "step":
        B, T = case["B"], case["T"]
        H, Hk, dk = case["heads"], case["kv_heads"], case["dk"]
        q, k, v = st["q"].float().view(B, 1, H, maps, dk), st["k"].float().view(B, T, Hk, maps, dk), st["v"].float().view(B, T, Hk, dv)
        with torch.no_grad():
            return {"out": _plain_attention(st, q, k, v, st["table"], _plain_lam(st["lam"]) if maps == 2 else None).to(dt)}
    with torch.set_grad_enabled(train):
        leaves = {"qkv": st["qkv"].float().detach().requires_grad_(train)}
        if st["table"] is not None:
            leaves["table"] = st["table"].detach().requires_grad_(train)
        if maps == 2:
            leaves["lam"] = st["lam"].detach().requires_grad_(train)
        q, k, v = _split(st, leaves["qkv"])
        out = _plain_attention(st, q, k, v, leaves.get("table"), _plain_lam(leaves["lam"]) if maps == 2 else None)
        res = {"out": out.detach().to(dt)}
        if train:
            grads = torch.autograd.grad(out, list(leaves.values()), st["dout"].float())
            for n, gr in zip(leaves, grads):
                res["d" + n] = gr.to(dt) if n == "qkv" else gr
    return res


def _plain_norm(v, g, b, rms):
    if rms:
        return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + _EPS) * g
    c = v - v.mean(dim=-1, keepdim=True)
    return c * torch.rsqrt((c * c).mean(dim=-1, keepdim=True) + _EPS) * g + b


def _plain_run_norm(st):
    case = st["case"]
    dt, rms, train = _DT[case["dtype"]], case["kind"] == "rms", case["mode"] == "train"
    rows = (torch.arange(case["T"], device=st["f"].device)[None, :] < st["lengths"].long()[:, None])[:, :, None]
    with torch.set_grad_enabled(train):
        leaves = {n: st[n].float().detach().requires_grad_(train) for n in ("f", "x", "gate", "post_g", "post_b", "pre_g", "pre_b")
                  if st[n] is not None}
        u = _plain_norm(leaves["f"], leaves["post_g"], leaves.get("post_b"), rms)
        if "gate" in leaves:
            u = u * (leaves["gate"][:, None] if case["gate"] == "utt" else leaves["gate"])
        y = (leaves["x"] + 0.5 * u) * rows
        z = _plain_norm(y, leaves["pre_g"], leaves.get("pre_b"), rms) * rows
        res = {"y": y.detach().to(dt), "z": z.detach().to(dt)}
        if train:
            grads = torch.autograd.grad((y, z), list(leaves.values()), (st["dy"].float(), st["dz"].float()))
            for n, gr in zip(leaves, grads):
                res["d" + n] = gr.to(dt) if n in ("f", "x") else gr
    return res


# ---------------------------------------------------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------------------------------------------------
def _own_run_attention(st):
    from promptttspp_amd import functional as PF

    case = st["case"]
    train, diff = case["mode"] == "train", case["op"] == "diff"
    kw = {"heads": case["heads"], "kv_heads": case["kv_heads"], "lengths": st["lengths"], "causal": case["causal"],
          "max_distance": _MAX_DISTANCE, "bidirectional": not case["causal"]}

    def call(q, k, v, table, lam):
        if diff:
            return PF.attention_diff(q, k, v, lam, _LAM_INIT, table=table, **kw)
        return PF.attention_bucket(q, k, v, table, **kw)

    if case["mode"] == "step":
        with torch.no_grad():
            kw["q_start"] = st["q_start"]
            return {"out": call(st["q"], st["k"], st["v"], st["table"], st.get("lam"))}
    if not train:
        with torch.no_grad():
            return {"out": call(st["qkv"], None, None, st["table"], st.get("lam"))}
    leaves = {n: st[n].detach().requires_grad_() for n in ("qkv", "table", "lam") if st.get(n) is not None}
    out = call(leaves["qkv"], None, None, leaves.get("table"), leaves.get("lam"))
    res = {"out": out.detach()}
    for n, gr in zip(leaves, torch.autograd.grad(out, list(leaves.values()), st["dout"])):
        res["d" + n] = gr
    return res


def _own_run_norm(st):
    from promptttspp_amd import functional as PF

    case = st["case"]
    kw = {"scale": 0.5, "eps": _EPS, "kind": case["kind"], "lengths": st["lengths"]}
    if case["mode"] != "train":
        with torch.no_grad():
            y, z = PF.residual_norm(st["f"], st["x"], gate=st["gate"], post=(st["post_g"], st["post_b"]), pre=(st["pre_g"], st["pre_b"]), **kw)
        return {"y": y, "z": z}
    leaves = {n: st[n].detach().requires_grad_() for n in ("f", "x", "gate", "post_g", "post_b", "pre_g", "pre_b") if st[n] is not None}
    y, z = PF.residual_norm(leaves["f"], leaves["x"], gate=leaves.get("gate"), post=(leaves["post_g"], leaves.get("post_b")),
                            pre=(leaves["pre_g"], leaves.get("pre_b")), **kw)
    res = {"y": y.detach(), "z": z.detach()}
    for n, gr in zip(leaves, torch.autograd.grad((y, z), list(leaves.values()), (st["dy"], st["dz"]))):
        res["d" + n] = gr
    return res


def run(state):
    if state["case"]["op"] == "norm":
        return _own_run_norm(state) if own else _plain_run_norm(state)
    return _own_run_attention(state) if own else _plain_run_attention(state)


# ---------------------------------------------------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e, lens = _SIZE[case["dtype"]], _lengths(case)
    rows = sum(lens)
    train = case["mode"] == "train"
    B, T = case["B"], case["T"]
    if case["op"] == "norm":
        C = case["C"]
        # forward: f, x in; y, z out (rows behind the utterances are written only); backward: dy, dz, f, x in; df, dx out
        par = C * (2 if case["kind"] == "rms" else 4) + {"utt": B * C, "chan": C, "none": 0}[case["gate"]]
        by = 2 * rows * C * e + 2 * B * T * C * e + 4 * par
        fl = 16 * rows * C
        if train:
            by += 4 * rows * C * e + 2 * B * T * C * e + 8 * par
            fl += 40 * rows * C
        return {"bytes": by, "flops": fl}
    maps, dv = _spread(case)
    H, Hk, dk = case["heads"], case["kv_heads"], case["dk"]
    wq, wk, wv, wo = H * maps * dk, Hk * maps * dk, Hk * dv, H * dv
    small = 4 * ((case["buckets"] * H) + (4 * dk if maps == 2 else 0))
    if case["mode"] == "step":
        pairs = rows
        by = B * wq * e + rows * (wk + wv) * e + B * wo * e + small
    else:
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        by = rows * (wq + wk + wv) * e + B * T * wo * e + small
        if train:
            by += rows * (wq + wk + wv + wo) * e + B * T * (wq + wk + wv) * e + 2 * small
    fl = 2 * H * pairs * maps * (dk + dv)
    if train:  # scores again, dP (one for all maps), dV (one for all maps), dQ, dK
        fl += 2 * H * pairs * (3 * maps * dk + 2 * dv)
    return {"bytes": by, "flops": fl}


def _exact_buckets(case, dist):
    """Bucket of every whole-number distance in ``dist``, from least whole numbers per logarithmic step."""
    n_all = case["buckets"]
    half = n_all if case["causal"] else n_all // 2
    e, D = half // 2, _MAX_DISTANCE
    steps = half - e
    edges = []  # edges[t - 1]: least n in step t
    for t in range(1, steps):
        lo = e
        while (lo ** steps) * (e ** t) < (D ** t) * (e ** steps):
            lo += 1
        edges.append(lo)
    n = (-dist).clamp(min=0) if case["causal"] else dist.abs()
    b = torch.where(n < e, n, torch.full_like(n, e))
    for lo in edges:
        b = b + (n >= lo)
    if not case["causal"]:
        b = b + half * (dist > 0)
    return b


def _exact_attention(case, st):
    maps, dv = _spread(case)
    H, Hk, dk = case["heads"], case["kv_heads"], case["dk"]
    B, train, step = case["B"], case["mode"] == "train", case["mode"] == "step"
    if step:
        q, k, v = (st[n].double().unflatten(2, s) for n, s in (("q", (H, maps, dk)), ("k", (Hk, maps, dk)), ("v", (Hk, dv))))
    else:
        q, k, v = _split(st, st["qkv"].double())
    Tq = q.shape[1]
    dev = q.device
    out = torch.zeros(B, Tq, H, dv, dtype=torch.float64, device=dev)
    lam = 0.0
    if maps == 2:
        lv = st["lam"].double()[:, 0]
        e1, e2 = float((lv[0] @ lv[1]).exp()), float((lv[2] @ lv[3]).exp())
        lam = e1 - e2 + _LAM_INIT
    tab = st["table"].double() if st["table"] is not None else None
    if train:
        do = st["dout"].double().unflatten(2, (H, dv))
        dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dtab = torch.zeros_like(tab) if tab is not None else None
        dlam = 0.0
    scale = dk ** -0.5
    for b, n in enumerate(_lengths(case)):
        nq = 1 if step else n
        first = n - 1 if step else 0
        i, j = torch.arange(first, first + nq, device=dev), torch.arange(n, device=dev)
        dist = j[None, :] - i[:, None]
        bk = _exact_buckets(case, dist) if tab is not None else None
        hide = dist > 0 if case["causal"] else None
        for h in range(H):
            kh = h // (H // Hk)
            ps = []
            for m in range(maps):
                s = (q[b, :nq, h, m] @ k[b, :n, kh, m].T) * scale
                if tab is not None:
                    s = s + tab[:, h][bk]
                if hide is not None:
                    s = s.masked_fill(hide, -math.inf)
                ps.append(torch.softmax(s, dim=-1))
            w = ps[0] - lam * ps[1] if maps == 2 else ps[0]
            vb = v[b, :n, kh]
            out[b, :nq, h] = w @ vb
            if not train:
                continue
            dob = do[b, :nq, h]
            dv_[b, :n, kh] += w.T @ dob
            dw = dob @ vb.T
            for m in range(maps):
                c = 1.0 if m == 0 else -lam
                D = (ps[m] * dw).sum(dim=-1, keepdim=True)
                ds = c * ps[m] * (dw - D)
                dq[b, :nq, h, m] = scale * (ds @ k[b, :n, kh, m])
                dk_[b, :n, kh, m] += scale * (ds.T @ q[b, :nq, h, m])
                if dtab is not None:
                    dtab[:, h] += torch.zeros(case["buckets"], dtype=torch.float64, device=dev).index_add_(0, bk.reshape(-1), ds.reshape(-1))
                if m == 1:
                    dlam -= float(D.sum())
    res = {"out": out.flatten(2)}
    if train:
        res["dqkv"] = torch.cat([dq.flatten(2), dk_.flatten(2), dv_.flatten(2)], dim=2)
        if dtab is not None:
            res["dtable"] = dtab
        if maps == 2:
            res["dlam"] = torch.stack([dlam * e1 * lv[1], dlam * e1 * lv[0], -dlam * e2 * lv[3], -dlam * e2 * lv[2]])[:, None]
    return res


def _exact_norm(case, st):
    rms, C = case["kind"] == "rms", case["C"]
    d = {n: (st[n].double() if st.get(n) is not None else None) for n in ("f", "x", "gate", "post_g", "post_b", "pre_g", "pre_b", "dy", "dz")}
    rows = (torch.arange(case["T"], device=st["f"].device)[None, :] < st["lengths"].long()[:, None])[:, :, None].double()

    def hat(v):
        mu = 0.0 if rms else v.mean(-1, keepdim=True)
        r = ((v - mu).square().mean(-1, keepdim=True) + _EPS).rsqrt()
        return (v - mu) * r, r

    def hat_back(gh, h, r):
        t = gh - h * (gh * h).mean(-1, keepdim=True)
        return r * (t if rms else t - gh.mean(-1, keepdim=True))

    fh, fr = hat(d["f"])
    u = fh * d["post_g"] + (0.0 if rms else d["post_b"])
    gate = 1.0 if d["gate"] is None else (d["gate"][:, None] if case["gate"] == "utt" else d["gate"])
    y = (d["x"] + 0.5 * gate * u) * rows
    yh, yr = hat(y)
    z = (yh * d["pre_g"] + (0.0 if rms else d["pre_b"])) * rows
    res = {"y": y, "z": z}
    if case["mode"] == "train":
        dz = d["dz"] * rows
        dx = (d["dy"] + hat_back(dz * d["pre_g"], yh, yr)) * rows
        du = 0.5 * gate * dx
        res["df"], res["dx"] = hat_back(du * d["post_g"], fh, fr), dx
        if d["gate"] is not None:
            dg = 0.5 * u * dx
            res["dgate"] = dg.sum(1) if case["gate"] == "utt" else dg.sum((0, 1))
        res["dpost_g"] = (du * fh).sum((0, 1))
        if not rms:
            res["dpost_b"] = du.sum((0, 1))
        res["dpre_g"] = (dz * yh).sum((0, 1))
        if not rms:
            res["dpre_b"] = dz.sum((0, 1))
    return res


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(case, st) if case["op"] == "norm" else _exact_attention(case, st)
