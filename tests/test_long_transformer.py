"""The long-input forms of the FFT-block Transformer (modules/transformer.py: attention="bucket" / "diff", norm="sandwich") -- bucketed-bias
and differential attention and the residual-norm step together, as the model's encoder slot runs them -- against a plain
implementation of the same modules in 64 bits."""
import os

import pytest
import torch
import torch.nn.functional as F

from conftest import ROOT
from test_encoder_block_ops import ref_bucket

CONF = os.path.join(ROOT, "egs", "proposed", "bin", "conf", "model")


def l2(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / (b.norm() + 1e-30))


def conv(x, c):
    k = c.weight.shape[-1]
    return F.conv1d(x.transpose(1, 2), c.weight, c.bias, padding=k // 2).transpose(1, 2)


def ln(x, n):
    return F.layer_norm(x, x.shape[-1:], n.gamma.reshape(-1), n.beta.reshape(-1), n.eps)


def ref_attention(m, x, lens):
    B, T, _ = x.shape
    H, G = m.n_heads, m.kv_heads
    diff = hasattr(m, "lam")
    qkv = conv(x, m.qkv)
    w = qkv.shape[2] // (H + 2 * G)
    q, k, v = qkv.split([H * w, G * w, G * w], dim=2)
    maps = 2 if diff else 1
    d = w // maps
    q, k = q.view(B, T, H, maps, d), k.view(B, T, G, maps, d).repeat_interleave(H // G, dim=2)
    v = v.view(B, T, G, w).repeat_interleave(H // G, dim=2)
    see = torch.arange(T)[None] < lens[:, None]
    dist = torch.arange(T)[None] - torch.arange(T)[:, None]
    bias = 0.0
    if m.rel_bias is not None:
        bias = m.rel_bias[ref_bucket(dist, m.rel_bias.shape[0], m.max_distance, True)].permute(2, 0, 1)[None]
    ps = []
    for i in range(maps):
        s = torch.einsum("bihd,bjhd->bhij", q[:, :, :, i], k[:, :, :, i]) * d ** -0.5 + bias
        ps.append(s.masked_fill(~see[:, None, None], float("-inf")).softmax(-1))
    a = ps[0]
    if diff:
        lam = (m.lam[0, 0] @ m.lam[1, 0]).exp() - (m.lam[2, 0] @ m.lam[3, 0]).exp() + m.lam_init
        a = ps[0] - lam * ps[1]
    ctx = torch.einsum("bhij,bjhd->bihd", a, v)
    if diff:
        ctx = ctx * torch.rsqrt(ctx.square().mean(-1, keepdim=True) + 1e-5) * m.sub_norm * (1.0 - m.lam_init)
    ctx = ctx.reshape(B, T, H * w) * see[:, :, None]
    return conv(ctx, m.out)


def ref_ffn(m, x, mask):
    return conv(conv(x * mask, m.conv1).relu() * mask, m.conv2) * mask


def ref_transformer(m, x, lens, g=None):
    mask = (torch.arange(x.shape[1])[None] < lens[:, None])[:, :, None].to(x.dtype)
    if m.norm_form == "post":
        for lay in m.layers:
            a = lay.attention
            x = ln(x + ref_attention(a.attention_layer, x, lens), a.norm)
            x = ln(x + ref_ffn(lay.ffn.ffn, x, mask), lay.ffn.norm) * mask
        return x
    st = m.stack
    gates = [s.gate for s in st.steps]
    if g is not None:
        c = F.linear(g, st.cond.weight, st.cond.bias).view(g.shape[0], len(st.steps), -1)
        gates = [(c[:, i] + s.gate)[:, None] for i, s in enumerate(st.steps)]
    z = ln(x, st.norm) * mask
    for i, s in enumerate(st.steps):
        f = ref_attention(st.attentions[i // 2], z, lens) if i % 2 == 0 else ref_ffn(st.ffns[i // 2], z, mask)
        x = (x + st.residual_scale * gates[i] * ln(f, s.post)) * mask
        z = ln(x, s.pre) * mask
    return z


def build(seed=0, **kw):
    from promptttspp_amd.modules.transformer import Transformer

    torch.manual_seed(seed)
    m = Transformer(channels=256, num_head=4, num_layers=2, kernel_size=3, dropout=0.1, scale=2, num_buckets=16, max_distance=40, **kw)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if n.endswith(("gamma", "sub_norm", "gate")):
                p.add_(0.1 * torch.randn_like(p))
            elif n.endswith(("beta", "rel_bias")) or ".cond." in n:
                p.add_(0.1 * torch.randn_like(p))
    return m


FORMS = [dict(attention="bucket"), dict(attention="diff", kv_heads=2), dict(attention="bucket", norm="sandwich", residual_scale=0.5),
         dict(attention="diff", norm="sandwich", cond_channels=64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 3e-5), (torch.bfloat16, 4e-2)])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_transformer_against_64_bits(dev, dtype, tol, form):
    """Outputs and every gradient of a two-layer stack.  f32: each of the ~15 operators in a row is off by a few 2^-24 of its terms, which two
    layers of norms amplify to below 3e-5 (relative 2-norm); bf16: about 20 roundings of 2^-9 root mean square each in a row, likewise
    amplified: below 4e-2."""
    import copy

    from promptttspp_amd import config, ops

    m = build(**FORMS[form])
    ref = copy.deepcopy(m).double()
    B, T = 3, 150
    lens = torch.tensor([150, 1, 97])
    gen = torch.Generator().manual_seed(5)
    x, dy = torch.randn(B, 256, T, generator=gen), torch.randn(B, 256, T, generator=gen)
    g = torch.randn(B, 1, 64, generator=gen) if "cond_channels" in FORMS[form] else None
    if dtype == torch.bfloat16:
        x, dy = x.bfloat16().float(), dy.bfloat16().float()
        g = None if g is None else g.bfloat16().float()
    xr = x.transpose(1, 2).double().requires_grad_()
    yr = ref_transformer(ref, xr, lens, None if g is None else g.double())
    yr.backward(dy.transpose(1, 2).double() * (torch.arange(T)[None] < lens[:, None])[:, :, None])
    m = m.to(dev).eval()
    with config.use_dtype(dtype):
        xc = ops.bct_to_btc(x.to(dev), dtype).requires_grad_()
        y = m.forward_cl(xc, lens.to(dev).int(), None if g is None else g.to(dev).to(dtype))
        y.backward(dy.transpose(1, 2).contiguous().to(dev).to(dtype))
        assert l2(y.float(), yr) < tol
        valid = (torch.arange(T)[None] < lens[:, None])[:, :, None]
        assert l2(xc.grad.float().cpu() * valid, xr.grad) < 2 * tol
        P = dict(m.named_parameters())
        for n, p in ref.named_parameters():
            assert P[n].grad is not None, n
            # a key bias moves every score of a row alike: its gradient is zero but for roundings; compare the q and v parts and scale
            got, want = P[n].grad.double().cpu(), p.grad
            err = float((got - want).norm() / (want.norm() + 1e-4 * max(float(q.grad.norm()) for q in ref.parameters())))
            assert err < 3 * tol, (n, err)
        if "norm" in FORMS[form]:  # the reference signature, mask and (B, C, 1) conditioning included
            mask = (torch.arange(T)[None] < lens[:, None])[:, None].float().to(dev)
            with torch.no_grad():
                y2 = m(x.to(dev), mask, g=None if g is None else g.transpose(1, 2).to(dev))
            assert l2(y2.transpose(1, 2), y.float()) < tol


@pytest.mark.gpu
def test_gradients_land_in_the_flat_buffer(dev):
    """With the trainer's flat gradient buffer the kernels add the parameters' gradients in place: twice the gradient after two passes"""
    from promptttspp_amd import config
    from promptttspp_amd import functional as PF
    from promptttspp_amd.parallel import FlatGradReducer

    with config.use_dtype(torch.float32):
        m = build(**FORMS[2]).to(dev).eval()
        x = torch.randn(2, 60, 256, device=dev)
        lens = torch.tensor([60, 33], device=dev, dtype=torch.int32)

        def step():
            (m.forward_cl(x, lens).float() ** 2).sum().backward()

        step()
        want = {n: p.grad.clone() for n, p in m.named_parameters()}
        m.zero_grad(set_to_none=True)
        try:
            red = FlatGradReducer(list(m.parameters()))
            red.zero_grad()
            step()
            step()
            red.finish()
            torch.cuda.synchronize()
            for n, p in m.named_parameters():
                assert l2(p.grad, 2 * want[n]) < 1e-5 or float(want[n].norm()) < 1e-3, n
        finally:
            PF.enable_direct_grads(False)


def test_a_parameter_given_twice_is_not_added_to_in_place():
    """in the flat buffer's mode one launch would add to the same gradient from two blocks at once"""
    from promptttspp_amd import functional as PF

    a, b = (torch.nn.Parameter(torch.ones(8)) for _ in range(2))
    a.grad, b.grad = torch.zeros(8), torch.zeros(8)
    on = PF._direct["on"]
    PF._direct["on"] = True
    try:
        assert PF._param_sinks([a, b]) == [a, b]
        assert PF._param_sinks([a, b, a]) is None
    finally:
        PF._direct["on"] = on


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 60, 256), (40, 33, 64)])
def test_one_norm_behind_and_before_a_block(dev, shape):
    """the same (gamma, beta) as post and pre norm: the flat buffer gets the sum of both gradients, which is what the norms given
    separately get"""
    from promptttspp_amd import functional as PF
    from promptttspp_amd.parallel import FlatGradReducer

    B, T, C = shape
    gen = torch.Generator(device=dev).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    f, x, dy, dz = r(B, T, C), r(B, T, C), r(B, T, C), r(B, T, C)
    gamma, beta = torch.nn.Parameter(1 + 0.1 * r(C)), torch.nn.Parameter(0.1 * r(C))
    apart = [p.detach().clone().requires_grad_() for p in (gamma, beta, gamma, beta)]
    want = torch.autograd.grad(PF.residual_norm(f, x, post=tuple(apart[:2]), pre=tuple(apart[2:])), apart, (dy, dz))
    try:
        red = FlatGradReducer([gamma, beta])
        red.zero_grad()
        for _ in range(2):
            torch.autograd.backward(PF.residual_norm(f, x, post=(gamma, beta), pre=(gamma, beta)), (dy, dz))
        red.finish()
        torch.cuda.synchronize()
        for p, a, b in ((gamma, want[0], want[2]), (beta, want[1], want[3])):
            # each sum is the same f32 value in both calls: three additions of them remain
            assert bool(((p.grad - 2 * (a + b)).abs() <= 4 * 2.0 ** -24 * 2 * (a.abs() + b.abs())).all())
    finally:
        PF.enable_direct_grads(False)


@pytest.mark.gpu
@pytest.mark.parametrize("form", [1, 3])
def test_training_mode_runs_with_dropout(dev, form):
    from promptttspp_amd import config

    with config.use_dtype(torch.bfloat16):
        m = build(**FORMS[form]).to(dev).train()
        x = torch.randn(2, 70, 256, device=dev).bfloat16().requires_grad_()
        g = torch.randn(2, 1, 64, device=dev).bfloat16() if form == 3 else None
        lens = torch.tensor([70, 20], device=dev, dtype=torch.int32)
        a, b = m.forward_cl(x, lens, g), m.forward_cl(x, lens, g)
        assert not torch.equal(a, b)
        a.float().sum().backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())
        assert float(a[1, 20:].abs().max()) == 0.0 and float(x.grad[1, 20:].abs().max()) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(attention="bucket"), dict(attention="diff", norm="sandwich")])
def test_model_takes_it_in_the_encoder_slot(dev, kw):
    """the acoustic model with this encoder: a forward with all losses and a backward that reaches its parameters"""
    import test_hip_acoustic as A
    from conftest import load_golden
    from promptttspp_amd import config
    from promptttspp_amd import hydra_lite as H

    cfg = H.load_node(os.path.join(CONF, "prompttts_mdn_v2_wo_erg_final.yaml"))
    cfg["encoder"] = {"_target_": "promptttspp.modules.transformer.Transformer", "channels": 256, "num_head": 2, "num_layers": 2, "kernel_size": 3,
                      "dropout": 0.1, "scale": 4, **kw}
    cfg["decoder"]["in_dim"] = 256
    with config.use_dtype(torch.float32):
        model = H.instantiate(cfg).to(dev).train()
        out = model(A._batch(load_golden("model_forward"), dev))
        assert bool(torch.isfinite(out["loss"]))
        out["loss"].backward()
        for n, p in model.encoder.named_parameters():
            assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n


def test_forms_and_defaults():
    from promptttspp_amd.modules.transformer import Transformer

    base = Transformer(256, 2, 2, 3, 0.1)
    assert [n for n in base.state_dict()] == [n for n in Transformer(256, 2, 2, 3, 0.1, scale=4, window_size=4, use_rel=False).state_dict()]
    assert "layers.0.attention.attention_layer.rel_bias" in Transformer(256, 2, 1, 3, 0.1, attention="bucket").state_dict()
    assert "stack.attentions.0.rel_bias" not in Transformer(256, 2, 1, 3, 0.1, attention="diff", norm="sandwich", num_buckets=0).state_dict()
    for kw in (dict(attention="other"), dict(norm="other"), dict(norm="sandwich"), dict(norm="sandwich", attention=None)):
        with pytest.raises(ValueError):
            Transformer(256, 2, 1, 3, 0.1, **kw)


def test_a_conditioned_stack_needs_its_conditioning():
    from promptttspp_amd.modules.transformer import Transformer

    x, g = torch.zeros(2, 5, 64), torch.zeros(2, 1, 16)
    kw = dict(attention="bucket", norm="sandwich")
    with pytest.raises(ValueError, match="conditioning vector"):
        Transformer(64, 2, 1, 3, 0.1, cond_channels=16, **kw).forward_cl(x, None)
    with pytest.raises(ValueError, match="cond_channels"):
        Transformer(64, 2, 1, 3, 0.1, **kw).forward_cl(x, None, g)
