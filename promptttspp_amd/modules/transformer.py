"""FFT-block Transformer encoder plug-in (reference: promptttspp/modules/transformer.py:23-263) -- the alternative
occupant of the model's ``encoder:`` slot (model.py:95: ``self.encoder(x, phone_mask)``), SURVEY section 8f n3.

Same classes, constructor arguments and state-dict keys as the reference.  Everything GEMM-shaped runs on the
package's kernels, channels-last: the fused q|k|v projection and the output projection (``ptpp_conv1d_fwd``), the
plain multi-head attention core incl. probability dropout (``ptpp_attention_fwd/bwd``, PLAIN variant), the
k-tap / 1x1 feed-forward convolutions with ReLU, masks and dropout fused, and the residual + dropout + LayerNorm of
every sub-layer (``ptpp_layernorm_fwd/bwd``).  The windowed relative-position attention core (``use_rel=True``,
Shaw et al. window of +-4) is one launch forward and three backward since round 4 (``ptpp_attention_win_fwd/bwd``: the row
kernels with the band terms as index arithmetic); the tensor-op form it replaced stays as the test's second opinion.

Masking note: the reference fills masked scores with -1e4 (not -inf), which gives PADDED query rows a uniform
attention over all positions; every layer ends in ``x * mask`` and every convolution reads ``x * mask``, so padded
rows never reach a valid row or the output.  The PLAIN kernel writes zeros there instead: outputs are identical.

Beyond the reference, for long inputs (memory linear in the sequence length): ``attention="bucket"`` -- a learned relative-position
bias by buckets -- and ``attention="diff"`` -- differential attention with a norm per head --, and ``norm="sandwich"``: a residual
stream with a norm before and behind every sub-layer, a gate (learned, or from the conditioning vector) and a residual scale, one
launch between two sub-layers.  The defaults are the reference's.
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import functional as PF
from .. import ops
from ..config import compute_dtype
from ..layers.norm import LayerNorm


def _lengths_of(mask):
    """(B,1,T) prefix mask -> (B,) int32 lengths"""
    return mask.sum(dim=(1, 2)).to(torch.int32)


class MultiHeadAttention(nn.Module):
    def __init__(self, channels, n_heads, dropout):
        super().__init__()
        assert channels % n_heads == 0
        self.inter_channels = channels // n_heads
        self.n_heads = n_heads
        self.scale = 1 / math.sqrt(self.inter_channels)
        self.qkv = nn.Conv1d(channels, channels * 3, 1)
        self.out = nn.Conv1d(channels, channels, 1)
        self.drop = nn.Dropout(dropout)

    def forward_cl(self, x, lengths):
        """x (B,T,C).  The reference views the 3C projection as [3][H][D]: q | k | v with contiguous heads -- the
        layout the attention kernel reads."""
        qkv = PF.conv1d(x, self.qkv.weight, self.qkv.bias)
        ctx = PF.attention(qkv, None, None, None, lengths, self.n_heads, "plain",
                           drop_p=float(self.drop.p) if self.training else 0.0)
        return PF.conv1d(ctx, self.out.weight, self.out.bias)

    def forward(self, x, mask):
        """Reference signature: x (B,C,T), mask (B,1,T,T) or None -> (B,C,T)."""
        B, C, T = x.shape
        lengths = None if mask is None else mask[:, 0].amax(dim=1).sum(dim=-1).to(torch.int32)
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), lengths))


class RelativeMultiHeadAttention(nn.Module):
    """Windowed relative positional attention: scores += q . emb_rel_k[j - i] and output += p . emb_rel_v[j - i]
    for |j - i| <= window_size (the reference's pad / view re-indexing, written as band gathers)."""

    def __init__(self, channels, n_heads, dropout, window_size=4):
        super().__init__()
        assert channels % n_heads == 0
        self.inter_channels = channels // n_heads
        self.n_heads = n_heads
        self.window_size = window_size
        self.scale = math.sqrt(self.inter_channels)
        self.conv_q = nn.Conv1d(channels, channels, 1)
        self.conv_k = nn.Conv1d(channels, channels, 1)
        self.conv_v = nn.Conv1d(channels, channels, 1)
        self.conv_o = nn.Conv1d(channels, channels, 1)
        self.drop = nn.Dropout(dropout)
        rel_stddev = self.inter_channels ** -0.5
        self.emb_rel_k = nn.Parameter(torch.randn(1, window_size * 2 + 1, self.inter_channels) * rel_stddev)
        self.emb_rel_v = nn.Parameter(torch.randn(1, window_size * 2 + 1, self.inter_channels) * rel_stddev)
        nn.init.xavier_uniform_(self.conv_q.weight)
        nn.init.xavier_uniform_(self.conv_k.weight)
        nn.init.xavier_uniform_(self.conv_v.weight)

    WINDOW_KERNEL = not __import__("os").environ.get("PTPP_NO_WINDOW_ATTN_KERNEL")  # (tests compare with the tensor-op form)

    def forward_cl(self, x, lengths):
        B, T, C = x.shape
        H, D, w = self.n_heads, self.inter_channels, self.window_size
        if self.WINDOW_KERNEL and x.is_cuda and D in (64, 128, 256) and T <= 2048:
            # the core as one launch (ptpp_attention_win_fwd / _bwd): band terms as index arithmetic, softmax in registers;
            # padded query rows come out zero (the tensor-op form below gives them a uniform attention that the layer's
            # mask removes: identical layer outputs)
            qkv = PF.linear_fused(x, [self.conv_q, self.conv_k, self.conv_v]).contiguous()
            ctx = PF.attention_window(qkv, self.emb_rel_k[0], self.emb_rel_v[0], lengths, H, w,
                                      drop_p=float(self.drop.p) if self.training else 0.0)
            return PF.conv1d(ctx, self.conv_o.weight, self.conv_o.bias)
        return self._forward_cl_tensor_ops(x, lengths)

    def _forward_cl_tensor_ops(self, x, lengths):
        B, T, C = x.shape
        H, D, w = self.n_heads, self.inter_channels, self.window_size
        qkv = PF.linear_fused(x, [self.conv_q, self.conv_k, self.conv_v]).float()
        q, k, v = (t.reshape(B, T, H, D).transpose(1, 2) for t in qkv.split(C, dim=-1))  # (B,H,T,D)
        q = q / self.scale
        scores = q @ k.transpose(-2, -1)
        # relative part: r = j - i + w in [0, 2w]; entries outside the band are the reference's zero padding
        i = torch.arange(T, device=x.device)
        r = i[None, :] - i[:, None] + w                                 # (T, T)
        band = (r >= 0) & (r <= 2 * w)
        rc = r.clamp(0, 2 * w)
        rel = q @ self.emb_rel_k[0].float().t()                         # (B,H,T,2w+1)
        scores = scores + rel.gather(-1, rc.expand(B, H, T, T)) * band
        if lengths is not None:
            valid = i[None, :] < lengths[:, None]                        # (B,T)
            scores = scores.masked_fill(~(valid[:, None, :, None] & valid[:, None, None, :]), -1e4)
        p = self.drop(F.softmax(scores, dim=-1))
        out = p @ v
        # relative_weights[i, r] = p[i, i + r - w] (0 outside the sequence)
        jj = i[:, None] + torch.arange(2 * w + 1, device=x.device)[None, :] - w   # (T, 2w+1)
        inside = (jj >= 0) & (jj < T)
        relw = p.gather(-1, jj.clamp(0, T - 1).expand(B, H, T, 2 * w + 1)) * inside
        out = out + relw @ self.emb_rel_v[0].float()
        out = out.transpose(1, 2).reshape(B, T, C).to(x.dtype).contiguous()
        return PF.conv1d(out, self.conv_o.weight, self.conv_o.bias)

    def forward(self, x, mask):
        lengths = None if mask is None else mask[:, 0].amax(dim=1).sum(dim=-1).to(torch.int32)
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), lengths))


class BucketAttention(nn.Module):
    """Self-attention with a learned bias per head and relative-position bucket (``PF.attention_bucket``).  ``kv_heads`` < ``n_heads``:
    key / value heads shared by groups of query heads.  Dropout applies to the output projection."""

    def __init__(self, channels, n_heads, dropout, num_buckets=32, max_distance=128, kv_heads=None):
        super().__init__()
        assert channels % n_heads == 0
        self.n_heads, self.kv_heads, self.max_distance = n_heads, kv_heads or n_heads, max_distance
        width = channels // n_heads
        self.qkv = nn.Conv1d(channels, (n_heads + 2 * self.kv_heads) * width, 1)
        self.out = nn.Conv1d(channels, channels, 1)
        self.rel_bias = nn.Parameter(torch.randn(num_buckets, n_heads) * 0.02)
        self.drop = nn.Dropout(dropout)

    def _context(self, x, lengths):
        qkv = PF.conv1d(x, self.qkv.weight, self.qkv.bias)
        return PF.attention_bucket(qkv, None, None, self.rel_bias, self.n_heads, kv_heads=self.kv_heads, max_distance=self.max_distance,
                                   lengths=lengths)

    def forward_cl(self, x, lengths):
        return PF.conv1d(self._context(x, lengths), self.out.weight, self.out.bias, drop_p=float(self.drop.p) if self.training else 0.0)

    def forward(self, x, mask):
        lengths = None if mask is None else mask[:, 0].amax(dim=1).sum(dim=-1).to(torch.int32)
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), lengths))


class DifferentialAttention(BucketAttention):
    """Differential self-attention (``PF.attention_diff``; Ye et al. 2024): every head is the difference of two softmax maps with learned
    lam (vectors shared by the heads, lam_init from the layer's depth), then a root-mean-square norm per head scaled by 1 - lam_init
    (``PF.residual_norm`` without a residual).  ``num_buckets`` = 0: no position bias."""

    def __init__(self, channels, n_heads, dropout, num_buckets=32, max_distance=128, kv_heads=None, depth=0):
        super().__init__(channels, n_heads, dropout, max(num_buckets, 1), max_distance, kv_heads)
        if not num_buckets:
            del self.rel_bias
            self.rel_bias = None
        self.head_width = channels // n_heads
        assert self.head_width % 2 == 0
        self.lam_init = 0.8 - 0.6 * math.exp(-0.3 * depth)
        self.lam = nn.Parameter(torch.randn(4, 1, self.head_width // 2) * 0.1)
        self.sub_norm = nn.Parameter(torch.ones(self.head_width))

    def _context(self, x, lengths):
        B, T, _ = x.shape
        qkv = PF.conv1d(x, self.qkv.weight, self.qkv.bias)
        ctx = PF.attention_diff(qkv, None, None, self.lam, self.lam_init, self.n_heads, kv_heads=self.kv_heads, table=self.rel_bias,
                                max_distance=self.max_distance, lengths=lengths)
        y, _ = PF.residual_norm(ctx.view(B, T * self.n_heads, self.head_width), post=(self.sub_norm, None), kind="rms", scale=1.0 - self.lam_init,
                                lengths=None if lengths is None else lengths * self.n_heads)
        return y.view(B, T, -1)


class FFN(nn.Module):
    def __init__(self, channels, kernel_size, dropout, scale):
        super().__init__()
        self.conv1 = nn.Conv1d(channels, channels * scale, kernel_size, padding=kernel_size // 2)
        self.conv2 = nn.Conv1d(channels * scale, channels, 1)
        self.drop = nn.Dropout(dropout)

    def forward_cl(self, x, lengths, drop_out=0.0):
        """drop_out(conv2(drop(relu(conv1(x * m))) * m)) * m"""
        k = self.conv1.kernel_size[0]
        h = PF.conv1d(x, self.conv1.weight, self.conv1.bias, ks=k, pad=k // 2, act="relu", lengths=lengths, in_mask=True,
                      drop_p=float(self.drop.p) if self.training else 0.0)
        return PF.conv1d(h, self.conv2.weight, self.conv2.bias, lengths=lengths, in_mask=True, out_mask=True, drop_p=drop_out)

    def forward(self, x, x_mask):
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), _lengths_of(x_mask)))


class _AttnSubLayer(nn.Module):
    """x = norm(x + dropout(attention(x)))"""

    def forward_cl(self, x, lengths):
        y = self.attention_layer.forward_cl(x, lengths)
        return self.norm.forward_cl(y, res=x, drop_in=float(self.dropout.p) if self.training else 0.0)

    def forward(self, x, attn_mask):
        lengths = None if attn_mask is None else attn_mask[:, 0].amax(dim=1).sum(dim=-1).to(torch.int32)
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), lengths))


class AttentionLayer(_AttnSubLayer):
    def __init__(self, channels, num_head, dropout):
        super().__init__()
        self.attention_layer = MultiHeadAttention(channels, num_head, dropout)
        self.norm = LayerNorm(channels)
        self.dropout = nn.Dropout(dropout)


class RelativeAttentionLayer(_AttnSubLayer):
    def __init__(self, channels, num_head, dropout, window_size):
        super().__init__()
        self.attention_layer = RelativeMultiHeadAttention(channels, num_head, dropout, window_size)
        self.norm = LayerNorm(channels)
        self.dropout = nn.Dropout(dropout)


class FFNLayer(nn.Module):
    def __init__(self, channels, kernel_size, dropout, scale):
        super().__init__()
        self.ffn = FFN(channels, kernel_size, dropout, scale)
        self.norm = LayerNorm(channels)
        self.dropout = nn.Dropout(dropout)

    def forward_cl(self, x, lengths):
        """norm(x + dropout(ffn(x))) * mask"""
        y = self.ffn.forward_cl(x, lengths)
        return self.norm.forward_cl(y, res=x, drop_in=float(self.dropout.p) if self.training else 0.0, lengths=lengths,
                                    out_mask=True)

    def forward(self, x, mask):
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), _lengths_of(mask)))


class LongAttentionLayer(_AttnSubLayer):
    """x = norm(x + dropout(attention(x))) around ``BucketAttention`` / ``DifferentialAttention`` (built without a dropout of their own)"""

    def __init__(self, channels, attention, dropout):
        super().__init__()
        self.attention_layer = attention
        self.norm = LayerNorm(channels)
        self.dropout = nn.Dropout(dropout)


def long_attention(kind, channels, num_head, dropout, depth, num_buckets, max_distance, kv_heads):
    if kind == "bucket":
        return BucketAttention(channels, num_head, dropout, num_buckets, max_distance, kv_heads)
    if kind == "diff":
        return DifferentialAttention(channels, num_head, dropout, num_buckets, max_distance, kv_heads, depth)
    raise ValueError(f"attention {kind!r}: None (plain, or windowed with use_rel), 'bucket' or 'diff'")


class TransformerLayer(nn.Module):
    def __init__(self, channels, num_head, kernel_size, dropout, scale, window_size=None, use_rel=False, attention=None, depth=0, num_buckets=32,
                 max_distance=128, kv_heads=None):
        super().__init__()
        if attention is not None:
            self.attention = LongAttentionLayer(channels, long_attention(attention, channels, num_head, 0.0, depth, num_buckets, max_distance, kv_heads),
                                                dropout)
        elif use_rel:
            self.attention = RelativeAttentionLayer(channels, num_head, dropout, window_size)
        else:
            self.attention = AttentionLayer(channels, num_head, dropout)
        self.ffn = FFNLayer(channels, kernel_size, dropout, scale)

    def forward_cl(self, x, lengths):
        return self.ffn.forward_cl(self.attention.forward_cl(x, lengths), lengths)

    def forward(self, x, mask, attn_mask):
        return ops.btc_to_bct(self.forward_cl(ops.bct_to_btc(x, compute_dtype()), _lengths_of(mask)))


class _SandwichNorms(nn.Module):
    """What stands between two sub-layers of a ``norm="sandwich"`` stack: the norm behind the first, its gate, the norm before the next"""

    def __init__(self, channels):
        super().__init__()
        self.post, self.pre = LayerNorm(channels), LayerNorm(channels)
        self.gate = nn.Parameter(torch.ones(channels))

    def step(self, f, x, gate, scale, lengths):
        return PF.residual_norm(f, x, gate=gate, post=(self.post.gamma, self.post.beta), pre=(self.pre.gamma, self.pre.beta), scale=scale,
                                eps=self.post.eps, lengths=lengths)


class SandwichStack(nn.Module):
    """The layers of ``Transformer(norm="sandwich")``: z = norm(x); then for every attention and feed-forward sub-layer
    x <- x + residual_scale * gate * norm(sub-layer(z)), z <- norm(x) in one launch; the last z is the output.

    ``cond_channels``: the conditioning vector g (B, 1, cond_channels) gates every sub-layer through one projection (zero at the start:
    the learned gates alone), gate = learned + projection(g).  Such a stack is always called with g; the acoustic model's encoder slot has
    none to give, so there the gates are the learned ones (no ``cond_channels``)."""

    def __init__(self, channels, num_head, num_layers, kernel_size, dropout, scale, attention, num_buckets, max_distance, kv_heads, residual_scale,
                 cond_channels):
        super().__init__()
        self.residual_scale = residual_scale
        self.attentions = nn.ModuleList([long_attention(attention, channels, num_head, dropout, i, num_buckets, max_distance, kv_heads)
                                         for i in range(num_layers)])
        self.ffns = nn.ModuleList([FFN(channels, kernel_size, dropout, scale) for _ in range(num_layers)])
        self.drop = nn.Dropout(dropout)
        self.norm = LayerNorm(channels)
        self.steps = nn.ModuleList([_SandwichNorms(channels) for _ in range(2 * num_layers)])
        self.cond = None
        if cond_channels:
            self.cond = nn.Linear(cond_channels, 2 * num_layers * channels)
            nn.init.zeros_(self.cond.weight)
            nn.init.zeros_(self.cond.bias)

    def _gates(self, g):
        if g is None:
            if self.cond is not None:
                raise ValueError("norm='sandwich' was built with cond_channels: it needs the conditioning vector (its projection would never learn)")
            return [s.gate for s in self.steps]
        if self.cond is None or g.shape[1] != 1:
            raise ValueError("norm='sandwich' takes its conditioning as one vector per utterance, through gates (cond_channels)")
        c = PF.linear(g.contiguous(), self.cond.weight, self.cond.bias).float()              # (B, 1, steps * C)
        c = c.view(g.shape[0], len(self.steps), -1).transpose(0, 1).contiguous()              # (steps, B, C)
        return [c[i] + s.gate for i, s in enumerate(self.steps)]

    def forward_cl(self, x, lengths, g=None):
        gates = self._gates(g)
        z = self.norm.forward_cl(x, lengths=lengths, out_mask=True)
        for i, (attention, ffn) in enumerate(zip(self.attentions, self.ffns)):
            x, z = self.steps[2 * i].step(attention.forward_cl(z, lengths), x, gates[2 * i], self.residual_scale, lengths)
            f = ffn.forward_cl(z, lengths, drop_out=float(self.drop.p) if self.training else 0.0)
            x, z = self.steps[2 * i + 1].step(f, x, gates[2 * i + 1], self.residual_scale, lengths)
        return z


class Transformer(nn.Module):
    """``attention``: None (the reference's: plain, or windowed relative with ``use_rel``), "bucket" or "diff"; ``norm``: "post" (the
    reference's) or "sandwich".  ``num_buckets`` / ``max_distance`` / ``kv_heads``: of the two long forms; ``residual_scale`` /
    ``cond_channels``: of the sandwich (see ``SandwichStack``)."""

    def __init__(self, channels, num_head, num_layers, kernel_size, dropout, scale=4, window_size=None, use_rel=False, attention=None, norm="post",
                 num_buckets=32, max_distance=128, kv_heads=None, residual_scale=1.0, cond_channels=None):
        super().__init__()
        self.channels = channels
        self.norm_form = norm
        if norm == "sandwich":
            self.stack = SandwichStack(channels, num_head, num_layers, kernel_size, dropout, scale, attention, num_buckets, max_distance, kv_heads,
                                       residual_scale, cond_channels)
        elif norm == "post":
            self.layers = nn.ModuleList([TransformerLayer(channels, num_head, kernel_size, dropout, scale, window_size, use_rel, attention, i, num_buckets,
                                                          max_distance, kv_heads) for i in range(num_layers)])
        else:
            raise ValueError(f"norm {norm!r}: 'post' or 'sandwich'")

    def forward_cl(self, x, lengths, g=None):
        """x (B,T,C) channels-last in the compute dtype; g: optional (B,1,C) / (B,T,C) conditioning added before
        every layer (transformer.py:258-260); with ``norm="sandwich"`` (B,1,cond_channels), through the gates."""
        if self.norm_form == "sandwich":
            return self.stack.forward_cl(x, lengths, g)
        for layer in self.layers:
            if g is not None:
                x = x + g
            x = layer.forward_cl(x, lengths)
        return x

    def forward(self, x, mask, g=None):
        """Reference signature: x (B,C,T), mask (B,1,T), g (B,C,1) -> (B,C,T)."""
        gc = None if g is None else g.transpose(1, 2).to(compute_dtype())
        y = self.forward_cl(ops.bct_to_btc(x, compute_dtype()), _lengths_of(mask), gc)
        return ops.btc_to_bct(y)
