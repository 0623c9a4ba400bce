"""Drop-in for the reference's models/fusion_nets.py SelfAttention and
Working (FCFM).  Parameter names match the reference (query_proj, key_proj,
value_proj, conv, bn_img, ...), so reference state dicts load unchanged.

The attention core (QK^T, softmax, PV and their backward) runs in the gfx950
kernels (kernels.AttentionCore); the 1x1 projections are plain GEMMs on a
channels-last view of the maps, so no NCHW<->NHWC copies are made.
"""
from __future__ import annotations

import numpy as np
import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import kernels as K

__all__ = ["SelfAttention", "CrossAttention", "Working", "conv1x1"]


def conv1x1(in_planes, out_planes):
    return nn.Conv2d(in_planes, out_planes, kernel_size=1, stride=1, padding=0, bias=False)


def _cl(x):
    """[N, C, H, W] (any strides) -> [N, H*W, C] view/copy, channels last."""
    n, c, h, w = x.shape
    return x.permute(0, 2, 3, 1).reshape(n, h * w, c)


class SelfAttention(nn.Module):
    """fusion_nets.py:82-118.

    forward(x, y): query role = key_proj(x), key role = query_proj(y),
    value = value_proj(x); softmax over y's positions; output [N, C, H, W]
    (returned as a channels-last strided view).
    """

    def __init__(self, channel_dim, scale=2):
        super().__init__()
        self.inplanes = channel_dim
        self.query_proj = nn.Conv2d(self.inplanes, self.inplanes // scale, 1)
        self.key_proj = nn.Conv2d(self.inplanes, self.inplanes // scale, 1)
        self.value_proj = nn.Conv2d(self.inplanes, self.inplanes, 1)
        self.sqrt_dim = np.sqrt(channel_dim / scale)
        self.precision = "fp32"

    def _w(self, conv):
        return conv.weight.reshape(conv.weight.shape[0], -1)

    def packed_self(self):
        """[key_proj; query_proj; value_proj] as one [2 C' + C, C] weight and
        bias: the query role, key role and value of self-attention."""
        w = torch.cat([self._w(self.key_proj), self._w(self.query_proj),
                       self._w(self.value_proj)], 0)
        b = torch.cat([self.key_proj.bias, self.query_proj.bias, self.value_proj.bias])
        return w, b

    def core_self(self, px):
        """Attention on packed [Qr | Kr | V] rows [N, HW, 2 C' + C]."""
        cq = self.key_proj.weight.shape[0]
        return K.attention_core(px, None, cq, cq, 2 * cq, 1.0 / float(self.sqrt_dim),
                                self.precision)

    def forward_cl(self, x_cl, y_cl):
        """Channels-last core: x_cl, y_cl [N, HW, C] -> [N, HW, C]."""
        mode = self.precision
        cq = self.key_proj.weight.shape[0]
        if y_cl is x_cl:
            w, b = self.packed_self()
            return self.core_self(K.linear_rows(x_cl, w, b, mode=mode))
        w = torch.cat([self._w(self.key_proj), self._w(self.value_proj)], 0)
        b = torch.cat([self.key_proj.bias, self.value_proj.bias])
        px = K.linear_rows(x_cl, w, b, mode=mode)                     # [Qr | V]
        py = K.linear_rows(y_cl, self._w(self.query_proj), self.query_proj.bias, mode=mode)
        return K.attention_core(px, py, cq, 0, cq, 1.0 / float(self.sqrt_dim), mode)

    def forward(self, x, y):
        n, c, h, w = y.shape
        assert x.shape[2] * x.shape[3] == h * w, "x and y need the same H*W (:105)"
        x_cl = _cl(x)
        y_cl = x_cl if y is x else _cl(y)
        o = self.forward_cl(x_cl, y_cl)
        return o.reshape(n, h, w, c).permute(0, 3, 1, 2)


class CrossAttention(nn.Module):
    """Attention of one side's tokens to the other side's states of another
    length (SelfAttention.forward needs one H*W on both, fusion_nets.py:105):
    regions reading a caption's words, words reading the regions, or single
    tokens against states that are kept.

    `heads` query heads on `kv_heads` key heads (default: as many) of
    channel_dim / heads elements; queries and keys are RMS-normed per head and,
    with `rope` (kernels.Rope), rotated by their positions in the same launch
    (kernels.qk_norm_rope), then kernels.cross_attention; 1x1 projections
    around them as in SelfAttention.  precision "fp32" runs the attention in
    fp32, "bf16" / "fp16" on tensors of that type."""

    def __init__(self, channel_dim, context_dim=None, heads=4, kv_heads=None, rope=None,
                 eps=1e-6):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if channel_dim % heads or heads % kv_heads:
            raise ValueError(f"{channel_dim} channels, {heads} heads on {kv_heads} key heads")
        self.heads, self.kv_heads = heads, kv_heads
        self.head_dim = channel_dim // heads
        kv = 2 * kv_heads * self.head_dim
        self.query_proj = nn.Linear(channel_dim, channel_dim)
        self.kv_proj = nn.Linear(channel_dim if context_dim is None else context_dim, kv)
        self.out_proj = nn.Linear(channel_dim, channel_dim)
        self.query_norm = nn.Parameter(torch.ones(self.head_dim))
        self.key_norm = nn.Parameter(torch.ones(self.head_dim))
        self.rope, self.eps = rope, eps
        self.precision = "fp32"

    def _dtype(self):
        return {"fp32": torch.float32, "bf16": torch.bfloat16,
                "fp16": torch.float16}[self.precision]

    def _queries(self, x):
        q = K.linear_rows(x, self.query_proj.weight, self.query_proj.bias, mode=self.precision)
        return q.unflatten(-1, (self.heads, self.head_dim))

    def _states(self, y):
        kv = K.linear_rows(y, self.kv_proj.weight, self.kv_proj.bias, mode=self.precision)
        return kv.unflatten(-1, (2, self.kv_heads, self.head_dim)).unbind(2)

    def context(self, y, y_pos=None):
        """The keys (normed, rotated) and values of y [N, T, context_dim], for
        forward(..., context=...) of any number of later steps."""
        k, v = self._states(y)
        _, k = K.qk_norm_rope(None, k, None, self.key_norm, eps=self.eps, rope=self.rope,
                              k_pos=y_pos, out_dtype=self._dtype())
        return k, v.to(self._dtype())

    def forward(self, x, y=None, x_pos=None, y_pos=None, x_lens=None, y_lens=None, y_mask=None,
                context=None):
        """x [N, Tx, channel_dim] reads y [N, Ty, context_dim] (or the kept
        `context` of it) -> [N, Tx, channel_dim].  x_lens, y_lens [N]: tokens
        of each sample; y_mask [N, Ty] (bool): False leaves a state out."""
        if (y is None) == (context is None):
            raise ValueError("either y or its context")
        q, dtype = self._queries(x), self._dtype()
        if context is None:
            k, v = self._states(y)
            q, k = K.qk_norm_rope(q, k, self.query_norm, self.key_norm, eps=self.eps,
                                  rope=self.rope, q_pos=x_pos, k_pos=y_pos, out_dtype=dtype)
            v = v.to(dtype)
        else:
            k, v = context
            q, _ = K.qk_norm_rope(q, None, self.query_norm, None, eps=self.eps, rope=self.rope,
                                  q_pos=x_pos, out_dtype=dtype)
        o = K.cross_attention(q, k, v, q_lens=x_lens, kv_lens=y_lens, mask=y_mask)
        return K.linear_rows(o.flatten(-2).float(), self.out_proj.weight, self.out_proj.bias,
                             mode=self.precision)


class Working(nn.Module):
    """fusion_nets.py:217-258 (FCFM).  The channel_dim argument is ignored
    exactly as in the reference (:220)."""

    def __init__(self, channel_dim):
        super().__init__()
        channel_dim = 36
        self.bn_img = nn.BatchNorm2d(channel_dim)
        self.bn_word = nn.BatchNorm2d(channel_dim)
        self.projection = nn.Linear(256, channel_dim)
        self.sa = SelfAttention(channel_dim, scale=1)
        self.maxpool = nn.MaxPool2d(kernel_size=2)
        self.conv = nn.Conv2d(256, channel_dim, kernel_size=(3, 3), padding=0)
        self.relu = nn.ReLU()
        self.ln = nn.LayerNorm([channel_dim, 6, 6])
        self.ln_gl_image = nn.LayerNorm([256])
        self.ln_sent = nn.LayerNorm([256])
        self.linear = nn.Linear(324, 128)

    def forward(self, img, word, gl_img, sent):
        mode = self.sa.precision
        sa = self.sa
        # conv3x3 + ReLU + maxpool (:236-237): one fused kernel each way
        img = K.conv_relu_pool(img, self.conv.weight, self.conv.bias, mode=mode)   # [B,36,6,6]
        # word projection and its Gram matrix / 6 (:240-242)
        wd = K.linear_rows(word.transpose(1, 2), self.projection.weight, self.projection.bias,
                           mode=mode)                                    # [B, T, 36]
        wd = K.gram(wd, 1.0 / np.sqrt(36), mode=mode)                    # [B, 36, 36]
        wd = wd.view(wd.size(0), wd.size(1), 6, 6)
        # bn_img / bn_word (:237, :243) folded into the attention's 1x1
        # projections (query role = key_proj(img), value = value_proj(img),
        # key role = query_proj(word), :248 -> :97-99)
        wx = torch.cat([sa._w(sa.key_proj), sa._w(sa.value_proj)], 0)
        bx = torch.cat([sa.key_proj.bias, sa.value_proj.bias])
        px = K.bn_linear(img, self.bn_img, wx, bx, mode=mode)                # [B, 36, Qr | V]
        py = K.bn_linear(wd, self.bn_word, sa._w(sa.query_proj), sa.query_proj.bias,
                         mode=mode)                                        # [B, 36, Kr]
        cq = sa.key_proj.weight.shape[0]
        iw = K.attention_core(px, py, cq, 0, cq, 1.0 / float(sa.sqrt_dim), mode)   # [B, HW, C]
        # LayerNorm [36, 6, 6] on the channels-last rows, maxpool, flatten (:249-253)
        iw = K.layer_norm_rows(iw, self.ln.weight, self.ln.bias, self.ln.eps, ch=iw.shape[2])
        iw = K.maxpool2_cl(iw, 6, 6).reshape(iw.size(0), -1)             # [B, 324]
        iw = K.linear_rows(iw, self.linear.weight, self.linear.bias, mode=mode)
        gl_img = K.layer_norm_rows(gl_img, self.ln_gl_image.weight, self.ln_gl_image.bias,
                                   self.ln_gl_image.eps)
        sent = K.layer_norm_rows(sent, self.ln_sent.weight, self.ln_sent.bias, self.ln_sent.eps)
        return torch.concat((iw, gl_img, sent), dim=1)


def set_precision(module, mode):
    """Set the MFMA precision mode ("fp32" split or "bf16") of every drop-in
    module under ``module``."""
    for m in module.modules():
        if hasattr(m, "precision"):
            m.precision = mode
    return module
