"""Transformer-block operators (LayerNorm, GeLU, attention, cross-entropy) as autograd functions.

CUDA tensors use the kernels in ``csrc/nn.cu`` and ``csrc/attention.cu``; CPU tensors use plain
torch math (the oracle the GPU tests compare against).
"""
import ctypes
import math
import os
import struct

import torch
import torch.nn.functional as F

from msamp.ops import cast as _c, native
from msamp.ops.autograd import once
from msamp.ops.rotary import rotary, rotary_frequencies, rotary_raw    # noqa: F401

_i64x24 = ctypes.c_int64 * 24


def _use_native(t):
    return t.is_cuda


# ---------------------------------------------------------------------------------------- LayerNorm
class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        shape = x.shape
        x2 = x.reshape(-1, shape[-1]).contiguous()
        rows, cols = x2.shape
        y = torch.empty_like(x2)
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        native.check(
            native.lib().msamp_layernorm_fwd(
                native.ptr(x2), native.ptr(weight), native.ptr(bias), native.dt(x2.dtype), native.dt(weight.dtype), native.ptr(y),
                native.ptr(mean), native.ptr(rstd), rows, cols, ctypes.c_float(eps), native.stream()
            ), 'layernorm_fwd'
        )
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.has_bias = bias is not None
        ctx.shape = shape
        return y.view(shape)

    @staticmethod
    def backward(ctx, dy):
        x2, weight, mean, rstd = ctx.saved_tensors
        rows, cols = x2.shape
        dy2 = dy.reshape(rows, cols).contiguous()
        dx = torch.empty_like(x2)
        dgamma = torch.empty_like(weight)
        dbeta = torch.empty_like(weight) if ctx.has_bias else None
        nparts = native.lib().msamp_layernorm_bwd_parts()
        part = torch.empty(nparts * 2 * cols, dtype=torch.float32, device=x2.device)
        native.check(
            native.lib().msamp_layernorm_bwd(
                native.ptr(dy2), native.ptr(x2), native.ptr(weight), native.dt(x2.dtype), native.dt(weight.dtype), native.ptr(mean),
                native.ptr(rstd), native.ptr(dx), native.ptr(dgamma), native.ptr(dbeta), native.ptr(part), rows, cols, native.stream()
            ), 'layernorm_bwd'
        )
        return dx.view(ctx.shape), dgamma, dbeta, None


def _ln_supported(x, weight, bias):
    cols = x.shape[-1]
    vec = 4 if x.dtype == torch.float32 else 8
    return (cols % vec == 0 and cols <= native.lib().msamp_layernorm_max_cols(native.dt(x.dtype))
            and weight.dtype in (torch.float32, torch.float16, torch.bfloat16) and (bias is None or bias.dtype == weight.dtype))


def layer_norm_fwd_raw(x2, weight, bias, eps, want_y=True, y8_scale=None, amax_in=None, amax_out=None, scale_inv_out=None, want_y8=False):
    """LayerNorm forward without autograd on a contiguous 2-D ``x2``.

    Returns ``(y or None, y8 or None, mean, rstd)``.  ``y8`` is the e4m3 copy of the output quantised with
    ``y8_scale`` (a 0-d fp32 tensor); with ``amax_in`` the scale is first derived from that amax by the power-of-two
    rule and written back to ``y8_scale``.  ``amax_out`` receives ``max|y|`` and ``scale_inv_out`` ``1 / scale``.
    The quantised values are taken from the output as rounded to the dtype of ``x2``, so they equal a separate cast
    of ``y`` bit for bit.  With ``want_y=False`` and ``want_y8=False`` only the statistics and ``amax_out`` are produced.
    """
    rows, cols = x2.shape
    if x2.is_cuda:
        if not _ln_supported(x2, weight, bias):
            raise RuntimeError(f'layer_norm: unsupported shape/dtype on CUDA (cols={cols}, dtype={x2.dtype}, param={weight.dtype})')
        y = torch.empty_like(x2) if want_y else None
        y8 = torch.empty((rows, cols), dtype=torch.uint8, device=x2.device) if want_y8 else None
        mean = torch.empty(rows, dtype=torch.float32, device=x2.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x2.device)
        native.check(
            native.lib().msamp_layernorm_fwd_q(
                x2.data_ptr(), weight.data_ptr(), native.addr(bias), native.dt(x2.dtype), native.dt(weight.dtype), native.addr(y),
                mean.data_ptr(), rstd.data_ptr(), rows, cols, eps, native.addr(y8), native.addr(y8_scale), native.addr(amax_in),
                native.addr(amax_out), native.addr(scale_inv_out), native.raw_stream()
            ), 'layernorm_fwd'
        )
        return y, y8, mean, rstd
    from msamp.common.dtype import Dtypes
    xf = x2.float()
    mean = xf.mean(1)
    var = xf.var(1, unbiased=False)
    rstd = torch.rsqrt(var + eps)
    yf = (xf - mean[:, None]) * rstd[:, None] * weight.float()
    if bias is not None:
        yf = yf + bias.float()
    y = yf.to(x2.dtype)
    y8 = None
    if amax_out is not None:
        _c.amax(y, out=amax_out)
    if want_y8:
        y8 = _c.cast_to_fp8(y, Dtypes.kfloat8_e4m3, y8_scale, scale_inv_out=scale_inv_out, amax_in=amax_in)
    return (y if want_y else None), y8, mean, rstd


def layer_norm_bwd_raw(dy2, x2, weight, mean, rstd, has_bias, dres=None, amax_out=None):
    """LayerNorm backward without autograd: returns ``(dx, dgamma, dbeta or None)``.

    ``dres`` (same shape and dtype as ``x2``) is added to ``dx`` in the same pass - the gradient that reaches the
    input through the skip connection around the normalised branch; ``amax_out`` receives ``max|dx|``.
    """
    rows, cols = x2.shape
    if x2.is_cuda:
        dx = torch.empty_like(x2)
        dgamma = torch.empty_like(weight)
        dbeta = torch.empty_like(weight) if has_bias else None
        nparts = native.lib().msamp_layernorm_bwd_parts()
        part = torch.empty(nparts * 2 * cols, dtype=torch.float32, device=x2.device)
        native.check(
            native.lib().msamp_layernorm_bwd_ex(
                native.ptr(dy2), native.ptr(x2), native.ptr(weight), native.dt(x2.dtype), native.dt(weight.dtype), native.ptr(mean),
                native.ptr(rstd), native.ptr(dx), native.ptr(dgamma), native.ptr(dbeta), native.ptr(part), rows, cols, native.ptr(dres),
                native.ptr(amax_out), native.stream()
            ), 'layernorm_bwd'
        )
        return dx, dgamma, dbeta
    xh = (x2.float() - mean[:, None]) * rstd[:, None]
    d = dy2.float()
    gd = d * weight.float()
    m1 = gd.mean(1, keepdim=True)
    m2 = (gd * xh).mean(1, keepdim=True)
    dxf = rstd[:, None] * (gd - m1 - xh * m2)
    if dres is not None:
        dxf = dxf + dres.float()
    dx = dxf.to(x2.dtype)
    if amax_out is not None:
        _c.amax(dx, out=amax_out)
    dgamma = (d * xh).sum(0).to(weight.dtype)
    dbeta = d.sum(0).to(weight.dtype) if has_bias else None
    return dx, dgamma, dbeta


def layer_norm(x, weight, bias=None, eps=1e-5):
    """LayerNorm over the last dimension."""
    if _use_native(x):
        cols = x.shape[-1]
        vec = 4 if x.dtype == torch.float32 else 8
        if cols % vec == 0 and cols <= native.lib().msamp_layernorm_max_cols(native.dt(x.dtype)) and weight.dtype in (
            torch.float32, torch.float16, torch.bfloat16
        ) and (bias is None or bias.dtype == weight.dtype):
            return _LayerNormFn.apply(x, weight, bias, eps)
        raise RuntimeError(f'layer_norm: unsupported shape/dtype on CUDA (cols={cols}, dtype={x.dtype}, param={weight.dtype})')
    return F.layer_norm(x.float(), (x.shape[-1], ), weight.float(), None if bias is None else bias.float(), eps).to(x.dtype)


# ---------------------------------------------------------------------------------------- GeLU
class _GeluFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x = x.contiguous()
        y = torch.empty_like(x)
        native.check(native.lib().msamp_gelu_fwd(native.ptr(x), native.ptr(y), native.i64(x.numel()), native.dt(x.dtype), native.stream()), 'gelu_fwd')
        ctx.save_for_backward(x)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, = ctx.saved_tensors
        dy = dy.contiguous()
        dx = torch.empty_like(x)
        native.check(
            native.lib().msamp_gelu_bwd(native.ptr(x), native.ptr(dy), native.ptr(dx), native.i64(x.numel()), native.dt(x.dtype), native.stream()),
            'gelu_bwd'
        )
        return dx


class _GeluKeepFn(torch.autograd.Function):
    """GeLU whose input is kept as e4m3 blocks: written by the forward kernel next to the output, read by the backward kernel."""
    @staticmethod
    def forward(ctx, x):
        if x.is_cuda:
            kept, y = _c._gelu_keep(x.contiguous())
            ctx.save_for_backward(kept)
            return y
        ctx.save_for_backward(*_c.cast_blocks_to_fp8(x))
        return F.gelu(x.float(), approximate='tanh').to(x.dtype)

    @staticmethod
    @once
    def backward(ctx, dy):
        kept, *rest = ctx.saved_tensors
        if rest:
            return gelu_bwd_blocks(kept, rest[0], dy)
        at = kept.data_ptr()
        return _c._gelu_keep_bwd(at, at + dy.numel(), dy.contiguous())


def gelu_bwd_blocks(codes, exponents, dy):
    """``dy * gelu'(x)`` for the ``x`` that the e4m3 blocks stand for (see ``cast.cast_blocks_to_fp8``), in the type of ``dy``."""
    _c._check_blocks(codes, exponents)
    if codes.shape != dy.shape or codes.device != dy.device:
        raise ValueError(f'gelu: codes {tuple(codes.shape)} and gradient {tuple(dy.shape)} differ')
    if dy.is_cuda:
        codes, exponents = codes.contiguous(), exponents.contiguous()
        return _c._gelu_keep_bwd(codes.data_ptr(), exponents.data_ptr(), dy.contiguous())
    with torch.enable_grad():
        x = _c.cast_blocks_from_fp8(codes, exponents, torch.float32).requires_grad_(True)
        grad, = torch.autograd.grad(F.gelu(x, approximate='tanh'), x, dy.float())
    return grad.to(dy.dtype)


def gelu(x, keep_fp8=False):
    """GeLU, tanh form.

    ``keep_fp8`` keeps the input of the backward pass as e4m3 with a power-of-two scale per 32 elements (1.03 bytes each, see
    ``cast.cast_blocks_to_fp8``) instead of ``x`` itself: the output is the same, the gradient is the slope at the kept value.
    """
    if keep_fp8:
        if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise TypeError(f'gelu: unsupported dtype {x.dtype}')
        if (torch.is_grad_enabled() and x.requires_grad) or (x.is_cuda and x.data_ptr() % 16):
            return _GeluKeepFn.apply(x)
    if _use_native(x):
        return _GeluFn.apply(x)
    return F.gelu(x.float(), approximate='tanh').to(x.dtype)


# ---------------------------------------------------------------------------------------- attention
def _attn_entry(which):
    """Native entry point: the tcgen05 kernels (``MSAMP_ATTN_IMPL=mma`` selects the mma.sync kernels, to which this entry also
    sends views with a zero stride and short rows)."""
    tc = os.environ.get('MSAMP_ATTN_IMPL', 'tc') != 'mma'
    return getattr(native.lib(), f'msamp_attention_{"tc_" if tc else ""}{which}')


def _strides(t):
    # t is a [B, S, nh, d] view; kernel wants element strides (batch, seq, head)
    assert t.stride(3) == 1
    return [t.stride(0), t.stride(1), t.stride(2)]


def _rows16(t):
    """``t`` if its rows can be read 16 bytes at a time (unit inner stride, other strides and start in whole 16 bytes), else a
    contiguous copy: an incoming gradient may be a view with any strides that starts anywhere in its buffer."""
    s = t.stride()
    if s[3] != 1 or s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


class _AttentionFn(torch.autograd.Function):
    """Inputs are [B, S, nh, d] bf16 views (arbitrary batch/seq/head strides); output is contiguous [B, S, nh, d]."""
    @staticmethod
    def forward(ctx, q, k, v, causal, scale, grad_layout):
        B, S, nh, d = q.shape
        o = torch.empty((B, S, nh, d), dtype=q.dtype, device=q.device)
        lse = torch.empty((B, nh, S), dtype=torch.float32, device=q.device)
        st = _strides(q) + _strides(k) + _strides(v) + _strides(o) + [0] * 12
        native.check(
            _attn_entry('fwd')(
                native.ptr(q), native.ptr(k), native.ptr(v), native.ptr(o), native.ptr(lse), _i64x24(*st), B, nh, S, d,
                ctypes.c_float(scale), int(causal), native.stream()
            ), 'attention_fwd'
        )
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal, ctx.scale, ctx.grad_layout = causal, scale, grad_layout
        return o

    @staticmethod
    def backward(ctx, d_o):
        q, k, v, o, lse = ctx.saved_tensors
        B, S, nh, d = q.shape
        o, d_o = _rows16(o), _rows16(d_o)
        if ctx.grad_layout == 'packed':
            # one [B, S, 3, nh, d] buffer so that the gradient of a fused QKV projection needs no concatenation
            dqkv = torch.empty((B, S, 3, nh, d), dtype=q.dtype, device=q.device)
            dq, dk, dv = dqkv[:, :, 0], dqkv[:, :, 1], dqkv[:, :, 2]
        else:
            dq, dk, dv = torch.empty_like(o), torch.empty_like(o), torch.empty_like(o)
        delta = torch.empty((B, nh, S), dtype=torch.float32, device=q.device)
        st = _strides(q) + _strides(k) + _strides(v) + _strides(o) + _strides(d_o) + _strides(dq) + _strides(dk) + _strides(dv)
        native.check(
            _attn_entry('bwd')(
                native.ptr(q), native.ptr(k), native.ptr(v), native.ptr(o), native.ptr(lse), native.ptr(d_o), native.ptr(dq),
                native.ptr(dk), native.ptr(dv), native.ptr(delta), _i64x24(*st), B, nh, S, d, ctypes.c_float(ctx.scale), int(ctx.causal),
                native.stream()
            ), 'attention_bwd'
        )
        return dq, dk, dv, None, None, None


def _packed_strides(B, S, nh, d):
    """(batch, seq, head) strides of q, k and v inside a contiguous ``[B, S, 3, nh, d]`` tensor, then of a contiguous output."""
    return [3 * S * nh * d, 3 * nh * d, d] * 3 + [S * nh * d, nh * d, d]


def _packed_fwd(qkv, causal, scale):
    """Attention on a contiguous packed tensor (the callers have checked that): q, k and v are addresses inside it."""
    B, S, _, nh, d = qkv.shape
    o = torch.empty((B, S, nh, d), dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty((B, nh, S), dtype=torch.float32, device=qkv.device)
    q, sub = qkv.data_ptr(), nh * d * qkv.element_size()
    native.check(
        _attn_entry('fwd')(
            q, q + sub, q + 2 * sub, o.data_ptr(), lse.data_ptr(), _i64x24(*_packed_strides(B, S, nh, d)), B, nh, S, d, scale, int(causal),
            native.raw_stream()
        ), 'attention_fwd'
    )
    return o, lse


def _packed_bwd(qkv, o, lse, d_o, causal, scale):
    B, S, _, nh, d = qkv.shape
    if not qkv.is_contiguous() or qkv.data_ptr() % 16:    # a saved tensor may come back with other strides (saved-tensor hooks)
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    o, d_o = _rows16(o), _rows16(d_o)
    dqkv = torch.empty_like(qkv)
    delta = torch.empty((B, nh, S), dtype=torch.float32, device=qkv.device)
    packed = _packed_strides(B, S, nh, d)[:9]
    q, dq, sub = qkv.data_ptr(), dqkv.data_ptr(), nh * d * qkv.element_size()
    native.check(
        _attn_entry('bwd')(
            q, q + sub, q + 2 * sub, o.data_ptr(), lse.data_ptr(), d_o.data_ptr(), dq, dq + sub, dq + 2 * sub, delta.data_ptr(),
            _i64x24(*packed, *_strides(o), *_strides(d_o), *packed), B, nh, S, d, scale, int(causal), native.raw_stream()
        ), 'attention_bwd'
    )
    return dqkv


class _AttentionPackedFn(torch.autograd.Function):
    """Attention on a fused ``[B, S, 3, heads, d]`` QKV tensor; the gradient comes back in the same packed layout.

    Taking the packed tensor as the one autograd input (instead of three ``select`` views of it) keeps
    autograd from materialising three zero-filled full-size gradients and adding them up.
    """
    @staticmethod
    def forward(ctx, qkv, causal, scale):
        o, lse = _packed_fwd(qkv, causal, scale)
        ctx.save_for_backward(qkv, o, lse)
        ctx.causal, ctx.scale = causal, scale
        return o

    @staticmethod
    def backward(ctx, d_o):
        qkv, o, lse = ctx.saved_tensors
        return _packed_bwd(qkv, o, lse, d_o, ctx.causal, ctx.scale), None, None


def attention_qkv_fwd_raw(qkv, causal=True, scale=None):
    """Self-attention forward without autograd on a packed ``[B, S, 3, heads, d]`` tensor: returns ``(o [B,S,heads,d], lse or None)``."""
    B, S, _, nh, d = qkv.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if _use_native(qkv):
        if qkv.dtype != torch.bfloat16 or d not in (64, 128) or not qkv.is_contiguous() or qkv.data_ptr() % 16:
            raise RuntimeError(f'attention_qkv: CUDA kernel needs contiguous bf16 with head_dim 64/128 (got {qkv.dtype}, {d})')
        return _packed_fwd(qkv, causal, scale)
    with torch.no_grad():
        return attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], causal=causal, scale=scale), None


def attention_qkv_bwd_raw(qkv, o, lse, d_o, causal=True, scale=None):
    """Gradient of :func:`attention_qkv_fwd_raw` with respect to the packed ``qkv`` (same layout)."""
    B, S, _, nh, d = qkv.shape
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if _use_native(qkv):
        return _packed_bwd(qkv, o, lse, d_o, causal, scale)
    with torch.enable_grad():
        leaf = qkv.detach().clone().requires_grad_(True)
        out = attention(leaf[:, :, 0], leaf[:, :, 1], leaf[:, :, 2], causal=causal, scale=scale)
        grad, = torch.autograd.grad(out, leaf, d_o)
    return grad


def attention_qkv(qkv, causal=True, scale=None):
    """Self-attention on a fused ``[B, S, 3, heads, head_dim]`` projection output; returns ``[B, S, heads, head_dim]``."""
    d = qkv.shape[-1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if _use_native(qkv):
        if qkv.dtype != torch.bfloat16 or d not in (64, 128) or not qkv.is_contiguous() or qkv.data_ptr() % 16:
            raise RuntimeError(f'attention_qkv: CUDA kernel needs contiguous bf16 with head_dim 64/128 (got {qkv.dtype}, {d})')
        return _AttentionPackedFn.apply(qkv, causal, scale)
    return attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], causal=causal, scale=scale)


# Attention whose query heads share key / value heads, on rows that may end early.  ``q [B, S, heads, d]``, ``k`` and ``v [B, S, kv_heads, d]``
# as strided views, ``lengths`` ``[B]`` (int32 or int64) or None.  The argument blocks of the native entry points: addresses, sizes and scale, strides.
_pack_fwd, _pack_bwd = struct.Struct('7q').pack, struct.Struct('13q').pack
_pack_sizes, _pack_st = struct.Struct('6qd').pack, [struct.Struct(f'{3 * n}q').pack for n in range(9)]


def _map_strides(t):
    """(batch, seq, head) element strides for a tensor map; the stride of an axis of extent 1 is never used and may be any number."""
    a, b, c, _ = t.stride()
    if (a | b | c) & 7 == 0:
        return a, b, c
    return tuple(s if n > 1 else t.shape[3] for s, n in zip((a, b, c), t.shape))


def _dense_strides(S, n, d):
    """The same of a contiguous ``[B, S, n, d]`` tensor."""
    return S * n * d, n * d, d


def _mappable(t):
    """``t``, or a copy of it where it repeats a batch, position or head (a tensor map has no zero stride)."""
    a, b, c, _ = t.stride()
    if a and b and c:
        return t
    return t.contiguous() if any(s == 0 and n > 1 for s, n in zip((a, b, c), t.shape)) else t


class _SharedCall:
    """What calls of the same sizes and strides share: their checks, and the fields of both argument blocks that are no addresses."""
    __slots__ = ('fields', 'tail', 'strides', 'partial', 'work', 'lse_shape', 'plan_size', 'split', 'args')

    def __init__(self, q, k, v, causal, scale, packed, lengths):
        B, S, nh, d = q.shape
        nkv = k.shape[2]
        if q.dtype != torch.bfloat16 or d not in (64, 128):
            raise RuntimeError(f'attention: CUDA kernel supports bf16 with head_dim 64/128 (got {q.dtype}, {d})')
        for t in (q, k, v):
            if t.stride(3) != 1 or any(s & 7 for s in _map_strides(t)):
                raise RuntimeError('attention: operands must have unit inner stride and 16-byte aligned rows')
        ragged = lengths is not None
        flags = int(causal) | (2 if lengths == torch.int64 else 0)
        self.args = (flags, scale)
        dense = _dense_strides(S, nh, d)
        self.fields = _pack_sizes(B, nh, nkv, S, d, flags, scale) + _pack_st[4](*_map_strides(q), *_map_strides(k), *_map_strides(v), *dense)
        # dO as a rule in the layout of o, then dq, dk and dv
        grads = _dense_strides(S, nh + 2 * nkv, d) * 3 if packed else dense + _dense_strides(S, nkv, d) * 2
        self.tail = _pack_st[4](*dense, *grads)
        self.strides = (q.stride(), k.stride(), v.stride(), torch.empty((B, S, nh, d), device='meta').stride())
        with native.on_device(q):
            # floats of the backward pass's workspace: partial sums of dK and dV where there may be several, rowsum(dO * O) behind them
            self.partial = native.lib().msamp_attention_shared_partial(B, nh, nkv, S, d, causal, ragged)
        self.work = self.partial + B * nh * S
        self.lse_shape = (B, nh, S)
        # with lengths: the tiles that are not padding, listed by the forward pass for both passes, and the lengths within 0 .. S
        self.plan_size = 2 + (B + 1) * ((S + 127) // 128) + B if ragged else 0
        self.split = ((B, S, nh + 2 * nkv, d), [nh, nkv, nkv]) if packed else None


_shared_calls = {}


def _shared_call(q, k, v, causal, scale, packed, lengths):
    """Checks and shared fields of a call, remembered by its sizes and strides."""
    kind = None if lengths is None else lengths.dtype
    key = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), causal, scale, packed, kind, q.device)
    call = _shared_calls.get(key)
    if call is None or q.dtype != torch.bfloat16:
        _check_shared(q, k, v, scale, lengths)
        if len(_shared_calls) > 1024:
            _shared_calls.clear()
        call = _shared_calls[key] = _SharedCall(q, k, v, causal, scale, packed, kind)
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.device != q.device or v.device != q.device:
        _check_shared(q, k, v, scale, lengths)
    if (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        raise RuntimeError('attention: operands must have unit inner stride and 16-byte aligned rows')
    if lengths is not None:
        _check_lengths(q, lengths)
    return call


def _shared_fwd(q, k, v, call, lengths):
    """``(o, lse, plan)``; ``lse`` is ``[B, heads, S]``."""
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty(call.lse_shape, dtype=torch.float32)
    plan = q.new_empty(call.plan_size, dtype=torch.int32) if call.plan_size else None
    with native.on_device(q):
        native.check(
            native.lib().msamp_attention_shared_fwd(
                _pack_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                          0 if plan is None else plan.data_ptr()) + call.fields, native.raw_stream()
            ), 'attention_fwd'
        )
    return o, lse, plan


def _shared_bwd(q, k, v, o, lse, d_o, dq, dk, dv, plan, fields, call, tail):
    """Gradients into ``dq``, ``dk`` and ``dv``; ``tail``: packed strides of ``d_o`` and of theirs."""
    lse = lse.contiguous()
    plan = None if plan is None else plan.contiguous()
    plan_at = 0 if plan is None else plan.data_ptr()    # holds the lengths too
    # of this call alone: saved tensors may serve several backward passes, captured ones too
    space = q.new_empty(call.work, dtype=torch.float32)
    at = space.data_ptr()
    with native.on_device(q):
        native.check(
            native.lib().msamp_attention_shared_bwd(
                _pack_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), lse.data_ptr(), plan_at, plan_at, d_o.data_ptr(),
                          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), at + 4 * call.partial, at if call.partial else 0) + fields + tail, native.raw_stream()
            ), 'attention_bwd'
        )


class _AttentionSharedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, call):
        o, lse, plan = _shared_fwd(q, k, v, call, lengths)
        # int32 lengths are saved for the check that nothing has overwritten them; the backward pass has those of the plan
        ctx.save_for_backward(q, k, v, o, lse, plan, lengths if lengths is not None and lengths.dtype == torch.int32 else None)
        ctx.call = call
        return o

    @staticmethod
    @once
    def backward(ctx, d_o):
        q, k, v, o, lse, plan, _ = ctx.saved_tensors
        call = ctx.call
        fields, tail = call.fields, call.tail
        if (q.stride(), k.stride(), v.stride(), o.stride()) != call.strides or (q.data_ptr() | k.data_ptr() | v.data_ptr() | o.data_ptr()) & 15:
            # saved tensors may come back with other strides (saved-tensor hooks)
            q, k, v, o = (_rows16(_mappable(t)) for t in (q, k, v, o))
            B, S, nh, d = q.shape
            fields = _pack_sizes(B, nh, k.shape[2], S, d, *call.args) + _pack_st[4](*(s for t in (q, k, v, o) for s in _map_strides(t)))
        if not d_o.is_contiguous() or d_o.data_ptr() & 15:
            d_o = _rows16(_mappable(d_o))
            tail = _pack_st[1](*_map_strides(d_o)) + tail[24:]
        if call.split is None:
            dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
        else:
            dq, dk, dv = q.new_empty(call.split[0]).split(call.split[1], dim=2)
        _shared_bwd(q, k, v, o, lse, d_o, dq, dk, dv, plan, fields, call, tail)
        return dq, dk, dv, None, None


def _attention_plain(q, k, v, causal, scale, lengths):
    """The same in torch operations on any device (the CPU form)."""
    B, S, nh, d = q.shape
    if lengths is not None:
        valid = torch.arange(S, device=q.device) < lengths.to(q.device)[:, None]
        q, k, v = (torch.where(valid[:, :, None, None], t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (q, k, v))
    qf, kf, vf = (t.float().permute(0, 2, 1, 3) for t in (q, k, v))
    # a single head is broadcast, as is everything to a single query head
    kf, vf = (t if t.shape[1] in (1, nh) or nh == 1 else t.repeat_interleave(nh // t.shape[1], dim=1) for t in (kf, vf))
    s = (qf @ kf.transpose(-1, -2)) * scale
    if causal:
        s = s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=q.device).triu(1), float('-inf'))
    if lengths is not None:
        s = s.masked_fill(~valid[:, None, None, :], float('-inf'))
        seen = valid[:, None, :, None]
        s = torch.where(seen, s, torch.zeros((), device=q.device))    # padding sees nothing: cleared below
        p = torch.where(seen, torch.softmax(s, dim=-1), torch.zeros((), device=q.device))
    else:
        p = torch.softmax(s, dim=-1)
    out = (p @ vf).permute(0, 2, 1, 3).to(q.dtype)
    if lengths is not None:    # keeps what the gradient holds at padding out of the products of the backward pass
        out = torch.where(valid[:, :, None, None], out, torch.zeros((), dtype=out.dtype, device=out.device))
    return out.contiguous()


def _check_lengths(q, lengths):
    if lengths.shape != q.shape[:1] or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f'attention: lengths must be an int32 or int64 tensor [{q.shape[0]}] (got {lengths.dtype} {tuple(lengths.shape)})')
    if lengths.device != q.device:
        raise ValueError('attention: lengths must be on the device of q')


def _check_shared(q, k, v, scale, lengths):
    shape, kv = q.shape, k.shape
    if len(shape) != 4 or len(kv) != 4 or v.shape != kv or kv[:2] != shape[:2] or kv[3] != shape[3]:
        raise ValueError(f'attention: q {tuple(shape)}, k {tuple(kv)} and v {tuple(v.shape)} do not fit together')
    if kv[2] == 0 or shape[2] % kv[2]:
        raise ValueError(f'attention: {shape[2]} query heads do not share {kv[2]} key/value heads evenly')
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise ValueError('attention: q, k and v must have one dtype and one device')
    if not 0.0 < scale < 3e38:
        raise ValueError(f'attention: scale must be positive (got {scale})')
    if lengths is not None:
        _check_lengths(q, lengths)


def _shared_operands(q, k, v, causal, scale, packed, lengths):
    """Mappable views, dense lengths, and the shared fields of the call."""
    if len(q.shape) == len(k.shape) == len(v.shape) == 4:
        q, k, v = _mappable(q), _mappable(k), _mappable(v)
    call = _shared_call(q, k, v, bool(causal), float(scale), packed, lengths)
    if lengths is not None:
        lengths = lengths.contiguous()
    return q, k, v, lengths, call


def attention_shared_fwd_raw(q, k, v, causal=True, scale=None, lengths=None):
    """Forward pass of :func:`attention` with shared key/value heads or row lengths, without autograd: ``(o, lse, plan)`` for its gradients."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if _use_native(q) and q.numel():
        q, k, v, lengths, call = _shared_operands(q, k, v, causal, scale, False, lengths)
        return _shared_fwd(q, k, v, call, lengths)
    _check_shared(q, k, v, scale, lengths)
    with torch.no_grad():
        return _attention_plain(q, k, v, causal, scale, lengths), None, None


def attention_shared_bwd_raw(q, k, v, o, lse, plan, d_o, dq, dk, dv, causal=True, scale=None, lengths=None):
    """Its gradients, written into ``dq``, ``dk`` and ``dv`` (views with unit inner stride and 16-byte aligned rows)."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    if _use_native(q) and q.numel():
        q, k, v, lengths, call = _shared_operands(q, k, v, causal, scale, False, lengths)
        for t, like in ((o, q), (d_o, q), (dq, q), (dk, k), (dv, v)):
            if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
                raise ValueError(f'attention: {tuple(t.shape)} {t.dtype} in the place of {tuple(like.shape)} {like.dtype}')
            if t.stride(3) != 1 and t is not o and t is not d_o:
                raise ValueError('attention: gradients must have unit inner stride')
        B, S, nh, d = q.shape
        if lse.shape != (B, nh, S) or lse.dtype != torch.float32 or lse.device != q.device:
            raise ValueError(f'attention: log-sum-exps {tuple(lse.shape)} {lse.dtype} of another forward pass')
        if (plan is not None) != bool(call.plan_size) or (plan is not None and (plan.numel() != call.plan_size or plan.dtype != torch.int32 or
                                                                                plan.device != q.device)):
            raise ValueError('attention: plan of another forward pass')
        o, d_o = _rows16(_mappable(o)), _rows16(_mappable(d_o))
        fields = _pack_sizes(B, nh, k.shape[2], S, d, *call.args) + _pack_st[4](*(x for t in (q, k, v, o) for x in _map_strides(t)))
        _shared_bwd(q, k, v, o, lse, d_o, dq, dk, dv, plan, fields, call,
                    _pack_st[4](*(x for t in (d_o, dq, dk, dv) for x in _map_strides(t))))
        return
    with torch.enable_grad():
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        grads = torch.autograd.grad(_attention_plain(*leaves, causal, scale, lengths), leaves, d_o)
    for dst, g in zip((dq, dk, dv), grads):
        dst.copy_(g)


def _attention_shared(q, k, v, causal, scale, grad_layout, lengths):
    if not q.is_cuda or q.numel() == 0:
        _check_shared(q, k, v, scale, lengths)
        return _attention_plain(q, k, v, causal, scale, lengths)
    q, k, v, lengths, call = _shared_operands(q, k, v, causal, scale, grad_layout == 'packed', lengths)
    if native.needs_function(q, k, v):
        return _AttentionSharedFn.apply(q, k, v, lengths, call)
    return _shared_fwd(q, k, v, call, lengths)[0]


def attention(q, k, v, causal=True, scale=None, grad_layout='separate', lengths=None):
    """Softmax attention on ``[B, S, heads, head_dim]`` tensors; returns ``[B, S, heads, head_dim]``.

    ``k`` and ``v`` may have fewer heads than ``q``: each of theirs then serves ``heads / kv_heads`` consecutive query heads, and its
    gradient is the sum over those.  ``lengths`` (``[B]``, int32 or int64, on the device of ``q``) makes positions at or behind a row's
    length padding: they are neither seen nor see, their outputs and gradients are zero, and whatever they hold stays out of every other
    row; lengths outside ``0 .. S`` count as 0 or S.

    ``grad_layout='packed'`` makes backward return dq/dk/dv as views of one ``[B,S,3,heads,d]`` buffer (``[B,S,heads + 2 kv_heads,d]`` with
    shared heads or lengths; use it when q, k, v are themselves views of a fused QKV tensor of that layout).
    """
    d = q.shape[-1]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    shared = q.dim() == k.dim() == 4 and k.shape[2] != q.shape[2]
    # CPU form: other batches or numbers of keys, and heads that broadcast, are whatever its products allow
    if lengths is not None or (shared and (q.is_cuda or (k.shape[:2] == q.shape[:2] and 1 not in (q.shape[2], k.shape[2])))):
        return _attention_shared(q, k, v, causal, scale, grad_layout, lengths)
    if _use_native(q):
        if q.dtype != torch.bfloat16 or d not in (64, 128):
            raise RuntimeError(f'attention: CUDA kernel supports bf16 with head_dim 64/128 (got {q.dtype}, {d})')
        for t in (k, v):
            if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
                raise ValueError(f'attention: q {tuple(q.shape)} {q.dtype} and {tuple(t.shape)} {t.dtype} do not fit together')
        for t in (q, k, v):
            if t.stride(3) != 1 or any(s % 8 for s in t.stride()[:3]) or t.data_ptr() % 16:
                raise RuntimeError('attention: operands must have unit inner stride and 16-byte aligned rows')
        return _AttentionFn.apply(q, k, v, causal, scale, grad_layout)
    return _attention_plain(q, k, v, causal, scale, None)


# ---------------------------------------------------------------------------------------- cross entropy
class _XentFn(torch.autograd.Function):
    """Mean token cross-entropy; backward overwrites the logits buffer with its gradient."""
    @staticmethod
    def forward(ctx, logits, target, ignore_index):
        rows, vocab = logits.shape
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        lse = torch.empty(rows, dtype=torch.float32, device=logits.device)
        native.check(
            native.lib().msamp_xent_fwd(
                native.ptr(logits), native.ptr(target), native.ptr(loss), native.ptr(lse), rows, vocab, native.i64(logits.stride(0)),
                native.i64(ignore_index), native.dt(logits.dtype), native.stream()
            ), 'xent_fwd'
        )
        count = (target != ignore_index).sum().clamp(min=1).float()
        ctx.save_for_backward(logits, target, lse, count)
        ctx.ignore_index = ignore_index
        return loss.sum() / count

    @staticmethod
    def backward(ctx, dloss):
        logits, target, lse, count = ctx.saved_tensors
        rows, vocab = logits.shape
        gscale = (dloss.float() / count).reshape(1).contiguous()
        native.check(
            native.lib().msamp_xent_bwd(
                native.ptr(logits), native.ptr(target), native.ptr(lse), native.ptr(gscale), rows, vocab, native.i64(logits.stride(0)),
                native.i64(ctx.ignore_index), native.dt(logits.dtype), native.stream()
            ), 'xent_bwd'
        )
        return logits, None, None


def cross_entropy(logits, target, ignore_index=-100):
    """Mean cross-entropy of ``logits [rows, vocab]`` against ``target [rows]`` (int64).

    On CUDA the backward pass reuses the logits buffer for the gradient, so ``logits`` must not be
    read again after ``backward``.
    """
    if _use_native(logits):
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        return _XentFn.apply(logits, target.contiguous(), ignore_index)
    return F.cross_entropy(logits.float(), target, ignore_index=ignore_index)
