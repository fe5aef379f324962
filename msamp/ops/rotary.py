"""Rotary positions: frequencies with their long-context scalings, and the rotation of query and key heads.

CUDA tensors use the kernel in ``csrc/rotary.cu``; CPU tensors use plain torch math with the same 64-bit angles (the oracle of
the GPU tests).
"""
import math
import struct

import torch

from msamp.ops import native


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, trained=None, fast=32.0, slow=1.0, device=None):
    """Angle per position of each of the ``dim / 2`` pairs, in radians, as a float64 vector: ``base ** (-2 i / dim)``.

    ``scaling`` stretches them by ``factor`` for contexts longer than the ``trained`` one:

    * ``'linear'``: every frequency is divided by ``factor``;
    * ``'base'``: ``base`` grows to ``base * factor ** (dim / (dim - 2))``, which divides the slowest frequency by ``factor`` and keeps
      the fastest;
    * ``'parts'``: pairs that turn at least ``fast`` times over the ``trained`` positions stay, pairs that turn at most ``slow`` times
      are divided by ``factor``, those between are mixed linearly in their number of turns.
    """
    if dim < 2 or dim % 2:
        raise ValueError(f'rotary_frequencies: dim must be even and positive (got {dim})')
    if not base > 0 or not factor > 0:
        raise ValueError(f'rotary_frequencies: base and factor must be positive (got {base}, {factor})')
    if scaling == 'base':
        if dim == 2:
            raise ValueError('rotary_frequencies: one pair has the frequency 1 at every base')
        base = base * factor**(dim / (dim - 2))
    elif scaling not in (None, 'linear', 'parts'):
        raise ValueError(f"rotary_frequencies: scaling is None, 'linear', 'base' or 'parts' (got {scaling!r})")
    f = torch.tensor([base**(-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device=device)
    if scaling == 'linear':
        f = f / factor
    elif scaling == 'parts':
        if not trained or not fast > slow:
            raise ValueError('rotary_frequencies: parts needs the trained number of positions and fast > slow')
        turns = f * (trained / (2.0 * math.pi))
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f


_TYPES = {torch.float32: native.DT_F32, torch.float16: native.DT_F16, torch.bfloat16: native.DT_BF16}


def _check_all(q, k, freqs, positions):
    if q.dim() != 4:
        raise ValueError(f'rotary: q must be [batch, seq, heads, head_dim] (got {tuple(q.shape)})')
    batch, seq, _, dim = q.shape
    if q.dtype not in _TYPES:
        raise TypeError(f'rotary: unsupported dtype {q.dtype}')
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not 1 <= freqs.numel() <= 512:
        raise ValueError(f'rotary: frequencies are a float64 vector of 1 to 512 pairs (got {freqs.dtype}, {tuple(freqs.shape)})')
    if 2 * freqs.numel() > dim:
        raise ValueError(f'rotary: {freqs.numel()} pairs do not fit a head of {dim}')
    if freqs.requires_grad:
        raise ValueError('rotary: the frequencies get no gradient')
    if freqs.device != q.device:
        raise ValueError('rotary: q and the frequencies must be on one device')
    if k is not None:
        if k.dim() != 4 or k.shape[:2] != (batch, seq) or k.shape[3] != dim or k.dtype != q.dtype or k.device != q.device:
            raise ValueError(f'rotary: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in more than their heads')
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f'rotary: positions must be int32 or int64 (got {positions.dtype})')
        if tuple(positions.shape) not in ((seq, ), (batch, seq)):
            raise ValueError(f'rotary: positions {tuple(positions.shape)} are neither [seq] nor [batch, seq] of {tuple(q.shape)}')
        if positions.device != q.device:
            raise ValueError('rotary: q and the positions must be on one device')


# The argument block of the native entry point: addresses and strides of the tensors, then what a call and its gradient share, then
# inverse and dtype.
_pack_tensors, _pack_common, _pack_end = struct.Struct('16q').pack, struct.Struct('12q').pack, struct.Struct('2q').pack


def _common(freqs, positions, batch, seq, heads0, heads1, dim, interleaved):
    """The fields that the rotation and its gradient share; ``freqs`` is contiguous."""
    part = 2 * freqs.numel()
    if positions is None:
        return _pack_common(freqs.data_ptr(), 0, 0, 0, 0, batch, seq, heads0, heads1, dim, part, interleaved)
    st = positions.stride()
    return _pack_common(freqs.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64, st[0] if len(st) == 2 else 0, st[-1], batch, seq,
                        heads0, heads1, dim, part, interleaved)


def _turn(x0, y0, x1, y1, common, inverse):
    """One launch on one or two tensors whose inner strides are one."""
    a, b = x0.stride(), y0.stride()
    if x1 is None:
        block = _pack_tensors(x0.data_ptr(), y0.data_ptr(), 0, 0, a[0], a[1], a[2], b[0], b[1], b[2], 0, 0, 0, 0, 0, 0)
    else:
        c, d = x1.stride(), y1.stride()
        block = _pack_tensors(x0.data_ptr(), y0.data_ptr(), x1.data_ptr(), y1.data_ptr(), a[0], a[1], a[2], b[0], b[1], b[2], c[0], c[1], c[2],
                              d[0], d[1], d[2])
    with native.on_device(x0):
        native.check(native.lib().msamp_rotary(block + common + _pack_end(inverse, _TYPES[x0.dtype]), native.raw_stream()), 'rotary')


def rotary_raw(xs, ys, freqs, positions, interleaved, inverse):
    """Turns one or two ``[batch, seq, heads, head_dim]`` tensors ``xs`` into ``ys`` (which may be ``xs``: in place), without autograd.

    Inner strides are one; the others are free.  ``inverse`` turns back, which is also the gradient.
    """
    x = xs[0]
    _check_all(x, xs[1] if len(xs) > 1 else None, freqs, positions)
    if len(ys) != len(xs) or len(xs) > 2:
        raise ValueError(f'rotary: one or two tensors and as many results (got {len(xs)} and {len(ys)})')
    for src, dst in zip(xs, ys):
        if dst is not src and (dst.shape != src.shape or dst.dtype != src.dtype or dst.device != src.device):
            raise ValueError(f'rotary: {tuple(src.shape)} {src.dtype} does not go into {tuple(dst.shape)} {dst.dtype}')
        if (src.stride(3) != 1 or dst.stride(3) != 1) and src.shape[3] != 1 and src.numel():
            raise ValueError('rotary: the elements of a head must be adjacent')
    if not x.is_cuda:
        for src, dst in zip(xs, ys):
            dst.copy_(_emulated(src, freqs, positions, interleaved, inverse))
        return
    freqs = freqs.contiguous()
    two = len(xs) > 1
    common = _common(freqs, positions, x.shape[0], x.shape[1], x.shape[2], xs[1].shape[2] if two else 0, x.shape[3], interleaved)
    _turn(x, ys[0], xs[1] if two else None, ys[1] if two else None, common, inverse)


def _emulated(x, freqs, positions, interleaved, inverse):
    part = 2 * freqs.numel()
    pos = torch.arange(x.shape[1], device=x.device) if positions is None else positions
    angle = pos.double()[..., None] * freqs    # [seq, pairs] or [batch, seq, pairs]
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    if inverse:
        sin = -sin
    y = x.float().clone()
    first, second = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    a, b = x[..., first].float(), x[..., second].float()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    return y.to(x.dtype)


def _unit_inner(t):
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _forward(q, k, freqs, positions, interleaved, inverse):
    """``(q', k' or None, fields)``; the last are what the gradient needs again on CUDA."""
    if not q.is_cuda:
        return (_emulated(q, freqs, positions, interleaved, inverse).contiguous(),
                None if k is None else _emulated(k, freqs, positions, interleaved, inverse).contiguous(), None)
    q = _unit_inner(q)
    batch, seq, heads, dim = q.shape
    if k is None:
        common = _common(freqs, positions, batch, seq, heads, 0, dim, interleaved)
        y = _like(q)
        _turn(q, y, None, None, common, inverse)
        return y, None, common
    k = _unit_inner(k)
    common = _common(freqs, positions, batch, seq, heads, k.shape[2], dim, interleaved)
    yq, yk = _like(q), _like(k)
    _turn(q, yq, k, yk, common, inverse)
    return yq, yk, common


def _layout(freqs, positions):
    """What the fields of a call take from these two: saved tensors may come back with other strides, at the same address too."""
    if positions is None:
        return freqs.data_ptr(), freqs.stride()
    return freqs.data_ptr(), freqs.stride(), positions.data_ptr(), positions.stride(), positions.dtype


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, freqs, positions, interleaved, inverse):
        ctx.set_materialize_grads(False)
        yq, yk, ctx.common = _forward(q, k, freqs, positions, interleaved, inverse)
        ctx.save_for_backward(freqs, positions)
        ctx.interleaved, ctx.back, ctx.layout = interleaved, not inverse, _layout(freqs, positions)
        return yq if k is None else (yq, yk)

    @staticmethod
    def backward(ctx, gq, gk=None):
        freqs, positions = ctx.saved_tensors
        if torch.is_grad_enabled() and (gq is not None or gk is not None):    # create_graph: the gradient is a rotation and has one too
            given = [g for g in (gq, gk) if g is not None]
            out = _RotaryFn.apply(given[0], given[1] if len(given) == 2 else None, freqs, positions, ctx.interleaved, ctx.back)
            back = iter(out if len(given) == 2 else (out, ))
            return (None if gq is None else next(back)), (None if gk is None else next(back)), None, None, None, None
        both = gq is not None and gk is not None and gq.is_cuda and gq.is_contiguous() and gk.is_contiguous()
        if both and _layout(freqs, positions) == ctx.layout:
            # as a rule: both gradients, in the layout of the outputs, with the fields of the forward call
            dq, dk = torch.empty_like(gq), torch.empty_like(gk)
            _turn(gq, dq, gk, dk, ctx.common, ctx.back)
            return dq, dk, None, None, None, None
        given = [_unit_inner(g) for g in (gq, gk) if g is not None]
        out = [_like(g) for g in given]
        if given:
            rotary_raw(given, out, freqs, positions, ctx.interleaved, ctx.back)
        back = iter(out)
        return (None if gq is None else next(back)), (None if gk is None else next(back)), None, None, None, None


def rotary(q, k, freqs, positions=None, interleaved=False):
    """Rotary positions on the heads of ``q [batch, seq, heads, head_dim]`` and ``k`` (any number of heads, or None).

    ``freqs`` (float64, :func:`rotary_frequencies`) holds one angle per position for each pair of the first ``2 * len(freqs)`` elements
    of a head; the elements behind them are passed on.  Pairs are elements ``i`` and ``i + len(freqs)``, or ``2 i`` and ``2 i + 1`` when
    ``interleaved``.  ``positions`` (``[seq]`` or ``[batch, seq]``, int32 or int64, any values) default to ``0 .. seq - 1``.  fp32, fp16 and
    bf16; inputs may be strided views.  Returns new contiguous tensors, ``(q', k')`` or ``q'`` alone when ``k`` is None.
    """
    _check_all(q, k, freqs, positions)
    freqs = freqs.contiguous()
    if native.needs_function(q, k) if q.is_cuda else torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _RotaryFn.apply(q, k, freqs, positions, bool(interleaved), False)
    yq, yk, _ = _forward(q, k, freqs, positions, bool(interleaved), False)
    return yq if k is None else (yq, yk)
