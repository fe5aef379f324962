"""Rotary positions: frequencies with their long-context scalings, and the rotation of query and key heads.

CUDA tensors use the kernel in ``csrc/rotary.cu``; CPU tensors use plain torch math with the same 64-bit angles (the oracle of
the GPU tests).
"""
import ctypes
import math

import torch

from msamp.ops import native

_i64x12 = ctypes.c_int64 * 12


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
    f = torch.tensor([base**(-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64)
    if scaling == 'linear':
        f = f / factor
    elif scaling == 'parts':
        if not trained or not fast > slow:
            raise ValueError('rotary_frequencies: parts needs the trained number of positions and fast > slow')
        turns = f * (trained / (2.0 * math.pi))
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f.to(device) if device is not None else f


def _check(x, name, freqs, positions):
    if x.dim() != 4:
        raise ValueError(f'rotary: {name} must be [batch, seq, heads, head_dim] (got {tuple(x.shape)})')
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'rotary: unsupported dtype {x.dtype}')
    if 2 * freqs.numel() > x.shape[3]:
        raise ValueError(f'rotary: {freqs.numel()} pairs do not fit a head of {x.shape[3]}')
    if freqs.device != x.device or (positions is not None and positions.device != x.device):
        raise ValueError(f'rotary: {name}, frequencies and positions must be on one device')


def _check_all(q, k, freqs, positions):
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or not 1 <= freqs.numel() <= 512:
        raise ValueError(f'rotary: frequencies are a float64 vector of 1 to 512 pairs (got {freqs.dtype}, {tuple(freqs.shape)})')
    _check(q, 'q', freqs, positions)
    if k is not None:
        _check(k, 'k', freqs, positions)
        if k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or k.dtype != q.dtype or k.device != q.device:
            raise ValueError(f'rotary: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in more than their heads')
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f'rotary: positions must be int32 or int64 (got {positions.dtype})')
        if tuple(positions.shape) not in ((q.shape[1], ), tuple(q.shape[:2])):
            raise ValueError(f'rotary: positions {tuple(positions.shape)} are neither [seq] nor [batch, seq] of {tuple(q.shape)}')


def rotary_raw(xs, ys, freqs, positions, interleaved, inverse):
    """Turns one or two ``[batch, seq, heads, head_dim]`` tensors ``xs`` into ``ys`` (which may be ``xs``: in place), without autograd.

    Inner strides are one; the others are free.  ``inverse`` turns back, which is also the gradient.
    """
    x = xs[0]
    batch, seq, _, dim = x.shape
    if not x.is_cuda:
        for src, dst in zip(xs, ys):
            dst.copy_(_emulated(src, freqs, positions, interleaved, inverse))
        return
    st, ptrs, heads = [], [], []
    for src, dst in zip(xs, ys):
        st += [*src.stride()[:3], *dst.stride()[:3]]
        ptrs += [src.data_ptr(), dst.data_ptr()]
        heads.append(src.shape[2])
    if len(heads) == 1:
        ptrs += [None, None]
        heads.append(0)
    freqs = freqs.contiguous()
    p_sb = p_ss = pos64 = 0
    if positions is not None:
        pos64 = int(positions.dtype == torch.int64)
        p_ss = positions.stride(-1)
        p_sb = positions.stride(0) if positions.dim() == 2 else 0
    with native.on_device(x):
        native.check(
            native.lib().msamp_rotary(
                *ptrs, _i64x12(*st), freqs.data_ptr(), native.addr(positions), pos64, p_sb, p_ss, batch, seq, *heads, dim, 2 * freqs.numel(),
                int(interleaved), int(inverse), native.dt(x.dtype), native.raw_stream()
            ), 'rotary'
        )


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


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, freqs, positions, interleaved):
        ctx.set_materialize_grads(False)
        xs = [_unit_inner(t) for t in ((q, ) if k is None else (q, k))]
        ys = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in xs]
        rotary_raw(xs, ys, freqs, positions, interleaved, False)
        ctx.save_for_backward(freqs, positions)
        ctx.interleaved = interleaved
        return tuple(ys)

    @staticmethod
    def backward(ctx, *grads):
        freqs, positions = ctx.saved_tensors
        xs = [_unit_inner(g) for g in grads if g is not None]
        ys = [torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in xs]
        if xs:
            rotary_raw(xs, ys, freqs, positions, ctx.interleaved, True)
        back = iter(ys)
        out = [None if g is None else next(back) for g in grads]
        return out[0], (out[1] if len(out) > 1 else None), None, None, None


def rotary(q, k, freqs, positions=None, interleaved=False):
    """Rotary positions on the heads of ``q [batch, seq, heads, head_dim]`` and ``k`` (any number of heads, or None).

    ``freqs`` (float64, :func:`rotary_frequencies`) holds one angle per position for each pair of the first ``2 * len(freqs)`` elements
    of a head; the elements behind them are passed on.  Pairs are elements ``i`` and ``i + len(freqs)``, or ``2 i`` and ``2 i + 1`` when
    ``interleaved``.  ``positions`` (``[seq]`` or ``[batch, seq]``, int32 or int64, any values) default to ``0 .. seq - 1``.  fp32, fp16 and
    bf16; inputs may be strided views.  Returns new contiguous tensors, ``(q', k')`` or ``q'`` alone when ``k`` is None.
    """
    _check_all(q, k, freqs, positions)
    out = _RotaryFn.apply(q, k, freqs, positions, bool(interleaved))
    return out if k is not None else out[0]
