"""Activation recomputation from an input that is kept in 8 bits."""
import torch

from msamp.ops import cast as _c, native


def _outputs(out):
    return (out, ) if isinstance(out, torch.Tensor) else tuple(out)


def _tensors(args):
    """Every tensor in nested arguments."""
    if isinstance(args, torch.Tensor):
        return [args]
    if isinstance(args, dict):
        args = args.values()
    elif not isinstance(args, (tuple, list)):
        return []
    return [t for a in args for t in _tensors(a)]


def _versions(args):
    return [(t, t._version) for t in _tensors(args) if not t.is_inference()]


class _CheckpointFp8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, function, preserve_rng_state, args, x):
        ctx.function, ctx.args = function, args
        ctx.dtype, ctx.needs_x = x.dtype, x.requires_grad
        ctx.device = x.device
        ctx.autocast = (torch.is_autocast_enabled(x.device.type), torch.get_autocast_dtype(x.device.type), torch.is_autocast_cache_enabled())
        ctx.rng = None
        if preserve_rng_state:
            ctx.rng = (torch.get_rng_state(), torch.cuda.get_rng_state(x.device) if x.is_cuda else None)
        ctx.save_for_backward(*_c.cast_blocks_to_fp8(x))    # before the function, which may change x
        before = _versions(args)
        with torch.no_grad():
            out = function(x, *args)
        ctx.versions = _versions(args)    # after the function, which may change them (a cache, a counter)
        # Aliases of the outputs: the function may hand back a tensor that is the caller's (an argument, a buffer, a parameter), which
        # would otherwise become an output of this node itself.  x is an input of the node, autograd makes an alias of it.
        outs, plain = list(_outputs(out)), {id(a) for a, version in before if not a.requires_grad and a._version == version}
        constant = []
        for i, o in enumerate(outs):
            if isinstance(o, torch.Tensor) and o is not x:
                outs[i] = o.detach()
                if id(o) in plain:
                    constant.append(outs[i])
        ctx.mark_non_differentiable(*constant)
        return outs[0] if isinstance(out, torch.Tensor) else tuple(outs)

    @staticmethod
    def backward(ctx, *grads):
        if torch.is_grad_enabled():
            raise RuntimeError('checkpoint_fp8: no create_graph, as the gradients of the parameters get no graph')
        codes, exponents = ctx.saved_tensors
        if any(t._version != v for t, v in ctx.versions):
            raise RuntimeError('checkpoint_fp8: an argument was modified by an inplace operation before the backward pass ran the function again')
        x = _c.cast_blocks_from_fp8(codes, exponents, ctx.dtype).requires_grad_(ctx.needs_x)
        cuda = [ctx.device] if ctx.rng is not None and ctx.rng[1] is not None else []
        enabled, dtype, cache = ctx.autocast
        with torch.random.fork_rng(devices=cuda, enabled=ctx.rng is not None):
            if ctx.rng is not None:
                torch.set_rng_state(ctx.rng[0])
                if cuda:
                    torch.cuda.set_rng_state(ctx.rng[1], ctx.device)
            with torch.enable_grad(), torch.autocast(ctx.device.type, enabled=enabled, dtype=dtype, cache_enabled=cache):
                out = _outputs(ctx.function(x, *ctx.args))
        ctx.versions = _versions(ctx.args)
        pairs = [(o, g) for o, g in zip(out, grads) if g is not None and isinstance(o, torch.Tensor) and o.requires_grad]
        if pairs:
            torch.autograd.backward([o for o, _ in pairs], [g for _, g in pairs])
        return None, None, None, None, x.grad


def checkpoint_fp8(function, x, *args, preserve_rng_state=True):
    """``function(x, *args)`` whose activations are not kept: the backward pass runs it again, from an ``x`` kept in 8 bits.

    ``x`` (fp32, fp16 or bf16) is stored as e4m3 with a power-of-two scale per 32 elements (1.03 bytes each,
    :func:`msamp.ops.cast.cast_blocks_to_fp8`), so the outputs are those of ``function(x)`` and the gradients those at the stored
    value, which is within 2^-4 of every element (of the small ones of a block: within 2^-17 of its largest, or 2^-137 if that is more).
    Scaling metas of FP8 layers record the amaxes of the second run.  ``function`` returns a tensor or a tuple of tensors; what it returns of its ``args``, or of
    tensors that it holds, comes back as an alias.  Its outputs count as computed with gradients, except those of ``args`` that need none
    and are as they were: one that it detaches says that it requires a gradient and passes none on.  ``args`` are handed on as they
    are; a tensor among them that is computed from others with gradients is refused, as its gradient would not wait for its other uses.
    Parameters, also among ``args``, receive their gradients in ``.grad``: use ``backward()``, not ``torch.autograd.grad``, and not with
    ``create_graph``.  The random
    state of the first run is used again unless ``preserve_rng_state`` is false.
    """
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f'checkpoint_fp8: unsupported dtype {x.dtype}')
    if not torch.is_grad_enabled():
        return function(x, *args)
    if any(t.requires_grad and not t.is_leaf for t in _tensors(args)):
        raise ValueError('checkpoint_fp8: only x may be computed from other tensors with gradients; give it to the function first, or detach the argument')
    if any(native.carries_tangent(t) for t in _tensors(args)):
        raise ValueError('checkpoint_fp8: an argument has a forward-mode tangent, which the function would not pass on')
    # the anchor makes the outputs part of the graph where only parameters need gradients
    anchor = torch.empty(0, requires_grad=True)
    return _CheckpointFp8Fn.apply(anchor, function, preserve_rng_state, args, x)
