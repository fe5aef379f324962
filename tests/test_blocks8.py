"""Activations in 8 bits: the codes against their definition, the GeLU that reads them, recomputation from them.

The codes are exact (equal bytes); the GeLU gradient is half a step of its type from the slope at the kept value, up to the error of the
exponential and the division in 32 bits (a few ulp of numbers that are at most 1, times |dy| (1 + |v|): 2^-18 covers them).
"""
import math

import pytest
import torch

import msamp
from msamp.nn import checkpoint_fp8
from msamp.ops import cast, native
from msamp.ops import nn as K

CPU_GPU = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _values(n, dtype, seed):
    """Magnitudes over the whole range of the type, zeros, whole blocks of zeros, powers of two and numbers just beside 1.75 * 2^k."""
    gen = torch.Generator().manual_seed(seed)
    info = torch.finfo(dtype)
    lo, hi = math.log2(info.smallest_normal) - 3, math.log2(info.max)
    x = torch.randn(n, generator=gen, dtype=torch.float64)
    block = torch.arange(n) // 32
    x = x * torch.exp2(lo + (hi - lo - 3) * torch.rand(int(n // 32) + 1, generator=gen, dtype=torch.float64))[block]
    x[block % 7 == 3] = 0.0
    x[torch.rand(n, generator=gen) < 0.05] = 0.0
    edge = block % 5 == 2
    x[edge] = (1.75 * torch.exp2(torch.randint(-6, 6, (n, ), generator=gen).double()) * (1 + info.eps * torch.randint(-1, 2, (n, ), generator=gen)))[edge]
    return x.clamp(-info.max, info.max).to(dtype)


def _definition(x):
    """(codes' values, k) by the definition, in 64 bits."""
    flat = x.detach().double().cpu().reshape(-1)
    n = flat.numel()
    rows = torch.cat([flat, flat.new_zeros(-n % 32)]).view(-1, 32)
    finite = torch.isfinite(rows)
    top = torch.where(finite, rows.abs(), 0.0).amax(1)
    k = torch.zeros_like(top)
    for j in range(-127, 128):    # the largest shift that keeps the block within 448
        k = torch.where((top > 0) & (top * 2.0**j <= 448.0), torch.full_like(top, j), k)
    y = torch.where(finite, rows * torch.exp2(k)[:, None], float('nan'))
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)    # e4m3: 3 bits of fraction, no finer than 2^-9
    return (torch.round(y / step) * step).view(-1)[:n], k


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n', [1, 31, 32, 33, 100, 1024, 4097, 40000])
def test_codes(device, dtype, n):
    x = _values(n, dtype, n).to(device)
    codes, exps = cast.cast_blocks_to_fp8(x)
    want, k = _definition(x)
    assert codes.shape == x.shape and codes.dtype == torch.uint8 and exps.numel() == (n + 31) // 32
    assert torch.equal(127 - exps.cpu().double(), k)
    assert torch.equal(codes.cpu().view(torch.float8_e4m3fn).double(), want)
    back = cast.cast_blocks_from_fp8(codes, exps, dtype)
    top = torch.finfo(dtype).max
    exact = (want * torch.exp2(-k).repeat_interleave(32)[:n]).clamp(-top, top)
    assert torch.equal(back.cpu(), exact.to(dtype)) and torch.isfinite(back).all()
    for out in TYPES:
        other = cast.cast_blocks_from_fp8(codes, exps, out).cpu()
        lim = torch.finfo(out).max
        assert torch.equal(other, exact_to(want, k, n, lim).to(out))


def exact_to(want, k, n, lim):
    return (want * torch.exp2(-k).repeat_interleave(32)[:n]).clamp(-lim, lim)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', TYPES)
def test_distance(device, dtype):
    """The largest of a block is over 224 in steps of its unit 2^-k.  e4m3 rounds numbers from 2^-6 on by at most 2^-4 of themselves, so
    values above 2^-6 / 224 < 2^-13 of the largest; below, by half of 2^-9, which is under 2^-10 / 224 < 2^-17 of the largest."""
    x = torch.randn(64, 256, generator=torch.Generator().manual_seed(0)).mul_(0.02)
    x = (x * torch.exp2(-20 * torch.rand(64, 256, generator=torch.Generator().manual_seed(1)))).to(dtype).to(device)
    v = cast.cast_blocks_from_fp8(*cast.cast_blocks_to_fp8(x), torch.float32).double()
    top = x.double().abs().view(-1, 32).amax(1).repeat_interleave(32).view_as(x)
    err = (v - x.double()).abs()
    small = x.double().abs() < top * 2.0**-13
    assert small.any() and (err[~small] <= x.double().abs()[~small] * 2.0**-4).all() and (err[small] <= top[small] * 2.0**-17).all()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('offset', [0, 1])
def test_not_finite(device, dtype, offset):
    x = _values(200 + offset, dtype, 5)[offset:]
    plain = cast.cast_blocks_to_fp8(x.to(device))
    bad = x.clone()
    bad[3], bad[40], bad[41], bad[199] = float('inf'), float('nan'), -float('inf'), float('inf')
    at = torch.zeros(200, dtype=torch.bool)
    at[[3, 40, 41, 199]] = True
    codes, exps = cast.cast_blocks_to_fp8(bad.to(device))
    want, k = _definition(bad)
    assert torch.equal(127 - exps.cpu().double(), k)
    back = cast.cast_blocks_from_fp8(codes, exps, dtype).cpu()
    assert torch.equal(torch.isnan(back), at) and torch.isfinite(back[~at]).all()
    assert torch.equal(codes.cpu().view(torch.float8_e4m3fn).double()[~at], want[~at])
    untouched = torch.arange(200) // 32
    keep = (untouched != 0) & (untouched != 1) & (untouched != 6)
    assert torch.equal(codes.cpu()[keep], plain[0].cpu()[keep])


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', TYPES)
def test_gpu_equals_cpu_for_views(dtype):
    base = _values(3 * 70 * 50 + 1, dtype, 9)
    for view in (lambda t: t[1:], lambda t: t[:-1].view(3, 70, 50).transpose(0, 2), lambda t: t[:-1].view(3, 70, 50)[:, ::2]):
        a, b = cast.cast_blocks_to_fp8(view(base)), cast.cast_blocks_to_fp8(view(base.cuda()))
        assert torch.equal(a[0], b[0].cpu()) and torch.equal(a[1], b[1].cpu())
        for out in TYPES:
            assert torch.equal(cast.cast_blocks_from_fp8(*a, out), cast.cast_blocks_from_fp8(*b, out).cpu())
    odd = torch.empty(base.numel() + 1, dtype=torch.uint8, device='cuda')[1:]    # codes off the 16-byte grid
    c, e = cast.cast_blocks_to_fp8(base.cuda())
    odd.copy_(c)
    assert torch.equal(cast.cast_blocks_from_fp8(odd, e, dtype), cast.cast_blocks_from_fp8(c, e, dtype))


@pytest.mark.parametrize('device', CPU_GPU)
def test_empty(device):
    x = torch.empty(0, 7, device=device)
    codes, exps = cast.cast_blocks_to_fp8(x)
    assert codes.shape == (0, 7) and exps.numel() == 0 and cast.cast_blocks_from_fp8(codes, exps, torch.bfloat16).shape == (0, 7)
    y = K.gelu(x.requires_grad_(True), keep_fp8=True)
    y.sum().backward()
    assert x.grad.shape == (0, 7)


def _slope(v):
    c0, c1 = math.sqrt(2.0 / math.pi), 0.044715
    t = torch.tanh(c0 * (v + c1 * v**3))
    return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c0 * (1 + 3 * c1 * v * v)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('shape, offset', [((1, ), 0), ((33, ), 0), ((7, 100), 0), ((7, 100), 1), ((64, 512), 0), ((3, 5, 1000), 0)])
def test_gelu(device, dtype, shape, offset):
    n = math.prod(shape)
    gen = torch.Generator().manual_seed(n)
    x = (torch.randn(n + offset, generator=gen) * 3).to(dtype).to(device)[offset:].view(shape).requires_grad_(True)
    dy = torch.randn(n + offset, generator=gen).to(dtype).to(device)[offset:].view(shape)
    y = K.gelu(x, keep_fp8=True)
    if offset == 0 or device == 'cpu':
        assert torch.equal(y, K.gelu(x.detach()))    # the output does not know
    dx, = torch.autograd.grad(y, x, dy)
    v = cast.cast_blocks_from_fp8(*cast.cast_blocks_to_fp8(x.detach()), torch.float32).double()
    want = dy.double() * _slope(v)
    err = (dx.double() - want).abs()
    tiny = torch.finfo(dtype).smallest_normal
    assert (err <= want.abs() * torch.finfo(dtype).eps / 2 + dy.double().abs() * (1 + v.abs()) * 2.0**-18 + tiny).all()
    # against differences of the function itself, at the kept values
    h = 1e-4
    c0, c1 = math.sqrt(2.0 / math.pi), 0.044715
    f = lambda t: 0.5 * t * (1 + torch.tanh(c0 * (t + c1 * t**3)))    # noqa: E731
    diff = dy.double() * (f(v + h) - f(v - h)) / (2 * h)
    assert ((want - diff).abs() <= 1e-6 * (1 + dy.double().abs())).all()


@pytest.mark.gpu
def test_gelu_views_and_gradient_layouts():
    x = torch.randn(40, 64, device='cuda').bfloat16().requires_grad_(True)
    y = K.gelu(x, keep_fp8=True)
    dy = torch.randn(64, 40, device='cuda').bfloat16().t()
    a, = torch.autograd.grad(y, x, dy, retain_graph=True)
    b, = torch.autograd.grad(y, x, dy.contiguous(), retain_graph=True)
    c, = torch.autograd.grad(y.sum(), x)    # an expanded gradient
    d, = torch.autograd.grad(K.gelu(x, keep_fp8=True), x, torch.ones_like(y))
    assert torch.equal(a, b) and torch.equal(c, d)
    t = torch.randn(64, 40, device='cuda').bfloat16()
    u, v = t.t().detach().requires_grad_(True), t.t().contiguous().requires_grad_(True)
    (gu, ), (gv, ) = torch.autograd.grad(K.gelu(u, keep_fp8=True), u, dy[:40, :64]), torch.autograd.grad(K.gelu(v, keep_fp8=True), v, dy[:40, :64])
    assert torch.equal(gu, gv)


@pytest.mark.parametrize('device', CPU_GPU)
def test_gelu_without_gradients_keeps_nothing(device):
    x = torch.randn(65, 31, device=device).to(torch.bfloat16 if device == 'cuda' else torch.float32).requires_grad_(True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        K.gelu(x.detach(), keep_fp8=True)
        with torch.no_grad():
            y = K.gelu(x, keep_fp8=True)
    assert not seen and torch.equal(y, K.gelu(x.detach()))
    z = K.gelu(x.detach().flatten()[1:], keep_fp8=True)    # off the 16-byte grid
    assert torch.equal(z, K.gelu(x.detach().flatten()[1:].clone()))


def test_refusals():
    c, e = cast.cast_blocks_to_fp8(torch.randn(70))
    for bad in (lambda: cast.cast_blocks_to_fp8(torch.zeros(3, dtype=torch.float64)), lambda: cast.cast_blocks_to_fp8(torch.zeros(3, dtype=torch.int32)),
                lambda: cast.cast_blocks_from_fp8(c, e, torch.float64), lambda: cast.cast_blocks_from_fp8(c.float(), e, torch.float32),
                lambda: K.gelu(torch.zeros(3, dtype=torch.float64), keep_fp8=True), lambda: checkpoint_fp8(torch.sin, torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: cast.cast_blocks_from_fp8(c, e[:-1], torch.float32), lambda: K.gelu_bwd_blocks(c, e, torch.randn(2, 35))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.skipif(not native.available(), reason='kernel library not built')
def test_entry_points_refuse():
    """No launch: every call is refused by its arguments."""
    lib, at = native.lib(), 1 << 20
    assert lib.msamp_blocks_cast(None, None, at, at, 8, 0, None) == 1 and lib.msamp_blocks_cast(at, None, None, at, 8, 0, None) == 1
    assert lib.msamp_blocks_cast(at, None, at, None, 8, 0, None) == 1 and lib.msamp_blocks_cast(at, None, at, at, 8, 7, None) == 2
    assert lib.msamp_blocks_uncast(None, at, None, at, 8, 0, None) == 1 and lib.msamp_blocks_uncast(at, at, None, None, 8, 0, None) == 1
    assert lib.msamp_blocks_cast(None, None, None, None, 0, 0, None) == 0 and lib.msamp_blocks_uncast(None, None, None, None, 0, 0, None) == 0


# ------------------------------------------------------------------------------------------------------------- GEMM epilogues
@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('mnk, tile', [((1, 32, 16), 0), ((300, 160, 96), 2), ((300, 160, 96), 1), ((513, 544, 256), 1), ((257, 256, 128), 2),
                                       ((2048, 1024, 512), 0)])
def test_gemm_epilogues(device, dtype, mnk, tile):
    """The blocks that a GEMM writes are those of its output, and the GeLU slope it takes from blocks is that of their values: equal bits."""
    from msamp.common.dtype import Dtypes
    from msamp.ops import gemm
    m, n, k = mnk
    if device == 'cpu' and m * n > 400000:
        pytest.skip('the same code as at the other sizes')
    gen = torch.Generator().manual_seed(m)
    e4 = Dtypes.kfloat8_e4m3
    a, b = ((torch.randn(r, k, generator=gen) * 2).to(torch.float8_e4m3fn).view(torch.uint8).to(device) for r in (m, n))
    one = torch.tensor(0.5, device=device)
    bias = torch.randn(n, generator=gen).to(device)
    kept = (torch.empty(m, n, dtype=torch.uint8, device=device), torch.empty(m * n // 32, dtype=torch.uint8, device=device))
    want = gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, bias=bias, tile=tile)
    amax = torch.zeros((), device=device)
    got = gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, bias=bias, tile=tile, keep_blocks=kept, amax_out=amax, act='gelu')
    codes, exps = cast.cast_blocks_to_fp8(want)
    assert torch.equal(got, want) and torch.equal(kept[0], codes) and torch.equal(kept[1], exps)
    again = tuple(torch.zeros_like(t) for t in kept)
    assert gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, bias=bias, tile=tile, keep_blocks=again, store_out=False) is None
    assert torch.equal(again[0], codes) and torch.equal(again[1], exps)
    h = _values(m * n, dtype, n).clamp(-1e3, 1e3).view(m, n).to(device)
    blocks = cast.cast_blocks_to_fp8(h)
    h = cast.cast_blocks_from_fp8(*blocks, dtype)
    x = gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, tile=tile, gelu_src=h)
    y = gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, tile=tile, gelu_blocks=blocks)
    assert torch.equal(x, y)
    out8, sums, scale = torch.empty(m, n, dtype=torch.uint8, device=device), torch.empty(n, device=device), torch.tensor(2.0, device=device)
    gemm.gemm_fp8(a, e4, one, b, e4, one, dtype, tile=tile, gelu_blocks=blocks, out8=out8, out8_qtype=e4, out8_scale=scale, colsum_out=sums, store_out=False)
    assert torch.equal(out8, cast.cast_to_fp8(x, e4, scale))
    assert (sums - x.float().sum(0)).abs().max() <= 1e-4 * (1 + x.float().abs().sum(0).max())    # another order of 32-bit sums
    if device == 'cuda':
        torch.cuda.synchronize()
        assert native.device_status() == 0


def test_gemm_epilogues_of_not_finite_values():
    """What does not fit the output type becomes infinite there and NaN in the blocks."""
    from msamp.common.dtype import Dtypes
    from msamp.ops import gemm
    for device in ['cpu'] + (['cuda'] if torch.cuda.is_available() else []):
        a = torch.ones(3, 16, device=device).to(torch.float8_e4m3fn).view(torch.uint8)
        b = torch.ones(64, 16, device=device).to(torch.float8_e4m3fn).view(torch.uint8)
        bias = torch.zeros(64, device=device)
        bias[5], bias[40], bias[41] = 1e6, float('nan'), -1e6
        one = torch.tensor(1.0, device=device)
        kept = (torch.empty(3, 64, dtype=torch.uint8, device=device), torch.empty(6, dtype=torch.uint8, device=device))
        d = gemm.gemm_fp8(a, Dtypes.kfloat8_e4m3, one, b, Dtypes.kfloat8_e4m3, one, torch.float16, bias=bias, keep_blocks=kept)
        codes, exps = cast.cast_blocks_to_fp8(d)
        assert torch.equal(kept[0], codes) and torch.equal(kept[1], exps)
        v = cast.cast_blocks_from_fp8(*kept, torch.float16)
        assert torch.equal(torch.isnan(v), ~torch.isfinite(d)) and (v[:, :5] == 16).all()


def test_gemm_blocks_refused():
    from msamp.common.dtype import Dtypes
    from msamp.ops import gemm
    e4, one = Dtypes.kfloat8_e4m3, torch.tensor(1.0)
    a, b = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(48, 16, dtype=torch.uint8)
    u8 = lambda n: torch.zeros(n, dtype=torch.uint8)    # noqa: E731
    with pytest.raises(ValueError):
        gemm.gemm_fp8(a, e4, one, b, e4, one, torch.float32, keep_blocks=(u8(192), u8(6)))
    b = torch.zeros(64, 16, dtype=torch.uint8)
    with pytest.raises(ValueError):
        gemm.gemm_fp8(a, e4, one, b, e4, one, torch.float32, gelu_blocks=(u8(256), u8(8)), gelu_src=torch.zeros(4, 64))
    with pytest.raises(AssertionError):
        gemm.gemm_fp8(a, e4, one, b, e4, one, torch.float32, keep_blocks=(u8(256), u8(7)))


# ------------------------------------------------------------------------------------------------------------- recomputation
@pytest.mark.parametrize('device', CPU_GPU)
def test_checkpoint_gradients_are_those_at_the_kept_input(device):
    torch.manual_seed(0)
    lin = torch.nn.Linear(48, 40, device=device)
    x = torch.randn(6, 48, device=device, requires_grad=True)
    f = lambda t, s: torch.tanh(lin(t)) * s    # noqa: E731
    y = checkpoint_fp8(f, x, 2.0)
    assert torch.equal(y, f(x, 2.0))
    dy = torch.randn_like(y)
    y.backward(dy)
    v = cast.cast_blocks_from_fp8(*cast.cast_blocks_to_fp8(x.detach()), x.dtype).requires_grad_(True)
    wv, wb, wx = torch.autograd.grad(f(v, 2.0), (lin.weight, lin.bias, v), dy)
    assert torch.equal(x.grad, wx) and torch.equal(lin.weight.grad, wv) and torch.equal(lin.bias.grad, wb)


def test_checkpoint_dropout_tuple_and_frozen_input():
    torch.manual_seed(0)
    lin = torch.nn.Linear(32, 32)
    x = torch.ones(4, 32)    # exact in 8 bits, needs no gradient

    def f(t):
        z = torch.nn.functional.dropout(lin(t), 0.5)
        return z, z.sum(), torch.arange(3)

    z, total, count = checkpoint_fp8(f, x)
    state = torch.get_rng_state()
    (z.sum() + total).backward()
    assert torch.equal(state, torch.get_rng_state()) and torch.equal(count, torch.arange(3))
    kept = (z != 0).float()
    assert torch.allclose(lin.weight.grad, 2 * (kept * 2.0).t() @ x) and x.grad is None
    with torch.no_grad():
        assert not checkpoint_fp8(f, x)[0].requires_grad


def test_checkpoint_of_a_function_that_changes_its_input_and_returns_none():
    x = torch.ones(4, 32, requires_grad=True)
    lin = torch.nn.Linear(32, 32, bias=False)
    y, nothing = checkpoint_fp8(lambda t: (lin(t.mul_(2.0) if not t.requires_grad else t * 2.0), None), x * 1.0)
    y.sum().backward()
    assert nothing is None
    assert torch.equal(lin.weight.grad, torch.full((32, 32), 8.0)) and torch.allclose(x.grad, 2 * lin.weight.sum(0).expand(4, 32))


def test_checkpoint_arguments():
    torch.manual_seed(12)
    x, w, side = torch.randn(4, 32, requires_grad=True), torch.randn(32, requires_grad=True), torch.randn(4, 32)

    def f(x, parts):
        w, (side, ) = parts['w'], parts['side']
        return (x * w + side).sin()

    def run(**kw):
        return checkpoint_fp8(f, x, {**dict(w=w, side=(side, )), **kw})

    with pytest.raises(ValueError):
        run(w=w * 2)
    out = run()
    side.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    out = run()
    out.sum().backward(retain_graph=True)
    once = w.grad.clone(), x.grad.clone()
    out.sum().backward()
    assert torch.equal(w.grad, 2 * once[0]) and torch.equal(x.grad, 2 * once[1])
    kept = cast.cast_blocks_from_fp8(*cast.cast_blocks_to_fp8(x.detach()), torch.float32).requires_grad_(True)
    w.grad = None
    f(kept, dict(w=w, side=(side, ))).sum().backward()
    assert torch.equal(w.grad, once[0]) and torch.equal(kept.grad, once[1])


def test_checkpoint_keeps_one_byte_per_element():
    seen = []
    lin = torch.nn.Linear(64, 64)
    x = torch.randn(32, 64, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        checkpoint_fp8(lambda t: torch.tanh(lin(t)), x)
    assert sum(t.numel() * t.element_size() for t in seen) == 32 * 64 + 64


def test_public_names():
    assert msamp.nn.checkpoint_fp8 is checkpoint_fp8 and 'checkpoint_fp8' in msamp.nn.__all__


@pytest.mark.parametrize('device', CPU_GPU)
def test_checkpoint_leaves_what_the_function_hands_back_alone(device):
    """A function may return an argument, a buffer or a parameter: the caller's tensors keep their place in autograd."""
    x = torch.ones(2, 32, device=device, requires_grad=True)
    argument, buffer, nested = (torch.zeros(3, device=device) for _ in range(3))
    count = torch.zeros(2, dtype=torch.int64, device=device)
    weight = torch.nn.Parameter(torch.full((32, ), 3.0, device=device))
    handed = torch.nn.Parameter(torch.full((4, ), 2.0, device=device))

    def f(t, a, parts, w):
        count.add_(1)
        y = t * weight
        return y, a, buffer, weight, w, parts['n'], count, y, t

    out = checkpoint_fp8(f, x, argument, dict(n=nested), handed)
    for t in (argument, buffer, nested, count):
        assert not t.requires_grad and t.grad_fn is None and t.is_leaf
    for t in (weight, handed):
        assert t.requires_grad and t.grad_fn is None and t.is_leaf
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(out[1:7], (argument, buffer, weight, handed, nested, count)))
    # arguments that need no gradient come back as such, as does what is no floating-point number
    assert not out[1].requires_grad and not out[5].requires_grad and not out[6].requires_grad
    (out[0].sum() + 2 * out[7].sum() + 5 * out[8].sum() + 7 * out[3].sum() + 11 * out[4].sum()).backward()
    assert torch.equal(x.grad, torch.full((2, 32), 3.0 * 3 + 5, device=device))
    assert torch.equal(weight.grad, torch.full((32, ), 3.0 * 2 + 7, device=device)) and torch.equal(handed.grad, torch.full((4, ), 11.0, device=device))


def test_checkpoint_of_one_returned_argument():
    x, cache = torch.ones(2, 32, requires_grad=True), torch.zeros(4)
    out = checkpoint_fp8(lambda t, c: c, x, cache)
    assert out.data_ptr() == cache.data_ptr() and not out.requires_grad and not cache.requires_grad and cache.grad_fn is None


def test_checkpoint_of_a_returned_argument_that_the_function_fills():
    x, cache = torch.ones(2, 32, requires_grad=True), torch.zeros(2, 32)
    out = checkpoint_fp8(lambda t, c: c.copy_(t * 3), x, cache)
    assert out.requires_grad and not cache.requires_grad and torch.equal(cache, torch.full((2, 32), 3.0))
    out.sum().backward()
    assert torch.equal(x.grad, torch.full((2, 32), 3.0))


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('offset', [0, 1])
def test_gelu_does_not_drop_a_forward_mode_tangent(monkeypatch, device, offset):
    monkeypatch.setenv('PYTORCH_JIT', '0')    # make_dual compiles torch's own rules otherwise, which fails on functions that msamp wraps
    from torch.autograd import forward_ad as fwd
    x = torch.randn(1025, device=device)[offset:offset + 1024]
    with fwd.dual_level():
        x = fwd.make_dual(x, torch.ones_like(x))
        if device == 'cuda':
            with pytest.raises((NotImplementedError, RuntimeError), match='forward'):
                K.gelu(x, keep_fp8=True)
        else:
            assert fwd.unpack_dual(K.gelu(x, keep_fp8=True)).tangent is not None


def test_checkpoint_refuses_forward_mode_tangents(monkeypatch):
    """The function runs without gradients inside of the node, where a tangent would be lost."""
    monkeypatch.setenv('PYTORCH_JIT', '0')    # make_dual compiles torch's own rules otherwise, which fails on functions that msamp wraps
    from torch.autograd import forward_ad as fwd
    x, side = torch.ones(2, 32), torch.ones(2, 32)
    with fwd.dual_level():
        dual = fwd.make_dual(torch.ones(2, 32), torch.ones(2, 32))
        with pytest.raises((NotImplementedError, RuntimeError), match='forward'):
            checkpoint_fp8(lambda t, s: t * s, dual, side)
        with pytest.raises(ValueError, match='forward'):
            checkpoint_fp8(lambda t, s: t * s['side'], x, dict(side=dual))
        with torch.no_grad():
            assert fwd.unpack_dual(checkpoint_fp8(lambda t, s: t * s, x, dual)).tangent is not None


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('power', [1, 2])
def test_gelu_refuses_second_derivatives(device, power):
    """Its slope at the kept value has no gradient; a constant incoming gradient (power 1) does not hide that."""
    x = torch.randn(64, device=device, requires_grad=True)
    y = K.gelu(x, keep_fp8=True)
    plain, = torch.autograd.grad((y**power).sum(), x, retain_graph=True)
    first, = torch.autograd.grad((y**power).sum(), x, create_graph=True)
    assert torch.equal(plain, first)
    with pytest.raises(RuntimeError, match='twice'):
        (first.pow(2).sum() + x.sum()).backward()


def test_checkpoint_refuses_create_graph():
    """The gradients of the parameters go to .grad without a graph, so there is nothing to differentiate again."""
    x, w = torch.ones(2, 32, requires_grad=True), torch.ones(32, requires_grad=True)
    out = checkpoint_fp8(lambda t: (t * w)**2, x)
    with pytest.raises(RuntimeError, match='create_graph'):
        out.sum().backward(create_graph=True)
    assert w.grad is None and x.grad is None
    out.sum().backward()
    assert torch.equal(w.grad, torch.full((32, ), 4.0)) and torch.equal(x.grad, torch.full((2, 32), 2.0))


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_distance_of_the_smallest_blocks(device, dtype):
    """The shift ends at 127: below 2^-119 the largest of a block no longer comes near 448.  The steps of e4m3's numbers below 2^-6 are 2^-9, here
    2^-136, so a value is off by at most 2^-4 of itself or by 2^-137 (which may be all of it), whichever is more."""
    gen = torch.Generator().manual_seed(2)
    top = torch.exp2(-119.0 - 29.0 * torch.rand(256, 1, generator=gen, dtype=torch.float64))    # down to the last subnormal number
    x = (top * torch.exp2(-14 * torch.rand(256, 32, generator=gen, dtype=torch.float64)) * torch.randn(256, 32, generator=gen).sign()).to(dtype).to(device)
    codes, exps = cast.cast_blocks_to_fp8(x)
    largest = x.double().abs().amax(1)
    assert (exps[(largest < 2.0**-119) & (largest > 0)] == 0).all()    # k = 127 (blocks of zeros, which bf16 has here too: k = 0)
    v = cast.cast_blocks_from_fp8(codes, exps, torch.float32).double()
    err = (v - x.double()).abs()
    assert (err <= torch.maximum(x.double().abs() * 2.0**-4, torch.tensor(2.0**-137, device=device, dtype=torch.float64))).all()
    if dtype == torch.float32:    # the bounds for larger blocks do not hold here (bf16 has no numbers below 2^-133, which is 2^-6 2^-127)
        lost = (x != 0) & (v == 0)
        assert lost.any() and (err > x.double().abs() * 0.3)[~lost].any()


@pytest.mark.gpu
def test_more_elements_than_32_bits_count():
    n, tail = 2**31 + 1000, 4096 + 1000
    end = torch.randn(tail, device='cuda').half()
    x = torch.zeros(n, dtype=torch.float16, device='cuda')
    x[-tail:] = end
    start = n - tail    # a multiple of 32, so that the tail is whole blocks
    assert start % 32 == 0
    codes, exps = cast.cast_blocks_to_fp8(x)
    want, e = cast.cast_blocks_to_fp8(end)
    assert torch.equal(codes[start:], want) and torch.equal(exps[start // 32:], e) and (exps[:start // 32] == 127).all()
    back = cast.cast_blocks_from_fp8(codes, exps, torch.float16)
    assert torch.equal(back[start:], cast.cast_blocks_from_fp8(want, e, torch.float16)) and back[:start].count_nonzero() == 0
    del back, codes, exps
    y = K.gelu(x.requires_grad_(True), keep_fp8=True)
    small = end.clone().requires_grad_(True)
    z = K.gelu(small, keep_fp8=True)
    dz = torch.randn_like(z)
    dy = torch.zeros_like(y)
    dy[start:] = dz
    dx, = torch.autograd.grad(y, x, dy)
    assert torch.equal(y[start:], z) and torch.equal(dx[start:], torch.autograd.grad(z, small, dz)[0]) and dx[:start].count_nonzero() == 0
