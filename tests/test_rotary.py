"""Rotary positions against the rotation in 64 bits: layouts, parts of a head, far positions, strided views, gradients, refusals.

Tolerance of a value y1 = x1 cos - x2 sin: the angle in half turns is rounded to 32 bits (at most 2^-24 half turns, pi 2^-24 rad) and sine and
cosine are good to an ulp (2^-23 of at most 1); two products and a sum round to 2^-24 each.  Together less than 2^-20 (|x1| + |x2|), and half a
step of the output type relative to the value.
"""
import math

import pytest
import torch

from msamp.ops import native
from msamp.ops import nn as K

CPU_GPU = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def _exact(x, freqs, positions, interleaved, inverse=False):
    """The rotation as a complex product in 64 bits, and |x1| + |x2| beside it."""
    x, f = x.detach().double().cpu(), freqs.cpu()
    r, s = f.numel(), x.shape[1]
    pos = torch.arange(s) if positions is None else positions.cpu()
    angle = (pos.double()[..., None] * f).expand(x.shape[0], s, r)[:, :, None] * (-1.0 if inverse else 1.0)
    u = torch.polar(torch.ones_like(angle), angle)
    y, size = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, 2 * r, 2), slice(1, 2 * r, 2)) if interleaved else (slice(0, r), slice(r, 2 * r))
    w = torch.complex(x[..., one].contiguous(), x[..., two].contiguous()) * u
    y[..., one], y[..., two] = w.real, w.imag
    size[..., one] = size[..., two] = x[..., one].abs() + x[..., two].abs()
    return y, size


def _check(got, x, freqs, positions, interleaved, inverse=False):
    want, size = _exact(x, freqs, positions, interleaved, inverse)
    step = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * step    # below the smallest normal number steps stop shrinking
    err = (got.detach().double().cpu() - want).abs()
    assert (err <= want.abs() * step + size * 2.0**-20 + tiny).all(), (err - want.abs() * step).max().item()
    part = 2 * freqs.numel()
    assert torch.equal(got[..., part:], x.detach()[..., part:])


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('interleaved', [False, True])
@pytest.mark.parametrize('dim, part', [(64, 64), (64, 16), (128, 128), (96, 96), (80, 20), (32, 2), (256, 256), (7, 6), (640, 640)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
def test_values_and_gradients(device, interleaved, dim, part, dtype):
    torch.manual_seed(dim + part)
    freqs = K.rotary_frequencies(part, device=device)
    for batch, seq, heads, kv in ((2, 5, 4, 2), (1, 1, 3, 1), (3, 37, 2, 2)):
        q = torch.randn(batch, seq, heads, dim, device=device).to(dtype).requires_grad_(True)
        k = torch.randn(batch, seq, kv, dim, device=device).to(dtype).requires_grad_(True)
        yq, yk = K.rotary(q, k, freqs, interleaved=interleaved)
        assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
        _check(yq, q, freqs, None, interleaved)
        _check(yk, k, freqs, None, interleaved)
        gq, gk = torch.randn_like(yq), torch.randn_like(yk)
        dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
        _check(dq, gq, freqs, None, interleaved, inverse=True)
        _check(dk, gk, freqs, None, interleaved, inverse=True)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
@pytest.mark.parametrize('shared', [False, True])
def test_positions_far_and_negative(device, kind, shared):
    torch.manual_seed(1)
    freqs = K.rotary_frequencies(64, base=500000.0, device=device)
    pos = torch.randint(-5, 10_000_000, (9, ) if shared else (2, 9), device=device, dtype=kind)
    q = torch.randn(2, 9, 3, 64, device=device)
    _check(K.rotary(q, None, freqs, positions=pos), q, freqs, pos, False)
    # a column of a wider table of positions
    wide = torch.randint(0, 1 << 20, (2, 9, 2), device=device, dtype=kind)[..., 1]
    _check(K.rotary(q, None, freqs, positions=wide, interleaved=True), q, freqs, wide, True)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_views_of_a_packed_projection(device, dtype):
    """Strided heads, a start off the 16-byte grid, an expanded batch, other orders, an unused output."""
    torch.manual_seed(2)
    freqs = K.rotary_frequencies(32, device=device)
    packed = torch.randn(2, 6, 8, 64, device=device).to(dtype)
    q, k = packed[:, :, :4], packed[:, :, 4:6]
    yq, yk = K.rotary(q, k, freqs)
    _check(yq, q, freqs, None, False)
    _check(yk, k, freqs, None, False)
    off = torch.randn(2 * 6 * 4 * 64 + 3, device=device).to(dtype)[3:].view(2, 6, 4, 64)
    _check(K.rotary(off, None, freqs), off, freqs, None, False)
    wide = packed[:1].expand(3, 6, 8, 64)
    _check(K.rotary(wide, None, freqs), wide, freqs, None, False)
    heads_first = torch.randn(2, 4, 6, 64, device=device).to(dtype).transpose(1, 2)
    _check(K.rotary(heads_first, k, freqs)[0], heads_first, freqs, None, False)
    last_outer = torch.randn(2, 6, 64, 4, device=device).to(dtype).transpose(2, 3)
    _check(K.rotary(last_outer, None, freqs), last_outer, freqs, None, False)
    leaf_q, leaf_k = q.detach().clone().requires_grad_(True), k.detach().clone().requires_grad_(True)
    yq, yk = K.rotary(leaf_q, leaf_k, freqs)
    yk.sum().backward()    # an expanded gradient of one output
    assert leaf_q.grad is None
    _check(leaf_k.grad, torch.ones_like(leaf_k), freqs, None, False, inverse=True)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('interleaved', [False, True])
def test_in_place(device, interleaved):
    torch.manual_seed(3)
    freqs = K.rotary_frequencies(48, device=device)
    for offset in (0, 1):
        packed = torch.randn(2 * 5 * 6 * 64 + offset, device=device).bfloat16()[offset:].view(2, 5, 6, 64)
        before = packed.clone()
        K.rotary_raw([packed[:, :, :4]], [packed[:, :, :4]], freqs, None, interleaved, False)
        _check(packed[:, :, :4], before[:, :, :4], freqs, None, interleaved)
        assert torch.equal(packed[:, :, 4:], before[:, :, 4:])


@pytest.mark.parametrize('device', CPU_GPU)
def test_empty(device):
    freqs = K.rotary_frequencies(8, device=device)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8)):
        q = torch.empty(shape, device=device, requires_grad=True)
        y = K.rotary(q, None, freqs)
        assert y.shape == shape
        y.sum().backward()
        assert q.grad.shape == shape


def test_not_finite_values_stay_in_their_pair():
    freqs = K.rotary_frequencies(8)
    q = torch.randn(1, 2, 1, 8)
    q[0, 1, 0, 2] = float('inf')
    y = K.rotary(q, None, freqs)
    assert torch.isfinite(y).view(-1).tolist() == [i not in (10, 14) for i in range(16)]


def test_frequencies():
    f = K.rotary_frequencies(8)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(K.rotary_frequencies(8, scaling='linear', factor=4.0), f / 4.0)
    g = K.rotary_frequencies(8, scaling='base', factor=4.0)
    assert g[0] == 1.0 and math.isclose(g[-1].item(), f[-1].item() / 4.0, rel_tol=1e-12)
    h = K.rotary_frequencies(64, scaling='parts', factor=8.0, trained=2048, fast=32.0, slow=1.0)
    plain = K.rotary_frequencies(64)
    turns = plain * 2048 / (2 * math.pi)
    assert torch.equal(h[turns >= 32], plain[turns >= 32]) and torch.allclose(h[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (h[between] < plain[between]).all() and (h[between] > plain[between] / 8).all()


@pytest.mark.parametrize('kw', [dict(dim=0), dict(dim=7), dict(dim=8, base=0.0), dict(dim=8, factor=-1.0), dict(dim=8, scaling='yes'),
                                dict(dim=2, scaling='base'), dict(dim=8, scaling='parts'), dict(dim=8, scaling='parts', trained=64, fast=1.0, slow=2.0)])
def test_frequencies_refused(kw):
    with pytest.raises(ValueError):
        K.rotary_frequencies(**kw)


def test_refusals():
    f, q, k = K.rotary_frequencies(8), torch.randn(2, 3, 4, 8), torch.randn(2, 3, 1, 8)
    with pytest.raises(ValueError):
        K.rotary(q[0], None, f)
    with pytest.raises(ValueError):
        K.rotary(q, k[:, :2], f)
    with pytest.raises(ValueError):
        K.rotary(q, k[..., :6], K.rotary_frequencies(6))
    with pytest.raises(ValueError):
        K.rotary(q, k.bfloat16(), f)
    with pytest.raises(ValueError):
        K.rotary(q, None, K.rotary_frequencies(10))
    with pytest.raises(ValueError):
        K.rotary(q, None, f.float())
    with pytest.raises(ValueError):
        K.rotary(q, None, f, positions=torch.arange(4))
    with pytest.raises(TypeError):
        K.rotary(q, None, f, positions=torch.arange(3.0))
    with pytest.raises(TypeError):
        K.rotary(q.double(), None, f)
    with pytest.raises(ValueError):
        K.rotary(q, None, f.to('meta'))
    with pytest.raises(ValueError):
        K.rotary(q, None, f.clone().requires_grad_(True))


def test_raw_refusals():
    f, q, k = K.rotary_frequencies(8), torch.randn(2, 3, 4, 8), torch.randn(2, 3, 1, 8)
    for xs, ys, freqs, positions in (([q], [q], f, torch.arange(4)), ([q], [q], f, torch.arange(3, device='meta')), ([q], [q], f.to('meta'), None),
                                     ([q], [q], K.rotary_frequencies(10), None), ([q, k[:, :2]], [q, k[:, :2]], f, None), ([q], [q, k], f, None),
                                     ([q], [q[:, :, :2]], f, None), ([q], [q.bfloat16()], f, None), ([q], [torch.empty(2, 3, 8, 4).mT], f, None),
                                     ([q, k, k], [q, k, k], f, None)):
        with pytest.raises(ValueError):
            K.rotary_raw(xs, ys, freqs, positions, False, False)


@pytest.mark.skipif(not native.available(), reason='kernel library not built')
def test_entry_point_refuses():
    """No launch: every call is refused by its arguments."""
    import struct
    lib, at = native.lib(), 1 << 20
    st, other = [24, 8, 8] * 4, [24, 8, 8] + [48, 8, 8] + [24, 8, 8] * 2

    def call(x=at, y=at, strides=st, freqs=at, batch=1, part=8, dim=8, heads=1, dtype=0):
        return lib.msamp_rotary(struct.pack('30q', x, y, 0, 0, *strides, freqs, 0, 0, 0, 0, batch, 3, heads, 0, dim, part, 0, 0, dtype), None)

    for kw in (dict(x=0), dict(y=0), dict(freqs=0), dict(batch=-1), dict(part=7), dict(part=10), dict(part=0), dict(strides=other),
               dict(part=2048, dim=2048), dict(heads=-1), dict(batch=1 << 40)):
        assert call(**kw) == 1, kw
    assert call(dtype=5) == 2 and call(batch=0) == 0 and lib.msamp_rotary(None, None) == 1


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason='needs two GPUs')
def test_tensors_of_another_device_than_the_current_one():
    torch.manual_seed(6)
    freqs, q = K.rotary_frequencies(64, device='cuda:1'), torch.randn(2, 5, 4, 64, device='cuda:1')
    assert torch.cuda.current_device() == 0
    _check(K.rotary(q, None, freqs), q, freqs, None, False)
    with pytest.raises(ValueError):
        K.rotary(q, None, freqs.to('cuda:0'))


@pytest.mark.gpu
def test_captured_and_on_a_side_stream():
    torch.manual_seed(4)
    freqs = K.rotary_frequencies(64, device='cuda')
    q = torch.randn(2, 33, 4, 64, device='cuda').bfloat16()
    pos = torch.arange(33, device='cuda')
    K.rotary(q, None, freqs, positions=pos)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = K.rotary(q, None, freqs, positions=pos)
    pos += 1000
    q.normal_()
    g.replay()
    _check(y, q, freqs, pos, False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = K.rotary(q, None, freqs, positions=pos)
    s.synchronize()
    assert torch.equal(y, z)
    assert native.device_status() == 0


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('which', ['q', 'k'])
@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_tangents_are_not_dropped(monkeypatch, device, which, grad):
    """Plain operations carry a tangent (the CPU form where nothing asks for a gradient); the autograd function refuses one."""
    monkeypatch.setenv('PYTORCH_JIT', '0')    # make_dual compiles torch's own rules otherwise, which fails on functions that msamp wraps
    from torch.autograd import forward_ad as fwd
    freqs = K.rotary_frequencies(64, device=device)
    q, k, t = (torch.randn(2, 5, 4, 64, device=device).bfloat16() for _ in range(3))
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        given = dict(q=q, k=k)
        given[which] = fwd.make_dual(given[which], t)
        if device == 'cuda':
            with pytest.raises((NotImplementedError, RuntimeError), match='forward'):
                K.rotary(**given, freqs=freqs)
        else:
            y = K.rotary(**given, freqs=freqs)['qk'.index(which)]
            tangent = fwd.unpack_dual(y).tangent
            _check(tangent, t, freqs, None, False)


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('with_k', [False, True])
def test_second_derivatives(device, with_k):
    """y = R q, L = sum y^3: dL/dq = R^T 3 y^2, and the gradient of sum(w dL/dq) is R^T (6 y R w), which 64 bits give from the plain form."""
    torch.manual_seed(3)
    freqs, at = K.rotary_frequencies(16, device=device), torch.arange(5, device=device) + 100
    q, w = (torch.randn(2, 5, 3, 20, device=device) for _ in range(2))
    k, wk = (torch.randn(2, 5, 1, 20, device=device) for _ in range(2))

    def second(turn, leaves, weights):
        y = turn(*leaves)
        first = torch.autograd.grad(sum((t**3).sum() for t in y), leaves, create_graph=True)
        return first + torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, weights)), leaves)

    def mine(q, k=None):
        y = K.rotary(q, k, freqs, positions=at, interleaved=True)
        return y if k is not None else (y, )

    def plain(*xs):
        u = torch.polar(torch.ones(5, 8, dtype=torch.float64, device=device), at.double()[:, None] * freqs)[:, None]
        turned = [torch.view_as_real(torch.view_as_complex(x[..., :16].unflatten(-1, (8, 2)).contiguous()) * u).flatten(-2) for x in xs]
        return [torch.cat([t, x[..., 16:]], -1) for t, x in zip(turned, xs)]

    xs, weights = ([q, k], [w, wk]) if with_k else ([q], [w])
    got = second(mine, [x.clone().requires_grad_(True) for x in xs], weights)
    want = second(plain, [x.double().requires_grad_(True) for x in xs], [t.double() for t in weights])
    for a, b in zip(got, want):
        # three rotations and two products in 32 bits of numbers up to 6 * 5^3
        assert (a.double() - b).abs().max() <= 6 * 5.0**3 * 2.0**-20


def test_fields_of_the_forward_call_hold_for_the_same_layout_only():
    """Saved tensors may come back with other strides, in the place where the first ones were: their fields are worked out again."""
    from msamp.ops.rotary import _layout
    freqs, wide = K.rotary_frequencies(8), torch.arange(24).view(2, 12)
    pos = wide[:, ::2]
    here = _layout(freqs, pos)
    assert here == _layout(freqs, wide[:, ::2]) and _layout(freqs, None) == _layout(freqs, None)
    dense = torch.as_strided(wide, (2, 6), (6, 1))
    assert dense.data_ptr() == pos.data_ptr()
    for other in (dense, wide.int()[:, ::2], wide.clone()[:, ::2], None):
        assert _layout(freqs, other) != here
    assert _layout(freqs.clone(), pos) != here and _layout(torch.as_strided(freqs, (4, ), (0, )), pos) != here


@pytest.mark.gpu
def test_saved_positions_in_another_layout():
    """Hooks that bring the positions back dense, and a hook that leaves them alone, against the call without hooks."""
    torch.manual_seed(8)
    freqs = K.rotary_frequencies(64, device='cuda')
    q, k = torch.randn(2, 6, 4, 64, device='cuda'), torch.randn(2, 6, 2, 64, device='cuda')
    g = torch.randn_like(q), torch.randn_like(k)
    wide = torch.randint(0, 1000, (2, 12), device='cuda')
    results = []
    for pack in (None, lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t.cpu()):
        leaves = [t.clone().requires_grad_(True) for t in (q, k)]
        with torch.autograd.graph.saved_tensors_hooks(pack or (lambda t: t), lambda t: t.cuda()):
            y = K.rotary(*leaves, freqs, positions=wide[:, ::2])
        results.append(torch.autograd.grad(y, leaves, g))
    for dq, dk in results:
        assert torch.equal(dq, results[0][0]) and torch.equal(dk, results[0][1])
        _check(dq, g[0], freqs, wide[:, ::2], False, inverse=True)


@pytest.mark.gpu
@pytest.mark.parametrize('interleaved', [False, True])
def test_offsets_beyond_32_bits(interleaved):
    torch.manual_seed(2)
    buf = torch.zeros(2**31 + 4096, dtype=torch.bfloat16, device='cuda')
    x = buf.as_strided((2, 3, 2, 64), (2**31 + 256, 128, 64, 1))
    q = torch.randn(2, 3, 2, 64, device='cuda').bfloat16()
    x.copy_(q)
    freqs = K.rotary_frequencies(64, device='cuda')
    want = K.rotary(q, None, freqs, interleaved=interleaved)
    assert torch.equal(K.rotary(x, None, freqs, interleaved=interleaved), want)
    K.rotary_raw([x], [x], freqs, None, interleaved, False)    # in place
    assert torch.equal(x, want)
    assert native.device_status() == 0
