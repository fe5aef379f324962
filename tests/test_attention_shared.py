"""Attention whose query heads share key/value heads, and rows of a padded batch, against 64 bits.

Where the tolerances come from (bf16 half step u = 2^-8, relative).  Scores, sums and accumulators are in 32 bits; s = 2^-11 covers their
roundings, the 32-bit exponential and the error that the 32-bit score carries into it.  The CUDA kernels round each probability P to
bf16 for P V and for dV = P^T dO, and dS = P (dP - delta) for dQ and dK, where delta = rowsum(dO * O) is taken from the rounded O:

  |O error|     <= u |O| + (u + s) sum P |V|
  |delta error| <= sum |dO| (O error)
  |dV error|    <= u |dV| + (u + s) sum P |dO|
  |dS error|    <= u |dS| + P (delta error) + s P (sum |dO| |V| + sum |dO| |O|)
  |dQ error|    <= u |dQ| + scale sum (dS error) |K|,  dK likewise

The CPU form has no rounding but the last, within the same bounds.
"""
import math

import pytest
import torch

from msamp.ops import native
from msamp.ops import nn as K

CPU_GPU = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
U, SLACK = 2.0**-8, 2.0**-11


def _reference(q, k, v, do, causal, lengths, scale):
    """(value, bound on the error) of o, dq, dk, dv; padding is zero in both."""
    B, S, nh, d = q.shape
    nkv = k.shape[2]
    rep = nh // nkv
    at = torch.arange(S, device=q.device)
    valid = at < (torch.full((B, ), S, device=q.device) if lengths is None else lengths.clamp(0, S))[:, None]

    def heads(t, n):
        t = torch.where(valid[:, :, None, None], t.detach().double(), 0.0).permute(0, 2, 1, 3)
        return t if n == nh else t.repeat_interleave(rep, 1)

    q, k, v, do = heads(q, nh), heads(k, nkv), heads(v, nkv), heads(do, nh)
    see = valid[:, None, :, None] & valid[:, None, None, :]
    if causal:
        see = see & (at[None, :] <= at[:, None])
    x = torch.where(see, q @ k.transpose(-1, -2) * scale, -1e300)
    p = torch.where(see, torch.softmax(x, -1), 0.0)
    pt = p.transpose(-1, -2)
    o = p @ v
    o_err = U * o.abs() + (U + SLACK) * (p @ v.abs())
    dv, dv_err = pt @ do, (U + SLACK) * (pt @ do.abs())
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    size = (do.abs() @ v.abs().transpose(-1, -2)) + (do.abs() * o.abs()).sum(-1, keepdim=True)
    ds_err = U * ds.abs() + p * (do.abs() * o_err).sum(-1, keepdim=True) + SLACK * p * size
    dq, dq_err = scale * (ds @ k), scale * (ds_err @ k.abs())
    dk, dk_err = scale * (ds.transpose(-1, -2) @ q), scale * (ds_err.transpose(-1, -2) @ q.abs())

    def back(t, n):
        t = t if n == nh else t.view(B, nkv, rep, S, d).sum(2)
        return t.permute(0, 2, 1, 3)

    out = []
    for value, err, n in ((o, o_err, nh), (dq, dq_err, nh), (dk, dk_err, nkv), (dv, dv_err, nkv)):
        value, err = back(value, n), back(err, n)
        out.append((value, err + U * value.abs() + 1e-30))
    return out, valid


def _inputs(B, S, nh, nkv, d, device, seed=0, spread=1.0):
    gen = torch.Generator().manual_seed(seed + S)
    make = lambda n: torch.randn(B, S, n, d, generator=gen).bfloat16().to(device)    # noqa: E731
    return make(nh) * spread, make(nkv), make(nkv), make(nh)


def _compare(got, want, valid):
    for name, a, (value, bound) in zip(('o', 'dq', 'dk', 'dv'), got, want):
        err = (a.detach().double() - value).abs()
        assert (err <= bound).all(), (name, (err / bound).max().item(), err.max().item())
        pad = ~valid[:, :, None, None].expand_as(value)
        assert (a.detach()[pad] == 0).all(), name


def _run(q, k, v, do, causal, lengths, scale=None, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = K.attention(*leaves, causal=causal, scale=scale, lengths=lengths, **kw)
    return [o, *torch.autograd.grad(o, leaves, do)]


def _status_ok():
    torch.cuda.synchronize()
    assert native.device_status() == 0


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('S, nh, nkv', [(1, 4, 2), (2, 2, 1), (5, 4, 2), (63, 3, 1), (64, 8, 2), (65, 2, 1), (127, 4, 4), (128, 6, 2), (129, 4, 1),
                                        (200, 16, 1), (256, 4, 2), (385, 2, 1)])
def test_shared_heads(device, d, causal, S, nh, nkv):
    q, k, v, do = _inputs(2, S, nh, nkv, d, device)
    want, valid = _reference(q, k, v, do, causal, None, d**-0.5)
    if nh == nkv:    # the kernels of shared heads serve one query head each too
        got = _run(q, k, v, do, causal, torch.full((2, ), S, device=device))
    else:
        got = _run(q, k, v, do, causal, None)
    _compare(got, want, valid)
    if device == 'cuda':
        _status_ok()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('junk', [0.0, float('nan'), float('inf'), torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize('S, nh, nkv, lengths', [(130, 4, 2, (130, 0, 1, 129, 128, 127)), (300, 2, 2, (5, 300, 256, 255, 257, -3)),
                                                 (7, 6, 1, (0, 0, 3)), (7, 2, 1, (0, 0)), (520, 2, 1, (1000, 385, 130))])
def test_lengths(device, d, causal, junk, S, nh, nkv, lengths):
    q, k, v, do = _inputs(len(lengths), S, nh, nkv, d, device)
    n = torch.tensor(lengths, device=device, dtype=torch.int32 if S % 2 else torch.int64)
    want, valid = _reference(q, k, v, do, causal, n, d**-0.5)
    q, k, v, do = (torch.where(valid[:, :, None, None], t, junk) for t in (q, k, v, do))
    _compare(_run(q, k, v, do, causal, n), want, valid)
    if device == 'cuda':
        _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('B, S, nh, nkv, ragged', [(1, 2048, 8, 1, False), (4, 1000, 24, 8, True), (40, 200, 12, 4, True), (3, 700, 36, 12, False),
                                                   (2, 1500, 96, 96, True), (300, 10, 4, 2, True), (3000, 20, 2, 1, True)])
def test_many_work_items(d, B, S, nh, nkv, ragged):
    """Several waves of items, items in parts, rows of every length in one batch."""
    q, k, v, do = _inputs(B, S, nh, nkv, d, 'cuda')
    n = torch.randint(0, S + 1, (B, ), generator=torch.Generator().manual_seed(B)).to('cuda') if ragged else None
    got = _run(q, k, v, do, True, n)
    for b in range(0, B, max(1, B // 3)):
        one = slice(b, b + 1)
        for h in range(0, nkv, max(1, nkv // 2)):
            qs = slice(h * nh // nkv, (h + 1) * nh // nkv)
            want, valid = _reference(q[one, :, qs], k[one, :, h:h + 1], v[one, :, h:h + 1], do[one, :, qs], True, None if n is None else n[one], d**-0.5)
            _compare([got[0][one, :, qs], got[1][one, :, qs], got[2][one, :, h:h + 1], got[3][one, :, h:h + 1]], want, valid)
    again = _run(q, k, v, do, True, n)
    assert all(torch.equal(a, b) for a, b in zip(got, again))    # no atomics: the same bits
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('B, S', [(1, 1), (1, 5000), (7, 700), (33, 300), (100, 129), (2000, 130), (70000, 3)])
def test_list_of_tiles(B, S, causal):
    """The tiles that hold rows of a sequence, each once, by falling work, then by batch and tile."""
    n = torch.randint(-2, S + 3, (B, ), generator=torch.Generator().manual_seed(B))
    q = torch.zeros(B, S, 2, 64, device='cuda', dtype=torch.bfloat16)
    o, lse, plan = K.attention_shared_fwd_raw(q, q[:, :, :1], q[:, :, :1], causal, lengths=n.cuda())
    tiles, want = (S + 127) // 128, []
    for b, m in enumerate(((n.clamp(0, S) + 127) // 128).tolist()):
        want += [(-(i + 1 if causal else m), b, i) for i in range(m)]
    want = [b * tiles + i for _, b, i in sorted(want)]
    plan = plan.tolist()
    assert plan[0] == len(want) and plan[1] in (1, 2) and plan[2:2 + len(want)] == want
    pad = (torch.arange(S) >= n[:, None]).cuda()
    assert torch.equal(torch.isinf(lse).all(1), pad) and not o.any()
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('S', [1, 2, 3, 5, 9, 17, 100, 128])
def test_gradients_of_few_keys_in_norm(d, S):
    """dS = P (dP - delta) is a small difference where a row has few keys.  With delta exact, dS, its product's result and P carry a bf16
    rounding each: at most u = 2^-8 of every term, 2^-8 / sqrt(3) of the norm on average; two of them, and a half for the few values of a short
    row: 1.5 sqrt(2 / 3) u < 0.005."""
    q, k, v, do = _inputs(2, S, 4, 2, d, 'cuda', spread=1.5)
    q = q.bfloat16()
    for n in (None, torch.tensor([S, (S + 1) // 2], device='cuda')):
        want, _ = _reference(q, k, v, do, True, n, d**-0.5)
        for a, (value, _) in zip(_run(q, k, v, do, True, n), want):
            assert (a.double() - value).norm() <= 0.005 * value.norm()    # S == 1: dq and dk are exactly zero
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('scale, spread', [(0.5, 4.0), (1e-4, 1.0), (1.0, 8.0)])
def test_peaked_and_flat_rows(d, scale, spread):
    """Scores of several hundred (the running maximum moves far) and scores that are all alike.

    A score is a sum of d products rounded to 32 bits: an error of at most d 2^-24 of sum |q| |k| scale enters the exponent, which the
    bound takes on top where scores are large.
    """
    q, k, v, do = _inputs(1, 400, 4, 2, d, 'cuda', spread=spread)
    n = torch.tensor([390], device='cuda')
    want, valid = _reference(q, k, v, do, True, n, scale)
    top = (q.abs().double().sum(-1).max() * k.abs().double().max() * scale).item() * 2.0**-22
    want = [(w, b * (1 + top / SLACK)) for w, b in want]
    _compare(_run(q, k, v, do, True, n, scale=scale), want, valid)
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('lengths', [None, (150, 260)])
def test_equal_heads_agree_with_the_plain_form(d, lengths):
    """Every key head repeated: dq and o as with shared heads, dk and dv their parts."""
    q, k, v, do = _inputs(2, 260, 6, 2, d, 'cuda')
    n = None if lengths is None else torch.tensor(lengths, device='cuda')
    a = _run(q, k, v, do, True, n)
    b = _run(q, k.repeat_interleave(3, 2), v.repeat_interleave(3, 2), do, True, torch.tensor([260, 260], device='cuda') if n is None else n)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    want, valid = _reference(q, k, v, do, True, n, d**-0.5)
    for x, y, (value, bound) in zip(a[2:], b[2:], want[2:]):
        parts = y.double().view(2, 260, 2, 3, d)
        assert ((x.double() - parts.sum(3)).abs() <= 2 * bound + 2 * U * parts.abs().sum(3)).all()
    _status_ok()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('d', [64, 128])
def test_views_and_layouts(device, d):
    """Views of a packed projection, packed gradients, an expanded key, strides and starts of the incoming gradient."""
    B, S, nh, nkv = 2, 140, 4, 2
    packed = torch.randn(B, S, nh + 2 * nkv, d, generator=torch.Generator().manual_seed(d)).bfloat16().to(device)
    q, k, v = packed.split([nh, nkv, nkv], 2)
    do = torch.randn(B, S, nh, d, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    n = torch.tensor([140, 77], device=device)
    want, valid = _reference(q, k, v, do, True, n, d**-0.5)
    got = _run(q, k, v, do, True, n)
    _compare(got, want, valid)
    same = _run(q, k, v, do, True, n, grad_layout='packed')
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    if device == 'cuda':
        assert same[1].stride() == ((nh + 2 * nkv) * d * S, (nh + 2 * nkv) * d, d, 1)
    shifted = torch.empty(do.numel() + 1, dtype=do.dtype, device=device)[1:].view_as(do).copy_(do)
    turned = do.transpose(1, 3).contiguous().transpose(1, 3)
    for other in (shifted, turned):
        assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, other, True, n)))
    one = do[:, :1, :1].expand_as(do)    # a gradient that repeats
    want, valid = _reference(q, k, v, one, True, n, d**-0.5)
    _compare(_run(q, k, v, one, True, n), want, valid)
    wide_k, wide_v = k[:1].expand_as(k), v[:1].expand_as(v)    # keys that repeat
    want, valid = _reference(q, wide_k, wide_v, do, True, n, d**-0.5)
    _compare(_run(q, wide_k, wide_v, do, True, n), want, valid)
    leaf = k[:1].detach().requires_grad_(True)
    o = K.attention(q, leaf.expand_as(k), v, lengths=n)
    g, = torch.autograd.grad(o, leaf, do)
    want, _ = _reference(q, wide_k, v, do, True, n, d**-0.5)
    value, bound = want[2]
    assert ((g.double() - value.sum(0, keepdim=True)).abs() <= bound.sum(0, keepdim=True) + U * value.abs().sum(0, keepdim=True)).all()
    single = K.attention(q[:1, :, :, :].as_strided((1, S, nh, d), (3, *q.stride()[1:])), k[:1], v[:1])    # an odd stride of an axis of one
    assert torch.equal(single, K.attention(q[:1].contiguous(), k[:1].contiguous(), v[:1].contiguous()))
    if device == 'cuda':
        _status_ok()


@pytest.mark.parametrize('device', CPU_GPU)
def test_empty(device):
    for B, S in ((0, 4), (2, 0)):
        q = torch.empty(B, S, 4, 64, device=device, dtype=torch.bfloat16, requires_grad=True)
        k = torch.empty(B, S, 2, 64, device=device, dtype=torch.bfloat16)
        o = K.attention(q, k, k, lengths=torch.zeros(B, dtype=torch.int32, device=device))
        o.sum().backward()
        assert o.shape == q.shape and q.grad.shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('lengths', [None, (200, 90)])
def test_saved_tensors_in_other_layouts(d, lengths):
    """What saved-tensor hooks bring back may lie anywhere: other strides, off the 16-byte grid, via the host."""
    q, k, v, do = _inputs(2, 200, 4, 2, d, 'cuda')
    n = None if lengths is None else torch.tensor(lengths, device='cuda')
    want = _run(q, k, v, do, True, n)

    def turned(t):
        return t.transpose(0, t.dim() - 1).contiguous().transpose(0, t.dim() - 1)

    def strided(t):
        return torch.stack([t, t], -1)[..., 0]

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t) if t.dim() == 4 else t

    for unpack in (turned, strided, shifted, lambda t: t.cpu().cuda()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            got = _run(q, k, v, do, True, n)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('S, lengths', [(100, None), (300, None), (300, [300, 7, 0])])
def test_backward_leaves_saved_tensors_alone(S, lengths):
    """Two backward passes of one forward pass, captured ones too, share nothing that either writes."""
    q, k, v, do = _inputs(3, S, 4, 2, 64, 'cuda')
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    kept = []
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        out = K.attention(*leaves, causal=True, lengths=n)
    before = [t.clone() for t in kept]
    one = torch.autograd.grad(out, leaves, do, retain_graph=True)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kept, before))
    torch.autograd.grad(out, leaves, 2 * do, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(one, torch.autograd.grad(out, leaves, do)))
    _status_ok()


@pytest.mark.gpu
def test_raw_backward_refusals():
    q, k, v, do = _inputs(2, 40, 4, 2, 64, 'cuda')
    n = torch.tensor([40, 7], dtype=torch.int32, device='cuda')
    o, lse, plan = K.attention_shared_fwd_raw(q, k, v, lengths=n)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    good = [q, k, v, o, lse, plan, do, dq, dk, dv]
    for at, bad in ((3, o[:, :39]), (4, lse[0]), (4, lse.half()), (5, None), (5, plan[:2]), (6, do.float()), (7, dk), (8, dk[:1]), (9, dv.cpu()),
                    (7, torch.empty(2, 40, 64, 4, dtype=torch.bfloat16, device='cuda').mT)):
        with pytest.raises(ValueError):
            K.attention_shared_bwd_raw(*good[:at], bad, *good[at + 1:], lengths=n)
    K.attention_shared_bwd_raw(*good, lengths=n)
    assert all(t.isfinite().all() for t in (dq, dk, dv))
    _status_ok()


def test_other_numbers_of_keys_on_the_cpu():
    """Equal heads, more keys than queries: what attention on the CPU has always taken."""
    torch.manual_seed(0)
    q, k, v = torch.randn(2, 3, 4, 8), torch.randn(2, 5, 4, 8), torch.randn(2, 5, 4, 8)
    x = torch.einsum('bihd,bjhd->bhij', q, k) / 8**0.5
    want = torch.einsum('bhij,bjhd->bihd', torch.softmax(x, -1), v)
    assert torch.allclose(K.attention(q, k, v, causal=False), want, rtol=1e-5, atol=1e-6)


def test_gradients_against_differences():
    """The CPU form in 32 bits, central differences of sum(o * do) in random directions."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(2, 9, n, 8, dtype=torch.float32) for n in (4, 2, 2))
    do, n = torch.randn(2, 9, 4, 8), torch.tensor([9, 5])
    grads = _run(q, k, v, do, True, n)[1:]
    for i in range(3):
        way = torch.randn_like((q, k, v)[i])
        step = 1e-2
        f = []
        for sign in (1, -1):
            args = [t.clone() for t in (q, k, v)]
            args[i] += sign * step * way
            f.append((K.attention(*args, lengths=n).double() * do).sum().item())
        # third derivatives of a softmax of scores of order one: the step enters squared
        assert math.isclose((f[0] - f[1]) / (2 * step), (grads[i].double() * way).sum().item(), rel_tol=5e-3, abs_tol=5e-3)


def test_refusals():
    q, k = torch.randn(2, 3, 4, 8), torch.randn(2, 3, 2, 8)
    n = torch.tensor([3, 2])
    for bad in (lambda: K.attention(q, k, k[:, :, :1]), lambda: K.attention(q, k[:, :2], k[:, :2], lengths=n), lambda: K.attention(q, q[:, :, :3], q[:, :, :3]),
                lambda: K.attention(q, k[..., :4], k[..., :4]), lambda: K.attention(q, k.half(), k), lambda: K.attention(q, k[:, :, :0], k[:, :, :0]),
                lambda: K.attention(q, k, k, lengths=n[:1]), lambda: K.attention(q, k, k, lengths=n.float()),
                lambda: K.attention(q, k, k, lengths=n.to('meta')), lambda: K.attention(q, k, k, scale=0.0),
                lambda: K.attention(q, k, k, scale=float('nan')), lambda: K.attention(q, k, k, scale=float('inf')), lambda: K.attention(q[0], k, k, lengths=n)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.gpu
def test_refusals_on_cuda():
    q, k = torch.randn(2, 3, 4, 64, device='cuda'), torch.randn(2, 3, 2, 64, device='cuda')
    with pytest.raises(RuntimeError):
        K.attention(q, k, k)    # fp32
    q, k = q.bfloat16(), k.bfloat16()
    with pytest.raises(RuntimeError):
        K.attention(q[..., :32], k[..., :32], k[..., :32])
    off = torch.empty(2 * 3 * 2 * 64 + 1, device='cuda', dtype=torch.bfloat16)[1:].view(2, 3, 2, 64)
    with pytest.raises(RuntimeError):
        K.attention(q, off, k)
    with pytest.raises(ValueError):
        K.attention(q, k, k, lengths=torch.tensor([1, 2]))
    _status_ok()


@pytest.mark.skipif(not native.available(), reason='kernel library not built')
def test_entry_points_refuse():
    """No launch and no driver call: every call is refused by its arguments."""
    import struct
    lib, at = native.lib(), 1 << 20
    good = [768, 256, 64] * 8

    def fwd(ptrs=None, strides=good, sizes=(2, 4, 2, 3, 64), scale=0.125, lengths=0):
        return lib.msamp_attention_shared_fwd(struct.pack('7q6qd12q', *(ptrs or [at] * 5), lengths, 0, *sizes, 1, scale, *strides[:12]), None)

    def bwd(ptrs=None, strides=good, sizes=(2, 4, 2, 3, 64), scale=0.125, partial=at, lengths=0):
        p = ptrs or [at] * 9
        return lib.msamp_attention_shared_bwd(struct.pack('13q6qd24q', *p[:5], lengths, 0, *p[5:], at, partial, *sizes, 1, scale, *strides), None)

    odd = good[:4] + [260] + good[5:]
    for call in (fwd, bwd):
        assert call(strides=odd) == 1 and call(sizes=(2, 4, 2, 3, 96)) == 1 and call(sizes=(2, 4, 3, 3, 64)) == 1
        assert call(sizes=(0, 4, 2, 3, 64)) == 1 and call(sizes=(2, 4, 2, 0, 64)) == 1 and call(sizes=(2, 4, 0, 3, 64)) == 1
        assert call(lengths=at) == 1    # without a plan
        assert call(scale=0.0) == 1 and call(scale=-1.0) == 1 and call(scale=float('nan')) == 1
        assert call(sizes=(1 << 14, 1 << 14, 1, 1 << 10, 64)) == 1 and call(sizes=(2, 4, 2, 1 << 40, 64)) == 1 and call(sizes=(-2, 4, 2, 3, 64)) == 1
    p = [at] * 5 + [at, at] + [at] * 5 + [0]    # lengths, a plan, query heads in parts and nowhere to leave their sums
    assert lib.msamp_attention_shared_bwd(struct.pack('13q6qd24q', *p, 2, 4, 2, 3, 64, 1, 0.125, *good), None) == 1
    assert lib.msamp_attention_shared_fwd(None, None) == 1 and lib.msamp_attention_shared_bwd(None, None) == 1
    for i in (0, 1, 2, 3):
        assert fwd([at + 8 * (j == i) for j in range(5)]) == 1
    for i in (0, 1, 2, 3, 5, 6, 7, 8):
        assert bwd([at + 8 * (j == i) for j in range(9)]) == 1


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
def test_captured_twice_with_other_lengths(d):
    """Two graphs of the same shapes, replayed in turn on other inputs and lengths, against the call outside of a graph."""
    B, S, nh, nkv = 2, 150, 4, 1
    n = torch.tensor([150, 20], device='cuda', dtype=torch.int32)
    sets = []
    for seed in range(2):
        q, k, v, do = _inputs(B, S, nh, nkv, d, 'cuda', seed=seed)
        _run(q, k, v, do, True, n)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(q, k, v, do, True, n)
        sets.append((g, (q, k, v, do), out))
    for lengths in ((150, 150), (1, 0), (129, 64)):
        n.copy_(torch.tensor(lengths))
        for g, _, _ in sets:
            g.replay()
        for _, args, out in sets:
            assert all(torch.equal(a, b) for a, b in zip(out, _run(*args, True, n)))
    _status_ok()


@pytest.mark.gpu
def test_on_a_side_stream():
    q, k, v, do = _inputs(2, 300, 8, 2, 64, 'cuda')
    want = _run(q, k, v, do, True, None)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(q, k, v, do, True, None)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    _status_ok()


FAR = (2**63 - 1, 2**31 + 3, 2**32 + 2, 2**31, -2**63, -2**31 - 5, -2**32 + 2, 5)
NEAR = (9, 9, 9, 9, 0, 0, 0, 5)    # the same in rows of 9


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('d', [64, 128])
def test_far_lengths(device, d):
    """Lengths outside of 0 .. S count as 0 or S, int64 ones that no int32 holds as well."""
    q, k, v, do = _inputs(len(FAR), 9, 4, 2, d, device)
    near = torch.tensor(NEAR, device=device)
    want, valid = _reference(q, k, v, do, True, near, d**-0.5)
    got = _run(q, k, v, do, True, torch.tensor(FAR, device=device))
    _compare(got, want, valid)
    assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, do, True, near)))
    if device == 'cuda':
        _status_ok()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('which', [0, 1, 2])
def test_forward_mode_tangents_are_not_dropped(monkeypatch, device, which, grad):
    """Plain operations carry a tangent (the CPU form); the autograd function refuses one."""
    monkeypatch.setenv('PYTORCH_JIT', '0')    # make_dual compiles torch's own rules otherwise, which fails on functions that msamp wraps
    from torch.autograd import forward_ad as fwd
    args = list(_inputs(2, 9, 4, 2, 64, device)[:3])
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
        for n in (None, torch.tensor([9, 4], device=device)):
            if device == 'cuda':
                with pytest.raises((NotImplementedError, RuntimeError), match='forward'):
                    K.attention(*args, lengths=n)
            else:
                assert fwd.unpack_dual(K.attention(*args, lengths=n)).tangent is not None


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('lengths', [None, (9, 4)])
def test_second_derivatives(device, lengths):
    """The CPU form differentiates twice; on CUDA the gradients have no gradient and say so, also where the incoming one is a constant."""
    q, k, v, _ = _inputs(2, 9, 4, 2, 64, device)
    n = None if lengths is None else torch.tensor(lengths, device=device)
    for power in (1, 2):
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        o = K.attention(*leaves, lengths=n)
        plain = torch.autograd.grad((o.float()**power).sum(), leaves, retain_graph=True)
        first = torch.autograd.grad((o.float()**power).sum(), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, first)) and all(t.requires_grad for t in first[:2])
        total = first[0].float().pow(2).sum() + leaves[0].float().sum()
        if device == 'cuda':
            with pytest.raises(RuntimeError, match='twice'):
                total.backward()
        else:
            total.backward()
            assert (leaves[0].grad.float() - 1.0).abs().sum() > 0


@pytest.mark.gpu
def test_raw_backward_refuses_saved_tensors_of_another_place_or_type():
    """Addresses of the host's memory, or 64-bit words, never reach the kernels: the call is refused before its first launch."""
    q, k, v, do = _inputs(2, 40, 4, 2, 64, 'cuda')
    n = torch.tensor([40, 7], dtype=torch.int32, device='cuda')
    o, lse, plan = K.attention_shared_fwd_raw(q, k, v, lengths=n)
    dq, dk, dv = (torch.zeros_like(t) for t in (q, k, v))
    good = [q, k, v, o, lse, plan, do, dq, dk, dv]
    for at, bad in ((4, lse.cpu()), (4, lse.double()), (5, plan.cpu()), (5, plan.long()), (5, plan.float())):
        with pytest.raises(ValueError):
            K.attention_shared_bwd_raw(*good[:at], bad, *good[at + 1:], lengths=n)
    with pytest.raises(ValueError):
        K.attention_shared_bwd_raw(*good[:5], plan, *good[6:])    # a plan without lengths
    _status_ok()
    assert not dq.any() and not dk.any() and not dv.any()


@pytest.mark.parametrize('q_heads, k_heads, v_heads, keys, v_dim, scale', [(1, 4, 4, 5, 8, None), (1, 4, 4, 7, 8, None), (4, 1, 1, 5, 6, None),
                                                                           (4, 1, 4, 5, 8, None), (4, 4, 1, 5, 8, None), (4, 1, 1, 7, 8, None),
                                                                           (4, 1, 1, 5, 8, -0.3), (4, 1, 1, 5, 8, 0.0), (4, 2, 2, 7, 8, None)])
def test_single_heads_on_the_cpu(q_heads, k_heads, v_heads, keys, v_dim, scale):
    """On the CPU a single head has always served all heads of the other side, with any sizes that the products allow."""
    torch.manual_seed(0)
    q, k, v = torch.randn(2, 5, q_heads, 8), torch.randn(2, keys, k_heads, 8), torch.randn(2, keys, v_heads, v_dim)
    n = max(q_heads, k_heads)
    qn, kn, vn = (t.double().repeat_interleave(n // t.shape[2], 2) for t in (q, k, v))
    x = torch.einsum('bihd,bjhd->bhij', qn, kn) * (8**-0.5 if scale is None else scale)
    want = torch.einsum('bhij,bjhd->bihd', torch.softmax(x, -1), vn)
    got = K.attention(q, k, v, causal=False, scale=scale)
    assert got.shape == want.shape and torch.allclose(got.double(), want, rtol=1e-5, atol=1e-6)


@pytest.mark.gpu
def test_equal_heads_of_other_sizes_are_refused_on_cuda():
    """The kernels take the sizes of q for k and v as well: others would be read past their end."""
    q = torch.randn(2, 6, 4, 64, device='cuda').bfloat16()
    for k, v in ((q[:, :5], q[:, :5]), (q, q[:, :5]), (q[:1], q[:1]), (q, q[:1]), (q, q[:, :, :2]), (q, q.float()), (q.half(), q), (q, q.cpu())):
        with pytest.raises(ValueError):
            K.attention(q, k, v, causal=False)
    assert K.attention(q, q, q).isfinite().all()
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('S', [1, 2, 3, 4, 7, 9, 17, 33, 63, 64, 65, 100, 128, 200])
def test_gradients_of_few_keys_in_norm_with_equal_heads(d, S, causal, packed):
    """The bound of test_gradients_of_few_keys_in_norm, over several draws: the norm of two keys' gradients varies with how far they cancel.

    One key: dS = P (dP - P dP) is zero up to 32-bit rounding.  The exponent of P is a difference of numbers below 2^3, rounded to 2^-22, so
    P is within 2^-21 of 1 and |dS| <= 2^-21 |dP|; the product's own 2^-8 is of that.  2^-20 max |dP| covers it, times scale and |K| or |Q|.
    """
    for seed in range(6):
        q, k, v, do = _inputs(2, S, 4, 4, d, 'cuda', seed=1000 * seed, spread=1.5)
        q = q.bfloat16()
        want, _ = _reference(q, k, v, do, causal, None, d**-0.5)
        zero = 2.0**-20 * d**-0.5 * (do * v).float().sum(-1).abs().max().item() * max(q.float().norm().item(), k.float().norm().item()) if S == 1 else 0.0
        if packed:
            qkv = torch.stack([q, k, v], 2).requires_grad_(True)
            o = K.attention_qkv(qkv, causal=causal)
            got = [o, *torch.autograd.grad(o, qkv, do)[0].unbind(2)]
        else:
            got = _run(q, k, v, do, causal, None)
        for name, a, (value, _) in zip(('o', 'dq', 'dk', 'dv'), got, want):
            err, size = (a.detach().double() - value).norm().item(), value.norm().item()
            assert err <= 0.005 * size + zero, (seed, name, err / size if size else err)
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('kind', [torch.int32, torch.int64])
def test_backward_takes_the_lengths_of_its_forward_pass(kind):
    """Without autograd's version check (as in graphs that are replayed apart) other lengths in the same tensor change nothing between the passes."""
    q, k, v, do = _inputs(3, 150, 4, 2, 64, 'cuda')
    n = torch.tensor([150, 20, 0], dtype=kind, device='cuda')
    o, lse, plan = K.attention_shared_fwd_raw(q, k, v, lengths=n)
    grads = []
    for other in ((150, 20, 0), (0, 150, 140)):
        n.copy_(torch.tensor(other))
        grads.append([torch.full_like(t, float('nan')) for t in (q, k, v)])
        K.attention_shared_bwd_raw(q, k, v, o, lse, plan, do, *grads[-1], lengths=n)
    want, valid = _reference(q, k, v, do, True, torch.tensor([150, 20, 0], device='cuda'), 64**-0.5)
    _compare([o, *grads[0]], want, valid)
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('S, nh, nkv, lengths', [(5000, 2, 1, None), (4097, 2, 2, (4097, )), (6001, 1, 1, (5890, ))])
def test_long_rows(d, S, nh, nkv, lengths):
    q, k, v, do = _inputs(1, S, nh, nkv, d, 'cuda')
    n = None if lengths is None else torch.tensor(lengths, device='cuda')
    want, valid = _reference(q, k, v, do, True, n, d**-0.5)
    _compare(_run(q, k, v, do, True, n), want, valid)
    _status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize('lengths', [None, (150, 70)])
def test_offsets_beyond_32_bits(lengths):
    """Two batches of a packed projection that lie more than 2^31 elements apart."""
    S, nh, nkv, d = 150, 4, 2, 64
    width = (nh + 2 * nkv) * d
    buf = torch.zeros(2**31 + 8 * width + S * width, dtype=torch.bfloat16, device='cuda')
    x = buf.as_strided((2, S, nh + 2 * nkv, d), (2**31 + 8 * width, width, d, 1))
    q, k, v, do = _inputs(2, S, nh, nkv, d, 'cuda')
    for part, at in ((q, 0), (k, nh), (v, nh + nkv)):
        x[:, :, at:at + part.shape[2]] = part
    n = None if lengths is None else torch.tensor(lengths, device='cuda')
    want = _run(q, k, v, do, True, n)
    got = _run(*x.split([nh, nkv, nkv], 2), do, True, n)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _status_ok()


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason='needs two GPUs')
@pytest.mark.parametrize('lengths', [None, (150, 70)])
def test_tensors_of_another_device_than_the_current_one(lengths):
    q, k, v, do = _inputs(2, 150, 4, 2, 64, 'cuda:1')
    n = None if lengths is None else torch.tensor(lengths, device='cuda:1')
    assert torch.cuda.current_device() == 0
    want, valid = _reference(q, k, v, do, True, n, 64**-0.5)
    _compare(_run(q, k, v, do, True, n), want, valid)
    with pytest.raises(ValueError):
        K.attention(q, k, v, lengths=torch.tensor([150, 70], device='cuda:0'))
