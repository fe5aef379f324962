"""Rotary positions, shared key/value heads, padded rows and activations in 8 bits together, as a GPT block uses them."""
import math

import pytest
import torch

import msamp
from msamp.models import GPT, gpt_config
from msamp.nn import LinearReplacer
from msamp.nn import fused_layers as FL
from msamp.ops import cast, native
from msamp.ops import nn as K

CPU_GPU = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]


def _config(**kw):
    return gpt_config('gpt-tiny', **{**dict(n_layer=2, n_head=4, hidden=256, ffn_hidden=512, vocab_size=512, max_seq=64), **kw})


def _batch(device, batch=3, seq=24):
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 512, (batch, seq), generator=gen)
    lengths = torch.tensor([seq, 7, 1][:batch])
    labels = torch.where(torch.arange(seq) < lengths[:, None], tokens.roll(-1, 1), torch.tensor(-100))
    return tokens.to(device), labels.to(device), lengths.to(device)


def _model(device, **kw):
    torch.manual_seed(0)
    return GPT(_config(**kw), device=device, act_dtype=torch.bfloat16 if device == 'cuda' else torch.float32)


LONG = dict(n_kv_head=2, rotary_dim=32, keep_fp8=True)


def _plain_block(blk, x, batch, seq, freqs, valid):
    """A block in torch operations: what the framework's form has to compute."""
    h, d, n, m = x.shape[1], blk.head_dim, blk.n_head, blk.n_kv

    def norm(ln, t):
        return torch.nn.functional.layer_norm(t, (h, ), ln.weight, ln.bias, ln.eps)

    qkv = torch.nn.functional.linear(norm(blk.ln1, x), blk.qkv.weight, blk.qkv.bias).view(batch, seq, n + 2 * m, d)
    q, k, v = qkv.split([n, m, m], 2)
    angle = torch.arange(seq, dtype=torch.float64)[:, None] * freqs
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(t):
        r = freqs.numel()
        a, b = t[..., :r], t[..., r:2 * r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, t[..., 2 * r:]], -1)

    q, k = turn(q), turn(k).repeat_interleave(n // m, 2)
    v = v.repeat_interleave(n // m, 2)
    s = torch.einsum('bihd,bjhd->bhij', q, k) / d**0.5
    see = valid[:, None, None, :] & torch.ones(seq, seq, dtype=torch.bool).tril()
    p = torch.softmax(torch.where(see, s, torch.tensor(-1e30)), -1) * valid[:, None, :, None]
    o = torch.einsum('bhij,bjhd->bihd', p, v).reshape(batch * seq, -1)
    x = x + torch.nn.functional.linear(o, blk.proj.weight, blk.proj.bias)
    f = torch.nn.functional.linear(norm(blk.ln2, x), blk.fc1.weight, blk.fc1.bias)
    return x + torch.nn.functional.linear(torch.nn.functional.gelu(f, approximate='tanh'), blk.fc2.weight, blk.fc2.bias)


def test_model_computes_the_plain_block():
    """fp32 on the CPU: loss and gradients equal the plain form's up to 32-bit rounding (same matrices, other order of sums)."""
    model = _model('cpu', n_kv_head=2, rotary_dim=32)
    tokens, labels, lengths = _batch('cpu')
    loss = model(tokens, labels, lengths=lengths)
    loss.backward()
    mine = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    b, s = tokens.shape
    valid = torch.arange(s) < lengths[:, None]
    x = model.wte(tokens).view(b * s, -1)
    for blk in model.blocks:
        x = _plain_block(blk, x, b, s, model._freqs, valid)
    ln = model.ln_f
    logits = torch.nn.functional.layer_norm(x, (x.shape[1], ), ln.weight, ln.bias, ln.eps) @ model.lm_head.weight.t()
    want = torch.nn.functional.cross_entropy(logits, labels.reshape(-1), ignore_index=-100)
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5
    for n, p in model.named_parameters():
        assert (mine[n] - p.grad).norm() <= 1e-4 * p.grad.norm() + 1e-7, n


def test_padding_does_not_change_a_row():
    model = _model('cpu', **LONG)
    tokens, _, lengths = _batch('cpu')
    out = model(tokens, lengths=lengths)
    other = tokens.clone()
    other[torch.arange(tokens.shape[1]) >= lengths[:, None]] = 5
    again = model(other, lengths=lengths)
    short = model(tokens[1:2, :7])
    assert torch.equal(out[1, :7], again[1, :7]) and torch.allclose(out[1, :7], short[0], rtol=1e-5, atol=1e-5)


def test_positions_are_relative():
    """Rotary scores depend on differences of positions only: a shifted context gives the same logits up to 32-bit rounding."""
    model = _model('cpu', n_kv_head=1, rotary_dim=64, rotary_interleaved=True)
    tokens, _, _ = _batch('cpu')
    at = torch.arange(tokens.shape[1])
    a, b, c = model(tokens), model(tokens, positions=at + 123456), model(tokens, positions=at * 2)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-4) and not torch.allclose(a, c, rtol=1e-2, atol=1e-2)


def _train_grads(device, opt, recompute=False, steps=1, **kw):
    model = _model(device, recompute=recompute, **kw)
    optimizer = torch.optim.AdamW(model.parameters(), lr=1e-3)
    if opt:
        model, optimizer = msamp.initialize(model, optimizer, opt)
    tokens, labels, lengths = _batch(device)
    for _ in range(steps):
        optimizer.zero_grad()
        loss = model(tokens, labels, lengths=lengths)
        loss.backward()
        grads = {n: (p.grad.float() if p.grad is not None else None) for n, p in model.named_parameters()}
        optimizer.step()
    return loss.item(), grads


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('opt', [None, 'O1', 'O2'])
@pytest.mark.parametrize('recompute', [False, True, 'fp8'])
def test_trains_with_every_option(device, opt, recompute):
    if device == 'cuda' and opt is None:
        pytest.skip('bf16 activations against fp32 linears: the model runs on CUDA after msamp.initialize')
    loss, grads = _train_grads(device, opt, recompute, steps=3, rotary_scaling='parts', rotary_factor=2.0, rotary_trained=64, **LONG)
    assert math.isfinite(loss)
    for n, g in grads.items():
        assert g is not None and torch.isfinite(g).all() and g.abs().sum() > 0, n
    if device == 'cuda':
        torch.cuda.synchronize()
        assert native.device_status() == 0


def test_fused_sublayers_compute_what_the_separate_calls_compute():
    """FP8 on the CPU emulation: the attention sublayer with rope, shared heads and lengths against LayerNorm, FP8 linear, rotary, attention,
    FP8 linear one by one; the same quantisation points, so the same values."""
    torch.manual_seed(0)
    h, n, m, d, b, s = 256, 4, 2, 64, 2, 12

    class Parts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            from msamp.models.gpt import LayerNorm
            self.ln, self.qkv, self.proj = LayerNorm(h), torch.nn.Linear(h, (n + 2 * m) * d), torch.nn.Linear(h, h)

    parts = LinearReplacer.replace(Parts())
    x = torch.randn(b * s, h)
    freqs, lengths = K.rotary_frequencies(d), torch.tensor([12, 5])
    results = []
    for fused in (True, False):
        torch.manual_seed(1)
        for meta in (parts.qkv, parts.proj):
            for v in meta.scaling_metas.values():
                v.amax.zero_()
                v.scale.fill_(1.0)
            meta.weight.grad = None
        leaf = x.clone().requires_grad_(True)
        if fused:
            y = FL.attention_sublayer(leaf, parts.ln, parts.qkv, parts.proj, b, s, n, n_kv_head=m, rope=(freqs, None, False), lengths=lengths)
        else:
            q, k, v = parts.qkv(parts.ln(leaf)).view(b, s, -1, d).split([n, m, m], 2)
            q, k = K.rotary(q, k, freqs)
            y = leaf + parts.proj(K.attention(q, k, v, lengths=lengths).view(b * s, -1))
        y.backward(torch.randn(b * s, h))
        results.append((y.detach(), leaf.grad, parts.ln.weight.grad.clone(), parts.qkv.bias.grad.clone(), parts.proj.weight.grad.float()))
        parts.zero_grad()
    for a, c in zip(*results):
        # a 32-bit sum in another order can move a value across a rounding border of e4m3 / e5m2 (a step of 2^-3 of it): rare, so small in norm
        assert (a - c).norm() <= 1e-2 * c.norm()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('ffn', [512, 528])
def test_mlp_sublayer_with_delayed_scales(device, ffn):
    """Past the warm-up the fc1 GEMM writes the blocks and no h at all (rows of whole blocks), or a pass over h does: the same bytes, so
    the same gradients."""
    from msamp.nn import model_state
    torch.manual_seed(0)
    dt = torch.bfloat16 if device == 'cuda' else torch.float32

    class Parts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            from msamp.models.gpt import LayerNorm
            self.ln, self.fc1, self.fc2 = LayerNorm(128), torch.nn.Linear(128, ffn), torch.nn.Linear(ffn, 128)

    parts = LinearReplacer.replace(Parts().to(device))
    x, dy = torch.randn(40, 128, device=device).to(dt), torch.randn(40, 128, device=device).to(dt)
    for lin in (parts.fc1, parts.fc2):    # any scale that was found before
        for name, meta in lin.scaling_metas.items():
            meta.amax_counter.fill_(10**6) if isinstance(meta.amax_counter, torch.Tensor) else setattr(meta, 'amax_counter', 10**6)
            meta.scale.fill_(8.0)
    assert not parts.fc2.scaling_metas['input'].is_in_time_scaling()
    kept = []
    leaf = x.clone().requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = FL.mlp_sublayer(leaf, parts.ln, parts.fc1, parts.fc2, keep_fp8=True)
    assert not any(t.shape == (40, ffn) and t.dtype == dt for t in kept)
    y.backward(dy)
    plain = x.clone().requires_grad_(True)
    z = FL.mlp_sublayer(plain, parts.ln, parts.fc1, parts.fc2)
    z.backward(dy)
    assert torch.equal(y, z)
    a, c = plain.grad.float(), leaf.grad.float()
    assert 0 < (a - c).norm() <= 0.16 * a.norm()
    model_state.clear()


@pytest.mark.parametrize('device', CPU_GPU)
def test_mlp_sublayer_keeps_the_gelu_input_in_8_bits(device):
    torch.manual_seed(0)
    dt = torch.bfloat16 if device == 'cuda' else torch.float32

    class Parts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            from msamp.models.gpt import LayerNorm
            self.ln, self.fc1, self.fc2 = LayerNorm(128), torch.nn.Linear(128, 512), torch.nn.Linear(512, 128)

    parts = LinearReplacer.replace(Parts().to(device))
    x, dy = torch.randn(40, 128, device=device).to(dt), torch.randn(40, 128, device=device).to(dt)
    seen, out = {}, {}
    for keep in (False, True):
        leaf, kept = x.clone().requires_grad_(True), []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
            y = FL.mlp_sublayer(leaf, parts.ln, parts.fc1, parts.fc2, keep_fp8=keep)
        y.backward(dy)
        seen[keep], out[keep] = sum(t.numel() * t.element_size() for t in kept), (y.detach(), leaf.grad)
    assert torch.equal(out[False][0], out[True][0])
    n = 40 * 512
    assert seen[False] - seen[True] == n * dt.itemsize - n - n // 32
    # the slope of GeLU moves by at most its second derivative (0.8) times 2^-4 of an input of order one, e = 0.05; a gradient moved by e
    # crosses a border of e5m2 (steps of up to 1/4) with probability 4 e and then moves by a step: sqrt(e / 4) + e of the norm at most
    a, c = out[False][1].float(), out[True][1].float()
    assert 0 < (a - c).norm() <= 0.16 * a.norm()


def test_options_refused():
    with pytest.raises(ValueError):
        GPT(_config(n_kv_head=3))
    with pytest.raises(ValueError):
        GPT(_config(recompute='fp4'))
    with pytest.raises(ValueError):
        GPT(_config(rotary_dim=33))
    with pytest.raises(ValueError):
        _model('cpu')(torch.zeros(1, 4, dtype=torch.int64), positions=torch.arange(4))


@pytest.mark.parametrize('fp8', [False, True])
def test_positions_refused(fp8):
    model = _model('cpu', **LONG)
    model = LinearReplacer.replace(model) if fp8 else model
    for positions in (torch.arange(5), torch.arange(4, device='meta'), torch.zeros(2, 4, dtype=torch.int64)):
        with pytest.raises(ValueError):
            model(torch.zeros(1, 4, dtype=torch.int64), positions=positions)
    with pytest.raises(TypeError):
        model(torch.zeros(1, 4, dtype=torch.int64), positions=torch.arange(4.0))


# (on the CPU an unfused block has made its mask of the lengths in the forward pass: its gradients stay right)
@pytest.mark.parametrize('device,fp8,which', [('cpu', False, 'positions'), ('cpu', True, 'positions'), ('cpu', True, 'lengths')] +
                         [pytest.param('cuda', fp8, which, marks=pytest.mark.gpu) for fp8 in (False, True) for which in ('positions', 'lengths')])
def test_changed_before_the_backward_pass(device, fp8, which):
    """Gradients need the positions and lengths of the forward pass: overwritten ones are an error, not other gradients."""
    model = _model(device, **LONG)
    model = LinearReplacer.replace(model) if fp8 else model.to(model.act_dtype)
    tokens, labels, lengths = _batch(device)
    given = dict(lengths=lengths.int(), positions=torch.arange(24, device=device))
    loss = model(tokens, labels, **given)
    given[which] += 1
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_parameters_and_defaults():
    for kw in ({}, LONG, dict(n_kv_head=1), dict(rotary_dim=64)):
        model = GPT(_config(**kw))
        assert sum(p.numel() for p in model.parameters()) == model.cfg.num_params()
    plain = GPT(_config())
    assert 'wpe.weight' in plain.state_dict() and plain.cfg.kv_heads == 4 and not any('freq' in n for n in plain.state_dict())
    assert GPT(_config(rotary_dim=32)).bfloat16()._freqs.dtype == torch.float64


def test_block_casts_are_in_the_public_module():
    assert cast.cast_blocks_to_fp8(torch.zeros(3))[1].tolist() == [127]


@pytest.mark.parametrize('recompute', [None, 0, 1, 2, [], [3], ''])
def test_recompute_goes_by_its_truth(recompute):
    """Any value but a string other than 'fp8', as before there was one."""
    from unittest import mock
    model = _model('cpu', recompute=recompute)
    with mock.patch('torch.utils.checkpoint.checkpoint', side_effect=torch.utils.checkpoint.checkpoint) as again, \
            mock.patch('msamp.models.gpt.checkpoint_fp8') as fp8:
        model(*_batch('cpu')[:2]).backward()
    assert again.called == bool(recompute) and not fp8.called


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('first', ['inference', 'meta'])
def test_frequencies_of_the_model_serve_every_mode(device, first):
    """A model whose first call, or whose construction, was under another mode or default device trains."""
    if first == 'meta':
        with torch.device('meta'):
            model = GPT(_config(**LONG), act_dtype=torch.float32)
        assert model._freqs.device.type == 'cpu'
        return
    model = GPT(_config(**LONG), device='cpu', act_dtype=torch.bfloat16 if device == 'cuda' else torch.float32).to(device)
    model = model.to(model.act_dtype)
    tokens, labels, _ = _batch(device)
    with torch.inference_mode():
        model(tokens)
    assert not model._freqs.is_inference()
    model(tokens, labels).backward()


@pytest.mark.parametrize('device', CPU_GPU)
@pytest.mark.parametrize('ffn', [512, 528])
@pytest.mark.parametrize('delayed', [False, True])
def test_mlp_sublayer_keeps_the_blocks_of_its_gelu_input(device, ffn, delayed):
    """The kept bytes are those of a cast of the GeLU input that the sublayer without blocks keeps, and the input's gradient is bit for bit the one that this
    sublayer gives when its kept GeLU input is replaced by what the bytes stand for."""
    torch.manual_seed(0)
    dt = torch.bfloat16 if device == 'cuda' else torch.float32

    class Parts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            from msamp.models.gpt import LayerNorm
            self.ln, self.fc1, self.fc2 = LayerNorm(128), torch.nn.Linear(128, ffn), torch.nn.Linear(ffn, 128)

    parts = LinearReplacer.replace(Parts().to(device))
    x, dy = (3 * torch.randn(40, 128, device=device)).to(dt), torch.randn(40, 128, device=device).to(dt)
    if delayed:
        for lin in (parts.fc1, parts.fc2):
            for meta in lin.scaling_metas.values():
                meta.amax_counter.fill_(10**6) if isinstance(meta.amax_counter, torch.Tensor) else setattr(meta, 'amax_counter', 10**6)
                meta.scale.fill_(8.0)
    assert parts.fc2.scaling_metas['input'].is_in_time_scaling() != delayed

    def run(keep, unpack):
        leaf, kept = x.clone().requires_grad_(True), []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, unpack):
            y = FL.mlp_sublayer(leaf, parts.ln, parts.fc1, parts.fc2, keep_fp8=keep)
        y.backward(dy)
        return leaf.grad, kept

    got, kept = run(True, lambda t: t)
    exps = [t for t in kept if t.dtype == torch.uint8 and t.shape == (40 * ffn // 32, )]
    assert len(exps) == 1
    replaced = []

    def unpack(t):
        if t.shape == (40, ffn) and t.dtype == dt:    # the GeLU input
            codes, e = cast.cast_blocks_to_fp8(t)
            assert torch.equal(e, exps[0]) and any(k.shape == (40, ffn) and k.dtype == torch.uint8 and torch.equal(k, codes) for k in kept)
            replaced.append(t)
            return cast.cast_blocks_from_fp8(codes, e, dt)
        return t

    want, _ = run(False, unpack)
    assert len(replaced) == 1 and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize('d, n, m, interleaved, lengths, seq', [(64, 4, 2, False, (150, 5, 0), 150), (64, 4, 4, True, (140, 129, 128), 150),
                                                                (128, 4, 1, True, None, 200), (64, 6, 2, False, None, 40)])
def test_fused_attention_sublayer_on_cuda_computes_what_the_separate_calls_compute(d, n, m, interleaved, lengths, seq):
    """The rotation in place on the packed projection and on its packed gradient, and the attention on its strided views, against LayerNorm,
    FP8 linear, rotary, attention, FP8 linear one by one.  All of them see the same bytes on both ways, so the weight gradients are equal bit for bit;
    sums over the rows are in 32 bits in any order (fewer than 2^10 terms: 2^-14 of the sum of their sizes, far less in norm).  The fused
    forms add the residual, or its gradient, before the rounding to bf16 and the separate ones after it as well: with u = 2^-8 and r the residual,
    the sum s and the other term t = s - r the two differ by at most u |t| + 2 u |s| <= u (3 |s| + |r|)."""
    torch.manual_seed(0)
    h, b = n * d, 3

    class Parts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            from msamp.models.gpt import LayerNorm
            self.ln, self.qkv, self.proj = LayerNorm(h), torch.nn.Linear(h, (n + 2 * m) * d), torch.nn.Linear(h, h)

    parts = LinearReplacer.replace(Parts().cuda())
    x, dy = (torch.randn(b * seq, h, device='cuda').bfloat16() for _ in range(2))
    freqs = K.rotary_frequencies(d // 2, device='cuda')
    at = torch.randint(0, 10000, (b, seq), device='cuda')
    lens = None if lengths is None else torch.tensor(lengths, device='cuda')
    results = []
    for fused in (True, False):
        for lin in (parts.qkv, parts.proj):
            for meta in lin.scaling_metas.values():
                meta.amax.zero_()
                meta.scale.fill_(1.0)
            lin.weight.grad = None
        parts.zero_grad()
        leaf = x.clone().requires_grad_(True)
        if fused:
            y = FL.attention_sublayer(leaf, parts.ln, parts.qkv, parts.proj, b, seq, n, n_kv_head=m, rope=(freqs, at, interleaved), lengths=lens)
        else:
            q, k, v = parts.qkv(parts.ln(leaf)).view(b, seq, -1, d).split([n, m, m], 2)
            q, k = K.rotary(q, k, freqs, positions=at, interleaved=interleaved)
            y = leaf + parts.proj(K.attention(q, k, v, lengths=lens).view(b * seq, -1))
        y.backward(dy)
        results.append((y.detach().float(), leaf.grad.float(), parts.qkv.weight.grad.float(), parts.proj.weight.grad.float(), parts.qkv.bias.grad.float(),
                        parts.ln.weight.grad.float()))
    (y, dx, *sums), (y2, dx2, *sums2) = results
    u = 2.0**-8
    assert (y - y2).norm() <= u * (3 * y2.norm() + x.float().norm()) and (dx - dx2).norm() <= u * (3 * dx2.norm() + dy.float().norm())
    assert torch.equal(sums[0], sums2[0]) and torch.equal(sums[1], sums2[1])
    for a, c in zip(sums[2:], sums2[2:]):
        assert (a - c).norm() <= 2.0**-14 * c.norm()
    for a in results[0]:
        assert torch.isfinite(a).all() and a.abs().sum() > 0
    assert native.device_status() == 0
