"""Layer norm, token log probabilities and gradient clipping: the eager forms on
the CPU, the kernels on the GPU, both against 64-bit formulas, and what they refuse.

Tolerances are counted in roundings: u = 2**-24 is half a step of the 32-bit
sums, `half(t)` half a step of a stored type.  A sum over n terms taken one after
the other is off by at most n u times the sum of their magnitudes.
"""
import math

import pytest
import torch

from distar_amd.ops.grad_norm import clip_grad_norm, grad_norm
from distar_amd.ops.layer_norm import FusedLayerNorm, add_layer_norm, layer_norm
from distar_amd.ops.linear_act import LinearAct, linear_act
from distar_amd.ops.token_logprobs import token_logprobs
from distar_amd.utils.grad_clip import GradClip

U = 2.0 ** -24
DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, want, tol):
    """|got - want| <= tol + the rounding of the result to its type."""
    tol = tol + half(got.dtype) * want.abs() * 1.01 + torch.finfo(got.dtype).tiny
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((off <= tol).all()), (off / tol).max()


# ------------------------------------------------------------------ layer norm

def _ln_reference(s, w, b, eps, dy=None, ds=None):
    s, w, b = (t.double() for t in (s, w, b))
    mean, var = s.mean(-1, keepdim=True), s.var(-1, unbiased=False, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (s - mean) * r
    out = {'y': h * w + b, 'h': h, 'r': r}
    if dy is not None:
        g = dy.double() * w
        out['dx'] = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        if ds is not None:
            out['dx'] = out['dx'] + ds.double()
        flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
        out['dw'], out['db'] = flat(dy.double() * h).sum(0), flat(dy.double()).sum(0)
        out['dw_abs'] = flat((dy.double() * h).abs()).sum(0)
        out['db_abs'] = flat(dy.double().abs()).sum(0)
    return out


def _ln_check(x, r, w, b, dy, ds, eps=1e-5):
    leaves = [t.clone().requires_grad_() if t is not None else None for t in (x, r, w, b)]
    if r is None:
        y, s = layer_norm(leaves[0], leaves[2], leaves[3], eps), x
        grads = torch.autograd.grad(y, [leaves[0], leaves[2], leaves[3]], dy)
    else:
        y, s = add_layer_norm(*leaves, eps)
        assert torch.equal(s, x + r)
        grads = torch.autograd.grad([y, s], leaves, [dy, ds])
        assert torch.equal(grads[0], grads[1])
        grads = grads[1:]
    ref = _ln_reference(s.detach(), w, b, eps, dy, ds)
    # a mean over C values by lanes and a tree, the difference, 1/sqrt, two products
    n = 32 + x.shape[-1] / 64
    top, wmax = (s.detach().double().abs() * ref['r']).amax(-1, keepdim=True), w.double().abs().max()
    near(y, ref['y'], n * U * (top * wmax * 2 + b.double().abs().max()))
    g = (dy.double() * w.double()).abs().amax(-1, keepdim=True)
    tol = n * U * 4 * ref['r'] * g * (1 + top * top)
    if r is not None and x.device.type == 'cpu':
        # autograd adds the two gradients of the stream after rounding each to its type
        tol = tol + half(x.dtype) * ((ref['dx'] - ds.double()).abs() + ds.double().abs()) * 1.01
    near(grads[0], ref['dx'], tol)
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    hmax = top.max() if top.numel() else 0.
    near(grads[1], ref['dw'], (n + rows) * U * (ref['dw_abs'] + 2 * hmax * ref['db_abs']))
    near(grads[2], ref['db'], (n + rows) * U * ref['db_abs'])
    with torch.no_grad():
        again = layer_norm(x, w, b, eps) if r is None else add_layer_norm(x, r, w, b, eps)[0]
    assert torch.equal(again, y.detach())
    return y, grads


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 2), (5, 7), (33, 64), (70, 65), (129, 256),
                                        (40, 257), (9, 1000), (301, 997), (7, 2049), (3, 5001),
                                        (2, 16383), (3, 16390), (5, 20001)])
def test_layer_norm(device, dtype, rows, width):
    gen = torch.Generator().manual_seed(rows * 31 + width)
    make = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, r, dy, ds = ((make(rows, width) * 2 + 0.5).to(device, dtype) for _ in range(4))
    for residual in (False, True):
        for wdtype in {dtype, torch.float32}:
            w, b = (1 + 0.2 * make(width)).to(device, wdtype), make(width).to(device, wdtype)
            _ln_check(x, r if residual else None, w, b, dy, ds if residual else None)


@pytest.mark.parametrize('device', DEVICES)
def test_layer_norm_far_mean_constant_rows_and_leading_shape(device):
    x = torch.randn(2, 3, 4, 320) + 1000.
    x[0, 1] = 7.
    dy, w, b = torch.randn(2, 3, 4, 320), torch.randn(320), torch.randn(320)
    _ln_check(*(t.to(device) if t is not None else None for t in (x, None, w, b, dy, None)))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
def test_layer_norm_strided_rows(device, dtype):
    big = torch.randn(12, 6, 300).to(device, dtype)
    w, b = torch.randn(96).to(device), torch.randn(96).to(device)
    for x in (big[:, :, 5:101], big[:, 2, 1:97], big[1, 0, 3:99], big.transpose(0, 1)[..., :96],
              big[..., ::3][..., :96], big[:, :1, :96].expand(12, 6, 96)):
        dy = torch.randn(x.shape).to(device, dtype)
        want = layer_norm(x.contiguous(), w, b)
        assert torch.equal(layer_norm(x, w, b), want)
        leaf = x.detach().requires_grad_()
        got, = torch.autograd.grad(layer_norm(leaf, w, b), leaf, dy[:1].expand(x.shape))
        plain = x.contiguous().requires_grad_()
        ref, = torch.autograd.grad(layer_norm(plain, w, b), plain, dy[:1].expand(x.shape).contiguous())
        assert torch.equal(got, ref)


@pytest.mark.parametrize('device', DEVICES)
def test_layer_norm_empty_partial_gradients_and_module(device):
    w, b = torch.randn(8, device=device, requires_grad=True), torch.randn(8, device=device, requires_grad=True)
    x = torch.zeros(0, 8, device=device, requires_grad=True)
    y = layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
    assert gx.shape == (0, 8) and not gw.any() and not gb.any()
    x = torch.randn(5, 8, device=device, requires_grad=True)
    r = torch.randn(5, 8, device=device)
    torch.testing.assert_close(layer_norm(x), torch.nn.functional.layer_norm(x, (8,)))
    for weight, bias in ((w, None), (None, b)):
        got = torch.autograd.grad(layer_norm(x, weight, bias).square().sum(), [x, w if weight is not None else b])
        ref = torch.autograd.grad(torch.nn.functional.layer_norm(x, (8,), weight, bias).square().sum(),
                                  [x, w if weight is not None else b])
        torch.testing.assert_close(got, ref, rtol=1e-4, atol=1e-4)
    y, s = add_layer_norm(x, r, w, b)                       # the stream alone
    torch.testing.assert_close(torch.autograd.grad(s.sum(), x)[0], torch.ones_like(x))
    module, plain = FusedLayerNorm(8).to(device), torch.nn.LayerNorm(8).to(device)
    module.load_state_dict(plain.state_dict())
    torch.testing.assert_close(module(x), plain(x), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(module(x, r)[0], plain(x + r), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize('device', DEVICES)
def test_layer_norm_refusals(device):
    x = torch.randn(4, 8, device=device)
    w = torch.ones(8, device=device)
    with pytest.raises(ValueError):
        layer_norm(x, w[:7])
    with pytest.raises(ValueError):
        layer_norm(x, w, eps=-1.)
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(4, 0, device=device))
    with pytest.raises(ValueError):
        layer_norm(x[0, 0])
    with pytest.raises(TypeError):
        layer_norm(x.long())
    with pytest.raises(ValueError):
        add_layer_norm(x, x[:1])
    with pytest.raises(TypeError):
        add_layer_norm(x, x.bfloat16())
    with pytest.raises(ValueError):
        FusedLayerNorm((4, 8))
    if device == 'cuda':
        with pytest.raises(TypeError):
            layer_norm(x.double())
        with pytest.raises(TypeError):
            layer_norm(x, w, w.bfloat16())
        with pytest.raises(TypeError):
            layer_norm(x.bfloat16(), w.half())
        with pytest.raises(ValueError):
            layer_norm(x, w.cpu())


def test_formulas_against_differences():
    gen = torch.Generator().manual_seed(3)
    x, r = (torch.randn(3, 6, generator=gen, dtype=torch.float64).requires_grad_() for _ in range(2))
    w, b = (torch.randn(6, generator=gen, dtype=torch.float64).requires_grad_() for _ in range(2))
    assert torch.autograd.gradcheck(add_layer_norm, (x, r, w, b))
    tokens = torch.tensor([1, -100, 5])
    mask = torch.tensor([[1, 1, 0, 1, 0, 0], [0] * 6, [1] * 6]).bool()
    assert torch.autograd.gradcheck(
        lambda t: token_logprobs(t, tokens, mask=mask, temperature=0.7)[:2], (x,))


# ------------------------------------------------------- token log probabilities

def _lp_reference(logits, tokens, mask, temperature, top_k, ignore):
    raw = logits.double()
    ok = raw > -math.inf
    if mask is not None:
        ok = ok & mask
        raw = torch.where(mask, raw, -math.inf)
    some = ok.any(-1, keepdim=True)
    x = torch.where(ok, raw, 0.) / temperature
    logp = torch.where(ok, x - torch.where(ok, x, -math.inf).logsumexp(-1, keepdim=True), -math.inf)
    p = logp.exp()
    entropy = -torch.where(ok, p * torch.where(ok, logp, 0.), 0.).sum(-1)
    at = tokens.clamp(min=0).unsqueeze(-1)
    lp = torch.where(tokens == ignore, 0., logp.gather(-1, at).squeeze(-1))
    order = torch.sort(raw, dim=-1, descending=True, stable=True)[1][..., :top_k]
    tlp = logp.gather(-1, order)
    return {'lp': lp, 'h': entropy, 'tlp': tlp, 'tt': torch.where(tlp > -math.inf, order, -1),
            'p': p, 'logp': logp, 'ok': ok, 'some': some,
            'range': (torch.where(ok, x, -math.inf).amax(-1) - torch.where(ok, x, math.inf).amin(-1)).clamp(min=0)
            .nan_to_num(0., posinf=0.)}


def _lp_check(logits, tokens, mask, temperature=1.0, top_k=0, ignore=-100):
    ref = _lp_reference(logits, tokens, mask, temperature, top_k, ignore)
    leaf = logits.detach().requires_grad_()
    got = token_logprobs(leaf, tokens, mask=mask, temperature=temperature, top_k=top_k)
    # a logit's distance to the maximum is exact but for 2 roundings of up to
    # `range`; exp, the sums and log add their own
    off = U * (64 + 8 * ref['range'])
    finite = ref['lp'] > -math.inf
    assert torch.equal(finite, got.logprob > -math.inf)
    near(got.logprob[finite], ref['lp'][finite], off[finite])
    near(got.entropy, ref['h'], off * (1 + ref['h']))
    if top_k:
        assert torch.equal(got.top_tokens, ref['tt'])
        there = ref['tt'] >= 0
        assert bool((got.top_logprobs[~there] == -math.inf).all())
        near(got.top_logprobs[there], ref['tlp'][there], off.unsqueeze(-1).expand_as(ref['tlp'])[there])
    gen = torch.Generator().manual_seed(9)
    a, b = (torch.randn(tokens.shape, generator=gen).to(logits.device) for _ in range(2))
    d, = torch.autograd.grad([got.logprob, got.entropy], leaf, [a, b])
    a, b = a.double().unsqueeze(-1), b.double().unsqueeze(-1)
    g = torch.where((tokens == ignore).unsqueeze(-1), 0., a)
    one = torch.zeros_like(ref['p']).scatter_(-1, tokens.clamp(min=0).unsqueeze(-1), 1.)
    logp = torch.where(ref['ok'], ref['logp'], 0.)
    h = ref['h'].unsqueeze(-1)
    want = (g * (one - ref['p']) - b * ref['p'] * (logp + h)) / temperature
    inside = torch.ones_like(ref['ok']) if mask is None else mask.expand(logits.shape)
    want = torch.where(ref['some'] & inside, want, 0.)
    near(d, want, off.unsqueeze(-1) * 4 / temperature * (g.abs() + b.abs() * (1 + h)))
    with torch.no_grad():
        again = token_logprobs(logits, tokens, mask=mask, temperature=temperature, top_k=top_k)
    for x, y in zip(got, again):
        assert x is None and y is None or torch.equal(x, y)
    return got


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width,top_k', [(1, 1, 1), (3, 2, 2), (5, 7, 9), (16, 327, 5), (67, 513, 0),
                                              (9, 1000, 64), (33, 1025, 3), (3, 4097, 20), (2, 24320, 5),
                                              (2, 33001, 32), (2, 70001, 7)])
def test_token_logprobs(device, dtype, rows, width, top_k):
    gen = torch.Generator().manual_seed(rows + width)
    logits = (torch.randn(rows, width, generator=gen) * 3).to(device, dtype)
    tokens = torch.randint(0, width, (rows,), generator=gen).to(device)
    _lp_check(logits, tokens, None, 1.0, top_k)
    # ragged lengths with one empty row and one row of a single token; what is
    # masked holds the type's lowest value, infinities and NaN
    lengths = torch.randint(1, width + 1, (rows,), generator=gen)
    lengths[rows // 2], lengths[0] = 0, 1
    mask = (torch.arange(width) < lengths.unsqueeze(1)).to(device)
    tokens = (torch.rand(rows, generator=gen) * lengths).long().to(device)
    tokens[rows // 2] = -100
    fill = torch.tensor([torch.finfo(dtype).min, math.inf, -math.inf, math.nan], device=device).to(dtype)
    junk = fill[torch.randint(0, 4, (rows, width), generator=gen).to(device)]
    _lp_check(torch.where(mask, logits, junk), tokens, mask, 0.7, top_k)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [40, 300, 3000, 40000])
def test_token_logprobs_ties_and_infinities(device, dtype, width):
    gen = torch.Generator().manual_seed(width)
    tokens = torch.zeros(4, dtype=torch.long, device=device)
    same = torch.full((4, width), 1.5).to(device, dtype)
    got = _lp_check(same, tokens, None, 1.0, 33)
    assert torch.equal(got.top_tokens, torch.arange(33, device=device).expand(4, 33))
    few = torch.randint(-2, 3, (4, width), generator=gen).to(device, dtype)
    _lp_check(few, tokens, None, 1.3, 64)
    holes = few.clone()
    holes[:, ::2] = -math.inf
    holes[1] = -math.inf                                    # a row with nothing
    holes[2, 5:] = -math.inf                                # fewer than top_k
    _lp_check(holes, tokens + 1, None, 1.0, 8)
    low = torch.full((4, width), torch.finfo(dtype).min, dtype=dtype, device=device)
    low[:, 3] = 0.
    got = token_logprobs(low, tokens + 3, top_k=2)
    assert torch.equal(got.logprob, torch.zeros(4, device=device))
    assert got.top_tokens[0].tolist() == [3, 0]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('width', [40, 3000, 40000])
def test_token_logprobs_bad_rows_and_tokens(device, width):
    logits = torch.randn(5, width, device=device)
    logits[1, width - 1] = math.nan
    logits[2, 7] = math.inf
    tokens = torch.tensor([0, 0, 0, width, -1], device=device)
    leaf = logits.requires_grad_()
    got = token_logprobs(leaf, tokens, top_k=3)
    assert torch.isnan(got.logprob).tolist() == [False, True, True, True, True]
    assert torch.isnan(got.entropy).tolist() == [False, True, True, False, False]
    assert got.top_tokens[1].tolist() == got.top_tokens[2].tolist() == [-1] * 3
    assert bool(torch.isnan(got.top_logprobs[1:3]).all())
    d, = torch.autograd.grad(got.logprob[0], leaf)
    assert bool(torch.isfinite(d[0]).all()) and d[0].abs().sum() > 0


@pytest.mark.parametrize('device', DEVICES)
def test_token_logprobs_shapes_masks_and_strides(device):
    gen = torch.Generator().manual_seed(4)
    big = torch.randn(3, 4, 50, generator=gen).to(device)
    logits, tokens = big[:, :, 3:40], torch.randint(0, 37, (3, 4), generator=gen).to(device)
    for shape in ((37,), (1, 1, 37), (3, 1, 37), (1, 4, 37), (3, 4, 37)):
        mask = (torch.rand(shape, generator=gen) < 0.6).to(device)
        _lp_check(logits, tokens, mask, 1.0, 4)
    _lp_check(big.transpose(0, 1)[..., :37], tokens.t(), None, 1.0, 4)
    _lp_check(big[..., ::2], tokens.clamp(max=24), None, 1.0, 4)
    _lp_check(big[0, 0], torch.tensor(7, device=device), None, 1.0, 4)
    got = token_logprobs(torch.zeros(0, 9, device=device, requires_grad=True),
                         torch.zeros(0, dtype=torch.long, device=device), top_k=3)
    assert got.logprob.shape == (0,) and got.top_tokens.shape == (0, 3)
    leaf = big.clone().requires_grad_()
    lp, h = token_logprobs(leaf, torch.zeros(3, 4, dtype=torch.int32, device=device))[:2]
    both, = torch.autograd.grad(lp.sum() + h.sum(), leaf, retain_graph=True)
    one, = torch.autograd.grad(lp.sum(), leaf, retain_graph=True)
    two, = torch.autograd.grad(h.sum(), leaf)
    torch.testing.assert_close(both, one + two, rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize('device', DEVICES)
def test_token_logprobs_refusals(device):
    logits, tokens = torch.randn(4, 9, device=device), torch.zeros(4, dtype=torch.long, device=device)
    for bad in (dict(top_k=-1), dict(top_k=65), dict(temperature=0.), dict(temperature=math.nan),
                dict(mask=torch.ones(4, 8, device=device).bool())):
        with pytest.raises(ValueError):
            token_logprobs(logits, tokens, **bad)
    with pytest.raises(ValueError):
        token_logprobs(logits, tokens[:3])
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(4, 0, device=device), tokens)
    with pytest.raises(TypeError):
        token_logprobs(logits, tokens.float())
    with pytest.raises(TypeError):
        token_logprobs(logits, tokens, mask=torch.ones(4, 9, device=device))
    with pytest.raises(TypeError):
        token_logprobs(logits.long(), tokens)
    if device == 'cuda':
        with pytest.raises(TypeError):
            token_logprobs(logits.double(), tokens)
        with pytest.raises(ValueError):
            token_logprobs(logits, tokens.cpu())


# ------------------------------------------------------------- gradient clipping

def _grads(device, gen, types, sizes=(1, 3, 1000, 0, 70001, 16385, 256)):
    flat = torch.randn(sum(sizes) + 5, generator=gen)
    out, at = [], 0
    for i, n in enumerate(sizes):
        t = types[i % len(types)]
        out.append(flat[at:at + n].to(device, t))
        at += n
    buffer = torch.randn(999, generator=gen).to(device)
    out += [buffer[1:8], buffer[8:501], buffer[501:900].view(19, 21).t()]     # views, one of them transposed
    out.append(torch.randn((), generator=gen).to(device))
    out.append(torch.randn(6, 5, 4, 3, generator=gen).to(device, types[-1]).contiguous(memory_format=torch.channels_last))
    return out


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('norm_type', [1, 2, 2.0, math.inf])
@pytest.mark.parametrize('types', [TYPES[:1], TYPES[1:2], TYPES])
def test_clip_grad_norm(device, norm_type, types):
    gen = torch.Generator().manual_seed(1)
    grads = _grads(device, gen, types)
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    want = torch.linalg.vector_norm(flat, float(norm_type))
    # 64-bit sums, one rounding of the norm
    near(grad_norm(grads, norm_type), want, 2 * U * want)
    for max_norm in (1e9, float(want) * 0.37, 0.):
        scale = min(1., max_norm / (float(want) + 1e-6))
        copies = [g.clone(memory_format=torch.preserve_format) for g in grads]
        norm = clip_grad_norm(copies, max_norm, norm_type)
        near(norm, want, 2 * U * want)
        for c, g in zip(copies, grads):
            near(c, g.double() * scale, 8 * U * g.double().abs() * scale)
            assert scale < 1 or torch.equal(c, g)
        out = [torch.full_like(g, math.nan, dtype=torch.float32) for g in grads]
        out[2] = out[2].bfloat16()
        keep = [g.clone() for g in grads]
        assert torch.equal(clip_grad_norm(grads, max_norm, norm_type, out=out), norm)
        for o, g, k in zip(out, grads, keep):
            near(o, g.double() * scale, 8 * U * g.double().abs() * scale)
            assert torch.equal(g, k)


@pytest.mark.parametrize('device', DEVICES)
def test_clip_grad_norm_many_strided_and_neighbours(device):
    gen = torch.Generator().manual_seed(2)
    sizes = [1 + (37 * i) % 400 for i in range(700)]
    flat = torch.randn(sum(sizes) + 700, generator=gen).to(device)
    grads, at = [], 0
    for n in sizes:                                          # one element between neighbours
        grads.append(flat[at:at + n])
        at += n + 1
    before, want = flat.clone(), torch.linalg.vector_norm(torch.cat(grads).double())
    near(clip_grad_norm(grads, 1.0), want, 2 * U * want)
    scale = 1 / (float(want) + 1e-6)
    gaps = torch.ones_like(flat, dtype=torch.bool)
    at = 0
    for n in sizes:
        gaps[at:at + n] = False
        at += n + 1
    assert torch.equal(flat[gaps], before[gaps])
    near(flat[~gaps], before[~gaps].double() * scale, 8 * U * before[~gaps].double().abs() * scale)
    wide = torch.randn(40, 30, generator=gen).to(device)
    kept = wide.clone()
    part = wide[:, 3:17:2]
    want = torch.linalg.vector_norm(part.double())
    near(clip_grad_norm([part], 0.5), want, 2 * U * want)
    near(part, kept[:, 3:17:2].double() * (0.5 / (float(want) + 1e-6)), 8 * U * kept[:, 3:17:2].double().abs())
    wide[:, 3:17:2] = kept[:, 3:17:2]
    assert torch.equal(wide, kept)
    out = torch.zeros(7, 40, device=device).t()              # another order than its input's
    clip_grad_norm([part], 1e9, out=[out])
    assert torch.equal(out, part)


@pytest.mark.parametrize('device', DEVICES)
def test_clip_grad_norm_bucket_views(device):
    gen = torch.Generator().manual_seed(3)
    sizes = [1, 7, 300, 0, 8192, 5, 16385, 40000]
    bucket = torch.randn(sum(sizes), generator=gen).to(device, torch.bfloat16)
    out = torch.full((sum(sizes),), math.nan, device=device)
    want = torch.linalg.vector_norm(bucket.double())
    scale = 0.5 / (float(want) + 1e-6)
    for order in (list(range(8)), [3, 1, 0, 2, 7, 6, 5, 4]):   # in memory's order, and not
        grads, outs = ([list(t.split(sizes))[i] for i in order] for t in (bucket, out))
        near(clip_grad_norm(grads, 0.5, out=outs), want, 2 * U * want)
        near(out, bucket.double() * scale, 8 * U * bucket.double().abs() * scale)
    # neighbours on one side only, and another type between neighbours
    apart = [torch.empty(n, device=device) for n in sizes]
    clip_grad_norm(list(bucket.split(sizes)), 0.5, out=apart)
    assert torch.equal(torch.cat(apart), out)
    mixed = list(bucket.split(sizes))
    mixed[2] = mixed[2].float()
    clip_grad_norm(mixed, 0.5, out=apart)
    near(torch.cat(apart), bucket.double() * scale, 8 * U * bucket.double().abs() * scale)


@pytest.mark.parametrize('device', DEVICES)
def test_clip_grad_norm_extremes(device):
    big = [torch.full((1000,), 1e30, device=device), torch.full((3,), -1e37, device=device)]
    want = torch.linalg.vector_norm(torch.cat(big).double())
    near(clip_grad_norm(big, 1.0), want, 2 * U * want)
    assert bool(torch.isfinite(big[0]).all()) and big[1][0] < 0
    small = [torch.full((100,), 1e-30, device=device)]       # squares below the smallest 32-bit value
    near(grad_norm(small), torch.tensor(1e-29, dtype=torch.float64, device=device), 4 * U * 1e-29)
    for norm_type in (1, 2, math.inf):
        for value in (math.nan, math.inf):
            g = [torch.ones(300, device=device), torch.ones(5, device=device)]
            g[0][211] = value
            norm = clip_grad_norm(g, 1.0, norm_type)
            if math.isnan(value):
                assert torch.isnan(norm) and bool(torch.isnan(g[1]).all())
            else:
                assert norm == math.inf and not g[1].any() and torch.isnan(g[0][211])
    zero = [torch.zeros(10, device=device)]
    assert clip_grad_norm(zero, 1.0) == 0 and not zero[0].any()
    assert grad_norm([torch.zeros(0, device=device)]) == 0
    assert grad_norm(torch.full((4,), 2., device=device)) == 4


@pytest.mark.parametrize('device', DEVICES)
def test_clip_grad_norm_refusals(device):
    g = torch.ones(10, device=device)
    for bad in (lambda: grad_norm([]), lambda: grad_norm([g], 3), lambda: clip_grad_norm([g], -1.),
                lambda: clip_grad_norm([g], math.nan), lambda: clip_grad_norm([g], 1., eps=-1.),
                lambda: clip_grad_norm([g], 1., out=[g, g]), lambda: clip_grad_norm([g], 1., out=[g[:9]])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        grad_norm([g.long()])
    with pytest.raises(TypeError):
        clip_grad_norm([g], 1., out=[g.long()])
    if device == 'cuda':
        with pytest.raises(TypeError):
            grad_norm([g.double()])
        with pytest.raises(ValueError):
            grad_norm([g, g.cpu()])
        wide = torch.ones(6, 4, device=device)
        for bad in ([g, g], [g[:6], g[5:]], [g[5:], g[:6]], [wide[:, :2], wide[:, :2]]):
            with pytest.raises(ValueError):
                clip_grad_norm(bad, 1.)
        with pytest.raises(ValueError):
            clip_grad_norm([g[:5], g[5:]], 1., out=[g[5:], torch.empty(5, device=device)])
        with pytest.raises(ValueError):
            clip_grad_norm([torch.ones(3, device=device)], 1., out=[torch.zeros(1, device=device).expand(3)])
    assert torch.equal(g, torch.ones(10, device=device))


@pytest.mark.parametrize('device', DEVICES)
def test_grad_clip_global_norm_type(device):
    gen = torch.Generator().manual_seed(6)
    params = [torch.nn.Parameter(torch.zeros(n, device=device, dtype=t)) for n, t in ((40, torch.float32), (77, torch.bfloat16))]
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(device, p.dtype)
    want = torch.linalg.vector_norm(torch.cat([p.grad.double() for p in params]))
    kept = [p.grad.clone() for p in params]
    norm = GradClip('global_norm', threshold=1.0).apply(params)
    assert abs(norm - float(want)) <= 2 * U * float(want)
    for p, k in zip(params, kept):
        near(p.grad, k.double() / (float(want) + 1e-6), 8 * U * k.double().abs())
    assert GradClip('global_norm', threshold=1.0, norm_type=float('inf')).apply(params) <= 1.0
    assert GradClip('global_norm').apply([torch.nn.Parameter(torch.zeros(3))]) == 0.


# ------------------------------------------------------------------ linear layers

LOW = [torch.bfloat16, torch.float16]
SLOPE = {None: lambda z: torch.ones_like(z), 'relu': lambda z: (z > 0).double(),
         'gelu': lambda z: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
         'silu': lambda z: torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))}
ACT = {None: lambda z: z, 'relu': torch.relu, 'gelu': torch.nn.functional.gelu, 'silu': torch.nn.functional.silu}


def _linear_check(x, w, b, act, residual, dy):
    """Against 64 bits. A sum of K products is off by K u of their magnitudes; the
    slope is taken at the stored z (|act''| < 1), and dz is stored once."""
    flat = lambda t: t.double().reshape(-1, t.shape[-1])  # noqa: E731
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, w, b, residual)]
    y = linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3])
    grads = iter(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    t, k, rows = half(x.dtype), x.shape[-1], flat(x).shape[0]
    xd, wd, dyd = flat(x), w.to(x.dtype).double(), flat(dy)
    z = xd @ wd.t() + (0. if b is None else b.double())
    z_off = 2 * (k + 8) * U * (xd.abs() @ wd.abs().t() + (0. if b is None else b.double().abs()))
    want = ACT[act](z) + (0. if residual is None else flat(residual))
    near(y.reshape(z.shape), want, 1.2 * z_off + 16 * U * (z.abs() + want.abs()))
    dz = dyd * SLOPE[act](z)
    dz_off = dyd.abs() * 16 * U
    if act == 'relu':
        dz_off = dz_off + dyd.abs() * (z.abs() <= z_off + torch.finfo(x.dtype).tiny)
    elif act:
        dz_off = dz_off + dyd.abs() * (z_off + t * z.abs() * 1.01 + torch.finfo(x.dtype).tiny)
    db_off = dz_off
    if act:
        dz_off = dz_off + t * dz.abs() * 1.01 + torch.finfo(x.dtype).tiny
    if x.device.type == 'cpu':          # the eager form casts weights of another type there and back
        dz_off = dz_off + t * dz.abs()
    n = w.shape[0]
    near(next(grads).reshape(xd.shape), dz @ wd, dz_off @ wd.abs() + 2 * (n + 8) * U * (dz.abs() @ wd.abs()))
    dw = next(grads)
    assert dw.dtype == w.dtype
    dw_off = dz_off.t() @ xd.abs() + 2 * (rows + 8) * U * (dz.abs().t() @ xd.abs())
    if x.device.type == 'cpu':
        dw_off = dw_off + t * (dz.t() @ xd).abs()
    near(dw, dz.t() @ xd, dw_off)
    if b is not None:
        db = next(grads)
        assert db.dtype == b.dtype
        near(db, dz.sum(0), db_off.sum(0) + 2 * (rows + 8) * U * dz.abs().sum(0))
    if residual is not None:
        assert torch.equal(next(grads), dy)
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, act, residual), y)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', LOW)
@pytest.mark.parametrize('rows,k,n', [(1, 1, 1), (3, 5, 7), (1, 1024, 256), (16, 1024, 256), (17, 997, 33), (64, 64, 64),
                                      (65, 72, 129), (130, 997, 256), (300, 128, 260), (257, 264, 520), (1000, 8, 8),
                                      (2100, 40, 136), (129, 2056, 24)])
def test_linear_act(device, dtype, rows, k, n):
    gen = torch.Generator().manual_seed(rows + k + n)
    make = lambda *s: torch.randn(*s, generator=gen).to(device, dtype)  # noqa: E731
    x, w, b, dy, r = make(rows, k), (make(n, k) * k ** -0.5).to(dtype), make(n), make(rows, n), make(rows, n)
    for act in (None, 'relu', 'gelu', 'silu'):
        _linear_check(x, w, b, act, r if act in (None, 'gelu') or rows % 2 else None, dy)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', LOW)
@pytest.mark.parametrize('rows,k,n', [(2600, 72, 2568), (520, 2568, 2568), (2600, 2568, 40), (5000, 256, 1024),
                                      (3600, 1032, 3400), (3600, 3400, 1032), (4104, 2600, 2600)])
def test_linear_act_large(dtype, rows, k, n):
    gen = torch.Generator('cuda').manual_seed(rows + k + n)
    make = lambda *s: torch.randn(*s, generator=gen, device='cuda').to(dtype)  # noqa: E731
    x, w, b, dy, r = make(rows, k), (make(n, k) * k ** -0.5).to(dtype), make(n), make(rows, n), make(rows, n)
    _linear_check(x, w, b, 'gelu', r, dy)
    _linear_check(x, w, b, 'relu', None, dy)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', LOW)
def test_linear_act_strides_and_master_weights(device, dtype):
    gen = torch.Generator().manual_seed(5)
    make = lambda *s: torch.randn(*s, generator=gen).to(device, dtype)  # noqa: E731
    big, wide = make(4, 50, 300), make(90, 300)
    for lo, hi in ((0, 128), (8, 136), (3, 131), (1, 98)):
        x, w = big[..., lo:hi], wide[:, lo:hi] * (hi - lo) ** -0.5
        dy = make(4, 50, 90)
        _linear_check(x, w, make(90), 'relu', big[..., 5:95], dy)
        _linear_check(x, w.float(), make(90).float(), 'silu', None, dy[:1, :1].expand(4, 50, 90))
        _linear_check(x, w.float(), make(90), None, big[..., 5:95], make(90, 50, 4).transpose(0, 2))
    _linear_check(big.transpose(0, 1)[..., :64], wide.t()[:70, :64], None, 'gelu', None, make(50, 4, 70))
    _linear_check(big[0, 0], wide[:, :300], make(90), 'gelu', make(90), make(90))


@pytest.mark.parametrize('device', DEVICES)
def test_linear_act_needed_gradients_empty_and_module(device):
    dtype = torch.bfloat16
    x, w, b = (torch.randn(*s, device=device).to(dtype) for s in ((9, 16), (8, 16), (8,)))
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(linear_act(*full, 'gelu').float().sum(), full)
    for i in range(3):
        leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(linear_act(*leaves, 'gelu').float().sum(), leaves[i])
        assert torch.equal(got, want[i])
    none = torch.zeros(0, 16, device=device, dtype=dtype, requires_grad=True)
    y = linear_act(none, full[1], full[2], 'relu')
    got = torch.autograd.grad(y.float().sum(), [none, *full[1:]])
    assert y.shape == (0, 8) and got[0].shape == (0, 16) and not got[1].any() and not got[2].any()
    nan = x.clone()
    nan[4, 3] = math.nan
    for act in (None, 'relu', 'gelu', 'silu'):
        y = linear_act(nan, w, b, act)
        assert bool(torch.isnan(y[4]).all()) and bool(torch.isfinite(y[[0, 1, 2, 3, 5, 6, 7, 8]]).all())
    module = LinearAct(16, 8, activation='relu').to(device)
    module.load_state_dict(torch.nn.Linear(16, 8).state_dict())
    with torch.autocast(device, dtype=dtype):
        y = module(x.float(), x[:, :8].float())
    assert y.dtype == dtype
    y.float().sum().backward()
    assert module.weight.grad.dtype == torch.float32 and bool(torch.isfinite(module.weight.grad).all())


@pytest.mark.parametrize('device', DEVICES)
def test_linear_act_refusals(device):
    x, w = torch.randn(4, 8, device=device).bfloat16(), torch.randn(3, 8, device=device).bfloat16()
    for bad in (lambda: linear_act(x, w, activation='tanh'), lambda: linear_act(x[:, :7], w), lambda: linear_act(x, w[0]),
                lambda: linear_act(x, w, w[0]), lambda: linear_act(x, w, residual=x), lambda: linear_act(x[0, 0], w),
                lambda: linear_act(x, w[:0]), lambda: LinearAct(3, 4, activation='no')):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: linear_act(x, w.half()), lambda: linear_act(x.long(), w),
                lambda: linear_act(x, w, residual=torch.zeros(4, 3, device=device))):
        with pytest.raises(TypeError):
            bad()
    if device == 'cuda':
        with pytest.raises(TypeError):
            linear_act(x.float(), w.float())
        with pytest.raises(ValueError):
            linear_act(x, w.cpu())


# ------------------------------------------------------------------ together

def _block(p, x, tokens, mask, eager=None):
    """A pre-norm sublayer, its policy head and its loss."""
    ln, add_ln, lin = (layer_norm, add_layer_norm, linear_act) if eager is None else eager
    h = lin(ln(x, p['w1'], p['b1']), p['up'], p['ub'], 'gelu')
    y, s = add_ln(lin(h, p['down'], p['db'], 'relu', x), x, p['w2'], p['b2'])
    logits = lin(y, p['head'], p['hb'])
    lp, entropy = token_logprobs(logits, tokens, mask=mask)[:2]
    return -(lp.clamp(min=-50.).mean()) - 0.1 * entropy.mean() + 0.01 * s.float().square().mean()


def _block_inputs(device, dtype):
    gen = torch.Generator().manual_seed(8)
    make = lambda *s, scale=0.1: (torch.randn(*s, generator=gen) * scale).to(device, dtype)  # noqa: E731
    p = {'w1': 1 + make(96), 'b1': make(96), 'up': make(200, 96), 'ub': make(200), 'down': make(96, 200), 'db': make(96),
         'w2': 1 + make(96), 'b2': make(96), 'head': make(37, 96), 'hb': make(37)}
    x = make(6, 11, 96, scale=1.)
    tokens = torch.randint(0, 37, (6, 11), generator=gen)
    mask = torch.rand(6, 11, 37, generator=gen) < 0.8
    mask.scatter_(-1, tokens.unsqueeze(-1), True)
    mask[2, 3], tokens[2, 3], tokens[0, 0] = False, -100, -100
    return p, x, tokens.to(device), mask.to(device)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', LOW)
def test_block_step_together(dtype):
    p, x, tokens, mask = _block_inputs('cuda', dtype)
    p = {k: v.requires_grad_() for k, v in p.items()}
    got = torch.autograd.grad(_block(p, x, tokens, mask), list(p.values()))
    wide = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    ref = torch.autograd.grad(_block(wide, x.cpu().double(), tokens.cpu(), mask.cpu()), list(wide.values()))
    for g, r, name in zip(got, ref, p):
        # about ten stored values lie between the loss and a weight, each off by half
        # a step in independent directions, and the relu's flips are of their order
        off = torch.linalg.vector_norm(g.cpu().double() - r) / torch.linalg.vector_norm(r)
        assert off <= 16 * half(dtype), (name, float(off))
    master = [torch.empty_like(g, dtype=torch.float32) for g in got]
    norm = clip_grad_norm(got, 0.01, out=master)
    near(norm, torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in got])), 2 * U * norm.double())
    assert abs(float(grad_norm(master)) - 0.01) <= 1e-6


@pytest.mark.gpu
def test_block_step_in_graph_and_on_another_stream():
    def step(p, x, tokens, mask):
        leaves = {k: v.detach().requires_grad_() for k, v in p.items()}
        loss = _block(leaves, x, tokens, mask)
        grads = list(torch.autograd.grad(loss, list(leaves.values())))
        norm = clip_grad_norm(grads, 0.05)
        return [loss.detach(), norm, *grads]

    inputs = [_block_inputs('cuda', torch.bfloat16)]
    eager = step(*inputs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*inputs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(eager, other):
        assert torch.equal(a, b)
    p, x, tokens, mask = inputs[0]
    x = x.clone()
    graphs = []
    for _ in range(2):                              # two graphs with workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(p, x, tokens, mask)
        graphs.append((graph, out))
    for turn in range(4):
        x.copy_(torch.randn(x.shape, device='cuda'))
        want = step(p, x, tokens, mask)
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize('device', DEVICES)
def test_second_derivatives_are_refused_and_versions_kept(device):
    if device == 'cuda':
        x = torch.randn(4, 8, device=device, dtype=torch.bfloat16, requires_grad=True)
        w = torch.randn(8, 8, device=device, dtype=torch.bfloat16, requires_grad=True)
        tokens = torch.zeros(4, dtype=torch.long, device=device)
        for y in (layer_norm(x, w[0]), linear_act(x, w, None, 'gelu'), token_logprobs(x, tokens)[0]):
            g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
            with pytest.raises(RuntimeError):
                g.float().sum().backward()
    a = torch.randn(5, device=device, requires_grad=True)
    b = torch.randn(5, device=device)
    y = (a * b).sum()
    clip_grad_norm([b], 0.1)
    with pytest.raises(RuntimeError):
        y.backward()


# ------------------------------------------------------------------ in the framework

@pytest.mark.parametrize('device', DEVICES)
def test_transformer_on_block_operators(device):
    from distar_amd.models.nn.transformer import Transformer
    torch.manual_seed(0)
    args = dict(input_dim=48, head_dim=128, hidden_dim=160, output_dim=96, head_num=2, layer_num=2)
    plain, fused = Transformer(**args).to(device), Transformer(**args, fused=True).to(device)
    fused.load_state_dict(plain.state_dict())
    assert list(plain.state_dict()) == list(fused.state_dict())
    x = torch.randn(3, 20, 48, device=device)
    mask = torch.arange(20, device=device) < torch.tensor([[20], [7], [1]], device=device)
    dy = torch.randn(3, 20, 96, device=device)
    want = plain(x, mask)
    ref = torch.autograd.grad(want, list(plain.parameters()), dy)
    if device == 'cpu':
        got = fused(x, mask)
        off = 1e-5
    else:
        with torch.autocast('cuda', dtype=torch.bfloat16):
            got = fused(x, mask)
        assert got.dtype == torch.bfloat16
        off = 16 * half(torch.bfloat16)       # some twenty stored values on the way
    grads = torch.autograd.grad(got, list(fused.parameters()), dy.to(got.dtype))
    # A relu's input carries the noise n of about four stored values, 4 half steps of
    # its own size; of normal values the share 0.8 n lies that near to zero, and each of
    # those may change sides, which takes its whole gradient along: a relative error of
    # sqrt(0.8 n) for one relu, and of sqrt(5 * 0.8 n) for the five of this model.
    flips = math.sqrt(5 * 0.8 * 4 * half(got.dtype)) if device == 'cuda' else 0.
    for a, b, most in zip([got, *grads], [want, *ref], [off] + [off + flips] * len(grads)):
        a, b = a.double(), b.double()
        assert torch.linalg.vector_norm(a - b) <= most * torch.linalg.vector_norm(b) + 1e-6
    with pytest.raises(ValueError):
        Transformer(**args, fused=True, ln_type='post')
    with pytest.raises(ValueError):
        Transformer(**args, fused=True, dropout_ratio=0.1)


@pytest.mark.parametrize('device', DEVICES)
def test_rl_loss_with_fused_logprobs(device):
    from distar_amd.lib.fake_data import fake_rl_learner_data
    from distar_amd.losses import ReinforcementLoss
    from distar_amd.models import Model
    from distar_amd.utils.config import Config
    from distar_amd.utils.data import to_device
    torch.manual_seed(0)
    model = Model(Config({'common': {'type': 'train'}, 'model': {'enable_baselines': ['winloss']}}),
                  use_value_network=True).to(device)
    data = fake_rl_learner_data(batch_size=2, unroll_len=3, entity_num_range=(32, 48))
    for key in ('model_last_iter', 'aux_type'):
        data.pop(key)
    out = model.rl_learner_forward(**to_device(data, device))
    total, grads = [], []
    for fused in (False, True):
        loss = ReinforcementLoss(Config({'fused_logprobs': fused}), 'MP0')
        assert loss.fused_logprobs is fused
        leaves = {k: v.detach().requires_grad_() for k, v in out['target_logit'].items()}
        values = {k: v.detach().clone() for k, v in out['value'].items()}
        total.append(loss.compute_loss({**out, 'target_logit': leaves, 'value': values})['total_loss'])
        grads.append(torch.autograd.grad(total[-1], list(leaves.values())))
    # the same quantities in 32 bits by two ways
    torch.testing.assert_close(total[0], total[1], rtol=1e-4, atol=1e-5)
    for a, b in zip(*grads):
        assert torch.linalg.vector_norm(a - b) <= 1e-4 * torch.linalg.vector_norm(a) + 1e-7


@pytest.mark.parametrize('device', DEVICES)
def test_inference_alternatives_and_fused_norm_blocks(device):
    from distar_amd.lib.fake_data import fake_sl_batch
    from distar_amd.models import Model
    from distar_amd.models.nn.blocks import ResFCBlock2, build_normalization
    from distar_amd.utils.config import Config
    from distar_amd.utils.data import to_device
    torch.manual_seed(0)
    model = Model(Config({'common': {'type': 'train'}})).to(device)
    data = to_device(fake_sl_batch(batch_size=2, traj_len=1, entity_num=32), device)
    hidden = [(torch.zeros(2, 384, device=device), torch.zeros(2, 384, device=device)) for _ in range(3)]
    obs = {k: data[k] for k in ('spatial_info', 'entity_info', 'scalar_info', 'entity_num')}
    with torch.no_grad():
        out = model.compute_logp_action(**obs, hidden_state=hidden, top_k=4)
    for head, (tokens, logp) in out['action_alternatives'].items():
        logit = out['logit'][head]
        k = min(4, logit.shape[-1])
        assert tokens.shape == (*logit.shape[:-1], k)
        best, where = logit.max(-1)
        assert torch.equal(logit.gather(-1, tokens[..., :1]).squeeze(-1), best)
        want = torch.log_softmax(logit.double(), -1).gather(-1, tokens.clamp(min=0))
        torch.testing.assert_close(logp.double(), want, rtol=1e-5, atol=1e-4)
    with torch.no_grad():
        assert 'action_alternatives' not in model.compute_logp_action(**obs, hidden_state=hidden)
    plain, fused = ResFCBlock2(24, norm_type='LN').to(device), ResFCBlock2(24, norm_type='FusedLN').to(device)
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(5, 24, device=device)
    torch.testing.assert_close(fused(x), plain(x), rtol=1e-5, atol=1e-5)
    assert build_normalization('FusedLN', dim=1) is FusedLayerNorm


# ------------------------------------------------------------------ sizes and streams

@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    gen = torch.Generator('cuda').manual_seed(0)
    x = torch.randn(70001, 32000, generator=gen, device='cuda', dtype=torch.bfloat16)     # 2.2e9 elements
    w, b = torch.randn(2, 32000, generator=gen, device='cuda')
    y = layer_norm(x, w, b)
    for part in (slice(0, 2), slice(67105, 67112), slice(-3, None)):
        assert torch.equal(y[part], layer_norm(x[part], w, b))
    del y
    tokens = torch.randint(0, 32000, (70001,), generator=gen, device='cuda')
    leaf = x.requires_grad_()
    got = token_logprobs(leaf, tokens, top_k=2)
    d, = torch.autograd.grad(got.logprob.sum(), leaf)
    for part in (slice(0, 2), slice(67105, 67112), slice(-3, None)):
        some = x.detach()[part].clone().requires_grad_()
        ref = token_logprobs(some, tokens[part], top_k=2)
        assert torch.equal(got.top_tokens[part], ref.top_tokens)
        torch.testing.assert_close(got.logprob[part], ref.logprob, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(d[part], torch.autograd.grad(ref.logprob.sum(), some)[0], rtol=1e-2, atol=1e-5)
    del d, got
    x = x.detach()
    weight = torch.randn(24, 32000, generator=gen, device='cuda').bfloat16() * 0.01
    y = linear_act(x, weight, None, 'relu')
    torch.testing.assert_close(y[-200:], linear_act(x[-200:].clone(), weight, None, 'relu'))
    wide = linear_act(y, weight.t().contiguous()[:, :24])                                # 2.2e9 outputs
    torch.testing.assert_close(wide[-200:], linear_act(y[-200:], weight.t().contiguous()))
    del wide, y
    x.fill_(1.0)
    want = math.sqrt(70001 * 32000)
    norm = clip_grad_norm([x], want / 2)
    assert abs(float(norm) - want) <= 4 * U * want
    assert bool((x[-1] == 0.5).all()) and bool((x[0] == 0.5).all()) and bool((x[67108] == 0.5).all())


@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    def work(seed):
        gen = torch.Generator('cuda').manual_seed(seed)
        x = torch.randn(3000, 264, generator=gen, device='cuda').bfloat16().requires_grad_()
        w = torch.randn(520, 264, generator=gen, device='cuda').bfloat16().requires_grad_()
        t = torch.randint(0, 520, (3000,), generator=gen, device='cuda')
        return x, w, t

    def run(x, w, t):
        y = linear_act(layer_norm(x), w, None, 'silu')
        got = token_logprobs(y, t, top_k=4)
        grads = torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), [x, w])
        return [got.logprob.detach(), got.top_tokens, clip_grad_norm(grads, 1.0), *grads]

    inputs = [work(1), work(2)]
    want = [run(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(3):
        got = []
        for stream, i in zip(streams, inputs):
            with torch.cuda.stream(stream):
                got.append(run(*i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_layer_norm_of_very_wide_rows():
    # more columns than a launch has threads at 16 columns a block
    gen = torch.Generator('cuda').manual_seed(1)
    x, dy = torch.randn(2, 2, 2 ** 25 + 9, generator=gen, device='cuda')
    w, b = torch.randn(2, 2 ** 25 + 9, generator=gen, device='cuda')
    _ln_check(x, None, w, b, dy, None)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [9, 40, 3000])
def test_token_logprobs_extreme_temperatures(device, dtype, width):
    gen = torch.Generator().manual_seed(width)
    logits = torch.randn(5, width, generator=gen).to(device, dtype)
    logits[:, 3] = 9.
    mask = torch.ones(5, width, dtype=torch.bool, device=device)
    mask[:, 5] = False
    logits[1, 6] = -math.inf
    tokens = torch.full((5,), 3, device=device)
    leaf = logits.clone().requires_grad_()
    cold = token_logprobs(leaf, tokens, mask=mask, temperature=1e-30, top_k=2)
    assert bool((cold.logprob == 0).all()) and bool((cold.entropy == 0).all())
    assert bool((cold.top_tokens[:, 0] == 3).all()) and bool((cold.top_logprobs[:, 0] == 0).all())
    grad, = torch.autograd.grad(cold.logprob.sum() + cold.entropy.sum(), leaf)
    assert bool((grad == 0).all())
    hot = token_logprobs(leaf, tokens, mask=mask, temperature=1e30)
    # the log of the count, by a sum, a logarithm and two products
    want = torch.full((5,), math.log(width - 1), dtype=torch.float64, device=device)
    want[1] = math.log(width - 2)
    near(hot.logprob, -want, (8 + width / 64) * U * (1 + want))
    near(hot.entropy, want, (8 + width / 64) * U * (1 + want))
    for bad in (9e-31, 2e30, math.inf, -1.):
        with pytest.raises(ValueError):
            token_logprobs(logits, tokens, temperature=bad)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', LOW)
@pytest.mark.parametrize('rows,k,n', [(512, 1024, 1024), (1024, 384, 1000), (2048, 997, 256), (600, 1201, 1003), (30000, 64, 136),
                                      (20000, 33, 41), (5000, 333, 777), (48, 3001, 200), (20, 4104, 264), (64, 2048, 520),
                                      (40, 4096, 1000), (100, 1500, 8), (4104, 3000, 4104)])
def test_linear_act_tiles_and_parts(dtype, rows, k, n):
    gen = torch.Generator('cuda').manual_seed(rows + k + n)
    make = lambda *s: torch.randn(*s, generator=gen, device='cuda').to(dtype)  # noqa: E731
    x, w, b, dy, r = make(rows, k), (make(n, k) * k ** -0.5).to(dtype), make(n), make(rows, n), make(rows, n)
    _linear_check(x, w, b, 'silu', r, dy)
    _linear_check(x, w, b, 'relu', None, dy)


@pytest.mark.parametrize('device', DEVICES)
def test_clip_grad_norm_own_output(device):
    gen = torch.Generator().manual_seed(3)
    a, b, c = (torch.randn(n, generator=gen).to(device, t) for n, t in
               ((20003, torch.float32), (517, torch.bfloat16), (64, torch.float16)))
    wide = torch.empty(517, device=device)
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in (a, b, c)))
    want = [t.double() * min(1., 0.5 / (norm + 1e-6)) for t in (a, b, c)]
    got = clip_grad_norm([a, b, c], 0.5, out=[a, wide, c])
    near(got, torch.tensor(norm, device=device, dtype=torch.float64), 4 * U * norm)
    for t, w in zip((a, wide, c), want):
        near(t, w, 4 * U * w.abs())          # the norm, the quotient, the scale, a product


@pytest.mark.gpu
def test_each_operator_in_a_graph_at_several_sizes():
    gen = torch.Generator('cuda').manual_seed(4)
    make = lambda *s, t=torch.bfloat16: torch.randn(*s, generator=gen, device='cuda').to(t)  # noqa: E731

    def norm_pass(x, r, w, b):
        leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
        y, s = add_layer_norm(*leaves)
        return [y.detach(), s.detach(), *torch.autograd.grad((y * s).sum(), leaves)]

    def linear_pass(x, w, b, r):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = linear_act(*leaves[:3], 'gelu', leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, r)]

    def logit_pass(x, tokens):
        leaf = x.detach().requires_grad_()
        got = token_logprobs(leaf, tokens, mask=x > -1.5, top_k=3)
        live = got.logprob.clamp(min=-30.) + got.entropy
        return [got.entropy.detach(), got.top_logprobs, got.top_tokens, *torch.autograd.grad(live, leaf, got.entropy)]

    def clip_pass(*tensors):
        outs = [torch.empty(t.shape, device='cuda') for t in tensors]
        return [clip_grad_norm(list(tensors), 0.1, out=outs), *outs]

    cases = [(norm_pass, [make(700, 1536), make(700, 1536), make(1536), make(1536)]),
             (norm_pass, [make(64, 9), make(64, 9), make(9), make(9)])]
    for m, k, n in ((40, 1024, 200), (512, 1024, 1024), (2048, 997, 256), (9000, 64, 72), (70, 5001, 33)):
        cases.append((linear_pass, [make(m, k), make(n, k) * 0.03, make(n), make(m, n)]))
    for m, n in ((300, 5000), (40, 327), (9, 40000)):
        cases.append((logit_pass, [make(m, n), torch.randint(0, n, (m,), generator=gen, device='cuda')]))
    cases.append((clip_pass, [make(3 * i * i + 1, t=TYPES[i % 3]) for i in range(300)]))
    for run, inputs in cases:
        run(*inputs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*inputs)
        for _ in range(3):
            inputs[0].copy_(make(*inputs[0].shape, t=inputs[0].dtype))
            want = run(*inputs)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
        del graph, out, want


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width,top_k', [(255, 7), (257, 7), (512, 6), (513, 64), (1024, 9), (1025, 2), (2049, 7)])
def test_token_logprobs_alternatives_at_batch_ends(device, dtype, width, top_k):
    gen = torch.Generator().manual_seed(width)
    logits = (torch.randn(37, width, generator=gen) * 3).to(device, dtype)
    tokens = torch.randint(0, width, (37,), generator=gen).to(device)
    mask = (torch.rand(37, width, generator=gen) < 0.7).to(device)
    mask.scatter_(-1, tokens.unsqueeze(-1), True)
    _lp_check(logits, tokens, mask, top_k=top_k)
    _lp_check(logits, tokens, None, temperature=0.8, top_k=top_k)


@pytest.mark.gpu
def test_kernels_are_switched_off_by_the_environment(monkeypatch):
    from distar_amd.ops import hip_ext
    x = torch.zeros(2, 8, device='cuda')
    for value, off in (('1', True), ('0', False), ('', False), ('1', True), (None, False)):
        if value is None:
            monkeypatch.delenv('DISTAR_AMD_DISABLE_HIP')
        else:
            monkeypatch.setenv('DISTAR_AMD_DISABLE_HIP', value)
        assert (hip_ext.maybe_ext(x) is None) == off
    assert hip_ext.maybe_ext(x.cpu()) is None


# ------------------------------------------------------------------ corners

@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', LOW)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
@pytest.mark.parametrize('rows,n', [(5, 16), (600, 16), (700, 264)])
def test_linear_act_slope_of_the_unrounded_sum(device, dtype, act, rows, n):
    # an identity as the weight: z = x + b has more digits than the operands' type, and
    # dx is dz. z comes with one 32-bit rounding, dz with the half step that `near` adds
    # (stored twice, the second time exactly)
    gen = torch.Generator().manual_seed(rows + n)
    x, dy = ((torch.randn(rows, n, generator=gen) * 2).to(device, dtype) for _ in range(2))
    b = torch.randn(n, generator=gen).to(device)
    w, leaf = torch.eye(n, dtype=dtype, device=device), x.clone().requires_grad_()
    dx, = torch.autograd.grad(linear_act(leaf, w, b, act, x), leaf, dy)
    z = x.double() + b.double()
    near(dx, dy.double() * SLOPE[act](z), dy.double().abs() * (16 * U + U * z.abs()))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('act', ['gelu', 'silu'])
def test_linear_act_sums_beyond_fp16(device, act):
    # z of up to 120000 either way, where the slope is 1 or 0
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(40, 16, generator=gen).to(device, torch.float16)
    x[7] = 60000.
    w = torch.eye(16, device=device) * 2
    w[3:9] *= -1
    dy = torch.randn(40, 16, generator=gen).to(device, torch.float16)
    dy[7] /= 64                                                 # for dw is below 65504
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_(), torch.zeros(16, device=device, requires_grad=True)]
    y = linear_act(*leaves, act)
    assert bool((y[7, 3:9] == 0).all())
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t()
    dz = dy.double() * SLOPE[act](z).nan_to_num(0.)             # the formula's 0 times infinity
    dz[7] = dy[7].double() * (z[7] > 0)
    t = half(torch.float16)
    off = dy.double().abs() * 32 * U + t * dz.abs() * 1.01 + torch.finfo(torch.float16).tiny
    near(dx, dz @ w.double(), off @ w.double().abs())
    near(dw, dz.t() @ x.double(), off.t() @ x.double().abs() + 64 * U * (dz.abs().t() @ x.double().abs()))
    near(db, dz.sum(0), off.sum(0))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('width', [7, 40, 513, 3000, 40000])
@pytest.mark.parametrize('flat', [True, False])
def test_token_logprobs_gradient_of_impossible_tokens(device, dtype, width, flat):
    # rows whose token has a logit of -inf, is masked, or lies outside [0, C): the first
    # two fall with the log of the sum, at the possible places alone, the last has no gradient
    gen = torch.Generator().manual_seed(width)
    logits = torch.randn(6, width + 3, generator=gen).to(device, dtype)[:, :width]
    logits = logits.contiguous() if flat else logits
    logits[:, 5] = -math.inf
    mask = torch.ones(6, width, dtype=torch.bool, device=device)
    mask[:, 2] = False
    tokens = torch.tensor([5, 2, -1, width, 1 << 40, 3], device=device)
    g, gh = torch.randn(2, 6, generator=gen).to(device)
    for m, entropy in ((None, False), (mask, False), (mask, True)):
        leaf = logits.detach().requires_grad_()
        got = token_logprobs(leaf, tokens, mask=m)
        d, = torch.autograd.grad([got.logprob, got.entropy], leaf, [g, gh * entropy])
        ok = (logits > -math.inf) & (mask if m is not None else True)
        logp = torch.where(ok, logits.double(), -math.inf).log_softmax(-1)
        p, logp = logp.exp(), torch.where(ok, logp, 0.)
        h = -(p * logp).sum(-1, keepdim=True)
        one = torch.zeros_like(p)
        one[5, 3] = 1.
        if m is None:
            one[1, 2] = 1.
        glp = g.double().masked_fill((tokens < 0) | (tokens >= width), 0.).unsqueeze(-1)
        want = glp * (one - p) - gh.double().unsqueeze(-1) * entropy * p * (logp + h)
        # as in _lp_check; the logits range over some 10
        off = U * (64 + 8 * 16) * 4 * (glp.abs() + gh.double().abs().unsqueeze(-1) * (1 + h))
        near(d, want, off.expand_as(want))
        assert bool((d[0] == 0)[5]) and bool((d[2:5] == 0).all()) or entropy
        assert bool((d[:, 5] == 0).all())


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype', LOW)
@pytest.mark.parametrize('k', [1, 3, 7, 8, 11])
def test_linear_act_channels_last(device, dtype, k):
    gen = torch.Generator().manual_seed(k)
    w, b = torch.randn(9, k, generator=gen).to(device, dtype), torch.randn(9, generator=gen).to(device, dtype)
    for shape, order in (((2, 5, 6, k), torch.channels_last), ((2, 3, 4, 5, k), torch.channels_last_3d)):
        x = torch.randn(shape, generator=gen).to(device, dtype)
        for n in (9, 3):                                  # rows of dy are narrow too
            dy = torch.randn(*shape[:-1], n, generator=gen).to(device, dtype)
            results = []
            for fmt in (torch.contiguous_format, order):
                leaves = [x.contiguous(memory_format=fmt).requires_grad_(), w[:n].clone().requires_grad_()]
                y = linear_act(*leaves, b[:n], 'gelu')
                results.append([y.detach(), *torch.autograd.grad(y, leaves, dy.contiguous(memory_format=fmt))])
            for a, c in zip(*results):
                assert a.shape == c.shape and torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', LOW)
def test_linear_act_gelu_far_below_zero(dtype):
    # z is x itself. z * cdf is off by the fit of the cdf (4.2e-6 of it), by three
    # roundings of z^2 / 2 in the exponent, and by some ten others
    x = -torch.linspace(0.5, 12.5, 4096, dtype=torch.float64, device='cuda').reshape(256, 16).to(dtype)
    w = torch.eye(16, dtype=dtype, device='cuda')
    y = linear_act(x, w, None, 'gelu')
    z = x.double().cpu()
    want = (z * 0.5 * torch.special.erfc(z * -0.5 ** 0.5)).cuda()      # ndtr loses the tail by 1 + erf
    z = z.cuda()
    near(y, want, want.abs() * (4.2e-6 + (16 + 1.5 * z * z) * U))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('width', [40, 3000])
def test_token_logprobs_large_gradients_of_entropy(device, width):
    # a scaled loss: places without probability stay without gradient
    gen = torch.Generator().manual_seed(width)
    logits = torch.randn(3, width, generator=gen).to(device)
    logits[:, ::3] = -math.inf
    logits[1, 1::3] = -1e9
    grads = []
    for scale in (1., 2. ** 34):
        leaf = logits.clone().requires_grad_()
        got = token_logprobs(leaf, torch.ones(3, dtype=torch.long, device=device))
        grads.append(torch.autograd.grad(got.entropy.sum() * scale, leaf)[0])
    assert bool(torch.isfinite(grads[0]).all())
    assert torch.equal(grads[1], grads[0] * 2. ** 34)           # a power of two: no rounding


@pytest.mark.parametrize('device', DEVICES)
def test_refused_clip_leaves_everything_as_it_was(device):
    a = torch.randn(5, device=device, requires_grad=True)
    b, c = torch.randn(5, device=device), torch.randn(5, device=device)
    bad = [lambda: clip_grad_norm([b, c], 0.1, out=[b, c.long()]), lambda: clip_grad_norm([b, c], 0.1, out=[b, c[:3]]),
           lambda: clip_grad_norm([b, c.long()], 0.1)]
    if device == 'cuda':
        bad += [lambda: clip_grad_norm([b, b], 0.1), lambda: clip_grad_norm([b, c.cpu()], 0.1),
                lambda: clip_grad_norm([b, c], 0.1, out=[c, b])]
    for call in bad:
        y, kept = (a * b * c).sum(), (b.clone(), c.clone())
        with pytest.raises((ValueError, TypeError)):
            call()
        assert torch.equal(b, kept[0]) and torch.equal(c, kept[1])
        y.backward()                                       # b and c are as they were saved


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    x, w, v = torch.randn(4, 8, device='cuda'), torch.randn(8, 8, device='cuda'), torch.randn(8, device='cuda')
    tokens = torch.zeros(4, dtype=torch.long, device='cuda')
    low = lambda t: t.bfloat16()  # noqa: E731
    with fwd.dual_level():
        dx, dw, dv = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, v))
        lx, lw, lv = (fwd.make_dual(low(t), torch.ones_like(low(t))) for t in (x, w, v))
        calls = [lambda: layer_norm(dx, v), lambda: layer_norm(x, dv), lambda: layer_norm(x, v, dv), lambda: add_layer_norm(x, dx),
                 lambda: linear_act(lx, low(w)), lambda: linear_act(low(x), lw), lambda: linear_act(low(x), low(w), lv),
                 lambda: linear_act(low(x), low(w), None, 'relu', lx), lambda: token_logprobs(dx, tokens),
                 lambda: grad_norm([v, dx]), lambda: clip_grad_norm([v, dx], 1.),
                 lambda: clip_grad_norm([v], 1., out=[dv])]
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call()
        assert torch.equal(layer_norm(x, v), layer_norm(fwd.unpack_dual(dx).primal, v))
    layer_norm(x, v)


def test_fused_transformer_refuses_the_tanh_gelu():
    from distar_amd.models.nn.transformer import Transformer
    args = dict(input_dim=16, head_dim=8, hidden_dim=32, output_dim=16, head_num=2, layer_num=1, fused=True)
    Transformer(**args, activation=torch.nn.GELU())
    with pytest.raises(ValueError):
        Transformer(**args, activation=torch.nn.GELU(approximate='tanh'))


@pytest.mark.gpu
def test_fused_transformer_in_float32():
    # as an actor without a batch server and a learner without autocast run it
    from distar_amd.models.nn.transformer import Transformer
    torch.manual_seed(0)
    args = dict(input_dim=48, head_dim=128, hidden_dim=160, output_dim=96, head_num=2, layer_num=2)
    plain, fused = Transformer(**args).cuda(), Transformer(**args, fused=True).cuda()
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(3, 20, 48, device='cuda')
    mask = torch.arange(20, device='cuda') < torch.tensor([[20], [7], [1]], device='cuda')
    dy = torch.randn(3, 20, 96, device='cuda')
    want, got = plain(x, mask), fused(x, mask)
    assert got.dtype == torch.float32
    ref, grads = (torch.autograd.grad(y, list(m.parameters()), dy) for y, m in ((want, plain), (got, fused)))
    # sums of up to 256 products, some twenty of them in a row, 32-bit; a relu whose input
    # lies within that noise may change sides, as in the test of the 16-bit stream
    noise = 20 * 16 * U
    flips = math.sqrt(5 * 0.8 * noise)
    for a, b, most in zip([got, *grads], [want, *ref], [noise] + [noise + flips] * len(grads)):
        assert torch.linalg.vector_norm((a - b).double()) <= most * torch.linalg.vector_norm(b.double()) + 1e-6
    module = LinearAct(48, 8, activation='silu').cuda()
    torch.testing.assert_close(module(x), torch.nn.functional.silu(torch.nn.functional.linear(x, module.weight, module.bias)))
    with torch.autocast('cuda', dtype=torch.bfloat16):
        assert module(x).dtype == torch.bfloat16


@pytest.mark.parametrize('device', DEVICES)
def test_linear_act_sums_stay_32_bit_under_autocast(device, monkeypatch):
    if device == 'cuda':
        monkeypatch.setenv('DISTAR_AMD_DISABLE_HIP', '1')
    gen = torch.Generator().manual_seed(1)
    x, w = torch.randn(30, 64, generator=gen).to(device).bfloat16(), torch.randn(9, 64, generator=gen).to(device)
    b, dy = torch.randn(9, generator=gen).to(device), torch.randn(30, 9, generator=gen).to(device).bfloat16()
    results = []
    for autocast in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        with torch.autocast(device, dtype=torch.bfloat16, enabled=autocast):
            y = linear_act(*leaves, 'gelu')
        results.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    for a, c in zip(*results):
        assert a.dtype == c.dtype and torch.equal(a, c)


@pytest.mark.gpu
def test_layer_norm_of_very_wide_rows_closely():
    # A block of 1024 threads adds up a row, n values each. Roundings of either sign add up
    # to 6 sqrt(n) of them but for 4 sums in 10^8 (Hoeffding's bound for n independent ones
    # of at most u each gives 2 exp(-18)), so a mean is off by that many u of the mean
    # magnitude, where the worst case, n, would be as large as the values themselves.
    width = 2 ** 25 + 9
    gen = torch.Generator('cuda').manual_seed(1)
    x, dy = torch.randn(2, 2, width, generator=gen, device='cuda') + 0.25
    w, b = torch.randn(2, width, generator=gen, device='cuda')
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    ref = _ln_reference(x, w, b, 1e-5, dy)
    e = (6 * math.sqrt(width / 1024) + 32) * U
    assert e < 1e-4
    size = x.double().abs().mean(-1, keepdim=True)
    h_off = e * (ref['r'] * size + ref['h'].abs())             # of the mean, and of 1 / the deviation
    near(y, ref['y'], h_off * w.double().abs() + 4 * U * (ref['y'].abs() + b.double().abs()))
    g = dy.double() * w.double()
    m1, m2 = g.abs().mean(-1, keepdim=True), (g * ref['h']).abs().mean(-1, keepdim=True)
    near(dx, ref['dx'], ref['r'] * (e * (2 * m1 + 2 * m2 * (1 + ref['h'].abs()) + g.abs()) + h_off * m2) + 8 * U * g.abs() * ref['r'])
    near(dw, ref['dw'], (dy.double().abs() * h_off).sum(0) + 4 * U * ref['dw_abs'])
    near(db, ref['db'], 2 * U * ref['db_abs'])


def test_linear_act_of_meta_tensors():
    # a device that autocast does not know
    x, module = torch.empty(4, 8, device='meta', requires_grad=True), LinearAct(8, 3, activation='gelu', device='meta')
    for y in (linear_act(x, module.weight, module.bias, 'gelu'), module(x)):
        assert y.shape == (4, 3) and y.device.type == 'meta'
