"""The training and inference operators around the policy transformer, as cases that can be timed:
layer normalisation with its residual stream, linear layers with their epilogue, log probabilities of given
tokens, and the clipping of a list of gradients."""
import math
import random

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decision of 16 environments: the residual joins the stream before the next sublayer
        {'name': 'ln_actor', 'op': 'ln', 'rows': 16, 'width': 256, 'dtype': 'bf16', 'wdtype': 'fp32', 'residual': True, 'train': False},
        # the gates of the LSTM core (4 x 384) over a ragged batch of trajectories, in full precision
        {'name': 'ln_gates', 'op': 'ln', 'rows': 4095, 'width': 1536, 'dtype': 'fp32', 'wdtype': 'fp32', 'residual': False, 'train': True},
        # the entity transformer's stream: 8 x 64 observations of 512 entities
        {'name': 'ln_entities', 'op': 'ln', 'rows': 262144, 'width': 256, 'dtype': 'bf16', 'wdtype': 'fp32', 'residual': True, 'train': True},
        # one decision of 16 environments: the action type over 327 actions with the race's mask and five alternatives
        {'name': 'lp_actor', 'op': 'lp', 'rows': 16, 'width': 327, 'dtype': 'fp32', 'mask': True, 'top_k': 5, 'temperature': 0.8, 'train': False},
        # selected units: 16 x 64 steps, up to 64 selections each over 513 ragged entities, padded selections ignored
        {'name': 'lp_units', 'op': 'lp', 'rows': 65536, 'width': 513, 'dtype': 'bf16', 'mask': True, 'top_k': 0, 'temperature': 1.0, 'train': True},
        # the target location: 32 x 64 steps over a 152 x 160 map
        {'name': 'lp_location', 'op': 'lp', 'rows': 2048, 'width': 24320, 'dtype': 'bf16', 'mask': False, 'top_k': 5, 'temperature': 1.0, 'train': True},
        # the same map while acting, in full precision, with more alternatives
        {'name': 'lp_location_eval', 'op': 'lp', 'rows': 33, 'width': 24320, 'dtype': 'fp32', 'mask': False, 'top_k': 20, 'temperature': 1.0, 'train': False},
        # a whole model's gradients, each aligned as an allocator aligns it, below the threshold: the ordinary step
        {'name': 'clip_model', 'op': 'clip', 'count': 332, 'total': 56_000_000, 'sizes': 1, 'dtype': 'fp32', 'norm': '2', 'packed': False, 'master': False},
        # bf16 gradients end to end in a reduction's flat bucket, clipped into 32-bit ones for the optimiser
        {'name': 'clip_master', 'op': 'clip', 'count': 1015, 'total': 170_000_000, 'sizes': 2, 'dtype': 'bf16', 'norm': '2', 'packed': True, 'master': True},
        # one decision of 16 environments: a head's first layer
        {'name': 'linear_actor', 'op': 'linear', 'rows': 16, 'k': 1024, 'n': 256, 'dtype': 'bf16', 'act': 'relu', 'residual': False, 'train': False},
        # the entity embedding: 64 observations of 512 entities, 997 features
        {'name': 'linear_embed', 'op': 'linear', 'rows': 32768, 'k': 997, 'n': 256, 'dtype': 'bf16', 'act': 'relu', 'residual': False, 'train': True},
        # a wide block's projection back onto its residual stream
        {'name': 'linear_wide', 'op': 'linear', 'rows': 16384, 'k': 4096, 'n': 2048, 'dtype': 'fp16', 'act': 'gelu', 'residual': True, 'train': True},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(['ln', 'lp', 'clip', 'linear'])
    if op == 'ln':
        width = _log(rng, 8, 8192)
        return {'op': 'ln', 'rows': min(_log(rng, 1, 262144), max(1, 2 ** 26 // width)), 'width': width,
                'dtype': rng.choice(['fp32', 'bf16', 'fp16']), 'wdtype': rng.choice(['fp32', 'same']),
                'residual': rng.random() < 0.5, 'train': rng.random() < 0.6}
    if op == 'lp':
        width = _log(rng, 2, 50000)
        return {'op': 'lp', 'rows': min(_log(rng, 1, 65536), max(1, 2048 * 24320 // width)), 'width': width,
                'dtype': rng.choice(['fp32', 'bf16', 'fp16']), 'mask': rng.random() < 0.5,
                'top_k': rng.choice([0, 0, 1, 2, 5, 8, 20, 32]), 'temperature': rng.choice([1.0, 1.0, 0.7, 1.6]),
                'train': rng.random() < 0.6}
    if op == 'clip':
        count = _log(rng, 1, 1200)
        return {'op': 'clip', 'count': count, 'total': max(count, _log(rng, 2000, 150_000_000)), 'sizes': rng.randrange(1 << 20),
                'dtype': rng.choice(['fp32', 'bf16', 'fp16', 'mixed']), 'norm': rng.choice(['2', '2', '2', '1', 'inf']),
                'packed': rng.random() < 0.5, 'master': rng.random() < 0.5}
    k, n = _log(rng, 8, 4096), _log(rng, 8, 4096)
    return {'op': 'linear', 'rows': min(_log(rng, 1, 131072), max(1, 2 ** 36 // (k * n))), 'k': k, 'n': n,
            'dtype': rng.choice(['bf16', 'fp16']), 'act': rng.choice(['none', 'relu', 'gelu', 'silu']),
            'residual': rng.random() < 0.5, 'train': rng.random() < 0.6}


def _sizes(case):
    """The tensors' sizes: a few large weights, many biases and norms."""
    rng = random.Random(case['sizes'])
    parts = [rng.lognormvariate(0.0, 2.5) for _ in range(case['count'])]
    scale = (case['total'] - case['count']) / sum(parts)
    return [1 + int(p * scale) for p in parts]


def _clip_types(case):
    if case['dtype'] != 'mixed':
        return [case['dtype']] * case['count']
    rng = random.Random(case['sizes'] + 1)
    return [rng.choice(['fp32', 'bf16', 'fp16']) for _ in range(case['count'])]


def _views(case, types, fill):
    """One tensor for each size, as views of one buffer of each type: end to end, or each on a boundary
    of 256 elements. Returns the buffers and the views."""
    ends, places = {}, []
    for n, t in zip(_sizes(case), types):
        start = ends.get(t, 0)
        places.append((t, start, n))
        ends[t] = start + (n if case['packed'] else -(-n // 256) * 256)
    buffers = {t: torch.zeros(n, device='cuda', dtype=DTYPES[t]) for t, n in ends.items()}
    views = [buffers[t][start:start + n] for t, start, n in places]
    if fill is not None:
        values = fill(sum(n for _, _, n in places)).split([n for _, _, n in places])
        for view, value in zip(views, values):
            view.copy_(value)
    return list(buffers.values()), views


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, device='cuda', generator=gen) * scale).to(dtype)

    state = {'case': case}
    if case['op'] == 'ln':
        rows, width, dtype = case['rows'], case['width'], DTYPES[case['dtype']]
        wdtype = torch.float32 if case['wdtype'] == 'fp32' else dtype
        channel = 1 + 4 * (torch.rand(width, device='cuda', generator=gen) < 0.02)
        state['x'] = (normal(rows, width) * channel + 0.2).to(dtype)
        state['residual'] = normal(rows, width, scale=2.0, dtype=dtype) if case['residual'] else None
        state['weight'] = (1 + normal(width, scale=0.1)).to(wdtype)
        state['bias'] = normal(width, scale=0.1, dtype=wdtype)
        if case['train']:
            state['dy'] = normal(rows, width, dtype=dtype)
            state['ds'] = normal(rows, width, dtype=dtype) if case['residual'] else None
            for name in ('x', 'residual', 'weight', 'bias'):
                if state[name] is not None:
                    state[name].requires_grad_()
    elif case['op'] == 'lp':
        rows, width, dtype = case['rows'], case['width'], DTYPES[case['dtype']]
        logits = normal(rows, width, scale=2.0)
        if case['mask']:
            # a ragged number of allowed entries in each row, a few rows with none
            allowed = torch.randint(1, width + 1, (rows, 1), device='cuda', generator=gen)
            empty = torch.rand(rows, 1, device='cuda', generator=gen) < 0.05
            allowed = allowed.masked_fill(empty, 0) if rows > 1 else allowed
            mask = torch.arange(width, device='cuda') < allowed
            logits = logits.masked_fill(~mask, -6e4)
            tokens = (torch.rand(rows, device='cuda', generator=gen) * allowed[:, 0]).long().clamp(max=width - 1)
            tokens = tokens.masked_fill(allowed[:, 0] == 0, -100)
        else:
            mask = None
            tokens = torch.randint(0, width, (rows,), device='cuda', generator=gen)
        state.update(logits=logits.to(dtype), tokens=tokens, mask=mask)
        if case['train']:
            state['logits'].requires_grad_()
            state['dlogprob'] = normal(rows)
            state['dentropy'] = normal(rows, scale=0.1)
    elif case['op'] == 'clip':
        scale, p = 0.01, case['norm']
        n = sum(_sizes(case))
        buffers, grads = _views(case, _clip_types(case), lambda n: normal(n, scale=scale))
        norm = scale * (5.0 if p == 'inf' else 0.8 * n if p == '1' else math.sqrt(n))
        state.update(grads=grads, buffers=buffers, out=None, max_norm=norm * (0.3 if case['master'] else 3.0))
        if case['master']:
            state['buffers'], state['out'] = _views(case, ['fp32'] * case['count'], None)
    else:
        rows, k, n, dtype = case['rows'], case['k'], case['n'], DTYPES[case['dtype']]
        state['x'] = normal(rows, k, dtype=dtype)
        state['weight'] = normal(n, k, scale=k ** -0.5, dtype=dtype)
        state['bias'] = normal(n, scale=0.1, dtype=dtype)
        state['residual'] = normal(rows, n, dtype=dtype) if case['residual'] else None
        if case['train']:
            state['dy'] = normal(rows, n, dtype=dtype)
            for name in ('x', 'weight', 'bias', 'residual'):
                if state[name] is not None:
                    state[name].requires_grad_()
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    return (_own if own else _plain)[state['case']['op']](state)


def _ln_own(state):
    from distar_amd.ops.layer_norm import add_layer_norm, layer_norm
    case = state['case']
    with torch.set_grad_enabled(case['train']):
        if case['residual']:
            y, s = add_layer_norm(state['x'], state['residual'], state['weight'], state['bias'], 1e-5)
        else:
            y, s = layer_norm(state['x'], state['weight'], state['bias'], 1e-5), None
    out = {'y': y.detach(), 's': None if s is None else s.detach()}
    if case['train']:
        names = [m for m in ('x', 'residual', 'weight', 'bias') if state[m] is not None]
        outs, douts = ([y], [state['dy']]) if s is None else ([y, s], [state['dy'], state['ds']])
        out.update(zip(['d' + m for m in names], torch.autograd.grad(outs, [state[m] for m in names], douts)))
    return {m: t for m, t in out.items() if t is not None}


@torch.no_grad()
def _ln_plain(state):
    case, x, w = state['case'], state['x'], state['weight'].float()
    s = x if not case['residual'] else (x.float() + state['residual'].float()).to(x.dtype)
    sf = s.float()
    centred = sf - sf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    xhat = centred * rstd
    out = {'y': (xhat * w + state['bias'].float()).to(x.dtype)}
    if case['residual']:
        out['s'] = s
    if case['train']:
        dy = state['dy'].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        if case['residual']:
            dx = dx + state['ds'].float()
        out['dx'] = dx.to(x.dtype)
        if case['residual']:
            out['dresidual'] = out['dx']
        out['dweight'] = (dy * xhat).sum(0).to(state['weight'].dtype)
        out['dbias'] = dy.sum(0).to(state['bias'].dtype)
    return out


def _lp_own(state):
    from distar_amd.ops.token_logprobs import token_logprobs
    case = state['case']
    with torch.set_grad_enabled(case['train']):
        got = token_logprobs(state['logits'], state['tokens'], mask=state['mask'],
                             temperature=case['temperature'], top_k=case['top_k'])
    out = {'logprob': got.logprob.detach(), 'entropy': got.entropy.detach()}
    if case['top_k']:
        out.update(top_logprobs=got.top_logprobs, top_tokens=got.top_tokens)
    if case['train']:
        out['dlogits'], = torch.autograd.grad([got.logprob, got.entropy], [state['logits']],
                                              [state['dlogprob'], state['dentropy']])
    return out


@torch.no_grad()
def _lp_plain(state):
    case, tokens, mask = state['case'], state['tokens'], state['mask']
    raw = state['logits'].float()
    if mask is not None:
        raw = raw.masked_fill(~mask, -math.inf)
    logits = raw / case['temperature']
    top = logits.amax(-1, keepdim=True)
    shifted = logits - top.masked_fill(top == -math.inf, 0.0)
    e = torch.exp(shifted)
    total = e.sum(-1, keepdim=True)
    logp = shifted - torch.log(total)
    empty = total == 0
    p = torch.where(empty, 0.0, e / total)
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(-1)
    given = tokens >= 0
    at = tokens.clamp(min=0).unsqueeze(-1)
    logp = logp.masked_fill(empty, -math.inf)
    out = {'logprob': logp.gather(-1, at)[:, 0].masked_fill(~given, 0.0), 'entropy': entropy}
    k = min(case['top_k'], case['width'])
    if k:
        order = torch.sort(raw, dim=-1, descending=True, stable=True)[1][:, :k]
        found = raw.gather(-1, order) > -math.inf
        out['top_logprobs'] = logp.gather(-1, order).masked_fill(~found, -math.inf)
        out['top_tokens'] = order.masked_fill(~found, -1)
    if case['train']:
        dlogprob = state['dlogprob'].masked_fill(~given, 0.0).unsqueeze(-1)
        d = -dlogprob * p - state['dentropy'].unsqueeze(-1) * (plogp + p * entropy.unsqueeze(-1))
        d.scatter_add_(-1, at, dlogprob.masked_fill(empty, 0.0))
        out['dlogits'] = (d / case['temperature']).to(state['logits'].dtype)
    return out


def _clip_own(state):
    from distar_amd.ops.grad_norm import clip_grad_norm
    norm = clip_grad_norm(state['grads'], state['max_norm'], norm_type=float(state['case']['norm']), out=state['out'])
    return {'norm': norm, 'clipped': state['buffers']}


@torch.no_grad()
def _clip_plain(state):
    grads, p = state['grads'], state['case']['norm']
    flat = torch.cat([g.float() for g in grads]).abs()
    norm = flat.amax() if p == 'inf' else flat.sum() if p == '1' else flat.square().sum().sqrt()
    scale = (state['max_norm'] / (norm + 1e-6)).clamp(max=1.0)
    if state['out'] is None:
        [g.mul_(scale) for g in grads]
    else:
        [torch.mul(g.float(), scale, out=o) for g, o in zip(grads, state['out'])]
    return {'norm': norm, 'clipped': state['buffers']}


def _linear_own(state):
    from distar_amd.ops.linear_act import linear_act
    case = state['case']
    act = None if case['act'] == 'none' else case['act']
    with torch.set_grad_enabled(case['train']):
        y = linear_act(state['x'], state['weight'], state['bias'], activation=act, residual=state['residual'])
    out = {'y': y.detach()}
    if case['train']:
        names = [m for m in ('x', 'weight', 'bias', 'residual') if state[m] is not None]
        out.update(zip(['d' + m for m in names], torch.autograd.grad(y, [state[m] for m in names], state['dy'])))
    return out


@torch.no_grad()
def _linear_plain(state):
    case, x, w = state['case'], state['x'].float(), state['weight'].float()
    dtype, act = state['x'].dtype, case['act']
    z = x @ w.t() + state['bias'].float()
    if act == 'relu':
        y = z.clamp(min=0.0)
    elif act == 'gelu':
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        y = z * cdf
    elif act == 'silu':
        gate = 1.0 / (1.0 + torch.exp(-z))
        y = z * gate
    else:
        y = z
    if case['residual']:
        y = y + state['residual'].float()
    out = {'y': y.to(dtype)}
    if case['train']:
        dz = state['dy'].float()
        if act == 'relu':
            dz = dz * (z > 0)
        elif act == 'gelu':
            dz = dz * (cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
        elif act == 'silu':
            dz = dz * gate * (1.0 + z * (1.0 - gate))
        out.update(dx=(dz @ w).to(dtype), dweight=(dz.t() @ x).to(dtype), dbias=dz.sum(0).to(dtype))
        if case['residual']:
            out['dresidual'] = state['dy']
    return out


_own = {'ln': _ln_own, 'lp': _lp_own, 'clip': _clip_own, 'linear': _linear_own}
_plain = {'ln': _ln_plain, 'lp': _lp_plain, 'clip': _clip_plain, 'linear': _linear_plain}


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = {'fp32': 4, 'bf16': 2, 'fp16': 2, 'mixed': 8 / 3}[case['dtype']]
    if case['op'] == 'ln':
        cells = case['rows'] * case['width']
        forward = 4 if case['residual'] else 2           # x, (residual) -> y, (s)
        backward = 0 if not case['train'] else 3 if case['residual'] else 2   # dy, (ds) -> dx
        params = case['width'] * (4 if case['wdtype'] == 'fp32' else size) * (4 if case['train'] else 2)
        return {'bytes': cells * size * (forward + backward) + params, 'flops': cells * (20 if case['train'] else 8)}
    if case['op'] == 'lp':
        cells = case['rows'] * case['width']
        read = cells * (size + (1 if case['mask'] else 0)) + case['rows'] * 8
        write = case['rows'] * (8 + 12 * min(case['top_k'], case['width']))
        if case['train']:
            read, write = read + case['rows'] * 8, write + cells * size
        return {'bytes': read + write, 'flops': cells * (16 if case['train'] else 8)}
    if case['op'] == 'clip':
        n = sum(_sizes(case))
        return {'bytes': n * size + (n * 4 if case['master'] else 0), 'flops': n * (3 if case['master'] else 2)}
    m, k, n = case['rows'], case['k'], case['n']
    cells = m * k + n * k + n + m * n * (2 if case['residual'] else 1)
    if case['train']:
        cells += m * n + m * k + n * k + n
    return {'bytes': cells * size, 'flops': 2 * m * n * k * (3 if case['train'] else 1)}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {'ln': _ln_exact, 'lp': _lp_exact, 'clip': _clip_exact, 'linear': _linear_exact}[case['op']](state)


def _ln_exact(state):
    # the stream is what is stored and normalised: the sum in x's own type
    case, x = state['case'], state['x'].detach()
    w, b = (state[m].detach().double() for m in ('weight', 'bias'))
    s = (x.double() + state['residual'].detach().double()).to(x.dtype).double() if case['residual'] else x.double()
    var, mean = torch.var_mean(s, -1, correction=0, keepdim=True)
    z = (s - mean) / (var + 1e-5).sqrt()
    out = {'y': torch.addcmul(b, z, w)}
    if case['residual']:
        out['s'] = s
    if case['train']:
        dy = state['dy'].double()
        dz = dy * w
        width = case['width']
        dx = (width * dz - dz.sum(-1, keepdim=True) - z * torch.linalg.vecdot(dz, z).unsqueeze(-1)) / (width * (var + 1e-5).sqrt())
        out['dx'] = dx + state['ds'].double() if case['residual'] else dx
        if case['residual']:
            out['dresidual'] = out['dx']
        out['dweight'] = torch.linalg.vecdot(dy, z, dim=0)
        out['dbias'] = dy.sum(0)
    return out


def _lp_exact(state):
    case, tokens, mask = state['case'], state['tokens'], state['mask']
    raw = state['logits'].detach().double()
    if mask is not None:
        raw = torch.where(mask, raw, -math.inf)
    given, lse = tokens >= 0, torch.logsumexp(raw / case['temperature'], -1, keepdim=True)
    some = lse > -math.inf
    logp = torch.where(some, raw / case['temperature'] - lse, -math.inf)
    p = logp.exp()
    entropy = torch.special.entr(p).sum(-1)
    at = torch.where(given, tokens, 0).unsqueeze(-1)
    out = {'logprob': torch.where(given, torch.take_along_dim(logp, at, -1)[:, 0], 0.0), 'entropy': entropy}
    k = min(case['top_k'], case['width'])
    if k:
        best, where = torch.sort(raw, dim=-1, descending=True, stable=True)
        best, where = best[:, :k], where[:, :k]
        out['top_logprobs'] = torch.where(best > -math.inf, best / case['temperature'] - lse, -math.inf)
        out['top_tokens'] = torch.where(best > -math.inf, where, -1)
    if case['train']:
        g = torch.where(given, state['dlogprob'].double(), 0.0).unsqueeze(-1)
        one = torch.zeros_like(p).scatter_(-1, at, 1.0)
        d = torch.where(some, g * (one - p), 0.0)
        d += state['dentropy'].double().unsqueeze(-1) * (torch.special.entr(p) - p * entropy.unsqueeze(-1))
        out['dlogits'] = d / case['temperature']
    return out


def _clip_exact(state):
    order = float(state['case']['norm'])
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double(), order) for g in state['grads']]), order)
    scale = min(1.0, state['max_norm'] / (float(norm) + 1e-6))
    if state['out'] is None:
        return {'norm': norm, 'clipped': [b.double() * scale for b in state['buffers']]}
    flat = state['buffers'][0].double()
    for o, g in zip(state['out'], state['grads']):
        flat[o.storage_offset():o.storage_offset() + o.numel()] = g.double() * scale
    return {'norm': norm, 'clipped': [flat]}


def _linear_exact(state):
    case = state['case']
    x, w, b = (state[m].detach().double() for m in ('x', 'weight', 'bias'))
    z = torch.addmm(b, x, w.t())
    one = torch.ones_like(z)
    if case['act'] == 'relu':
        y, slope = torch.relu(z), (z > 0).double()
    elif case['act'] == 'gelu':
        slope = torch.special.ndtr(z)
        y = z * slope
        slope = slope + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
    elif case['act'] == 'silu':
        slope = torch.sigmoid(z)
        y = z * slope
        slope = slope + y * (1 - slope)
    else:
        y, slope = z, one
    out = {'y': y + state['residual'].detach().double() if case['residual'] else y}
    if case['train']:
        dz = state['dy'].double() * slope
        out.update(dx=torch.mm(dz, w), dweight=torch.mm(dz.t(), x), dbias=dz.sum(0))
        if case['residual']:
            out['dresidual'] = state['dy'].double()
    return out
