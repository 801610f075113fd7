"""Workloads of the expert-MLP operators (``ops/experts.py``) and of the
4-bit products (``ops/mxfp4.py``), and their plain forms.

Five operators: ``route`` (router logits to a plan), ``grouped`` (one matrix
product per expert over ragged row groups, bf16 or MXFP4 weights),
``combine`` (the experts' rows back to their tokens), ``quantize`` (a tensor
through MXFP4 and back) and ``mxgemm`` (bf16 activations through MXFP4
against MXFP4 weights).  :func:`run` makes one pass through one of them:
with ``own`` false in elementary torch operations in 32 bits, with ``own``
true by the framework's calls.
"""
import math

import torch

own = False

BLOCK = 32                      # elements under one MXFP4 scale
#: magnitudes of the eight e2m1 codes
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GELU_C = 0.7978845608028654     # sqrt(2 / pi)

LISTED = (
    # one request's token through a router: pure latency
    dict(name='route-one', op='route', tokens=1, experts=16, k=2,
         dtype='float32', padded=0.0),
    # a prefill batch with many small experts, an eighth of its rows padding
    dict(name='route-batch', op='route', tokens=16384, experts=128, k=8,
         dtype='bfloat16', padded=0.125),
    # up-projection of one request's token: two experts' weights are read
    dict(name='up-one', op='grouped', mx=False, tokens=1, experts=8, k=2,
         inner=4096, outer=16384, epilogue='gelu', gather=True, padded=0.0),
    # up-projection of a prefill batch, groups of very different sizes
    dict(name='up-batch', op='grouped', mx=False, tokens=2048, experts=8,
         k=2, inner=4096, outer=16384, epilogue='gelu', gather=True,
         padded=0.05),
    # 4-bit down-projection of a decode batch: few rows for each expert, the
    # weights are what is read
    dict(name='mx-down-decode', op='grouped', mx=True, tokens=32, experts=64,
         k=4, inner=4096, outer=4096, epilogue='bias', gather=False,
         padded=0.0),
    # 4-bit down-projection of a prefill batch
    dict(name='mx-down-batch', op='grouped', mx=True, tokens=2048, experts=8,
         k=2, inner=16384, outer=4096, epilogue='bias', gather=False,
         padded=0.05),
    # the two expert rows of one token
    dict(name='combine-one', op='combine', tokens=1, k=2, width=4096,
         padded=0.0),
    # the expert rows of a prefill batch, an eighth of its tokens padding
    dict(name='combine-batch', op='combine', tokens=8192, k=4, width=4096,
         padded=0.125),
    # one token's activations
    dict(name='quantize-row', op='quantize', rows=1, inner=4096,
         dtype='bfloat16'),
    # one projection's weights when a model is loaded
    dict(name='quantize-weights', op='quantize', rows=16384, inner=4096,
         dtype='bfloat16'),
    # one token through a 4-bit down-projection with its residual
    dict(name='mxgemm-one', op='mxgemm', rows=1, inner=16384, outer=4096,
         epilogue='residual'),
    # the worker's batch through a 4-bit up-projection
    dict(name='mxgemm-batch', op='mxgemm', rows=2048, inner=4096,
         outer=16384, epilogue='gelu'),
)


def listed():
    """The listed cases."""
    return [dict(case) for case in LISTED]


def _log(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], spread over the logarithm."""
    value = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return min(max(int(value) // step * step, max(lo, step)), hi)


def draw(rng):
    """One more case of the listed ones' ranges."""
    largest = {}
    for case in LISTED:
        cost = work(case)
        for key in cost:
            largest[key] = max(largest.get(key, 0), cost[key])
    while True:
        case = _draw(rng)
        cost = work(case)
        if cost['flops'] <= largest['flops'] and \
                cost['bytes'] <= largest['bytes']:
            return case


def _draw(rng):
    op = rng.choice(('route', 'grouped', 'grouped', 'combine', 'quantize',
                     'mxgemm'))
    padded = rng.choice((0.0, 0.05, 0.125, 0.5))
    if op == 'route':
        experts = _log(rng, 4, 256)
        return dict(op=op, tokens=_log(rng, 1, 16384), experts=experts,
                    k=min(experts, rng.randint(1, 8)), padded=padded,
                    dtype=rng.choice(('float32', 'bfloat16')))
    if op == 'grouped':
        mx = rng.random() < 0.5
        experts = _log(rng, 4, 64)
        return dict(op=op, mx=mx, tokens=_log(rng, 1, 4096),
                    experts=experts, k=rng.randint(1, min(4, experts)),
                    inner=_log(rng, 128, 16384, 128 if mx else 64),
                    outer=_log(rng, 64, 16384, 16),
                    epilogue=rng.choice(('none', 'bias', 'gelu')),
                    gather=rng.random() < 0.5, padded=padded)
    if op == 'combine':
        return dict(op=op, tokens=_log(rng, 1, 8192), k=rng.randint(1, 8),
                    width=_log(rng, 64, 8192, 8), padded=padded)
    if op == 'quantize':
        return dict(op=op, rows=_log(rng, 1, 16384),
                    inner=_log(rng, 64, 16384, 32),
                    dtype=rng.choice(('float32', 'bfloat16')))
    return dict(op=op, rows=_log(rng, 1, 4096),
                inner=_log(rng, 128, 16384, 128),
                outer=_log(rng, 64, 16384, 16),
                epilogue=rng.choice(('none', 'gelu', 'residual')))


def _touched(case):
    """How many experts a case's rows can reach."""
    return min(case['experts'], case['tokens'] * case['k'])


def _assigned(case):
    """Tokens of a case that are not padding."""
    return case['tokens'] - int(case['tokens'] * case['padded'])


def work(case):
    """Bytes and operations one pass cannot do without."""
    op = case['op']
    if op == 'route':
        tokens, experts, k = case['tokens'], case['experts'], case['k']
        size = 4 if case['dtype'] == 'float32' else 2
        return {'bytes': tokens * experts * size + 16 * tokens * k
                + 4 * (experts + 1), 'flops': 4 * tokens * experts}
    if op == 'grouped':
        rows = _assigned(case) * case['k']
        inner, outer = case['inner'], case['outer']
        size = 17 / 32 if case['mx'] else 2
        source = _assigned(case) if case['gather'] else rows
        size_a = 17 / 32 if case['mx'] and not case['gather'] else 2
        total = (_touched(case) * outer * inner * size
                 + source * inner * size_a
                 + case['tokens'] * case['k'] * outer * 2)
        if case['epilogue'] != 'none':
            total += 4 * _touched(case) * outer
        return {'bytes': int(total), 'flops': 2 * rows * outer * inner}
    if op == 'combine':
        tokens, width = case['tokens'], case['width']
        rows = _assigned(case) * case['k']
        return {'bytes': 2 * width * (rows + 2 * tokens)
                + 8 * tokens * case['k'], 'flops': 2 * rows * width}
    if op == 'quantize':
        size = 4 if case['dtype'] == 'float32' else 2
        count = case['rows'] * case['inner']
        return {'bytes': count * (size + size), 'flops': 4 * count}
    rows, inner, outer = case['rows'], case['inner'], case['outer']
    total = rows * inner * 2 + outer * inner * 17 / 32 + rows * outer * 2
    if case['epilogue'] != 'none':
        total += 4 * outer
    if case['epilogue'] == 'residual':
        total += 2 * rows * outer
    return {'bytes': int(total), 'flops': 2 * rows * inner * outer}


# ---------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed))


def _normal(shape, gen, scale=1.0, dtype=torch.bfloat16):
    """Normal values, made a slice at a time where there are many."""
    out = torch.empty(shape, dtype=dtype, device='cuda')
    flat = out.view(-1)
    for start in range(0, flat.numel(), 1 << 27):
        part = flat[start:start + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=gen, device='cuda')
                   * scale)
    return out


def _logits(tokens, experts, padded, dtype, gen):
    """Router logits: some experts are sought more than others, the padded
    tail of the batch has every expert masked."""
    out = torch.randn(tokens, experts, generator=gen, device='cuda')
    out = out + torch.randn(experts, generator=gen, device='cuda')
    out = out.to(getattr(torch, dtype))
    count = int(tokens * padded)
    if count:
        out[tokens - count:] = float('-inf')
    return out


def _quantized(shape, gen, scale):
    """MXFP4 codes and scales of normal values, a matrix at a time."""
    codes = torch.empty(shape[:-1] + (shape[-1] // 2,), dtype=torch.uint8,
                        device='cuda')
    scales = torch.empty(shape[:-1] + (shape[-1] // BLOCK,),
                         dtype=torch.uint8, device='cuda')
    pairs = zip(codes.view(-1, *codes.shape[-2:]),
                scales.view(-1, *scales.shape[-2:]))
    for part_codes, part_scales in pairs:
        x = _normal(shape[-2:], gen, scale, torch.float32)
        index, exponent = plain_quantize(x)
        part_codes.copy_(index[..., 0::2] | (index[..., 1::2] << 4))
        part_scales.copy_((exponent + 127).to(torch.uint8))
    return codes, scales


def prepare(case, seed):
    """What a user's program holds before the call."""
    gen = _generator(seed)
    op = case['op']
    state = {'case': dict(case)}
    if op == 'route':
        state['logits'] = _logits(case['tokens'], case['experts'],
                                  case['padded'], case['dtype'], gen)
    elif op == 'grouped':
        tokens, experts, k = case['tokens'], case['experts'], case['k']
        inner, outer = case['inner'], case['outer']
        plan = plain_route(_logits(tokens, experts, case['padded'],
                                   'float32', gen), k)
        state['offsets'] = plan['offsets']
        # the plain form walks the groups on the host
        state['bounds'] = plan['offsets'].tolist()
        state['rows'] = plan['tokens'] if case['gather'] else None
        count = tokens if case['gather'] else tokens * k
        if case['mx']:
            state['b'] = _quantized((experts, outer, inner), gen,
                                    inner ** -0.5)
            # gathered rows are quantised within the call, expert rows are
            # what the last product's quantisation left
            state['a'] = _normal((count, inner), gen) if case['gather'] \
                else _quantized((count, inner), gen, 1.0)
        else:
            state['b'] = _normal((experts, outer, inner), gen, inner ** -0.5)
            state['a'] = _normal((count, inner), gen)
        state['bias'] = None if case['epilogue'] == 'none' else \
            _normal((experts, outer), gen, 0.5, torch.float32)
    elif op == 'combine':
        tokens, k = case['tokens'], case['k']
        logits = _logits(tokens, max(8, k), case['padded'], 'float32', gen)
        plan = plain_route(logits, k)
        state['positions'], state['weights'] = \
            plan['positions'], plan['weights']
        state['y'] = _normal((tokens * k, case['width']), gen)
        state['residual'] = _normal((tokens, case['width']), gen)
    elif op == 'quantize':
        # activations: a few channels are much larger than the rest
        x = _normal((case['rows'], case['inner']), gen, 1.0,
                    getattr(torch, case['dtype']))
        x[:, ::67] *= 24
        state['x'] = x
    else:
        rows, inner, outer = case['rows'], case['inner'], case['outer']
        state['a'] = _normal((rows, inner), gen)
        state['b'] = _quantized((outer, inner), gen, inner ** -0.5)
        state['bias'] = None if case['epilogue'] == 'none' else \
            _normal((outer,), gen, 0.5, torch.float32)
        state['residual'] = _normal((rows, outer), gen) \
            if case['epilogue'] == 'residual' else None
    return state


# ---------------------------------------------------------------------------
# plain forms

def plain_route(logits, k):
    tokens, experts = logits.shape
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    top, index = order.values[:, :k], order.indices[:, :k]
    masked = top == float('-inf')
    weights = torch.where(masked, 0.0, torch.exp(top - top[:, :1]))
    total = weights.sum(1, keepdim=True)
    weights = torch.where(total == 0, 0.0, weights / total)
    key = torch.where(masked, experts, index).reshape(-1)
    rows = torch.sort(key, stable=True)
    places = torch.arange(tokens * k, device=logits.device)
    positions = torch.empty_like(places)
    positions[rows.indices] = places
    positions = torch.where(masked, -1, positions.view(tokens, k))
    offsets = torch.searchsorted(
        rows.values, torch.arange(experts + 1, device=logits.device))
    row_tokens = torch.where(rows.values == experts, -1, rows.indices // k)
    return {'experts': torch.where(masked, -1, index).to(torch.int32),
            'weights': weights, 'tokens': row_tokens.to(torch.int32),
            'positions': positions.to(torch.int32),
            'offsets': offsets.to(torch.int32)}


def plain_quantize(x):
    """e2m1 codes (uint8, one an element) and the blocks' exponents."""
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    peak = blocks.abs().amax(-1)
    exponent = torch.where(peak > 0, torch.frexp(peak).exponent - 3, -127)
    exponent = exponent.clamp(min=-127)
    v = torch.ldexp(blocks, -exponent.unsqueeze(-1)).abs()
    code = ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25)
            + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5))
    code = code + 8 * torch.signbit(blocks).to(torch.uint8)
    return code.flatten(-2), exponent


def plain_dequantize(index, exponent):
    table = torch.tensor(VALUES + tuple(-v for v in VALUES),
                         device=index.device)
    values = table[index.int()].unflatten(-1, (-1, BLOCK))
    return torch.ldexp(values, exponent.unsqueeze(-1)).flatten(-2)


def plain_values(quantized):
    """What packed codes and scale bytes stand for."""
    codes, scales = quantized
    index = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return plain_dequantize(index, scales.int() - 127)


def plain_gelu(x):
    return 0.5 * x * (1.0 + torch.tanh(GELU_C * (x + 0.044715 * x ** 3)))


def _plain_grouped(state):
    case, bounds = state['case'], state['bounds']
    a = state['a']
    if case['mx']:
        a = plain_dequantize(*plain_quantize(a)) if case['gather'] \
            else plain_values(a)
    a = a.float()
    if state['rows'] is not None:
        a = a[state['rows'].clamp(min=0).long()]
    out = torch.zeros(a.shape[0], case['outer'], dtype=torch.bfloat16,
                      device=a.device)
    for e in range(case['experts']):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        b = plain_values([part[e] for part in state['b']]) if case['mx'] \
            else state['b'][e].float()
        y = a[lo:hi] @ b.t()
        if case['epilogue'] != 'none':
            y = y + state['bias'][e]
        if case['epilogue'] == 'gelu':
            y = plain_gelu(y)
        out[lo:hi] = y.to(torch.bfloat16)
    return out


def _plain_combine(state):
    positions, weights = state['positions'], state['weights']
    rows = state['y'][positions.clamp(min=0).long()].float()
    rows = torch.where((positions < 0).unsqueeze(-1), 0.0,
                       rows * weights.unsqueeze(-1))
    return (state['residual'].float() + rows.sum(1)).to(torch.bfloat16)


def _plain_mxgemm(state):
    case = state['case']
    a = plain_dequantize(*plain_quantize(state['a']))
    y = a @ plain_values(state['b']).t()
    if case['epilogue'] != 'none':
        y = y + state['bias']
    if case['epilogue'] == 'gelu':
        y = plain_gelu(y)
    if case['epilogue'] == 'residual':
        y = y + state['residual'].float()
    return y.to(torch.bfloat16)


def _plain(state):
    case = state['case']
    op = case['op']
    if op == 'route':
        return plain_route(state['logits'], case['k'])
    if op == 'grouped':
        return _plain_grouped(state)
    if op == 'combine':
        return _plain_combine(state)
    if op == 'quantize':
        x = state['x']
        return plain_dequantize(*plain_quantize(x)).to(x.dtype)
    return _plain_mxgemm(state)


def _own(state):
    from kiosk_autoscaler_amd.ops import experts, mxfp4
    case = state['case']
    op = case['op']
    if op == 'route':
        plan = experts.route(state['logits'], case['k'])
        return {'experts': plan.experts, 'weights': plan.weights,
                'tokens': plan.tokens, 'positions': plan.positions,
                'offsets': plan.offsets}
    if op == 'grouped':
        a, b = state['a'], state['b']
        if case['mx']:
            a = mxfp4.quantize(a) if case['gather'] else mxfp4.Mxfp4(*a)
            b = mxfp4.Mxfp4(*b)
        return experts.grouped_gemm(a, b, state['offsets'],
                                    bias=state['bias'],
                                    epilogue=case['epilogue'],
                                    rows=state['rows'])
    if op == 'combine':
        return experts.combine(state['y'], state['positions'],
                               state['weights'],
                               residual=state['residual'])
    if op == 'quantize':
        x = state['x']
        return mxfp4.dequantize(mxfp4.quantize(x), dtype=x.dtype)
    return mxfp4.gemm(mxfp4.quantize(state['a']), mxfp4.Mxfp4(*state['b']),
                      bias=state['bias'], residual=state['residual'],
                      epilogue=case['epilogue'])


def run(state):
    """One pass through the case's operator, and its outputs."""
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_route(state):
    logits, k = state['logits'].double().cpu(), state['case']['k']
    tokens, experts = logits.shape
    low = float('-inf')
    # the rank of an expert in its row: how many stand before it
    left = logits.clone()
    chosen = torch.full((tokens, k), -1, dtype=torch.int64)
    weights = torch.zeros(tokens, k, dtype=torch.float64)
    peak = logits.amax(1)
    span = torch.arange(experts)
    for j in range(k):
        best = left.amax(1, keepdim=True)
        first = torch.where(left == best, span, experts).amin(1)
        live = best[:, 0] > low
        chosen[:, j] = torch.where(live, first, -1)
        weights[:, j] = torch.where(live, (best[:, 0] - peak).exp(), 0.0)
        left[torch.arange(tokens), first] = low
    weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-300)
    flat = chosen.reshape(-1)
    offsets = torch.zeros(experts + 1, dtype=torch.int64)
    positions = torch.full((tokens * k,), -1, dtype=torch.int64)
    row_tokens = torch.full((tokens * k,), -1, dtype=torch.int64)
    for e in range(experts):
        slots = (flat == e).nonzero()[:, 0]
        start = int(offsets[e])
        offsets[e + 1] = start + len(slots)
        positions[slots] = torch.arange(start, start + len(slots))
        row_tokens[start:start + len(slots)] = slots // k
    return {'experts': chosen.to(torch.int32), 'weights': weights,
            'tokens': row_tokens.to(torch.int32),
            'positions': positions.view(tokens, k).to(torch.int32),
            'offsets': offsets.to(torch.int32)}


def _exact_codec(x):
    """Each value's nearest neighbour on its block's grid, in 64 bits."""
    x = x.double()
    blocks = x.reshape(-1, BLOCK)
    out = torch.empty_like(blocks)
    # grid points with an even code first: a tie then falls to them
    grid = torch.tensor((0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0),
                        dtype=torch.float64, device=x.device)
    for start in range(0, len(blocks), 1 << 18):
        part = blocks[start:start + (1 << 18)]
        peak = part.abs().amax(1, keepdim=True)
        power = torch.floor(torch.log2(peak.clamp(min=2.0 ** -160)))
        # log2 may round up to a whole number just below a power of two
        power = power - (torch.pow(2.0, power) > peak).double()
        step = torch.pow(2.0, (power - 2).clamp(min=-127.0))
        nearest = (part.abs().unsqueeze(-1) / step.unsqueeze(-1)
                   - grid).abs().argmin(-1)
        out[start:start + (1 << 18)] = torch.copysign(grid[nearest] * step,
                                                      part)
    return out.view(x.shape)


def _exact_values(codes, scales):
    """What packed codes and scale bytes stand for, by the fields' bits."""
    fields = torch.stack((codes % 16, codes // 16), -1).flatten(-2).int()
    exponent, mantissa = (fields >> 1) & 3, (fields & 1).double()
    magnitude = torch.where(exponent == 0, mantissa * 0.5,
                            (1 + mantissa / 2)
                            * torch.pow(2.0, exponent.double() - 1))
    sign = 1.0 - 2.0 * (fields >> 3).double()
    scale = torch.pow(2.0, scales.double() - 127)
    return sign * magnitude * scale.repeat_interleave(BLOCK, -1)


def _exact_epilogue(y, epilogue, bias, residual=None):
    if epilogue != 'none':
        y = y + bias.double()
    if epilogue == 'gelu':
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi)
                               * (y + 0.044715 * y * y * y)))
    if residual is not None:
        y = y + residual.double()
    return y


def exact(case, seed):
    """What :func:`run` returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    op = case['op']
    if op == 'route':
        return _exact_route(state)
    if op == 'quantize':
        return _exact_codec(state['x'])
    if op == 'combine':
        out = state['residual'].double()
        y = state['y']
        for j in range(case['k']):
            place = state['positions'][:, j].long()
            live = place >= 0
            out[live] += y[place[live]].double() \
                * state['weights'][live, j].double().unsqueeze(1)
        return out
    if op == 'mxgemm':
        y = _exact_codec(state['a']) @ _exact_values(*state['b']).t()
        return _exact_epilogue(y, case['epilogue'], state['bias'],
                               state['residual'])
    a = state['a']
    if case['mx']:
        a = _exact_codec(a) if case['gather'] else _exact_values(*a)
    a = a.double()
    bounds, rows = state['bounds'], state['rows']
    out = torch.zeros(case['tokens'] * case['k'], case['outer'],
                      dtype=torch.float64, device=a.device)
    for e in range(case['experts']):
        span = torch.arange(bounds[e], bounds[e + 1], device=a.device)
        if len(span) == 0:
            continue
        b = _exact_values(state['b'][0][e], state['b'][1][e]) \
            if case['mx'] else state['b'][e].double()
        source = span if rows is None else rows[span].long()
        bias = None if state['bias'] is None else state['bias'][e]
        out[span] = _exact_epilogue(a[source] @ b.t(), case['epilogue'],
                                    bias)
    return out
