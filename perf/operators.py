"""The operators of a mixture-of-experts layer around the grouped FP8 GEMMs, as cases that can be timed and compared: the
router with its balance loss, the way of tokens into the experts' rows and back, and the weight gradients of the experts
with the quantiser that makes their operands. Forward for serving, forward and backward for training.

`run` computes a case in elementary torch operations, or with the framework's entry points where `own` is true.
"""
import math

import torch

own = False

BLOCK = 128         # elements along K that share a scale; also the alignment of an expert's rows
FP8_MAX = 448.0
LEAST_AMAX = 2.0 ** -100            # a block of zeros has the exponent of this maximum
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
    return [
        # a decode step of 64 sequences: one small router, all latency
        {'name': 'route_decode', 'op': 'route', 'tokens': 64, 'experts': 256, 'top_k': 8, 'dtype': 'bf16', 'scoring': 'softmax',
         'renormalize': True, 'padding': 0.0, 'train': False},
        # a training batch with padding at the ends of its sequences: loss, counts and the gradient of the logits
        {'name': 'route_train', 'op': 'route', 'tokens': 16384, 'experts': 256, 'top_k': 8, 'dtype': 'fp32', 'scoring': 'sigmoid',
         'renormalize': True, 'padding': 0.07, 'train': True},
        # the same decode step's tokens on their way to 32 experts in fixed slots of 64 rows
        {'name': 'dispatch_decode', 'op': 'dispatch', 'layout': 'masked', 'tokens': 64, 'hidden': 7168, 'experts': 32, 'top_k': 4, 'm_max': 64,
         'dtype': 'bf16', 'skew': 0.5},
        # a prefill of 8192 tokens, eight experts each, into the contiguous layout
        {'name': 'dispatch_prefill', 'op': 'dispatch', 'layout': 'contiguous', 'tokens': 8192, 'hidden': 7168, 'experts': 64, 'top_k': 8, 'm_max': 0,
         'dtype': 'bf16', 'skew': 1.0},
        # the experts' outputs of a decode step back to its tokens
        {'name': 'combine_decode', 'op': 'combine', 'tokens': 64, 'hidden': 7168, 'experts': 32, 'top_k': 4, 'skew': 0.5, 'weighted': True, 'train': False},
        # an odd number of training tokens, there and back: outputs, then the gradients of expert outputs and weights
        {'name': 'combine_train', 'op': 'combine', 'tokens': 4097, 'hidden': 4096, 'experts': 64, 'top_k': 8, 'skew': 1.0, 'weighted': True, 'train': True},
        # gradients of a dense layer's outputs for a ragged number of tokens, in fp32, on their way into a weight gradient
        {'name': 'cast_ragged', 'op': 'cast', 'rows': 1023, 'columns': 2112, 'dtype': 'fp32', 'gather': 0, 'skew': 0.0},
        # activations of 4096 tokens, gathered into the rows of sixteen experts (four each) and turned round
        {'name': 'cast_gathered', 'op': 'cast', 'rows': 4096, 'columns': 7168, 'dtype': 'bf16', 'gather': 4, 'skew': 1.0},
        # the weight gradient of a small projection over a short sequence
        {'name': 'wgrad_small', 'op': 'wgrad', 'm': 512, 'n': 1536, 'tokens': 1024, 'accumulate': False},
        # the weight gradient of a large layer over 16384 tokens, added to what earlier micro-batches left
        {'name': 'wgrad_large', 'op': 'wgrad', 'm': 7168, 'n': 4096, 'tokens': 16384, 'accumulate': True},
        # 32 experts of a fine-grained layer, most of them with few tokens, some with none
        {'name': 'wgrad_experts_few', 'op': 'wgrad_experts', 'groups': 32, 'm': 2048, 'n': 1024, 'tokens': 2000, 'skew': 2.0, 'accumulate': True},
        # sixteen experts, 6144 rows in all, as many each as the router sends
        {'name': 'wgrad_experts', 'op': 'wgrad_experts', 'groups': 16, 'm': 4096, 'n': 7168, 'tokens': 6144, 'skew': 1.0, 'accumulate': False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _multiple(rng, low, high, of):
    return min(high, max(low, _log(rng, low, high) // of * of))


def draw(rng):
    op = rng.choice(['route', 'dispatch', 'combine', 'cast', 'wgrad', 'wgrad_experts'])
    if op == 'route':
        experts = _log(rng, 4, 512)
        return {'op': op, 'tokens': _log(rng, 1, min(32768, 16384 * 256 // experts)), 'experts': experts, 'top_k': rng.randint(1, min(8, experts)),
                'dtype': rng.choice(['bf16', 'fp32']), 'scoring': rng.choice(['softmax', 'sigmoid']), 'renormalize': rng.random() < 0.7,
                'padding': rng.choice([0.0, 0.1, 0.5]), 'train': rng.random() < 0.6}
    if op == 'dispatch':
        tokens, experts, hidden = _log(rng, 1, 8192), _log(rng, 2, 256), _multiple(rng, 128, 7168, 128)
        masked = tokens <= 256 and rng.random() < 0.6
        return {'op': op, 'layout': 'masked' if masked else 'contiguous', 'tokens': tokens, 'hidden': hidden, 'experts': experts,
                'top_k': rng.randint(1, min(8, experts)), 'm_max': rng.choice([16, 64, 100, 256]) if masked else 0, 'dtype': rng.choice(['bf16', 'fp32']),
                'skew': rng.choice([0.0, 1.0, 2.0])}
    if op == 'combine':
        tokens, experts = _log(rng, 1, 4097), _log(rng, 2, 256)
        return {'op': op, 'tokens': tokens, 'hidden': _multiple(rng, 64, 4096, 8), 'experts': experts, 'top_k': rng.randint(1, min(8, experts)),
                'skew': rng.choice([0.0, 1.0, 2.0]), 'weighted': rng.random() < 0.7, 'train': rng.random() < 0.5}
    if op == 'cast':
        gather = rng.choice([0, 0, 1, 4])
        return {'op': op, 'rows': _log(rng, 1, 4096), 'columns': _multiple(rng, 8, 7168, 8), 'dtype': rng.choice(['bf16', 'fp32']), 'gather': gather,
                'skew': rng.choice([0.0, 1.0])}
    if op == 'wgrad':
        while True:
            m, n, tokens = _log(rng, 16, 8192), _multiple(rng, 16, 8192, 4), _log(rng, 1, 32768)
            if 2.0 * m * n * tokens <= 9.6e11 and (m + n) * tokens <= 3e8:
                return {'op': op, 'm': m, 'n': n, 'tokens': tokens, 'accumulate': rng.random() < 0.5}
    while True:
        groups, m, n, tokens = _log(rng, 2, 64), _log(rng, 64, 4096), _multiple(rng, 64, 7168, 4), _log(rng, 1, 32768)
        if 2.0 * m * n * tokens <= 9.6e11 and 4 * groups * m * n <= 1.9e9 and (m + n) * tokens <= 3e8:
            return {'op': op, 'groups': groups, 'm': m, 'n': n, 'tokens': tokens, 'skew': rng.choice([0.0, 1.0, 2.0]), 'accumulate': rng.random() < 0.5}


def _ceil(x, y):
    return -(-x // y)


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) % (1 << 62) + 1)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device='cuda').to(dtype)


def _activations(g, rows, columns, dtype):
    """Normal values with a few columns a good deal larger than the others, as the activations of language models have them."""
    x = _normal(g, rows, columns)
    loud = torch.rand(columns, generator=g, device='cuda') < 0.01
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _routing(g, tokens, experts, top_k, skew):
    """int32 [tokens, top_k]: different experts for every token, some of them asked for more than others."""
    liking = skew * torch.randn(experts, generator=g, device='cuda')
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, generator=g, device='cuda').clamp(1e-9, 1 - 1e-7)))
    return torch.sort(liking + noise, dim=1, descending=True, stable=True).indices[:, :top_k].to(torch.int32).contiguous()


def _counts(flat, experts):
    return torch.zeros(experts, dtype=torch.long, device='cuda').scatter_add_(0, flat, torch.ones_like(flat))


def _layout(indices, experts, capacity):
    """(rows [tokens, top_k], tokens [capacity], starts [experts + 1]) of the contiguous layout: an expert's rows in the order of the tokens,
    every expert from a multiple of BLOCK on."""
    tokens, top_k = indices.shape
    flat = indices.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    counts = _counts(flat, experts)
    starts = torch.zeros(experts + 1, dtype=torch.long, device='cuda')
    starts[1:] = ((counts + BLOCK - 1) // BLOCK * BLOCK).cumsum(0)
    before = counts.cumsum(0) - counts
    by_expert = flat[order]
    place = starts[by_expert] + torch.arange(flat.numel(), device='cuda') - before[by_expert]
    rows = torch.empty_like(flat)
    rows[order] = place
    source = torch.full((capacity, ), -1, dtype=torch.int32, device='cuda')
    source[place] = (order // top_k).to(torch.int32)
    return rows.view(tokens, top_k).to(torch.int32), source, starts.to(torch.int32)


def _capacity(tokens, top_k, experts):
    """Rows that the contiguous layout takes at most."""
    pairs = tokens * top_k
    return (pairs + (BLOCK - 1) * min(experts, pairs)) // BLOCK * BLOCK


def _power_of_two_cast(x):
    """x [rows, K] fp32 with K % BLOCK == 0 -> (e4m3 codes, exponents + 127 as uint8, their rows a multiple of four bytes apart)."""
    rows, k = x.shape
    blocks = x.view(rows, k // BLOCK, BLOCK)
    fraction, exponent = torch.frexp(blocks.abs().amax(-1).clamp(min=LEAST_AMAX))
    exponent = exponent - 9 + (fraction > FP8_MAX / 512).int()          # the smallest with amax <= 448 * 2 ** exponent
    codes = torch.ldexp(blocks, -exponent[..., None]).to(torch.float8_e4m3fn).view(rows, k)
    scales = torch.zeros(rows, _ceil(k // BLOCK, 4) * 4, dtype=torch.uint8, device=x.device)[:, :k // BLOCK]
    scales.copy_(exponent + 127)
    return codes, scales


def _operand(g, rows, valid):
    """A weight gradient's operand [rows, K]: gradients or activations with the tokens along K, quantised; `valid` [K] marks the columns that hold one."""
    k = valid.numel()
    x = _normal(g, rows, k) * torch.exp(0.5 * _normal(g, rows, 1))
    return _power_of_two_cast(x * valid)


def prepare(case, seed):
    g, op = _generator(seed), case['op']
    s = dict(case)
    if op == 'route':
        t, e, k = case['tokens'], case['experts'], case['top_k']
        s['logits'] = (1.5 * _normal(g, t, e) + 0.7 * _normal(g, 1, e)).to(DTYPES[case['dtype']])
        s['mask'] = torch.rand(t, generator=g, device='cuda') >= case['padding'] if case['padding'] else None
        if case['train']:
            s['grad_weights'], s['grad_loss'] = _normal(g, t, k), torch.full((), 0.01 * t, device='cuda') * (1 + 0.1 * _normal(g, 1)[0])
    elif op == 'dispatch':
        t, h, e = case['tokens'], case['hidden'], case['experts']
        s['x'] = _activations(g, t, h, DTYPES[case['dtype']])
        s['indices'] = _routing(g, t, e, case['top_k'], case['skew'])
        shape = (e, case['m_max']) if case['layout'] == 'masked' else (_capacity(t, case['top_k'], e), )
        s['codes'] = torch.zeros(*shape, h, dtype=torch.float8_e4m3fn, device='cuda')
        s['scales'] = torch.zeros(*shape[:-1], h // BLOCK, shape[-1], device='cuda').transpose(-1, -2)
    elif op == 'combine':
        t, h, e, k = case['tokens'], case['hidden'], case['experts'], case['top_k']
        s['rows'], s['source'], _ = _layout(_routing(g, t, e, k, case['skew']), e, _capacity(t, k, e))
        s['y'] = _normal(g, s['source'].numel(), h, dtype=torch.bfloat16)
        s['weights'] = torch.softmax(_normal(g, t, k), 1) if case['weighted'] else None
        s['out'] = torch.empty(t, h, dtype=torch.bfloat16, device='cuda')
        s['grad_out'] = _normal(g, t, h, dtype=torch.bfloat16) if case['train'] else None
    elif op == 'cast':
        s['x'] = _activations(g, case['rows'], case['columns'], DTYPES[case['dtype']])
        s['source'] = None
        if case['gather']:
            s['source'] = _layout(_routing(g, case['rows'], 16, case['gather'], case['skew']), 16, _capacity(case['rows'], case['gather'], 16))[1]
    elif op == 'wgrad':
        k = _ceil(case['tokens'], BLOCK) * BLOCK
        valid = (torch.arange(k, device='cuda') < case['tokens']).float()
        s['lhs'], s['rhs'] = _operand(g, case['m'], valid), _operand(g, case['n'], valid)
        s['out'] = _normal(g, case['m'], case['n'])
    else:
        groups, tokens = case['groups'], case['tokens']
        _, source, starts = _layout(_routing(g, tokens, groups, 1, case['skew']), groups, _capacity(tokens, 1, groups))
        valid = (source >= 0).float()
        s['lhs'], s['rhs'] = _operand(g, case['m'], valid), _operand(g, case['n'], valid)
        s['offsets'], s['ends'] = starts, starts.tolist()
        s['out'] = _normal(g, groups, case['m'], case['n'])
    return s


# The plain forms

def _route(s):
    logits, k, e = s['logits'].float(), s['top_k'], s['experts']
    live = torch.ones(logits.size(0), dtype=torch.bool, device='cuda') if s['mask'] is None else s['mask']
    score = torch.softmax(logits, 1) if s['scoring'] == 'softmax' else torch.sigmoid(logits)
    picked = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    weights = score.gather(1, picked)
    chosen = weights.sum(1, keepdim=True)
    if s['renormalize']:
        weights = weights / chosen
    weights = weights * live[:, None]
    total = score.sum(1, keepdim=True)
    share = score if s['scoring'] == 'softmax' else score / total
    counts = torch.zeros(e, device='cuda').scatter_add_(0, picked.reshape(-1), live[:, None].expand(-1, k).reshape(-1).float())
    tokens = live.sum().clamp(min=1)
    pull = e * counts / (k * tokens * tokens)
    loss = (pull * (share * live[:, None]).sum(0)).sum()
    out = {'weights': weights, 'indices': torch.where(live[:, None], picked, -1).to(torch.int32), 'counts': counts.to(torch.int32), 'loss': loss}
    if s['train']:
        down = s['grad_weights']
        if s['renormalize']:
            down = (down - (weights * down).sum(1, keepdim=True)) / chosen
        grad = torch.zeros_like(score).scatter_(1, picked, down)
        pull = s['grad_loss'] * pull
        if s['scoring'] == 'softmax':
            grad = grad + pull
            grad = score * (grad - (score * grad).sum(1, keepdim=True))
        else:
            grad = (grad + (pull - (share * pull).sum(1, keepdim=True)) / total) * score * (1 - score)
        out['grad_logits'] = (grad * live[:, None]).to(s['logits'].dtype)
    return out


def _quantise_tokens(x):
    groups = x.float().view(x.size(0), -1, BLOCK)
    amax = groups.abs().amax(-1).clamp(min=1e-4)
    factor = torch.full_like(amax, FP8_MAX) / amax
    return (groups * factor[..., None]).to(torch.float8_e4m3fn).view(x.shape), amax / torch.full_like(amax, FP8_MAX)


def _dispatch(s):
    indices, e = s['indices'], s['experts']
    t, k = indices.shape
    codes, scales = _quantise_tokens(s['x'])
    if s['layout'] == 'masked':
        slots, flat = s['m_max'], indices.reshape(-1).long()
        order = torch.sort(flat, stable=True).indices
        counts = _counts(flat, e)
        rank = torch.empty_like(flat)
        rank[order] = torch.arange(flat.numel(), device='cuda') - (counts.cumsum(0) - counts)[flat[order]]
        kept = rank < slots
        row = flat * slots + rank
        token = torch.arange(t * k, device='cuda') // k
        s['codes'].view(torch.uint8).view(e * slots, -1)[row[kept]] = codes.view(torch.uint8)[token[kept]]
        s['scales'][flat[kept], rank[kept]] = scales[token[kept]]
        return {'codes': s['codes'], 'scales': s['scales'], 'rows': torch.where(kept, row, -1).view(t, k).to(torch.int32),
                'masked_m': counts.clamp(max=slots).to(torch.int32)}
    rows, source, starts = _layout(indices, e, s['codes'].size(0))
    row, token = rows.reshape(-1).long(), torch.arange(t * k, device='cuda') // k
    s['codes'].view(torch.uint8)[row] = codes.view(torch.uint8)[token]
    s['scales'][row] = scales[token]
    row = torch.arange(source.numel(), device='cuda', dtype=torch.int32)
    group = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    m_indices = torch.where(row < starts[-1], group, -1).to(torch.int32)
    return {'codes': s['codes'], 'scales': s['scales'], 'rows': rows, 'm_indices': m_indices, 'source': source, 'offsets': starts}


def _combine(s):
    t, h, k = s['tokens'], s['hidden'], s['top_k']
    weights = torch.ones(t, k, device='cuda') if s['weights'] is None else s['weights']
    taken = s['y'][s['rows'].reshape(-1).long()].view(t, k, h).float()
    out = {'out': (taken * weights[..., None]).sum(1).to(torch.bfloat16)}
    if s['train']:
        grad = s['grad_out'].float()
        grad_y = torch.zeros_like(s['y'])
        grad_y[s['rows'].reshape(-1).long()] = (weights[..., None] * grad[:, None]).to(torch.bfloat16).view(t * k, h)
        out['grad_y'] = grad_y
        if s['weights'] is not None:
            out['grad_weights'] = (taken * grad[:, None]).sum(-1)
    return out


def _cast(s):
    x, source = s['x'].float(), s['source']
    if source is None:
        wide = torch.zeros(_ceil(x.size(0), BLOCK) * BLOCK, x.size(1), device='cuda')
        wide[:x.size(0)] = x
    else:
        wide = x[source.clamp(min=0).long()] * (source >= 0)[:, None]
    return dict(zip(('codes', 'scales'), _power_of_two_cast(wide.t().contiguous())))


def _decoded(operand):
    codes, scales = operand
    rows, k = codes.shape
    return torch.ldexp(codes.float().view(rows, -1, BLOCK), (scales.int() - 127)[..., None]).view(rows, k)


def _wgrad(s):
    product = _decoded(s['lhs']) @ _decoded(s['rhs']).t()
    if s['accumulate']:
        s['out'] += product
    else:
        s['out'].copy_(product)
    return s['out']


def _wgrad_experts(s):
    lhs, rhs, ends = _decoded(s['lhs']), _decoded(s['rhs']), s['ends']
    for g in range(s['groups']):            # the experts' numbers of tokens differ: a product for each
        product = lhs[:, ends[g]:ends[g + 1]] @ rhs[:, ends[g]:ends[g + 1]].t()
        if s['accumulate']:
            s['out'][g] += product
        else:
            s['out'][g] = product
    return s['out']


# The framework's calls

def _own(s):
    import yan_amd as yan
    op = s['op']
    if op == 'route':
        weights, indices, counts, loss = yan.moe_route(s['logits'], s['top_k'], s['scoring'], s['renormalize'], s['mask'])
        out = {'weights': weights, 'indices': indices, 'counts': counts, 'loss': loss}
        if s['train']:
            out['grad_logits'] = yan.moe_route_backward(s['logits'], indices, counts, s['grad_weights'], s['grad_loss'], s['scoring'], s['renormalize'])
        return out
    if op == 'dispatch':
        buffers = (s['codes'], s['scales'])
        if s['layout'] == 'masked':
            rows, masked_m = yan.moe_dispatch_to_fp8_masked(s['x'], s['indices'], buffers)
            return {'codes': s['codes'], 'scales': s['scales'], 'rows': rows, 'masked_m': masked_m}
        rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(s['x'], s['indices'], s['experts'], buffers)
        return {'codes': s['codes'], 'scales': s['scales'], 'rows': rows, 'm_indices': m_indices, 'source': source, 'offsets': offsets}
    if op == 'combine':
        yan.moe_combine(s['y'], s['rows'], s['weights'], s['out'])
        out = {'out': s['out']}
        if s['train']:
            out['grad_y'], grad_weights = yan.moe_combine_backward(s['grad_out'], s['y'], s['rows'], s['weights'], s['source'])
            if s['weights'] is not None:
                out['grad_weights'] = grad_weights
        return out
    if op == 'cast':
        return dict(zip(('codes', 'scales'), yan.per_channel_cast_to_fp8(s['x'], s['source'])))
    if op == 'wgrad':
        yan.gemm_fp8_fp8_fp32_nt(s['lhs'], s['rhs'], s['out'], accumulate=s['accumulate'])
    else:
        yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(s['lhs'], s['rhs'], s['out'], s['offsets'], accumulate=s['accumulate'])
    return s['out']


_PLAIN = {'route': _route, 'dispatch': _dispatch, 'combine': _combine, 'cast': _cast, 'wgrad': _wgrad, 'wgrad_experts': _wgrad_experts}


def run(s):
    if own:
        return _own(s)
    return _PLAIN[s['op']](s)


def work(case):
    op = case['op']
    if op == 'route':
        t, e, k = case['tokens'], case['experts'], case['top_k']
        size = 2 if case['dtype'] == 'bf16' else 4
        nbytes, flops = t * e * size + t * k * 8 + e * 4 + (t if case['padding'] else 0), 8.0 * t * e
        if case['train']:
            nbytes += 2 * t * e * size + t * k * 8 + e * 4
            flops += 12.0 * t * e
    elif op == 'dispatch':
        t, h, k = case['tokens'], case['hidden'], case['top_k']
        kept = t * k if case['layout'] == 'contiguous' else min(t * k, case['experts'] * case['m_max'])
        nbytes, flops = t * h * (2 if case['dtype'] == 'bf16' else 4) + t * k * 8 + kept * (h + h // BLOCK * 4), 3.0 * t * h
        if case['layout'] == 'contiguous':
            nbytes += 8 * _capacity(t, k, case['experts'])
    elif op == 'combine':
        t, h, k = case['tokens'], case['hidden'], case['top_k']
        nbytes, flops = t * k * h * 2 + t * h * 2 + t * k * 8, 2.0 * t * k * h
        if case['train']:
            nbytes += t * h * 2 + (t * k * h * 2 if case['weighted'] else 0) + _capacity(t, k, case['experts']) * h * 2
            flops += 3.0 * t * k * h
    elif op == 'cast':
        n = case['columns']
        m = _capacity(case['rows'], case['gather'], 16) if case['gather'] else _ceil(case['rows'], BLOCK) * BLOCK
        nbytes, flops = case['rows'] * n * (2 if case['dtype'] == 'bf16' else 4) + m * n + m * n // BLOCK, 3.0 * m * n
    else:
        groups, tokens = case.get('groups', 1), case['tokens']
        outputs = groups * case['m'] * case['n']
        nbytes = (case['m'] + case['n']) * tokens * (1 + 1 / BLOCK) + outputs * (8 if case['accumulate'] else 4)
        flops = 2.0 * case['m'] * case['n'] * tokens
    return {'bytes': float(nbytes), 'flops': float(flops)}


# The definitions in 64 bits

def _e4m3(v):
    """Nearest e4m3 value of every element, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s, op = prepare(case, seed), case['op']
    if op == 'route':
        l, k, e = s['logits'].double(), case['top_k'], case['experts']
        live = torch.ones(l.size(0), device='cuda').double() if s['mask'] is None else s['mask'].double()
        exps = torch.exp(l - l.max(1, keepdim=True).values)
        score = exps / exps.sum(1, keepdim=True) if case['scoring'] == 'softmax' else 1 / (1 + torch.exp(-l))
        p = score / score.sum(1, keepdim=True)
        at = torch.argsort(l, dim=1, descending=True, stable=True)[:, :k]
        hot = torch.zeros_like(l).scatter_(1, at, 1.0)
        norm = (score * hot).sum(1, keepdim=True) if case['renormalize'] else torch.ones_like(l[:, :1])
        weights = (score / norm).gather(1, at) * live[:, None]
        counts, n = (hot * live[:, None]).sum(0), max(1.0, float(live.sum()))
        force = e * counts / (k * n * n)
        out = {'weights': weights, 'indices': None, 'counts': None, 'loss': (force * (p * live[:, None]).sum(0)).sum()}
        if case['train']:
            dw = torch.zeros_like(l).scatter_(1, at, s['grad_weights'].double())
            slope = score if case['scoring'] == 'softmax' else score * (1 - score)         # of the score, or its own part of it
            ds = hot * (dw - ((score / norm) * dw).sum(1, keepdim=True)) / norm if case['renormalize'] else dw
            dp = s['grad_loss'].double() * force
            if case['scoring'] == 'softmax':
                grad = slope * (ds + dp) - score * (score * (ds + dp)).sum(1, keepdim=True)
            else:
                grad = slope * (ds + (dp - (p * dp).sum(1, keepdim=True)) / score.sum(1, keepdim=True))
            out['grad_logits'] = grad * live[:, None]
        return out
    if op == 'dispatch':
        t, k = s['indices'].shape
        x = s['x'].double().view(t, -1, BLOCK)
        amax = x.abs().amax(2).clamp(min=float(torch.tensor(1e-4)))
        codes = _e4m3(x * (FP8_MAX / amax)[..., None]).view(t, -1)
        scales = amax / FP8_MAX
        out_codes, out_scales = torch.zeros(s['codes'].shape, device='cuda', dtype=torch.float32), torch.zeros(s['scales'].shape, device='cuda').double()
        chosen = s['indices'].cpu().tolist()
        filled, places = {}, []
        for token in range(t):
            for expert in chosen[token]:
                places.append((expert, filled.get(expert, 0), token))
                filled[expert] = filled.get(expert, 0) + 1
        if case['layout'] == 'masked':
            kept = torch.tensor([p for p in places if p[1] < case['m_max']], device='cuda')
            out_codes[kept[:, 0], kept[:, 1]] = codes[kept[:, 2]].float()
            out_scales[kept[:, 0], kept[:, 1]] = scales[kept[:, 2]]
            return {'codes': out_codes, 'scales': out_scales, 'rows': None, 'masked_m': None}
        start, at = 0, {}
        for expert in range(case['experts']):
            at[expert], start = start, start + _ceil(filled.get(expert, 0), BLOCK) * BLOCK
        kept = torch.tensor([(at[p[0]] + p[1], p[2]) for p in places], device='cuda')
        out_codes[kept[:, 0]] = codes[kept[:, 1]].float()
        out_scales[kept[:, 0]] = scales[kept[:, 1]]
        return {'codes': out_codes, 'scales': out_scales, 'rows': None, 'm_indices': None, 'source': None, 'offsets': None}
    if op == 'combine':
        t, h, k = case['tokens'], case['hidden'], case['top_k']
        y, rows = s['y'].double(), s['rows'].long()
        w = torch.ones(t, k, device='cuda').double() if s['weights'] is None else s['weights'].double()
        total = torch.zeros(t, h, device='cuda').double()
        for i in range(k):
            total += w[:, i, None] * y[rows[:, i]]
        out = {'out': total}
        if case['train']:
            d = s['grad_out'].double()
            grad_y, grad_w = torch.zeros_like(y), torch.zeros(t, k, device='cuda').double()
            for i in range(k):
                grad_y[rows[:, i]] = w[:, i, None] * d
                grad_w[:, i] = (d * y[rows[:, i]]).sum(1)
            out['grad_y'] = grad_y
            if s['weights'] is not None:
                out['grad_weights'] = grad_w
        return out
    if op == 'cast':
        x, source = s['x'].double(), s['source']
        if source is None:
            wide = torch.cat([x, x.new_zeros(-x.size(0) % BLOCK, x.size(1))])
        else:
            wide = torch.where((source >= 0)[:, None], x[source.clamp(min=0).long()], x.new_zeros(()))
        v = wide.view(-1, BLOCK, x.size(1))
        e = torch.ceil(torch.log2(v.abs().amax(1).clamp(min=LEAST_AMAX) / FP8_MAX))
        return {'codes': _e4m3(v / torch.exp2(e)[:, None]).reshape(wide.shape).t().contiguous(), 'scales': None}
    a, b = ((c.double().view(c.size(0), -1, BLOCK) * torch.exp2(e.double() - 127)[..., None]).view(c.shape) for c, e in (s['lhs'], s['rhs']))
    keep = s['out'].double() if case['accumulate'] else torch.zeros_like(s['out'], dtype=torch.float64)
    if op == 'wgrad':
        return keep + a @ b.t().contiguous()
    for g in range(case['groups']):
        lo, hi = s['ends'][g], s['ends'][g + 1]
        keep[g] += a[:, lo:hi].contiguous() @ b[:, lo:hi].t().contiguous()
    return keep
