"""The operators around a layer of experts that stays in 16 bits, as cases that can be timed and compared: the norm in front of it, which adds the
residual and leaves the FP8 GEMM's operand, and its gradient; the layout of tokens sorted by expert without padding; and the experts' products on
groups of any size, forward, for the gradient of the rows and for the gradient of the weights.

`run` computes a case in elementary torch operations, or with the framework's entry points where `own` is true.
"""
import math

import torch

own = False

BLOCK = 128         # elements that share a scale
FP8_MAX = 448.0
EPS = 1e-6
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.half, 'fp32': torch.float32}


def listed():
    return [
        # a decode step of 64 sequences between two projections in FP8: one small launch, all latency
        {'name': 'norm_decode', 'op': 'norm', 'rows': 64, 'hidden': 7168, 'dtype': 'bf16', 'residual': 'bf16', 'codes': True, 'normed': False, 'col_major': True},
        # a prefill of 8192 tokens: codes for the projections, 16 bits for the router
        {'name': 'norm_prefill', 'op': 'norm', 'rows': 8192, 'hidden': 7168, 'dtype': 'bf16', 'residual': 'bf16', 'codes': True, 'normed': True, 'col_major': True},
        # the gradient of a norm without a residual, a ragged number of tokens of a width that is no multiple of 128
        {'name': 'norm_grad_ragged', 'op': 'norm_grad', 'rows': 1023, 'hidden': 2112, 'dtype': 'bf16', 'h': 'bf16', 'residual': False, 'accumulate': False},
        # the gradient of a training batch of 8192 tokens, the residual's added, the weight's onto what earlier micro-batches left
        {'name': 'norm_grad_train', 'op': 'norm_grad', 'rows': 8192, 'hidden': 7168, 'dtype': 'bf16', 'h': 'bf16', 'residual': True, 'accumulate': True},
        # a decode step's picks sorted by expert
        {'name': 'layout_decode', 'op': 'layout', 'tokens': 64, 'experts': 256, 'top_k': 8, 'padding': 0.0, 'skew': 1.0},
        # those of a training batch with padding at the ends of its sequences
        {'name': 'layout_train', 'op': 'layout', 'tokens': 16384, 'experts': 256, 'top_k': 8, 'padding': 0.07, 'skew': 1.0},
        # 64 tokens of a decode step, four experts each: the weights of 32 experts are read for a few rows each
        {'name': 'experts_decode', 'op': 'experts', 'tokens': 64, 'top_k': 4, 'groups': 32, 'n': 4096, 'k': 7168, 'dtype': 'bf16', 'gather': True, 'skew': 0.5},
        # a prefill of 4096 tokens, eight of 64 experts each, rows gathered out of the tokens' activations
        {'name': 'experts_prefill', 'op': 'experts', 'tokens': 4096, 'top_k': 8, 'groups': 64, 'n': 2048, 'k': 7168, 'dtype': 'bf16', 'gather': True, 'skew': 1.0},
        # the rows' gradient of a short fp16 sequence on fine-grained experts, many of them with a row or none
        {'name': 'rows_grad_few', 'op': 'rows_grad', 'tokens': 137, 'top_k': 2, 'groups': 32, 'n': 1024, 'k': 2048, 'dtype': 'fp16', 'skew': 2.0},
        # the rows' gradient of sixteen experts, 6144 rows in all, as many each as the router sends
        {'name': 'rows_grad_train', 'op': 'rows_grad', 'tokens': 1536, 'top_k': 4, 'groups': 16, 'n': 7168, 'k': 4096, 'dtype': 'bf16', 'skew': 1.0},
        # weight gradients of 32 fine-grained experts, most with few tokens, some with none, added to what earlier micro-batches left
        {'name': 'weights_grad_few', 'op': 'weights_grad', 'tokens': 2000, 'top_k': 1, 'groups': 32, 'm': 2048, 'n': 1024, 'dtype': 'bf16', 'gather': False, 'skew': 2.0,
         'accumulate': True},
        # weight gradients of sixteen experts, the activations of 1536 tokens gathered, four experts each
        {'name': 'weights_grad_train', 'op': 'weights_grad', 'tokens': 1536, 'top_k': 4, 'groups': 16, 'm': 4096, 'n': 7168, 'dtype': 'bf16', 'gather': True, 'skew': 1.0,
         'accumulate': False},
    ]


MOST_FLOP = 2.0 * 4096 * 8 * 2048 * 7168            # experts_prefill
MOST_WEIGHTS = 64 * 2048 * 7168


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _multiple(rng, low, high, of):
    return min(high, max(low, _log(rng, low, high) // of * of))


def draw(rng):
    op = rng.choice(['norm', 'norm_grad', 'layout', 'experts', 'rows_grad', 'weights_grad'])
    if op in ('norm', 'norm_grad'):
        codes = rng.random() < 0.6
        hidden = _multiple(rng, 128, 16384, 128) if codes else _multiple(rng, 8, 16384, 8)
        rows = _log(rng, 1, min(262144, 8192 * 7168 // hidden))
        if op == 'norm':
            return {'op': op, 'rows': rows, 'hidden': hidden, 'dtype': rng.choice(['bf16', 'bf16', 'fp32']), 'residual': rng.choice(['none', 'bf16', 'fp32']), 'codes': codes,
                    'normed': not codes or rng.random() < 0.3, 'col_major': rng.random() < 0.6}
        return {'op': op, 'rows': rows, 'hidden': hidden, 'dtype': rng.choice(['bf16', 'bf16', 'fp32']), 'h': rng.choice(['bf16', 'bf16', 'fp32']),
                'residual': rng.random() < 0.6, 'accumulate': rng.random() < 0.5}
    if op == 'layout':
        experts = _log(rng, 2, 512)
        return {'op': op, 'tokens': _log(rng, 1, 16384), 'experts': experts, 'top_k': rng.randint(1, min(8, experts)), 'padding': rng.choice([0.0, 0.1, 0.5]),
                'skew': rng.choice([0.0, 1.0, 2.0])}
    while True:
        groups = _log(rng, 2, 128)
        case = {'op': op, 'tokens': _log(rng, 1, 8192), 'top_k': rng.randint(1, min(8, groups)), 'groups': groups}
        first, second = _multiple(rng, 64, 7168, 8), _multiple(rng, 64, 7168, 8)
        case.update({'m': first, 'n': second} if op == 'weights_grad' else {'n': first, 'k': second})
        case.update(dtype=rng.choice(['bf16', 'bf16', 'fp16']), skew=rng.choice([0.0, 1.0, 2.0]))
        if op != 'rows_grad':
            case['gather'] = rng.random() < 0.6
        if op == 'weights_grad':
            case['accumulate'] = rng.random() < 0.5
        pairs = case['tokens'] * case['top_k']
        outputs = groups * first * second if op == 'weights_grad' else 0
        if 2.0 * pairs * first * second <= MOST_FLOP and groups * first * second <= MOST_WEIGHTS and 4 * outputs <= 2e9 and pairs * (first + second) <= 4e8:
            return case


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(int(seed) % (1 << 62) + 1)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device='cuda').to(dtype)


def _activations(g, rows, columns, dtype):
    """Normal values with a few columns a good deal larger than the others, as the activations of language models have them."""
    x = _normal(g, rows, columns)
    loud = torch.rand(columns, generator=g, device='cuda') < 0.01
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _routing(g, tokens, experts, top_k, skew, padding=0.0):
    """int32 [tokens, top_k]: different experts for every token, some of them asked for more than others; -1 for the tokens that are padding."""
    liking = skew * torch.randn(experts, generator=g, device='cuda')
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, generator=g, device='cuda').clamp(1e-9, 1 - 1e-7)))
    picks = torch.sort(liking + noise, dim=1, descending=True, stable=True).indices[:, :top_k]
    if padding:
        picks = torch.where((torch.rand(tokens, generator=g, device='cuda') < padding)[:, None], -1, picks)
    return picks.to(torch.int32).contiguous()


def _layout(indices, experts):
    """rows [tokens, top_k], source [tokens * top_k] and offsets [experts + 1]: an expert's rows in the order of the tokens, right behind those of the
    expert before it; -1 where a pick is none and, in `source`, behind the last row."""
    tokens, top_k = indices.shape
    flat = indices.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device='cuda')
    counts = torch.zeros(experts + 1, dtype=torch.long, device='cuda').scatter_add_(0, key, torch.ones_like(key))[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.long, device='cuda')
    offsets[1:] = counts.cumsum(0)
    source = torch.where(key[order] < experts, order // top_k, -1)
    return torch.where(flat < 0, -1, place).view(tokens, top_k).to(torch.int32), source.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    g, op = _generator(seed), case['op']
    s = dict(case)
    if op == 'norm':
        t, h = case['rows'], case['hidden']
        s['x'] = _activations(g, t, h, DTYPES[case['dtype']])
        s['sum'] = None if case['residual'] == 'none' else _activations(g, t, h, DTYPES[case['residual']])
        s['weight'] = (1 + 0.2 * _normal(g, h)).to(torch.bfloat16)
        s['out'] = torch.empty(t, h, dtype=torch.bfloat16, device='cuda') if case['normed'] else None
    elif op == 'norm_grad':
        t, h = case['rows'], case['hidden']
        s['grad'] = _normal(g, t, h, dtype=DTYPES[case['dtype']])
        s['x'] = _activations(g, t, h, DTYPES[case['h']])
        s['weight'] = (1 + 0.2 * _normal(g, h)).to(torch.bfloat16)
        s['inverse_rms'] = (s['x'].double().square().mean(1) + EPS).rsqrt().float()
        s['grad_residual'] = _normal(g, t, h, dtype=DTYPES[case['dtype']]) if case['residual'] else None
        s['grad_weight'] = _normal(g, h)
    elif op == 'layout':
        s['indices'] = _routing(g, case['tokens'], case['experts'], case['top_k'], case['skew'], case['padding'])
    else:
        groups, dtype, tokens, top_k = case['groups'], DTYPES[case['dtype']], case['tokens'], case['top_k']
        _, source, offsets = _layout(_routing(g, tokens, groups, top_k, case['skew']), groups)
        pairs, gather = tokens * top_k, case.get('gather', False)
        s['offsets'], s['ends'], s['source'] = offsets, offsets.tolist(), source if gather else None
        if op == 'weights_grad':
            s['lhs'] = _normal(g, pairs, case['m'], dtype=dtype)
            s['rhs'] = _activations(g, tokens if gather else pairs, case['n'], dtype)
            s['out'] = _normal(g, groups, case['m'], case['n'])
        else:
            n, k = case['n'], case['k']
            s['lhs'] = _activations(g, tokens if gather else pairs, k, dtype)
            s['rhs'] = (_normal(g, groups, *((k, n) if op == 'rows_grad' else (n, k))) / math.sqrt(k)).to(dtype)
            s['out'] = torch.empty(pairs, n, dtype=dtype, device='cuda')
    return s


# The plain forms

def _norm(s):
    x = s['x'].float()
    if s['sum'] is not None:
        s['sum'].copy_(x + s['sum'].float())
        x = s['sum'].float()
    inverse = 1 / torch.sqrt((x * x).sum(1) / x.size(1) + EPS)
    y = x * inverse[:, None] * s['weight'].float()
    out = {'inverse_rms': inverse}
    if s['sum'] is not None:
        out['sum'] = s['sum']
    if s['codes']:
        blocks = y.view(y.size(0), -1, BLOCK)
        amax = blocks.abs().amax(-1).clamp(min=1e-4)
        top = torch.full_like(amax, FP8_MAX)
        out['codes'], out['scales'] = (blocks * (top / amax)[..., None]).to(torch.float8_e4m3fn).view(y.shape), amax / top
        if s['col_major']:
            out['scales'] = out['scales'].t().contiguous().t()
    if s['normed']:
        s['out'].copy_(y)
        out['normed'] = s['out']
    return out


def _norm_grad(s):
    x, grad, inverse = s['x'].float(), s['grad'].float(), s['inverse_rms'][:, None]
    unit, pulled = x * inverse, grad * s['weight'].float()
    down = inverse * (pulled - unit * ((pulled * unit).sum(1, keepdim=True) / x.size(1)))
    if s['grad_residual'] is not None:
        down = down + s['grad_residual'].float()
    for_weight = (grad * unit).sum(0)
    if s['accumulate']:
        s['grad_weight'] += for_weight
    else:
        s['grad_weight'].copy_(for_weight)
    return {'grad': down.to(s['grad'].dtype), 'grad_weight': s['grad_weight']}


def _experts(s):
    lhs, rhs, ends = s['lhs'].float(), s['rhs'], s['ends']
    if s['source'] is not None:
        lhs = lhs[s['source'].long()]
    for g in range(s['groups']):            # the experts' numbers of rows differ: a product for each
        if ends[g] < ends[g + 1]:
            weight = rhs[g].float()
            s['out'][ends[g]:ends[g + 1]] = lhs[ends[g]:ends[g + 1]] @ (weight if s['op'] == 'rows_grad' else weight.t())
    return s['out']


def _weights_grad(s):
    lhs, rhs, ends = s['lhs'].float(), s['rhs'].float(), s['ends']
    if s['source'] is not None:
        rhs = rhs[s['source'].long()]
    for g in range(s['groups']):
        product = lhs[ends[g]:ends[g + 1]].t() @ rhs[ends[g]:ends[g + 1]]
        if s['accumulate']:
            s['out'][g] += product
        else:
            s['out'][g] = product
    return s['out']


def _plain_layout(s):
    return dict(zip(('rows', 'source', 'offsets'), _layout(s['indices'], s['experts'])))


# The framework's calls

def _own(s):
    import yan_amd as yan
    op = s['op']
    if op == 'norm':
        out = {}
        if s['codes']:
            out['codes'], out['scales'], out['inverse_rms'] = yan.rms_norm_to_fp8(s['x'], s['weight'], EPS, s['sum'], s['col_major'], s['out'])
        else:
            out['inverse_rms'] = yan.rms_norm(s['x'], s['weight'], s['out'], EPS, s['sum'])
        if s['sum'] is not None:
            out['sum'] = s['sum']
        if s['normed']:
            out['normed'] = s['out']
        return out
    if op == 'norm_grad':
        grad = yan.rms_norm_backward(s['grad'], s['x'], s['weight'], s['inverse_rms'], s['grad_weight'], s['grad_residual'], s['accumulate'])
        return {'grad': grad, 'grad_weight': s['grad_weight']}
    if op == 'layout':
        return dict(zip(('rows', 'source', 'offsets'), yan.moe_ragged_layout(s['indices'], s['experts'])))
    half = s['dtype'] == 'fp16'
    if op == 'experts':
        product = yan.m_grouped_gemm_fp16_fp16_fp16_nt_ragged if half else yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged
        product(s['lhs'], s['rhs'], s['out'], s['offsets'], s['source'])
    elif op == 'rows_grad':
        product = yan.m_grouped_gemm_fp16_fp16_fp16_nn_ragged if half else yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged
        product(s['lhs'], s['rhs'], s['out'], s['offsets'])
    else:
        product = yan.k_grouped_gemm_fp16_fp16_fp32_tn_ragged if half else yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged
        product(s['lhs'], s['rhs'], s['out'], s['offsets'], s['accumulate'], s['source'])
    return s['out']


_PLAIN = {'norm': _norm, 'norm_grad': _norm_grad, 'layout': _plain_layout, 'experts': _experts, 'rows_grad': _experts, 'weights_grad': _weights_grad}


def run(s):
    if own:
        return _own(s)
    return _PLAIN[s['op']](s)


def work(case):
    op = case['op']
    size = lambda name: torch.finfo(DTYPES[name]).bits // 8
    if op == 'norm':
        t, h = case['rows'], case['hidden']
        nbytes = t * h * size(case['dtype']) + 2 * h + 4 * t
        if case['residual'] != 'none':
            nbytes += 2 * t * h * size(case['residual'])
        nbytes += (t * h * (1 + 4 / BLOCK) if case['codes'] else 0) + (2 * t * h if case['normed'] else 0)
        flops = 8.0 * t * h
    elif op == 'norm_grad':
        t, h = case['rows'], case['hidden']
        nbytes = t * h * (2 * size(case['dtype']) + size(case['h']) + (size(case['dtype']) if case['residual'] else 0)) + 4 * t + h * (10 if case['accumulate'] else 6)
        flops = 12.0 * t * h
    elif op == 'layout':
        pairs = case['tokens'] * case['top_k']
        nbytes, flops = 12 * pairs + 4 * case['experts'] + 4, 2.0 * pairs
    else:
        pairs, groups = case['tokens'] * case['top_k'], case['groups']
        used = min(groups, pairs)           # groups that can have rows
        if op == 'weights_grad':
            m, n = case['m'], case['n']
            nbytes = 2 * (pairs * m + (case['tokens'] if case['gather'] else pairs) * n) + (8 * used if case['accumulate'] else 4 * groups) * m * n
        else:
            n, k = case['n'], case['k']
            m = k
            nbytes = 2 * ((case['tokens'] if case.get('gather') else pairs) * k + used * n * k + pairs * n)
        nbytes += 4 * groups + 4 + (4 * pairs if case.get('gather') else 0)
        flops = 2.0 * pairs * m * n
    return {'bytes': float(nbytes), 'flops': float(flops)}


# The definitions in 64 bits

def _e4m3(v):
    """Nearest e4m3 value of every element, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s, op = prepare(case, seed), case['op']
    if op == 'norm':
        v = s['x'].double()
        if s['sum'] is not None:
            v = (v + s['sum'].double()).to(s['sum'].dtype).double()
        rms = torch.sqrt(v.pow(2).mean(1, keepdim=True) + EPS)
        y = v / rms * s['weight'].double()
        out = {'inverse_rms': (1 / rms)[:, 0]}
        if s['sum'] is not None:
            out['sum'] = v
        if case['codes']:
            groups = y.unflatten(1, (-1, BLOCK))
            top = groups.abs().max(2, keepdim=True).values.clamp(min=float(torch.tensor(1e-4)))
            out['codes'], out['scales'] = _e4m3(groups * FP8_MAX / top).flatten(1), (top / FP8_MAX)[..., 0]
        if case['normed']:
            out['normed'] = y
        return out
    if op == 'norm_grad':
        v, d, w = s['x'].double(), s['grad'].double(), s['weight'].double()
        r = s['inverse_rms'].double()[:, None]
        dot = (d * w * v).mean(1, keepdim=True)
        down = r * d * w - r.pow(3) * v * dot
        if case['residual']:
            down = down + s['grad_residual'].double()
        total = (d * v * r).sum(0)
        return {'grad': down, 'grad_weight': total + s['grad_weight'].double() if case['accumulate'] else total}
    if op == 'layout':
        return None
    lhs, rhs = s['lhs'].double(), s['rhs']
    if op == 'weights_grad':
        rhs = rhs.double()
        out = s['out'].double() if case['accumulate'] else torch.zeros_like(s['out'], dtype=torch.float64)
        for g in range(case['groups']):
            at = slice(s['ends'][g], s['ends'][g + 1])
            picked = rhs[at] if s['source'] is None else rhs.index_select(0, s['source'][at].long())
            out[g] += torch.mm(lhs[at].t().contiguous(), picked)
        return out
    out = torch.zeros(s['out'].shape, dtype=torch.float64, device='cuda')
    for g in range(case['groups']):
        at = slice(s['ends'][g], s['ends'][g + 1])
        picked = lhs[at] if s['source'] is None else lhs.index_select(0, s['source'][at].long())
        weight = rhs[g].double()
        out[at] = torch.mm(picked, weight if op == 'rows_grad' else weight.t().contiguous())
    return out
