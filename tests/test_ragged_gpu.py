"""The ragged layout and the 16-bit products on it, on the GPU: each against its definition in 64 bits, and all of them in a row."""
import pytest
import torch

import harness as testing
import yan_amd as yan
from yan_amd.jit_kernels import ragged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _close(got, want, bound, what=''):
    off = (got.double() - want.double()).abs()
    assert bool((off <= bound).all()), f'{what}: {int((~(off <= bound)).sum())} of {off.numel()} further off than they may be, by up to {float((off - bound).max()):.3g}'


# The layout

def _layout_reference(indices, experts):
    flat = indices.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device='cuda')
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device='cuda')
    offsets[1:] = counts.cumsum(0)
    rows = torch.where(key < experts, place, -1).view(indices.shape).int()
    source = torch.where(key[order] < experts, order // indices.size(1), -1).int()
    return rows, source, offsets


@pytest.mark.parametrize('tokens,experts,top_k', [(0, 4, 2), (1, 1, 1), (1, 256, 8), (64, 256, 8), (37, 7, 5), (511, 3, 16), (1024, 1024, 8), (1025, 65, 8), (5000, 64, 3),
                                                  (16384, 256, 8), (70001, 100, 4), (40000, 1000, 16)])
def test_layout(tokens, experts, top_k):
    g = _gen(tokens + experts)
    for kind in ('spread', 'padded', 'one', 'none', 'foreign'):
        picks = torch.randint(0, experts, (tokens, top_k), generator=g, device='cuda', dtype=torch.int32)         # (an expert may come twice)
        if kind == 'padded':
            picks[torch.rand(tokens, generator=g, device='cuda') < 0.3] = -1
        elif kind == 'one':
            picks.fill_(experts - 1)
        elif kind == 'none':
            picks.fill_(-1)
        elif kind == 'foreign':
            picks = torch.where(torch.rand(tokens, top_k, generator=g, device='cuda') < 0.2, experts + (1 << 20), picks)
        want = _layout_reference(picks, experts)
        for _ in range(2):
            got = yan.moe_ragged_layout(picks, experts)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), kind


# The products

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.half}
NT = {'bf16': yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged, 'fp16': yan.m_grouped_gemm_fp16_fp16_fp16_nt_ragged}
NN = {'bf16': yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged, 'fp16': yan.m_grouped_gemm_fp16_fp16_fp16_nn_ragged}
TN = {'bf16': yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged, 'fp16': yan.k_grouped_gemm_fp16_fp16_fp32_tn_ragged}


def _inside(values, around=float('nan')):
    """The values in the middle of a larger allocation, of which the rest is NaN: what is read beyond them shows."""
    flat = torch.full((values.numel() + 4096, ), around, dtype=values.dtype, device='cuda')
    flat[2048:2048 + values.numel()] = values.reshape(-1)
    return flat[2048:2048 + values.numel()].view(values.shape)


def _whole(g, *shape, dtype, top=3):
    """Whole numbers: products of a few thousand of them are summed without rounding, whatever the order."""
    return torch.randint(-top, top + 1, shape, generator=g, device='cuda').to(dtype)


def _offsets(rows, before=0):
    return torch.tensor([before] + rows, device='cuda').cumsum(0).to(torch.int32)


def _groups(offsets):
    ends = offsets.tolist()
    return [slice(ends[i], ends[i + 1]) for i in range(len(ends) - 1)]


def _call(mode, dtype, kernel, lhs, rhs, out, offsets, source=None, accumulate=False):
    named = () if kernel == 'kGroupedAny' else (kernel, )
    if mode == 'TN':
        if named:
            ragged._k_grouped(TYPES[dtype], lhs, rhs, out, offsets, accumulate, source, named)
        else:
            TN[dtype](lhs, rhs, out, offsets, accumulate, source)
    elif named:
        ragged._m_grouped(ragged.RAGGED_NT if mode == 'NT' else ragged.RAGGED_NN, TYPES[dtype], lhs, rhs, out, offsets, source, named)
    elif mode == 'NT':
        NT[dtype](lhs, rhs, out, offsets, source)
    else:
        NN[dtype](lhs, rhs, out, offsets)


KERNELS = [('kGroupedAny', 'bf16'), ('kGroupedAny', 'fp16')] + [(k, 'bf16') for k in testing.GROUPED16_KERNELS[1:]]
# rows of the groups, columns of the output, depth
M_SIZES = [([1], 8, 8), ([0, 3, 0, 0, 1], 72, 56), ([5, 130, 64, 0, 257], 136, 200), ([33, 31, 1, 128, 129], 264, 64), ([300, 17], 520, 1000), ([0, 0], 16, 24),
           ([1] * 70 + [0] * 60 + [9], 40, 136), ([600], 1024, 72), ([64, 192, 320], 128, 128)]


@pytest.mark.parametrize('kernel,dtype', KERNELS)
@pytest.mark.parametrize('mode', ['NT', 'NN', 'gathered'])
@pytest.mark.parametrize('size', range(len(M_SIZES)))
def test_products_of_whole_numbers(size, mode, kernel, dtype):
    rows, n, k = M_SIZES[size]
    g = _gen(size)
    before, behind = 7, 5                   # rows that no group has
    offsets = _offsets(rows, before)
    m = int(offsets[-1]) + behind
    gather = mode == 'gathered'
    weights = _inside(_whole(g, len(rows), *((k, n) if mode == 'NN' else (n, k)), dtype=TYPES[dtype]))
    source = None
    if gather:
        lhs = _inside(_whole(g, 50, k, dtype=TYPES[dtype]))
        source = torch.randint(-3, 55, (m, ), generator=g, device='cuda', dtype=torch.int32)          # some are none of lhs' rows
        source[:before], source[m - behind:] = 1 << 30, -5
        there = (source >= 0) & (source < 50)
        taken = torch.where(there[:, None], lhs.double()[source.clamp(0, 49).long()], 0.0)
    else:
        lhs = _whole(g, m, k, dtype=TYPES[dtype])
        lhs[:before], lhs[m - behind:] = float('nan'), float('nan')
        lhs = _inside(lhs)
        taken = lhs.double()
    want = torch.full((m, n), 7.0, dtype=TYPES[dtype], device='cuda')
    for i, at in enumerate(_groups(offsets)):
        w = weights[i].double()
        want[at] = (taken[at] @ (w if mode == 'NN' else w.t().contiguous())).to(TYPES[dtype])
    for _ in range(2):
        around = torch.full((m * n + 4096, ), 7.0, dtype=TYPES[dtype], device='cuda')
        out = around[2048:2048 + m * n].view(m, n)
        _call('NN' if mode == 'NN' else 'NT', dtype, kernel, lhs, weights, out, offsets, source)
        assert torch.equal(out, want)
        assert bool((around[:2048] == 7).all()) and bool((around[2048 + m * n:] == 7).all())


# rows of the groups, rows and columns of the gradients
K_SIZES = [([1], 8, 8), ([0, 3, 0, 0, 1], 72, 56), ([5, 130, 64, 0, 257], 136, 200), ([33, 31, 1, 128, 129], 264, 64), ([300, 17], 8, 520), ([0, 0], 16, 24),
           ([1] * 70 + [0] * 60 + [9], 40, 136), ([600, 1], 256, 72), ([64, 192, 320], 128, 128), ([1000], 384, 264)]


@pytest.mark.parametrize('kernel,dtype', [k for k in KERNELS if k[0] != 'kGrouped32'])
@pytest.mark.parametrize('gather', [False, True])
@pytest.mark.parametrize('size', range(len(K_SIZES)))
def test_weight_gradients_of_whole_numbers(size, gather, kernel, dtype):
    rows, m, n = K_SIZES[size]
    g = _gen(size + 100)
    before, behind = 3, 70
    offsets = _offsets(rows, before)
    total = int(offsets[-1]) + behind
    lhs = _whole(g, total, m, dtype=TYPES[dtype])
    lhs[:before], lhs[total - behind:] = float('nan'), float('nan')
    lhs, source = _inside(lhs), None
    if gather:
        rhs = _inside(_whole(g, 50, n, dtype=TYPES[dtype]))
        source = torch.randint(-3, 55, (total, ), generator=g, device='cuda', dtype=torch.int32)
        source[:before], source[total - behind:] = 1 << 30, -5
        there = (source >= 0) & (source < 50)
        taken = torch.where(there[:, None], rhs.double()[source.clamp(0, 49).long()], 0.0)
    else:
        rhs = _whole(g, total, n, dtype=TYPES[dtype])
        rhs[:before], rhs[total - behind:] = float('nan'), float('nan')
        rhs = _inside(rhs)
        taken = rhs.double()
    left = _whole(g, len(rows), m, n, dtype=torch.float32)
    for accumulate in (False, True):
        want = left.double() if accumulate else torch.zeros_like(left, dtype=torch.float64)
        for i, at in enumerate(_groups(offsets)):
            want[i] += lhs[at].double().t().contiguous() @ taken[at]
        for _ in range(2):
            around = torch.full((left.numel() + 2048, ), 7.0, device='cuda')
            out = around[1024:1024 + left.numel()].view(left.shape)
            out.copy_(left)
            _call('TN', dtype, kernel, lhs, rhs, out, offsets, source, accumulate)
            assert torch.equal(out.double(), want)
            assert bool((around[:1024] == 7).all()) and bool((around[1024 + left.numel():] == 7).all())


@pytest.fixture
def capped():
    """Sets the compute-unit cap for a test and takes it back."""
    before = yan.get_num_sms()
    yield yan.set_num_sms
    yan.set_num_sms(before)


@pytest.mark.parametrize('kernel', testing.GROUPED16_KERNELS[1:])
@pytest.mark.parametrize('cap', [1, 3, 8, 24])
def test_walks_of_many_tiles(cap, kernel, capped):
    """Few workgroups walk over all tiles: of one k-tile each, of several, of depths that are no multiple, of groups without rows in between."""
    capped(cap)
    g = _gen(cap)
    for rows, n, k in (([300, 0, 1, 129, 0, 513, 64], 520, 8), ([257, 100, 0, 128], 264, 72), ([140, 600, 3], 776, 264), ([20] * 30, 264, 64)):
        offsets = _offsets(rows)
        m = int(offsets[-1])
        lhs, weights, source = _whole(g, m, k, dtype=torch.bfloat16), _whole(g, len(rows), n, k, dtype=torch.bfloat16), torch.randperm(m, generator=g, device='cuda').int()
        for mode in ('NT', 'NN', 'gathered'):
            taken = lhs[source.long()] if mode == 'gathered' else lhs
            want = torch.cat([taken[at].double() @ weights[i].double().t().contiguous() for i, at in enumerate(_groups(offsets))]).bfloat16()
            out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device='cuda')
            _call('NN' if mode == 'NN' else 'NT', 'bf16', kernel, lhs, weights.transpose(1, 2).contiguous() if mode == 'NN' else weights, out, offsets,
                  source if mode == 'gathered' else None)
            assert torch.equal(out, want), (mode, rows)
    if kernel == 'kGrouped32':
        return
    for rows, m, n in (([5, 0, 64, 1, 63, 0, 0, 64, 2], 264, 520), ([65, 128, 0, 200, 1], 520, 264), ([1000, 30], 264, 136)):
        offsets = _offsets(rows)
        total = int(offsets[-1])
        lhs, rhs, source = _whole(g, total, m, dtype=torch.bfloat16), _whole(g, total, n, dtype=torch.bfloat16), torch.randperm(total, generator=g, device='cuda').int()
        for gather in (False, True):
            taken = rhs[source.long()] if gather else rhs
            products = torch.stack([lhs[at].double().t().contiguous() @ taken[at].double() for at in _groups(offsets)])
            for accumulate in (False, True):
                out = torch.full((len(rows), m, n), 7.0, device='cuda')
                _call('TN', 'bf16', kernel, lhs, rhs, out, offsets, source if gather else None, accumulate)
                assert torch.equal(out.double(), products + (7 if accumulate else 0)), (gather, accumulate, rows)


def test_many_groups():
    """More groups than a wave has lanes, most of them empty, runs of empty ones at both ends."""
    g = _gen(9)
    for groups in (64, 65, 129, 1000, 1024):
        counts = torch.where(torch.rand(groups, generator=g, device='cuda') < 0.2, torch.randint(1, 40, (groups, ), generator=g, device='cuda'), 0)
        counts[:5], counts[-70 % groups:] = 0, 0
        counts[groups // 2] = 700
        offsets = _offsets(counts.tolist())
        m = int(offsets[-1])
        lhs, weights = _whole(g, m, 72, dtype=torch.bfloat16), _whole(g, groups, 136, 72, dtype=torch.bfloat16)
        want = torch.cat([lhs[at].double() @ weights[i].double().t().contiguous() for i, at in enumerate(_groups(offsets))]).bfloat16()
        grads = torch.stack([want[at].double().t().contiguous() @ lhs[at].double() for at in _groups(offsets)])
        for kernel in testing.GROUPED16_KERNELS:
            out = torch.empty(m, 136, dtype=torch.bfloat16, device='cuda')
            _call('NT', 'bf16', kernel, lhs, weights, out, offsets)
            assert torch.equal(out, want), (groups, kernel)
            if kernel != 'kGrouped32':
                grad = torch.empty(groups, 136, 72, device='cuda')
                _call('TN', 'bf16', kernel, want, lhs, grad, offsets)
                _close(grad, grads, 40 * U * 700 * want.double().abs().max() * 3, 'gradients')


# An fp32 sum of n products of 16-bit numbers is off by at most n steps, a step of 2 u at most of the sum of the products' magnitudes (whether the matrix cores round or cut off).
REAL_SIZES = [([700, 0, 300, 24, 1], 520, 2048), ([64] * 8, 1032, 520), ([2000], 256, 7168), ([3, 1, 0, 2], 4096, 7168), ([129, 255, 257, 511], 776, 1544)]


@pytest.mark.parametrize('kernel,dtype', KERNELS)
@pytest.mark.parametrize('size', range(len(REAL_SIZES)))
def test_products_of_normal_numbers(size, kernel, dtype):
    rows, n, k = REAL_SIZES[size]
    g = _gen(size + 50)
    offsets, half = _offsets(rows), 2.0 ** (-8 if dtype == 'bf16' else -11)
    m = int(offsets[-1])
    lhs = torch.randn(m, k, generator=g, device='cuda').to(TYPES[dtype])
    weights = (torch.randn(len(rows), n, k, generator=g, device='cuda') / k ** 0.5).to(TYPES[dtype])
    grad = torch.randn(m, n, generator=g, device='cuda').to(TYPES[dtype])
    out, back, for_weights = torch.empty_like(grad), torch.empty_like(lhs), torch.empty(len(rows), n, k, device='cuda')
    _call('NT', dtype, kernel, lhs, weights, out, offsets)
    _call('NN', dtype, kernel, grad, weights, back, offsets)
    if kernel != 'kGrouped32':
        _call('TN', dtype, kernel, grad, lhs, for_weights, offsets)
    for i, at in enumerate(_groups(offsets)):
        a, w, d = lhs[at].double(), weights[i].double(), grad[at].double()
        for got, x, y, depth, step in ((out[at], a, w.t().contiguous(), k, half), (back[at], d, w, n, half), (for_weights[i], d.t().contiguous(), a, a.size(0), 0.0)):
            if not got.numel() or (step == 0.0 and kernel == 'kGrouped32'):
                continue
            want, size_of = x @ y, x.abs() @ y.abs()
            _close(got, want, 2 * depth * U * size_of * (1 + step) + step * want.abs() + (2.0 ** -25 if dtype == 'fp16' else 0), 'product')


def test_offsets_past_32_bits():
    """Outputs and operands of more than 4 GiB: the last rows are where they belong, and so are those of a group that starts far into its operand."""
    g = _gen(12)
    m, n = (1 << 20) + 131, 2056
    offsets = torch.tensor([0, 1, m - 300, m], dtype=torch.int32, device='cuda')
    lhs, weights = _whole(g, m, 8, dtype=torch.bfloat16), _whole(g, 3, n, 8, dtype=torch.bfloat16)
    for kernel in ('kGroupedTall', 'kGrouped128'):
        out = torch.zeros(m, n, dtype=torch.bfloat16, device='cuda')
        _call('NT', 'bf16', kernel, lhs, weights, out, offsets)
        for i, at in ((0, slice(0, 1)), (1, slice(1, 300)), (1, slice(m - 700, m - 300)), (2, slice(m - 300, m))):
            assert torch.equal(out[at], (lhs[at].double() @ weights[i].double().t().contiguous()).bfloat16())
        del out
    # both operands of the weights' gradient, and the rows' one, read from beyond 4 GiB on
    wide = torch.zeros(m, n, dtype=torch.bfloat16, device='cuda')
    tail = _whole(g, 700, n, dtype=torch.bfloat16)
    wide[m - 700:] = tail
    offsets = torch.tensor([m - 700, m - 640, m], dtype=torch.int32, device='cuda')
    for kernel in ('kGroupedTall', 'kGrouped128', 'kGrouped64'):
        grad = torch.empty(2, n, 8, device='cuda')
        _call('TN', 'bf16', kernel, wide, lhs, grad, offsets)
        for i, (first, last) in enumerate(((0, 60), (60, 700))):
            assert torch.equal(grad[i].double(), tail[first:last].double().t().contiguous() @ lhs[m - 700 + first:m - 700 + last].double())
    back = torch.empty(m, 8, dtype=torch.bfloat16, device='cuda')
    _call('NN', 'bf16', 'kGroupedTall', wide, weights[:2].contiguous(), back, offsets)
    assert torch.equal(back[m - 640:], (tail[60:].double() @ weights[1].double()).bfloat16())


def test_offsets_that_make_no_sense_stay_within_the_operands():
    """Whatever the offsets hold, rows and groups are within theirs: nothing outside is written, and ascending groups among them are right."""
    g = _gen(13)
    m, n, k = 500, 264, 72
    lhs, weights = _inside(_whole(g, m, k, dtype=torch.bfloat16)), _inside(_whole(g, 4, n, k, dtype=torch.bfloat16))
    grad = _inside(_whole(g, m, n, dtype=torch.bfloat16))
    for values in ([-5, 100, 1 << 30, 1 << 30, 2147483647], [400, 300, 200, 100, 0], [-2147483648, -1, 0, 0, 0], [500, 500, 500, 500, 500], [0, 500, 0, 500, 0], [0, 700, 100, 900, 501]):
        offsets = torch.tensor(values, dtype=torch.int64, device='cuda').to(torch.int32)
        for kernel in testing.GROUPED16_KERNELS:
            around = torch.full((m * n + 4096, ), 7.0, dtype=torch.bfloat16, device='cuda')
            _call('NT', 'bf16', kernel, lhs, weights, around[2048:2048 + m * n].view(m, n), offsets)
            assert bool((around[:2048] == 7).all()) and bool((around[2048 + m * n:] == 7).all())
            if kernel == 'kGrouped32':
                continue
            around = torch.full((4 * n * k + 2048, ), 7.0, device='cuda')
            _call('TN', 'bf16', kernel, grad, lhs, around[1024:1024 + 4 * n * k].view(4, n, k), offsets)
            assert bool((around[:1024] == 7).all()) and bool((around[1024 + 4 * n * k:] == 7).all())


def _layer_inputs(g, tokens, hidden, inner, experts, top_k, padded):
    x = torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16()
    logits = torch.randn(tokens, experts, generator=g, device='cuda')
    w1 = (torch.randn(experts, inner, hidden, generator=g, device='cuda') / hidden ** 0.5).bfloat16()
    w2 = (torch.randn(experts, hidden, inner, generator=g, device='cuda') / inner ** 0.5).bfloat16()
    mask = torch.rand(tokens, generator=g, device='cuda') > 0.2 if padded else None
    return x, logits, w1, w2, mask


@pytest.mark.parametrize('padded', [False, True])
def test_training_step_of_a_layer_in_16_bits(padded):
    """A norm, the router, two expert products with an activation between them and the way back, as they are used together; gradients against 64 bits."""
    g = _gen(21)
    tokens, hidden, inner, experts, top_k = testing.RAGGED_LAYER
    x, logits, w1, w2, mask = _layer_inputs(g, tokens, hidden, inner, experts, top_k, padded)
    gain, grad_out = (1 + 0.2 * torch.randn(hidden, generator=g, device='cuda')).bfloat16(), torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16()
    normed = torch.empty_like(x)
    inverse = yan.rms_norm(x, gain, normed)
    weights, indices, counts, _ = yan.moe_route(logits, top_k, mask=mask)
    rows, source, offsets = yan.moe_ragged_layout(indices, experts)
    m = source.numel()
    y1, y2 = torch.zeros(m, inner, dtype=torch.bfloat16, device='cuda'), torch.zeros(m, hidden, dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(normed, w1, y1, offsets, source)
    h = torch.relu(y1)
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(h, w2, y2, offsets)
    out = torch.empty_like(x)
    yan.moe_combine(y2, rows, weights, out)
    # and back
    grad_y2, grad_weights = yan.moe_combine_backward(grad_out, y2, rows, weights, source)
    grad_h, grad_rows, grad_normed = torch.zeros_like(h), torch.zeros(m, hidden, dtype=torch.bfloat16, device='cuda'), torch.empty_like(x)
    yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged(grad_y2, w2, grad_h, offsets)
    grad_w2, grad_w1 = torch.zeros(experts, hidden, inner, device='cuda'), torch.zeros(experts, inner, hidden, device='cuda')
    yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(grad_y2, h, grad_w2, offsets, accumulate=True)
    grad_y1 = grad_h * (y1 > 0)
    yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged(grad_y1, w1, grad_rows, offsets)
    yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(grad_y1, normed, grad_w1, offsets, accumulate=True, source=source)
    yan.moe_combine(grad_rows, rows, None, grad_normed)
    grad_gain = torch.empty(hidden, device='cuda')
    grad_x = yan.rms_norm_backward(grad_normed, x, gain, inverse, grad_gain)

    # the same in 64 bits, by autograd
    leaves = [t.double().requires_grad_() for t in (x, w1, w2, gain)]
    dx, dw1, dw2, dgain = leaves
    v = dx / torch.sqrt(dx.square().mean(1, keepdim=True) + 1e-6) * dgain
    live = torch.ones(tokens, device='cuda') if mask is None else mask.double()
    picked = torch.softmax(logits.double(), 1).gather(1, indices.clamp(min=0).long())
    share = picked / picked.sum(1, keepdim=True) * live[:, None]
    total = torch.zeros_like(v)
    for e in range(experts):
        through = torch.relu(v @ dw1[e].t()) @ dw2[e].t()
        total = total + through * (share * (indices == e)).sum(1, keepdim=True)
    (total * grad_out.double()).sum().backward()
    # every product and every sum over them is rounded to 8 bits on the way: 5 such roundings to out, 9 to the farthest gradient, each half a step of 2^-8 of its value at most. Of
    # sums of many terms with signs of their own what that comes to relative to the norm is less than twice the largest of them, in quadrature below a tenth of that
    for name, got, want, roundings in (('out', out, total, 5), ('grad_w2', grad_w2, dw2.grad, 7), ('grad_w1', grad_w1, dw1.grad, 8), ('grad_x', grad_x, dx.grad, 9), ('grad_gain', grad_gain, dgain.grad, 9)):
        off = (got.double() - want.detach()).norm() / want.detach().norm()
        assert float(off) <= roundings * 2.0 ** -8, f'{name}: {float(off):.4f}'


def test_padded_groups_of_the_contiguous_layout():
    """The 128-row groups of the FP8 layout are groups as well: padding has no source, and comes out as zeros."""
    g = _gen(22)
    tokens, experts, top_k, k, n = 150, 5, 2, 256, 136
    x = _whole(g, tokens, k, dtype=torch.bfloat16)
    indices = torch.stack([torch.randperm(experts, generator=g, device='cuda')[:top_k] for _ in range(tokens)]).int()
    m = yan.get_contiguous_layout_rows(tokens, top_k, experts)
    codes, scales = torch.zeros(m, k, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn), torch.zeros(m, k // 128, device='cuda')
    rows, _, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, experts, (codes, scales))
    weights = _whole(g, experts, n, k, dtype=torch.bfloat16)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(x, weights, out, offsets, source)
    grad = torch.empty(experts, n, k, device='cuda')
    dy = _whole(g, m, n, dtype=torch.bfloat16)
    yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(dy, x, grad, offsets, False, source)
    taken = torch.where((source >= 0)[:, None], x[source.clamp(min=0).long()], 0).double()
    for i, at in enumerate(_groups(offsets)):
        assert torch.equal(out[at], (taken[at] @ weights[i].double().t().contiguous()).bfloat16())
        assert torch.equal(grad[i].double(), dy[at].double().t().contiguous() @ taken[at])
    assert bool((out[int(offsets[-1]):] == 7).all())


def test_edges_of_ragged_products():
    """No rows, no depth, no columns, one of each; outputs that are not asked for stay."""
    empty = torch.zeros(3, dtype=torch.int32, device='cuda')
    w = torch.ones(2, 16, 8, dtype=torch.bfloat16, device='cuda')
    out = torch.zeros(0, 16, dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(torch.zeros(0, 8, dtype=torch.bfloat16, device='cuda'), w, out, empty)
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(torch.zeros(0, 8, dtype=torch.bfloat16, device='cuda'), w, out, empty, empty[:0])
    out = torch.full((4, 16), 7.0, dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(torch.ones(4, 8, dtype=torch.bfloat16, device='cuda'), w, out, empty)
    assert bool((out == 7).all())
    offsets = torch.tensor([1, 1, 3], dtype=torch.int32, device='cuda')
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(torch.zeros(4, 0, dtype=torch.bfloat16, device='cuda'), w[:, :, :0], out, offsets)
    assert bool((out[1:3] == 0).all()) and bool((out[[0, 3]] == 7).all())
    grad = torch.full((2, 16, 8), 7.0, device='cuda')
    nothing = torch.zeros(0, 16, dtype=torch.bfloat16, device='cuda')
    yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(nothing, nothing[:, :8], grad, empty, True)
    assert bool((grad == 7).all())
    yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(nothing, nothing[:, :8], grad, empty)
    assert bool((grad == 0).all())


def test_infinities_and_nan_stay_in_their_rows():
    """A row that is not finite makes itself not finite and no other one, whichever tile they share; rows without a group are not read into any sum."""
    g = _gen(23)
    for kernel in testing.GROUPED16_KERNELS:
        offsets = torch.tensor([2, 40, 170], dtype=torch.int32, device='cuda')
        lhs = _whole(g, 200, 72, dtype=torch.bfloat16)
        lhs[0], lhs[180] = float('nan'), float('inf')
        weights = _whole(g, 2, 136, 72, dtype=torch.bfloat16)
        clean = torch.empty(200, 136, dtype=torch.bfloat16, device='cuda')
        _call('NT', 'bf16', kernel, lhs, weights, clean, offsets)
        assert bool(clean[2:170].isfinite().all())
        dirty, out = lhs.clone(), torch.empty_like(clean)
        dirty[39], dirty[100] = float('inf'), float('nan')
        _call('NT', 'bf16', kernel, dirty, weights, out, offsets)
        rest = torch.ones(200, dtype=torch.bool, device='cuda')
        rest[:2], rest[170:], rest[39], rest[100] = False, False, False, False
        assert torch.equal(out[rest], clean[rest]) and bool((~out[39].isfinite()).all()) and bool(out[100].isnan().all())


def test_ragged_products_in_a_graph_and_on_other_streams():
    g = _gen(24)
    tokens, hidden, inner, experts, top_k = testing.RAGGED_LAYER
    x, logits, w1, _, _ = _layer_inputs(g, tokens, hidden, inner, experts, top_k, False)
    grad = torch.zeros(experts, inner, hidden, device='cuda')

    def step(out, back):
        _, indices, _, _ = yan.moe_route(logits, top_k)
        rows, source, offsets = yan.moe_ragged_layout(indices, experts)
        yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(x, w1, out, offsets, source)
        yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged(out, w1, back, offsets)
        yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(out, x, grad, offsets, True, source)
        return rows, source, offsets

    m = tokens * top_k
    buffers = [(torch.empty(m, inner, dtype=torch.bfloat16, device='cuda'), torch.empty(m, hidden, dtype=torch.bfloat16, device='cuda')) for _ in range(3)]
    made = step(*buffers[0])
    want = [t.clone() for t in (*made, *buffers[0], grad)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    grad.zero_()
    with torch.cuda.stream(side):
        got = step(*buffers[1])
    torch.cuda.synchronize()
    for a, b in zip((*got, *buffers[1]), want):
        assert torch.equal(a, b)
    grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*buffers[2])
    for turn in range(3):
        for t in (*got, *buffers[2]):
            t.zero_()
        grad.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, *buffers[2], grad), want):
            assert torch.equal(a, b), turn
        x.mul_(1)               # eager work between the replays


@pytest.mark.parametrize('kernel', testing.GROUPED16_KERNELS)
def test_rows_without_a_source_are_nothing_to_what_is_not_finite(kernel):
    """Weights that are not finite leave the outputs of such rows zeros, and gradients that nobody has written into their rows leave the weights' gradients as they were."""
    g = _gen(31)
    rows = [70, 0, 130, 257, 1, 64]
    offsets, total = _offsets(rows), sum(rows)
    source = torch.randint(0, 50, (total, ), generator=g, device='cuda', dtype=torch.int32)
    none = torch.rand(total, generator=g, device='cuda') < 0.3
    none[70:73] = True
    source[none] = -1
    source[none.nonzero()[::2]] = 50            # one row behind the last one
    tokens = _whole(g, 50, 136, dtype=torch.bfloat16)
    weights = _whole(g, 6, 264, 136, dtype=torch.bfloat16)
    weights[2, 5], weights[3, 17], weights[5] = float('inf'), float('nan'), float('nan')
    out = torch.full((total, 264), 9.0, dtype=torch.bfloat16, device='cuda')
    _call('NT', 'bf16', kernel, tokens, weights, out, offsets, source)
    assert bool((out[none] == 0).all())
    for i, at in enumerate(_groups(offsets)):
        live = ~none[at]
        want = (tokens[source[at][live].long()].float() @ weights[i].float().t().contiguous()).bfloat16()
        assert torch.equal(out[at][live].nan_to_num(7, 7, 7), want.nan_to_num(7, 7, 7))
    if kernel == 'kGrouped32':
        return
    grads = _whole(g, total, 72, dtype=torch.bfloat16)
    want = torch.zeros(6, 72, 136, device='cuda')
    for i, at in enumerate(_groups(offsets)):
        live = ~none[at]
        want[i] = grads[at][live].float().t().contiguous() @ tokens[source[at][live].long()].float()
    grads[none] = float('nan')
    grads[none.nonzero()[::3]] = float('inf')
    for accumulate in (False, True):
        got = torch.full((6, 72, 136), 2.0, device='cuda')
        _call('TN', 'bf16', kernel, grads, tokens, got, offsets, source, accumulate)
        assert torch.equal(got, want + 2 if accumulate else want)


def test_more_tiles_than_a_launch_has_workgroups():
    """The widest weights there may be, of 1024 groups with a row or two: more tiles than a launch may have threads for."""
    g = _gen(32)
    n, groups = (1 << 21) - 8, 1024
    rows = [1] * groups
    rows[7], rows[1000] = 40, 38
    offsets, total = _offsets(rows), sum(rows)
    weights = torch.zeros(groups, n, 8, dtype=torch.bfloat16, device='cuda')
    lhs = _whole(g, total, 8, dtype=torch.bfloat16)
    out = torch.full((total, n), 9.0, dtype=torch.bfloat16, device='cuda')
    known = (0, 7, 511, 1000, 1023)
    for i in known:
        weights[i] = _whole(g, n, 8, dtype=torch.bfloat16)
    yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(lhs, weights, out, offsets)
    for i, at in enumerate(_groups(offsets)):
        if i in known:
            assert torch.equal(out[at], (lhs[at].float() @ weights[i].float().t().contiguous()).bfloat16())
        else:
            assert not bool(out[at].any())
