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
