"""The norm, the ragged layout and the ragged products at the ends of their ranges, on the GPU."""
import pytest
import torch

import harness as testing
import yan_amd as yan
from yan_amd.jit_kernels import ragged

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _whole(g, *shape, dtype=BF16, top=3):
    """Whole numbers: products of a few thousand of them are summed without rounding, whatever the order."""
    return torch.randint(-top, top + 1, shape, generator=g, device='cuda').to(dtype)


def _nearly_2_gib(g, tokens, columns):
    """Tokens of zeros but for the first two and the last eight, and 2048 picks of those."""
    x = torch.zeros(tokens, columns, dtype=BF16, device='cuda')
    x[:2], x[-8:] = _whole(g, 2, columns), _whole(g, 8, columns)
    picks = torch.randint(-8, 2, (2048, ), generator=g, device='cuda')
    return x, torch.where(picks < 0, picks + tokens, picks).int()


@pytest.mark.parametrize('kernel', ['kGroupedAny', 'kGroupedTall', 'kGrouped128'])
@pytest.mark.parametrize('tokens,k', [(508400, 2112), (2097151, 512), (1048575, 1024), ((1 << 27) - 1, 8)])
def test_rows_gathered_from_the_end_of_2_gib(tokens, k, kernel):
    g = _gen(k)
    x, source = _nearly_2_gib(g, tokens, k)
    n, offsets = 4608, torch.tensor([0, 1000, 2048], dtype=torch.int32, device='cuda')        # two long groups: large tiles by the rule as well
    weights = _whole(g, 2, n, k)
    out = torch.full((2048, n), 7.0, dtype=BF16, device='cuda')
    if kernel == 'kGroupedAny':
        yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged(x, weights, out, offsets, source)
    else:
        ragged._m_grouped(ragged.RAGGED_NT, BF16, x, weights, out, offsets, source, (kernel, ))
    taken = x[source.long()].double()
    for group, at in enumerate((slice(0, 1000), slice(1000, 2048))):
        assert torch.equal(out[at], (taken[at] @ weights[group].double().t().contiguous()).bfloat16())


@pytest.mark.parametrize('kernel', ['kGroupedAny', 'kGroupedTall', 'kGrouped128'])
@pytest.mark.parametrize('tokens,n', [(2064888, 520), (2097151, 512), ((1 << 27) - 1, 8)])
def test_weight_gradients_gathered_from_the_end_of_2_gib(tokens, n, kernel):
    g = _gen(n + 1)
    x, source = _nearly_2_gib(g, tokens, n)
    m, offsets = 1 << 15, torch.tensor([0, 1000, 2048], dtype=torch.int32, device='cuda')     # (m: as many tiles as the rule wants for large ones)
    grads = _whole(g, 2048, m)
    out = torch.full((2, m, n), 7.0, device='cuda')
    if kernel == 'kGroupedAny':
        yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged(grads, x, out, offsets, False, source)
    else:
        ragged._k_grouped(BF16, grads, x, out, offsets, False, source, (kernel, ))
    taken = x[source.long()].double()
    for group, at in enumerate((slice(0, 1000), slice(1000, 2048))):
        assert torch.equal(out[group].double(), grads[at].double().t().contiguous() @ taken[at])


@pytest.mark.parametrize('groups', [1, 2, 3, 9])
def test_shallow_products_on_large_tiles(groups):
    """Depths of a few rows, where a k-tile of one group's weights reaches over several groups behind it, and the last of them end inside; what lies behind the operands is NaN."""
    g = _gen(groups)
    rows = [(140, 0, 1, 300, 64)[i % 5] for i in range(groups)]
    offsets = torch.tensor([0] + rows, device='cuda').cumsum(0).int()
    m, n, ends = sum(rows), 264, [0, *offsets.tolist()[1:]]
    for k in (8, 16, 24, 32, 40, 48, 56, 64, 72, 120):
        flat = torch.full((groups * k * n + 64 * n, ), float('nan'), dtype=BF16, device='cuda')
        weights = flat[:groups * k * n].view(groups, k, n)
        weights.copy_(_whole(g, groups, k, n))
        lhs = _whole(g, m, k)
        want = torch.cat([lhs[ends[i]:ends[i + 1]].double() @ weights[i].double() for i in range(groups)]).bfloat16()
        for kernel in ('kGroupedTall', 'kGrouped128'):
            out = torch.full((m, n), 7.0, dtype=BF16, device='cuda')
            ragged._m_grouped(ragged.RAGGED_NN, BF16, lhs, weights, out, offsets, None, (kernel, ))
            assert torch.equal(out, want), (k, kernel)


def test_norm_gradient_of_as_many_rows_as_there_are_numbers_for():
    """2^31 - 1 rows, one tensor for the gradient and the rows: dh = r (g - h r mean(g h r)) is 3/8 for ones and 0 for twos where r is 1/2, and the weight's sums follow."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip('wants 78 GB of memory')
    rows, twos = (1 << 31) - 1, 40
    h = torch.ones(rows, 8, dtype=BF16, device='cuda')
    h[-twos:] = 2
    inverse, grad_weight = torch.full((rows, ), 0.5, device='cuda'), torch.empty(8, device='cuda')
    got = yan.rms_norm_backward(h, h, torch.ones(8, device='cuda'), inverse, grad_weight)
    assert bool((got[-twos:] == 0).all())
    for first in range(0, rows - twos, 1 << 28):
        assert bool((got[first:min(first + (1 << 28), rows - twos)] == 0.375).all())
    # a part's sums of halves are exact; 8192 parts, 32 sums of every 32nd and those added up
    total = 0.5 * (rows - twos) + 2 * twos
    assert bool(((grad_weight.double() - total).abs() <= (256 + 32) * 2.0 ** -24 * total).all())
    del h, inverse, got
    torch.cuda.empty_cache()


def test_norm_refuses_views_of_its_residual_also_after_calls_that_it_took():
    x, residual, out = (torch.ones(4, 256, dtype=BF16, device='cuda') for _ in range(3))
    w = torch.ones(256, device='cuda')
    for _ in range(2):
        yan.rms_norm(x, w, out, 1e-6, residual)
        yan.rms_norm_to_fp8(x, w, 1e-6, residual, False, out)
    before = residual.clone()
    for _ in range(2):
        with pytest.raises(AssertionError, match='a place of their own'):
            yan.rms_norm(x, w, residual.view(4, 256), 1e-6, residual)
        with pytest.raises(AssertionError, match='a place of their own'):
            yan.rms_norm_to_fp8(x, w, 1e-6, residual, False, residual[:])
    assert torch.equal(residual, before)


def test_entries_of_one_type_refuse_the_others_tensors_after_calls_of_the_other():
    g = _gen(3)
    offsets, source = torch.tensor([0, 5, 12], dtype=torch.int32, device='cuda'), torch.arange(12, dtype=torch.int32, device='cuda')
    pairs = {BF16: (yan.m_grouped_gemm_bf16_bf16_bf16_nt_ragged, yan.m_grouped_gemm_bf16_bf16_bf16_nn_ragged, yan.k_grouped_gemm_bf16_bf16_fp32_tn_ragged),
             torch.half: (yan.m_grouped_gemm_fp16_fp16_fp16_nt_ragged, yan.m_grouped_gemm_fp16_fp16_fp16_nn_ragged, yan.k_grouped_gemm_fp16_fp16_fp32_tn_ragged)}
    for dtype, other in ((BF16, torch.half), (torch.half, BF16)):
        lhs, weights, grad = _whole(g, 12, 64, dtype=dtype), _whole(g, 2, 64, 64, dtype=dtype), torch.zeros(2, 64, 64, device='cuda')
        out = torch.zeros(12, 64, dtype=dtype, device='cuda')
        calls = [lambda f: f[0](lhs, weights, out, offsets), lambda f: f[0](lhs, weights, out, offsets, source), lambda f: f[1](lhs, weights, out, offsets),
                 lambda f: f[2](lhs, out, grad, offsets), lambda f: f[2](lhs, out, grad, offsets, True, source)]
        for call in calls:
            call(pairs[dtype])
            call(pairs[dtype])
            before = out.clone(), grad.clone()
            with pytest.raises(AssertionError):
                call(pairs[other])
            assert torch.equal(out, before[0]) and torch.equal(grad, before[1])


@pytest.mark.parametrize('rows,k,codes', testing.NORM_LONG)
def test_norm_of_more_rows_than_a_launch_has_threads(rows, k, codes):
    """Rows of ones and, in places, of twos whose root mean square is 1 and 2: the normed rows are the weight, and the reciprocals say which is which."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip('wants up to 110 GB of memory')
    x = torch.ones(rows, k, dtype=BF16, device='cuda')
    places = torch.tensor([0, 17, rows // 2, (1 << 24) - 9, (1 << 24) - 1, (1 << 26) - 1, (1 << 28) - 129, (1 << 28) - 1, 1 << 28, 1 << 26, 1 << 24, rows - 2, rows - 1], device='cuda')
    places = places[places < rows].unique()
    x[places] = 2
    weight = (1 + torch.arange(k, device='cuda') % 3).float()
    if codes:
        # (token-contiguous scales: the pieces of a column follow each other. Quotients rounded once: torch divides a tensor by a number as a product with its reciprocal, a rounding more)
        got, scales, inverse = yan.rms_norm_to_fp8(x, weight, 0.0, col_major_scales=True)
        assert bool((scales == torch.tensor(3 / 448, device='cuda')).all())
        want = (weight * torch.tensor(448 / 3, device='cuda')).to(torch.float8_e4m3fn).view(torch.uint8)
        same = lambda part: bool((got[part].view(torch.uint8) == want).all())
    else:
        got = torch.zeros(rows, k, dtype=BF16, device='cuda')
        inverse = yan.rms_norm(x, weight, got, 0.0)
        same = lambda part: bool((got[part] == weight.bfloat16()).all())
    step = (1 << 31) // k
    assert all(same(slice(first, first + step)) for first in range(0, rows, step))
    assert bool((inverse[places] == 0.5).all()) and int((inverse == 0.5).sum()) == places.numel() and int((inverse == 1).sum()) == rows - places.numel()
    del x, got, inverse
    torch.cuda.empty_cache()


def test_layout_with_a_table_of_more_than_2_gib():
    """2^29 pairs and a few of 1024 experts: pair p asks for expert p mod 1000, and every 1000th for none."""
    torch.cuda.empty_cache()
    tokens, top_k, experts, none = (1 << 25) + 3, 16, 1024, 7
    pairs, step = tokens * top_k, 1 << 26
    indices = torch.empty(pairs, dtype=torch.int32, device='cuda')
    for first in range(0, pairs, step):
        e = torch.arange(first, min(first + step, pairs), dtype=torch.int32, device='cuda') % 1000
        indices[first:first + step] = torch.where(e == none, -1, e)
    rows, source, offsets = yan.moe_ragged_layout(indices.view(tokens, top_k), experts)
    counts = torch.tensor([(pairs - e + 999) // 1000 if e < 1000 and e != none else 0 for e in range(experts)], device='cuda')
    starts = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    assert torch.equal(offsets.long(), starts)
    total, starts, flat = int(starts[-1]), starts.int(), rows.view(-1)
    for first in range(0, pairs, step):
        p = torch.arange(first, min(first + step, pairs), dtype=torch.int32, device='cuda')
        e, part = p % 1000, flat[first:first + step]
        assert torch.equal(part, torch.where(e == none, -1, starts[e.long()] + p // 1000))
        real = e != none
        assert torch.equal(source[part[real].long()], p[real] // top_k)
    assert bool((source[total:] == -1).all())
    del indices, rows, source, flat
    torch.cuda.empty_cache()
