"""The norm with the residual's addition and its gradient on the GPU, against the formulas in 64 bits.

Tolerances, u = 2^-24 being half a step of fp32, 2^-8 that of bf16, 2^-4 that of e4m3 relative to a normal number. A sum of n terms of one sign that is
taken in d additions one after the other is off by d u of itself, each of its terms by what it was off by.
"""
import pytest
import torch

import harness as testing
import yan_amd as yan
from yan_amd.jit_kernels import norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = testing.NORM_TYPES


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _close(got, want, bound, what=''):
    off = (got.double() - want.double()).abs()
    assert bool((off <= bound).all()), f'{what}: {int((~(off <= bound)).sum())} of {off.numel()} further off than they may be, by up to {float((off - bound).max()):.3g}'


def _rows(g, rows, k, dtype):
    x = torch.randn(rows, k, generator=g, device='cuda') * torch.exp(torch.randn(rows, 1, generator=g, device='cuda'))
    return (x * torch.where(torch.rand(k, generator=g, device='cuda') < 0.02, 20.0, 1.0)).to(dtype)


# The squares: 8 runs of 8 fused multiplications and additions a lane at most, 6 steps over a wave, 16 waves; of their mean's root half of that and a quotient,
# an addition, a root and a quotient.
INVERSE_OFF = ((64 + 6 + 16 + 2) / 2 + 2) * U
Y_OFF = INVERSE_OFF + 2 * U


def _check_norm(got, x, weight, eps, h, k):
    """got: dict of what a call gave; h: what was normed, exact."""
    v = h.double()
    r = 1 / torch.sqrt(v.square().mean(1, keepdim=True) + eps)
    y = v * r * weight.double()
    _close(got['inverse_rms'], r[:, 0], INVERSE_OFF * r[:, 0], 'reciprocal')
    if got.get('normed') is not None:
        _close(got['normed'], y, (2.0 ** -8 + 2 * Y_OFF) * y.abs(), '16 bits')
    if got.get('codes') is not None:
        blocks = y.view(y.size(0), -1, 128)
        amax = blocks.abs().amax(-1).clamp(min=float(torch.tensor(1e-4)))
        _close(got['scales'], amax / 448, (Y_OFF + U) * amax / 448, 'scales')
        decoded = got['codes'].double().view_as(blocks) * got['scales'].double()[..., None]
        # half a step of a normal code or, below 2^-6, of the smallest ones; y, the factor, the product and the scale are off by less than 2 Y_OFF together
        _close(decoded, blocks, torch.maximum(2.0 ** -4 * blocks.abs(), 2.0 ** -10 * (amax / 448)[..., None]) * (1 + 32 * Y_OFF) + 4 * Y_OFF * blocks.abs(), 'codes')


@pytest.mark.parametrize('rows,k', testing.NORM_SHAPES)
def test_norm(rows, k):
    g = _gen(rows + k)
    for i, (xt, ht, wt, codes, normed) in enumerate(testing.NORM_CALLS):
        if codes and k % 128:
            continue
        x, weight, eps = _rows(g, rows, k, TYPES[xt]), (1 + 0.3 * torch.randn(k, generator=g, device='cuda')).to(TYPES[wt]), (1e-6, 1e-2)[i % 2]
        before = None if ht is None else _rows(g, rows, k, TYPES[ht])
        h = x if before is None else (x.float() + before.float()).to(before.dtype)
        for turn in range(2):               # the second call is made natively
            residual = None if before is None else before.clone()
            out = torch.full((rows, k), 7.0, dtype=torch.bfloat16, device='cuda') if normed else None
            got = {'normed': out}
            if codes:
                got['codes'], got['scales'], got['inverse_rms'] = yan.rms_norm_to_fp8(x, weight, eps, residual, i % 4 == 0, out)
                assert got['codes'].dtype == torch.float8_e4m3fn and got['scales'].shape == (rows, k // 128)
                assert got['scales'].stride() == ((1, rows) if i % 4 == 0 else (k // 128, 1)) or rows == 1 or k == 128
            else:
                got['inverse_rms'] = yan.rms_norm(x, weight, out, eps, residual)
            if residual is not None:
                assert torch.equal(residual, h)
            _check_norm(got, x, weight, eps, h, k)


def test_norm_to_fp8_is_the_quantiser_of_the_normed_rows():
    """Codes and scales are those of per_token_cast_to_fp8 applied to the normed rows, where these are numbers that 16 bits hold."""
    rows, k = 40, 512
    g = _gen(1)
    # rows whose root mean square is 1: +-1 throughout, and weights of few bits
    x = (torch.randint(0, 2, (rows, k), generator=g, device='cuda') * 2 - 1).to(torch.bfloat16)
    weight = (torch.randint(1, 255, (k, ), generator=g, device='cuda') / 64).to(torch.bfloat16)
    out = torch.empty_like(x)
    codes, scales, inverse = yan.rms_norm_to_fp8(x, weight, 0.0, normed=out)
    assert bool((inverse == 1).all()) and torch.equal(out, x * weight)
    want, want_scales = yan.per_token_cast_to_fp8(out)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)


@pytest.mark.parametrize('rows,k', testing.NORM_SHAPES)
def test_norm_gradient(rows, k):
    g = _gen(rows * 3 + k)
    lanes, runs = norm.norm_backward_lanes(k)
    parts = norm.norm_backward_workgroups(rows, k) * max(1, 256 // lanes)
    for gt, ht, wt, residual, with_weight in testing.NORM_BACKWARD_CALLS:
        grad, h = _rows(g, rows, k, TYPES[gt]), _rows(g, rows, k, TYPES[ht])
        weight = (1 + 0.3 * torch.randn(k, generator=g, device='cuda')).to(TYPES[wt])
        r = (1 / torch.sqrt(h.double().square().mean(1) + 1e-5)).float()
        kept = _rows(g, rows, k, TYPES[gt]) if residual else None
        u, p = h.double() * r.double()[:, None], grad.double() * weight.double()
        want = r.double()[:, None] * (p - u * (p * u).mean(1, keepdim=True))
        # a term of the sum over k: two products and one that is fused, 4 runs of 8 a lane, 6 steps over a wave, 8 waves, a quotient; around it five more roundings
        size = r.double()[:, None] * (p.abs() + u.abs() * (p * u).abs().mean(1, keepdim=True))
        bound = (3 + 32 + 6 + 8 + 1 + 5) * U * size
        if residual:
            want = want + kept.double()
            bound = bound + U * (want.abs() + bound)
        if gt == 'bf16':
            bound = bound + 2.0 ** -8 * (want.abs() + bound)
        terms = grad.double() * u
        for accumulate in ((False, True) if with_weight else (False, )):
            before = torch.randn(k, generator=g, device='cuda')
            grad_weight = before.clone() if with_weight else None
            got = yan.rms_norm_backward(grad, h, weight, r, grad_weight, kept, accumulate)
            assert got.dtype == grad.dtype
            _close(got, want, bound, 'gradient')
            if with_weight:
                want_weight = terms.sum(0) + (before.double() if accumulate else 0)
                # a part's rows one after the other, every 32nd part, the 32 sums of those; u and its product
                depth = -(-rows // parts) + -(-parts // 32) + 32 + 3
                _close(grad_weight, want_weight, depth * U * (terms.abs().sum(0) + (before.double().abs() if accumulate else 0)), 'weight')
                again = before.clone()
                assert torch.equal(yan.rms_norm_backward(grad, h, weight, r, again, kept, accumulate), got) and torch.equal(again, grad_weight)


def test_norm_gradient_against_differences():
    g = _gen(5)
    rows, k = 3, 24
    x, weight = torch.randn(rows, k, generator=g, device='cuda'), 1 + 0.3 * torch.randn(k, generator=g, device='cuda')
    down, eps = torch.randn(rows, k, generator=g, device='cuda'), 1e-3
    out = torch.empty(rows, k, dtype=torch.bfloat16, device='cuda')
    inverse = yan.rms_norm(x, weight, out, eps)
    grad_weight = torch.empty(k, device='cuda')
    got = yan.rms_norm_backward(down, x, weight, inverse, grad_weight)

    def value(h, w):
        return float((h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w * down.double()).sum())

    step = 1e-5
    for r in range(rows):
        for c in range(k):
            up, low = x.double().clone(), x.double().clone()
            up[r, c] += step
            low[r, c] -= step
            # third order in the step: below 1e-8 here; the gradient is off by a hundred u of terms of size 10
            assert abs(float(got[r, c]) - (value(up, weight.double()) - value(low, weight.double())) / (2 * step)) < 1e-8 + 1000 * U
    for c in range(k):
        up, low = weight.double().clone(), weight.double().clone()
        up[c] += step
        low[c] -= step
        assert abs(float(grad_weight[c]) - (value(x.double(), up) - value(x.double(), low)) / (2 * step)) < 1e-8 + 1000 * U


def test_norm_rows_of_zeros_infinities_and_nan():
    """A row's own and nobody else's: zeros give zeros, an infinity or a NaN makes its row what the formula makes it."""
    k = 256
    x = torch.ones(70, k, dtype=torch.bfloat16, device='cuda')
    x[3] = 0
    x[10, 5], x[20, 250] = float('inf'), float('nan')
    weight = torch.ones(k, dtype=torch.bfloat16, device='cuda')
    out = torch.empty_like(x)
    codes, scales, inverse = yan.rms_norm_to_fp8(x, weight, 1e-6, normed=out)
    assert bool((out[3] == 0).all()) and bool((codes[3].float() == 0).all()) and bool((scales[3] == torch.tensor(1e-4, device='cuda') / 448).all())
    assert float(inverse[10]) == 0 and bool(out[10, 5].isnan()) and bool((out[10, :5] == 0).all())
    assert bool(inverse[20].isnan()) and bool(out[20].isnan().all()) and bool(codes[20].float().isnan().all())
    rest = torch.ones(70, dtype=torch.bool, device='cuda')
    rest[[3, 10, 20]] = False
    assert bool((out[rest] == 1).all()) and bool((codes[rest].float() == 448).all())


def test_norm_in_place_and_empty():
    x = _rows(_gen(2), 65, 384, torch.bfloat16)
    weight = torch.ones(384, device='cuda')
    want = torch.empty_like(x)
    inverse = yan.rms_norm(x, weight, want)
    same = x.clone()
    assert torch.equal(yan.rms_norm(same, weight, same), inverse) and torch.equal(same, want)
    nothing = x[:0]
    codes, scales, inverse = yan.rms_norm_to_fp8(nothing, weight)
    assert codes.shape == (0, 384) and scales.shape == (0, 3) and inverse.shape == (0, )
    grad_weight = torch.ones(384, device='cuda')
    assert yan.rms_norm_backward(nothing, nothing, weight, inverse, grad_weight, accumulate=True).shape == (0, 384) and bool((grad_weight == 1).all())
    yan.rms_norm_backward(nothing, nothing, weight, inverse, grad_weight)
    assert bool((grad_weight == 0).all())


def test_norm_in_a_graph_and_on_another_stream():
    g = _gen(4)
    x, weight = _rows(g, 300, 1024, torch.bfloat16), torch.ones(1024, device='cuda')
    grad, residual = _rows(g, 300, 1024, torch.bfloat16), _rows(g, 300, 1024, torch.bfloat16)
    grad_weight = torch.zeros(1024, device='cuda')
    start = residual.clone()

    def step():
        codes, scales, inverse = yan.rms_norm_to_fp8(x, weight, 1e-6, residual)
        return codes, scales, yan.rms_norm_backward(grad, residual, weight, inverse, grad_weight, accumulate=True)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    residual.copy_(start)
    grad_weight.zero_()
    want = [t.clone() for t in step()] + [residual.clone(), grad_weight.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        residual.copy_(start)
        grad_weight.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, residual, grad_weight), want):
            assert torch.equal(a.view(torch.uint8) if a.dtype == torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
        x.mul_(1)               # eager work between the replays


@pytest.mark.parametrize('rows,k', [(1, 128), (5, 1024), (37, 7168), (3, 16384)])
def test_norm_of_one_tensor_in_two_places(rows, k):
    """The rows are their own residual, and a gradient its own residual's: as of two tensors that hold the same."""
    g = torch.Generator(device='cuda').manual_seed(rows * 31 + k)
    x, w = torch.randn(rows, k, generator=g, device='cuda').bfloat16(), torch.rand(k, generator=g, device='cuda')
    twin, residual = x.clone(), x.clone()
    want = yan.rms_norm_to_fp8(x.clone(), w, 1e-6, residual)
    got = yan.rms_norm_to_fp8(twin, w, 1e-6, twin)
    assert torch.equal(twin, residual) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    out, again = torch.empty_like(x), x.clone()
    yan.rms_norm(again, w, out, 1e-6, again)
    want_out, residual = torch.empty_like(x), x.clone()
    yan.rms_norm(x, w, want_out, 1e-6, residual)
    assert torch.equal(again, residual) and torch.equal(out, want_out)
    grad, dw, want_dw = torch.randn(rows, k, generator=g, device='cuda').bfloat16(), torch.zeros(k, device='cuda'), torch.zeros(k, device='cuda')
    want = yan.rms_norm_backward(grad, residual, w, got[2], want_dw, grad.clone())
    assert torch.equal(yan.rms_norm_backward(grad, residual, w, got[2], dw, grad), want) and torch.equal(dw, want_dw)
