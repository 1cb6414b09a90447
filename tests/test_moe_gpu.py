"""The mixture-of-experts entries and the weight-gradient products on the GPU, each against its definition in 64 bits, and all of them in a row.

Tolerances, u = 2^-24 being half a step of fp32, 2^-8 that of bf16: what an fp32 sum of n terms is off by is at most n u times the sum of their
magnitudes, a product or quotient u of its value, a score 4 u (two units of its exponential, one of its division, one of what it divides by) and, by the
rounding of its argument, |l - top| u more.
"""
import pytest
import torch

import harness as testing
import yan_amd as yan
from yan_amd.jit_kernels import wgrad

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _close(got, want, bound, what=''):
    off = (got.double() - want.double()).abs()
    worst = (off - bound).max() if off.numel() else torch.tensor(0.0)
    assert bool((off <= bound).all()), f'{what}: {int((off > bound).sum())} of {off.numel()} further off than they may be, by up to {float(worst):.3g}'


# Router

def _route_reference(logits, top_k, scoring, renormalize, mask):
    """weights, indices, counts, loss, and per token what its scores may be off by, relatively; all in 64 bits."""
    l = logits.double()
    live = torch.ones(l.size(0), dtype=torch.bool, device=l.device) if mask is None else mask
    l = torch.where(l == float('inf'), torch.full_like(l, torch.finfo(torch.float32).max), l)
    top = l.max(1, keepdim=True).values
    top = torch.where(top == -float('inf'), torch.zeros_like(top), top)
    s = torch.exp(l - top) if scoring == 'softmax' else 1 / (1 + torch.exp(-l))
    total = s.sum(1, keepdim=True)
    p = torch.where(total == 0, s, s / total)
    if scoring == 'softmax':
        s = p
    order = torch.argsort(l, dim=1, descending=True, stable=True)[:, :top_k]
    w = s.gather(1, order)
    if renormalize:
        chosen = w.sum(1, keepdim=True)
        w = torch.where(chosen == 0, w, w / chosen)
    w = w * live[:, None]
    indices = torch.where(live[:, None], order, -1).int()
    counts = torch.zeros(l.size(1), dtype=torch.long, device=l.device).scatter_add_(0, order[live].reshape(-1), torch.ones_like(order[live].reshape(-1)))
    n = int(live.sum())
    e = l.size(1)
    loss = (e / (top_k * n * n) * (counts * (p * live[:, None]).sum(0)).sum()) if n else torch.zeros((), dtype=torch.float64, device=l.device)
    return w, indices, counts.int(), loss, s, p, total, order, live


ROUTES = [(1, 4, 1), (1, 256, 8), (3, 7, 7), (64, 256, 8), (17, 60, 6), (33, 64, 16), (100, 65, 3), (129, 128, 2), (1000, 130, 8), (5, 257, 4), (257, 512, 8),
          (40, 1000, 16), (9, 1024, 5), (4099, 16, 4)]


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('tokens,experts,top_k', ROUTES)
def test_route_and_its_gradient(tokens, experts, top_k, dtype, scoring):
    g = _gen(tokens + experts)
    for renormalize, padded in ((True, False), (False, True)):
        logits = (2 * torch.randn(tokens, experts, generator=g, device='cuda')).to(dtype)
        mask = (torch.rand(tokens, generator=g, device='cuda') < 0.7) if padded else None
        w, i, c, loss, s, p, total, order, live = _route_reference(logits, top_k, scoring, renormalize, mask)
        got_w, got_i, got_c, got_loss = yan.moe_route(logits, top_k, scoring, renormalize, mask)
        assert torch.equal(got_i, i) and torch.equal(got_c, c)
        # a score 4 u and |l - top| <= 24 of it, a sum over the row (lanes and steps: 16 + 6 additions), one over the picks, two quotients
        score_off = (4 + 24 + 22 + 6 + 2) * U
        _close(got_w, w, score_off * w, 'weights')
        # shares the same, summed over the tokens in steps: a lane's own, 16 waves, 4 groups, 64 and 16 rows
        _close(got_loss, loss, (score_off + (tokens / 256 + 100) * U) * loss.abs(), 'loss')
        again = yan.moe_route(logits, top_k, scoring, renormalize, mask)
        assert all(torch.equal(a, b) for a, b in zip(again, (got_w, got_i, got_c, got_loss)))
        # backward
        dw = torch.randn(tokens, top_k, generator=g, device='cuda')
        dl = torch.randn(1, generator=g, device='cuda')
        for grad_w, grad_l in ((dw, dl), (dw, None), (None, dl), (None, None)):
            got = yan.moe_route_backward(logits, got_i, got_c, grad_w, grad_l, scoring, renormalize)
            assert got.dtype == dtype and got.shape == logits.shape
            n = max(1, int(live.sum()))
            pull = (0.0 if grad_l is None else float(grad_l)) * experts * c.double() / (top_k * n * n)
            h_of = torch.zeros(tokens, top_k, dtype=torch.float64, device='cuda') if grad_w is None else grad_w.double()
            size_of = h_of.abs()
            if renormalize:
                chosen = s.gather(1, order).sum(1, keepdim=True)
                r = s.gather(1, order) / chosen
                h_of, size_of = (h_of - (r * h_of).sum(1, keepdim=True)) / chosen, (size_of + (r * size_of).sum(1, keepdim=True)) / chosen
            h = torch.zeros_like(s).scatter_(1, order, h_of)
            size = torch.zeros_like(s).scatter_(1, order, size_of)
            if scoring == 'softmax':
                d = h + pull
                want = s * (d - (s * d).sum(1, keepdim=True))
                size = s * (size + pull.abs() + (s * (size + pull.abs())).sum(1, keepdim=True))
            else:
                want = s * (1 - s) * (h + (pull - (p * pull).sum(1, keepdim=True)) / total)
                size = s * (size + (pull.abs() + (p * pull.abs()).sum(1, keepdim=True)) / total)        # 1 - s is off by u of 1, not of itself
            want, size = want * live[:, None], size * live[:, None]
            # every factor of a term is off by a score's bound at most, of which there are five in the longest, and 30 additions
            bound = (5 * score_off + 30 * U) * size
            if dtype == torch.bfloat16:
                bound = bound + 2.0 ** -8 * (want.abs() + bound)
            _close(got, want, bound, f'gradient with {grad_w is not None} {grad_l is not None}')


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
def test_route_gradient_against_differences(scoring):
    """The gradient against central differences of the definition in 64 bits, the picks and counts held."""
    g = _gen(3)
    tokens, experts, top_k = 6, 12, 3
    logits = torch.randn(tokens, experts, generator=g, device='cuda')
    dw, dl = torch.randn(tokens, top_k, generator=g, device='cuda'), torch.tensor(1.5, device='cuda')
    w, i, c, loss = yan.moe_route(logits, top_k, scoring, True)
    got = yan.moe_route_backward(logits, i, c, dw, dl, scoring, True)

    def value(l):
        s = torch.softmax(l, 1) if scoring == 'softmax' else torch.sigmoid(l)
        picked = s.gather(1, i.long())
        weights = picked / picked.sum(1, keepdim=True)
        share = s / s.sum(1, keepdim=True)
        return (weights * dw.double()).sum() + dl.double() * experts / (top_k * tokens * tokens) * (c.double() * share.sum(0)).sum()

    step = 1e-5
    for t in range(tokens):
        for e in range(experts):
            up, down = logits.double().clone(), logits.double().clone()
            up[t, e] += step
            down[t, e] -= step
            difference = float(value(up) - value(down)) / (2 * step)
            # of the third order in the step, below 1e-9 here; the gradient itself about a hundred u of terms of size 3
            assert abs(float(got[t, e]) - difference) < 1e-8 + 100 * U * 3


def test_route_ties_and_rows_without_a_choice():
    inf = float('inf')
    logits = torch.zeros(8, 40, device='cuda')
    logits[1] = -inf                                    # nothing to choose: the first experts, with weight 0
    logits[2, 5:] = -inf                                # fewer than top_k
    logits[3, 7] = inf
    logits[4, ::2] = -0.0                               # the same value as 0
    logits[5] = torch.finfo(torch.float32).min          # a mask's lowest value
    logits[5, 39] = 0.0
    logits[6, 3:6] = inf
    logits[7, 30:] = 1.0
    for scoring in ('softmax', 'sigmoid'):
        w, i, c, loss = yan.moe_route(logits, 8, scoring, True)
        first = list(range(8))
        assert i[0].tolist() == first and i[1].tolist() == first and i[2].tolist() == first and i[4].tolist() == first
        assert i[3].tolist() == [7] + first[:7] and i[5].tolist() == [39] + first[:7] and i[6].tolist() == [3, 4, 5, 0, 1, 2, 6, 7]
        assert i[7].tolist() == list(range(30, 38))
        assert torch.isfinite(w).all() and torch.isfinite(loss)
        assert bool((w[1] == 0).all()) and bool((w[2, 5:] == 0).all())
        assert abs(float(w[0].sum()) - 1) < 16 * U and abs(float(w[0, 0]) - 0.125) < 8 * U
        if scoring == 'softmax':
            assert w[3].tolist() == [1.0] + [0.0] * 7 and w[5].tolist() == [1.0] + [0.0] * 7
            assert abs(float(w[6, 0]) - 1 / 3) < 8 * U and bool((w[6, 3:] == 0).all())
        assert int(c.sum()) == 64
        dx = yan.moe_route_backward(logits, i, c, torch.randn(8, 8, device='cuda'), torch.ones((), device='cuda'), scoring, True)
        assert torch.isfinite(dx).all() and bool((dx[1] == 0).all())
    # a NaN is told: the weights of its token and the loss
    logits[0, 11] = float('nan')
    w, i, c, loss = yan.moe_route(logits, 8)
    assert bool(torch.isnan(w[0]).all()) and bool(torch.isfinite(w[1:]).all()) and bool(torch.isnan(loss))
    assert sorted(i[0].tolist()) == list(range(8)) and int(c.sum()) == 64
    # ... but not one of a token that is masked
    mask = torch.ones(8, dtype=torch.bool, device='cuda')
    mask[0] = False
    w, i, c, loss = yan.moe_route(logits, 8, mask=mask)
    assert torch.isfinite(w).all() and torch.isfinite(loss) and i[0].tolist() == [-1] * 8 and int(c.sum()) == 56


@pytest.mark.parametrize('tokens', [0, 5, 300])
def test_route_of_nothing(tokens):
    """No tokens, and tokens all of which are padding."""
    mask = torch.zeros(tokens, dtype=torch.bool, device='cuda')
    logits = torch.randn(tokens, 32, device='cuda')
    w, i, c, loss = yan.moe_route(logits, 4, mask=mask)
    assert float(loss) == 0 and int(c.abs().sum()) == 0 and bool((w == 0).all()) and bool((i == -1).all()) and w.shape == i.shape == (tokens, 4)
    dx = yan.moe_route_backward(logits, i, c, torch.ones(tokens, 4, device='cuda'), torch.ones(1, device='cuda'))
    assert bool((dx == 0).all()) and dx.shape == logits.shape


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('experts,top_k', [(40, 5), (256, 8), (1000, 3)])
def test_sigmoid_rows_far_below_zero(experts, top_k, dtype):
    """What is a quotient of scores is defined however small they are: weights, shares and their gradient, large gradients of the weights included."""
    g = _gen(experts)
    centre = torch.tensor([-20.0, -60, -80, -86, -88, -95, -103, -200, -1000, -1e6, 3.0, -0.5], device='cuda')
    logits = (centre[:, None] + torch.randn(12, experts, generator=g, device='cuda').clamp(-6, 6)).to(dtype)
    logits[10, 1:] = -95.0                          # but one
    logits[10, :1] = 2.0
    w, i, c, loss = yan.moe_route(logits, top_k, 'sigmoid', True)
    leaf = logits.double().requires_grad_()
    log_s = torch.nn.functional.logsigmoid(leaf)
    p, order = torch.softmax(log_s, 1), torch.argsort(logits.double(), dim=1, descending=True, stable=True)[:, :top_k]
    want = torch.softmax(log_s.gather(1, order), 1)
    assert torch.equal(i.long(), order) and int(c.sum()) == 12 * top_k
    # a score 4 u, and |l - largest| <= 13 of it (row 10: those far below the one are less than 2^-126), a sum over the row, one over the picks, two quotients
    score_off = (4 + 13 + 22 + 6 + 2) * U
    normal = torch.full_like(want, 2.0 ** -126)
    _close(w, want, (score_off * want + normal).detach(), 'weights')
    loss_want = experts / (top_k * 144) * (c.double() * p.sum(0)).sum()
    _close(loss, loss_want, (score_off + 112 * U) * loss_want.detach(), 'loss')
    dw, dl = 1e6 * torch.randn(12, top_k, generator=g, device='cuda'), torch.tensor(50.0, device='cuda')
    got = yan.moe_route_backward(logits, i, c, dw, dl, 'sigmoid', True)
    ((want * dw.double()).sum() + dl.double() * loss_want).backward()
    pull = 50.0 * experts * c.double() / (top_k * 144)
    size = torch.zeros_like(p).scatter_(1, order, want * (dw.double().abs() + (want * dw.double().abs()).sum(1, keepdim=True)))
    size = (size + p * (pull + (p * pull).sum(1, keepdim=True))).detach()
    bound = (5 * score_off + 30 * U) * size + 1e7 * 2.0 ** -126
    if dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (leaf.grad.abs() + bound)
    _close(got, leaf.grad, bound, 'gradient')
    # without renormalising a weight is the score, which is 0 below the smallest normal number
    w, i, _, _ = yan.moe_route(logits, top_k, 'sigmoid', False)
    want = torch.sigmoid(logits.double()).gather(1, order)
    _close(w, want, score_off * want + 2.0 ** -126, 'scores')


@pytest.mark.parametrize('renormalize', [True, False])
def test_sigmoid_gradient_of_confident_logits(renormalize):
    """The slope of a score near one is as exact, relatively, as anywhere else: 1 - s is not a difference of rounded numbers."""
    g = _gen(17)
    tokens, experts, top_k = 64, 32, 4
    logits = 60 * torch.rand(tokens, experts, generator=g, device='cuda') - 30
    logits[:8] = 20 + 10 * torch.rand(8, experts, generator=g, device='cuda')
    w, i, c, loss = yan.moe_route(logits, top_k, 'sigmoid', renormalize)
    dw = torch.randn(tokens, top_k, generator=g, device='cuda')
    for dl in (None, torch.tensor(3.0, device='cuda')):
        got = yan.moe_route_backward(logits, i, c, dw, dl, 'sigmoid', renormalize)
        l = logits.double()
        s, slope = torch.sigmoid(l), torch.sigmoid(-l)
        p = s / s.sum(1, keepdim=True)
        weight = s.gather(1, i.long())
        if renormalize:
            weight = weight / weight.sum(1, keepdim=True)
            inner, spread = dw.double() - (weight * dw.double()).sum(1, keepdim=True), dw.double().abs() + (weight * dw.double().abs()).sum(1, keepdim=True)
        else:
            inner, spread = dw.double(), dw.double().abs()
        pull = (0.0 if dl is None else 3.0) * experts * c.double() / (top_k * tokens * tokens)
        back = p * (pull - (p * pull).sum(1, keepdim=True))
        want = slope * (torch.zeros_like(s).scatter_(1, i.long(), weight * inner) + back)
        size = slope * (torch.zeros_like(s).scatter_(1, i.long(), weight * spread) + p * (pull + (p * pull).sum(1, keepdim=True)))
        # as for the gradient above, an exponential's argument of up to 30
        _close(got, want, (5 * (4 + 30 + 22 + 6 + 2) * U + 30 * U) * size + 2.0 ** -126, f'gradient with loss {dl is not None}')


def test_route_of_more_picks_than_a_number_of_31_bits_counts():
    """The limits are 2^30 tokens and 16 picks, whose product no 32 bits hold: loss and gradient of 402653184 equal tokens with 8 picks."""
    tokens, experts, top_k = 3 << 27, 16, 8
    row = torch.linspace(1, -1, experts, device='cuda').bfloat16()
    logits = row.expand(tokens, experts).contiguous()
    w, i, c, loss = yan.moe_route(logits, top_k)
    assert c.tolist() == [tokens] * top_k + [0] * (experts - top_k) and i[-1].tolist() == list(range(top_k))
    p = torch.softmax(row.double(), 0)
    _close(w[-1], p[:top_k] / p[:top_k].sum(), 50 * U * torch.ones(top_k, device='cuda'))
    # a lane adds up the shares of every 16384th token, then come the sums over a workgroup and over 256 of them
    want = experts / top_k * p[:top_k].sum()
    _close(loss, want, (tokens / 16384 + 100 + 50) * U * want, 'loss')
    del w
    got = yan.moe_route_backward(logits, i, c, None, torch.full((1, ), float(tokens), device='cuda'))
    pull = torch.zeros_like(p)
    pull[:top_k] = experts / top_k
    want = p * (pull - (p * pull).sum())
    bound = 200 * U * p * (pull + (p * pull).sum())
    for at in (0, tokens // 2, tokens - 1):
        _close(got[at], want, bound + 2.0 ** -8 * (want.abs() + bound), 'gradient')


# Dispatch

def _places(indices, experts):
    """(expert, rank) of every pair that has an expert, by the definition."""
    seen, places = [0] * experts, []
    for t, row in enumerate(indices.cpu().tolist()):
        for i, e in enumerate(row):
            if 0 <= e < experts:
                places.append((t, i, e, seen[e]))
                seen[e] += 1
    return places, seen


def _routing(g, tokens, experts, top_k, skew, holes=0.0):
    noise = torch.rand(tokens, experts, generator=g, device='cuda').log().neg().log().neg()
    indices = torch.topk(noise + skew * torch.randn(experts, generator=g, device='cuda'), top_k, dim=1).indices.int()
    if holes:
        indices = torch.where(torch.rand(tokens, 1, generator=g, device='cuda') < holes, torch.full_like(indices, -1), indices)
    return indices.contiguous()


DISPATCHES = [(1, 128, 4, 1), (1, 7168, 256, 8), (64, 2048, 32, 4), (3, 256, 1, 1), (511, 384, 9, 8), (512, 128, 64, 8), (513, 256, 64, 8), (600, 1152, 130, 7),
              (2000, 128, 1000, 16), (4100, 512, 3, 1)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tokens,k,experts,top_k', DISPATCHES)
def test_dispatch_contiguous(tokens, k, experts, top_k, dtype):
    g = _gen(tokens + k)
    x = torch.randn(tokens, k, generator=g, device='cuda').to(dtype)
    indices = _routing(g, tokens, experts, top_k, 1.0, holes=0.1)
    want_codes, want_scales = yan.per_token_cast_to_fp8(x)
    places, seen = _places(indices, experts)
    starts = [0]
    for n in seen:
        starts.append(starts[-1] + (n + 127) // 128 * 128)
    m_sum = yan.get_contiguous_layout_rows(tokens, top_k, experts) + 128
    for token_contiguous in (False, True):
        codes = torch.full((m_sum, k), 0x55, dtype=torch.uint8, device='cuda').view(F8)
        scales = torch.full((k // 128, m_sum), -3.0, device='cuda').t() if token_contiguous else torch.full((m_sum, k // 128), -3.0, device='cuda')
        rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, experts, (codes, scales))
        assert offsets.tolist() == starts
        want_rows, want_source = torch.full((tokens, top_k), -1), torch.full((m_sum, ), -1)
        for t, i, e, rank in places:
            want_rows[t, i] = starts[e] + rank
            want_source[starts[e] + rank] = t
        assert torch.equal(rows.cpu().long(), want_rows) and torch.equal(source.cpu().long(), want_source)
        want_m = torch.full((m_sum, ), -1)
        for e in range(experts):
            want_m[starts[e]:starts[e + 1]] = e
        assert torch.equal(m_indices.cpu().long(), want_m)
        held = source >= 0
        at = source[held].long()
        assert torch.equal(codes.view(torch.uint8)[held], want_codes.view(torch.uint8)[at]) and torch.equal(scales[held], want_scales[at])
        assert bool((codes.view(torch.uint8)[~held] == 0x55).all()) and bool((scales[~held] == -3.0).all())         # left as they were


@pytest.mark.parametrize('tokens,k,experts,top_k,m_max', [(1, 128, 4, 2, 1), (64, 7168, 32, 4, 64), (200, 256, 8, 3, 16), (700, 384, 16, 8, 100), (0, 128, 4, 2, 8)])
def test_dispatch_masked_drops_what_does_not_fit(tokens, k, experts, top_k, m_max):
    g = _gen(tokens + k)
    x = torch.randn(tokens, k, generator=g, device='cuda').bfloat16()
    indices = _routing(g, tokens, experts, top_k, 1.0, holes=0.05)
    want_codes, want_scales = yan.per_token_cast_to_fp8(x)
    places, seen = _places(indices, experts)
    for layout in range(3):
        codes = torch.full((experts, m_max, k), 0x55, dtype=torch.uint8, device='cuda').view(F8)
        shape = {0: (experts, m_max, k // 128), 1: (experts, k // 128, m_max), 2: (m_max, k // 128, experts)}[layout]
        scales = torch.full(shape, -3.0, device='cuda').permute({0: (0, 1, 2), 1: (0, 2, 1), 2: (2, 0, 1)}[layout])
        rows, masked_m = yan.moe_dispatch_to_fp8_masked(x, indices, (codes, scales))
        assert masked_m.tolist() == [min(n, m_max) for n in seen]
        want_rows = torch.full((tokens, top_k), -1)
        held = torch.zeros(experts, m_max, dtype=torch.bool)
        for t, i, e, rank in places:
            if rank < m_max:
                want_rows[t, i] = e * m_max + rank
                held[e, rank] = True
        assert torch.equal(rows.cpu().long(), want_rows)
        for t, i, e, rank in places[:50]:
            if rank < m_max:
                assert torch.equal(codes[e, rank].view(torch.uint8), want_codes[t].view(torch.uint8)) and torch.equal(scales[e, rank], want_scales[t])
        held = held.cuda()
        assert bool((codes.view(torch.uint8)[~held] == 0x55).all()) and bool((scales[~held] == -3.0).all())


@pytest.mark.parametrize('tokens', [40, 900])
def test_dispatch_into_too_few_rows_and_an_expert_twice(tokens):
    """Pairs past the rows that there are go nowhere, the offsets end with them; an expert that a token names twice gets it twice."""
    g = _gen(8)
    x = torch.randn(tokens, 128, generator=g, device='cuda').bfloat16()
    indices = torch.randint(0, 3, (tokens, 8), generator=g, device='cuda').int()
    places, seen = _places(indices, 3)
    assert tokens * 8 > 256
    codes, scales = torch.zeros(256, 128, dtype=torch.uint8, device='cuda').view(F8), torch.zeros(256, 1, device='cuda')
    rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, 3, (codes, scales))
    starts = [0]
    for n in seen:
        starts.append(starts[-1] + (n + 127) // 128 * 128)
    assert offsets.tolist() == [min(s, 256) for s in starts]
    for t, i, e, rank in places:
        row = starts[e] + rank
        assert int(rows[t, i]) == (row if row < 256 else -1) or tokens > 100
    want = torch.tensor([starts[e] + rank if starts[e] + rank < 256 else -1 for _, _, e, rank in places]).view(tokens, 8)
    assert torch.equal(rows.cpu().long(), want)
    assert m_indices.tolist() == [next((e for e in range(3) if starts[e] <= r < starts[e + 1]), -1) for r in range(256)]


# Combine

@pytest.mark.parametrize('weighted', [True, False])
@pytest.mark.parametrize('tokens,n,m,top_k', [(1, 8, 1, 1), (1, 7168, 512, 8), (64, 512, 640, 4), (33, 520, 384, 3), (100, 2056, 1024, 7), (700, 128, 8192, 8), (5, 4096, 128, 16),
                                              (0, 64, 128, 2), (3, 64, 0, 2)])
def test_combine_and_its_gradient(tokens, n, m, top_k, weighted):
    g = _gen(tokens + n + m)
    y = torch.randn(m, n, generator=g, device='cuda').bfloat16()
    free = torch.randperm(m, generator=g, device='cuda')[:tokens * top_k]
    rows = torch.full((tokens * top_k, ), -1, device='cuda')
    rows[:free.numel()] = free
    rows = torch.where(torch.rand(tokens * top_k, generator=g, device='cuda') < 0.1, torch.full_like(rows, -1), rows).view(tokens, top_k)
    source = torch.full((m, ), -1, dtype=torch.int32, device='cuda')
    held = rows >= 0
    source[rows[held]] = torch.arange(tokens, device='cuda')[:, None].expand(-1, top_k)[held].int()
    y[source < 0] = float('nan')                                            # nobody reads those
    rows = torch.where(rows < 0, torch.full_like(rows, -1 if top_k % 2 else m), rows).int()         # outside of y on either side
    w = torch.randn(tokens, top_k, generator=g, device='cuda') if weighted else None
    weights = (torch.ones(tokens, top_k, device='cuda') if w is None else w).double() * held
    taken = y[rows.clamp(0, max(m - 1, 0)).long().reshape(-1)].view(tokens, top_k, n).double() if m else torch.zeros(tokens, top_k, n, device='cuda').double()
    taken = torch.where(held[..., None], taken, torch.zeros_like(taken))
    out = torch.full((tokens + 1, n), 7.0, device='cuda').bfloat16()
    yan.moe_combine(y, rows, w, out[:tokens])
    want, size = (weights[..., None] * taken).sum(1), (weights[..., None] * taken).abs().sum(1)
    bound = (top_k + 1) * U * size
    _close(out[:tokens], want, bound + 2.0 ** -8 * (want.abs() + bound), 'out')
    assert bool((out[tokens:] == 7.0).all())
    d = torch.randn(tokens, n, generator=g, device='cuda').bfloat16()
    grad_y, grad_w = yan.moe_combine_backward(d, y, rows, w, source)
    want_y = torch.zeros(m, n, dtype=torch.float64, device='cuda')
    want_y[rows[held].long()] = (weights[..., None] * d.double()[:, None])[held]
    _close(grad_y, want_y, (2.0 ** -8 + 2 * U) * want_y.abs(), 'grad_y')
    if weighted:
        want_w, size_w = (taken * d.double()[:, None]).sum(-1), (taken * d.double()[:, None]).abs().sum(-1)
        _close(grad_w, want_w, (n / 64 + 16) * U * size_w, 'grad_weights')          # a lane's own (of 64 or more), then 8 steps
    else:
        assert grad_w is None


def test_combine_of_no_columns():
    rows = torch.tensor([[0, 1], [2, -1], [3, 5]], dtype=torch.int32, device='cuda')
    source = torch.tensor([0, 0, 1, 2, -1, 2], dtype=torch.int32, device='cuda')
    y, out, w = torch.empty(6, 0, dtype=torch.bfloat16, device='cuda'), torch.empty(3, 0, dtype=torch.bfloat16, device='cuda'), torch.ones(3, 2, device='cuda')
    for _ in range(2):          # the second natively
        yan.moe_combine(y, rows, w, out)
        grad_y, grad_w = yan.moe_combine_backward(out, y, rows, w, source)
        assert grad_y.shape == y.shape and grad_y.dtype == y.dtype and grad_w.shape == w.shape and bool((grad_w == 0).all())
        grad_y, grad_w = yan.moe_combine_backward(out, y, rows, None, source)
        assert grad_y.shape == y.shape and grad_w is None


# Quantiser

def _turned(x, source):
    """codes (as values) and exponent bytes by the definition, in 64 bits on the CPU."""
    x = x.double().cpu()
    if source is None:
        wide = torch.cat([x, x.new_zeros(-x.size(0) % 128, x.size(1))])
    else:
        s = source.cpu().long()
        inside = (s >= 0) & (s < x.size(0))
        wide = torch.where(inside[:, None], x[s.clamp(0, x.size(0) - 1)] if x.size(0) else x.new_zeros(s.numel(), x.size(1)), x.new_zeros(()))
    v = wide.t().reshape(x.size(1), wide.size(0) // 128, 128)
    amax = torch.where(torch.isfinite(v), v.abs(), v.new_zeros(())).amax(-1).clamp(min=2.0 ** -100)
    fraction, exponent = torch.frexp(amax)
    e = exponent - 9 + (fraction > 0.875).int()
    scaled = torch.ldexp(v, -e[..., None])
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6, max=448))) - 3)
    q = torch.where(torch.isfinite(v), torch.round(scaled / step) * step, v.new_full((), float('nan')))
    return q.reshape(x.size(1), wide.size(0)), e + 127


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n', [(1, 8), (127, 64), (128, 72), (129, 8), (1000, 136), (300, 2112), (0, 16), (5, 0), (513, 64)])
def test_per_channel_cast(m, n, dtype):
    g = _gen(m + n)
    x = (torch.randn(m, n, generator=g, device='cuda') * torch.exp(3 * torch.randn(1, n, generator=g, device='cuda'))).to(dtype)
    if m > 100:
        x[:, 0] = 0
        x[3, 1], x[5, 1], x[7, 1] = float('nan'), float('inf'), -float('inf')
        x[:, 2] *= 1e-30
        x[0, 3] = 448.0                     # on a border between two exponents
        x[0, 4] = 3e38
    codes, scales = yan.per_channel_cast_to_fp8(x)
    k = (m + 127) // 128 * 128
    assert codes.shape == (n, k) and scales.shape == (n, k // 128) and scales.dtype == torch.uint8
    want, want_e = _turned(x, None)
    assert torch.equal(scales.cpu().int(), want_e.int())
    assert torch.equal(codes.float().cpu().nan_to_num(500.0), want.float().nan_to_num(500.0))
    if m and n:
        source = torch.randint(-2, m + 2, (384, ), generator=g, device='cuda').int()
        codes, scales = yan.per_channel_cast_to_fp8(x, source)
        want, want_e = _turned(x, source)
        assert torch.equal(scales.cpu().int(), want_e.int())
        assert torch.equal(codes.float().cpu().nan_to_num(500.0), want.float().nan_to_num(500.0))


@pytest.mark.parametrize('dtype,m,n', [(torch.bfloat16, 600, 7168), (torch.float32, 4000, 6000)])
def test_per_channel_cast_of_many_gathered_rows(dtype, m, n):
    """The same bits from one call as from one for every 1280 rows."""
    g = _gen(n)
    x = torch.randn(m, n, generator=g, device='cuda').to(dtype)
    source = torch.randint(-1, m, (8 * 1280, ), generator=g, device='cuda').int()
    codes, scales = yan.per_channel_cast_to_fp8(x, source)
    for r in range(0, source.numel(), 1280):
        part, part_scales = yan.per_channel_cast_to_fp8(x, source[r:r + 1280].contiguous())
        assert torch.equal(codes[:, r:r + 1280].contiguous().view(torch.uint8), part.view(torch.uint8))
        assert torch.equal(scales[:, r // 128:r // 128 + 10], part_scales)


# Weight gradients

def _operand(g, rows, k, wide=False):
    """Codes and scales of an operand with `rows` rows, the scales' rows a multiple of four bytes apart and, with `wide`, further than they have to be."""
    codes = torch.randint(0, 256, (rows, k), generator=g, device='cuda', dtype=torch.uint8)
    codes = torch.where((codes & 0x7f) == 0x7f, codes & 0x80, codes)                      # no NaN
    pitch = (k // 128 + 3) // 4 * 4 + (8 if wide else 0)
    scales = torch.randint(118, 131, (rows, pitch), generator=g, device='cuda', dtype=torch.uint8)[:, :k // 128]
    return codes.view(F8), scales


def _decode(operand):
    codes, scales = operand
    return codes.double() * torch.exp2(scales.double() - 127).repeat_interleave(128, 1)


def _check_product(got, a, b, before, bound_terms=None):
    want, size = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    if before is not None:
        want, size = want + before, size + before.abs()
    # a sum of 32 products in the matrix core, k / 32 of those behind each other, then parts and what was there; each addition off by a step at most
    _close(got, want, (a.size(1) / 32 + 32 + 16) * 2 * U * size, 'product')


KERNELS = testing.WGRAD_KERNELS


@pytest.mark.parametrize('m,n,k', [(1, 4, 128), (16, 16, 128), (64, 64, 512), (65, 68, 640), (128, 256, 256), (257, 132, 1280), (300, 516, 2048), (520, 260, 384), (33, 1000, 5120)])
@pytest.mark.parametrize('kernel', KERNELS)
def test_weight_gradient_kernels(kernel, m, n, k):
    g = _gen(m + n + k)
    a, b = _operand(g, m, k), _operand(g, n, k, wide=True)
    for accumulate in (False, True):
        held = torch.randn(m + 2, n, generator=g, device='cuda')
        out = held.clone()
        wgrad._wgrad(a, b, out[:m], None, accumulate, kernel)
        _check_product(out[:m], _decode(a), _decode(b), held[:m].double() if accumulate else None)
        assert torch.equal(out[m:], held[m:])
        again = held.clone()
        wgrad._wgrad(a, b, again[:m], None, accumulate, kernel)
        assert torch.equal(again, out)


@pytest.mark.parametrize('m,n,tiles', [(64, 64, [1, 0, 2, 5]), (200, 132, [0, 0, 3]), (300, 520, [1, 1, 0, 9, 2]), (513, 260, [4]), (130, 36, [0]), (16, 2000, [7, 1, 6, 2, 0, 0, 3, 1])])
@pytest.mark.parametrize('kernel', KERNELS)
def test_grouped_weight_gradient_kernels(kernel, m, n, tiles):
    """Groups of uneven lengths, some without columns, that start anywhere in a dword of scales."""
    g = _gen(m + n)
    groups, k = len(tiles), max(1, sum(tiles)) * 128
    if kernel[1] > 1 and kernel[1] * groups * ((-(-m // 64) * -(-n // 64) + 7) // 8 * 8) > 1024:           # more parts than a workspace holds are refused
        a, b = _operand(g, m, k), _operand(g, n, k)
        with pytest.raises(AssertionError):
            wgrad._wgrad(a, b, torch.zeros(groups, m, n, device='cuda'), torch.zeros(groups + 1, dtype=torch.int32, device='cuda'), False, kernel)
        return
    a, b = _operand(g, m, k), _operand(g, n, k)
    ends = torch.tensor([0] + tiles).cumsum(0) * 128
    for accumulate in (False, True):
        held = torch.randn(groups, m, n, generator=g, device='cuda')
        out = held.clone()
        wgrad._wgrad(a, b, out, ends.int().cuda(), accumulate, kernel)
        for q in range(groups):
            lo, hi = int(ends[q]), int(ends[q + 1])
            if lo == hi:
                assert torch.equal(out[q], held[q]) if accumulate else bool((out[q] == 0).all())
            else:
                _check_product(out[q], _decode(a)[:, lo:hi].contiguous(), _decode(b)[:, lo:hi].contiguous(), held[q].double() if accumulate else None)


@pytest.mark.parametrize('m,n', [(1, 64), (3, 100), (8, 2000), (65, 132), (72, 64), (136, 4), (193, 260), (257, 68), (264, 520)])
@pytest.mark.parametrize('kernel', KERNELS)
def test_weight_gradients_of_one_k_tile_with_few_rows_in_the_last_tile(kernel, m, n):
    """Right behind the copies of the only k-tile the sums are turned round, in the smaller kernels in the same LDS; rows behind the last one are none of theirs."""
    g = _gen(m * n)
    a, b = _operand(g, m, 128), _operand(g, n, 128)
    out = torch.full((m + 1, n), 7.0, device='cuda')
    wgrad._wgrad(a, b, out[:m], None, False, kernel)
    _check_product(out[:m], _decode(a), _decode(b), None)
    assert bool((out[m:] == 7.0).all())
    groups = 2 if kernel[1] > 8 else 3
    if kernel[1] * groups * ((-(-m // 64) * -(-n // 64) + 7) // 8 * 8) > 1024:              # more parts than a workspace holds
        return
    a, b = _operand(g, m, 128 * groups), _operand(g, n, 128 * groups)
    held = torch.randn(groups, m, n, generator=g, device='cuda')
    grouped = held.clone()
    wgrad._wgrad(a, b, grouped, torch.arange(groups + 1, device='cuda').int() * 128, True, kernel)
    for q in range(groups):
        _check_product(grouped[q], _decode(a)[:, 128 * q:128 * q + 128].contiguous(), _decode(b)[:, 128 * q:128 * q + 128].contiguous(), held[q].double())


@pytest.mark.parametrize('low,high', [(10, 246), (246, 10), (10, 10), (19, 235)])
def test_weight_gradients_with_scales_at_the_ends_of_their_range(low, high):
    """Every code times a scale of 2^-117 to 2^119 is a normal bf16 number, so products of both ends are those of the definition."""
    g = _gen(low)
    for kernel in KERNELS[:4]:
        a, b = _operand(g, 72, 512), _operand(g, 68, 512)
        a[1].fill_(low)
        b[1].fill_(high)
        out = torch.zeros(72, 68, device='cuda')
        wgrad._wgrad(a, b, out, None, False, kernel)
        want = _decode(a) @ _decode(b).t().contiguous()
        size = _decode(a).abs() @ _decode(b).abs().t().contiguous()
        # (of two small scales the products are less than the smallest normal number of fp32)
        _close(out, want, (512 / 32 + 48) * 2 * U * size + 2.0 ** -126, 'product')


def test_weight_gradient_edges():
    """K of zero, NaN codes, offsets that do not ascend or leave K (whatever they say, nothing outside is read), a cap on compute units."""
    g = _gen(1)
    a, b = _operand(g, 40, 0), _operand(g, 24, 0)
    out = torch.ones(40, 24, device='cuda')
    yan.gemm_fp8_fp8_fp32_nt(a, b, out, accumulate=True)
    assert bool((out == 1).all())
    yan.gemm_fp8_fp8_fp32_nt(a, b, out)
    assert bool((out == 0).all())
    a, b = _operand(g, 40, 640), _operand(g, 24, 640)
    a[0].view(torch.uint8)[7, 300] = 0x7f
    out = torch.zeros(40, 24, device='cuda')
    yan.gemm_fp8_fp8_fp32_nt(a, b, out)
    assert bool(torch.isnan(out[7]).all()) and not bool(torch.isnan(out[:7]).any()) and not bool(torch.isnan(out[8:]).any())
    a, b = _operand(g, 40, 640), _operand(g, 24, 640)
    out = torch.full((4, 40, 24), 5.0, device='cuda')
    yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(a, b, out, torch.tensor([-256, 256, 128, 512, 1 << 30], dtype=torch.int32, device='cuda'))
    for q, (lo, hi) in enumerate([(0, 256), (256, 256), (128, 512), (512, 640)]):
        _check_product(out[q], _decode(a)[:, lo:hi].contiguous(), _decode(b)[:, lo:hi].contiguous(), None)
    want = torch.zeros(600, 700, device='cuda')
    a, b = _operand(g, 600, 1280), _operand(g, 700, 1280)
    for kernel in KERNELS[:4]:
        wgrad._wgrad(a, b, want, None, False, kernel)
        for cap in (1, 7, 40):
            try:
                yan.set_num_sms(cap)
                out = torch.zeros_like(want)
                wgrad._wgrad(a, b, out, None, False, kernel)
            finally:
                yan.set_num_sms(torch.cuda.get_device_properties(0).multi_processor_count)
            _check_product(out, _decode(a), _decode(b), None)


def test_offsets_past_32_bits():
    """Rows of operands, activations and expert outputs that lie 4 GiB and more behind the first."""
    g = _gen(4)
    k = (1 << 23) - 128
    a = (torch.zeros(520, k, dtype=torch.uint8, device='cuda').view(F8), torch.full((520, 65536), 127, dtype=torch.uint8, device='cuda')[:, :k // 128])
    b = (torch.zeros(4, k, dtype=torch.uint8, device='cuda').view(F8), torch.full((4, 65536), 127, dtype=torch.uint8, device='cuda')[:, :k // 128])
    a[0].view(torch.uint8)[519, k - 1], b[0].view(torch.uint8)[3, k - 1] = 0x40, 0x44                        # 2 and 3
    a[0].view(torch.uint8)[515, 5], b[0].view(torch.uint8)[2, 5] = 0x40, 0x40
    out = torch.zeros(520, 4, device='cuda')
    yan.gemm_fp8_fp8_fp32_nt(a, b, out)
    want = torch.zeros_like(out)
    want[519, 3], want[515, 2] = 6.0, 4.0
    assert torch.equal(out, want)
    del a, b
    m, n = 300032, 8192                     # 4.9 GB of bf16, 2.5 GB of codes
    y = torch.zeros(m, n, dtype=torch.bfloat16, device='cuda')
    y[-3:] = torch.randn(3, n, generator=g, device='cuda').bfloat16()
    rows = torch.tensor([[m - 1, 0], [m - 2, m - 3]], dtype=torch.int32, device='cuda')
    out = torch.empty(2, n, dtype=torch.bfloat16, device='cuda')
    yan.moe_combine(y, rows, None, out)
    assert torch.equal(out[0], y[-1]) and torch.equal(out[1], (y[-2].float() + y[-3].float()).bfloat16())
    source = torch.full((m, ), -1, dtype=torch.int32, device='cuda')
    source[rows.long().reshape(-1)] = torch.tensor([0, 0, 1, 1], dtype=torch.int32, device='cuda')
    d = torch.randn(2, n, generator=g, device='cuda').bfloat16()
    grad_y, _ = yan.moe_combine_backward(d, y, rows, None, source)
    assert torch.equal(grad_y[-3:], d[[1, 1, 0]]) and torch.equal(grad_y[0], d[0]) and int((grad_y[1:-3] != 0).sum()) == 0
    del grad_y, source
    picked = torch.full((128, ), -1, dtype=torch.int32, device='cuda')
    picked[5] = m - 1
    codes, scales = yan.per_channel_cast_to_fp8(y, picked)
    want, want_e = _turned(torch.cat([y[-1:]]), torch.where(picked < 0, -1, 0).int())
    assert torch.equal(codes.float().cpu(), want.float()) and torch.equal(scales.cpu().int(), want_e.int())
    del y
    codes, scales = torch.zeros(2, 300032, n, dtype=torch.uint8, device='cuda').view(F8), torch.zeros(2, 300032, n // 128, device='cuda')
    x = torch.randn(8, n, generator=g, device='cuda').bfloat16()
    rows, masked_m = yan.moe_dispatch_to_fp8_masked(x, torch.ones(8, 1, dtype=torch.int32, device='cuda'), (codes, scales))
    assert rows.flatten().tolist() == list(range(300032, 300040)) and masked_m.tolist() == [0, 8]
    want_codes, want_scales = yan.per_token_cast_to_fp8(x)
    assert torch.equal(codes[1, :8].view(torch.uint8), want_codes.view(torch.uint8)) and torch.equal(scales[1, :8], want_scales)


# All of them in a row, as a layer uses them

def _layer(tokens, hidden, inner, experts, top_k, seed):
    g = _gen(seed)
    x = torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16()
    logits = torch.randn(tokens, experts, generator=g, device='cuda')
    stacked = [yan.per_block_cast_to_fp8(torch.randn(inner, hidden, generator=g, device='cuda').bfloat16() * 0.05) for _ in range(experts)]
    w8, ws = torch.stack([c.view(torch.uint8) for c, _ in stacked]).view(F8), torch.stack([s for _, s in stacked])
    return x, logits, w8, ws, torch.randn(tokens, inner, generator=g, device='cuda').bfloat16()


def _weights_of(w8, ws):
    inner, hidden = w8.shape[1:]
    return w8.double() * ws.double().repeat_interleave(128, 1)[:, :inner].repeat_interleave(128, 2)


def test_training_step_of_a_layer():
    """Route, dispatch, the experts' GEMM, combine, and back: outputs and all gradients against 64 bits on the same quantised operands."""
    tokens, hidden, inner, experts, top_k = testing.MOE_TRAINING_LAYER
    x, logits, w8, ws, dout = _layer(tokens, hidden, inner, experts, top_k, 11)
    mask = torch.arange(tokens, device='cuda') % 50 != 7
    weights, indices, counts, loss = yan.moe_route(logits, top_k, 'softmax', True, mask)
    m_sum = yan.get_contiguous_layout_rows(tokens, top_k, experts)
    codes, scales = torch.empty(m_sum, hidden, dtype=F8, device='cuda'), torch.empty(hidden // 128, m_sum, device='cuda').t()
    rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, experts, (codes, scales))
    assert int((m_indices >= 0).sum()) == int(((counts + 127) // 128 * 128).sum())
    y = torch.empty(m_sum, inner, dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_fp8_fp8_bf16_nt_contiguous((codes, scales), (w8, ws), y, m_indices)
    out = torch.empty(tokens, inner, dtype=torch.bfloat16, device='cuda')
    yan.moe_combine(y, rows, weights, out)
    # the same from the definition
    x8, xs = yan.per_token_cast_to_fp8(x)
    xd = x8.double() * xs.double().repeat_interleave(128, 1)
    wd = _weights_of(w8, ws)
    per_expert = torch.stack([xd @ wd[e].t() for e in range(experts)], 1)                      # [tokens, experts, inner]
    picked = per_expert.gather(1, indices.clamp(min=0).long()[..., None].expand(-1, -1, inner))
    want = (weights.double()[..., None] * picked).sum(1)
    size = (weights.double()[..., None] * picked.abs()).sum(1)
    assert bool((out[~mask] == 0).all())
    # y is rounded to bf16, then the sum; what the matrix core leaves out of fp8 products is about 1e-4 of their magnitudes
    loose = 1e-4 * (weights.double()[..., None] * (xd.abs().norm(dim=1)[:, None, None] * wd.norm(dim=2).max())).sum(1)
    _close(out, want, 2.0 ** -7 * size + 2.0 ** -8 * want.abs() + loose, 'out')
    # back
    grad_y, grad_weights = yan.moe_combine_backward(dout, y, rows, weights, source)
    assert bool((grad_y[source < 0] == 0).all())
    a, b = yan.per_channel_cast_to_fp8(grad_y), yan.per_channel_cast_to_fp8(x, source)
    grad_w = torch.zeros(experts, inner, hidden, device='cuda')
    yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(a, b, grad_w, offsets)
    first = grad_w.clone()
    yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(a, b, grad_w, offsets, accumulate=True)
    assert torch.equal(grad_w, 2 * first)
    ends = offsets.tolist()
    for e in range(experts):
        if ends[e] < ends[e + 1]:
            _check_product(first[e], _decode(a)[:, ends[e]:ends[e + 1]].contiguous(), _decode(b)[:, ends[e]:ends[e + 1]].contiguous(), None)
    # against the gradient of the layer itself: e4m3 is off by 2^-4 of a value at most on either side, 2^-3 of the products' magnitudes in all
    for e in range(experts):
        use = (indices == e) * weights.double()
        want = (use.sum(1)[:, None] * dout.double()).t() @ x.double()
        size = (use.sum(1)[:, None] * dout.double().abs()).t() @ x.double().abs()
        _close(first[e], want, (2.0 ** -3 + 2.0 ** -7) * size + 1e-30, 'gradient of the experts')
    want = (dout.double()[:, None] * torch.where((rows >= 0)[..., None], y[rows.clamp(min=0).long().reshape(-1)].view(tokens, top_k, inner).double(),
                                                 torch.zeros((), device='cuda', dtype=torch.float64))).sum(-1)
    _close(grad_weights, want, 1e-4 * want.abs() + 1e-3, 'gradient of the weights')
    grad_logits = yan.moe_route_backward(logits, indices, counts, grad_weights, torch.ones((), device='cuda'))
    leaf = logits.double().requires_grad_()
    s = torch.softmax(leaf, 1)
    w = s.gather(1, indices.clamp(min=0).long())
    w = w / w.sum(1, keepdim=True) * mask[:, None]
    n = int(mask.sum())
    aux = experts / (top_k * n * n) * (counts.double() * (s * mask[:, None]).sum(0)).sum()
    ((w * grad_weights.double()).sum() + aux).backward()
    _close(grad_logits, leaf.grad, 1e-5 * grad_weights.abs().sum(1, keepdim=True) + 1e-7, 'gradient of the logits')
    # the tokens' gradient: what the experts hand back, summed over the picks
    grad_x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device='cuda')
    rows_back = torch.randn(m_sum, hidden, device='cuda').bfloat16()
    yan.moe_combine(rows_back, rows, None, grad_x)
    want = torch.where((rows >= 0)[..., None], rows_back[rows.clamp(min=0).long().reshape(-1)].view(tokens, top_k, hidden).double(), torch.zeros((), device='cuda', dtype=torch.float64))
    _close(grad_x, want.sum(1), 2.0 ** -8 * want.sum(1).abs() + 8 * U * want.abs().sum(1), 'gradient of the tokens')


@pytest.mark.parametrize('m_sum', [0, 128])
def test_training_step_of_no_tokens(m_sum):
    """An empty batch goes through the layer, forward and backward; its layout has no rows, or more than it needs."""
    hidden, inner, experts, top_k = 256, 384, 6, 3
    x, logits, w8, ws, dout = _layer(0, hidden, inner, experts, top_k, 13)
    assert yan.get_contiguous_layout_rows(0, top_k, experts) == 0
    for _ in range(2):          # the second natively
        weights, indices, counts, loss = yan.moe_route(logits, top_k)
        codes, scales = torch.zeros(m_sum, hidden, dtype=torch.uint8, device='cuda').view(F8), torch.zeros(hidden // 128, m_sum, device='cuda').t()
        rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, experts, (codes, scales))
        assert rows.shape == (0, top_k) and offsets.tolist() == [0] * (experts + 1) and m_indices.tolist() == source.tolist() == [-1] * m_sum
        y, out = torch.zeros(m_sum, inner, dtype=torch.bfloat16, device='cuda'), torch.empty(0, inner, dtype=torch.bfloat16, device='cuda')
        yan.moe_combine(y, rows, weights, out)
        grad_y, grad_weights = yan.moe_combine_backward(dout, y, rows, weights, source)
        assert grad_y.shape == y.shape and bool((grad_y == 0).all()) and grad_weights.shape == (0, top_k)
        grad_w = torch.full((experts, inner, hidden), 3.0, device='cuda')
        sides = yan.per_channel_cast_to_fp8(grad_y), yan.per_channel_cast_to_fp8(x, source)
        yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(*sides, grad_w, offsets, accumulate=True)
        assert bool((grad_w == 3.0).all())
        yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(*sides, grad_w, offsets)
        assert bool((grad_w == 0).all())
        assert yan.moe_route_backward(logits, indices, counts, grad_weights, loss).shape == (0, experts)


def test_tokens_that_find_no_row_at_all():
    """A layout without rows: every pair has none."""
    g = _gen(9)
    x, indices = torch.randn(40, 128, generator=g, device='cuda').bfloat16(), torch.randint(0, 3, (40, 2), generator=g, device='cuda').int()
    for tokens in (40, 40 * 64):          # few pairs and many
        many, chosen = x.repeat(tokens // 40, 1), indices.repeat(tokens // 40, 1)
        codes, scales = torch.zeros(0, 128, dtype=torch.uint8, device='cuda').view(F8), torch.zeros(0, 1, device='cuda')
        rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(many, chosen, 3, (codes, scales))
        assert bool((rows == -1).all()) and m_indices.numel() == source.numel() == 0 and offsets.tolist() == [0] * 4


def test_decode_step_of_a_layer():
    tokens, hidden, inner, experts, top_k, m_max, expected_m = testing.MOE_DECODE_LAYER
    x, logits, w8, ws, _ = _layer(tokens, hidden, inner, experts, top_k, 12)
    weights, indices, counts, _ = yan.moe_route(logits, top_k)
    codes, scales = torch.zeros(experts, m_max, hidden, dtype=torch.uint8, device='cuda').view(F8), torch.zeros(experts, m_max, hidden // 128, device='cuda')
    rows, masked_m = yan.moe_dispatch_to_fp8_masked(x, indices, (codes, scales))
    assert torch.equal(masked_m, counts.clamp(max=m_max))
    y = torch.full((experts, m_max, inner), float('nan'), dtype=torch.bfloat16, device='cuda')
    yan.m_grouped_gemm_fp8_fp8_bf16_nt_masked((codes, scales), (w8, ws), y, masked_m, expected_m)
    out = torch.empty(tokens, inner, dtype=torch.bfloat16, device='cuda')
    yan.moe_combine(y.view(experts * m_max, inner), rows, weights, out)
    x8, xs = yan.per_token_cast_to_fp8(x)
    xd, wd = x8.double() * xs.double().repeat_interleave(128, 1), _weights_of(w8, ws)
    picked = torch.stack([xd @ wd[e].t() for e in range(experts)], 1).gather(1, indices.long()[..., None].expand(-1, -1, inner))
    kept = (weights.double() * (rows >= 0))[..., None]
    loose = 1e-4 * (kept * (xd.abs().norm(dim=1)[:, None, None] * wd.norm(dim=2).max())).sum(1)
    _close(out, (kept * picked).sum(1), 2.0 ** -7 * (kept * picked.abs()).sum(1) + 2.0 ** -8 * (kept * picked).sum(1).abs() + loose, 'out')


# Graphs, streams, repeated calls

def _pass(x, logits, grad, buffers, sums):
    codes, scales, out = buffers
    weights, indices, counts, loss = yan.moe_route(logits, 4)
    rows, m_indices, source, offsets = yan.moe_dispatch_to_fp8_contiguous(x, indices, 40, (codes, scales))
    y = codes.float().bfloat16()
    yan.moe_combine(y, rows, weights, out)
    grad_y, grad_weights = yan.moe_combine_backward(grad, y, rows, weights, source)
    grad_logits = yan.moe_route_backward(logits, indices, counts, grad_weights, loss)
    a, b = yan.per_channel_cast_to_fp8(grad_y), yan.per_channel_cast_to_fp8(x, source)
    yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(a, b, sums, offsets)
    few = torch.empty(16, 16, device=x.device)
    yan.gemm_fp8_fp8_fp32_nt((a[0][:16].contiguous(), a[1][:16]), (b[0][:16].contiguous(), b[1][:16]), few)          # in parts
    return weights, indices, counts, loss, rows, m_indices, source, offsets, out.clone(), grad_y, grad_weights, grad_logits, sums.clone(), few


def _inputs(seed, tokens=900, hidden=256):
    g = _gen(seed)
    return torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16(), torch.randn(tokens, 40, generator=g, device='cuda'), torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16()


def _buffers(tokens=900, hidden=256):
    m_sum = yan.get_contiguous_layout_rows(tokens, 4, 40)
    codes = torch.zeros(m_sum, hidden, dtype=torch.uint8, device='cuda').view(F8)
    return (codes, torch.zeros(m_sum, hidden // 128, device='cuda'), torch.zeros(tokens, hidden, dtype=torch.bfloat16, device='cuda')), torch.zeros(40, hidden, hidden, device='cuda')


def test_captured_and_replayed():
    """A forward and backward pass in two graphs, replayed in turn with eager calls in between, each time with other inputs."""
    graphs = []
    for seed in (1, 2):
        held, (buffers, sums) = _inputs(seed), _buffers()
        _pass(*held, buffers, sums)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = _pass(*held, buffers, sums)
        graphs.append((graph, held, made, buffers, sums))          # a graph's memory stays
    for round_ in range(3):
        for n, (graph, held, made, *_) in enumerate(graphs):
            fresh = _inputs(10 + 2 * round_ + n)
            for to, value in zip(held, fresh):
                to.copy_(value)
            graph.replay()
            want = _pass(*fresh, *_buffers())
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(made, want)):
                assert torch.equal(a, b), (round_, n, i)


def test_on_other_streams_and_at_the_same_time():
    """The same bits from two streams side by side as from one call after the other."""
    inputs, homes = [_inputs(21), _inputs(22)], [_buffers(), _buffers()]
    want = [[t.clone() for t in _pass(*i, *_buffers())] for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(4):
        got = []
        for stream, i, home in zip(streams, inputs, homes):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(_pass(*i, *home))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b)), round_


@pytest.mark.parametrize('tokens,experts,top_k', [(5, 256, 8), (256, 256, 8), (257, 256, 8), (1024, 64, 6), (1025, 64, 6), (100, 500, 4), (70, 1024, 2)])
def test_route_joined_by_the_last_workgroup_and_by_a_second_kernel(tokens, experts, top_k, monkeypatch):
    """Counts and loss of few tokens are joined in the split-K workspace, which products use too; without it, by a second kernel."""
    logits = 2 * torch.randn(tokens, experts, generator=_gen(tokens), device='cuda')
    a = torch.randint(0, 100, (16, 4096), generator=_gen(1), device='cuda').to(torch.uint8).view(F8), torch.full((16, 32), 120, dtype=torch.uint8, device='cuda')
    products = torch.zeros(2, 16, 16, device='cuda')
    joined = []
    for n in range(2):          # the second natively
        joined.append(yan.moe_route(logits, top_k))
        yan.gemm_fp8_fp8_fp32_nt(a, a, products[n])
    monkeypatch.setenv('YAN_SPLIT_K', '0')
    apart = yan.moe_route(logits, top_k)
    assert all(torch.equal(p, q) for p, q in zip(*joined)) and torch.equal(products[0], products[1])
    assert all(torch.equal(p, q) for p, q in zip(joined[0][:3], apart[:3]))
    # the sums of a share have at most 64 rows added in one order or in another, each addition off by u of what is not negative
    _close(joined[0][3], apart[3].double(), 2 * 64 * U * apart[3].double().abs())


def test_repeated_calls_take_what_each_is_given():
    """Calls of known sizes are made natively: other inputs, other settings, other layouts and other memory each time, and new outputs."""
    x, logits, grad = _inputs(31)
    first = yan.moe_route(logits, 4)
    again = yan.moe_route(logits, 4)
    assert all(torch.equal(a, b) and a.data_ptr() != b.data_ptr() for a, b in zip(first, again))
    other = yan.moe_route(logits + 1e-3 * logits.square(), 4)
    assert not torch.equal(other[0], first[0])
    sigmoid = yan.moe_route(logits, 4, 'sigmoid')
    assert torch.equal(sigmoid[1], first[1]) and not torch.equal(sigmoid[0], first[0])
    raw = yan.moe_route(logits, 4, 'sigmoid', False)
    assert not torch.equal(sigmoid[0], raw[0])
    mask = torch.rand(900, device='cuda') < 0.5
    for m in (mask, ~mask, mask):
        got = yan.moe_route(logits, 4, mask=m)
        assert torch.equal(got[1] >= 0, m[:, None].expand(-1, 4))
    with pytest.raises(AssertionError):
        yan.moe_route(logits, 4, 'tanh')
    codes, scales = yan.per_channel_cast_to_fp8(x)
    for _ in range(3):
        more = yan.per_channel_cast_to_fp8(x)
        assert torch.equal(more[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(more[1], scales) and more[1].stride() == scales.stride()
    out, size = torch.zeros(256, 256, device='cuda'), torch.zeros(256, 256, device='cuda')
    for n in range(4):
        yan.gemm_fp8_fp8_fp32_nt((codes, scales), (codes, scales), out, accumulate=n > 0)
    yan.gemm_fp8_fp8_fp32_nt((codes, scales), (codes, scales), size)
    # four times the same product, added three times: each addition off by half a step of a sum up to four of it
    _close(out, 4 * size.double(), 3 * 4 * U * size.abs().double())


def test_a_call_with_one_tensor_twice_and_then_with_two():
    """A call that gives the same tensor twice says nothing about the next call of its sizes."""
    g = _gen(41)
    a, b = _operand(g, 192, 1152), _operand(g, 192, 1152)
    turns = [(a, a), (a, b), (b, a), (b, b), (a, (b[0], a[1])), (a, b), ((b[0], a[1]), a)]
    for lhs, rhs in turns:
        out, grouped = torch.zeros(192, 192, device='cuda'), torch.zeros(2, 192, 192, device='cuda')
        yan.gemm_fp8_fp8_fp32_nt(lhs, rhs, out)
        _check_product(out, _decode(lhs), _decode(rhs), None)
        yan.k_grouped_gemm_fp8_fp8_fp32_nt_contiguous(lhs, rhs, grouped, torch.tensor([0, 256, 1152], dtype=torch.int32, device='cuda'))
        for q, (lo, hi) in enumerate([(0, 256), (256, 1152)]):
            _check_product(grouped[q], _decode(lhs)[:, lo:hi].contiguous(), _decode(rhs)[:, lo:hi].contiguous(), None)
    y, d = [torch.randn(48, 136, generator=g, device='cuda').bfloat16() for _ in range(2)]
    rows = torch.arange(48, dtype=torch.int32, device='cuda')[:, None].contiguous()
    w = torch.randn(48, 1, generator=g, device='cuda')
    for grad_out, of in ((y, y), (d, y), (y, d), (d, d)):
        grad_y, grad_w = yan.moe_combine_backward(grad_out, of, rows, w, rows[:, 0].contiguous())
        _close(grad_y, w.double() * grad_out.double(), (2.0 ** -8 + 2 * U) * (w.double() * grad_out.double()).abs(), 'grad_y')
        size = (grad_out.double() * of.double()).abs().sum(1, keepdim=True)
        _close(grad_w, (grad_out.double() * of.double()).sum(1, keepdim=True), (136 / 64 + 16) * U * size, 'grad_weights')
    logits, dw = torch.randn(40, 6, generator=g, device='cuda'), torch.randn(40, 6, generator=g, device='cuda')
    _, indices, counts, _ = yan.moe_route(logits, 6)
    apart = yan.moe_route_backward(logits, indices, counts, logits.clone(), None)
    assert torch.equal(yan.moe_route_backward(logits, indices, counts, logits, None), apart)
    leaf = logits.double().requires_grad_()
    (torch.softmax(leaf, 1).gather(1, indices.long()) * dw.double()).sum().backward()
    # the terms are products of a score and a gradient of up to 5, each off by 60 u at most, of which there are 7 in a sum
    _close(yan.moe_route_backward(logits, indices, counts, dw, None), leaf.grad, torch.full_like(leaf, 7 * 5 * 60 * U).detach(), 'grad_logits')
