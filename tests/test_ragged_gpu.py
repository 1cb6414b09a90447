"""The ragged layout and the 16-bit products on it, on the GPU: each against its definition in 64 bits, and all of them in a row."""
import pytest
import torch

import harness as testing
import yan_amd as yan

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
