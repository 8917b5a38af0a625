"""The router on bf16 logits of more experts than have distinct values, and on more tokens than a 16-bit number of blocks."""
import pytest
import torch

from mooncake_amd import route
from tests.gpu_util import announce
from tests.test_gpu_route import TOLERANCE, compare

pytestmark = pytest.mark.gpu


def some_equal(T, E, seed):
    """Logits in steps of 1/32 within +-2, exact in bf16, equal ones among them, one large group of equals at the top of a token."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(-64, 65, (T, E), generator=gen).float() / 32
    x[0] = x[0].clamp(max=1.0)
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("K", [1, 4, 5, 6, 8, 16])
@pytest.mark.parametrize("E,groups", [(257, 1), (264, 1), (264, 8), (384, 1), (384, 8), (511, 1), (512, 1), (512, 8), (1000, 1),
                                      (1000, 8), (1024, 1), (1024, 8)])
def test_bf16(gpu_device, E, groups, K, score):
    announce(f"route bf16 E {E} K {K} {score} groups {groups}")
    x = some_equal(6, E, E + K).to(gpu_device)
    want = compare(x, K, margin=0, score=score, num_groups=groups, topk_groups=max(1, groups // 2))
    # rows that begin at an odd element, an even one, and aligned ones with a stride of their own
    for pad in (1, 2, 8):
        wide = torch.full((6, E + pad), float("nan"), dtype=torch.bfloat16, device=gpu_device)
        wide[:, pad:] = x
        got = route(wide[:, pad:], K, score=score, num_groups=groups, topk_groups=max(1, groups // 2))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("E,K", [(16, 3), (72, 2)])
def test_more_than_65535_blocks(gpu_device, E, K):
    """A wave per token, four tokens a block."""
    T = 300_001
    announce(f"route {T} tokens of {E}")
    x = torch.zeros(T, E, device=gpu_device)
    t = torch.arange(T, device=gpu_device)
    want = (t.unsqueeze(1) * 5 + torch.arange(K, device=gpu_device)) % E
    for k in range(K):
        x[t, want[:, k]] = 4.0 - k
    idx, w = route(x, K, renormalize=False)
    assert torch.equal(idx, want)
    top = torch.exp(4.0 - torch.arange(K, dtype=torch.float64, device=gpu_device))
    exact = top / (top.sum() + E - K)           # (where the experts lie decides the order of the sum)
    assert bool(((w.double() - exact).abs() <= TOLERANCE * exact).all())
