"""Sigmoid scores below the smallest normal number (logits of about -87.34 down to -88.72): the weights keep their ratios."""
import pytest
import torch

from mooncake_amd import route
from tests import operators_ref as ref
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu


def logits(T, E):
    """From -88.7 (a score of 2^-127.97) up to -86.7, 1/64 apart or more for up to 128 of them, in another order per token."""
    gen = torch.Generator().manual_seed(E)
    step = 2.0 / max(E, 8)
    return torch.stack([torch.randperm(E, generator=gen) for _ in range(T)]).float() * step - 88.7


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("E,K", [(8, 8), (5, 3), (16, 16), (64, 6), (100, 16)])
def test_weights_of_small_scores(gpu_device, E, K, bias):
    announce(f"route small scores E {E} K {K} bias {bias}")
    x = logits(9, E)
    b = None
    if bias:        # (the scores vanish beside it: it alone decides)
        b = (torch.randperm(E, generator=torch.Generator().manual_seed(K)).float() * 0.01).to(gpu_device)
    for renormalize in (False, True):
        idx, weights = route(x.to(gpu_device), K, score="sigmoid", renormalize=renormalize, bias=b)
        want_idx, want, _ = ref.route(x, K, score="sigmoid", renormalize=renormalize, bias=b)
        assert torch.equal(idx.cpu(), want_idx)
        # an exponential within 2 ulp, an addition and a quotient: 2^-21 of a score, and half of the smallest subnormal.  Divided
        # by their sum twice that and three roundings, with half of 2^-149 no more than 2^-22 of the smallest score
        allowed = want * 2.0 ** -19 if renormalize else want * 2.0 ** -21 + 2.0 ** -150
        assert bool(((weights.cpu().double() - want).abs() <= allowed).all())


@pytest.mark.parametrize("E", [8, 16])
def test_scores_that_are_zero_in_32_bits(gpu_device, E):
    announce(f"route scores that are zero E {E}")
    x = torch.full((3, E), -89.0)
    x[1, 2] = -88.0
    x[2, 1] = float("-inf")
    idx, weights = route(x.to(gpu_device), 2, score="sigmoid")
    assert idx.tolist() == [[0, 1], [2, 0], [0, 2]]
    assert weights.tolist() == [[0, 0], [1, 0], [0, 0]]
