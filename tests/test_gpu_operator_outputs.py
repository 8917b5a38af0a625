"""The operators' outputs and the memory they stand in."""
import pytest
import torch

from mooncake_amd import route
from tests.gpu_util import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,K", [(1, 8), (5, 3), (64, 8)])
def test_router_outputs_grow_without_meeting(gpu_device, T, K):
    """Each has memory of its own: one that grows does not grow into the other, and one kept does not keep the other."""
    announce(f"route outputs that grow, {T} x {K}")
    logits = torch.randn((T, 24), device=gpu_device)
    idx, weights = route(logits, K)
    assert idx.untyped_storage().data_ptr() != weights.untyped_storage().data_ptr()
    assert idx.untyped_storage().nbytes() == T * K * 8 and weights.untyped_storage().nbytes() == T * K * 4
    want = weights.clone()
    for rows in (T + 1, T + 40, 2 * T):
        idx.resize_(rows, K)
        idx.fill_(-1)
        assert torch.equal(weights, want)
