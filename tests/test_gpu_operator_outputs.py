"""The operators' outputs and the memory they stand in."""
import pytest
import torch

from mooncake_amd import expert_gate_up, route
from tests.gpu_util import announce
from tests.test_gpu_experts import empty_act, make

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


def test_activations_come_with_their_scales_or_not_at_all(gpu_device):
    """The same from both bindings: fp8 values without scales are no place to write to, nor are scales for bf16."""
    announce("activations handed in without scales")
    for fp8 in (True, False):
        x, count, w1, _ = make(2, 8, 256, 128, [8, 3], fp8)
        values, scales = empty_act(2, 8, 128, True, gpu_device)
        bad = values if fp8 else (empty_act(2, 8, 128, False, gpu_device), scales)
        with pytest.raises(AssertionError):
            expert_gate_up(x, count, w1, act=bad)
