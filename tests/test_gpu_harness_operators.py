"""The whole-world driver's route and experts with outputs that do not exist yet, on another stream, over loaded routing, and
with a silent rank."""
import pytest
import torch

from mooncake_amd.benchmarks import moe_layer
from tests.gpu_util import announce
from tests.test_gpu_moe_layer import config

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])


@BOTH
def test_a_first_step_on_another_stream(gpu_device, fp8):
    announce(f"harness: first step on another stream fp8={fp8}")
    layer = moe_layer.MoELayer(config(fp8), 256, seed=3)
    h = layer.harness
    h.expert_out = h.combined = None
    layer.gate()
    logits = layer.logits.view(h.cfg.num_ranks, h.cfg.tokens_per_rank, -1)
    loaded = h.topk_idx, h.topk_weights
    before = [t.clone() for t in loaded]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h.route(logits, stream=side)
    h.dispatch(stream=side)
    h.experts(layer.w_gate_up, layer.w_down, stream=side)
    h.combine(stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(loaded, before))
    assert h.topk_idx is not loaded[0] and h.topk_weights is not loaded[1]
    other = moe_layer.MoELayer(config(fp8), 256, seed=3)
    want = other()
    torch.cuda.synchronize()
    assert torch.equal(h.topk_idx, other.harness.topk_idx) and torch.equal(h.combined, want)


@BOTH
def test_a_silent_rank(gpu_device, fp8):
    announce(f"harness: a silent rank fp8={fp8}")
    layer = moe_layer.MoELayer(config(fp8), 256, seed=4)
    h, R = layer.harness, layer.harness.cfg.num_ranks
    present = [1, 0, 1, 1]
    layer.gate()
    layer.route()
    h.recv_count.fill_(1 << 20)             # (as memory may be: the silent rank's stay so)
    h.expert_out.fill_(-7.0)
    h.dispatch(present=present)
    h.experts(layer.w_gate_up, layer.w_down, present=present)
    torch.cuda.synchronize()
    got = h.expert_out.clone()
    assert bool((got[1] == -7.0).all()) and bool((h.recv_count[1] == 1 << 20).all())
    h.recv_count[1] = 0
    h.expert_out.fill_(-7.0)
    h.experts(layer.w_gate_up, layer.w_down)
    torch.cuda.synchronize()
    assert all(int(h.recv_count[r].sum()) > 0 for r in range(R) if present[r])
    assert torch.equal(got.view(torch.int16), h.expert_out.view(torch.int16))
