"""The whole-world driver around the router and the experts: which stream their outputs are allocated for.  (No GPU: streams
are names, and the operators write down what they are given.)"""
import contextlib

import pytest
import torch

from mooncake_amd import harness as module
from mooncake_amd.harness import WorldHarness
from mooncake_amd.workloads import EPConfig

R, T, H, E, K, I = 3, 4, 128, 6, 2, 128


class Recorder:
    """Stands in for the allocator, the streams and the operators."""

    def __init__(self, monkeypatch):
        self.current, self.allocated_on, self.used_on, self.calls = "caller", {}, {}, []
        self.kept = []              # (so that no address comes twice)
        empty = torch.empty

        def counted_empty(*args, **kwargs):
            t = empty(*args, **kwargs)
            self.kept.append(t)
            self.allocated_on[t.data_ptr()] = self.current
            return t

        @contextlib.contextmanager
        def on(stream):
            before, self.current = self.current, stream if stream is not None else self.current
            yield
            self.current = before

        monkeypatch.setattr(torch, "empty", counted_empty)
        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.current)
        monkeypatch.setattr(torch.Tensor, "record_stream",
                            lambda t, stream: self.used_on.setdefault(t.data_ptr(), set()).add(stream))
        monkeypatch.setattr(module.operators, "route", self.route)
        monkeypatch.setattr(module.operators, "expert_mlp", self.expert_mlp)

    def route(self, logits, num_topk, out, **kwargs):
        self.calls.append(("route", self.current, out))
        for t in out:
            t.fill_(7)

    def expert_mlp(self, x, count, w_gate_up, w_down, out):
        self.calls.append(("experts", self.current, x, count, w_gate_up, w_down, out))


class World:
    num_ranks = R


def make(fp8=False):
    h = WorldHarness(EPConfig("operators", R, T, H, E, K, fp8), device="cpu", world=World())
    h.alloc_dispatch_outputs()
    return h


@pytest.mark.parametrize("stream", [None, "side"])
def test_routing_is_allocated_for_the_stream_that_writes_it(monkeypatch, stream):
    seen = Recorder(monkeypatch)
    h = make()
    h.route(torch.zeros(R, T, E), stream=stream)
    for t in (h.topk_idx, h.topk_weights):
        assert seen.allocated_on[t.data_ptr()] == (stream or "caller")
        # and its memory goes to nobody else while either stream may still use it
        assert stream is None or seen.used_on[t.data_ptr()] == {"caller", "side"}
    assert seen.calls[0][1] == (stream or "caller")


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("stream", [None, "side"])
def test_expert_rows_are_allocated_for_the_stream_that_writes_them(monkeypatch, stream, fp8):
    seen = Recorder(monkeypatch)
    h = make(fp8)
    h.experts(torch.zeros(E, 2 * I, H), torch.zeros(E, H, I), stream=stream)
    for t in (h.expert_out, h.combined):
        assert seen.allocated_on[t.data_ptr()] == (stream or "caller")
        assert stream is None or seen.used_on[t.data_ptr()] == {"caller", "side"}
    for t in (h.recv_x, h.recv_count) + ((h.recv_scales_phys,) if fp8 else ()):
        assert stream is None or "side" in seen.used_on[t.data_ptr()]
    assert seen.calls[0][1] == (stream or "caller")


def test_what_was_loaded_is_not_written_over(monkeypatch):
    Recorder(monkeypatch)
    h = make()
    data = {"x": torch.zeros(R, T, H, dtype=torch.bfloat16), "topk_idx": torch.full((R, T, K), 5),
            "topk_weights": torch.full((R, T, K), 0.5)}
    h.load(data)
    h.route(torch.zeros(R, T, E))
    assert bool((data["topk_idx"] == 5).all()) and bool((data["topk_weights"] == 0.5).all())
    assert bool((h.topk_idx == 7).all()) and bool((h.topk_weights == 7).all())
    # the next step's choices come to the same place, which a recorded dispatch reads; loaded ones come back by loading
    at = h.topk_idx.data_ptr(), h.topk_weights.data_ptr()
    h.route(torch.zeros(R, T, E))
    assert at == (h.topk_idx.data_ptr(), h.topk_weights.data_ptr())
    h.load(data)
    assert bool((h.topk_idx == 5).all())
    h.route(torch.zeros(R, T, E))
    assert bool((data["topk_idx"] == 5).all()) and at == (h.topk_idx.data_ptr(), h.topk_weights.data_ptr())


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("present,runs", [(None, [(0, 3)]), ((1, 1, 1), [(0, 3)]), ((1, 0, 1), [(0, 1), (2, 3)]),
                                          ((0, 1, 1), [(1, 3)]), ((0, 0, 0), [])])
def test_experts_of_silent_ranks_are_left_out(monkeypatch, present, runs, fp8):
    seen = Recorder(monkeypatch)
    h = make(fp8)
    w_gate_up, w_down = torch.zeros(E, 2 * I, H), torch.zeros(E, H, I)
    if fp8:
        w_gate_up, w_down = (w_gate_up, torch.zeros(E, 2 * I // 128, H // 128)), (w_down, torch.zeros(E, H // 128, I // 128))
    h.experts(w_gate_up, w_down, **({} if present is None else {"present": present}))
    L = E // R
    assert len(seen.calls) == len(runs)
    for (first, last), (_, _, x, count, w1, w2, out) in zip(runs, seen.calls):
        x, w1, w2 = (v if fp8 else (v,) for v in (x, w1, w2))
        for got, of in ([(x[0], h.recv_x.view(E, R * T, H)), (count, h.recv_count.view(E)), (out, h.expert_out.view(E, R * T, H))]
                        + list(zip(w1, w_gate_up if fp8 else (w_gate_up,))) + list(zip(w2, w_down if fp8 else (w_down,)))
                        + ([(x[1], h.recv_scales_phys.view(E, -1, R * T).transpose(1, 2))] if fp8 else [])):
            part = of[first * L:last * L]
            assert got.shape == part.shape and got.data_ptr() == part.data_ptr() and got.stride() == part.stride()
