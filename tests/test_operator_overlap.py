"""The experts' products are refused where they would write over what they read (before anything is enqueued, so without a
GPU): other blocks of the same kernel may still need it."""
import pytest

from tests.test_operator_refusals import P, down, gate_up, refused

L, ROWS, H = 2, 8, 256


@pytest.mark.parametrize("fp8", [0, 1])
def test_input_and_output_lie_apart(fp8):
    size = 1 if fp8 else 2
    far = {"w": P << 8, "ws": P << 9, "xs": P << 10, "act_s": P << 11, "count": P << 12, "fp8": fp8}
    x = L * ROWS * H * size
    act = L * ROWS * 128 * size
    for at in (P, P + x - 16, P - act + 16):
        refused(gate_up(x=P, act=at, H=H, I=128, **far), "apart")
    del far["xs"]
    act, out = L * ROWS * H * size, L * ROWS * H * 2        # (as wide as the rows: in place would fit)
    for at in (P, P + act - 16, P - out + 16):
        refused(down(act=P, out=at, H=H, I=H, **far), "apart")


def test_scales_lie_apart():
    refused(gate_up(x=P, act=P << 8, xs=P << 9, act_s=P << 9, H=H, I=H), "apart")
