"""Which tiles the experts' products are cut into (the library's choice, asked for on the host), and that the cases of
test_gpu_expert_tiles.py run all of them."""
import pytest

from tests import expert_tiles as tiles


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("product", [0, 1], ids=["gate_up", "down"])
def test_the_cases_run_every_tile_shape(product, fp8):
    assert tiles.covered(tiles.CASES, fp8, product) == tiles.every_shape(fp8, product == 0)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_blocks_go_on_with_other_shapes_too(fp8):
    for product in (0, 1):
        assert max(c.products()[product].switches for c in tiles.CASES if c.fp8 == fp8) > 20


def test_no_rows_and_counts_out_of_range():
    assert tiles.products([0, 0, -4], 8, 256, 256, True)[0].runs == {}
    assert tiles.products([1 << 30, -5, 20], 20, 256, 256, True) == tiles.products([20, 0, 20], 20, 256, 256, True)


@pytest.mark.parametrize("gate_up", [False, True])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_prices_of_very_many_tiles(fp8, gate_up):
    """Experts of as many rows as the entry points take: the prices' sums pass 32 bits, the plan stays the one that fewer
    rows of the kind get."""
    want = tiles.plan([1 << 15] * 4, 1 << 24, 128, 256, fp8, gate_up, 256)[:2]
    for L in range(1, 64):
        assert tiles.plan([1 << 24] * L, 1 << 24, 128, 256, fp8, gate_up, 256)[:2] == want, L
