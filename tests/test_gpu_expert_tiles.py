"""The experts' products through every tile shape of the kernels, with blocks that go from tile to tile (expert_tiles.CASES),
and on inputs whose sums are exact in 32 bits, where a single product that is missing or counted twice shows."""
import pytest
import torch

from mooncake_amd import expert_down, expert_gate_up
from tests import expert_tiles as tiles
from tests import operators_ref as ref
from tests.gpu_util import announce
from tests.test_gpu_experts import POISON, column_major, empty_act, poison, run_and_check, untouched, wide

pytestmark = pytest.mark.gpu

EACH = pytest.mark.parametrize("case", tiles.CASES, ids=lambda c: c.name)


def cus(device):
    return torch.cuda.get_device_properties(device).multi_processor_count


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("product", [0, 1], ids=["gate_up", "down"])
def test_the_cases_run_every_tile_shape_here(gpu_device, product, fp8):
    assert tiles.covered(tiles.CASES, fp8, product, cus(gpu_device)) == tiles.every_shape(fp8, product == 0)


@EACH
def test_tiles(gpu_device, case):
    announce(f"expert tiles {case.name}: " + ", ".join(str(p.plan) for p in case.products(cus(gpu_device))))
    run_and_check(case.experts, case.rows, case.hidden, case.intermediate, case.counts, case.fp8, seed=case.experts)


def whole(shape, gen, device):
    """Values -1, 0 and 1, different in every row."""
    return torch.randint(-1, 2, shape, generator=gen, device=device, dtype=torch.int8)


def operands(shape, fp8, unit, block, gen, device):
    """[L, rows, columns] values times scales that are unit or unit / 2 (fp8: of each 128, or of blocks), exact in any order of
    summation: products are multiples of one unit and fewer than 2^22 of them add up."""
    values = whole(shape, gen, device)
    L, rows, columns = shape
    if not fp8:
        return (values * unit).to(torch.bfloat16)
    scales = torch.randint(1, 3, (L, rows // 128 if block else rows, columns // 128), generator=gen, device=device) * (unit / 2)
    return values.to(ref.FP8), scales.float()


@EACH
def test_every_product_counts(gpu_device, case):
    announce(f"expert tiles exactly {case.name}")
    fp8, L, RM, H, I = case.fp8, case.experts, case.rows, case.hidden, case.intermediate
    gen = torch.Generator(device=gpu_device).manual_seed(case.hidden)
    count = torch.tensor(case.counts, dtype=torch.int32, device=gpu_device)
    # gate and up of about 1: 4/9 of H products of one unit squared
    unit = 2.0 ** -round(torch.tensor(H * 4 / 9).log2().item() / 4)

    x = operands((L, RM, H), fp8, unit, False, gen, gpu_device)
    x = (poison(x[0], count), column_major(poison(x[1], count))) if fp8 else poison(x, count)
    w1 = operands((L, 2 * I, H), fp8, unit, True, gen, gpu_device)
    act = empty_act(L, RM, I, fp8, gpu_device)
    expert_gate_up(x, count, w1, act=act)

    a = operands((L, RM, I), fp8, 1.0, False, gen, gpu_device)
    a = (poison(a[0], count), column_major(poison(a[1], count))) if fp8 else poison(a, count)
    w2 = operands((L, H, I), fp8, 1.0, True, gen, gpu_device)
    out = expert_down(a, count, w2, out=torch.full((L, RM, H), POISON, dtype=torch.bfloat16, device=gpu_device))
    torch.cuda.synchronize()
    for e, n in enumerate(case.counts):
        # the sums are exact: rounded once, they are the output bit for bit
        assert torch.equal(out[e, :n], (wide(a, e, n) @ wide(w2, e, block=True).T).to(torch.bfloat16)), f"expert {e}: down"
        g, u = (wide(x, e, n) @ wide(w1, e, block=True).T).split(I, 1)
        want = g * torch.sigmoid(g) * u
        # the exponential's argument is rounded (|g| 2^-24), its value, the quotient and the products are a few roundings
        off = want.abs() * (g.abs() + 8) * 2.0 ** -23
        if not fp8:
            low, high = (want - off).to(torch.bfloat16), (want + off).to(torch.bfloat16)        # (rounding keeps the order)
            assert bool(((low <= act[e, :n]) & (act[e, :n] <= high)).all()), f"expert {e}"
            continue
        s = act[1][e, :n].double()
        top = want.unflatten(1, (-1, 128)).abs().amax(2)
        room = off.unflatten(1, (-1, 128)).amax(2) / 448
        assert bool(((s - top.clamp(min=1e-4) / 448).abs() <= room + s * 2.0 ** -22).all()), f"expert {e}: scales"
        # half a step of the fp8 value (2^-4 of it, or 2^-10 below the smallest normal), of a quotient that is roundings away
        s = s.repeat_interleave(128, 1)
        step = torch.maximum(want.abs() * 2.0 ** -4, 2.0 ** -10 * s) * (1 + 2.0 ** -10)
        assert bool(((act[0][e, :n].double() * s - want).abs() <= step + off + want.abs() * 2.0 ** -20).all()), f"expert {e}"
    assert untouched(out, count) and all(untouched(t, count) for t in (act if fp8 else (act,)))
