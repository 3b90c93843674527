"""GPU tier: values at which the token-wise operators' arithmetic can lose what the formulas keep, against float64.

Tolerances count roundings as in test_gpu_token_ops.py, whose oracles are used: u = 2^-24 is half a step of f32, h(T) half a step
of the storage type."""
import math

import pytest
import torch

from test_gpu_token_ops import lp_check

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs an MI355X")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------------------------------------- log probabilities far from zero
# rows in a wave's registers (a part of a wave, a wave), a wave per long row, a block per row, split rows
FAR_SHAPES = [(1, 40), (1, 2048), (130, 2500), (1, 5003), (1, 70001)]


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("repeat,v", FAR_SHAPES)
def test_token_logprobs_rows_and_parts_far_from_zero(repeat, v, dt):
    """Finite mask fills and logits of any size: a row's exponents are of the distance to its maximum, wherever that lies.  Rows
    all at the fill, halves and stripes of it (a thread's first accesses may be nothing else), distances of a few steps there."""
    g = gen(v)
    fills = (-1e9, -1e10, -1e12, -1e20, -1e30, 1e10, 1e30, 2.0 ** 20, -2.0 ** 20, 2.0 ** 20 + 64)
    rows = []
    for f in fills:
        n = lambda: torch.randn(v, device="cuda", generator=g)      # noqa: E731
        x = [torch.full((v,), f, device="cuda"), n(), n(), n(), n(), f + torch.randint(-3, 4, (v,), device="cuda", generator=g)]
        x[1][: v // 2] = f
        x[2][v // 2:] = f
        x[3][::2] = f
        x[4][:] = -math.inf
        x[4][: v // 3] = f
        x[4][v - 1] = 1.0
        rows += x
    # the sums of one row about maxima on both sides of where the exponents' form changes
    border = torch.full((v,), 2.0 ** 20 - 6, device="cuda")
    border[v // 2:] += torch.randint(0, 12, (v - v // 2,), device="cuda", generator=g)
    rows += [border, border.flip(0), -border]
    x = torch.stack(rows).to(dt).repeat(repeat if repeat == 1 else repeat // 2, 1)
    if repeat > 1:
        assert x.shape[0] >= 2048
    t = torch.randint(0, v, (x.shape[0],), device="cuda", generator=g)
    lp_check(x, t, top=min(v, 5))


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("v", [3, 2500, 70001])
def test_token_logprobs_distances_near_the_end_of_the_range(v, dt):
    """ln p = x - m - ln s is finite wherever x - m is, although (x - m) log2 e is not."""
    x = torch.full((4, v), -math.inf, device="cuda")
    x[0, :3] = torch.tensor([3e38, 0.0, 1e38])
    x[1, :3] = torch.tensor([1.9e38, -1e38, 1.9e38])
    x[2, :3] = torch.tensor([0.0, -3e38, -2.5e38])
    x[3, :3] = torch.tensor([1.5e38, -1.5e38, 7.0])
    x = x.to(dt)
    lp_check(x, torch.ones(4, dtype=torch.int64, device="cuda"), top=3)
    lp_check(x, torch.full((4,), 2, device="cuda"), top=3)
