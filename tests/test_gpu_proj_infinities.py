"""drb_proj_q8_lora where an infinity has one sign all the way: the outputs are that infinity, by every form of the call, and no other row sees it.

The first half's f16 rows and the second half's v meet the adapters in several bf16 terms; what an infinity leaves for the second term is nothing, not a NaN."""

import pytest
import torch

from tests.test_gpu_proj_lora import make, run

pytestmark = pytest.mark.gpu
AT = 17  # the input that is large
# the mma.sync form with one to four column tiles and several passes, and the tcgen05 form with one tile of rows and with three
FORMS = [(3, 300), (12, 300), (20, 300), (40, 300), (70, 300), (33, 9000), (70, 9000), (170, 9000)]


def case(rows, n, x_type):
    """All adapters' B and all their weights for input AT are positive."""
    t = make(rows + n, rows, n, 512, 3, 16, x_type, who=[r % 4 - 1 for r in range(rows)])
    t["b"] = t["b"].abs().clamp_min(0.01)
    t["a"][:, :, AT] = 0.5
    t["q"][:, AT] = 3
    t["x"][:, AT] = 0
    return t


@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("rows,n", FORMS)
def test_an_infinite_input(rows, n, x_type):
    t = case(rows, n, x_type)
    y = run(t)
    t["x"][1, AT] = float("inf")  # a row with an adapter
    if rows > 4:
        t["x"][4, AT] = float("-inf")  # and one without
    z = run(t)
    assert (z[1] == float("inf")).all()
    assert rows <= 4 or (z[4] == float("-inf")).all()
    others = [r for r in range(rows) if r not in (1, 4)]
    assert torch.equal(z[others], y[others])


@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("rows,n", FORMS)
def test_a_first_half_that_overflows(rows, n, x_type):
    t = case(rows, n, x_type)
    y = run(t)
    t["q"][:, AT] = 0
    t["a"][:, :, AT] = 1e38
    t["x"][1, AT] = 1e4
    z = run(t)
    assert (z[1] == float("inf")).all()
    others = [r for r in range(rows) if r != 1]
    assert torch.equal(z[others], y[others])


@pytest.mark.parametrize("bad", [float("-inf"), float("nan")])
@pytest.mark.parametrize("x_type", [1, 2])
@pytest.mark.parametrize("rows,n", FORMS)
def test_a_negative_infinity_and_a_nan(rows, n, x_type, bad):
    t = case(rows, n, x_type)
    t["b"][:, :, 0] = 500  # beside the largest rest that a second term may be: finite
    y = run(t)
    t["x"][1, AT] = bad
    z = run(t)
    assert torch.isnan(z[1]).all() if bad != bad else (z[1] == bad).all()
    others = [r for r in range(rows) if r != 1]
    assert torch.equal(z[others], y[others])
