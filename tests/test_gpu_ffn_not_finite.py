"""The gated feed-forward projections on the GPU where a row of x, or of the weights, has a value
that is not finite: it reaches the results that are formed of it and no other."""

import math

import pytest
import torch

from tests import _block as T
from tests.test_gpu_ffn import inputs, run

pytestmark = pytest.mark.gpu

# (an fp32 value above 3.39e38 counts as one: its first bf16 plane is infinite)
BAD = [(dt, v) for dt in T.DTYPES for v in (math.nan, math.inf, -math.inf)] + [(torch.float32, 3.4e38)]


@pytest.mark.parametrize("dt,bad", BAD)
@pytest.mark.parametrize("R", [9, 90, 700])
def test_a_row_of_x(lib, R, dt, bad):
    """Its results are not finite, in fp32 NaN, whichever way the work is cut up; the other rows' results
    and gradients have the same bits as without it, and so have the biases' but for what it adds."""
    d = T.dev(inputs(R, 100, 60, dt, seed=5))
    ref = run(d)
    e = {**d, "x": d["x"].clone()}
    e["x"][4, 99] = bad
    got = run(e)
    keep = [i for i in range(R) if i != 4]
    for k in ("y", "dx"):
        assert torch.equal(got[k][keep], ref[k][keep]), k
    assert not torch.isfinite(got["y"][4].float()).any()
    if dt == torch.float32:
        assert torch.isnan(got["y"][4]).all()
    for k in ("dw_gate", "dw_up", "db_gate", "db_up"):
        assert not torch.isfinite(got[k].float()).any(), k


@pytest.mark.parametrize("dt,bad", BAD)
@pytest.mark.parametrize("R", [9, 90])
@pytest.mark.parametrize("which", ["w_gate", "w_up"])
def test_a_row_of_the_weights(lib, R, dt, bad, which):
    """It reaches its own column of y, and its own row of the weights' gradients."""
    d = T.dev(inputs(R, 100, 60, dt, seed=6))
    ref = run(d)
    e = {**d, which: d[which].clone()}
    e[which][7, 3] = bad
    got = run(e)
    keep = [i for i in range(60) if i != 7]
    assert torch.equal(got["y"][:, keep], ref["y"][:, keep]) and not torch.isfinite(got["y"][:, 7].float()).any()
    for k in ("dw_gate", "dw_up", "db_gate", "db_up"):
        assert torch.equal(got[k][keep], ref[k][keep]), k
    assert not torch.isfinite(got["dx"].float()).any()
