"""The scan's results value by value: sums of few terms show what formed values are rounded
to on the way."""

import pytest
import torch

from tests import _ssm as T
from tests import _ssm_values as V

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L,H,P,G,N", [(64, 1, 4, 32, 1, 16), (40, 2, 4, 64, 2, 16), (16, 16, 4, 64, 1, 32),
                                         (4, 100, 6, 32, 2, 64), (2, 260, 5, 64, 5, 128), (3, 90, 12, 64, 1, 64)])
def test_scan_values(lib, dt, B, L, H, P, G, N):
    d = T.dev(T.scan_inputs(B, L, H, P, G, N, dt, seed=60 + B + L))
    V.scan_each(d, T.scan_run(d))


@pytest.mark.parametrize("t", [0, 5, 31, 40, 70])
def test_largest_fp32_value(lib, t):
    """Above 3.39e38 an fp32 value rounds to infinity in bf16 and counts as not finite: it reaches
    the outputs of its feature from its token on, and no other.  Below, it is a value."""
    d = T.scan_inputs(2, 90, 2, 32, 1, 16, torch.float32, seed=75)
    want = T.scan_run(T.dev(d), grads=False)["y"]
    d["x"] = d["x"].clone()
    d["x"][1, t, 1, 9] = torch.finfo(torch.float32).max
    got = T.scan_run(T.dev(d), grads=False)["y"]
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[1, t:, 1, 9] = True
    assert torch.equal(got[~hit], want[~hit])
    d["x"][1, t, 1, 9] = 1e37
    assert torch.isfinite(T.scan_run(T.dev(d), grads=False)["y"]).all()
