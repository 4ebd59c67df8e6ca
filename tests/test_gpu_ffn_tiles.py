"""The gated feed-forward projections' large tiles, and whole rounds of them with small ones behind,
for either activation, and from planes where 16-bit rows are not whole pieces of 16 bytes."""

import pytest
import torch

from tests import _block as T
from tests.test_gpu_ffn import BF16, F16, check, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R,D,F,bias", [(6200, 24, 1030, True), (4099, 400, 2100, False), (4099, 4200, 200, True)])
def test_activations(lib, dt, R, D, F, bias, act):
    d = inputs(R, D, F, dt, bias=bias, seed=R + D + 1)
    check(d, run(T.dev(d), act), act)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("R,D,F,bias", [(6200, 21, 1030, True), (4099, 397, 2100, False), (4099, 4197, 203, True)])
def test_rows_from_planes(lib, dt, R, D, F, bias, act):
    """D that is no multiple of 8: the rows are padded in the workspace."""
    d = inputs(R, D, F, dt, bias=bias, seed=R + D + 2)
    check(d, run(T.dev(d), act), act)
