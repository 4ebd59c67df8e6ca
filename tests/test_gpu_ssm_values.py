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
