"""States of the scan that begin off 16 bytes, on the GPU: the same bits as from whole ones."""

import pytest
import torch

from tests import _ssm as T

pytestmark = pytest.mark.gpu


def test_states_off_16_bytes(lib):
    """An initial state, and a gradient of the last one, that begin in the middle of 16 bytes."""
    d = T.dev(T.scan_inputs(2, 70, 3, 32, 1, 16, torch.bfloat16, seed=54))
    want = T.scan_run(d)
    for by in (1, 2, 3):
        q = dict(d)
        for k in ("state", "dlast"):
            q[k] = torch.empty(d[k].numel() + 4, device="cuda")[by:by + d[k].numel()].view(d[k].shape).copy_(d[k])
            assert q[k].data_ptr() % 16 == 4 * by
        got = T.scan_run(q)
        for k in want:
            assert torch.equal(got[k], want[k]), (by, k)
