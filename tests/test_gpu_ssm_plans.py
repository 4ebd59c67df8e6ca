"""The scan against float64 in every way that its work is cut up: one segment of many chunks,
a few segments that the workgroups join, many that are joined beforehand, and in the backward
several heads to a workgroup, shared out evenly or not.  Each case asserts, by the library's
own sizes, that it is cut up so."""

import pytest
import torch

from tests import _ssm as T
from tests import _ssm_values as V

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODE = {F32: 0, BF16: 1, F16: 2}


def _up(n):
    return -(-n // 256) * 256


def plan(lib, dt, B, L, H, P, G, N):
    """(chunks, segments forwards, segments back, workgroups that share a group's heads)"""
    NP = 32 if N <= 32 else 64 if N <= 64 else 128
    Q = 32 if dt == F32 or (dt == F16 and NP == 128) else 64
    NC, chains = -(-L // Q), B * H

    def ends(S):  # the end states of the segments and their decays
        return chains * S * P * NP * 4 + _up(chains * S * 4) if S > 1 else 0

    fwd = lib.ttt_scan_workspace_bytes(B, L, H, P, N, CODE[dt])
    (S,) = [s for s in range(1, NC + 1) if ends(s) == fwd]
    states = lib.ttt_scan_states_bytes(B, L, H, P, N, CODE[dt])
    assert states == chains * NC * P * NP * 4
    back = lib.ttt_scan_bwd_workspace_bytes(B, L, H, P, G, N, CODE[dt]) - _up(states) - _up(3 * chains * NC * 4)
    ((Sb, shares),) = [(s, k) for s in range(1, NC + 1) for k in range(1, H // G + 1)
                       if ends(s) + (2 * k * B * L * G * N * 4 if k > 1 else 0) == back]
    return NC, S, Sb, shares


def check(lib, dt, shape, seed):
    d = T.dev(T.scan_inputs(*shape, dt, seed=seed))
    V.scan_each(d, T.scan_run(d))


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,H,P,N", [(104, 5, 64, 64), (104, 5, 64, 128), (104, 5, 64, 16), (206, 5, 32, 64),
                                     (154, 5, 32, 32), (206, 5, 32, 112)])
def test_one_segment(lib, dt, B, H, P, N):
    """The state stays in registers over five chunks (in fp32 nine), the last one ragged; the
    backward's workgroups have all five heads."""
    shape = (B, 273, H, P, 1, N)
    NC, S, Sb, shares = plan(lib, dt, *shape)
    assert NC >= 5 and S == Sb == 1 and shares == 1
    check(lib, dt, shape, 70)


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,H,P,G,N", [(16, 12, 64, 1, 64), (16, 12, 64, 1, 128), (16, 12, 64, 2, 32), (16, 20, 32, 1, 64),
                                       (16, 20, 32, 2, 16), (16, 20, 32, 1, 128)])
def test_segments_that_workgroups_join(lib, dt, B, H, P, G, N):
    """A few segments of several chunks each, the last one shorter or ragged."""
    shape = (B, 850, H, P, G, N)
    NC, S, Sb, shares = plan(lib, dt, *shape)
    assert 2 <= S <= 8 and 2 <= Sb <= 8 and NC > 2 * max(S, Sb) and -(-H // G // shares) >= 3
    check(lib, dt, shape, 71)


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,H,P,N", [(9, 5, 64, 64), (9, 5, 64, 128), (9, 5, 64, 32), (9, 5, 32, 64), (9, 5, 32, 32)])
def test_segments_joined_beforehand(lib, dt, B, H, P, N):
    """More segments than a workgroup joins, of two chunks and more; the heads are shared
    out unevenly, three and two."""
    shape = (B, 2291, H, P, 1, N)
    NC, S, Sb, shares = plan(lib, dt, *shape)
    assert S > 8 and Sb > 8 and NC >= 2 * max(S, Sb) - 1 and shares <= 2
    check(lib, dt, shape, 72)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_uneven_shares_of_heads(lib, dt):
    """Seven heads of a group by fours and threes, three groups."""
    shape = (10, 1000 if dt != F32 else 500, 21, 64, 3, 48)
    NC, S, Sb, shares = plan(lib, dt, *shape)
    assert shares == 2
    check(lib, dt, shape, 73)
