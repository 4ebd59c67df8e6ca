"""How a scan is cut into segments: by the workgroups of the walks that a compute unit holds,
forwards and backwards, as the built kernels' registers and LDS say (no GPU)."""

import pytest

from tests.test_kernel_resources import kernels  # noqa: F401

TYPES = {0: ("f", 3, 3), 1: ("DF16b", 1, 2), 2: ("DF16_", 2, 3)}  # mangled name, planes of an input, of a formed value
F32, BF16, F16 = 0, 1, 2


def _chunk(dtype, NP):
    return 32 if dtype == F32 or (dtype == F16 and NP == 128) else 64


def _lds(dtype, P, NP):
    """Bytes of a walk's workgroup: planes of x, keys and queries (16 bytes of padding to a row),
    the masked products by tiles of 64 lanes, two chunks' decays."""
    _, IN, MID = TYPES[dtype]
    Q = _chunk(dtype, NP)
    tb = Q // 16
    rows = 2 * IN * Q * ((P + 8) + 2 * (NP + 8))
    return rows + MID * tb * (tb + 1) // 2 * 64 * 8 + 2 * -(-(6 * Q + 2) * 4 // 16) * 16


def _segments(lib, dtype, P, NP, back):
    """Workgroups of one sequence and head of 256 x 60 chunks, 256 compute units: as many segments as
    are held at once."""
    Q = _chunk(dtype, NP)
    NC = 256 * 60
    L = NC * Q
    up = lambda n: -(-n // 256) * 256  # noqa: E731
    if not back:
        n = lib.ttt_scan_workspace_bytes(1, L, 1, P, NP, dtype)
    else:
        n = lib.ttt_scan_bwd_workspace_bytes(1, L, 1, P, 1, NP, dtype)
        n -= up(lib.ttt_scan_states_bytes(1, L, 1, P, NP, dtype)) + up(3 * NC * 4)
    (found,) = [s for s in range(2, NC + 1) if s * P * NP * 4 + up(4 * s) == n]
    return found


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("NP", [32, 64, 128])
@pytest.mark.parametrize("P", [32, 64])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_segments_fill_one_round(kernels, dtype, P, NP, back):  # noqa: F811
    from ttt_amd import _lib
    name = f"scan_walk_kernelI{TYPES[dtype][0]}Li{P}ELi{NP}ELNS0_4WalkE{int(back)}ELb1E"
    (k,) = [r for n, r in kernels if name in n]
    waves = min(8, 512 // (-(-k["vgpr_count"] // 8) * 8))  # of a SIMD
    held = min(4 * waves // (P // 16), 160 * 1024 // _lds(dtype, P, NP))
    assert _segments(_lib.load(), dtype, P, NP, back) == 256 * held
