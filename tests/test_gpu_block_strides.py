"""A gated delta-rule block's operators on the GPU on rows that are far apart, past the reach of 32-bit
offsets and of what is read in place: the same bits as from contiguous tensors."""

import pytest
import torch

from tests import _block as T
from tests import test_gpu_block_norm as N
from tests import test_gpu_ffn as FF

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("needs 64 GB of the GPU's memory")
    yield
    torch.cuda.empty_cache()


def far(t, lead, apart):
    """t with its first `lead` axes as rows `apart` bytes apart"""
    rows, flat = t.shape[:lead].numel(), t.flatten(lead) if t.dim() > lead else t.unsqueeze(-1)
    m = torch.empty(rows, apart // t.element_size(), device=t.device, dtype=t.dtype)[:, 8:8 + flat.shape[-1]]
    m.copy_(flat.reshape(rows, -1))
    return m.unflatten(1, t.shape[lead:]).unflatten(0, t.shape[:lead])


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("R", [9, 70])
def test_gated_linear(lib, dt, R):
    d = T.dev(FF.inputs(R, 48, 40, dt, seed=3))
    ref = FF.run(d)
    for apart in (1 << 22, (1 << 22) + 64, 1 << 27):
        for k, t in FF.run({**d, "x": far(d["x"], 1, apart), "dy": far(d["dy"], 1, apart)}).items():
            assert torch.equal(t, ref[k]), (apart, k)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_block_norm(lib, dt):
    d = T.dev(N.inputs((5, 7, 3, 64), dt, "wgsrn", F32, seed=3))
    ref = N.run(d)
    for lead in (2, 3):
        e = {k: far(t, lead, 1 << 27) if t is not None and k in ("x", "gate", "residual") else t for k, t in d.items()}
        for k, t in N.run(e).items():
            assert torch.equal(t, ref[k]), (lead, k)


@pytest.mark.parametrize("dt", T.DTYPES)
@pytest.mark.parametrize("B,L", [(1, 70), (2, 33), (40, 1)])
def test_gated_delta(lib, dt, B, L):
    from ttt_amd.delta import gated_delta_step
    d = T.dev(T.delta_inputs(B, L, 4, 2, 32, 64, dt, seed=7))
    ref = T.delta_run(d)
    for apart in (1 << 25, 1 << 26, 1 << 27):
        e = {k: far(t, 2, apart) if k in ("q", "k", "v", "g", "beta", "do") else t for k, t in d.items()}
        for k, t in T.delta_run(e).items():
            assert torch.equal(t, ref[k]), (apart, k)
        states = d["state"].clone(), d["state"].clone()
        ys = [gated_delta_step(*(t[k][:, 0] for k in ("q", "k", "v", "g", "beta")), s) for t, s in zip((d, e), states)]
        assert torch.equal(*ys) and torch.equal(*states)
        del e
