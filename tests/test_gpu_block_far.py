"""A gated delta-rule block's operators on the GPU over tensors of more than 2^31 values, and the block
norm over more rows than a launch has threads for: the results at both ends and at the borders are
those of calls on these parts alone."""

import math

import pytest
import torch

from tests import _block as T
from tests import test_gpu_block_norm as N
from tests import test_gpu_ffn as FF

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def room():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GB of the GPU's memory")
    yield
    torch.cuda.empty_cache()


def _norm_parts(R, D, spots, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, dt=BF16: torch.empty(*s, device="cuda", dtype=dt).normal_(generator=g)  # noqa: E731
    d = dict(x=r(R, D), weight=1 + 0.1 * r(D, dt=F32), residual=r(R, D, dt=BF16), gate=r(R, D), scale=0.5 + 0.1 * r(D, dt=F32),
             next_weight=1 + 0.1 * r(D, dt=F32), dr=r(R, D), dy=r(R, D))
    got = N.run(d)
    for a, b in spots:
        part = {k: t[a:b] if t.dim() == 2 else t for k, t in d.items()}
        want = N.run(part)
        for k in ("r", "y", "dx", "dresidual", "dgate"):
            assert torch.equal(got[k][a:b], want[k]), (k, a)
    return d, got


def test_norm_of_wide_rows(lib):
    """270,000 rows of 8,192 values: 2.2e9 of them"""
    R = 270_000
    _norm_parts(R, 8192, ((0, 3), (131071, 131074), (262142, 262146), (R - 3, R)), 1)


def test_norm_in_several_launches(lib):
    """Rows of one value, eight threads to a row: a launch has 2^29 of them"""
    R = (1 << 29) + 4099
    _norm_parts(R, 1, ((0, 100), ((1 << 28) - 50, (1 << 28) + 50), ((1 << 29) - 64, (1 << 29) + 64), (R - 100, R)), 2)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("D,F", [(64, 2048), (2048, 64)])
def test_gated_linear(lib, dt, D, F):
    R = 1_100_003
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.empty(*s, device="cuda", dtype=dt).normal_(generator=g)  # noqa: E731
    d = dict(x=r(R, D), w_gate=r(F, D) / D ** 0.5, w_up=r(F, D) / D ** 0.5, b_gate=None, b_up=None, dy=r(R, F))
    got = FF.run(d)
    for a in (0, 1 << 20, R - 200):
        part = {k: t if t is None or k[0] == "w" else t[a:a + 200] for k, t in d.items()}
        FF.check({k: None if t is None else t.cpu() for k, t in part.items()}, {k: got[k][a:a + 200] for k in ("y", "dx")})
    # the weights' gradients, of the rows in two calls that are each within 2^31 values
    halves = [FF.run({k: t if t is None or k[0] == "w" else t[a:b] for k, t in d.items()}) for a, b in ((0, R // 2), (R // 2, R))]
    for k in ("dw_gate", "dw_up"):
        want = sum(h[k].double() for h in halves)
        # (a rounding at the store of each, and of three calls' sums of da and db, rounded to the type, by fp32 sums of R
        # terms, whose sizes are like the root of R times those of a term: sqrt(R) 2^-24 of the whole at most)
        assert float((got[k].double() - want).norm() / want.norm()) <= 3 * T.half_step(dt) + 3 * T.U * (8 + math.sqrt(R)), k


@pytest.mark.parametrize("dt", [BF16, F16])
def test_gated_delta(lib, dt):
    """16 heads of 256 features: 2.2e9 values of v.  A decay of nothing left before the last 300 tokens: they, and their
    gradients, stand alone."""
    H, P, n, L = 16, 256, 16, 530_000 // 64 * 64 + 300
    tail = T.delta_inputs(1, 300, H, 1, n, P, dt, seed=4, packed=False)
    tail["g"][:, 0] = -math.inf
    d = {}
    g = torch.Generator(device="cuda").manual_seed(5)
    for k, t in tail.items():
        if k in ("state", "dlast"):
            d[k] = t.cuda()
            continue
        d[k] = torch.empty(1, L, *t.shape[2:], device="cuda", dtype=t.dtype)
        d[k].normal_(generator=g) if k in ("q", "k", "v", "do") else d[k].uniform_(-1, 0, generator=g) if k == "g" else d[k].uniform_(0, 1, generator=g)
        d[k][:, -300:] = t.cuda()
    got = T.delta_run(d)
    part = {k: t[:, -300:] for k, t in got.items() if k not in ("last", "dstate")}
    part["last"] = got["last"]
    T.delta_check({**tail, "g": tail["g"].clamp(min=-1e4), "state": torch.zeros_like(tail["state"])}, part)
    # the first tokens see no later ones
    ref = T.delta_run({k: t if k in ("state", "dlast") else t[:, :320].contiguous() for k, t in d.items()}, grads=False)
    assert float((got["o"][:, :320].double() - ref["o"].double()).norm() / ref["o"].double().norm()) <= 2 * T.half_step(dt) + 4 * 2.0 ** -17
    assert all(torch.isfinite(got[k].float()).all() for k in ("o", "last", "dv", "dq", "dk", "dg", "dbeta", "dstate"))
