"""The block norm and the gated feed-forward projections, forward and backward, on another stream than
the current one was and captured into a graph, and the delta rule's backward: each replay on new
values, with eager calls in between, gives the eager call's bits."""

import pytest
import torch

from tests import _block as T
from tests import test_gpu_block_norm as N
from tests import test_gpu_ffn as FF

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def norm_case(shape, parts, res_dt):
    def f(seed):
        return N.inputs(shape, BF16, parts, res_dt, seed=seed)

    def call(leaves, d):
        from ttt_amd.norm import block_norm
        out = block_norm(*(leaves.get(k) for k in N.ARGS))
        out = list(out) if isinstance(out, tuple) else [out]
        return [t.detach() for t in out], torch.autograd.grad(out, list(leaves.values()), [d["dr"], d["dy"]][:len(out)])

    return f, call, N.ARGS


def ffn_case(R, D, F, dt, bias):
    def f(seed):
        return FF.inputs(R, D, F, dt, bias=bias, seed=seed)

    def call(leaves, d):
        from ttt_amd.ffn import gated_linear
        y = gated_linear(*(leaves.get(k) for k in FF.ARGS), activation="gelu")
        return [y.detach()], torch.autograd.grad(y, list(leaves.values()), d["dy"])

    return f, call, FF.ARGS


def delta_case(dt):
    def f(seed):
        return T.delta_inputs(3, 130, 4, 2, 32, 64, dt, seed=seed)

    def call(leaves, d):
        from ttt_amd.delta import gated_delta
        out = gated_delta(*(leaves[k] for k in T.DELTA_ARGS), return_final_state=True)
        return [t.detach() for t in out], torch.autograd.grad(out, list(leaves.values()), [d["do"], d["dlast"]])

    return f, call, T.DELTA_ARGS


CASES = {"norm": norm_case((300, 768), "wsrn", F32), "norm of heads": norm_case((5, 40, 6, 64), "wg", None),
         "norm of wide rows": norm_case((9, 5000), "wgsrn", F32), "ffn": ffn_case(300, 96, 72, BF16, True),
         "ffn of few rows": ffn_case(5, 96, 72, F16, False), "ffn in shares": ffn_case(700, 501, 333, F32, True),
         "ffn in fp16": ffn_case(700, 96, 40, F16, True), "delta": delta_case(BF16), "delta in fp32": delta_case(F32)}


def _leaves(d, args):
    return {k: d[k].detach().clone().requires_grad_(True) for k in args if d[k] is not None}


@pytest.mark.parametrize("name", CASES)
def test_on_another_stream(lib, name):
    inputs, call, args = CASES[name]
    d = T.dev(inputs(1))
    want = call(_leaves(d, args), d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(_leaves(d, args), d)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip([*want[0], *want[1]], [*got[0], *got[1]]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", CASES)
def test_forward_and_backward_in_a_graph(lib, name):
    inputs, call, args = CASES[name]
    d = T.dev(inputs(2))
    leaves = _leaves(d, args)
    d = {k: t if t is None or k in leaves else t.clone() for k, t in d.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(leaves, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = call(leaves, d)
    for seed in (3, 4, 5, 6):
        e = T.dev(inputs(seed))
        with torch.no_grad():
            for k, t in d.items():
                if t is not None:
                    (leaves[k] if k in leaves else t).copy_(e[k])
        graph.replay()
        want = call(_leaves(e, args), e)
        torch.cuda.synchronize()
        for a, b in zip([*out, *grads], [*want[0], *want[1]]):
            assert torch.equal(a, b), seed
