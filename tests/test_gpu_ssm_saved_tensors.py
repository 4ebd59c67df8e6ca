"""Gradients of the state-space operators and of their layer under hooks on saved tensors
(activations kept on the CPU, copies, other layouts, recomputation): the same bits as without."""

import contextlib

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from tests import _ssm as T

pytestmark = pytest.mark.gpu


def _transposed(t):
    return t.transpose(0, -1).contiguous().transpose(0, -1)


def _wider(t):
    wide = torch.full((*t.shape[:-1], t.shape[-1] + 56), 7, dtype=t.dtype, device=t.device)
    return wide[..., 8:8 + t.shape[-1]].copy_(t)


HOOKS = {"on the CPU": lambda: save_on_cpu(), "on the CPU, pinned": lambda: save_on_cpu(pin_memory=True),
         "copies": lambda: saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t),
         "transposed": lambda: saved_tensors_hooks(lambda t: t, _transposed),
         "wider": lambda: saved_tensors_hooks(lambda t: t, _wider)}


ROWS = ["on the CPU", "on the CPU, pinned", "copies"]  # hooks that leave contiguous rows


def _same(run, names=HOOKS):
    want = run(contextlib.nullcontext())
    for name in names:
        got = run(HOOKS[name]())
        for k in want:
            assert torch.equal(got[k], want[k]), (name, k)


@pytest.mark.parametrize("dt", T.DTYPES)
def test_conv(lib, dt):
    d = T.dev(T.conv_inputs(3, 70, 36, 4, dt, seed=50, pad=20))

    def run(hooks):
        with hooks:
            return T.conv_run(d, "silu")

    _same(run)
    T.conv_check({k: v.cpu() for k, v in d.items()}, run(save_on_cpu()), "silu")


@pytest.mark.parametrize("dt", T.DTYPES)
def test_scan(lib, dt):
    c = T.scan_inputs(2, 150, 4, 64, 2, 48, dt, seed=51)
    d = T.dev(c)

    def run(hooks):
        with hooks:
            return T.scan_run(d)

    _same(run)
    T.scan_check(c, run(save_on_cpu()))


@pytest.mark.parametrize("dt", T.DTYPES)
def test_norm(lib, dt):
    from ttt_amd.norm import layer_norm
    g = torch.Generator().manual_seed(52)
    wide = torch.randn(40, 3, 200, generator=g).to(dt).cuda()
    w, b = (torch.randn(72, generator=g).cuda() for _ in range(2))
    dy = torch.randn(40, 3, 72, generator=g).to(dt).cuda()

    def run(hooks):
        x, z = (wide[..., k:k + 72].detach().requires_grad_(True) for k in (5, 101))
        par = [t.detach().requires_grad_(True) for t in (w, b)]
        with hooks:
            y = layer_norm(x, *par, gate=z)
        return dict(zip(("y", "x", "z", "w", "b"), [y.detach(), *torch.autograd.grad(y, [x, z, *par], dy)]))

    _same(run)


@pytest.mark.parametrize("dt", [None, torch.bfloat16])
def test_layer(lib, dt):
    """The layer hands its operators columns of one projection.  (Contiguous rows alone: torch's
    products beside them round as their operands lie in memory.)"""
    from torch.utils.checkpoint import checkpoint

    from ttt_amd.model import ModelConfig, TTTWrapper
    torch.manual_seed(53)
    m = TTTWrapper(ModelConfig(seq_len=128, model_dim=256, num_heads=4, ssm_layer="selective_scan",
                               mini_batch_size=16)).cuda()
    x, dy = torch.randn(2, 100, 256, device="cuda"), torch.randn(2, 100, 256, device="cuda")

    def run(hooks, again=False):
        with hooks, torch.autocast("cuda", dtype=dt or torch.bfloat16, enabled=dt is not None):
            y = checkpoint(m, x, use_reentrant=False) if again else m(x)
        gs = torch.autograd.grad(y, list(m.parameters()), dy.to(y.dtype))
        return dict(zip(["y", *(n for n, _ in m.named_parameters())], [y.detach(), *gs]))

    want = run(contextlib.nullcontext())
    _same(run, ROWS)
    got = run(contextlib.nullcontext(), again=True)
    for k in want:
        assert torch.equal(got[k], want[k]), k
