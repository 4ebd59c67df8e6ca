"""Bounds value by value for the state-space operators, beside those of tests/_ssm.py for
whole tensors, and references that are computed on the GPU."""

from __future__ import annotations

import math

import torch

from tests import _ssm as T

U = 2.0 ** -24  # half a step of fp32


def each_within(got, ref, size, terms, what, planes=0.0):
    """Every value of got against ref in 64 bits.  It may be off by
    - half a step of got's own type, where that is a 16-bit one (2^-25 where fp16 has no
      smaller steps);
    - 8 half steps of fp32 of `size`, the sum of the absolute values of its terms, for the
      factors of a term, and 4 sqrt(terms) for adding them up: a rounding is off by up to half
      a step, U / sqrt(3) root mean square, those of `terms` sums add up to
      U sqrt(terms / 3), and the largest of 2^23 values is 5.3 standard deviations off;
    - `planes` of `size`: what formed values are rounded to where they are multiplied."""
    dt = got.dtype
    got, ref, size = got.detach().double(), ref.double(), size.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    bound = ((8 + 4 * math.sqrt(terms)) * U + planes) * size + 1e-30
    if dt != torch.float32:
        bound = bound + T.half_step(dt) * (ref.abs() + bound) + (2.0 ** -25 if dt == torch.float16 else 0.0)
    off = (got - ref).abs()
    worst = (off / bound).argmax()
    assert (off <= bound).all(), (f"{what}: {float(got.flatten()[worst])} for {float(ref.flatten()[worst])}, "
                                  f"{float(off.flatten()[worst]):.3e} off, {float(bound.flatten()[worst]):.3e} allowed")


def scan_each(d, got, softplus=True, grads=True):
    """All outputs of a scan on the GPU inputs d, value by value and as whole tensors.  bf16
    results come of formed values in two planes, 2^-17 of them, one in each term."""
    ref, size = T.scan_reference(d, softplus, grads)
    B, L, H, P = d["x"].shape
    N, G = d["Bm"].shape[-1], d["Bm"].shape[2]
    for k in got:
        terms = L + P + N + (B * L if k in ("dA", "dD", "ddt_bias") else 0) + (H // G if k in ("dBm", "dCm") else 0)
        dt = got[k].dtype
        what = f"{k} {tuple(d['x'].shape)} G{G} N{N} {d['x'].dtype}"
        each_within(got[k], ref[k], size[k], terms, what, 2.0 ** -17 if dt == torch.bfloat16 else 0.0)
        T.within(got[k], ref[k].cpu(), size[k].cpu(), terms, what, None if dt == torch.float32 else dt)
