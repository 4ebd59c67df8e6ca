"""The state-space operators' Python side on CPU tensors, with the library's launches
replaced: what a launch is handed is looked at in host memory."""

from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch


class Launches:
    """Stands in for the loaded library: sizes come from the real one, launches are kept as
    (name, arguments) in `calls` and, where `look` names one, handed to it first."""

    def __init__(self, real):
        self.real, self.calls, self.look = real, [], {}

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return getattr(self.real, name)

        def launch(*args):
            if name in self.look:
                self.look[name](*args)
            self.calls.append((name, args))
            return 0

        return launch


@pytest.fixture
def launches(monkeypatch):
    from ttt_amd import _lib, norm, ssm
    real = _lib.load()
    fake = Launches(real)
    monkeypatch.setattr(_lib, "load", lambda *a: fake)
    for m in (ssm, norm):
        monkeypatch.setattr(m, "check_device", lambda *ts: ts[0].device)
        monkeypatch.setattr(m, "on_device", lambda dev: contextlib.nullcontext())
        monkeypatch.setattr(m, "_stream", lambda dev: 0)
    ssm._bytes.cache_clear()
    return fake


def rows_at(address, ld, rows, width, dtype):
    """[rows, width]: the values of rows `ld` elements apart from `address` on, copied"""
    es = torch.tensor([], dtype=dtype).element_size()
    n = (rows - 1) * ld + width
    raw = (ctypes.c_char * (n * es)).from_address(address)
    flat = torch.frombuffer(bytearray(raw), dtype=dtype)
    return flat.as_strided((rows, width), (ld, 1)).clone()
