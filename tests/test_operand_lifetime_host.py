"""CPU: what a C entry gets a pointer to is alive until it returns.

The entries run without the interpreter's lock, so the memory of a copy that is freed before the
call can be another thread's by the time the kernel is launched on the stream they share."""
from __future__ import annotations

import weakref

import torch

import metalblas_b200 as mb
from metalblas_b200 import _lib, router


class Library:
    """Stands for the library: looks at the copies when an entry is called."""

    def __init__(self, copies):
        self.copies, self.called = copies, 0

    def __getattr__(self, name):
        def entry(*args):
            self.called += 1
            assert self.copies and all(t() is not None for t in self.copies), f"{name}: a copy was freed before the call"
            return _lib.MB_OK
        return entry


def test_strided_operands_of_the_balance_gradient(monkeypatch):
    copies = []
    contiguous = torch.Tensor.contiguous

    def record(t, *args, **kw):
        c = contiguous(t, *args, **kw)
        if c is not t:
            copies.append(weakref.ref(c))
        return c

    library = Library(copies)
    monkeypatch.setattr(torch.Tensor, "contiguous", record)
    monkeypatch.setattr(router._lib, "load", lambda: library)
    monkeypatch.setattr(router, "_stream_of", lambda device: None)
    every_other = (lambda *shape, dtype: torch.zeros(*shape[:-1], 2 * shape[-1], dtype=dtype)[..., ::2])
    logits = every_other(4, 8, dtype=torch.float32)
    mask, counts = every_other(4, dtype=torch.bool), every_other(8, dtype=torch.int32)
    balance = mb.ExpertBalance(None, counts, torch.zeros((), dtype=torch.int32))
    router._balance_backward.__wrapped__(logits, torch.ones(()), balance, mask)
    assert library.called == 1 and len(copies) == 3
