"""CPU: an extension and a library of different builds say so.

The extension may be older than the library while the builder runs (it imports the package
first), so a list of functions that it refuses is no error; but every later call would pay for
its arguments' checks in Python, and a program has to be told."""
from __future__ import annotations

import types
import warnings

import pytest

from metalblas_b200 import _lib


class Library:
    """A library that has every function but those named."""

    def __init__(self, real, without=()):
        self.real, self.without = real, without

    def __getattr__(self, name):
        if name in self.without:
            raise AttributeError(name)
        return getattr(self.real, name)


def refuse(addresses):
    raise RuntimeError("set_ops: 8 addresses expected")


def test_the_present_build_is_registered_without_a_word(lib):
    got = []
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        _lib.register_ops(types.SimpleNamespace(set_ops=got.extend), lib)
    assert len(got) == len(_lib._FAST_OPS) and all(got)


@pytest.mark.parametrize("mod,without", [
    (types.SimpleNamespace(set_ops=refuse), ()),                            # built for another list
    (types.SimpleNamespace(), ()),                                          # built before there was one
    (types.SimpleNamespace(set_ops=lambda a: None), ("mb_expert_route",))])  # newer than the library
def test_other_builds_are_reported(lib, mod, without):
    with pytest.warns(RuntimeWarning, match="metalblas_b200.build"):
        _lib.register_ops(mod, Library(lib, without))
