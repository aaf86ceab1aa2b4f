"""What Engine.sample_groups makes of its settings, on the CPU: the library is
stood in for by a function that keeps what it was given."""
import ctypes as C

import numpy as np
import pytest

from grande_b200 import engine
from grande_b200.engine import BranchTokens, Engine, Group, OmgError

ONE = [Group([2, 3], [BranchTokens([5, 6], [1])])]
THREE = [Group([2, 3], [BranchTokens([5, 6], [0, 1]), BranchTokens([7], [0])])]


class Library:
    def omg_engine_sample_groups(self, h, groups, n, s, tokens, probs, capacity, srcs):
        s = s._obj
        self.all = (s.temperature_all, s.top_k_all, s.top_p_all, s.min_p_all)
        of = (("temperature", C.c_float), ("top_k", C.c_int32), ("top_p", C.c_float),
              ("min_p", C.c_float), ("u", C.c_float))
        self.rows = {k: list(C.cast(getattr(s, k), C.POINTER(t))[:capacity])
                     for k, t in of if getattr(s, k)}
        return 0

    def omg_engine_destroy(self, h):
        pass


@pytest.fixture
def call(monkeypatch):
    fake = Library()
    monkeypatch.setattr(engine, "lib", lambda: fake)
    eng = object.__new__(Engine)
    eng._h = None

    def run(groups, uniforms, **kw):
        eng.sample_groups(groups, uniforms, **kw)
        return fake
    return run


def test_none_is_off(call):
    for groups, u in ((ONE, [0.25]), (THREE, [0.25, 0.5, 0.75])):
        f = call(groups, u, temperature=None, top_k=None, top_p=None, min_p=None)
        assert f.all == (1.0, 0, 1.0, 0.0) and f.rows == {"u": u}
