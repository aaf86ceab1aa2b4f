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


def test_numbers_of_any_kind(call):
    f = call(ONE, np.array([0.25]), temperature=np.float64(0.5), top_k=np.int64(7),
             top_p=np.float32(0.75), min_p=np.array(0.125))
    assert f.all == (0.5, 7, 0.75, 0.125)
    f = call(THREE, [0.25, 0.5, 0.75], temperature=(0, 1, 2), top_k=[3.0, 2.0, 0.0],
             top_p=np.array([1, 0.5, 1], np.float16), min_p=[0, 0.5, 0])
    assert f.rows == {"u": [0.25, 0.5, 0.75], "temperature": [0, 1, 2], "top_k": [3, 2, 0],
                      "top_p": [1, 0.5, 1], "min_p": [0, 0.5, 0]}
    assert call(ONE, [0.5], temperature=1e300).all[0] == float("inf")


@pytest.mark.parametrize("kw,text", [
    (dict(top_k=2 ** 32 + 5), "top_k: whole numbers of 32 bits"),
    (dict(top_k=[2 ** 32 + 5]), "top_k: whole numbers of 32 bits"),
    (dict(top_k=0.5), "top_k: whole numbers of 32 bits"),
    (dict(top_k=[1.5]), "top_k: whole numbers of 32 bits"),
    (dict(top_k=float("nan")), "top_k: whole numbers of 32 bits"),
    (dict(top_p="a"), "top_p: numbers expected"),
    (dict(temperature=[None]), "temperature: numbers expected"),
    (dict(min_p=[0.1, 0.2]), "min_p: .2. values for 1 rows"),
])
def test_refused(call, kw, text):
    with pytest.raises(OmgError, match=text):
        call(ONE, [0.5], **kw)


@pytest.mark.parametrize("u", [None, 0.5, ["a"], [None], [], [0.1, 0.2], [[0.1]]])
def test_uniforms_refused(call, u):
    with pytest.raises(OmgError, match="uniforms"):
        call(ONE, u)
