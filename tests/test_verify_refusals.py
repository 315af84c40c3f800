"""CPU checks of the verification's arguments: the C entry refuses them before
anything touches a device."""
from __future__ import annotations

import ctypes as C

import pytest

from util import load_pkg


@pytest.fixture(scope="module")
def sa():
    pkg = load_pkg()
    yield pkg
    pkg.lib().sa_prefill_window(None, None, None, pkg.SA_DTYPE_F32, 1, 1, 1, 0, 64, None, None, None, 1, 0, 1.0, None,
                                None)   # nothing to do: leaves no error behind


def test_refusals(sa):
    lib = sa.lib()
    buf = (C.c_uint8 * 8192)()
    base = (C.addressof(buf) + 15) // 16 * 16
    V = 10
    good = dict(target=base, target_stride=V, draft=base + 512, draft_stride=V, tokens=base + 1024, ua=base + 1088,
                us=base + 1152, n=2, counts=[2, 1], vocab=V, T=1.0, acc=base + 1280, out=base + 1344, width=3, ws=base + 2048,
                ws_bytes=1 << 40)

    def call(**k):
        a = dict(good, **k)
        counts = None if a["counts"] is None else (C.c_int32 * len(a["counts"]))(*a["counts"])
        st = lib.sa_draft_verify(a["target"], a["target_stride"], a["draft"], a["draft_stride"], a["tokens"], a["ua"],
                                 a["us"], a["n"], counts, a["vocab"], a["T"], a["acc"], a["out"], a["width"], a["ws"],
                                 a["ws_bytes"], None)
        return st, lib.sa_last_error().decode()

    bad = [dict(n=0), dict(n=(1 << 20) + 1, counts=None), dict(counts=[65, 0]), dict(counts=[-1, 1]), dict(vocab=0),
           dict(vocab=(1 << 30) + 1), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(target=None),
           dict(tokens=None), dict(ua=None), dict(us=None), dict(acc=None), dict(out=None), dict(target_stride=V - 1),
           dict(draft_stride=V - 1), dict(width=2), dict(ws=base + 2052), dict(out=base + 1028), dict(out=base + 4),
           dict(acc=base + 1152), dict(acc=base + 1348), dict(acc=base + 520),
           dict(n=1 << 20, counts=None, vocab=1 << 30, target_stride=1 << 30, draft=None)]
    for k in bad:
        st, msg = call(**k)
        assert st == sa.SA_EINVAL and msg, (k, st, msg)
    for k in (dict(ws=None), dict(ws_bytes=100)):
        st, msg = call(**k)
        assert st == sa.SA_ENOMEM and "workspace" in msg
    assert lib.sa_draft_verify_ws_bytes(2, (C.c_int32 * 2)(65, 0), V) == 0
    assert lib.sa_draft_verify_ws_bytes(2, None, V) > 0


def test_python_arguments(sa):
    import torch
    x = torch.zeros(3, 10)
    with pytest.raises(ValueError):           # not on a GPU
        sa.draft_verify(x, torch.zeros(2, dtype=torch.int32), torch.zeros(2), torch.zeros(1), [2])
