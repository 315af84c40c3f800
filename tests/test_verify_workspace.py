"""CPU check of the verification's workspace: one that lies on an input or an output is
refused before anything touches a device."""
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


def test_overlaps_are_refused(sa):
    lib, V, counts = sa.lib(), 10, (C.c_int32 * 2)(2, 1)
    need = lib.sa_draft_verify_ws_bytes(2, counts, V)
    buf = (C.c_uint8 * (4096 + 2 * need))()
    base = (C.addressof(buf) + 15) // 16 * 16
    at = dict(target=base, draft=base + 512, tokens=base + 1024, ua=base + 1088, us=base + 1152, acc=base + 1280,
              out=base + 1344, ws=base + 2048)

    def call(T=1.0, **k):
        a = dict(at, **k)
        st = lib.sa_draft_verify(a["target"], V, a["draft"], V, a["tokens"], a["ua"], a["us"], 2, counts, V, T, a["acc"],
                                 a["out"], 3, a["ws"], need, None)
        return st, lib.sa_last_error().decode()

    last = at["ws"] + need - 4
    for k in [dict(ws=at[name] // 16 * 16) for name in ("target", "draft", "tokens", "ua", "us", "acc", "out")] + \
            [{name: last} for name in ("target", "draft", "tokens", "ua", "us", "acc", "out")]:
        st, msg = call(**k)
        assert st == sa.SA_EINVAL and "overlap" in msg, (k, st, msg)
    for k in (dict(ws=at["target"]), dict(tokens=last), dict(acc=last), dict(out=last)):
        st, msg = call(T=0.0, **k)                       # draft and uniform numbers are not read
        assert st == sa.SA_EINVAL and "overlap" in msg, (k, st, msg)
