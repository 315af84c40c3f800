"""GPU test of a prompt's chunks, each over what is committed by then, against 64-bit
attention, with the tolerances of the attention of chunks."""
from __future__ import annotations

import math

import pytest
import torch

from kv_rows import Rows, attend
from test_gpu_extend import PAIRS, TYPE, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("parts", [[1, 64, 300, 335], [65, 1, 1, 200], [513, 3, 31, 64, 65]])
def test_chunks_of_a_prompt(sa, q, kv, Hq, Hkv, D, parts):
    rows = Rows(sa, kv, Hkv, D, [0], seed=33, room=sum(parts))
    at, scale = 0, 1 / math.sqrt(D)
    for n in parts:
        rows.append([n])
        x = rows.normal(n, Hq, D, dtype=TYPE[q])
        check(rows.cache.extend(0, x, scale, [n]), *attend(x, rows.k[0], rows.v[0], scale, at))
        rows.cache.commit(n, n_seqs=1)
        at += n
