"""GPU tests of what sa_paged_extend refuses before it enqueues anything: workspaces that
are too small for a part of a call."""
from __future__ import annotations

import pytest
import torch

from kv_rows import Rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,counts", [([0, 2000], [32, 3]), ([2000, 0], [3, 32])])
def test_a_call_in_two_parts_is_refused_as_a_whole(sa, lens, counts):
    """A long chunk behind nothing needs no workspace, a short one behind 2000 tokens does."""
    rows = Rows(sa, "f32", 2, 64, lens, seed=31, room=32)
    rows.append(counts)
    x = rows.normal(sum(counts), 4, 64)
    out = torch.full_like(x, 7.0)
    with pytest.raises(sa.SaError, match="workspace"):
        rows.cache.extend(0, x, 0.125, counts, out=out, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    assert (out == 7.0).all()
    rows.cache.extend(0, x, 0.125, counts, out=out)
    assert torch.equal(out, rows.cache.extend(0, x, 0.125, counts))
