"""GPU tests of what sa_paged_extend refuses before it enqueues anything: workspaces that
are too small for a part of a call, and overlapping arguments."""
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


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "fp8")])
@pytest.mark.parametrize("n", [5, 300])
def test_overlaps_are_refused(sa, q, kv, n):
    rows = Rows(sa, kv, 2, 64, [1000], seed=32, room=n)
    rows.append([n])
    buf = rows.normal(2 * n + 1, 4, 64, dtype={"f32": torch.float32, "bf16": torch.bfloat16}[q])
    before = buf.clone()
    ext = lambda x, **k: rows.cache.extend(0, x, 0.125, [n], **k)  # noqa: E731
    for at in (0, 1, n - 1):
        for x, out in ((buf[:n], buf[at:at + n]), (buf[at:at + n], buf[:n])):
            with pytest.raises(sa.SaError, match="overlap"):
                ext(x, out=out)
    need = rows.cache.extend_ws_bytes([n], 4)
    raw = buf.view(torch.uint8).view(-1)
    assert 16 < need
    big = torch.empty(need + 2 * raw.numel(), dtype=torch.uint8, device="cuda")
    inside = big[need - 16:need - 16 + n * 4 * 64 * buf.element_size()].view(buf.dtype).view(n, 4, 64)
    with pytest.raises(sa.SaError, match="overlap"):
        ext(buf[:n], out=inside, ws=big[:need])          # the workspace's last bytes
    with pytest.raises(sa.SaError, match="overlap"):
        ext(inside, out=buf[:n], ws=big[:need])
    torch.cuda.synchronize()
    assert torch.equal(buf, before)
    beside = big[need + (-need) % 16:][:n * 4 * 64 * buf.element_size()].view(buf.dtype).view(n, 4, 64)
    want = ext(buf[:n])
    assert torch.equal(ext(buf[:n], out=buf[n:2 * n]), want) and torch.equal(ext(buf[:n], out=beside, ws=big[:need]), want)
