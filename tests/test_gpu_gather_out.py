"""GPU test of reading a cache back into outputs of any alignment, or one of K and V
only: the same bits as into aligned ones, and nothing beside them."""
from __future__ import annotations

import pytest
import torch

from kv_rows import KV, Rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 65, 700])
def test_outputs_of_any_alignment(sa, kv, D, n):
    rows = Rows(sa, kv, 2, D, [n, 5], seed=34)
    want = rows.cache.gather(0, 0, n)
    assert torch.equal(want[0].transpose(0, 1).double(), rows.k[0])
    size = 2 * n * D
    for at in range(1, 4):
        bufs = [torch.full((size + 8,), 7.0, device="cuda") for _ in range(2)]
        for which in ((0, 1), (0,), (1,)):
            for b in bufs:
                b.fill_(7.0)
            sa.check(sa.lib().sa_kvcache_gather(rows.cache.handle, 0, 0, n,
                                                *(bufs[i].data_ptr() + 4 * at if i in which else None for i in (0, 1)),
                                                torch.cuda.current_stream().cuda_stream))
            for i, b in enumerate(bufs):
                part = b[at:at + size]
                assert torch.equal(part.view(2, n, D), want[i]) if i in which else (part == 7.0).all()
                assert (b[:at] == 7.0).all() and (b[at + size:] == 7.0).all()
