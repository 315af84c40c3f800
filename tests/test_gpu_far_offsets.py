"""GPU tests of tensors and pools whose far ends lie beyond 2^32 bytes: pages at
the end of a large pool (decoded, forked, reordered), prompts of far apart rows
and logits of far apart rows, each against the same data laid out densely."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_pages_at_the_end_of_a_large_pool(sa, kv):
    dt, elem = (sa.SA_DTYPE_BF16, 2) if kv == "bf16" else (sa.SA_DTYPE_F32, 4)
    Hkv, D, n, rows, layers = 8, 128, 200, 4, 2
    pages = (5 << 30) // (64 * Hkv * D * elem)          # K and V of a layer: 5 GiB each
    far = sa.KVCache(layers, Hkv, D, rows, 8, pages, dt)
    near = sa.KVCache(layers, Hkv, D, rows, 8, rows * 8, dt)
    for c, first in ((far, pages - rows * 4), (near, 0)):
        gen = torch.Generator(device="cuda").manual_seed(1)
        for r in range(rows):
            c.set_pages(r, [first + 4 * r + j for j in range(4)])
        for layer in range(layers):
            c.append(layer, None, *(torch.randn(rows, n, Hkv, D, device="cuda", generator=gen) for _ in range(2)))
        c.commit(n, n_seqs=rows)
    q = torch.randn(rows, 2 * Hkv, D, device="cuda")

    def compare():
        for layer in range(layers):
            assert torch.equal(far.decode_window(layer, q, 0.09, 90, 3), near.decode_window(layer, q, 0.09, 90, 3))
            assert torch.equal(far.decode_shared(layer, q, 0.09), near.decode_shared(layer, q, 0.09))
            for r in range(rows):
                for a, b in zip(far.gather(layer, r, far.length(r)), near.gather(layer, r, near.length(r))):
                    assert torch.equal(a, b)

    compare()
    for c in (far, near):
        c.fork(1, 3, 150)
    compare()
    for c in (far, near):
        c.reorder([0, 1, 2, 3], [3, 3, 3, 0])
    compare()
    far.close()
    near.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompt_of_far_apart_rows(sa, dtype):
    """Rows almost 2^24 elements apart, the largest stride that k and v take."""
    Hq, Hkv, L, D, step = 4, 2, 200, 64, (1 << 24) - 8
    buf = torch.empty(L, step, dtype=dtype, device="cuda")
    x = [torch.randn(1, h, L, D, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv)]
    views, at = [], step - (2 * Hq + 2 * Hkv) * D      # the end of each row
    for t in (*x, x[0]):
        h = t.shape[1]
        views.append(buf[:, at:at + h * D].view(L, h, D).permute(1, 0, 2)[None])
        at += h * D
    for v, t in zip(views, x):
        v.copy_(t)
    out = views[3]
    sa.prefill_window(*views[:3], 0.1, 70, 5, out=out)
    assert torch.equal(out, sa.prefill_window(*x, 0.1, 70, 5))


def test_logits_of_far_apart_rows(sa):
    B, V, step = 5, 2001, (1 << 29) + 1
    buf = torch.empty((B - 1) * step + V, device="cuda")
    x = torch.randn(1, B, V, device="cuda")
    far = buf.as_strided((1, B, V), (B * step, step, 1))
    far.copy_(x)
    s = -torch.rand(1, B, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(sa.beam_select(far, s, 12), sa.beam_select(x, s, 12)))
