"""Paged caches of the GPU tests with what they hold in 64 bits, and the plain
attention that they are compared with."""
from __future__ import annotations

import torch

KV = ("f32", "bf16", "fp8")


def e4m3(y):
    """The nearest value of 4 exponent and 3 mantissa bits to y (64 bits, |y| <= 448), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def held_fp8(x):
    """Rows of the last axis as an 8-bit cache holds them: (values in 64 bits, exponents)."""
    x = x.double()
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** -100)))
    y = x / torch.exp2(e)
    limit = torch.where(e >= 120, 240.0, 448.0)
    v = e4m3(torch.minimum(torch.maximum(torch.where(x.isfinite(), y, 0.0), -limit), limit)) * torch.exp2(e)
    return torch.where(x.isfinite(), v, float("nan")), e.long()


def held(x, kv):
    if kv == "fp8":
        return held_fp8(x)[0]
    return (x.bfloat16() if kv == "bf16" else x).double()


def code(sa, kv):
    return {"f32": sa.SA_DTYPE_F32, "bf16": sa.SA_DTYPE_BF16, "fp8": sa.SA_DTYPE_FP8}[kv]


def poison(sa, cache, layer=0):
    """Every place of the pools that no append has written holds NaN."""
    for view in sa.kv_pool_views(cache, layer):
        if view.dtype == torch.float8_e4m3fn:
            view.view(torch.uint8).fill_(0x7f)
        else:
            view.fill_(float("nan"))
    if cache.desc.kv_dtype == sa.SA_DTYPE_FP8:
        for view in sa.kv_scale_views(cache, layer):
            view.fill_(255)


class Rows:
    """A cache on shuffled pages, and its rows' keys and values as they are held."""

    def __init__(self, sa, kv, Hkv, D, lens, seed, room=0, spare=3):
        self.sa, self.kv, self.Hkv, self.D = sa, kv, Hkv, D
        counts = [(n + room + 63) // 64 for n in lens]
        pages = sum(counts) + spare
        self.cache = sa.KVCache(1, Hkv, D, len(lens), max(*counts, 1) + 1, pages, code(sa, kv))
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        poison(sa, self.cache)
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        at = 0
        for r, c in enumerate(counts):
            self.cache.set_pages(r, perm[at:at + c])
            at += c
        self.k = [torch.empty(0, Hkv, D, device="cuda", dtype=torch.float64) for _ in lens]
        self.v = list(self.k)
        self.append(lens, commit=True)

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=self.gen).to(dtype)

    def append(self, counts, commit=False, change=None):
        """New tokens of every row; change(k, v) alters what is appended."""
        T = sum(counts)
        if T == 0:
            return
        k, v = self.normal(T, self.Hkv, self.D), self.normal(T, self.Hkv, self.D)
        if change:
            change(k, v)
        self.cache.append(0, None, k, v, counts=counts)
        at = 0
        for r, n in enumerate(counts):
            self.k[r] = torch.cat([self.k[r], held(k[at:at + n], self.kv)])
            self.v[r] = torch.cat([self.v[r], held(v[at:at + n], self.kv)])
            at += n
            if commit and n:
                self.cache.commit(n, seqs=[r])


def attend(q, k, v, scale, past):
    """q [n, Hq, D] of tokens past .. past + n - 1, k and v [T, Hkv, D], T >= past + n -> (out, sum of w |v|) in 64 bits."""
    n, Hq, D = q.shape
    rep = Hq // k.shape[1]
    out, mag = [], []
    for j in range(n):
        kk, vv = (x[:past + j + 1].repeat_interleave(rep, 1) for x in (k, v))      # [T, Hq, D]
        w = torch.softmax((kk * q[j].double()).sum(-1) * scale, 0)[..., None]
        out.append((w * vv).sum(0))
        mag.append((w * vv.abs()).sum(0))
    return torch.stack(out), torch.stack(mag)
