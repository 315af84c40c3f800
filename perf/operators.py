"""Performance cases of the serving operators over long, shared and searched contexts.

Kinds:

  prefill_window  causal prefill attention in which a query sees the last `window` keys up to its own and the
                  first `sink` keys of the prompt (prefill_window)
  decode_window   the same rule for one token of each of a batch of sequences over a paged cache
                  (KVCache.decode_window)
  decode_shared   one token of each of a batch of sequences whose leading pages are shared in groups: the pages
                  of a group are read once for all its rows (KVCache.decode_shared)
  beam_select     one beam search selection over beams and vocabulary: the best continuations by accumulated log
                  probability (beam_select)

`own` chooses between the plain form of each operator (elementary torch operations) and the framework's call.
A case is a dict of plain values; `draw` gives more of the same ranges.  Outputs and workspaces are allocated
once per state, as a serving loop does.
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
PAGE = 64
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
VOCAB = 151936


def _package():
    name = "streaming_attention_amd"
    if name not in sys.modules:
        pkg = ROOT / "streaming-attention_amd"
        spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ---------------------------------------------------------------- cases

def listed():
    return [
        # A long prompt of a streaming session: a window much shorter than the prompt, four sink tokens.
        {"name": "prefill-window-bf16-l8192", "kind": "prefill_window", "dtype": "bf16", "B": 1, "L": 8192, "Hq": 16,
         "Hkv": 8, "D": 128, "window": 1024, "sink": 4},
        # An ordinary prompt at the reference's precision.
        {"name": "prefill-window-f32-l2048", "kind": "prefill_window", "dtype": "f32", "B": 1, "L": 2048, "Hq": 16,
         "Hkv": 8, "D": 128, "window": 512, "sink": 4},
        # A few short prompts of a length that is no multiple of any tile, narrow heads, no sinks.
        {"name": "prefill-window-bf16-b3-l777", "kind": "prefill_window", "dtype": "bf16", "B": 3, "L": 777, "Hq": 16,
         "Hkv": 4, "D": 64, "window": 200, "sink": 0},
        # Interactive generation of one session, fp32 cache: all latency.
        {"name": "decode-window-b1-f32", "kind": "decode_window", "kv": "f32", "B": 1, "lo": 5000, "hi": 5000,
         "Hq": 16, "Hkv": 8, "D": 128, "window": 1024, "sink": 4},
        # Batched serving of sessions of very different lengths, bf16 cache.
        {"name": "decode-window-b64-bf16", "kind": "decode_window", "kv": "bf16", "B": 64, "lo": 512, "hi": 32768,
         "Hq": 16, "Hkv": 8, "D": 128, "window": 4096, "sink": 4},
        # Odd sizes: sinks that end inside the second page, a window that starts anywhere, wide head groups.
        {"name": "decode-window-b7-odd", "kind": "decode_window", "kv": "bf16", "B": 7, "lo": 1, "hi": 3001,
         "Hq": 32, "Hkv": 8, "D": 64, "window": 333, "sink": 70},
        # 64 requests behind one long system prompt or document, bf16 cache.
        {"name": "decode-shared-b64-p32768", "kind": "decode_shared", "kv": "bf16", "groups": 1, "rows": 64,
         "prefix_lo": 32768, "prefix_hi": 32768, "suffix": 512, "Hq": 16, "Hkv": 8, "D": 128},
        # Beam searches over several prompts of odd lengths, fp32 cache.
        {"name": "decode-shared-4x4-f32", "kind": "decode_shared", "kv": "f32", "groups": 4, "rows": 4,
         "prefix_lo": 1500, "prefix_hi": 2100, "suffix": 65, "Hq": 16, "Hkv": 8, "D": 128},
        # One beam search over a short prompt: all latency.
        {"name": "decode-shared-1x4-bf16", "kind": "decode_shared", "kv": "bf16", "groups": 1, "rows": 4,
         "prefix_lo": 512, "prefix_hi": 512, "suffix": 33, "Hq": 16, "Hkv": 8, "D": 128},
        # One beam search over the decoder's vocabulary; twice as many continuations as beams, so that ended ones
        # can be set aside.
        {"name": "beam-select-1x4", "kind": "beam_select", "groups": 1, "beams": 4, "vocab": VOCAB, "select": 8},
        # A batch of searches.
        {"name": "beam-select-8x8", "kind": "beam_select", "groups": 8, "beams": 8, "vocab": VOCAB, "select": 16},
        # A vocabulary of an odd size: rows start at any 4-byte address.
        {"name": "beam-select-3x5-odd", "kind": "beam_select", "groups": 3, "beams": 5, "vocab": 32003, "select": 10},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(query heads, KV heads): the decoder's shape most often, other groups beside it."""
    return rng.choice([(16, 8), (16, 8), (32, 8), (16, 4), (8, 8), (32, 4)])


def draw(rng):
    kind = rng.choice(["prefill_window", "decode_window", "decode_shared", "beam_select"])
    if kind == "beam_select":
        groups = _log_int(rng, 1, 8)
        beams = _log_int(rng, 1, 16 if groups <= 4 else 8)
        return {"kind": kind, "groups": groups, "beams": beams, "vocab": _log_int(rng, 1000, 160000),
                "select": min(32, rng.choice([1, 2, 2]) * beams)}
    Hq, Hkv = _heads(rng)
    D = rng.choice([128, 128, 64])
    if kind == "prefill_window":
        dtype = rng.choice(["f32", "bf16", "bf16"])
        L = _log_int(rng, 16, 2048 if dtype == "f32" else 8192)
        B = rng.randint(1, max(1, min(4, 4096 // L)))
        return {"kind": kind, "dtype": dtype, "B": B, "L": L, "Hq": 16, "Hkv": min(Hkv, 8), "D": D,
                "window": _log_int(rng, 1, max(2, min(L, 1024))), "sink": rng.choice([0, 0, 1, 4, _log_int(rng, 1, 128)])}
    kv = rng.choice(["f32", "bf16", "bf16"])
    if kind == "decode_window":
        B, hi = _log_int(rng, 1, 64), _log_int(rng, 64, 16384)
        return {"kind": kind, "kv": kv, "B": B, "lo": rng.randint(1, hi), "hi": hi, "Hq": Hq, "Hkv": Hkv, "D": D,
                "window": _log_int(rng, 1, 4096), "sink": rng.choice([0, 1, 4, 4, _log_int(rng, 1, 200)])}
    groups = _log_int(rng, 1, 8)
    rows = _log_int(rng, 1, max(2, 64 // groups))
    hi = _log_int(rng, 65, 16384 // groups)
    return {"kind": kind, "kv": kv, "groups": groups, "rows": rows, "prefix_lo": max(1, hi - hi // 3),
            "prefix_hi": hi, "suffix": _log_int(rng, 1, 512), "Hq": Hq, "Hkv": Hkv, "D": D}


# ---------------------------------------------------------------- inputs

def _gen(seed, tag, device="cuda"):
    return torch.Generator(device=device).manual_seed((seed * 1000003 + tag * 7919 + 17) % (1 << 62))


def _normal(seed, tag, shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=_gen(seed, tag))


def _pages_for(tokens):
    return -(-tokens // PAGE)


def _case_rng(case, tag):
    return random.Random(sum((i + 1) * 7919 * int(v) for i, v in enumerate(case.values()) if isinstance(v, int)) + tag)


def _window_lengths(case):
    """Cached tokens of each sequence: fixed by the case, the longest and the shortest among them."""
    r = _case_rng(case, 1)
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["B"])]
    lens[0] = case["hi"]
    if case["B"] > 1:
        lens[-1] = case["lo"]
    return lens


def _shared_lengths(case):
    """(prompt tokens of each group, tokens of each row behind its group's prompt): fixed by the case."""
    r = _case_rng(case, 2)
    prompts = [r.randint(case["prefix_lo"], case["prefix_hi"]) for _ in range(case["groups"])]
    return prompts, [r.randint(1, case["suffix"]) for _ in range(case["groups"] * case["rows"])]


def _window_layout(case, seed):
    """Shuffled pages of every sequence, and the pools that hold the cached keys and values."""
    lens = _window_lengths(case)
    counts = [_pages_for(n) for n in lens]
    perm = torch.randperm(sum(counts), generator=_gen(seed, 5, "cpu")).tolist()
    ends = [sum(counts[:i + 1]) for i in range(len(counts))]
    lists = [perm[e - n:e] for e, n in zip(ends, counts)]
    shape = (sum(counts), case["Hkv"], PAGE, case["D"])
    k, v = (_normal(seed, t, shape, DTYPE[case["kv"]]) for t in (2, 3))
    return lens, lists, k, v


def _shared_tensors(case, seed):
    """Keys and values of the groups' prompts [G, P, Hkv, D] and of what the rows have behind them [N, S, Hkv, D],
    padded to the longest."""
    prompts, tails = _shared_lengths(case)
    kp, vp = (_normal(seed, t, (case["groups"], max(prompts), case["Hkv"], case["D"])) for t in (2, 3))
    ks, vs = (_normal(seed, t, (len(tails), max(tails), case["Hkv"], case["D"])) for t in (4, 5))
    return prompts, tails, [x.to(DTYPE[case["kv"]]) for x in (kp, vp, ks, vs)]


def _queries(case, seed, rows):
    return _normal(seed, 1, (rows, case["Hq"], case["D"]))


def _beam_inputs(case, seed):
    """Logits of a few confident and many unlikely tokens, and the beams' accumulated log probabilities."""
    G, B, V = case["groups"], case["beams"], case["vocab"]
    logits = _normal(seed, 1, (G, B, V)) * 2.5
    scores = -20.0 * torch.rand(G, B, device="cuda", generator=_gen(seed, 2))
    return logits, scores


def _prefill_inputs(case, seed):
    B, L, Hq, Hkv, D, dt = (case[n] for n in ("B", "L", "Hq", "Hkv", "D", "dtype"))
    return [_normal(seed, t, (B, H, L, D), DTYPE[dt]) for t, H in ((1, Hq), (2, Hkv), (3, Hkv))]


def _table(lists):
    width = max(len(p) for p in lists)
    return torch.tensor([p + [0] * (width - len(p)) for p in lists], dtype=torch.int64, device="cuda")


def _kv_code(case):
    sa = _package()
    return sa.SA_DTYPE_BF16 if case["kv"] == "bf16" else sa.SA_DTYPE_F32


def prepare(case, seed):
    kind = case["kind"]
    if kind == "beam_select":
        logits, scores = _beam_inputs(case, seed)
        s = {"case": case, "logits": logits, "scores": scores}
        if own:
            G, N = case["groups"], case["select"]
            s["out"] = (torch.empty(G, N, device="cuda"), torch.empty(G, N, dtype=torch.int32, device="cuda"),
                        torch.empty(G, N, dtype=torch.int32, device="cuda"))
            need = _package().beam_select_ws_bytes(G, case["beams"], case["vocab"], N)
            s["ws"] = torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")
        return s
    s = {"case": case, "scale": 1.0 / math.sqrt(case["D"])}
    if kind == "prefill_window":
        q, k, v = _prefill_inputs(case, seed)
        s.update(q=q, k=k, v=v, out=torch.empty_like(q))
        return s
    if kind == "decode_window":
        lens, lists, k, v = _window_layout(case, seed)
        s["q"] = _queries(case, seed, len(lens))
        if own:
            sa = _package()
            cache = sa.KVCache(1, case["Hkv"], case["D"], len(lens), max(map(len, lists)), sum(map(len, lists)),
                               _kv_code(case))
            for view, pool in zip(sa.kv_pool_views(cache, 0), (k, v)):
                view.copy_(pool.reshape(-1))
            for i, (n, pages) in enumerate(zip(lens, lists)):
                cache.set_pages(i, pages)
                cache.set_len(i, n)
            need = cache.decode_window_ws_bytes(len(lens), case["Hq"], case["window"], case["sink"])
            s.update(cache=cache, out=torch.empty_like(s["q"]),
                     ws=torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda"))
        else:
            s.update(k=k, v=v, table=_table(lists), lens=torch.tensor(lens, device="cuda"))
        return s
    prompts, tails, (kp, vp, ks, vs) = _shared_tensors(case, seed)
    G, R = case["groups"], case["rows"]
    s["q"] = _queries(case, seed, G * R)
    if own:
        sa = _package()
        per_row = max(_pages_for(p + max(tails)) for p in prompts)
        cache = sa.KVCache(1, case["Hkv"], case["D"], G * R, per_row, G * R * (_pages_for(max(tails)) + 2) + G * per_row,
                           _kv_code(case))
        for g, n in enumerate(prompts):
            first = g * R
            cache.reserve(first, n)
            cache.append(0, None, kp[g:g + 1, :n].float(), vp[g:g + 1, :n].float(), seq_ids=[first])
            cache.commit(n, seqs=[first])
            for r in range(first + 1, first + R):
                cache.fork(r, first, n)
        for r, n in enumerate(tails):
            cache.reserve(r, prompts[r // R] + n)
            cache.append(0, None, ks[r:r + 1, :n].float(), vs[r:r + 1, :n].float(), seq_ids=[r])
            cache.commit(n, seqs=[r])
        need = cache.decode_shared_ws_bytes(G * R, case["Hq"])
        s.update(cache=cache, groups=[R] * G, out=torch.empty_like(s["q"]),
                 ws=torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda"))
    else:
        s.update(kp=kp, vp=vp, ks=ks, vs=vs, prompts=torch.tensor(prompts, device="cuda"),
                 tails=torch.tensor(tails, device="cuda"))
    return s


# ---------------------------------------------------------------- one pass: plain forms

def _weights(scores, seen):
    """Softmax over the last axis of the scores that are seen, and 0 elsewhere; a row that sees nothing is 0."""
    scores = scores.masked_fill(~seen, -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - m.masked_fill(m == -math.inf, 0.0))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-38)


def _plain_prefill_window(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    B, Hq, L, D = q.shape
    G = Hq // k.shape[1]
    i, j = torch.arange(L, device="cuda")[:, None], torch.arange(L, device="cuda")[None, :]
    seen = (j <= i) & ((i - j < c["window"]) | (j < c["sink"]))
    qf = q.float().reshape(B, -1, G, L, D)
    p = _weights(torch.matmul(qf, k.float()[:, :, None].transpose(-1, -2)) * s["scale"], seen)
    return torch.matmul(p, v.float()[:, :, None]).reshape(B, Hq, L, D).to(q.dtype)


def _plain_decode_window(s):
    c, q, lens = s["case"], s["q"], s["lens"][:, None]
    N, Hq, D = q.shape
    Hkv = c["Hkv"]
    sinks, back = torch.arange(c["sink"], device="cuda"), torch.arange(c["window"], device="cuda")
    start = (lens - c["window"]).clamp_min(0)
    idx = torch.cat([sinks.expand(N, -1), start + back], 1)
    seen = torch.cat([sinks < start, start + back < lens], 1)      # sinks inside the window count once
    idx = torch.where(seen, idx, 0)
    pages = torch.gather(s["table"], 1, idx // PAGE)
    k = s["k"][pages, :, idx % PAGE].float().transpose(1, 2)       # [N, Hkv, T, D]
    v = s["v"][pages, :, idx % PAGE].float().transpose(1, 2)
    p = _weights(torch.matmul(q.reshape(N, Hkv, -1, D), k.transpose(-1, -2)) * s["scale"], seen[:, None, None])
    return torch.matmul(p, v).reshape(N, Hq, D)


def _plain_decode_shared(s):
    c, q = s["case"], s["q"]
    N, Hq, D = q.shape
    G, R, Hkv = c["groups"], c["rows"], c["Hkv"]
    kp, vp, ks, vs = (s[n].float().transpose(1, 2) for n in ("kp", "vp", "ks", "vs"))   # [.., Hkv, T, D]
    P, S, rep = kp.shape[2], ks.shape[2], Hq // Hkv
    qg = q.reshape(G, R, Hkv, rep, D).transpose(1, 2).reshape(G, Hkv, R * rep, D)
    sp = torch.matmul(qg, kp.transpose(-1, -2)).reshape(G, Hkv, R, rep, P).transpose(1, 2).reshape(N, Hkv, rep, P)
    ss = torch.matmul(q.reshape(N, Hkv, rep, D), ks.transpose(-1, -2))
    in_prompt = (torch.arange(P, device="cuda") < s["prompts"][:, None]).repeat_interleave(R, 0)
    in_tail = torch.arange(S, device="cuda") < s["tails"][:, None]
    p = _weights(torch.cat([sp, ss], -1) * s["scale"], torch.cat([in_prompt, in_tail], 1)[:, None, None])
    pp = p[..., :P].reshape(G, R, Hkv, rep, P).transpose(1, 2).reshape(G, Hkv, R * rep, P)
    op = torch.matmul(pp, vp).reshape(G, Hkv, R, rep, D).transpose(1, 2).reshape(N, Hkv, rep, D)
    return (op + torch.matmul(p[..., P:], vs)).reshape(N, Hq, D)


def _plain_beam_select(s):
    c = s["case"]
    x = s["logits"].double()       # 64 bits: candidates of different beams lie close together
    m = x.amax(-1, keepdim=True)
    total = s["scores"].double()[..., None] + x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True)))
    best, at = torch.sort(total.reshape(c["groups"], -1), dim=-1, descending=True, stable=True)
    best, at = best[:, :c["select"]], at[:, :c["select"]]
    return {"scores": best.float(), "tokens": (at % c["vocab"]).int(), "beams": (at // c["vocab"]).int()}


# ---------------------------------------------------------------- one pass

def run(s):
    kind, c = s["case"]["kind"], s["case"]
    if not own:
        return {"prefill_window": _plain_prefill_window, "decode_window": _plain_decode_window,
                "decode_shared": _plain_decode_shared, "beam_select": _plain_beam_select}[kind](s)
    if kind == "prefill_window":
        return _package().prefill_window(s["q"], s["k"], s["v"], s["scale"], c["window"], c["sink"], out=s["out"])
    if kind == "decode_window":
        return s["cache"].decode_window(0, s["q"], s["scale"], c["window"], c["sink"], out=s["out"], ws=s["ws"])
    if kind == "decode_shared":
        return s["cache"].decode_shared(0, s["q"], s["scale"], s["groups"], out=s["out"], ws=s["ws"])
    scores, tokens, beams = _package().beam_select(s["logits"], s["scores"], c["select"], out=s["out"], ws=s["ws"])
    return {"scores": scores, "tokens": tokens, "beams": beams}


# ---------------------------------------------------------------- work

def _visible(n, window, sink):
    """Keys that the last of n tokens sees."""
    return min(n, window) + min(sink, max(0, n - window))


def work(case):
    kind = case["kind"]
    if kind == "beam_select":
        G, B, V, N = case["groups"], case["beams"], case["vocab"], case["select"]
        return {"bytes": 4 * G * B * (V + 1) + 12 * G * N, "flops": 4 * G * B * V}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if kind == "prefill_window":
        B, L, elem = case["B"], case["L"], 2 if case["dtype"] == "bf16" else 4
        keys = sum(_visible(i + 1, case["window"], case["sink"]) for i in range(L))
        return {"bytes": B * L * D * (2 * Hq + 2 * Hkv) * elem, "flops": 4 * B * Hq * D * keys}
    elem = 2 if case["kv"] == "bf16" else 4
    if kind == "decode_window":
        rows = case["B"]
        read = scored = sum(_visible(n, case["window"], case["sink"]) for n in _window_lengths(case))
    else:
        prompts, tails = _shared_lengths(case)
        rows, read = len(tails), sum(prompts) + sum(tails)
        scored = case["rows"] * sum(prompts) + sum(tails)
    return {"bytes": read * 2 * Hkv * D * elem + 8 * rows * Hq * D, "flops": 4 * Hq * D * scored}


# ---------------------------------------------------------------- the definitions in 64 bits

def _attend64(q, k, v, scale):
    """softmax(scale q k^T) v for one token: q [Hq, D], k and v [T, Hkv, D] -> [Hq, D]."""
    rep = q.shape[0] // k.shape[1]
    k, v = (x.double().repeat_interleave(rep, 1) for x in (k, v))
    w = torch.einsum("hd,thd->ht", q.double(), k) * scale
    w = torch.exp(w - w.max(1, keepdim=True).values)
    return torch.einsum("ht,thd->hd", w, v) / w.sum(1, keepdim=True)


def exact(case, seed):
    kind = case["kind"]
    if kind == "beam_select":
        logits, scores = (x.cpu().double() for x in _beam_inputs(case, seed))
        out = {"scores": [], "tokens": [], "beams": []}
        for rows, base in zip(logits, scores):
            total = (base[:, None] + torch.log_softmax(rows, -1)).reshape(-1)
            best = sorted(torch.topk(total, min(total.numel(), case["select"] + 8)).indices.tolist(),
                          key=lambda i: (-float(total[i]), i))[:case["select"]]
            out["scores"].append(total[best])
            out["tokens"].append(torch.tensor([i % case["vocab"] for i in best], dtype=torch.int32))
            out["beams"].append(torch.tensor([i // case["vocab"] for i in best], dtype=torch.int32))
        return {n: torch.stack(v) for n, v in out.items()}
    scale = 1.0 / math.sqrt(case["D"])
    if kind == "prefill_window":
        q, k, v = _prefill_inputs(case, seed)
        B, Hq, L, D = q.shape
        rep = Hq // k.shape[1]
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        for b in range(B):
            for at in range(0, L, 1024):     # queries [at, end) see keys [0, sink) and [at - window + 1, end)
                end = min(L, at + 1024)
                first = max(0, at - case["window"] + 1)
                keys = sorted(set(range(min(case["sink"], end))) | set(range(first, end)))
                kk = torch.tensor(keys, device="cuda")
                gap = torch.arange(at, end, device="cuda")[:, None] - kk[None]
                hidden = (gap < 0) | ((gap >= case["window"]) & (kk >= case["sink"])[None])
                for h in range(Hq):
                    w = q[b, h, at:end].double() @ k[b, h // rep][kk].double().T * scale
                    w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                    out[b, h, at:end] = w @ v[b, h // rep][kk].double()
        return out
    if kind == "decode_window":
        lens, lists, k, v = _window_layout(case, seed)
        q = _queries(case, seed, len(lens))
        rows = []
        for i, (n, pages) in enumerate(zip(lens, lists)):
            at = [t for t in range(n) if t < case["sink"] or t >= n - case["window"]]
            page, row = torch.tensor([pages[t // PAGE] for t in at]), torch.tensor([t % PAGE for t in at])
            rows.append(_attend64(q[i], k[page.cuda(), :, row.cuda()], v[page.cuda(), :, row.cuda()], scale))
        return torch.stack(rows)
    prompts, tails, (kp, vp, ks, vs) = _shared_tensors(case, seed)
    q = _queries(case, seed, len(tails))
    rows = []
    for i, n in enumerate(tails):
        g = i // case["rows"]
        k, v = (torch.cat([a[g, :prompts[g]], b[i, :n]]) for a, b in ((kp, ks), (vp, vs)))
        rows.append(_attend64(q[i], k, v, scale))
    return torch.stack(rows)
