"""The attention half of a decoder layer as measurable cases: rotary positions, attention
over packed prompts, attention over the paged key/value cache, and the cache's pages.

Each case is a dict of plain values. `prepare` makes what a program holds before the
call, `run` makes one pass: with `own` through the framework's entry points
(AttentionBackend, KvCache, Rope), without it in elementary torch operations in 32 bits.
`exact` gives the same outputs in 64 bits from the definitions, `work` counts what a
pass cannot do without.

Ops: rope (AttentionBackend.rope_device), prompt (AttentionBackend.prompt_device),
cached (AttentionBackend.cached_device), append (KvCache.append_device), fork
(KvCache.free_device, fork_device, extend_device), step (KvCache.compact_device,
extend_device, append_device, compact_device: one speculative step).
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # decode of one token at the Qwen3-A3B head shape: launch latency counts
        {"name": "rope_f32_t1", "op": "rope", "tokens": 1, "heads": 32, "kv_heads": 4, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "none", "factor": 1.0, "first": 4103, "in": "f32", "out": "f32"},
        # a long prompt's queries and keys, half of each head rotated in pairs, far positions of a stretched context
        {"name": "rope_yarn_t8191", "op": "rope", "tokens": 8191, "heads": 64, "kv_heads": 8, "dim": 128, "rotary": 64,
         "layout": "interleaved", "scaling": "yarn", "factor": 32.0, "first": 122000, "in": "f32", "out": "bf16"},
        # prefill of one long prompt
        {"name": "prompt_bf16_8192", "op": "prompt", "seqs": 1, "tokens": 8192, "pad": 0, "heads": 32, "kv_heads": 4,
         "dim": 128, "causal": True, "type": "bf16"},
        # prefill of many short prompts packed behind one another, an empty one among them, padded rows behind
        {"name": "prompt_f16_ragged", "op": "prompt", "seqs": 23, "tokens": 4099, "pad": 61, "heads": 16, "kv_heads": 16,
         "dim": 80, "causal": True, "type": "f16"},
        # an encoder's pass (every token sees every token) in the framework's own float activations
        {"name": "prompt_f32_both", "op": "prompt", "seqs": 3, "tokens": 1531, "pad": 0, "heads": 8, "kv_heads": 2,
         "dim": 192, "causal": False, "type": "f32"},
        # decode of one token early in a chat: latency
        {"name": "cached_f32_b1", "op": "cached", "seqs": 1, "short": 517, "long": 517, "rows": 1, "tree": False,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 16, "type": "f32", "cache": "bf16"},
        # decode of 32 sequences of very different lengths
        {"name": "cached_bf16_b32", "op": "cached", "seqs": 32, "short": 301, "long": 8192, "rows": 1, "tree": False,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 16, "type": "bf16", "cache": "bf16"},
        # decode at the end of two very long contexts
        {"name": "cached_f16_long", "op": "cached", "seqs": 2, "short": 98765, "long": 131072, "rows": 1, "tree": False,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 64, "type": "f16", "cache": "f16"},
        # verifying trees of up to 64 drafted tokens for 8 sequences
        {"name": "cached_tree_b8", "op": "cached", "seqs": 8, "short": 2000, "long": 7001, "rows": 64, "tree": True,
         "heads": 32, "kv_heads": 4, "dim": 128, "page": 16, "type": "bf16", "cache": "bf16"},
        # the keys and values of one decode step of 32 sequences into the cache, queries rotated beside them
        {"name": "append_b32", "op": "append", "seqs": 32, "short": 301, "long": 8192, "rows": 1, "heads": 32,
         "kv_heads": 4, "dim": 128, "rotary": 128, "layout": "half", "page": 16, "type": "f32", "cache": "bf16"},
        # two branches forked from each of 24 sequences, every layer's last page copied on their first token
        {"name": "fork_24x2", "op": "fork", "seqs": 24, "branches": 2, "short": 40, "long": 1500, "grow": 1, "layers": 24,
         "kv_heads": 4, "dim": 128, "page": 16, "cache": "bf16"},
        # one speculative step's cache work: the last round's tokens taken back, drafts written, the accepted kept
        {"name": "step_b16", "op": "step", "seqs": 16, "short": 100, "long": 3000, "drafts": 48, "kept": 6, "layers": 4,
         "kv_heads": 4, "dim": 128, "page": 16, "type": "bf16", "cache": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    return kv * rng.choice([1, 2, 4, 5, 7, 8, 16]), kv


def draw(rng):
    u = rng.random()
    while True:
        heads, kv = _heads(rng)
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
        kind = rng.choice(["f32", "f16", "bf16", "bf16"])
        if u < 0.2:
            c = {"op": "rope", "tokens": _log_int(rng, 1, 8192), "heads": heads, "kv_heads": kv, "dim": dim,
                 "rotary": rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                 "layout": rng.choice(["half", "interleaved"]),
                 "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.0, 32.0]),
                 "first": _log_int(rng, 1, 1 << 20), "in": kind, "out": rng.choice([kind, "bf16"])}
            if c["tokens"] * (heads + kv) * dim <= 8191 * 72 * 128:
                return c
        elif u < 0.5:
            c = {"op": "prompt", "seqs": _log_int(rng, 1, 48), "tokens": _log_int(rng, 5, 8192), "pad": rng.choice([0, 0, 37]),
                 "heads": heads, "kv_heads": kv, "dim": dim, "causal": rng.random() < 0.8, "type": kind}
            slow = 8 if kind == "f32" else 1
            pairs = c["tokens"] ** 2 * heads * slow
            if max(pairs, pairs * dim * (1 if c["causal"] else 2) // 128) <= 8192 ** 2 * 32:
                return c
        elif u < 0.8:
            tree = rng.random() < 0.4
            short = _log_int(rng, 70, 20000)
            c = {"op": "cached", "seqs": _log_int(rng, 1, 64), "short": short,
                 "long": min(131072, int(short * rng.uniform(1, 12))),
                 "rows": rng.randint(2, 64) if tree else rng.choice([1, 1, 1, 2, 5, 70]), "tree": tree,
                 "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([8, 16, 16, 32, 64, 256]),
                 "type": kind, "cache": rng.choice([kind, "f16", "bf16"]) if kind == "f32" else kind}
            if (c["seqs"] * c["long"] * kv * dim <= 1 << 28 and c["seqs"] * c["long"] * heads * c["rows"] <= 1 << 28):
                return c
        elif u < 0.88:
            c = {"op": "append", "seqs": _log_int(rng, 1, 64), "short": 80, "long": _log_int(rng, 80, 8192),
                 "rows": rng.choice([1, 1, 7, 64]), "heads": heads, "kv_heads": kv, "dim": dim,
                 "rotary": rng.choice([dim, dim // 2]), "layout": rng.choice(["half", "interleaved"]),
                 "page": rng.choice([8, 16, 32, 64]), "type": kind, "cache": rng.choice([kind, "f16"])}
            if c["seqs"] * c["long"] * kv * dim <= 1 << 27:
                return c
        elif u < 0.94:
            c = {"op": "fork", "seqs": _log_int(rng, 1, 48), "branches": rng.randint(1, 4), "short": 1,
                 "long": _log_int(rng, 2, 1500), "grow": _log_int(rng, 1, 40), "layers": rng.randint(1, 24),
                 "kv_heads": kv, "dim": dim, "page": rng.choice([8, 16, 32, 64]), "cache": kind}
            if _pool_elements(c) <= 1 << 28:
                return c
        else:
            drafts = rng.randint(1, 64)
            c = {"op": "step", "seqs": _log_int(rng, 1, 48), "short": 70, "long": _log_int(rng, 70, 4000), "drafts": drafts,
                 "kept": rng.randint(0, drafts), "layers": rng.randint(1, 4), "kv_heads": kv, "dim": dim,
                 "page": rng.choice([8, 16, 32, 64]), "type": kind, "cache": kind}
            if _pool_elements(c) <= 1 << 28:
                return c


# ------------------------------------------------------------------ case plans
def _lengths(c):
    """The sequences' lengths, spread from the shortest to the longest over the logarithm, in mixed order."""
    n, lo, hi = c["seqs"], c["short"], c["long"]
    lens = [hi if n == 1 else int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    random.Random(n * 1009 + lo + hi).shuffle(lens)
    return lens


def _packed(c):
    """Ragged lengths of `seqs` packed prompts that add up to `tokens`; one of several is empty, one a single token."""
    n, total = c["seqs"], c["tokens"]
    if n == 1:
        return [total]
    r = random.Random(n * 7919 + total)
    w = [0.02 + r.random() ** 2 for _ in range(n)]
    lens = [int(total * x / sum(w)) for x in w]
    lens[n // 2] = 0
    if n > 2:
        lens[n // 3] = min(1, total)
    spare = total - sum(lens)
    lens[-1] = max(0, lens[-1] + spare)
    while sum(lens) > total:
        lens[lens.index(max(lens))] -= 1
    return lens


def _rows(c):
    """Query rows of each cached sequence: all alike for a step of one token, ragged up to `rows` otherwise."""
    n, m = c["seqs"], c["rows"]
    return [m if m == 1 or i % 3 == 0 else 1 + (m * (i % 7 + 1)) // 8 for i in range(n)]


def _page_count(c):
    p = c["page"]
    if c["op"] == "fork":
        kept = sum(-(-n // p) for n in _lengths(c))
        return kept + c["seqs"] * c["branches"] * (2 + c["grow"] // p) + 8
    if c["op"] == "step":
        return sum(-(-(n + c["kept"]) // p) + 1 + c["drafts"] // p for n in _lengths(c)) + 8
    return sum(-(-n // p) for n in _lengths(c)) + 5


def _pool_elements(c):
    return c.get("layers", 1) * _page_count(c) * c["kv_heads"] * c["page"] * c["dim"]


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _randn(g, *shape, kind="f32"):
    return torch.randn(shape, device="cuda", generator=g).to(TYPES[kind])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cumulative(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _cache(c, g, seqs, held):
    """A paged cache whose first sequences hold `held` tokens each, in pages of a mixed order."""
    p, n_pages = c["page"], _page_count(c)
    top = -(-(max(held) + c.get("drafts", 0) + c.get("grow", 0)) // p) + 1
    pages = [-(-n // p) for n in held]
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((seqs, top), -1, dtype=torch.int32, device="cuda")
    start = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[start:start + n]
        start += n
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[order[:start].long()] = 1
    shape = (c.get("layers", 1), n_pages, c["kv_heads"], p, c["dim"])
    return {"k": _randn(g, *shape, kind=c["cache"]), "v": _randn(g, *shape, kind=c["cache"]), "table": table,
            "lens": _ints(held + [0] * (seqs - len(held))), "refs": refs}


def _tree_masks(rows, seed):
    """For each row of each sequence the bits of its ancestors and itself among the drafts."""
    r, masks = random.Random(seed * 31 + 5), []
    for n in rows:
        own_bits = []
        for i in range(n):
            parent = r.randint(max(0, i - 9), i) - 1  # one before the first draft: the cached context itself
            own_bits.append((own_bits[parent] if parent >= 0 else 0) | 1 << i)
        masks += [b - (1 << 64) if b >> 63 else b for b in own_bits]
    return torch.tensor(masks, dtype=torch.int64, device="cuda")


def _inputs(c, seed):
    g, op = _generator(seed), c["op"]
    if op == "rope":
        t = c["tokens"]
        pos = c["first"] + torch.arange(t, device="cuda") + int(seed) % 97
        return {"q": _randn(g, t, c["heads"], c["dim"], kind=c["in"]), "k": _randn(g, t, c["kv_heads"], c["dim"], kind=c["in"]),
                "pos": pos.to(torch.int32)}
    if op == "prompt":
        t = c["tokens"] + c["pad"]
        return {"q": _randn(g, t, c["heads"], c["dim"], kind=c["type"]), "k": _randn(g, t, c["kv_heads"], c["dim"], kind=c["type"]),
                "v": _randn(g, t, c["kv_heads"], c["dim"], kind=c["type"]), "cu": _ints(_cumulative(_packed(c)))}
    lens = _lengths(c)
    if op in ("cached", "append"):
        rows = [min(a, b) for a, b in zip(_rows(c), lens)]
        d = {"cache": _cache(c, g, c["seqs"], lens), "cu": _ints(_cumulative(rows)),
             "seqs": torch.randperm(c["seqs"], device="cuda", generator=g).to(torch.int32) if op == "append"
             else torch.arange(c["seqs"], device="cuda", dtype=torch.int32)}
        n = sum(rows)
        d["q"] = _randn(g, n, c["heads"], c["dim"], kind=c["type"])
        if op == "cached":
            d["tree"] = _tree_masks(rows, seed) if c["tree"] else None
        else:
            if c["rows"] > 1:  # every sequence is long enough for the longest run
                d["seqs"] = torch.arange(c["seqs"], device="cuda", dtype=torch.int32)
            d["k"], d["v"] = (_randn(g, n, c["kv_heads"], c["dim"], kind=c["type"]) for _ in range(2))
            d["pos"] = torch.randint(0, 1 << 17, (n,), device="cuda", generator=g).to(torch.int32)
        return d
    n = c["seqs"]
    if op == "fork":
        b = n * c["branches"]
        return {"cache": _cache(c, g, n + b, lens), "src": _ints([i % n for i in range(b)]), "dst": _ints(list(range(n, n + b))),
                "counts": _ints([c["grow"]] * b)}
    r = random.Random(int(seed) * 17 + 3)
    keep = [sorted(r.sample(range(c["drafts"]), c["kept"])) + [-1] * (c["drafts"] - c["kept"]) for _ in range(n)]
    rows = n * c["drafts"]
    return {"cache": _cache(c, g, n, [x + c["kept"] for x in lens]), "seqs": _ints(list(range(n))), "old": _ints([c["kept"]] * n),
            "none": _ints([0] * n), "drafts": _ints([c["drafts"]] * n), "kept": _ints([c["kept"]] * n), "keep": _ints(keep),
            "cu": _ints(_cumulative([c["drafts"]] * n)), "k": _randn(g, c["layers"], rows, c["kv_heads"], c["dim"], kind=c["type"]),
            "v": _randn(g, c["layers"], rows, c["kv_heads"], c["dim"], kind=c["type"])}


def prepare(case, seed):
    c, d = case, _inputs(case, seed)
    s = {"case": c, "in": d}
    if c["op"] == "rope":
        s["q_out"], s["k_out"] = (torch.empty(d[x].shape, dtype=TYPES[c["out"]], device="cuda") for x in ("q", "k"))
    elif c["op"] in ("prompt", "cached"):
        s["out"] = torch.zeros_like(d["q"])  # rows behind the last sequence stay as they are
        s["lse"] = torch.zeros(d["q"].shape[:2], dtype=torch.float32, device="cuda")
    elif c["op"] == "append":
        s["q_out"] = torch.empty_like(d["q"])
    if own:
        s["rope"] = _own_rope(c) if "rotary" in c else None
        s["cache"] = _own_cache(c, d["cache"]) if "cache" in d else None
    torch.cuda.synchronize()
    return s


# ----------------------------------------------------------- the framework's calls
@functools.lru_cache(maxsize=None)
def _backend():
    from objeta_amd import AttentionBackend, HipBackend
    be = HipBackend(0, 1)
    return be, AttentionBackend(be)


_THETA, _ORIGINAL = 1.0e6, 4096


def _own_rope(c):
    from objeta_amd import Rope
    return Rope(c["rotary"], theta=_THETA, layout=c["layout"], scaling=c.get("scaling", "none"), factor=c.get("factor", 1.0),
                original_context=_ORIGINAL)


def _own_cache(c, t):
    from objeta_amd import KvCache
    layers, pages, kv, page, dim = t["k"].shape
    return KvCache(_backend()[0], layers, pages, kv, page, dim, t["table"].shape[0], t["table"].shape[1], dtype=c["cache"],
                   d_k=t["k"].data_ptr(), d_v=t["v"].data_ptr(), d_page_table=t["table"].data_ptr(),
                   d_seq_lens=t["lens"].data_ptr(), d_ref_counts=t["refs"].data_ptr())


def _run_own(s):
    att, c, d, at = _backend()[1], s["case"], s["in"], torch.Tensor.data_ptr
    op, cache = c["op"], s["cache"]
    if op == "rope":
        att.rope_device(s["rope"], at(d["pos"]), c["tokens"], c["dim"], at(d["q"]), at(s["q_out"]), c["heads"], at(d["k"]),
                        at(s["k_out"]), c["kv_heads"], dtype=c["in"], out_dtype=c["out"])
        return s["q_out"], s["k_out"]
    if op == "prompt":
        att.prompt_device(c["type"], at(d["q"]), at(d["k"]), at(d["v"]), at(s["out"]), c["heads"], c["kv_heads"], c["dim"],
                          c["tokens"] + c["pad"], at(d["cu"]), c["seqs"], causal=c["causal"], d_lse=at(s["lse"]))
        return s["out"], s["lse"]
    if op == "cached":
        att.cached_device(cache, 0, at(d["seqs"]), at(d["cu"]), c["seqs"], d["q"].shape[0], c["rows"], c["long"], c["type"],
                          at(d["q"]), at(s["out"]), c["heads"], d_tree=None if d["tree"] is None else at(d["tree"]),
                          d_lse=at(s["lse"]))
        return s["out"], s["lse"]
    if op == "append":
        cache.append_device(0, at(d["seqs"]), at(d["cu"]), c["seqs"], d["q"].shape[0], c["type"], at(d["k"]), at(d["v"]),
                            rope=s["rope"], d_positions=at(d["pos"]), d_q=at(d["q"]), d_q_out=at(s["q_out"]), n_q_heads=c["heads"])
        return s["q_out"], d["cache"]["k"], d["cache"]["v"]
    if op == "fork":
        n = d["dst"].numel()
        cache.free_device(at(d["dst"]), n)
        cache.fork_device(at(d["src"]), at(d["dst"]), n)
        cache.extend_device(at(d["dst"]), at(d["counts"]), n)
    else:
        n, rows = c["seqs"], c["seqs"] * c["drafts"]
        cache.compact_device(at(d["seqs"]), at(d["old"]), at(d["keep"]), at(d["none"]), n, c["drafts"])
        cache.extend_device(at(d["seqs"]), at(d["drafts"]), n)
        for layer in range(c["layers"]):
            cache.append_device(layer, at(d["seqs"]), at(d["cu"]), n, rows, c["type"], at(d["k"][layer]), at(d["v"][layer]))
        cache.compact_device(at(d["seqs"]), at(d["drafts"]), at(d["keep"]), at(d["kept"]), n, c["drafts"])
    t = d["cache"]
    return t["table"], t["lens"], t["refs"], t["k"], t["v"]


# ------------------------------------------------------------------ plain forms
def _frequencies(c):
    """Radians per position of each pair, in 64 bits, and the factor on cosines and sines."""
    r, scaling, factor = c["rotary"], c.get("scaling", "none"), c.get("factor", 1.0)
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    theta = _THETA * (factor ** (r / (r - 2)) if scaling == "ntk" and r > 2 else 1.0)
    f = torch.pow(theta, -2.0 * i / r)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    low, high = ((r * math.log(_ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(_THETA))) for turns in (32.0, 1.0))
    low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _rotate(x, pos, c):
    """x [tokens][heads][dim] rotated, in 32 bits; the angles in 64, which far positions need."""
    r = c["rotary"]
    f, amp = _frequencies(c)
    a = pos.double()[:, None] * f
    cos, sin = (torch.cos(a) * amp).float()[:, None], (torch.sin(a) * amp).float()[:, None]
    x = x.float()
    if c["layout"] == "half":
        u, w = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat((u * cos - w * sin, u * sin + w * cos), -1)
    else:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack((u * cos - w * sin, u * sin + w * cos), -1).flatten(-2)
    return torch.cat((y, x[..., r:]), -1)


def _attend(q, k, v, seen, dim):
    """q [.., rows, dim], k and v [.., keys, dim] in 32 bits, `seen` broadcast over the scores: (out, lse)."""
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    s = torch.where(seen, s, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (top + torch.log(total)).squeeze(-1)


def _plain_prompt(s):
    c, d = s["case"], s["in"]
    t, kv, group = d["q"].shape[0], c["kv_heads"], c["heads"] // c["kv_heads"]
    at = torch.arange(t, device="cuda", dtype=torch.int32)
    of = torch.searchsorted(d["cu"], at, right=True)  # the sequence of a token; one past the last: padding
    seen = of[:, None] == of[None, :]
    if c["causal"]:
        seen = seen & (at[None, :] <= at[:, None])
    q = d["q"].float().view(t, kv, group, -1).permute(1, 2, 0, 3)
    k, v = (d[x].float().permute(1, 0, 2)[:, None].expand(-1, group, -1, -1) for x in ("k", "v"))
    out, lse = _attend(q, k, v, seen, c["dim"])
    real = of <= c["seqs"]
    out = torch.where(real[None, None, :, None], out, torch.zeros_like(out))
    lse = torch.where(real, lse, torch.zeros_like(lse))
    return out.permute(2, 0, 1, 3).reshape(d["q"].shape).to(d["q"].dtype), lse.permute(2, 0, 1).reshape(t, -1)


def _plain_cached(s):
    c, d = s["case"], s["in"]
    t, kv, group, p = d["cache"], c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    n, rows = c["seqs"], c["rows"]
    seqs, cu = d["seqs"].long(), d["cu"].long()
    pages = t["table"][seqs][:, :-(-c["long"] // p)].clamp(min=0).long()
    k, v = (t[x][0][pages].float().permute(0, 2, 1, 3, 4).reshape(n, kv, -1, c["dim"]) for x in ("k", "v"))
    i = torch.arange(rows, device="cuda")
    at = cu[:-1, None] + i
    real = at < cu[1:, None]
    at = at.clamp(max=d["q"].shape[0] - 1)
    q = d["q"].float()[at].view(n, rows, kv, group, -1).permute(0, 2, 3, 1, 4).reshape(n, kv, group * rows, -1)
    slot = torch.arange(k.shape[2], device="cuda")
    lens = t["lens"].long()[seqs][:, None, None]
    base = lens - (cu[1:] - cu[:-1])[:, None, None]
    if d["tree"] is None:
        seen = slot <= base + i[:, None]
    else:
        bit = (slot - base).clamp(0, 63)
        seen = (slot < base) | ((d["tree"][at][..., None] >> bit) & 1 == 1) & (slot < lens)
    seen = seen[:, None, None].expand(-1, kv, group, -1, -1).reshape(n, kv, group * rows, -1)
    out, lse = _attend(q, k, v, seen, c["dim"])
    out = out.view(n, kv, group, rows, -1).permute(0, 3, 1, 2, 4).reshape(n, rows, c["heads"], -1)[real]
    lse = lse.view(n, kv, group, rows).permute(0, 3, 1, 2).reshape(n, rows, c["heads"])[real]
    return out.to(d["q"].dtype), lse


def _places(t, d, p):
    """(page, row in it) of each new row: a sequence's rows are its last ones."""
    cu, lens = d["cu"].long(), t["lens"].long()
    at = torch.arange(d["k"].shape[-3], device="cuda")
    b = torch.searchsorted(cu, at, right=True) - 1
    seq = d["seqs"].long()[b]
    slot = lens[seq] - cu[b + 1] + at
    return t["table"][seq, slot // p].long(), slot % p


def _plain_append(s):
    c, d = s["case"], s["in"]
    t = d["cache"]
    page, row = _places(t, d, c["page"])
    t["k"][0][page, :, row] = _rotate(d["k"], d["pos"], c).to(t["k"].dtype)
    t["v"][0][page, :, row] = d["v"].to(t["v"].dtype)
    return _rotate(d["q"], d["pos"], c).to(d["q"].dtype), t["k"], t["v"]


def _release(t, pages):
    held = pages >= 0
    t["refs"].index_add_(0, pages.clamp(min=0).long().flatten(), -held.int().flatten())


def _plain_free(t, seqs):
    _release(t, t["table"][seqs])
    t["table"][seqs] = -1
    t["lens"][seqs] = 0


def _plain_fork(t, src, dst):
    pages, lens = t["table"][src], t["lens"][src]
    _release(t, t["table"][dst])
    t["refs"].index_add_(0, pages.clamp(min=0).long().flatten(), (pages >= 0).int().flatten())
    t["table"][dst], t["lens"][dst] = pages, lens


def _plain_extend(t, seqs, counts, p):
    lens, counts = t["lens"].long()[seqs], counts.long()
    have, want = -(-lens // p), -(-(lens + counts) // p)
    part = (lens % p != 0) & (counts > 0)
    last = torch.where(part, t["table"][seqs, lens // p].long(), -1 - torch.arange(lens.numel(), device="cuda"))
    before = (last[:, None] == last[None, :]).tril(-1).sum(1)
    copy = part & (t["refs"].long()[last.clamp(min=0)] - before > 1)
    need = want - have + copy.long()
    start = need.cumsum(0) - need
    free = torch.nonzero(t["refs"] == 0).flatten()
    entry = torch.repeat_interleave(torch.arange(lens.numel(), device="cuda"), need)
    j = torch.arange(entry.numel(), device="cuda") - start[entry]
    new = free[:entry.numel()]
    t["table"][seqs[entry], have[entry] + j - copy[entry].long()] = new.int()
    t["refs"][new] = 1
    old, to, filled = last[copy], free[start[copy]], (lens % p)[copy]
    t["refs"].index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    some = torch.arange(p, device="cuda") < filled[:, None]
    for x in ("k", "v"):
        t[x][:, to] = torch.where(some[None, :, None, :, None], t[x][:, old], t[x][:, to])
    t["lens"][seqs] = (lens + counts).int()


def _plain_compact(t, seqs, drafts, keep, kept, p):
    base = t["lens"].long()[seqs] - drafts.long()
    kept = kept.long()
    j = torch.arange(keep.shape[1], device="cuda")
    entry, j = torch.nonzero(j < kept[:, None], as_tuple=True)
    src, dst = base[entry] + keep.long()[entry, j], base[entry] + j
    rows = t["table"][seqs[entry]].long()
    one = torch.arange(entry.numel(), device="cuda")
    for x in ("k", "v"):
        t[x][:, rows[one, dst // p], :, dst % p] = t[x][:, rows[one, src // p], :, src % p]
    held = t["table"][seqs]
    past = torch.arange(held.shape[1], device="cuda") >= (-(-(base + kept) // p))[:, None]
    _release(t, torch.where(past, held, -1))
    t["table"][seqs] = torch.where(past, -1, held)
    t["lens"][seqs] = (base + kept).int()


def _plain_pages(s):
    c, d = s["case"], s["in"]
    t, p = d["cache"], c["page"]
    if c["op"] == "fork":
        src, dst = d["src"].long(), d["dst"].long()
        _plain_free(t, dst)
        _plain_fork(t, src, dst)
        _plain_extend(t, dst, d["counts"], p)
    else:
        seqs = d["seqs"].long()
        _plain_compact(t, seqs, d["old"], d["keep"], d["none"], p)
        _plain_extend(t, seqs, d["drafts"], p)
        page, row = _places(t, d, p)
        t["k"][:, page, :, row] = d["k"].permute(1, 0, 2, 3).to(t["k"].dtype)
        t["v"][:, page, :, row] = d["v"].permute(1, 0, 2, 3).to(t["v"].dtype)
        _plain_compact(t, seqs, d["drafts"], d["keep"], d["kept"], p)
    return t["table"], t["lens"], t["refs"], t["k"], t["v"]


def run(state):
    if own:
        return _run_own(state)
    c, d = state["case"], state["in"]
    if c["op"] == "rope":
        return tuple(_rotate(d[x], d["pos"], c).to(TYPES[c["out"]]) for x in ("q", "k"))
    if c["op"] == "prompt":
        return _plain_prompt(state)
    if c["op"] == "cached":
        return _plain_cached(state)
    if c["op"] == "append":
        return _plain_append(state)
    return _plain_pages(state)


# ------------------------------------------------------------------------ work
def work(case):
    c, op = case, case["op"]
    if op == "rope":
        n = c["tokens"] * (c["heads"] + c["kv_heads"])
        return {"bytes": n * c["dim"] * (SIZES[c["in"]] + SIZES[c["out"]]) + 4 * c["tokens"], "flops": 3 * n * c["rotary"]}
    if op == "prompt":
        lens = _packed(c)
        t = sum(lens)
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lens)
        return {"bytes": t * c["dim"] * (2 * c["heads"] + 2 * c["kv_heads"]) * SIZES[c["type"]] + 4 * t * c["heads"],
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    lens, row = _lengths(c), c["kv_heads"] * c["dim"]
    if op in ("cached", "append"):
        rows = [min(a, b) for a, b in zip(_rows(c), lens)]
        q = sum(rows) * c["heads"] * c["dim"] * 2 * SIZES[c["type"]]
        if op == "append":
            return {"bytes": q + sum(rows) * row * 2 * (SIZES[c["type"]] + SIZES[c["cache"]]),
                    "flops": 3 * sum(rows) * (c["heads"] + c["kv_heads"]) * c["rotary"]}
        pairs = sum(r * (n - r) + r * (r + 1) // 2 for r, n in zip(rows, lens))
        return {"bytes": q + sum(rows) * c["heads"] * 4 + sum(lens) * row * 2 * SIZES[c["cache"]] + sum(-(-n // c["page"]) for n in lens) * 4,
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    size, p = SIZES[c["cache"]], c["page"]
    if op == "fork":
        copied = sum(n % p for n in lens) * c["branches"]
        entries = sum(-(-n // p) for n in lens) * c["branches"]
        return {"bytes": copied * row * 4 * size * c["layers"] + entries * 24 + _page_count(c) * 4, "flops": 0}
    rows = c["seqs"] * c["drafts"]
    return {"bytes": c["layers"] * row * (rows * 2 * (SIZES[c["type"]] + size) + c["seqs"] * c["kept"] * 4 * size) + _page_count(c) * 4,
            "flops": 0}


# ---------------------------------------------------------------- 64-bit results
def _exact_rope(x, pos, c):
    x, half = x.double().clone(), c["layout"] == "half"
    r, scaling, factor = c["rotary"], c.get("scaling", "none"), c.get("factor", 1.0)
    amp, y = 1.0, x.clone()
    for i in range(r // 2):
        w = _THETA ** (-2.0 * i / r)
        if scaling == "linear":
            w /= factor
        elif scaling == "ntk" and r > 2:
            w = (_THETA * factor ** (r / (r - 2.0))) ** (-2.0 * i / r)
        elif scaling == "yarn":
            def index(turns):
                return r * math.log(_ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(_THETA))
            low, high = max(math.floor(index(32.0)), 0), min(math.ceil(index(1.0)), r - 1)
            blend = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            w, amp = w * (1 - blend) + w / factor * blend, 0.1 * math.log(factor) + 1.0
        a = pos.double() * w
        e = torch.polar(torch.full_like(a, amp), a)[:, None]
        u, v = (i, i + r // 2) if half else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., u], x[..., v]) * e
        y[..., u], y[..., v] = z.real, z.imag
    return y


def _exact_rows(q, k, v, seen):
    """One head in 64 bits: q [rows][dim] against k, v [keys][dim]."""
    s = (q.double() @ k.double().T) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~seen, float("-inf"))
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    return w @ v.double(), lse


def _exact_prompt(c, d):
    out, lse = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda"), torch.zeros(d["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for n in _packed(c):
        seen = torch.ones((n, n), dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = seen.tril()
        for h in range(c["heads"] if n else 0):
            kv = h * c["kv_heads"] // c["heads"]
            out[at:at + n, h], lse[at:at + n, h] = _exact_rows(d["q"][at:at + n, h], d["k"][at:at + n, kv], d["v"][at:at + n, kv], seen)
        at += n
    return out, lse


def _exact_cached(c, d):
    t, out = d["cache"], torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(d["q"].shape[:2], dtype=torch.float64, device="cuda")
    cu, table, lens = d["cu"].tolist(), t["table"].tolist(), t["lens"].tolist()
    tree = None if d["tree"] is None else d["tree"].tolist()
    for b, seq in enumerate(d["seqs"].tolist()):
        n, lo, hi = lens[seq], cu[b], cu[b + 1]
        pages = torch.tensor([x for x in table[seq] if x >= 0], device="cuda")
        k, v = (t[x][0, pages].transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :n] for x in ("k", "v"))
        seen = torch.ones((hi - lo, n), dtype=torch.bool, device="cuda")
        base = n - (hi - lo)
        for i in range(hi - lo):
            if tree is None:
                seen[i, base + i + 1:] = False
            else:
                seen[i, base:] = torch.tensor([bool(tree[lo + i] >> j & 1) for j in range(hi - lo)], device="cuda")
        for h in range(c["heads"]):
            kv = h * c["kv_heads"] // c["heads"]
            out[lo:hi, h], lse[lo:hi, h] = _exact_rows(d["q"][lo:hi, h], k[kv], v[kv], seen)
    return out, lse


def _exact_append(c, d):
    t = d["cache"]
    k, v = t["k"].double(), t["v"].double()
    new = _exact_rope(d["k"], d["pos"], c)
    cu, table, lens, p = d["cu"].tolist(), t["table"].tolist(), t["lens"].tolist(), c["page"]
    for b, seq in enumerate(d["seqs"].tolist()):
        for r in range(cu[b], cu[b + 1]):
            slot = lens[seq] - cu[b + 1] + r
            page = table[seq][slot // p]
            k[0, page, :, slot % p], v[0, page, :, slot % p] = new[r], d["v"][r].double()
    return _exact_rope(d["q"], d["pos"], c), k, v


def _exact_pages(c, d):
    """The page operations one after the other on the host's lists."""
    t, p = d["cache"], c["page"]
    k, v = t["k"].double(), t["v"].double()
    table = [[x for x in row if x >= 0] for row in t["table"].tolist()]
    lens, refs, width = t["lens"].tolist(), t["refs"].tolist(), t["table"].shape[1]

    def cut(s, n):
        for x in table[s][-(-n // p):]:
            refs[x] -= 1
        table[s], lens[s] = table[s][:-(-n // p)], n

    def take():
        x = refs.index(0)
        refs[x] = 1
        return x

    def grow(todo):
        for s, count in todo:
            if count and lens[s] % p and refs[table[s][-1]] > 1:
                old, r = table[s][-1], lens[s] % p
                table[s][-1] = take()
                refs[old] -= 1
                for x in (k, v):
                    x[:, table[s][-1], :, :r] = x[:, old, :, :r]
            lens[s] += count
            while len(table[s]) * p < lens[s]:
                table[s].append(take())

    if c["op"] == "fork":
        dst = d["dst"].tolist()
        for s in dst:
            cut(s, 0)
        for a, b in zip(d["src"].tolist(), dst):
            table[b], lens[b] = list(table[a]), lens[a]
            for x in table[b]:
                refs[x] += 1
        grow([(s, c["grow"]) for s in dst])
    else:
        for s in range(c["seqs"]):
            cut(s, lens[s] - c["kept"])
        grow([(s, c["drafts"]) for s in range(c["seqs"])])
        for s, keep in enumerate(d["keep"].tolist()):
            base = lens[s] - c["drafts"]
            for i in range(c["drafts"]):
                page, row = table[s][(base + i) // p], (base + i) % p
                k[:, page, :, row], v[:, page, :, row] = d["k"][:, s * c["drafts"] + i].double(), d["v"][:, s * c["drafts"] + i].double()
            for j in range(c["kept"]):
                a, b = base + keep[j], base + j
                for x in (k, v):
                    x[:, table[s][b // p], :, b % p] = x[:, table[s][a // p], :, a % p]
            cut(s, base + c["kept"])
    rows = [r + [-1] * (width - len(r)) for r in table]
    return _ints(rows), _ints(lens), _ints(refs), k, v


def exact(case, seed):
    c, d = case, _inputs(case, seed)
    if c["op"] == "rope":
        return tuple(_exact_rope(d[x], d["pos"], c) for x in ("q", "k"))
    return {"prompt": _exact_prompt, "cached": _exact_cached, "append": _exact_append, "fork": _exact_pages, "step": _exact_pages}[c["op"]](c, d)
