"""The operators of checking drafted tokens over a paged 4-bit KV cache, as cases that can be timed and
compared: each in its plain form (elementary torch operations) and, with `own`, as a user calls it.

  rope     PagedKV4.append_rope: rows normed, rotated and written into 4-bit pages, and .read of what they stand for
  tree     PagedKV4.attend_tree: trees of drafted tokens over the slots' pages
  verify   verify_draft: which drafted tokens the target keeps, and the token that follows them
  keep     PagedKV4.keep: the kept rows moved together in all layers, the rest dropped
  round    draft_tree, append_rope and attend_tree of one layer: what a layer of a checking pass does

The cache format is the one that include/sx8_paged.h documents; both forms work on its bytes.
Heads are those of the decoder of bench.py (32 query heads over 8 of 128, 151936 tokens) and a few other groupings.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
GROUP = 64                       # values that share a scale and a minimum
SEVENTH = float(np.float32(1.0) / np.float32(15.0))     # 1/15 as a float32
EPS = 1e-6


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # a token of each of 64 conversations, norms of the decoder's heads included
        {"name": "rope_step", "kind": "rope", "n": 64, "lo": 40, "hi": 2000, "mix": 1, "new": 1, "tree": False, "nh": 32,
         "nk": 8, "hd": 128, "rot": 128, "inter": False, "norm": True, "pt": 64, "type": "fp16"},
        # prompts of different lengths packed into one pass, a quarter of the head rotated in interleaved pairs
        {"name": "rope_prompt", "kind": "rope", "n": 9, "lo": 200, "hi": 2000, "mix": 2, "new": 0, "tree": False, "nh": 32,
         "nk": 8, "hd": 128, "rot": 32, "inter": True, "norm": False, "pt": 64, "type": "bf16"},
        # one conversation, eight drafted tokens: the smallest attention call
        {"name": "tree_one", "kind": "tree", "n": 1, "lo": 700, "hi": 700, "mix": 3, "new": 8, "nh": 32, "nk": 8,
         "hd": 128, "pt": 64, "type": "fp16"},
        # 24 conversations of very different lengths, up to 24 drafted tokens each
        {"name": "tree_batch", "kind": "tree", "n": 24, "lo": 100, "hi": 8000, "mix": 4, "new": -24, "nh": 32, "nk": 8,
         "hd": 128, "pt": 64, "type": "fp16"},
        # wide trees of 64 tokens
        {"name": "tree_wide", "kind": "tree", "n": 8, "lo": 2500, "hi": 4100, "mix": 5, "new": 64, "nh": 32, "nk": 8,
         "hd": 128, "pt": 64, "type": "fp16"},
        # two very long contexts
        {"name": "tree_long", "kind": "tree", "n": 2, "lo": 61000, "hi": 100001, "mix": 6, "new": 31, "nh": 32, "nk": 4,
         "hd": 128, "pt": 128, "type": "bf16"},
        # one conversation, a chain of four drafted tokens behind the last one
        {"name": "verify_one", "kind": "verify", "n": 1, "lo": 5, "hi": 5, "mix": 7, "chain": True, "vocab": 151936,
         "probs": False, "greedy": 0, "type": "fp32"},
        # trees of 16 conversations, some of them greedy
        {"name": "verify_trees", "kind": "verify", "n": 16, "lo": 8, "hi": 48, "mix": 8, "chain": False, "vocab": 151936,
         "probs": False, "greedy": 3, "type": "fp32"},
        # chains of 32 conversations sampled from a draft model whose probabilities are at hand
        {"name": "verify_sampled", "kind": "verify", "n": 32, "lo": 4, "hi": 7, "mix": 9, "chain": True, "vocab": 151936,
         "probs": True, "greedy": 0, "type": "fp32"},
        # the kept rows of 48 trees in eight of the decoder's layers
        {"name": "keep_48", "kind": "keep", "n": 48, "lo": 100, "hi": 3000, "mix": 10, "new": -32, "nk": 8, "hd": 128,
         "pt": 64, "layers": 8},
        # one conversation in all 36 layers
        {"name": "keep_one", "kind": "keep", "n": 1, "lo": 900, "hi": 900, "mix": 30, "new": 12, "nk": 8, "hd": 128,
         "pt": 64, "layers": 36},
        # one layer of a checking pass over 16 conversations
        {"name": "round_16", "kind": "round", "n": 16, "lo": 100, "hi": 4000, "mix": 12, "new": -16, "tree": True, "nh": 32,
         "nk": 8, "hd": 128, "rot": 128, "inter": False, "norm": True, "pt": 64, "type": "fp16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 8, 128), (32, 4, 128), (16, 16, 64), (16, 4, 64), (20, 4, 128), (8, 1, 128), (16, 2, 256)]


def draw(rng):
    kind = rng.choice(["rope", "rope", "tree", "tree", "tree", "verify", "verify", "keep", "round"])
    nh, nk, hd = rng.choice(HEADS)
    mix, pt, kt = rng.randrange(1 << 20), rng.choice([32, 64, 128]), rng.choice(["fp16", "fp16", "bf16"])
    if kind == "verify":
        probs = rng.random() < 0.35
        vocab = rng.choice([151936, _log(rng, 500, 150000), _log(rng, 500, 150000) | 1])
        chain = probs or rng.random() < 0.4
        n = _log(rng, 1, 32)
        hi = min(_log(rng, 2, 12 if chain else 60), max(2, 450 // n))
        return {"kind": kind, "n": n, "lo": rng.randint(1, hi), "hi": hi, "mix": mix, "chain": chain, "vocab": vocab,
                "probs": probs, "greedy": rng.choice([0, 0, n // 3, n]), "type": rng.choice(["fp32", "fp32", "fp16", "bf16"])}
    if kind == "keep":
        hi = _log(rng, 64, 2500)
        return {"kind": kind, "n": _log(rng, 1, 40), "lo": max(33, hi // _log(rng, 1, 16)), "hi": hi, "mix": mix,
                "new": rng.choice([4, 9, -16, -32]), "nk": nk, "hd": min(hd, 128), "pt": pt, "layers": rng.choice([1, 3, 8])}
    n = _log(rng, 1, 32)
    if kind == "tree":
        new = rng.choice([2, 5, 8, 16, 33, 64, -12, -24, -48])
        hi = _log(rng, 70, max(80, min(100000, 2_600_000_000 // (n * abs(new) * nh * hd))))
        return {"kind": kind, "n": n, "lo": max(abs(new), 1, hi // _log(rng, 1, 32)), "hi": max(hi, abs(new)), "mix": mix,
                "new": new, "nh": nh, "nk": nk, "hd": hd, "pt": pt, "type": kt}
    new = rng.choice([0, 1, 5, -16]) if kind == "rope" else rng.choice([3, 8, -16])
    hi = _log(rng, 40, max(50, 6000 // n if new == 0 else 4000))
    return {"kind": kind, "n": n, "lo": max(abs(new), 1, hi // _log(rng, 1, 32)), "hi": hi, "mix": mix, "new": new,
            "tree": kind == "round" or abs(new) > 1, "nh": nh, "nk": nk, "hd": hd,
            "rot": rng.choice([hd, hd, hd // 2, hd // 4]), "inter": rng.random() < 0.4, "norm": rng.random() < 0.5, "pt": pt,
            "type": rng.choice([kt, "fp32"])}


def _lens(case):
    """The lengths of a case's sequences, new tokens included: longest, shortest, the rest spread over their logarithm."""
    rng = random.Random(case["mix"])
    ls = [case["hi"], case["lo"]] + [_log(rng, case["lo"], case["hi"]) for _ in range(case["n"] - 2)]
    ls = ls[:case["n"]]
    rng.shuffle(ls)
    return ls


def _new(case):
    """Rows that each sequence brings: `new`, all of its tokens (0), or 1 .. -new of them."""
    rng = random.Random(case["mix"] + 1)
    if case["kind"] == "verify":
        return [case["hi"]] + [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"] - 1)]
    if case["new"] == 0:
        return _lens(case)
    return [case["new"] if case["new"] > 0 else rng.randint(1, -case["new"]) for _ in range(case["n"])]


def _parents(case):
    """Drafted trees, a list a sequence: row 0 is the last token, most likely branches come first (or a chain)."""
    rng = random.Random(case["mix"] + 2)
    chain = case.get("chain", False)
    return [[-1] + [i - 1 if chain or rng.random() < 0.4 else rng.randrange(max(0, i - 9), i) for i in range(1, n)]
            for n in _new(case)]


def _depths(parents):
    out = []
    for ps in parents:
        d = []
        for p in ps:
            d.append(d[p] + 1 if p >= 0 else 0)
        out.append(d)
    return out


def _kept(case):
    """Rows that a checked tree keeps: the first branch up to a place, then rows of other branches."""
    rng, out = random.Random(case["mix"] + 3), []
    for n in _new(case):
        c = rng.randint(1, max(1, n // 2))
        j = rng.randint(1, c)
        out.append(list(range(j)) + sorted(rng.sample(range(c, n), c - j)))
    return out


def _block_bytes(hd):
    return 32 * hd + hd // GROUP * 256


def _page_bytes(case):
    return case["nk"] * (case["pt"] // 32) * _block_bytes(case["hd"])


# ------------------------------------------------------------------------------ the cache format
def _unpack_nibbles(words):
    sh = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=words.device, dtype=torch.int32)
    return (words[..., None] >> sh) & 15


def _pack_nibbles(lv):
    sh = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=lv.device, dtype=torch.int64)
    w = (lv.to(torch.int64) << sh).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _unpack(blocks, hd):
    """Blocks (B, bytes) of 32 tokens -> levels K, V (B, 32, hd) and (s, m) of K, V (B, 32, hd / 64)."""
    B, ng, W = blocks.shape[0], hd // GROUP, hd // 32
    n, wi = 16 * hd, min(W, 4)
    kw = blocks[:, :n].contiguous().view(torch.int32).view(B, 2, W // wi, 4, 16, wi)
    k = _unpack_nibbles(kw).permute(0, 1, 4, 2, 5, 3, 6).reshape(B, 32, hd)
    vw = blocks[:, n:2 * n].contiguous().view(torch.int32).view(B, hd // 64, 4, 16, 4)
    v = _unpack_nibbles(vw).view(B, hd // 64, 4, 16, 4, 2, 4).permute(0, 5, 2, 6, 1, 4, 3).reshape(B, 32, hd)
    p = blocks[:, 2 * n:].contiguous().view(torch.float16).view(B, 4, ng * 32)
    slots = lambda x: x.view(B, ng, 4, 2, 4).permute(0, 3, 2, 4, 1).reshape(B, 32, ng)  # noqa: E731
    return k, v, slots(p[:, 0]), p[:, 1].reshape(B, 32, ng), slots(p[:, 2]), slots(p[:, 3])


def _pack(k, v, ks, km, vs, vm):
    """The inverse of _unpack."""
    B, _, hd = k.shape
    ng, W = hd // GROUP, hd // 32
    wi = min(W, 4)
    kw = _pack_nibbles(k.view(B, 2, 16, W // wi, wi, 4, 8).permute(0, 1, 3, 5, 2, 4, 6))
    vw = _pack_nibbles(v.view(B, 2, 4, 4, hd // 64, 4, 16).permute(0, 4, 2, 6, 5, 1, 3).reshape(B, hd // 64, 4, 16, 4, 8))
    slots = lambda x: x.view(B, 2, 4, 4, ng).permute(0, 4, 2, 1, 3).reshape(B, ng * 32)  # noqa: E731
    p = torch.stack([slots(ks), km.reshape(B, -1), slots(vs), slots(vm)], 1).contiguous()
    return torch.cat([kw.reshape(B, -1).contiguous().view(torch.uint8), vw.reshape(B, -1).contiguous().view(torch.uint8),
                      p.view(B, -1).view(torch.uint8)], 1)


def _quantize(x):
    """Rows (..., hd) -> levels (..., hd) int32, scale and minimum (..., hd / 64) fp16."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) * SEVENTH).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    bad = ~torch.isfinite(g).all(-1)
    s, m = s.masked_fill(bad, math.nan), m.masked_fill(bad, math.nan)
    t = (g.double() - m.double()[..., None]) / s.double()[..., None]     # (64 bits: values next to a border)
    t = torch.where((s > 0)[..., None], t, 0.0)
    return t.round().clamp(0, 15).to(torch.int32).flatten(-2), s, m


def _values(lv, s, m):
    return torch.addcmul(m.float()[..., None], s.float()[..., None], lv.float().unflatten(-1, (-1, GROUP))).flatten(-2)


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _dtype(case):
    """The type of the rows that leave an operator (float32 inputs: fp16)."""
    return torch.bfloat16 if case["type"] == "bf16" else torch.float16


def _heads(g, rows, nh, hd, dt):
    """Query rows as they leave a per-head RMSNorm: unit mean square."""
    x = torch.randn(rows, nh, hd, generator=g, device=DEV)
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True))).to(dt)


def _kv(g, rows, nk, hd, dt):
    """Key rows with a few strong channels, value rows of different strengths."""
    k = torch.randn(rows, nk, hd, generator=g, device=DEV)
    k[..., 5::32] = k[..., 5::32] * 3 + 2
    v = torch.randn(rows, nk, hd, generator=g, device=DEV) * (0.3 + torch.rand(rows, nk, 1, generator=g, device=DEV))
    return k.to(dt), v.to(dt)


def _history(case, g, n_pages):
    """The K/V rows behind the pool's pages, a piece of the pages at a time."""
    piece = max(1, (1 << 24) // (case["pt"] * case["nk"] * case["hd"]))
    for p in range(0, n_pages, piece):
        c = min(piece, n_pages - p)
        k, v = _kv(g, c * case["pt"], case["nk"], case["hd"], torch.float16)
        yield p, c, k.view(c, case["pt"] // 32, 32, case["nk"], -1), v.view(c, case["pt"] // 32, 32, case["nk"], -1)


def _pool(case, seed, lens, spare=8):
    """Page table, lengths, reference counts (pages in random order, a few free) and the number of pages."""
    pt = case["pt"]
    counts = [(ln + pt - 1) // pt for ln in lens]
    n_pages, width = sum(counts) + spare, max(counts) + 2
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    table, refs, at = np.full((len(lens), width), -1, np.int32), np.zeros(n_pages, np.int32), 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        refs[order[at:at + c]] = 1
        at += c
    return (torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
            torch.from_numpy(refs).to(DEV), n_pages)


def _ints(xs):
    return torch.tensor(list(xs), dtype=torch.int32, device=DEV)


def _cu(ns):
    return _ints([0] + list(np.cumsum(ns)))


def _flat(xs):
    return [v for x in xs for v in x]


def _masks(parents, words):
    """Bit j of a row: row j of its sequence is the row itself or above it."""
    out = []
    for ps in parents:
        m = []
        for i, p in enumerate(ps):
            m.append((m[p] if p >= 0 else 0) | 1 << i)
        out += m
    low = (1 << 64) - 1
    words = np.array([[m >> 64 * w & low for w in range(words)] for m in out], dtype=np.uint64)
    return torch.from_numpy(words.view(np.int64)).to(DEV)


def _prepare_verify(case, g, st):
    parents, V, dt = _parents(case), case["vocab"], _TYPES[case["type"]]
    n = [len(p) for p in parents]
    T = sum(n)
    logits = torch.randn(T, V, generator=g, device=DEV) * 3
    st["parents"], st["cu"], st["n"] = _ints(_flat(parents)), _cu(n), n
    row0 = np.cumsum([0] + n[:-1])
    par = torch.tensor(_flat([[max(p, 0) + r for p in ps] for ps, r in zip(parents, row0)]), device=DEV)
    temp = torch.tensor([0.0 if i < case["greedy"] else 0.7 + 0.1 * (i % 5) for i in range(case["n"])], device=DEV)
    st["temp"] = temp
    st["u"] = torch.rand(T, generator=g, device=DEV)
    st["probs"] = None
    if case["probs"]:                                  # the draft model's opinion is near the target's
        d = (logits + torch.randn(T, V, generator=g, device=DEV)).div_(0.9)
        st["probs"] = torch.softmax(d, -1)
        st["tokens"] = torch.multinomial(st["probs"][par], 1, generator=g)[:, 0]
        del d
    else:                                              # one of the target's likely tokens, the first ones more often
        like = logits.topk(min(6, V), -1).indices[par]
        pick = (torch.rand(T, generator=g, device=DEV).square() * like.shape[1]).long()
        st["tokens"] = like.gather(1, pick[:, None])[:, 0].contiguous()
    st["logits"] = logits.to(dt)
    return st


def prepare(case, seed):
    g, st = _gen(seed), {"case": case}
    kind = case["kind"]
    if kind == "verify":
        return _prepare_verify(case, g, st)
    new = _new(case)
    lens = [max(a, b) for a, b in zip(_lens(case), new)]
    st["new"], st["most"] = new, (max(new), max(lens))
    st["table"], st["lens"], st["refs"], n_pages = _pool(case, seed, lens)
    st["cu"] = _cu(new)
    T = sum(new)
    if kind == "keep":
        st["pages"] = torch.randint(0, 256, (case["layers"], n_pages, _page_bytes(case)), generator=g, device=DEV,
                                    dtype=torch.uint8)
        kept = _kept(case)
        st["path"] = _ints(_flat([k + [-1] * (n - len(k)) for k, n in zip(kept, new)]))
        st["counts"] = _ints(len(k) for k in kept)
        st["was"] = (st["table"].clone(), st["lens"].clone(), st["refs"].clone())
        return st
    st["pages"] = torch.empty(1, n_pages, _page_bytes(case), dtype=torch.uint8, device=DEV)
    for p, c, k, v in _history(case, g, n_pages):
        kk, vv = (x.permute(0, 3, 1, 2, 4).reshape(-1, 32, case["hd"]) for x in (k, v))
        (kl, ks, km), (vl, vs, vm) = _quantize(kk), _quantize(vv)
        st["pages"][0, p:p + c] = _pack(kl, vl, ks, km, vs, vm).view(c, -1)
    dt = _TYPES[case["type"]]
    st["q"] = _heads(g, T, case["nh"], case["hd"], dt)
    if kind != "rope":
        parents = _parents(case)
        st["parents"] = _ints(_flat(parents))
        st["mask"] = _masks(parents, 1)
    if kind == "tree":
        return st
    st["k"], st["v"] = _kv(g, T, case["nk"], case["hd"], dt)
    # angles in 64 bits; frequencies stretched fourfold, as for contexts longer than those trained on
    inv = 1.0e6 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"]) / 4
    ang = torch.outer(torch.arange(max(lens), device=DEV, dtype=torch.float64), inv)
    st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    st["depth"] = _ints(_flat(_depths(_parents(case)))) if case["tree"] else None
    st["qw"] = st["kw"] = None
    if case["norm"]:
        st["qw"], st["kw"] = ((1 + 0.2 * torch.randn(case["hd"], generator=g, device=DEV)).to(_dtype(case)) for _ in range(2))
    return st


# ------------------------------------------------------------------------------ plain forms
def _padded(cu, most):
    """Row numbers (n, most) of packed rows, and which of them are rows."""
    cu = cu.long()
    i = torch.arange(most, device=cu.device)
    n = cu[1:] - cu[:-1]
    return torch.minimum(cu[:-1, None] + i, (cu[1:, None] - 1).clamp(min=0)), i < n[:, None]


def _slot_of(st, T):
    cu = st["cu"].long()
    return torch.searchsorted(cu[1:].contiguous(), torch.arange(T, device=DEV), right=True), cu


def _where(st):
    """Block number (page, head 0, block in page) and row in the block of every new token."""
    c = st["case"]
    T, bpp = sum(st["new"]), c["pt"] // 32
    slot, cu = _slot_of(st, T)
    pos = st["lens"].long()[slot] - cu[slot + 1] + torch.arange(T, device=DEV)
    page = st["table"][slot, pos // c["pt"]].long()
    return page * c["nk"] * bpp + pos % c["pt"] // 32, pos % 32


def _blocks(st, first):
    """Numbers of the blocks of all heads for blocks of head 0."""
    c = st["case"]
    return first[..., None] + torch.arange(c["nk"], device=DEV) * (c["pt"] // 32)


def _plain_write(st, k, v):
    c = st["case"]
    hd, nk = c["hd"], c["nk"]
    pool = st["pages"].view(-1, _block_bytes(hd))
    first, row = _where(st)
    some, at = torch.unique(first, return_inverse=True)
    ids = _blocks(st, some).flatten()
    parts = [x.view(some.numel(), nk, 32, -1).clone() for x in _unpack(pool[ids], hd)]
    kl, ks, km = _quantize(k)
    vl, vs, vm = _quantize(v)
    parts[0][at, :, row], parts[1][at, :, row], parts[2][at, :, row] = kl, vl, ks
    parts[3][at, :, row], parts[4][at, :, row], parts[5][at, :, row] = km, vs, vm
    pool[ids] = _pack(*[x.reshape(ids.numel(), 32, -1) for x in parts])


def _plain_read(st):
    c = st["case"]
    first, row = _where(st)
    ids = _blocks(st, first)
    parts = [x.view(first.numel(), c["nk"], 32, -1)
             for x in _unpack(st["pages"].view(-1, _block_bytes(c["hd"]))[ids.flatten()], c["hd"])]
    i, h = torch.arange(first.numel(), device=DEV)[:, None], torch.arange(c["nk"], device=DEV)
    kl, vl, ks, km, vs, vm = (x[i, h, row[:, None]] for x in parts)
    return _values(kl, ks, km).to(_dtype(c)), _values(vl, vs, vm).to(_dtype(c))


def _rotate(x, w, cos, sin, inter, eps):
    """Rows (T, heads, hd) in 64 bits: normed (with w), then their first dimensions rotated by the rows of cos, sin."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    r = 2 * cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    if inter:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., r:]], -1)


def _positions(st, depth):
    slot, cu = _slot_of(st, sum(st["new"]))
    first = st["lens"].long()[slot] - (cu[slot + 1] - cu[slot])
    return first + (torch.arange(slot.numel(), device=DEV) - cu[slot] if depth is None else depth.long())


def _plain_rope(st, depth):
    c, dt = st["case"], _dtype(st["case"])
    pos = _positions(st, depth)
    q, k = (_rotate(st[x], st[w], st["cos"][pos], st["sin"][pos], c["inter"], EPS).float().to(dt)
            for x, w in (("q", "qw"), ("k", "kw")))
    _plain_write(st, k, st["v"].to(dt))
    return q


def _softmax_product(q, k, v, keep, scale):
    """q (b, g, r, d), k / v (b, g, l, d) float32, keep (b, 1, r, l): rows that keep nothing give zeros."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill_(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _plain_tree(st, q, mask):
    c = st["case"]
    nh, nk, hd, pt = c["nh"], c["nk"], c["hd"], c["pt"]
    rep, (mq, mk) = nh // nk, st["most"]
    nb, pool = (mk + 31) // 32, st["pages"].view(-1, _block_bytes(hd))
    rq, isq = _padded(st["cu"], mq)
    out = torch.empty(q.shape, dtype=q.dtype, device=DEV)
    j, key = torch.arange(nb, device=DEV), torch.arange(nb * 32, device=DEV)
    for i in range(0, len(st["new"]), 8):                        # eight slots at a time
        rows, real = rq[i:i + 8], isq[i:i + 8]
        b = rows.shape[0]
        page = st["table"][i:i + 8, (j // (pt // 32)).clamp(max=st["table"].shape[1] - 1)].long().clamp(min=0)
        ids = _blocks(st, page * nk * (pt // 32) + j % (pt // 32))               # (b, nb, nk)
        kl, vl, ks, km, vs, vm = _unpack(pool[ids.flatten()], hd)
        k, v = _values(kl, ks, km), _values(vl, vs, vm)
        k, v = (x.view(b, nb, nk, 32, hd).permute(0, 2, 1, 3, 4).reshape(b, nk, nb * 32, hd) for x in (k, v))
        qq = q.float()[rows].view(b, mq, nk, rep, hd).permute(0, 2, 3, 1, 4).reshape(b, nk, rep * mq, hd)
        first = (st["lens"][i:i + 8].long() - real.sum(-1))[:, None, None]
        bit = (key - first).clamp(0, 63)
        see = (mask[rows, 0][..., None] >> bit & 1).bool() & (key < first + real.sum(-1)[:, None, None])
        keep = (key < first) | see
        keep = keep[:, None, None].expand(b, 1, rep, mq, nb * 32).reshape(b, 1, rep * mq, nb * 32)
        o = _softmax_product(qq, k, v, keep, 1 / math.sqrt(hd))
        o = o.view(b, nk, rep, mq, hd).permute(0, 3, 1, 2, 4).reshape(b, mq, nh, hd)
        out[rows[real]] = o[real].to(q.dtype)
    return out


def _plain_draft_tree(st):
    """Masks and depths from the parents, a row of every tree at a time."""
    cu, most = st["cu"].long(), st["most"][0]
    T = st["parents"].numel()
    mask, depth = torch.zeros(T, 1, dtype=torch.int64, device=DEV), torch.zeros(T, dtype=torch.int32, device=DEV)
    rows, real = _padded(st["cu"], most)
    for i in range(most):
        r, ok = rows[:, i], real[:, i]
        up = st["parents"][r].long()
        has = ok & (up >= 0) & (up < i)
        at = cu[:-1] + up.clamp(min=0)
        m = torch.where(has, mask[at.clamp(max=T - 1), 0], 0) | (1 << i if i < 63 else -(1 << 63))
        d = torch.where(has, depth[at.clamp(max=T - 1)] + 1, 0).int()
        mask[r, 0] = torch.where(ok, m, mask[r, 0])
        depth[r] = torch.where(ok, d, depth[r])
    return mask, depth


def _plain_verify(st):
    cu, tok, par, u = st["cu"].long(), st["tokens"], st["parents"].long(), st["u"].double()
    S, T = cu.numel() - 1, tok.numel()
    most = max(st["n"])
    start, n = cu[:-1], cu[1:] - cu[:-1]
    slot, _ = _slot_of(st, T)
    temp = st["temp"].double()
    w = st["logits"].double()
    best = w.argmax(-1)                                # (the lowest index of several)
    w -= w.amax(-1, keepdim=True)
    w /= torch.where(temp > 0, temp, 1.0)[slot][:, None]
    w.exp_()
    w /= w.sum(-1, keepdim=True)
    s = torch.arange(S, device=DEV)
    greedy = temp <= 0
    cur, left, count = torch.zeros(S, dtype=torch.long, device=DEV), torch.ones(S, dtype=torch.float64, device=DEV), n.clamp(max=1)
    path = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    path[start[n > 0]] = 0
    gone = torch.zeros(S, most, dtype=torch.bool, device=DEV)
    rows, _ = _padded(st["cu"], most)
    toks = tok[rows]
    rest = w[start].clone() if st["probs"] is not None else None
    for i in range(1, most):
        r = rows[:, i]
        child = (i < n) & (par[r] == cur)
        x = tok[r]
        if rest is None:
            p = w[start + cur, x]
            twice = ((toks == x[:, None]) & gone).any(-1)
            yes = child & torch.where(greedy, x == best[start + cur], ~twice & (u[r] * left < p))
            no = child & ~yes & ~twice & ~greedy
            left = torch.where(yes, 1.0, torch.where(no, left - p, left))
            gone[:, i] = no
            gone &= ~yes[:, None]
        else:
            q = st["probs"][start + cur].double()
            yes = child & torch.where(greedy, x == best[start + cur], u[r] * q[s, x] < rest[s, x])
            no = child & ~yes & ~greedy
            less = (rest - q).clamp_(min=0)
            total = less.sum(-1, keepdim=True)
            less = torch.where(total > 0, less / torch.where(total > 0, total, 1.0), w[start + cur])
            rest = torch.where(no[:, None], less, rest)
        path[(start + count).clamp(max=T - 1)[yes]] = i
        count = count + yes
        cur = torch.where(yes, i, cur)
        if rest is not None:
            rest = torch.where(yes[:, None], w[start + cur], rest)
    end = w[start + cur]
    if rest is None:
        off = torch.zeros_like(end).scatter_add_(1, toks, gone.double())
        end = torch.where((off > 0) & (end * (off == 0)).sum(-1, keepdim=True).gt(0), 0.0, end)
    else:
        end = rest
    c = end.cumsum(-1)
    total = c[:, -1:]
    k = torch.searchsorted(c, u[start][:, None] * total, right=True)[:, 0]
    last = torch.where(end > 0, torch.arange(end.shape[1], device=DEV), 0).amax(-1)
    nxt = torch.where(greedy, best[start + cur], torch.minimum(k, last))
    return path, count.int(), nxt


def _plain_keep(st):
    c = st["case"]
    hd, nk, pt = c["hd"], c["nk"], c["pt"]
    path, counts, cu = st["path"].long(), st["counts"].long(), st["cu"].long()
    T = path.numel()
    slot, _ = _slot_of(st, T)
    i = torch.arange(T, device=DEV) - cu[slot]
    base = st["lens"].long() - (cu[1:] - cu[:-1])
    move = (i < counts[slot]) & (path != i)
    slot, to, at = slot[move], (base[slot] + i)[move], (base[slot] + path)[move]
    bpp, layers = pt // 32, c["layers"]

    def block(pos):                                    # (moves, layers * heads) numbers of blocks
        b = _blocks(st, st["table"][slot, pos // pt].long() * nk * bpp + pos % pt // 32)
        per = st["pages"].shape[1] * nk * bpp
        return (b[:, None] + torch.arange(layers, device=DEV)[:, None] * per).flatten(1)

    pool = st["pages"].view(-1, _block_bytes(hd))
    src, dst = block(at), block(to)
    some, where = torch.unique(torch.cat([src.flatten(), dst.flatten()]), return_inverse=True)
    a, b = (x.view(src.shape) for x in where.view(2, -1))
    if some.numel():                                   # (some row moves)
        parts = [x.clone() for x in _unpack(pool[some], hd)]
        for x in parts:
            x[b, (to % 32)[:, None]] = x[a, (at % 32)[:, None]]
        pool[some] = _pack(*parts)
    st["lens"].copy_(torch.where(cu[1:] > cu[:-1], base + counts, st["lens"].long()).int())
    have = (st["lens"] + pt - 1) // pt
    col = torch.arange(st["table"].shape[1], device=DEV)
    drop = (col >= have[:, None]) & (st["table"] >= 0)
    st["refs"].index_add_(0, st["table"].long().clamp(min=0).flatten(), -drop.flatten().int())
    st["table"].masked_fill_(drop, -1)


# ------------------------------------------------------------------------------ one pass
def _module(name):
    at = os.path.join(os.getcwd(), "sx8-quantization_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    return __import__(name)


def _handle(st):
    """The framework's handle on the state's cache, which a program keeps."""
    if "pool" not in st:
        c = st["case"]
        st["pool"] = _module("sx8_paged_kv").PagedKV4.from_tensors(st["pages"], st["table"], st["lens"], st["refs"],
                                                                   n_kv=c["nk"], head_dim=c["hd"], page_tokens=c["pt"])
    return st["pool"]


def _own_rope(st, depth):
    c = st["case"]
    return _handle(st).append_rope(0, st["q"], st["k"], st["v"], st["cos"], st["sin"], st["cu"], depth=depth, q_norm=st["qw"],
                                   k_norm=st["kw"], eps=EPS, interleaved=c["inter"], dtype=_dtype(c))


def _run_rope(st):
    if own:
        q = _own_rope(st, st["depth"])
        return (q, *_handle(st).read(0, q.shape[0], st["cu"], dtype=q.dtype))
    q = _plain_rope(st, st["depth"])
    return (q, *_plain_read(st))


def _run_tree(st):
    if own:
        return _handle(st).attend_tree(0, st["q"], st["mask"], st["cu"])
    return _plain_tree(st, st["q"], st["mask"])


def _run_round(st):
    if own:
        mask, depth = _module("sx8_draft").draft_tree(st["parents"], st["cu"])
        q = _own_rope(st, depth)
        o = _handle(st).attend_tree(0, q, mask, st["cu"])
        return (mask, depth, o, *_handle(st).read(0, q.shape[0], st["cu"], dtype=q.dtype))
    mask, depth = _plain_draft_tree(st)
    q = _plain_rope(st, depth)
    return (mask, depth, _plain_tree(st, q, mask), *_plain_read(st))


def _run_verify(st):
    if own:
        return _module("sx8_draft").verify_draft(st["logits"], st["tokens"], st["parents"], st["cu"], st["u"],
                                                 temperature=st["temp"], draft_probs=st["probs"])
    return _plain_verify(st)


def _run_keep(st):
    st["table"].copy_(st["was"][0])                    # the slots with all of their new rows again
    st["lens"].copy_(st["was"][1])
    st["refs"].copy_(st["was"][2])
    if own:
        _handle(st).keep(st["path"], st["counts"], st["cu"])
    else:
        _plain_keep(st)
    return st["table"], st["lens"], st["refs"], st["pages"]


def run(state):
    return {"rope": _run_rope, "tree": _run_tree, "verify": _run_verify, "keep": _run_keep,
            "round": _run_round}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------ work
def work(case):
    kind, new = case["kind"], _new(case)
    T = sum(new)
    if kind == "verify":                               # the rows of one path through each tree, and its draft rows
        size = {"fp32": 4, "fp16": 2, "bf16": 2}[case["type"]]
        rows = sum(max(d) + 1 for d in _depths(_parents(case)))
        return {"bytes": rows * case["vocab"] * (size + (4 if case["probs"] else 0)) + 28 * T, "flops": 3 * rows * case["vocab"]}
    nk, hd = case["nk"], case["hd"]
    row = nk * (hd + hd // GROUP * 8)                  # packed bytes of a token
    if kind == "keep":
        moved = sum(sum(p != i for i, p in enumerate(k)) for k in _kept(case))
        return {"bytes": 2 * moved * row * case["layers"] + 8 * T, "flops": 0}
    lens, nh = [max(a, b) for a, b in zip(_lens(case), new)], case["nh"]
    size = 4 if case["type"] == "fp32" else 2
    rope = {"bytes": T * (nh * hd * (size + 2) + 2 * nk * hd * size + row + 4 * case.get("rot", 0)),
            "flops": T * (nh + nk) * (3 * case.get("rot", 0) + (4 * hd if case.get("norm") else 0)) + 12 * T * nk * hd}
    if kind == "rope":
        return {"bytes": rope["bytes"] + T * (row + 4 * nk * hd), "flops": rope["flops"]}
    depths = _depths(_parents(case))
    pairs = sum(n * (ln - n) + sum(d) + n for n, ln, d in zip(new, lens, depths))
    tree = {"bytes": sum(lens) * row + 4 * T * nh * hd + 8 * T, "flops": 4 * nh * hd * pairs}
    if kind == "round":
        return {"bytes": rope["bytes"] + tree["bytes"] + T * (row + 4 * nk * hd + 8), "flops": rope["flops"] + tree["flops"]}
    return tree


# ------------------------------------------------------------------------------ in 64 bits
def _exact_rows(x):
    """The values that rows stand for in 4 bits, from the definition."""
    a = x.double().reshape(-1, GROUP)
    lo, hi = torch.aminmax(a, dim=-1, keepdim=True)
    width = (hi.float() - lo.float()) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)
    s = torch.minimum(width, torch.tensor(65504.0, device=x.device)).half().double()
    m = torch.clip(lo.float(), -65504, 65504).half().double()
    lv = torch.clip(torch.round((a - m) / torch.where(s > 0, s, torch.ones_like(s))), 0, 15) * (s > 0)
    return (m + s * lv).view(x.shape)


def _exact_turn(x, w, pos, case, st):
    """Rows as complex numbers times cos + i sin."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    r = case["rot"]
    z = torch.complex(st["cos"].double(), st["sin"].double())[pos][:, None]
    pairs = x[..., :r].unflatten(-1, (r // 2, 2) if case["inter"] else (2, r // 2))
    a, b = pairs.unbind(-1 if case["inter"] else -2)
    y = torch.complex(a, b) * z
    y = torch.stack([y.real, y.imag], -1 if case["inter"] else -2).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def _exact_tree(q, k, v, first, parents):
    """q (n, nh, d), k / v (first + n, nk, d): a row sees the first keys, its own and those of the rows above it."""
    n, nh, d = q.shape
    out, rep = torch.empty_like(q), nh // k.shape[1]
    see = torch.zeros(n, k.shape[0], dtype=torch.bool)
    see[:, :first] = True
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, first + i] = True
    see = see.to(q.device)
    for h in range(nh):
        kh, vh = k[:, h // rep], v[:, h // rep]
        s = (q[:, h] @ kh.T.contiguous() / math.sqrt(d)).masked_fill(~see, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ vh
    return out


def _exact_verify(case, st):
    logits, cu = st["logits"], st["cu"].tolist()
    tokens, parents, u, temps = st["tokens"].tolist(), st["parents"].tolist(), st["u"].tolist(), st["temp"].tolist()
    path, counts, nxt = [-1] * len(tokens), [], []

    def target(row, t):
        x = logits[row].double().cpu().numpy()
        if t <= 0:
            p = np.zeros_like(x)
            p[int(np.flatnonzero(x == x.max())[0])] = 1.0
            return p
        e = np.exp((x - x.max()) / t)
        return e / e.sum()

    for s, t in enumerate(temps):
        a, n = cu[s], cu[s + 1] - cu[s]
        at, kept = 0, [0]
        p = target(a, t)
        while True:
            q = st["probs"][a + at].double().cpu().numpy() if case["probs"] and t > 0 else None
            for i in range(at + 1, n):
                if parents[a + i] != at:
                    continue
                x = tokens[a + i]
                if u[a + i] * (1.0 if q is None or t <= 0 else q[x]) < p[x]:
                    break
                if t > 0:
                    less = np.maximum(p - q, 0) if q is not None else np.where(np.arange(p.size) == x, 0.0, p)
                    p = less / less.sum() if less.sum() > 0 else target(a + at, t)
            else:
                break
            at = i
            kept.append(i)
            p = target(a + at, t)
        path[a:a + len(kept)] = kept
        counts.append(len(kept))
        c = np.cumsum(p)
        nxt.append(int(np.searchsorted(c, u[a] * c[-1], side="right")))
    return _ints(path), _ints(counts), torch.tensor(nxt, device=DEV)


def exact(case, seed):
    kind = case["kind"]
    if kind == "keep":
        return None
    st = prepare(case, seed)
    if kind == "verify":
        return _exact_verify(case, st) if sum(st["n"]) <= 1000 else None
    new, lens, dt = st["new"], st["lens"].tolist(), _dtype(case)
    depths = _depths(_parents(case)) if case.get("tree") else [range(n) for n in new]
    if kind != "tree":
        pos = torch.tensor([ln - n + d for n, ln, ds in zip(new, lens, depths) for d in ds], device=DEV)
        q, k = (_exact_turn(st[x], st[w], pos, case, st) for x, w in (("q", "qw"), ("k", "kw")))
        fresh = [_exact_rows(x.float().to(dt)) for x in (k, st["v"])]
        if kind == "rope":
            return q, fresh[0], fresh[1]
        q = q.float().to(dt).double()
    else:
        q = st["q"].double()
    old = [[], []]
    for _, c, k, v in _history(case, _gen(seed), st["pages"].shape[1]):
        for into, x in zip(old, (k, v)):
            into.append(_exact_rows(x).reshape(c, case["pt"], case["nk"], -1))
    old = [torch.cat(x) for x in old]
    outs, a, parents = [], 0, _parents(case)
    for i, (n, ln) in enumerate(zip(new, lens)):
        ids = st["table"][i, :(ln + case["pt"] - 1) // case["pt"]].long()
        k, v = (x[ids].flatten(0, 1)[:ln] for x in old)
        if kind == "round":
            k, v = (torch.cat([x[:ln - n], y[a:a + n]]) for x, y in ((k, fresh[0]), (v, fresh[1])))
        outs.append(_exact_tree(q[a:a + n], k, v, ln - n, parents[i]))
        a += n
    if kind == "round":
        return None, None, torch.cat(outs), fresh[0], fresh[1]
    return torch.cat(outs)
