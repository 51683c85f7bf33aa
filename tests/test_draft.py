"""Drafted tokens on the GPU (append_rope, attend_tree, draft_tree, verify_draft, keep) against plain implementations in 64
bits.

Tolerances.  append_rope computes in 64 bits and rounds once, as the reference does (to float32 and from there to 16 bits; an
exact value within 2^-50 of a rounding's border is not to be expected among the 10^6 here), so its rows and what is read back are
equal.  attend_tree is the arithmetic of PagedKV4.attend, with the bound that test_paged_kv.py derives: half a step of the output
and LOOSE = 2^-15 of the largest value averaged (the weights' sum is taken from the matrix cores here: two fp16 numbers a
weight, cut, 2^-21 of it, their products with a scale within 2^-22 of that or 2^-24: within 2^-15 with the rest).  verify_draft and keep
return whole numbers and moved bits: equal."""
import math
import random

import numpy as np
import pytest
import torch

from test_paged_kv import BF16, F16, LOOSE, close, cum, ints, make, q4, rand

pytestmark = pytest.mark.gpu

F32 = torch.float32


# ------------------------------------------------------------------------------ plain implementations
def turn(x, w, cos, sin, inter, eps=1e-6):
    """Rows (T, heads, hd) normed and rotated by the rows (T, r / 2) of cos and sin, in 64 bits."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    r = 2 * cos.shape[1]
    z = torch.complex(cos.double(), sin.double())[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    re, im = a * z.real - b * z.imag, b * z.real + a * z.imag
    y = torch.stack([re, im], -1).flatten(-2) if inter else torch.cat([re, im], -1)
    return torch.cat([y, x[..., r:]], -1)


def tables(n, rot, cuda, seed=0):
    """Angles of every size, and a length that is not 1."""
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(n, rot // 2, generator=g, dtype=torch.float64) * 6000
    return (1.1 * ang.cos()).float().to(cuda), (1.1 * ang.sin()).float().to(cuda)


def trees(ns, seed, chain=False):
    """Parents of trees of these sizes; row 0 is a root."""
    rng = random.Random(seed)
    return [[-1] + [i - 1 if chain or rng.random() < 0.3 else rng.randrange(max(0, i - 6), i) for i in range(1, n)] if n else []
            for n in ns]


def ancestors(ps):
    out = []
    for i, p in enumerate(ps):
        out.append((out[p] if 0 <= p < i else frozenset()) | {i})
    return out


def flat(xs):
    return [v for x in xs for v in x]


def words_of(sets, words):
    """Sets of row numbers as masks (rows, words) int64."""
    m = np.array([[sum(1 << j - 64 * w for j in s if 64 * w <= j < 64 * w + 64) for w in range(words)] for s in sets],
                 dtype=np.uint64).reshape(len(sets), words)
    return torch.from_numpy(m.view(np.int64))


def want_tree(q, k, v, first, sets, scale=None):
    """q (n, nh, d), k / v (first + n, nk, d) float64: row i sees the first keys and those of sets[i]; none: zeros."""
    n, nh, d = q.shape
    L, nk = k.shape[:2]
    if n == 0 or L == 0:
        return torch.zeros_like(q)
    rep = nh // nk
    see = torch.zeros(n, L, dtype=torch.bool)
    for i, s in enumerate(sets):
        see[i, :max(first, 0)] = True
        for j in s:
            if 0 <= first + j < L and j < n:
                see[i, first + j] = True
    see = see.to(q.device)
    kk = k.repeat_interleave(rep, 1).permute(1, 2, 0).contiguous()
    vv = v.repeat_interleave(rep, 1).permute(1, 0, 2).contiguous()
    w = torch.matmul(q.permute(1, 0, 2).contiguous(), kk) * (scale or 1 / math.sqrt(d))
    w = w.masked_fill(~see, -math.inf)
    p = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e300)).masked_fill(~see, 0.0)
    o = torch.matmul(p, torch.where(torch.isfinite(vv), vv, 0.0))
    seen = see.double().expand(nh, n, L).contiguous()
    odd = torch.matmul(seen, (~torch.isfinite(vv)).double()) > 0
    o = torch.where(odd, math.nan, o / p.sum(-1, keepdim=True).clamp(min=1e-300))
    return o.permute(1, 0, 2)


def want_verify(logits, tokens, parents, u, temp, probs=None):
    """One slot: (kept rows, next token), float64 on the host."""
    def target(row):
        x = logits[row].astype(np.float64)
        x = np.where(np.isnan(x), -np.inf, x)
        top = x.max()
        if top == -np.inf:
            return None, -1
        if temp <= 0:
            return None, int(np.flatnonzero(x == top)[0])
        with np.errstate(invalid="ignore"):
            e = np.where(x == top, 1.0, np.exp((x - top) / temp))
        e = np.where(np.isnan(e) | (x == -np.inf), 0.0, e)
        return e / e.sum(), int(np.flatnonzero(x == top)[0])

    cur, kept = 0, [0]
    p, best = target(0)
    n, V = len(tokens), logits.shape[1]
    while True:
        nxt = None
        q = probs[cur].astype(np.float64) if probs is not None else None
        for i in range(cur + 1, n):
            if parents[i] != cur:
                continue
            x = tokens[i]
            if best < 0 or not 0 <= x < V:
                ok = False
                if best >= 0 and temp > 0:
                    pass                                             # a token that is none: nothing is known of it
            elif temp <= 0:
                ok = x == best
            elif q is None:
                ok = p[x] > 0 and u[i] < p[x]
                if not ok and p[x] > 0:
                    less = p.copy()
                    less[x] = 0.0
                    p = less / less.sum() if less.sum() > 0 else target(cur)[0]
            else:
                ok = p[x] > 0 and u[i] * q[x] < p[x]
                if not ok:
                    less = np.maximum(p - q, 0)
                    p = less / less.sum() if less.sum() > 0 else target(cur)[0]
            if ok:
                nxt = i
                break
        if nxt is None:
            break
        cur = nxt
        kept.append(cur)
        p, best = target(cur)
    if best < 0 or temp <= 0:
        return kept, best
    c = np.cumsum(p)
    k = int(np.searchsorted(c, u[0] * c[-1], side="right"))
    return kept, min(k, int(np.flatnonzero(p > 0)[-1]))


# ------------------------------------------------------------------------------ append_rope
@pytest.mark.parametrize("hd,rot,inter", [(64, 64, False), (128, 128, False), (128, 32, True), (256, 64, False), (256, 256, True),
                                          (64, 16, True)])
@pytest.mark.parametrize("dt,wide", [(F16, False), (BF16, False), (F16, True), (BF16, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rope(hiplib, cuda, hd, rot, inter, dt, wide, norm):
    """Rotated query rows, and what is read back of K and V, in calls that end inside blocks and pages; later calls keep the
    tokens of earlier ones."""
    from sx8_paged_kv import PagedKV4
    nk, nh, pt = 2, 6, 32
    p = PagedKV4(1, nk, hd, 16, 4, 5, pt, device=cuda)
    cos, sin = tables(130, rot, cuda)
    lens, parts = [0] * 4, [[] for _ in range(4)]
    for step, ns in enumerate([[0, 1, 33, 70], [1, 0, 5, 13], [3, 31, 1, 32]]):
        p.reserve(ints(ns, cuda))
        T = sum(ns)
        q, k, v = (rand((T, n, hd), 7 * step + i, F32 if wide else dt, cuda, s) for i, (n, s) in enumerate(((nh, 1), (nk, 2), (nk, 0.3))))
        qw, kw = (1 + rand((hd,), 50 + i, dt, cuda, 0.3) for i in range(2)) if norm else (None, None)
        depth = [j // 2 for n in ns for j in range(n)] if step == 1 else None
        got = p.append_rope(0, q, k, v, cos, sin, cum(ns, cuda), depth=None if depth is None else ints(depth, cuda), q_norm=qw,
                            k_norm=kw, interleaved=inter, dtype=dt)
        at = [a + j for a, n in zip(lens, ns) for j in (range(n) if depth is None else [j // 2 for j in range(n)])]
        assert torch.equal(got, turn(q, qw, cos[at], sin[at], inter).float().to(dt))
        kk, a = turn(k, kw, cos[at], sin[at], inter).float().to(dt), 0
        for s, n in enumerate(ns):
            parts[s].append((kk[a:a + n], v[a:a + n].to(dt)))
            a, lens[s] = a + n, lens[s] + n
    p.check()
    gk, gv = p.read(0, sum(lens), cum(lens, cuda), dtype=dt)
    k, v = (torch.cat([x[j] for part in parts for x in part]) for j in range(2))
    assert torch.equal(gk, q4(k).to(dt)) and torch.equal(gv, q4(v).to(dt))


def test_append_rope_places_outside(hiplib, cuda):
    """Rows before and behind the tables: zeros, and the pages keep what they had; strided rows, an `out` with room between its
    rows, one row a slot without cu, more than 64 slots."""
    from sx8_paged_kv import PagedKV4
    S, hd = 70, 64
    p = PagedKV4(2, 1, hd, S, S, 2, 32, device=cuda)
    p.reserve(ints([5] * S, cuda))
    old = rand((S, 1, hd), 1, F16, cuda), rand((S, 1, hd), 2, F16, cuda)
    p.append(1, *old)
    cos, sin = tables(20, hd, cuda)
    big = rand((S, 4, hd + 8), 3, F16, cuda)
    q, k, v = big[:, :2, :hd], big[:, 2:3, :hd], big[:, 3:, :hd]
    place = torch.full((S, 2, 2 * hd), 7.0, dtype=F16, device=cuda)
    depth = ints([(0, -5, 16, 15, -2 ** 30, 2 ** 31 - 1)[s % 6] for s in range(S)], cuda)
    out = p.append_rope(1, q, k, v, cos, sin, depth=depth, out=place[..., :hd])
    at = 4 + depth.long()
    inside = (at >= 0) & (at < 20)
    want = turn(q, None, cos[at.clamp(0, 19)], sin[at.clamp(0, 19)], False).float().half()
    assert out.data_ptr() == place.data_ptr() and (place[..., hd:] == 7).all()
    assert torch.equal(out, torch.where(inside[:, None, None], want, 0.0))
    gk, gv = p.read(1, S)
    wk = turn(k, None, cos[at.clamp(0, 19)], sin[at.clamp(0, 19)], False).float().half()
    for got, new, was in ((gk, wk, old[0]), (gv, v, old[1])):
        assert torch.equal(got, torch.where(inside[:, None, None], q4(new), q4(was)).half())
    assert not p.pages[0].any()


# ------------------------------------------------------------------------------ trees
@pytest.mark.parametrize("words", [1, 2, 4])
def test_draft_tree(hiplib, cuda, words):
    """Masks and depths of trees, chains and forests; parents that are none; rows past the words; rows of no slot are left."""
    from sx8_draft import draft_tree
    ns = [1, 0, 5, 64, 63, 200, 256, 300, 2]
    ps = trees(ns, 1)
    ps[3] = trees([64], 0, chain=True)[0]
    ps[6] = trees([256], 0, chain=True)[0]
    ps[2] = [-1, 0, 2, 9, -7]                                        # itself, a later row, below -1: none
    mask, depth = draft_tree(ints(flat(ps) + [0, 0], cuda), cum(ns, cuda), words)
    sets = [ancestors(p) for p in ps]
    want = words_of(flat([[s if i < 64 * words else () for i, s in enumerate(x)] for x in sets]), words)
    far = flat([[len(s) - 1 if i < 64 * words else -2 ** 30 for i, s in enumerate(x)] for x in sets])
    assert torch.equal(mask[:-2].cpu(), want) and depth[:-2].tolist() == far


CASES = [  # hd, heads, kv heads, page tokens, tokens before, new rows
    (64, 4, 1, 32, [0, 1, 31, 500], [1, 3, 5, 8]),
    (128, 8, 2, 64, [700, 0, 33], [8, 40, 64]),
    (128, 4, 4, 128, [95, 96, 1000], [2, 1, 31]),
    (256, 16, 2, 32, [130, 20], [9, 64]),
    (256, 2, 2, 64, [0, 300], [0, 3]),
    (128, 40, 2, 64, [64, 4000], [11, 13]),
    (64, 16, 1, 256, [3000], [64]),
]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_tree(hiplib, cuda, case, dt):
    """Trees, and masks of any bits: rows that see nothing new, bits of rows that the slot does not have."""
    hd, nh, nk, pt, before, new = case
    lens = [a + b for a, b in zip(before, new)]
    p, k, v = make(cuda, lens, nk, hd, pt, dt)
    k, v = q4(k), q4(v)
    q = rand((sum(new), nh, hd), 9, dt, cuda, 2.0)
    for kind in ("tree", "any"):
        rng = random.Random(5)
        sets = [ancestors(t) if kind == "tree" else [frozenset(j for j in range(64) if rng.random() < rng.choice([0, 0.2, 1])) for _ in t]
                for t in trees(new, 3)]
        got = p.attend_tree(0, q, words_of(flat(sets), 1).to(cuda), cum(new, cuda))
        a, b, want = 0, 0, []
        for n, ln, s in zip(new, lens, sets):
            want.append(want_tree(q[a:a + n].double(), k[b:b + ln], v[b:b + ln], ln - n, s))
            a, b = a + n, b + ln
        close(got, torch.cat(want), dt, v.abs().max().item())


def test_attend_tree_words(hiplib, cuda):
    """More than 64 drafted tokens a slot, at offsets of the mask's words against the blocks of every kind; rows past the words."""
    p, k, v = make(cuda, [7 + 200, 256, 40 + 300], 1, 128, 32)
    k, v, new, lens = q4(k), q4(v), [200, 256, 300], [207, 256, 340]
    q = rand((sum(new), 2, 128), 9, F16, cuda, 2.0)
    sets = [ancestors(t) for t in trees(new, 3)]
    for words in (4, 3, 2):
        got = p.attend_tree(0, q, words_of(flat(sets), words).to(cuda), cum(new, cuda))
        a, b, want = 0, 0, []
        for n, ln, s in zip(new, lens, sets):
            cut = [{j for j in x if j < 64 * words} for x in s]
            want.append(want_tree(q[a:a + n].double(), k[b:b + ln], v[b:b + ln], ln - n, cut))
            a, b = a + n, b + ln
        close(got, torch.cat(want), F16, v.abs().max().item())


@pytest.mark.parametrize("hd,rep", [(64, 1), (128, 4), (256, 8)])
def test_attend_tree_is_attend(hiplib, cuda, hd, rep):
    """Chains are what `attend` computes; one row a slot without cu; 80 slots of very different lengths, cut over many
    work-groups; rows of no slot are left as they are, strided rows and outputs."""
    lens = [(s * 977) % 3000 + 9 for s in range(80)]
    p, k, v = make(cuda, lens, 1, hd, 64)
    new = [s % 8 + 1 for s in range(80)]
    T = sum(new)
    wide = rand((T + 3, rep, hd + 16), 4, F16, cuda)
    q = wide[..., 8:hd + 8]
    sets = flat([[range(i + 1) for i in range(n)] for n in new] + [[[0]] * 3])
    room = torch.full((T + 3, rep, hd + 8), 5.0, dtype=F16, device=cuda)
    got = p.attend_tree(0, q, words_of(sets, 1).to(cuda), cum(new, cuda), scale=0.2, out=room[..., :hd])
    want = p.attend(0, q, cum(new, cuda), scale=0.2)
    top = v.abs().max().item()
    close(got[:T], want[:T].double(), F16, top, more=2.0 ** -11)     # (two results of half a step each)
    assert (room[T:] == 5).all() and (room[..., hd:] == 5).all()
    one = p.attend_tree(0, q[:80].contiguous(), torch.ones(80, 1, dtype=torch.int64, device=cuda))
    close(one, p.attend(0, q[:80].contiguous()).double(), F16, top, more=2.0 ** -11)


def test_attend_tree_odd_values(hiplib, cuda):
    """A NaN in a drafted token's K or V reaches the rows that attend it and no others, however small its weight; large
    values of V; zero queries; pages that the table does not have."""
    new, lens = [12, 7], [12 + 50, 7 + 90]
    p, k, v = make(cuda, lens, 2, 128, 32, spare=2)
    T = sum(new)
    fresh_k, fresh_v = rand((T, 2, 128), 5, F16, cuda), rand((T, 2, 128), 6, F16, cuda)
    fresh_v[3, 0, 5] = math.nan                                      # first group of slot 0's row 3
    fresh_v[14, 1, 100] = math.inf                                   # second group of slot 1's row 2
    fresh_k[8, 1, 70] = math.nan
    fresh_v[1] *= 3000
    p.append(0, fresh_k, fresh_v, cum(new, cuda))
    kk, vv = torch.cat([k[:50], fresh_k[:12], k[62:62 + 90], fresh_k[12:]]), torch.cat([v[:50], fresh_v[:12], v[62:62 + 90], fresh_v[12:]])
    kk, vv = q4(kk), q4(vv)
    q = rand((T, 4, 128), 9, F16, cuda, 2.0)
    q[6] = 0
    fresh = torch.linspace(0, 30, T, device=cuda)[:, None, None].half()
    q = (q.float() * (1 + fresh.float() * 0.2)).half()
    sets = [ancestors(t) for t in trees(new, 8)]
    got = p.attend_tree(0, q, words_of(flat(sets), 1).to(cuda), cum(new, cuda))
    want = torch.cat([want_tree(q[:12].double(), kk[:62], vv[:62], 50, sets[0]), want_tree(q[12:].double(), kk[62:], vv[62:], 90, sets[1])])
    # (a NaN in K: every row that attends it, in all dimensions)
    for i, s in enumerate(sets[0]):
        if 8 in s:
            want[i, 2:] = math.nan
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    close(got, want, F16, vv[torch.isfinite(vv)].abs().max().item())
    # a page number that is none: its tokens are no tokens, wherever they lie
    p, k, v = make(cuda, lens, 2, 128, 32)
    kq, vq = q4(k), q4(v)
    p.table[0, 0], p.table[1, 2] = -1, 10 ** 6
    got = p.attend_tree(0, q, words_of(flat(sets), 1).to(cuda), cum(new, cuda))
    keep0, keep1 = list(range(32, 62)), [i for i in range(97) if not 64 <= i < 96]
    w0 = want_tree(q[:12].double(), kq[keep0], vq[keep0], 50 - 32, sets[0])
    w1 = want_tree(q[12:].double(), kq[[62 + i for i in keep1]], vq[[62 + i for i in keep1]], 64, [{j - 6 for j in s if j >= 6} for s in sets[1]])
    close(got, torch.cat([w0, w1]), F16, vq.abs().max().item())


def test_attend_tree_more_rows_than_tokens(hiplib, cuda):
    """A slot whose lens is below its number of rows: positions below zero are no tokens; no tokens at all: zeros."""
    p, k, v = make(cuda, [3, 0, 40], 1, 64, 32)
    kq, vq = q4(k), q4(v)
    new = [5, 2, 1]
    q = rand((8, 2, 64), 9, F16, cuda, 2.0)
    sets = [[{0}, {0, 1}, {1, 2}, {3, 4}, {4}], [{0}, {1}], [set()]]
    got = p.attend_tree(0, q, words_of(flat(sets), 1).to(cuda), cum(new, cuda))
    assert not got[0:2].any() and not got[5:7].any()
    want = want_tree(q[:5].double(), kq[:3], vq[:3], -2, sets[0])
    close(got[:5], torch.where(torch.isnan(want), 0.0, want), F16, vq.abs().max().item())
    close(got[7:], want_tree(q[7:].double(), kq[3:], vq[3:], 39, [set()]), F16, vq.abs().max().item())


# ------------------------------------------------------------------------------ verification
def run_verify(cuda, logits, ps, tokens, u, temp, probs=None, number=None):
    from sx8_draft import verify_draft
    ns = [len(p) for p in ps]
    t = number if number is not None else torch.tensor(temp, dtype=torch.float32, device=cuda)
    path, counts, nxt = verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cum(ns, cuda),
                                     None if u is None else torch.tensor(u, dtype=torch.float32, device=cuda), t, probs)
    a, want = 0, []
    host, hp = logits.float().cpu().numpy(), None if probs is None else probs.float().cpu().numpy()
    u = [0.0] * len(tokens) if u is None else torch.tensor(u, dtype=torch.float32).tolist()
    temp = torch.tensor(temp, dtype=torch.float32).tolist()
    for s, n in enumerate(ns):
        if n == 0:
            want.append(([], -1))
        else:
            want.append(want_verify(host[a:a + n], tokens[a:a + n], ps[s], u[a:a + n], temp[s], None if hp is None else hp[a:a + n]))
        a += n
    got_path, a = path.tolist(), 0
    for s, (kept, token) in enumerate(want):
        assert got_path[a:a + ns[s]] == kept + [-1] * (ns[s] - len(kept)), s
        assert counts[s].item() == len(kept) and nxt[s].item() == token, s
        a += ns[s]
    return path, counts, nxt


def drafts(cuda, ns, V, seed, dt=F32, chain=False, probs=False):
    """Trees whose tokens are likely ones of the target (or drawn from draft probabilities near it)."""
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    T, ps = sum(ns), trees(ns, seed, chain)
    logits = (torch.randn(T, V, generator=g) * 3).to(dt)
    q = torch.softmax(logits.float() + torch.randn(T, V, generator=g), -1) if probs else None
    tokens, a = [], 0
    for p in ps:
        for i, up in enumerate(p):
            row = a + max(up, 0)
            if probs:
                w = q[row].double().numpy()
                tokens.append(int(rng.choice(V, p=w / w.sum())))
            else:
                tokens.append(int(logits[row].float().topk(min(4, V)).indices[rng.integers(min(4, V))]))
        a += len(p)
    return logits.to(cuda), ps, tokens, rng.random(T, dtype=np.float32).tolist(), None if q is None else q.to(cuda)


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 8192, 8193, 40001])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_verify(hiplib, cuda, V, dt):
    """Trees and chains at several temperatures, greedy slots and empty ones among them."""
    ns = [1, 5, 0, 40, 2, 70, 7, 3]
    logits, ps, tokens, u, _ = drafts(cuda, ns, V, V, dt)
    run_verify(cuda, logits, ps, tokens, u, [0.7, 1.0, 1.0, 0.3, 0.0, 1.5, -1.0, 20.0])


@pytest.mark.parametrize("V", [2, 50, 8192, 20001])
@pytest.mark.parametrize("dt,pdt", [(F32, F32), (BF16, F16), (F16, BF16)])
@pytest.mark.parametrize("chain", [True, False])
def test_verify_with_draft_probabilities(hiplib, cuda, V, dt, pdt, chain):
    ns = [1, 6, 0, 17, 66, 4]
    logits, ps, tokens, u, q = drafts(cuda, ns, V, V + 1, dt, chain, probs=True)
    run_verify(cuda, logits, ps, tokens, u, [0.7, 1.0, 1.0, 0.9, 1.3, 0.0], q.to(pdt))


def test_verify_special(hiplib, cuda):
    """Rows without any finite logit, NaN and infinities, the same token twice, tokens outside the vocabulary, uniforms of 0
    and 1, an endless temperature, siblings that take the whole distribution, parents that are none."""
    V, inf, nan = 300, math.inf, math.nan
    base = torch.randn(40, V, generator=torch.Generator().manual_seed(1))

    def check(logits, parents, tokens, u, temp, probs=None):
        run_verify(cuda, torch.stack(logits).to(cuda), [parents], tokens, u, [temp], None if probs is None else torch.stack(probs).to(cuda))

    none = torch.full((V,), -inf)
    check([none], [-1], [5], [0.5], 1.0)
    check([none, base[0]], [-1, 0], [5, 5], [0.5, 0.0], 1.0)
    check([none, base[0]], [-1, 0], [5, 5], [0.5, 0.0], 0.0)
    two = base[1].clone()
    two[7] = two[200] = inf
    for u in (0.0, 0.49, 0.5, 0.75):
        check([two], [-1], [5], [u], 1.0)
        check([two, base[2]], [-1, 0], [5, 200], [u, u], 0.8)
    holes = base[3].clone()
    holes[::2] = nan
    holes[1:200:2] = -inf
    for u in (0.0, 0.3, 0.999):
        check([holes, base[1]], [-1, 0], [5, 201], [u, 0.001], 1.0)
        check([holes, base[1]], [-1, 0], [5, 2], [u, 0.0], inf)
    check([holes, base[1]], [-1, 0], [5, int(holes.nan_to_num(-inf).argmax())], [0.2, 0.2], 0.0)
    # the same token twice, and tokens that are none
    top = base[4].topk(3).indices.tolist()
    for t in ([top[0]] * 3, [top[0], top[1], top[0]], [-1, V, top[0]], [2 ** 40, top[1], -2 ** 40]):
        for u in ([0.5, 0.99, 0.99, 0.99], [0.9, 0.0, 0.0, 0.0], [0.1, 0.9, 0.0, 0.01]):
            check([base[4], base[5], base[6], base[7]], [-1, 0, 0, 0], [1] + t, u, 0.5)
            check([base[4], base[5], base[6], base[7]], [-1, 0, 0, 0], [1] + t, u, 0.5, [torch.softmax(base[8 + i], -1) for i in range(4)])
    # siblings of the whole vocabulary, all refused: the target's own again
    small = [torch.randn(3, generator=torch.Generator().manual_seed(i)) for i in range(4)]
    run_verify(cuda, torch.stack(small).to(cuda), [[-1, 0, 0, 0]], [0, 0, 1, 2], [0.4, 1.0, 1.0, 1.0], [1.0])
    # p = draft probabilities: nothing is left of p - q
    p = torch.tensor([0.5, 0.25, 0.25, 0.0])
    run_verify(cuda, p.log().repeat(2, 1).to(cuda), [[-1, 0]], [0, 1], [0.6, 1.0], [1.0], p.repeat(2, 1).to(cuda))
    # parents that are none: never a child
    check([base[9], base[10], base[11]], [-1, 1, 5], [0, top[0], top[0]], [0.3, 0.0, 0.0], 1.0)
    check([base[9], base[10], base[11]], [-1, -1, 0], [0, 3, 4], [0.3, 0.0, 0.0], 1.0)


def test_verify_numbers_and_strides(hiplib, cuda):
    """A number as temperature, greedy without uniforms, logits that are a part of wider rows, more than 64 slots, rows of no
    slot left as they are."""
    from sx8_draft import verify_draft
    ns = [s % 4 for s in range(150)]
    logits, ps, tokens, u, _ = drafts(cuda, ns, 777, 5)
    wide = torch.zeros(logits.shape[0], 1000, device=cuda)
    wide[:, 100:877] = logits
    run_verify(cuda, wide[:, 100:877], ps, tokens, u, [0.9] * 150, number=0.9)
    run_verify(cuda, logits, ps, tokens, None, [0.0] * 150, number=0)
    T = len(tokens)
    more = lambda x, n: torch.cat([x, x[:n]])  # noqa: E731
    path, counts, nxt = verify_draft(more(logits, 4), more(torch.tensor(tokens, device=cuda), 4), more(ints(flat(ps), cuda), 4),
                                     cum(ns, cuda), more(torch.tensor(u, device=cuda), 4), 0.9)
    first = verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cum(ns, cuda), torch.tensor(u, device=cuda), 0.9)
    assert torch.equal(path[:T], first[0]) and torch.equal(counts, first[1]) and torch.equal(nxt, first[2])


def test_verify_keeps_the_distribution(hiplib, cuda):
    """The first token that comes out (the first kept draft, or the drawn one) has the target's probabilities: 60000 slots'
    worth of draws of a vocabulary of 6, drafts chosen and drafts drawn.  Frequencies of n draws differ from p by
    sqrt(p (1 - p) / n) <= 0.0021 in the mean square; five of these are exceeded once in two million."""
    from sx8_draft import verify_draft
    S, V, n = 4000, 6, 4
    logits = torch.tensor([0.3, 1.2, -0.5, 0.0, 2.0, -1.0], device=cuda)
    want = torch.softmax(logits / 0.8, -1)
    q = torch.softmax(torch.tensor([1.0, 0.5, 0.5, 0.0, 0.5, 0.0], device=cuda), -1)
    rows = logits.repeat(S * n, 1)
    parents = ints([-1, 0, 0, 0] * S, cuda)
    cu = ints(range(0, S * n + 1, n), cuda)
    g = torch.Generator(device=cuda).manual_seed(3)
    for drawn in (False, True):
        hits, draws = torch.zeros(V, device=cuda), 0
        for _ in range(15):
            if drawn:
                tok = torch.multinomial(q, S * n, replacement=True, generator=g)
            else:
                tok = torch.tensor([0, 4, 1, 1], device=cuda).repeat(S)
            u = torch.rand(S * n, generator=g, device=cuda)
            path, counts, nxt = verify_draft(rows, tok, parents, cu, u, 0.8, q.repeat(S * n, 1) if drawn else None)
            kept = path.view(S, n)[:, 1].long().clamp(min=0)
            first = torch.where(counts > 1, tok.view(S, n).gather(1, kept[:, None])[:, 0], nxt)
            hits += torch.bincount(first, minlength=V)
            draws += S
        assert ((hits / draws - want).abs() < 5 * 0.0021).all(), (drawn, hits / draws, want)


# ------------------------------------------------------------------------------ keep
@pytest.mark.parametrize("hd,pt,nk", [(64, 32, 3), (128, 64, 2), (256, 32, 1), (128, 256, 2)])
def test_keep(hiplib, cuda, hd, pt, nk):
    """Kept rows of every layer lie together behind the earlier tokens, bit for bit; lens, tables and counts follow; other
    slots and a shared page keep theirs."""
    new = [1, 9, 40, 0, 33, 70, 8, 4]
    lens = [n + b for n, b in zip(new, [0, 30, 60, 5, 95, 127, 64, 3])]
    p, _, _ = make(cuda, lens, nk, hd, pt, layers=3, spare=3)
    rng = random.Random(2)
    kept = [[0], [0, 3, 8], sorted(rng.sample(range(40), 17)), [], list(range(33)), sorted(rng.sample(range(70), 35)), [], [3]]
    # bits, not values: layers of their own
    p.pages.copy_(torch.randint(0, 256, p.pages.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1)).to(cuda))
    for i in (0, 1):                                                 # (scales that are numbers, so that values can be compared)
        T = sum(lens)
        p.append(i, rand((T, nk, hd), 5 + i, F16, cuda), rand((T, nk, hd), 7 + i, F16, cuda), cum(lens, cuda))
    was = [p.read(i, sum(lens), cum(lens, cuda)) for i in (0, 1)]
    raw, table, refs = p.pages.clone(), p.table.clone(), p.refs.clone()
    path = flat([k + [-1] * (n - len(k)) for k, n in zip(kept, new)])
    p.keep(ints(path, cuda), ints([len(k) for k in kept], cuda), cum(new, cuda))
    p.check()
    after = [ln - n + len(k) for ln, n, k in zip(lens, new, kept)]
    assert p.lens.tolist() == after
    for s, ln in enumerate(after):
        have = (ln + pt - 1) // pt
        assert torch.equal(p.table[s, :have], table[s, :have]) and (p.table[s, have:] == -1).all()
        gone = table[s, have:]
        gone = gone[gone >= 0].long()
        assert (p.refs[gone] == 0).all()
    assert p.refs.sum() == refs.sum() - ((table >= 0).sum() - (p.table >= 0).sum())
    starts = [sum(lens[:s]) for s in range(len(lens))]
    at = flat([list(range(starts[s], starts[s] + lens[s] - new[s])) + [starts[s] + lens[s] - new[s] + j for j in kept[s]] for s in range(len(lens))])
    for i in (0, 1):
        got = p.read(i, sum(after), cum(after, cuda))
        for g, w in zip(got, was[i]):
            assert torch.equal(g, w[at])
    # a slot that kept its first rows, and pages that nobody moves in: untouched
    same = torch.ones(p.n_pages, dtype=torch.bool, device=cuda)
    for s in (1, 2, 5, 7):
        pages = table[s, (lens[s] - new[s]) // pt:]
        same[pages[pages >= 0].long()] = False
    assert torch.equal(p.pages[:, same], raw[:, same])


def test_keep_refuses(hiplib, cuda):
    """Counts and rows that are none: the status says which slot, and nothing changes; slots without rows; without cu."""
    for path, counts, new, slot in (([0, 1, 2, 0, -1], [3, 3], [3, 2], 1), ([0, 0, 2, 0, 1], [2, 1], [3, 2], 0), ([0, 3, 2, 0, 1], [2, 1], [3, 2], 0),
                                    ([0, 1, 2, 0, 1], [-1, 1], [3, 2], 0), ([0, 1, 2, 0, 1], [3, 1], [5, 0], 1), ([-1, 1, 2, 0, 1], [2, 2], [3, 2], 0),
                                    ([0, 1, 2, 3, 4], [0, 1], [0, 5], 1)):
        p, _, _ = make(cuda, [40, 4], 1, 64, 32)
        before = [t.clone() for t in (p.pages, p.table, p.lens, p.refs)]
        p.keep(ints(path, cuda), ints(counts, cuda), cum(new, cuda))
        with pytest.raises(RuntimeError, match=rf"bad slot or count \(slot or entry {slot}\)"):
            p.check()
        assert all(torch.equal(a, b) for a, b in zip(before, (p.pages, p.table, p.lens, p.refs)))
    p, _, _ = make(cuda, [40, 33], 1, 64, 32)
    p.keep(ints([0, 0], cuda), ints([1, 0], cuda))
    p.check()
    assert p.lens.tolist() == [40, 32] and p.table[1, 1] == -1 and p.refs.tolist() == [1, 1, 1, 0]
    p.keep(ints([], cuda), ints([0, 0], cuda), ints([0, 0, 0], cuda))
    # a cu that runs backwards names more rows than there are
    p.keep(ints([0] * 6, cuda), ints([0, 0], cuda), ints([0, 6, 0], cuda))
    p.check()


def test_keep_many_rows(hiplib, cuda):
    """Hundreds of kept rows of a slot; one of them out of order, anywhere, refuses the call."""
    n, before = 700, 50
    p, _, _ = make(cuda, [before + n, 3], 1, 64, 32, spare=2, width=30)
    kept = sorted(random.Random(3).sample(range(n), 403))
    was = p.read(0, before + n + 3, cum([before + n, 3], cuda))
    cu, counts = cum([n, 1], cuda), ints([len(kept), 1], cuda)
    state = [t.clone() for t in (p.pages, p.table, p.lens, p.refs)]
    for i in (1, 7, 8, 200, 402):
        for value in (kept[i - 1], n, -1):
            path = kept[:i] + [value] + kept[i + 1:] + [-1] * (n - len(kept)) + [0]
            p.keep(ints(path, cuda), counts, cu)
            with pytest.raises(RuntimeError, match=r"bad slot or count \(slot or entry 0\)"):
                p.check()
    assert all(torch.equal(a, b) for a, b in zip(state, (p.pages, p.table, p.lens, p.refs)))
    p.keep(ints(kept + [-1] * (n - len(kept)) + [0], cuda), counts, cu)
    p.check()
    lens = [before + len(kept), 3]
    at = list(range(before)) + [before + j for j in kept] + [before + n + j for j in range(3)]
    assert p.lens.tolist() == lens
    for g, w in zip(p.read(0, sum(lens), cum(lens, cuda)), was):
        assert torch.equal(g, w[at])


# ------------------------------------------------------------------------------ together
def round_of(p, seed, new, ps, cuda, cos, sin, V=500):
    """One checking pass of a single layer, as a program makes it; returns its outputs."""
    from sx8_draft import draft_tree, verify_draft
    T, cu = sum(new), cum(new, cuda)
    p.reserve(ints(new, cuda))
    q, k, v = (rand((T, n, 64), seed + i, F16, cuda) for i, n in enumerate((4, 2, 2)))
    logits, _, tokens, u, _ = drafts(cuda, new, V, seed)
    args = (q, k, v, logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), torch.tensor(u, device=cuda), cu)

    def run(q, k, v, logits, tokens, parents, u, cu):
        mask, depth = draft_tree(parents, cu)
        qr = p.append_rope(0, q, k, v, cos, sin, cu, depth=depth)
        o = p.attend_tree(0, qr, mask, cu)
        path, counts, nxt = verify_draft(logits, tokens, parents, cu, u, 0.8)
        p.keep(path, counts, cu)
        return mask, depth, qr, o, path, counts, nxt
    return run, args


def test_round_captured(hiplib, cuda):
    """A whole pass on a stream of its own, and captured: every replay, with eager work between them, gives what the eager
    calls give from the same cache."""
    p, _, _ = make(cuda, [40, 3, 0, 90], 2, 64, 32, spare=12, width=8)
    cos, sin = tables(200, 64, cuda)
    new = [5, 1, 0, 9]
    ps = trees(new, 4)
    run, args = round_of(p, 20, new, ps, cuda, cos, sin)
    state = [t.clone() for t in (p.pages, p.table, p.lens, p.refs)]

    def back():
        for t, w in zip((p.pages, p.table, p.lens, p.refs), state):
            t.copy_(w)

    def results(outs):
        torch.cuda.synchronize()
        return [t.clone() for t in (*outs, p.pages, p.table, p.lens, p.refs)]

    want = results(run(*args))
    p.check()
    side = torch.cuda.Stream()
    back()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = run(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results(outs), want))
    back()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run(*args)
    for i in range(4):
        back()
        g.replay()
        got = results(outs)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        back()
        assert all(torch.equal(a, b) for a, b in zip(results(run(*args)), want)), i
    p.check()
    # K, V and attention of the kept rows are those of a cache that only ever saw them
    kept = want[4].tolist()
    q4v = p.read(0, sum(p.lens.tolist()), cum(p.lens.tolist(), cuda))
    k, v = args[1], args[2]
    cu, a = cum(new, cuda).tolist(), 0
    for s, ln in enumerate(p.lens.tolist()):
        rows = [r for r in kept[cu[s]:cu[s + 1]] if r >= 0]
        first = ln - len(rows)
        if rows:
            at = [cu[s] + r for r in rows]
            place = list(range(first, ln))                           # (a kept row's depth is its place among the kept)
            want_k = turn(k[at], None, cos[place], sin[place], False).float().half()
            assert torch.equal(q4v[0][a + first:a + ln], q4(want_k).half()) and torch.equal(q4v[1][a + first:a + ln], q4(v[at]).half())
        a += ln


def test_round_of_long_trees(hiplib, cuda):
    """Trees of more than 64 rows through the whole pass: four words a mask, rows past them out of every later step."""
    from sx8_draft import draft_tree
    new, before = [200, 300, 256], [10, 0, 33]
    p, k0, v0 = make(cuda, before, 2, 64, 32, spare=40, width=12)
    cos, sin = tables(400, 64, cuda)
    ps, T, cu = trees(new, 6), sum(new), cum(new, cuda)
    p.reserve(ints(new, cuda))
    q, k, v = (rand((T, n, 64), 30 + i, F16, cuda) for i, n in enumerate((4, 2, 2)))
    p.append(0, torch.zeros_like(k), torch.zeros_like(v), cu)
    mask, depth = draft_tree(ints(flat(ps), cuda), cu, 4)
    qr = p.append_rope(0, q, k, v, cos, sin, cu, depth=depth)
    out = p.attend_tree(0, qr, mask, cu)
    a, b, want = 0, 0, []
    for n, f, tree in zip(new, before, ps):
        sets = [s if i < 256 else frozenset() for i, s in enumerate(ancestors(tree))]
        at = [f + len(s) - 1 for s in sets[:256]]
        turned = torch.zeros(n, 2, 64, dtype=F16, device=cuda)
        turned[:256] = turn(k[a:a + min(n, 256)], None, cos[at], sin[at], False).float().half()
        vv = v[a:a + n].clone()
        vv[256:] = 0
        kk, vv = torch.cat([k0[b:b + f], turned]), torch.cat([v0[b:b + f], vv])
        want.append(want_tree(qr[a:a + n].double(), q4(kk), q4(vv), f, sets))
        assert not qr[a + 256:a + n].any() or n <= 256
        a, b = a + n, b + f
    close(out, torch.cat(want), F16, q4(v).abs().max().item())
    kept = [list(range(0, n, 7))[:20] for n in new]
    was = p.read(0, sum(before) + T, cum([f + n for f, n in zip(before, new)], cuda))
    p.keep(ints(flat([x + [-1] * (n - len(x)) for x, n in zip(kept, new)]), cuda), ints([len(x) for x in kept], cuda), cu)
    p.check()
    lens = [f + len(x) for f, x in zip(before, kept)]
    assert p.lens.tolist() == lens
    starts = [0, 210, 510]
    at = flat([list(range(s, s + f)) + [s + f + j for j in x] for s, f, x in zip(starts, before, kept)])
    for g, w in zip(p.read(0, sum(lens), cum(lens, cuda)), was):
        assert torch.equal(g, w[at])


def test_two_rounds_at_once(hiplib, cuda):
    """Two caches on two streams at once, then as two captured graphs replayed side by side."""
    cos, sin = tables(1500, 64, cuda)
    pools = [make(cuda, [700 + 100 * i, 3, 40], 2, 64, 32, spare=12, width=32, seed=i)[0] for i in range(2)]
    states = [[t.clone() for t in (p.pages, p.table, p.lens, p.refs)] for p in pools]
    work = [round_of(p, 20 + i, [9, 1, 30], trees([9, 1, 30], i), cuda, cos, sin) for i, p in enumerate(pools)]

    def back(i):
        for t, w in zip((pools[i].pages, pools[i].table, pools[i].lens, pools[i].refs), states[i]):
            t.copy_(w)

    def grown(i):
        back(i)
        pools[i].reserve(ints([9, 1, 30], cuda))

    def all_of(i, outs):
        return [t.clone() for t in (*outs, pools[i].pages, pools[i].table, pools[i].lens, pools[i].refs)]

    want = []
    for i in range(2):
        grown(i)
        want.append(all_of(i, work[i][0](*work[i][1])))
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    add = ints([9, 1, 30], cuda)
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                back(i)
                pools[i].reserve(add)
                got.append(all_of(i, work[i][0](*work[i][1])))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    for i in range(2):
        grown(i)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = work[i][0](*work[i][1])
        graphs.append((g, outs))
    for _ in range(5):
        torch.cuda.synchronize()
        for i in range(2):
            grown(i)
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i, (_, outs) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(all_of(i, outs), want[i]))
    for p in pools:
        p.check()


# ------------------------------------------------------------------------------ where calls could go wrong
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_tree_query_sizes(hiplib, cuda, dt):
    """Queries from tiny to large (bf16: far past fp16's range) keep their precision."""
    p, k, v = make(cuda, [300] * 6, 1, 64, 64, F16)
    q = rand((6, 2, 64), 4, F32, cuda)
    mags = [1e-6, 1e-3, 1.0, 30.0, 300.0, 0.0] if dt is F16 else [1e-30, 1e-3, 1.0, 1e6, 1e20, 0.0]
    q = (q * torch.tensor(mags, device=cuda)[:, None, None]).to(dt)
    ones = torch.ones(6, 1, dtype=torch.int64, device=cuda)
    kk, vv = q4(k), q4(v)
    for scale, rows in ((0.125, [0, 1, 2, 5]), (2.0 ** -9, [3] if dt is F16 else []), (2.0 ** -23, [3] if dt is BF16 else [4]),
                        (2.0 ** -69, [4] if dt is BF16 else [])):
        if rows:
            got = p.attend_tree(0, q, ones, scale=scale)
            want = torch.cat([want_tree(q[i:i + 1].double(), kk[300 * i:300 * i + 300], vv[300 * i:300 * i + 300], 299, [{0}], scale)
                              for i in rows])
            close(got[rows], want, dt, vv.abs().max().item())


@pytest.mark.parametrize("hd,rep", [(64, 16), (128, 32), (256, 16)])
def test_attend_tree_value_sizes(hiplib, cuda, hd, rep):
    """Blocks whose values grow from nothing to fp16's ends and back, for one tile of rows a unit and for two."""
    sizes = [0.0, 1e-6, 1e-3, 1.0, 100.0, 65504.0, 1.0, 0.0, 30.0]
    from sx8_paged_kv import PagedKV4
    n = 32 * len(sizes)
    p = PagedKV4(1, 1, hd, 9, 1, 9, 32, device=cuda)
    p.reserve(ints([n], cuda))
    k, v = rand((n, 1, hd), 1, F16, cuda), torch.zeros(n, 1, hd, dtype=F16, device=cuda)
    for i, size in enumerate(sizes):
        g = torch.Generator().manual_seed(i)
        v[32 * i:32 * i + 32] = ((torch.rand(32, 1, hd, generator=g) * 2 - 1) * size).half().to(cuda)
    p.append(0, k, v, cum([n], cuda))
    T = 8
    q = rand((T, rep, hd), 3, F16, cuda)
    for i in range(9):                                               # (heads that pick out one block each)
        q[:, i] = k[32 * i + 5, 0] * 4
    sets = [{j for j in range(T) if (i + j) % 3} for i in range(T)]
    got = p.attend_tree(0, q, words_of(sets, 1).to(cuda), cum([T], cuda)).double()
    kk, vv = q4(k), q4(v)
    want = want_tree(q.double(), kk, vv, n - T, sets)
    # a row's bound goes by the values that it gives weight, as in the test of `attend`
    top = want_tree(q.double(), kk, vv.abs().amax(-1, keepdim=True).expand(-1, -1, hd).contiguous(), n - T, sets)
    err = (got - want).abs()
    assert (err <= (2.0 ** -11 + LOOSE) * torch.maximum(top, want.abs()) + 2.0 ** -25).all(), (err / top.clamp(min=1e-9)).max()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attend_tree_bits_do_not_depend_on_old_bytes(hiplib, cuda, hd):
    """What lies behind a slot's last token in its page does not change a bit of the result, whatever it is."""
    from sx8_paged_kv import PagedKV4
    lens, new, got = [45, 1, 130], [3, 1, 33], []
    k, v = rand((sum(lens), 2, hd), 1, F16, cuda), rand((sum(lens), 2, hd), 2, F16, cuda)
    q = rand((sum(new), 4, hd), 3, F16, cuda)
    mask = words_of(flat([ancestors(t) for t in trees(new, 3)]), 1).to(cuda)
    for seed in range(4):
        p = PagedKV4(1, 2, hd, 8, 3, 3, 64, device=cuda)
        if seed == 3:
            p.pages.fill_(255)                                       # (scales and minima that are NaN)
        elif seed:
            p.pages.copy_(torch.randint(0, 256, p.pages.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8))
        p.reserve(ints(lens, cuda))
        p.append(0, k, v, cum(lens, cuda))
        got.append(p.attend_tree(0, q, mask, cum(new, cuda)))
    assert not torch.isnan(got[0]).any() and all(torch.equal(g, got[0]) for g in got)


@pytest.mark.parametrize("n_slots", [64, 65, 4096])
def test_many_slots(hiplib, cuda, n_slots):
    """Slots without rows, with one, with trees, at 64 (the last number whose line a wave holds) and far more."""
    from sx8_draft import draft_tree, verify_draft
    from sx8_paged_kv import PagedKV4
    hd, nk, rng = 64, 2, random.Random(n_slots)
    new = [rng.choice([0, 0, 1, 2, 5]) for _ in range(n_slots)]
    new[n_slots // 2] = 20
    lens = [n + rng.choice([0, 1, 40]) for n in new]
    p = PagedKV4(1, nk, hd, 3 * n_slots, n_slots, 4, 32, device=cuda)
    p.reserve(ints(lens, cuda))
    k, v = rand((sum(lens), nk, hd), 1, F16, cuda), rand((sum(lens), nk, hd), 2, F16, cuda)
    p.append(0, k, v, cum(lens, cuda))
    cos, sin = tables(80, hd, cuda)
    T, cu, ps = sum(new), cum(new, cuda), trees(new, 1)
    q, nkr, nvr = (rand((T, n, hd), 5 + i, F16, cuda) for i, n in enumerate((4, nk, nk)))
    mask, depth = draft_tree(ints(flat(ps), cuda), cu)
    sets = [ancestors(t) for t in ps]
    assert torch.equal(mask.cpu(), words_of(flat(sets), 1)) and depth.tolist() == [len(s) - 1 for x in sets for s in x]
    qr = p.append_rope(0, q, nkr, nvr, cos, sin, cu, depth=depth)
    at = [ln - n + len(s) - 1 for ln, n, x in zip(lens, new, sets) for s in x]
    assert torch.equal(qr, turn(q, None, cos[at], sin[at], False).float().half())
    kt = turn(nkr, None, cos[at], sin[at], False).float().half()
    out = p.attend_tree(0, qr, mask, cu)
    a, b, checked = 0, 0, 0
    for n, ln, x in zip(new, lens, sets):
        if n and checked < 150:
            checked += 1
            kk, vv = (q4(torch.cat([old[b:b + ln - n], fresh[a:a + n]])) for old, fresh in ((k, kt), (v, nvr)))
            close(out[a:a + n], want_tree(qr[a:a + n].double(), kk, vv, ln - n, x), F16, 6.0)
        a, b = a + n, b + ln
    logits, _, tokens, u, _ = drafts(cuda, new, 40, 3)
    path, counts, nxt = run_verify(cuda, logits, ps, tokens, u, [0.8] * n_slots)
    assert [t.tolist() for t in verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cu,
                                             torch.tensor(u, device=cuda), 0.8)] == [path.tolist(), counts.tolist(), nxt.tolist()]
    p.keep(path, counts, cu)
    p.check()
    assert p.lens.tolist() == [ln - n + c for ln, n, c in zip(lens, new, counts.tolist())]


@pytest.mark.parametrize("top,temp", [(20.0, 1e-9), (20.0, 1e-8), (20.0, 1e-6), (1.0, 1e-30), (1.0, 1e-44), (1e10, 1.0), (1e30, 1.0),
                                      (65504.0, 1e-6), (1e10, 1e9), (3e38, 3e37), (-1e30, 0.7), (1e-30, 1.0), (1e-42, 1e-42)])
@pytest.mark.parametrize("drawn", [False, True])
def test_verify_steep(hiplib, cuda, top, temp, drawn):
    """Temperatures far below a step of the logits, and logits whose steps are far above the temperature: the weights are
    those of the formula."""
    V, n = 5000, 6
    g = torch.Generator().manual_seed(4)
    logits = (torch.randn(n, V, generator=g) * abs(top) / 10).clamp(-abs(top), abs(top))
    logits[:, 17], logits[:, 4321] = abs(top), abs(top)
    logits = logits - (2 * abs(top) if top < 0 else 0)
    tokens, u = [0, 5, 17, 4321, 17, 4321], [0.51, 0.0, 0.7, 0.3, 0.2, 0.9]
    probs = torch.softmax(torch.randn(n, V, generator=g), -1).to(cuda) if drawn else None
    run_verify(cuda, logits.to(cuda), [[-1, 0, 0, 0, 2, 3]], tokens, u, [temp], probs)
    run_verify(cuda, logits.to(cuda), [[-1]] * n, tokens, [0.1, 0.4, 0.499, 0.501, 0.8, 0.99], [temp] * n)


def test_cu_backwards(hiplib, cuda):
    """A cu that names the same rows for many slots, and ends below its beginnings: no call leaves its memory."""
    from sx8_draft import draft_tree, verify_draft
    from sx8_paged_kv import PagedKV4
    n_slots = 4096
    p = PagedKV4(1, 1, 64, 2, n_slots, 1, 32, device=cuda)
    p.reserve(ints([1, 1] + [0] * (n_slots - 2), cuda))
    q, k = rand((64, 256, 64), 1, F16, cuda), rand((64, 1, 64), 1, F16, cuda)
    cos, sin = tables(40, 64, cuda)
    for cu in (ints([0, 64] * 2048 + [64], cuda), ints([-5, 70, 3] + [64, -2 ** 31] * 2047, cuda), ints([64] * 4097, cuda),
               ints([2 ** 31 - 1, 0] * 2048 + [9], cuda)):
        mask, depth = draft_tree(ints([-1] + [0] * 63, cuda), cu, 2)
        assert p.append_rope(0, q, k, k, cos, sin, cu).shape == q.shape
        ones = torch.full((64, 2), -1, dtype=torch.int64, device=cuda)
        assert p.attend_tree(0, q, ones, cu).shape == q.shape
        torch.cuda.synchronize()
        assert p.refs.tolist() == [1, 1]
    # long slots over the same rows, whose lists of refused tokens share their places
    T, V = 600, 50
    logits = torch.randn(T, V, generator=torch.Generator().manual_seed(1)).to(cuda)
    tokens, parents = (torch.arange(T, device=cuda) % V), ints([-1] + [0] * (T - 1), cuda)
    u = torch.full((T,), 0.999, device=cuda)
    for cu in ([0, 600, 300, 600, 0, 500], [300, 600, 0, 600, 100, 600]):
        path, counts, nxt = verify_draft(logits, tokens, parents, ints(cu, cuda), u, 1.0)
        torch.cuda.synchronize()
        assert path.shape == (T,) and (counts >= 0).all() and (counts <= T).all()


def test_past_four_gib(hiplib, cuda):
    """Pages whose bytes lie past 2^32: rows rotated into them, read as a tree, kept."""
    from sx8_paged_kv import PagedKV4
    nk, hd, pt = 8, 128, 128
    n_pages = (1 << 32) // PagedKV4._page_bytes(nk, hd, pt) + 40
    big = PagedKV4(1, nk, hd, n_pages, 2, 4, pt, device=cuda)
    small = PagedKV4(1, nk, hd, 8, 2, 4, pt, device=cuda)
    big.refs[:n_pages - 8] = 1                                      # all but the last pages are taken
    cos, sin = tables(400, hd, cuda)
    new, got = [20, 64], []
    q, k, v = (rand((300, n, hd), i, F16, cuda) for i, n in enumerate((2 * nk, nk, nk)))
    mask = words_of(flat([ancestors(t) for t in trees(new, 2)]), 1).to(cuda)
    path = flat([[j for j in range(0, n, 3)] + [-1] * (n - len(range(0, n, 3))) for n in new])
    for p in (big, small):
        p.reserve(ints([200, 100], cuda))
        p.append_rope(0, q, k, v, cos, sin, cum([200, 100], cuda))
        p.reserve(ints(new, cuda))
        qr = p.append_rope(0, q[:84], k[84:168], v[84:168], cos, sin, cum(new, cuda))
        out = p.attend_tree(0, qr, mask, cum(new, cuda))
        p.keep(ints(path, cuda), ints([7, 22], cuda), cum(new, cuda))
        p.check()
        got.append((qr, out, *p.read(0, 329, cum([207, 122], cuda)), p.lens))
    assert big.table.max() == n_pages - 8 + small.table.max() and (n_pages - 8) * big.page_bytes > 1 << 32
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_rows_past_four_gib(hiplib, cuda):
    """Query rows, logits and probabilities whose offsets pass 2^32 bytes."""
    from sx8_draft import verify_draft
    T, ts = 2100, 1 << 20
    big = torch.zeros(T * ts, dtype=F16, device=cuda)
    far = torch.as_strided(big, (T, 2, 64), (ts, 64, 1))
    far.copy_(rand((T, 2, 64), 1, F16, cuda))
    out = torch.as_strided(big, (T, 2, 64), (ts, 64, 1), 256)
    p, _, _ = make(cuda, [T + 50], 1, 64, 64)
    near, k = far.clone(), far[:, :1].clone()
    cos, sin = tables(T + 50, 64, cuda)
    cu = cum([T], cuda)
    p.append_rope(0, far, far[:, :1], far[:, 1:], cos, sin, cu, out=out)
    pages = p.pages.clone()
    assert torch.equal(out, p.append_rope(0, near, k, near[:, 1:].clone(), cos, sin, cu)) and torch.equal(p.pages, pages)
    mask = torch.full((T, 4), 0x5A5A5A5A, dtype=torch.int64, device=cuda)
    assert torch.equal(p.attend_tree(0, far, mask, cu, out=out), p.attend_tree(0, near, mask, cu))
    del big, far, out
    rows, V, stride = 20, 9000, 1 << 28
    pool = torch.empty(rows * stride, dtype=F16, device=cuda)
    logits, probs = (torch.as_strided(pool, (rows, V), (stride, 1), i << 20) for i in range(2))
    x, ps, tokens, u, pr = drafts(cuda, [12, 8], V, 5, F16, probs=True)
    logits.copy_(x)
    probs.copy_(pr.half())
    run_verify(cuda, logits, ps, tokens, u, [0.8, 1.2], probs)


def test_rows_with_gradients(hiplib, cuda):
    """Rows that require a gradient are read as values; outputs have none."""
    from sx8_draft import verify_draft
    p, k, v = make(cuda, [40, 9], 2, 64, 32)
    cos, sin = tables(60, 64, cuda)
    q, kk = rand((2, 4, 64), 5, F16, cuda).requires_grad_(), rand((2, 2, 64), 6, F16, cuda).requires_grad_()
    w = torch.nn.Parameter(torch.ones(64, dtype=F16, device=cuda))
    got = p.append_rope(0, q, kk, kk, cos, sin, q_norm=w, k_norm=w)
    ones = torch.ones(2, 1, dtype=torch.int64, device=cuda)
    x = torch.randn(2, 30, device=cuda, requires_grad=True)
    outs = [got, p.attend_tree(0, q, ones), *verify_draft(x, torch.zeros(2, dtype=torch.int64, device=cuda), ints([-1, -1], cuda), cum([1, 1], cuda))]
    assert not any(o.requires_grad for o in outs)


def test_general_path_gives_the_same(hiplib, cuda, monkeypatch):
    """Without the host module every call takes the wrappers' general path: the same results."""
    import _sx8lib
    from sx8_draft import draft_tree, verify_draft

    def run():
        p, _, _ = make(cuda, [40, 0, 70], 2, 128, 32, spare=8, width=8, layers=2)
        cos, sin = tables(200, 64, cuda)
        new = [5, 0, 20]
        ps, cu, T = trees(new, 4), cum(new, cuda), 25
        p.reserve(ints(new, cuda))
        w = rand((128,), 9, F16, cuda)
        outs = []
        for dt in (F16, F32):
            q, k, v = (rand((T, n, 128), 20 + i, dt, cuda) for i, n in enumerate((4, 2, 2)))
            mask, depth = draft_tree(ints(flat(ps), cuda), cu, 2)
            qr = p.append_rope(1, q, k, v, cos, sin, cu, depth=depth, q_norm=w, k_norm=w, eps=1e-5, interleaved=dt is F32)
            outs += [mask, depth, qr, p.attend_tree(1, qr, mask, cu), p.attend_tree(0, qr, mask, cu, scale=0.3), p.pages.clone()]
        outs.append(p.append_rope(0, q[:3], k[:3], v[:3], cos, sin, dtype=BF16))
        for dt, probs, temp in ((F32, False, 0.8), (BF16, True, torch.tensor([0.5, 1.0, 0.0], device=cuda)), (F16, False, 0.0)):
            logits, _, tokens, u, pr = drafts(cuda, new, 900, 3, dt, probs=probs)
            u = None if dt is F16 else torch.tensor(u, device=cuda)
            got = verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cu, u, temp, pr)
            outs += got
        p.keep(got[0], got[1], cu)
        p.keep(ints([0, 0, 0], cuda), ints([1, 0, 1], cuda), ints([0, 1, 1, 2], cuda))
        p.check()
        return outs + [p.pages, p.table, p.lens, p.refs]

    fast = run()
    assert isinstance(_sx8lib.py().kv4_attend_tree, type(len))      # the module is there
    monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    for i, (a, b) in enumerate(zip(fast, run())):
        assert torch.equal(a, b), i


def test_views_that_negate(hiplib, cuda):
    """They are read as the values they stand for; as outputs, masks or whole numbers they are refused."""
    from sx8_draft import draft_tree, verify_draft
    p, _, _ = make(cuda, [40, 9], 2, 64, 32)
    cos, sin = tables(60, 64, cuda)
    n = torch._neg_view
    q, k, v, w = (rand(s, i, F16, cuda) for i, s in enumerate(((2, 4, 64), (2, 2, 64), (2, 2, 64), (64,))))
    want = p.append_rope(0, q, k, v, cos, sin, q_norm=w, k_norm=w)
    pages = p.pages.clone()
    got = p.append_rope(0, n(-q), n(-k), n(-v), n(-cos), n(-sin), q_norm=n(-w), k_norm=n(-w))
    assert torch.equal(got, want) and torch.equal(p.pages, pages)
    ones = torch.ones(2, 1, dtype=torch.int64, device=cuda)
    assert torch.equal(p.attend_tree(0, n(-q), ones), p.attend_tree(0, q, ones))
    x, pr, u = torch.randn(2, 30, device=cuda), torch.rand(2, 30, device=cuda), torch.rand(2, device=cuda)
    tokens, parents, cu, temp = torch.tensor([3, 4], device=cuda), ints([-1, 0], cuda), cum([2], cuda), torch.tensor([0.7], device=cuda)
    for a, b in zip(verify_draft(x, tokens, parents, cu, u, temp, pr), verify_draft(n(-x), tokens, parents, cu, n(-u), n(-temp), n(-pr))):
        assert torch.equal(a, b)
    for call in (lambda: p.append_rope(0, q, k, v, cos, sin, out=n(torch.empty_like(q))), lambda: p.append_rope(0, q, k, v, cos, sin, n(-cum([1, 1], cuda))),
                 lambda: p.append_rope(0, q, k, v, cos, sin, depth=n(ints([0, 0], cuda))), lambda: p.attend_tree(0, q, n(-ones)),
                 lambda: p.attend_tree(0, q, ones, out=n(torch.empty_like(q))), lambda: draft_tree(n(parents), cu), lambda: draft_tree(parents, n(-cu)),
                 lambda: verify_draft(x, n(tokens), parents, cu, u, 0.8), lambda: verify_draft(x, tokens, n(parents), cu, u, 0.8),
                 lambda: verify_draft(x, tokens, parents, n(-cu), u, 0.8), lambda: p.keep(n(ints([0, 0], cuda)), ints([1, 1], cuda)),
                 lambda: p.keep(ints([0, 0], cuda), n(ints([1, 1], cuda)))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("general", [False, True])
def test_wrappers_refuse(hiplib, cuda, monkeypatch, general):
    """What the documentation does not allow, by the host module and by the general path."""
    import _sx8lib
    from sx8_draft import draft_tree, verify_draft
    p, _, _ = make(cuda, [40], 1, 64, 32)
    if general:
        monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    cos, sin = tables(60, 64, cuda)
    q, k, w = rand((1, 2, 64), 1, F16, cuda), rand((1, 1, 64), 2, F16, cuda), rand((64,), 3, F16, cuda)
    cu, ones = cum([1], cuda), torch.ones(1, 1, dtype=torch.int64, device=cuda)
    x, tokens, parents, u = torch.randn(1, 30, device=cuda), torch.zeros(1, dtype=torch.int64, device=cuda), ints([-1], cuda), torch.rand(1, device=cuda)
    before = p.pages.clone()

    def rope(q=q, k=k, v=k, cos=cos, sin=sin, layer=0, **kw):
        return lambda: p.append_rope(layer, q, k, v, cos, sin, **kw)

    def tree(q=q, mask=ones, cu=None, **kw):
        return lambda: p.attend_tree(0, q, mask, cu, **kw)

    def verify(x=x, tokens=tokens, parents=parents, cu=cu, u=u, t=0.8, probs=None):
        return lambda: verify_draft(x, tokens, parents, cu, u, t, probs)

    for i, call in enumerate((
            rope(layer=1), rope(layer=-1), rope(q=q.double()), rope(q=q[..., :32]), rope(q=q[0]), rope(k=k.bfloat16()), rope(v=k.float()),
            rope(k=k[:0]), rope(k=q), rope(q=rand((1, 2, 64), 1, F16, cuda).cpu()), rope(cos=cos.half()), rope(cos=cos[:, :8]), rope(cos=cos[0], sin=sin[0]),
            rope(cos=cos[:, :20], sin=sin[:, :20]), rope(cos=torch.ones(60, 40, device=cuda), sin=torch.ones(60, 40, device=cuda)), rope(cos=cos.cpu()),
            rope(cos=cos[:0], sin=sin[:0]), rope(depth=ints([0, 0], cuda)), rope(depth=ints([0], cuda).long()), rope(q_norm=w.float()),
            rope(k_norm=w[:32]), rope(q_norm=w.cpu()), rope(eps=-1.0), rope(eps=math.nan), rope(eps=math.inf), rope(dtype=BF16), rope(dtype=F32),
            rope(out=q), rope(out=q.float()), rope(out=q[:, :1].expand(1, 2, 64)), rope(q=torch.cat([q, q]), k=torch.cat([k, k]), v=torch.cat([k, k])),
            rope(cu=cu.long()), rope(cu=cum([1, 1], cuda)),
            tree(mask=ones.int()), tree(mask=ones[0]), tree(mask=ones.expand(1, 5).contiguous()), tree(mask=torch.ones(2, 1, dtype=torch.int64, device=cuda)),
            tree(mask=ones.cpu()), tree(mask=torch.ones(1, 0, dtype=torch.int64, device=cuda)), tree(q=q.float()), tree(scale=0.0), tree(scale=math.nan),
            tree(out=q), tree(out=q.bfloat16()), tree(cu=cum([1, 1], cuda)), tree(q=torch.cat([q, q]), mask=torch.cat([ones, ones])),
            lambda: draft_tree(parents, cu, 0), lambda: draft_tree(parents, cu, 5), lambda: draft_tree(parents, cu, -1), lambda: draft_tree(parents.long(), cu),
            lambda: draft_tree(parents, cu.cpu()), lambda: draft_tree(parents.cpu(), cu), lambda: draft_tree([0], cu), lambda: draft_tree(parents, cu[:0]),
            lambda: draft_tree(parents, ints([0], cuda)), lambda: draft_tree(ints([0, 1, 2, 3], cuda)[::2], cu),
            verify(x=x.double()), verify(x=x[0]), verify(x=x.cpu()), verify(x=x[:, :0]), verify(tokens=tokens.int()), verify(tokens=torch.cat([tokens, tokens])),
            verify(parents=parents.long()), verify(parents=ints([0, 0], cuda)), verify(cu=cu.long()), verify(cu=cu[:1]), verify(u=None), verify(u=u.half()),
            verify(u=torch.rand(2, device=cuda)), verify(u=None, t=torch.zeros(1, device=cuda)), verify(t=torch.ones(2, device=cuda)),
            verify(t=torch.ones(1, device=cuda).half()), verify(t=torch.ones(1)), verify(probs=x[:, :29]), verify(probs=x.double()), verify(probs=x.cpu()),
            lambda: p.keep(ints([0], cuda).long(), ints([1], cuda)), lambda: p.keep(ints([0], cuda), ints([1, 1], cuda)),
            lambda: p.keep(ints([0, 0], cuda), ints([1], cuda)), lambda: p.keep([0], ints([1], cuda)), lambda: p.keep(ints([0], cuda), ints([1], cuda), cu.long()),
            lambda: p.keep(ints([0], cuda), ints([1], cuda).cpu()), lambda: p.keep(ints([0], cuda), ints([1], cuda), cum([1, 1], cuda)))):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} is not refused")
    assert torch.equal(p.pages, before) and p.lens.tolist() == [40]
    # calls without rows
    none = ints([0, 0], cuda)
    assert p.append_rope(0, q[:0], k[:0], k[:0], cos, sin, none).shape == (0, 2, 64) and p.attend_tree(0, q[:0], ones[:0], none).shape == (0, 2, 64)
    mask, depth = draft_tree(parents[:0], none)
    path, counts, nxt = verify_draft(x[:0], tokens[:0], parents[:0], none, u[:0], 0.8, x[:0])
    p.keep(path, counts, none)
    p.check()
    assert mask.shape == (0, 1) and depth.shape == (0,) and counts.tolist() == [0] and nxt.tolist() == [-1] and p.lens.tolist() == [40]
