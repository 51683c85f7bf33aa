"""Drafted tokens on the GPU (append_rope, attend_tree, draft_tree, verify_draft, keep) against plain implementations in 64
bits.

Tolerances.  append_rope computes in 64 bits and rounds once, as the reference does (to float32 and from there to 16 bits; an
exact value within 2^-50 of a rounding's border is not to be expected among the 10^6 here), so its rows and what is read back are
equal.  attend_tree is the arithmetic of PagedKV4.attend, with the bound that test_paged_kv.py derives: half a step of the output
and LOOSE = 2^-15 of the largest value averaged (the weights' sum is taken from the matrix cores here: two fp16 numbers a
weight, 22 bits, 2^-22 of the sum, and sums cut by 2^-24 a product: within 2^-15 with the rest).  verify_draft and keep
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
