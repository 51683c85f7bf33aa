"""What a pass over drafted tokens may leave in the cache: only rows whose K and V were written there.  Whole numbers and moved
bits: equal."""
import random

import pytest
import torch

from test_draft import F32, drafts, flat, run_verify, tables, trees, turn
from test_paged_kv import F16, cum, ints, make, q4, rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------ rows that are no part of a tree
def without(ps, dead):
    """The trees with the rows of `dead` as no one's children."""
    return [[-1 if (s, i) in dead else p for i, p in enumerate(tree)] for s, tree in enumerate(ps)]


@pytest.mark.parametrize("words", [1, 2, 4])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("dt", [F32, F16])
def test_rows_past_the_words_are_not_kept(hiplib, cuda, words, probs, dt):
    """Trees and chains with rows past the masks' words, greedy and drawn: the verification that knows the depths keeps what
    it would if these rows followed none, and never one of them."""
    from sx8_draft import draft_tree, verify_draft
    ns, V = [70, 64, 3, 140, 0, 300, 65], 50
    logits, ps, tokens, u, pr = drafts(cuda, ns, V, words, dt, probs=probs)
    ps[0], ps[6] = trees([70], 0, chain=True)[0], trees([65], 0, chain=True)[0]
    u = [0.0 if random.Random(i).random() < 0.9 else x for i, x in enumerate(u)]      # (most tokens are kept)
    temp = [1.0, 0.0, 0.7, 1.3, 1.0, 0.9, 1.0]
    cu, parents = cum(ns, cuda), ints(flat(ps), cuda)
    _, depth = draft_tree(parents, cu, words)
    dead = {(s, i) for s, n in enumerate(ns) for i in range(64 * words, n)}
    assert (depth < 0).sum() == len(dead)
    want = run_verify(cuda, logits, without(ps, dead), tokens, u, temp, pr)
    args = (logits, torch.tensor(tokens, device=cuda), parents, cu, torch.tensor(u, dtype=F32, device=cuda), torch.tensor(temp, device=cuda), pr)
    got = verify_draft(*args, depth=depth)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert got[0].max().item() < 64 * words
    # every first child kept: the chains up to their masks' last row
    u = [0.0] * len(u)
    want = run_verify(cuda, logits, without(ps, dead), tokens, u, [1.0] * 7, pr)
    got = verify_draft(*args[:4], torch.zeros(len(u), device=cuda), 1.0, pr, depth=depth)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert [got[1][s].item() for s in (0, 6)] == [min(70, 64 * words), min(65, 64 * words)]
    # all rows are part of their trees: as without depths
    _, depth = draft_tree(ints(flat(trees(ns, 3)), cuda), cu, 4)
    if words == 4:
        args = (*args[:2], ints([p if i < 256 else -1 for t in ps for i, p in enumerate(t)], cuda), *args[3:])
        assert all(torch.equal(a, b) for a, b in zip(verify_draft(*args, depth=depth), verify_draft(*args)))


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temp", [0.0, 0.9])
@pytest.mark.parametrize("general", [False, True])
def test_slots_whose_first_row_is_no_part(hiplib, cuda, monkeypatch, probs, temp, general):
    """Such a slot keeps nothing and has no token; its neighbours are as they were; scattered rows without a place."""
    import _sx8lib
    from sx8_draft import verify_draft
    if general:
        monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    ns = [5, 1, 300, 7, 0, 20]
    logits, ps, tokens, u, pr = drafts(cuda, ns, 33, 4, probs=probs)
    u = [x / 3 for x in u]
    dead = {(1, 0), (3, 0), (2, 7), (2, 280), (5, 1), (0, 3)}
    starts = cum(ns, cuda).tolist()
    depth = torch.zeros(sum(ns), dtype=torch.int32)
    for s, i in dead:
        depth[starts[s] + i] = -1 - s
    want = run_verify(cuda, logits, without(ps, dead), tokens, u, [temp] * 6, pr)
    got = verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cum(ns, cuda), torch.tensor(u, dtype=F32, device=cuda),
                       temp, pr, depth=depth.to(cuda))
    for s in range(6):
        rows = slice(starts[s], starts[s + 1])
        if s in (1, 3):
            assert got[1][s] == 0 and got[2][s] == -1 and (got[0][rows] == -1).all()
        else:
            assert all(torch.equal(a, b) for a, b in ((got[0][rows], want[0][rows]), (got[1][s], want[1][s]), (got[2][s], want[2][s])))
    for bad in (depth, depth.to(cuda).long(), depth[1:].to(cuda), torch._neg_view(depth.to(cuda)), [0] * sum(ns)):
        with pytest.raises(RuntimeError, match="depth"):
            verify_draft(logits, torch.tensor(tokens, device=cuda), ints(flat(ps), cuda), cum(ns, cuda), torch.tensor(u, dtype=F32, device=cuda),
                         temp, pr, depth=bad)


@pytest.mark.parametrize("words,kept", [(1, 64), (2, 70)])
def test_round_of_a_long_chain(hiplib, cuda, words, kept):
    """A chain of 70 tokens, all of them to be kept, through a whole pass: with masks of one word 64 are, and every token of
    the cache is one that was written."""
    from sx8_draft import draft_tree, verify_draft
    new, before = [70, 2], [40, 7]
    p, k0, v0 = make(cuda, before, 2, 64, 32, spare=8, width=8)
    cos, sin = tables(200, 64, cuda)
    cu, parents = cum(new, cuda), ints([*range(-1, 69), -1, 0], cuda)
    p.reserve(ints(new, cuda))
    q, k, v = (rand((72, n, 64), 30 + i, F16, cuda) for i, n in enumerate((4, 2, 2)))
    mask, depth = draft_tree(parents, cu, words)
    qr = p.append_rope(0, q, k, v, cos, sin, cu, depth=depth)
    p.attend_tree(0, qr, mask, cu)
    logits = torch.randn(72, 30, generator=torch.Generator().manual_seed(1)).to(cuda)
    tokens = torch.arange(72, device=cuda) % 30
    path, counts, following = verify_draft(logits, tokens, parents, cu, torch.zeros(72, device=cuda), 1.0, depth=depth)
    p.keep(path, counts, cu)
    p.check()
    assert counts.tolist() == [kept, 2] and p.lens.tolist() == [40 + kept, 9] and (following >= 0).all()
    place = list(range(40, 40 + kept))
    kk = torch.cat([k0[:40], turn(k[:kept], None, cos[place], sin[place], False).float().half()])
    got = p.read(0, 40 + kept + 9, cum(p.lens.tolist(), cuda))
    assert torch.equal(got[0][:40 + kept], q4(kk).half()) and torch.equal(got[1][:40 + kept], q4(torch.cat([v0[:40], v[:kept]])).half())


# ------------------------------------------------------------------------------ a reservation that is refused
def a_pass(p, new, seed, cuda, cos, sin, reserve=True):
    """One pass over drafted tokens of a single layer, nobody asking for the status in between; as a function of tensors."""
    from sx8_draft import draft_tree, verify_draft
    T = sum(new)
    q, k, v = (rand((T, n, 64), seed + i, F16, cuda) for i, n in enumerate((4, 2, 2)))
    logits, ps, tokens, u, _ = drafts(cuda, new, 40, seed)
    add, cu, parents = ints(new, cuda), cum(new, cuda), ints(flat(ps), cuda)
    tokens, u = torch.tensor(tokens, device=cuda), torch.tensor(u, dtype=F32, device=cuda) / 2

    def run():
        if reserve:
            p.reserve(add)
        mask, depth = draft_tree(parents, cu)
        qr = p.append_rope(0, q, k, v, cos, sin, cu, depth=depth)
        o = p.attend_tree(0, qr, mask, cu)
        path, counts, nxt = verify_draft(logits, tokens, parents, cu, u, 0.8, depth=depth)
        p.keep(path, counts, cu)
        return qr, o, counts
    return run


def state(p):
    return [t.clone() for t in (p.pages, p.table, p.lens, p.refs)]


def unmarked(p):
    return p.marks.tolist() == [[2 ** 31 - 1] + [0] * 8] * p.n_slots


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("new,error", [([3, 40, 0], "no free pages"), ([3, 200, 2], "table row is full"), ([3, 5, 9], "no free pages"), ([0, 0, 70], "no free pages")])
def test_refused_reservation_harms_no_token(hiplib, cuda, monkeypatch, general, new, error):
    """No page left, or no place in the table: the whole pass changes nothing, in slots with room as well, one with fewer tokens
    than rows among them; the error is there whenever it is asked for, and the next pass is that of a cache that never saw it."""
    import _sx8lib
    if general:
        monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    p, _, _ = make(cuda, [60, 64, 1], 2, 64, 32, spare=0, width=6)
    other, _, _ = make(cuda, [60, 64, 1], 2, 64, 32, spare=0, width=6)
    cos, sin = tables(200, 64, cuda)
    before = state(p)
    _, _, counts = a_pass(p, new, 30, cuda, cos, sin)()
    assert same(state(p), before) and counts.sum() > 0
    k, v = (rand((3, 2, 64), i, F16, cuda) for i in (5, 6))
    p.append_rope(0, rand((3, 4, 64), 4, F16, cuda), k, v, cos, sin)                                 # one row a slot
    want, _, _ = make(cuda, [60, 64, 1], 2, 64, 32, spare=0, width=6)
    want.append_rope(0, rand((3, 4, 64), 4, F16, cuda), k, v, cos, sin)
    for got, new_row, old in zip(p.read(0, 3), want.read(0, 3), other.read(0, 3)):
        grows = torch.tensor([n > 0 for n in new], device=cuda)[:, None, None]
        assert torch.equal(got, torch.where(grows, old, new_row)) and not torch.equal(old, new_row)
    p.pages.copy_(before[0])
    a_pass(p, new, 30, cuda, cos, sin)()                             # refused again
    with pytest.raises(RuntimeError, match=error):
        p.check()
    assert same(state(p), before)
    p.check()
    outs = [a_pass(c, [4, 0, 20], 50, cuda, cos, sin)() for c in (p, other)]
    for c in (p, other):
        c.check()
    assert same(*outs) and same(state(p), state(other)) and outs[0][2][0] > 0


def test_refused_reservation_captured(hiplib, cuda):
    """A captured pass, replayed while there is no page and again when there is one: nothing, then what the eager pass does."""
    p, _, _ = make(cuda, [60, 64, 40], 2, 64, 32, spare=0, width=6)
    other, _, _ = make(cuda, [60, 64, 40], 2, 64, 32, spare=0, width=6)
    cos, sin = tables(200, 64, cuda)
    run, want = a_pass(p, [3, 40, 0], 30, cuda, cos, sin), a_pass(other, [3, 40, 0], 30, cuda, cos, sin)
    run()
    with pytest.raises(RuntimeError, match="no free pages"):
        p.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = run()
    before = state(p)
    for _ in range(3):
        g.replay()
        assert same(state(p), before)
        run()
        assert same(state(p), before)
    with pytest.raises(RuntimeError, match="no free pages"):
        p.check()
    for c in (p, other):
        c.free(ints([2], cuda))
    g.replay()
    got = [t.clone() for t in outs] + state(p)
    assert same(got, [*want(), *state(other)])
    for c in (p, other):
        c.check()


def test_marks_are_of_the_slot(hiplib, cuda):
    """An error of another call stops no pass; a refusal for other slots neither; a slot's mark goes with its next reservation."""
    cos, sin = tables(200, 64, cuda)
    pools = [make(cuda, [60, 64, 1], 2, 64, 32, spare=1, width=6)[0] for _ in range(3)]
    p, late, want = pools
    p.fork(ints([0], cuda), ints([1], cuda))                         # the target is in use
    a_pass(p, [3, 0, 5], 30, cuda, cos, sin)()
    with pytest.raises(RuntimeError, match="in use"):
        p.check()
    # reserved, then other slots refused: the pass goes on
    late.reserve(ints([3, 0, 5], cuda))
    late.reserve(ints([0, 100, 0], cuda))
    assert late.marks[:, 0].tolist() == [2 ** 31 - 1, -1, 2 ** 31 - 1]
    a_pass(late, [3, 0, 5], 30, cuda, cos, sin, reserve=False)()
    with pytest.raises(RuntimeError, match="no free pages"):
        late.check()
    late.reserve(ints([0, 1, 0], cuda))
    assert unmarked(late) and late.lens[1] == 65
    a_pass(want, [3, 0, 5], 30, cuda, cos, sin)()
    want.check()
    assert same(state(p), state(want))
    want.reserve(ints([0, 1, 0], cuda))
    assert same(state(late), state(want))
    late.reserve(ints([-1, 0, 0], cuda))
    assert late.marks[:, 0].tolist() == [-1, 2 ** 31 - 1, 2 ** 31 - 1]
    with pytest.raises(RuntimeError, match="bad slot or count"):
        late.check()


# ------------------------------------------------------------------------------ rows that were never written
@pytest.mark.parametrize("general", [False, True])
@pytest.mark.parametrize("S", [3, 70])
def test_keep_refuses_rows_that_were_not_written(hiplib, cuda, monkeypatch, general, S):
    """Rows past the masks' words and behind the tables' end: a verification that does not know the depths keeps them, `keep` says
    so and changes nothing; fewer rows are kept as ever, and the next pass is one without a trace."""
    import _sx8lib
    from sx8_draft import draft_tree, verify_draft
    if general:
        monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    for new, table, slot, good in (([70, 4], 400, 0, [64, 4]), ([5, 12], 40, 1, [5, 7]), ([2, 1], 33, 1, [2, 0])):
        new, good = new + [0] * (S - 2), good + [0] * (S - 2)
        p, _, _ = make(cuda, [10, 33] + [1] * (S - 2), 2, 64, 32, spare=8, width=8, layers=2)
        cos, sin = tables(table, 64, cuda)
        T, cu, parents = sum(new), cum(new, cuda), ints([j - 1 for n in new for j in range(n)], cuda)
        p.reserve(ints(new, cuda))
        q, k, v = (rand((T, n, 64), 30 + i, F16, cuda) for i, n in enumerate((4, 2, 2)))
        mask, depth = draft_tree(parents, cu)
        for layer in range(2):
            p.attend_tree(layer, p.append_rope(layer, q, k, v, cos, sin, cu, depth=depth), mask, cu)
        x, tokens, u = torch.randn(T, 30, generator=torch.Generator().manual_seed(1)).to(cuda), torch.arange(T, device=cuda) % 30, torch.zeros(T, device=cuda)
        path, counts, _ = verify_draft(x, tokens, parents, cu, u, 1.0)
        assert counts.tolist() == new
        before = state(p)
        for _ in range(2):                                           # (refused as often as it is asked)
            p.keep(path, counts, cu)
            with pytest.raises(RuntimeError, match=rf"never written \(slot or entry {slot}\)"):
                p.check()
            assert same(state(p), before)
        p.keep(path, ints(good, cuda), cu)
        p.check()
        lens = [10 + good[0], 33 + good[1]]
        assert p.lens.tolist()[:2] == lens and unmarked(p)
        at = list(range(10, lens[0]))
        got = p.read(1, sum(lens), ints([0, lens[0], *[sum(lens)] * (S - 1)], cuda))
        assert torch.equal(got[0][10:lens[0]], q4(turn(k[:good[0]], None, cos[at], sin[at], False).float().half()).half())
        # a pass whose rows all have a place: nothing is left of the refusal
        p.reserve(ints([1] + [0] * (S - 1), cuda))
        one = cum([1] + [0] * (S - 1), cuda)
        p.append_rope(0, q[:1], k[:1], v[:1], cos, sin, one)
        p.keep(ints([0], cuda), ints([1] + [0] * (S - 1), cuda), one)
        p.check()
        assert p.lens[0] == lens[0] + 1


def test_rows_that_were_not_written_and_not_kept(hiplib, cuda):
    """Branches that end outside: what lies before them is kept, without depths too; a row that is out by its depth alone."""
    from sx8_draft import draft_tree, verify_draft
    p, _, _ = make(cuda, [10], 1, 64, 32, spare=4, width=8)
    cos, sin = tables(100, 64, cuda)
    new, parents = 80, ints([-1] + [0] * 79, cuda)
    cu = cum([new], cuda)
    p.reserve(ints([new], cuda))
    q, k = rand((new, 2, 64), 1, F16, cuda), rand((new, 1, 64), 2, F16, cuda)
    _, depth = draft_tree(parents, cu)
    p.append_rope(0, q, k, k, cos, sin, cu, depth=depth)
    assert not unmarked(p)
    x = torch.zeros(new, 100, device=cuda)
    u = torch.full((new,), 0.999, device=cuda)
    u[63] = 0.0
    path, counts, _ = verify_draft(x, torch.arange(new, device=cuda), parents, cu, u, 1.0)
    p.keep(path, counts, cu)
    p.check()
    assert path.tolist()[:3] == [0, 63, -1] and p.lens.tolist() == [12] and unmarked(p)
    p.reserve(ints([3], cuda))
    p.append_rope(0, q[:3], k[:3], k[:3], cos, sin, cum([3], cuda), depth=ints([0, -13, 1], cuda))
    p.keep(ints([0, 1, -1], cuda), ints([2], cuda), cum([3], cuda))
    with pytest.raises(RuntimeError, match="never written"):
        p.check()
    p.keep(ints([0, 2, -1], cuda), ints([2], cuda), cum([3], cuda))
    p.check()
    assert p.lens.tolist() == [14]


def test_branches_beside_a_row_that_was_not_written(hiplib, cuda):
    """A deep branch ends behind the tables; a row with a higher number that is written is kept, the deep ones are not: every
    single row of a tree of 256 and rows behind them, where one that is out takes all behind it with it."""
    p, _, _ = make(cuda, [10], 1, 64, 32, spare=14, width=20)
    cos, sin = tables(20, 64, cuda)
    q, k = rand((300, 2, 64), 1, F16, cuda), rand((300, 1, 64), 2, F16, cuda)
    rng = random.Random(1)
    depth = [0] + [rng.choice([1, 3, 9, 10, 11, 2 ** 31 - 1, -11, 2]) for _ in range(255)] + [1] * 20 + [10] + [1] * 23
    cu, d = cum([300], cuda), ints(depth, cuda)
    for row in [*range(1, 256, 5), 31, 32, 63, 64, 255, 256, 275, 276, 277, 299]:
        p.reserve(ints([300], cuda))
        p.append_rope(0, q, k, k, cos, sin, cu, depth=d)
        p.keep(ints([0, row] + [-1] * 298, cuda), ints([2], cuda), cu)
        if not 0 <= 10 + depth[row] < 20 or row > 276:
            with pytest.raises(RuntimeError, match="never written"):
                p.check()
            p.keep(ints([0] + [-1] * 299, cuda), ints([0], cuda), cu)
            assert p.lens.tolist() == [10]
        else:
            p.check()
            assert p.lens.tolist() == [12] and unmarked(p)
            p.lens.fill_(10)
        p.check()
        assert unmarked(p)
