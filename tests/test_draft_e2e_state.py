"""What PagedDecoder.verify leaves behind where it refuses, raises or finds no token, and how often it waits."""
import warnings

import pytest
import torch

from test_e2e import TINY
from test_paged_e2e import ids

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(hiplib, cuda):
    from e2e_decoder import SX8Decoder
    return SX8Decoder(TINY, device=cuda, seed=3, n_distinct=2, max_len=160)


def start(dec, **kw):
    """A decoder whose slots 0 and 2 of four hold tokens."""
    from e2e_decoder import PagedDecoder
    pd = PagedDecoder(dec, 4, max_len=120, page_tokens=32, **kw)
    pd.prompt([0, 2], [ids(30, 1, dec.device), ids(20, 2, dec.device)])
    return pd


def state(pd):
    """Everything that a later call reads: the slots' tokens, lengths, tables and counts, and the pages' used bytes as values."""
    c, lens = pd.cache, pd.cache.lens.tolist()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=c.device)
    rows = [t for layer in range(c.n_layers) for t in c.read(layer, sum(lens), cu)]
    return [list(pd.lens), pd.tok.clone(), c.table.clone(), c.lens.clone(), c.refs.clone(), *rows]


def same(a, b):
    return a[0] == b[0] and all(torch.equal(x, y) for x, y in zip(a[1:], b[1:]))


def test_drafts_are_whole_numbers(dec, cuda):
    """Vectors of another kind are refused before anything changes, an empty floating-point one too; other whole numbers are
    taken as what they are."""
    pd, other = start(dec), start(dec)
    three, before = ids(3, 5, cuda), state(pd)
    for bad in (torch.tensor([]), torch.tensor([], device=cuda), three.float(), three.half(), three[None], three[0], three.to(torch.complex64), three.tolist()):
        for slots, drafts in (([0, 2], [three, bad]), ([2], [bad])):
            with pytest.raises(ValueError, match="slot 2: drafts"):
                pd.verify(slots, drafts)
    assert same(state(pd), before)
    none = torch.tensor([], dtype=torch.int64)
    got, want = pd.verify([0, 2], [three.int(), none]), other.verify([0, 2], [three, none.to(cuda)])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and same(state(pd), state(other))
    assert torch.equal(pd.step()[[0, 2]], other.step()[[0, 2]])


@pytest.mark.parametrize("where", ["head", "layer", "verify", "check"])
@pytest.mark.parametrize("error", [torch.cuda.OutOfMemoryError, RuntimeError, KeyboardInterrupt])
def test_a_pass_that_raises_leaves_no_trace(dec, cuda, monkeypatch, where, error):
    """Whatever raises behind the reservation, with new pages among it: tokens, lengths, tables and counts are as before, and the
    next pass and step those of a decoder that never saw it."""
    import e2e_decoder
    pd, other = start(dec), start(dec)
    drafts, before = [ids(5, 5, cuda), ids(40, 6, cuda)], state(pd)

    def fails(*a, **kw):
        raise error("as if")

    with monkeypatch.context() as m:
        if where == "head":
            m.setattr(pd, "_head", fails)
        elif where == "layer":
            real = pd.cache.attend_tree
            m.setattr(pd.cache, "attend_tree", lambda li, *a: fails() if li == len(dec.layers) - 1 else real(li, *a))
        elif where == "verify":
            m.setattr(e2e_decoder, "verify_draft", fails)
        else:
            m.setattr(pd.cache, "check", fails)
        for _ in range(2):
            with pytest.raises(error, match="as if"):
                pd.verify([0, 2], drafts)
            assert same(state(pd), before)
    got, want = pd.verify([0, 2], drafts), other.verify([0, 2], drafts)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and same(state(pd), state(other))
    assert torch.equal(pd.step()[[0, 2]], other.step()[[0, 2]])
    pd.cache.check()


def test_an_earlier_error_is_raised_and_the_rows_are_dropped(dec, cuda):
    """An error that the program's own call on the cache left behind: verify raises it, and its places are given back; where its own
    reservation is refused, nothing is dropped."""
    pd = start(dec)
    before = state(pd)
    pd.cache.fork(*(torch.tensor([i], dtype=torch.int32, device=cuda) for i in (0, 2)))
    with pytest.raises(RuntimeError, match="in use"):
        pd.verify([0, 2], [ids(5, 5, cuda), ids(40, 6, cuda)])
    assert same(state(pd), before)
    small = start(dec, n_pages=2)
    before = state(small)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no free pages"):
            small.verify([2, 0], [ids(1, 5, cuda), ids(5, 6, cuda)])
        assert same(state(small), before)
    assert small.verify([2], [ids(1, 5, cuda)])[0].numel() >= 1 and small.lens == small.cache.lens.tolist()


@pytest.mark.parametrize("value", [float("nan"), -float("inf")])
@pytest.mark.parametrize("sampled", [False, True])
def test_a_slot_that_no_token_follows(dec, cuda, monkeypatch, value, sampled):
    """Logits that are no numbers give no token: the pass says which slots and is undone, and no slot's next input is -1."""
    pd, other = start(dec), start(dec)
    drafts, before = [ids(3, 5, cuda), ids(2, 6, cuda)], state(pd)
    how = dict(uniforms=[torch.zeros(4, device=cuda), torch.zeros(3, device=cuda)], temperature=1.0) if sampled else {}
    head = pd._head

    def broken(resid, d, n):
        x = head(resid, d, n)
        x[4:] = value                                                # the rows of slot 2
        return x

    with monkeypatch.context() as m:
        m.setattr(pd, "_head", broken)
        with pytest.raises(RuntimeError, match=r"slots \[2\]: no token follows"):
            pd.verify([0, 2], drafts, **how)
    assert same(state(pd), before)
    got, want = pd.verify([0, 2], drafts, **how), other.verify([0, 2], drafts, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and same(state(pd), state(other)) and (pd.tok >= 0).all()
    assert torch.equal(pd.step()[[0, 2]], other.step()[[0, 2]])


def test_waits(dec, cuda, monkeypatch):
    """One wait a pass; one more, before the buffers are replaced, where a slot needs a page or a prompt may still run on them."""
    pd = start(dec)
    order = []
    check, bufs = pd.cache.check, pd._bufs
    monkeypatch.setattr(pd.cache, "check", lambda: order.append("check") or check())
    monkeypatch.setattr(pd, "_bufs", lambda n: order.append("bufs") or bufs(n))
    torch.manual_seed(0)
    drafts = {n: ids(n, n, cuda) for n in (1, 2, 20)}
    u = {n: torch.rand(1 + n, device=cuda) for n in drafts}

    def one(slots, ns, **kw):
        order.clear()
        torch.cuda.synchronize()
        with warnings.catch_warnings(record=True) as said:
            warnings.simplefilter("always")
            torch.cuda.set_sync_debug_mode("warn")
            try:
                pd.verify(slots, [drafts[n] for n in ns], **kw)
            finally:
                torch.cuda.set_sync_debug_mode("default")
        return order, sum("called a synchronizing" in str(w.message) for w in said)

    assert one([2], [1]) == (["check", "bufs"], 2)                   # the prompt's buffers
    assert one([2], [2]) == (["bufs"], 1)
    assert one([2], [2], uniforms=[u[2]], temperature=[0.8]) == (["bufs"], 1)
    assert one([2], [20], uniforms=[u[20]], temperature=0.8) == (["check", "bufs"], 2)       # a page
    assert pd.lens == pd.cache.lens.tolist()
    pd.prompt([1], [ids(3, 1, cuda)])
    assert one([1], [2]) == (["bufs"], 1)                            # (three rows as well: the prompt's buffers stay)
    pd.prompt([3], [ids(4, 1, cuda)])
    assert one([3], [2]) == (["check", "bufs"], 2)
    pd.cache.check()


def test_an_earlier_error_where_no_page_is_needed(dec, cuda):
    """It is read with the counts, and the pass is undone."""
    pd, other = start(dec), start(dec)
    pd.verify([2], [ids(1, 5, cuda)])
    other.verify([2], [ids(1, 5, cuda)])
    before = state(pd)
    pd.cache.fork(*(torch.tensor([i], dtype=torch.int32, device=cuda) for i in (0, 2)))
    with pytest.raises(RuntimeError, match="in use"):
        pd.verify([2], [ids(2, 5, cuda)])
    assert same(state(pd), before)
    assert torch.equal(pd.verify([2], [ids(2, 5, cuda)])[0], other.verify([2], [ids(2, 5, cuda)])[0]) and same(state(pd), state(other))
