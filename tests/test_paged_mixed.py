"""Prompts of new slots and of slots that have tokens already, in one call of the batched decoder."""
import pytest
import torch

from test_e2e import TINY
from test_paged_e2e import ids

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(hiplib, cuda):
    from e2e_decoder import SX8Decoder
    return SX8Decoder(TINY, device=cuda, seed=3, n_distinct=2, max_len=160)


def start(dec, n_slots=4, **kw):
    """A decoder whose slots 0 and 2 hold tokens."""
    from e2e_decoder import PagedDecoder
    pd = PagedDecoder(dec, n_slots, max_len=160, page_tokens=32, **kw)
    pd.prompt([0, 2], [ids(11, 1, dec.device), ids(20, 2, dec.device)])
    return pd


def rel(a, b):
    return ((a - b).abs().max() / b.abs().max()).item()


@pytest.mark.parametrize("n_old", [4, 138])
def test_new_and_continuing_slots(dec, cuda, n_old):
    """Each sequence gets what it gets without the others (few rows behind earlier tokens, and so many that the pages are read
    back): its attention is the same, and its linears may sum in another order for another number of rows, which moves
    an fp16 activation by a rounding: 2^-11 of itself, some ten of them a layer, in other directions: 2^-8 of the
    largest logit for all of them."""
    from e2e_decoder import PagedDecoder
    new = {1: ids(25, 3, cuda), 3: ids(70, 4, cuda)}
    old = {0: ids(n_old, 5, cuda), 2: ids(n_old + 1, 6, cuda)}
    want = {}
    alone = PagedDecoder(dec, 4, max_len=160, page_tokens=32)
    alone.prompt(list(new), list(new.values()))
    want.update(zip(new, alone.logits))
    alone = start(dec)
    alone.prompt(list(old), list(old.values()))
    want.update(zip(old, alone.logits))
    pd = start(dec)
    slots = [3, 0, 1, 2]
    nxt = pd.prompt(slots, [{**new, **old}[s] for s in slots])
    far = {s: rel(pd.logits[s], want[s]) for s in range(4)}
    print("apart by", far, flush=True)
    assert max(far.values()) <= 2.0 ** -8
    assert torch.equal(nxt, pd.logits.argmax(-1)[torch.tensor(slots, device=cuda)]) and torch.equal(pd.tok, pd.logits.argmax(-1))
    assert pd.lens == pd.cache.lens.tolist() == [11 + n_old, 25, 21 + n_old, 70]
    pd.step()
    pd.cache.check()


def test_idle_slots_are_no_sequences(dec, cuda, monkeypatch):
    """The prompt attention gets the call's sequences alone: slots that bring nothing do not count when it cuts keys into
    parts, and launch nothing."""
    import e2e_decoder
    seen = []

    def spy(q, k, v, cu_q, cu_k=None, *args, **kw):
        seen.append((cu_q.tolist(), None if cu_k is None else cu_k.tolist()))
        return attn_varlen(q, k, v, cu_q, cu_k, *args, **kw)

    attn_varlen = e2e_decoder.attn_varlen
    monkeypatch.setattr(e2e_decoder, "attn_varlen", spy)
    pd = start(dec, 70)
    assert seen and all(s == ([0, 11, 31], None) for s in seen)
    del seen[:]
    pd.prompt([69, 0, 33], [ids(9, 1, cuda), ids(140, 2, cuda), ids(5, 3, cuda)])
    layers = TINY["n_layers"]
    assert seen == [([0, 5, 14], None), ([0, 140], [0, 151])] * layers
    assert pd.lens == pd.cache.lens.tolist()


def test_embedding_rows_are_the_decoders_own(dec, cuda):
    """Prompts and steps, captured ones too, write none of the embedding module's buffer, which a longer call replaces: a graph
    that wrote it would go on writing freed memory."""
    pd = start(dec)
    dec.embed(ids(90, 1, cuda))
    dec.embed._out.fill_(7)
    pd.step()
    pd.prompt([1], [ids(30, 2, cuda)])
    pd.step()
    pd.step(use_graph=False)
    torch.cuda.synchronize()
    assert (dec.embed._out == 7).all()
    kept = dec.embed._out.data_ptr()
    pd.prompt([3], [ids(150, 3, cuda)])
    assert dec.embed._out.data_ptr() == kept
    # the captured step after a longer prompt: the tokens of eager steps
    other = start(dec)
    other.step(use_graph=False)
    other.prompt([1], [ids(30, 2, cuda)])
    for _ in range(2):
        other.step(use_graph=False)
    other.prompt([3], [ids(150, 3, cuda)])
    for _ in range(4):
        assert torch.equal(pd.step(), other.step(use_graph=False))
    pd.cache.check()


def test_two_decoders_at_once(dec, cuda):
    """Two batched decoders over one set of weights, on two streams at once, give what they give one after the other."""
    def run(streams):
        pds = [start(dec) for _ in range(2)]
        for i, pd in enumerate(pds):
            pd.prompt([1], [ids(20 + i, 7 + i, cuda)])
            pd.step()
        torch.cuda.synchronize()
        out = [[], []]
        for _ in range(5):
            for i, pd in enumerate(pds):
                with torch.cuda.stream(streams[i]):
                    out[i].append(pd.step())
        torch.cuda.synchronize()
        return [torch.stack(o) for o in out]

    one = torch.cuda.current_stream()
    want = run([one, one])
    got = run([torch.cuda.Stream(), torch.cuda.Stream()])
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_slot_numbers_as_vectors(dec, cuda):
    """Slot numbers in torch or numpy vectors are the slots that ints name; numbers that are no integers are refused."""
    import numpy as np
    from e2e_decoder import PagedDecoder
    a, b = (PagedDecoder(dec, 5, max_len=100, page_tokens=32) for _ in range(2))
    prompts = [ids(9, 1, cuda), ids(40, 2, cuda)]
    want = a.prompt([3, 1], prompts)
    assert torch.equal(b.prompt(torch.tensor([3, 1]), prompts), want) and a.lens == b.lens == b.cache.lens.tolist()
    a.fork([1, 1], [0, 2])
    with pytest.raises(ValueError):
        b.fork(torch.tensor([1, 1]), torch.tensor([0, 0]))
    b.fork(np.array([1, 1]), torch.tensor([0, 2]))
    a.free([3])
    b.free(np.array([3]))
    assert a.lens == b.lens == b.cache.lens.tolist() == [40, 40, 40, 0, 0]
    assert torch.equal(a.step(), b.step())
    with pytest.raises(ValueError):
        b.prompt(torch.tensor([3, 3]), prompts)
    with pytest.raises(TypeError):
        b.prompt([3.0], prompts[:1])


def test_buffers_go_when_nothing_runs_on_them(dec, cuda, monkeypatch):
    """A prompt replaces the last one's buffers behind the wait of the cache's check, on whatever stream they were made and
    used; where there is no memory for the new ones, lengths are still the cache's."""
    pd = start(dec)
    order = []
    check, bufs = pd.cache.check, pd._bufs
    monkeypatch.setattr(pd.cache, "check", lambda: order.append("check") or check())
    monkeypatch.setattr(pd, "_bufs", lambda n: order.append("bufs") or bufs(n))
    pd.prompt([1], [ids(7, 1, cuda)])
    assert order == ["check", "bufs"]

    def none(n):
        raise torch.cuda.OutOfMemoryError("none left")

    monkeypatch.setattr(pd, "_bufs", none)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        pd.prompt([1, 3], [ids(7, 1, cuda), ids(9, 1, cuda)])
    assert pd.lens == pd.cache.lens.tolist() == [11, 14, 20, 9] and pd.active.tolist() == [1] * 4
    monkeypatch.setattr(pd, "_bufs", bufs)
    pd.free([1, 3])
    other = start(dec)
    assert torch.equal(pd.prompt([3], [ids(9, 1, cuda)]), other.prompt([3], [ids(9, 1, cuda)]))
    used = torch.tensor([0, 2, 3], device=cuda)
    assert torch.equal(pd.step()[used], other.step()[used]) and pd.active.tolist() == [1, 0, 1, 1]


def test_full_slots_are_named(dec, cuda):
    from e2e_decoder import PagedDecoder
    pd = PagedDecoder(dec, 3, max_len=40, page_tokens=32)
    pd.prompt([0, 2], [ids(12, 1, cuda), ids(40, 2, cuda)])
    with pytest.raises(ValueError, match=r"slots \[2\] are full"):
        pd.step()
    assert pd.lens == pd.cache.lens.tolist() == [12, 0, 40]
    pd.free([2])
    pd.step()
    assert pd.lens == pd.cache.lens.tolist() == [13, 0, 0]
