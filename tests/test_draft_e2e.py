"""PagedDecoder.verify: drafted tokens checked over the paged 4-bit cache, against a float32 decoder that is fed the kept tokens one
after another.  Tolerances are those of test_paged_e2e.py (its reference and its bound)."""
import pytest
import torch

from test_e2e import TINY, _dequant_all
from test_paged_e2e import Ref, ids, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(hiplib, cuda):
    from e2e_decoder import SX8Decoder
    d = SX8Decoder(TINY, device=cuda, seed=3, n_distinct=2, max_len=160)
    return d, _dequant_all(d, cuda)


def follow(refs, pd, slots, before, results, drafts, up):
    """Feed each reference the last token and the kept ones; the logits of the kept rows are those of the pass."""
    a = 0
    for s, first, got, t, p in sorted(zip(slots, before, results, drafts, up), key=lambda x: x[0]):
        kept, at = got[:-1].tolist(), 0
        near(pd.logits[a], refs[s].run(first.view(1)))
        for tok in kept:
            at = next(i + 1 for i in range(len(p)) if p[i] == at and t[i].item() == tok)
            near(pd.logits[a + at], refs[s].run(torch.tensor([tok], device=first.device)))
        assert got[-1] == pd.logits[a + at].argmax() and pd.tok[s] == got[-1]
        a += 1 + len(p)


def test_verify_greedy(dec, cuda):
    """Chains and trees of three slots of four, right and wrong tokens, two passes and a step behind them: logits of every kept
    row against the reference, the kept tokens those of greedy decoding by the pass's own logits."""
    from e2e_decoder import PagedDecoder
    d, W = dec
    pd = PagedDecoder(d, 4, max_len=120, page_tokens=32)
    slots = [3, 0, 2]
    refs = {s: Ref(d, W) for s in slots}
    prompts = [ids(n, n, cuda) for n in (5, 40, 31)]
    pd.prompt(slots, prompts)
    for s, p in zip(slots, prompts):
        refs[s].run(p)
    # what the model itself would say next: a copy of the cache decodes it
    probe = PagedDecoder(d, 4, max_len=120, page_tokens=32)
    probe.prompt(slots, prompts)
    says = torch.stack([probe.step() for _ in range(6)])
    wrong = ids(6, 99, cuda)
    for turn in range(2):
        if turn == 0:
            drafts = [says[:4, 3], torch.cat([says[:2, 0], wrong[:3]]), torch.cat([wrong[:2], says[:1, 2], wrong[2:4], says[1:2, 2]])]
            up = [[0, 1, 2, 3], [0, 1, 2, 3, 4], [0, 0, 0, 1, 3, 3]]
        else:
            drafts, up = [wrong[:0], wrong[:3], wrong[3:5]], [[], [0, 0, 1], [0, 1]]
        before, lens = [pd.tok[s].clone() for s in slots], list(pd.lens)
        out = pd.verify(slots, drafts, up if turn == 0 else [torch.tensor(p) for p in up])
        follow(refs, pd, slots, before, out, drafts, up)
        assert pd.cache.lens.tolist() == pd.lens == [lens[s] + (len(out[slots.index(s)]) if s in slots else 0) for s in range(4)]
    for i in range(3):
        fed = pd.tok.clone()
        pd.step(use_graph=i > 0)
        for s in slots:
            near(pd.logits[s], refs[s].run(fed[s:s + 1]))
    pd.cache.check()


def test_verify_sampled(dec, cuda):
    """Temperatures, uniforms and draft probabilities reach the verification in the order of the slots: the same as
    verify_draft on the pass's logits."""
    from e2e_decoder import PagedDecoder
    from sx8_draft import verify_draft
    d, _ = dec
    pd = PagedDecoder(d, 3, max_len=100, page_tokens=64)
    pd.prompt([0, 2, 1], [ids(n, n, cuda) for n in (9, 3, 70)])
    V, slots, ns = TINY["vocab"], [2, 0], [4, 2]
    g = torch.Generator().manual_seed(5)
    for probs in (None, [torch.softmax(torch.randn(1 + n, V, generator=g), -1).to(cuda) for n in ns]):
        lens, tok = list(pd.lens), pd.tok.clone()
        drafts = [ids(n, 7 + n, cuda) for n in ns]
        u = [torch.rand(1 + n, generator=g).to(cuda) for n in ns]
        out = pd.verify(slots, drafts, uniforms=u, temperature=[0.9, 1.4], draft_probs=probs)
        i32 = dict(dtype=torch.int32, device=cuda)
        rows = torch.cat([tok[0:1], drafts[1], tok[2:3], drafts[0]])
        path, counts, nxt = verify_draft(pd.logits, rows, torch.tensor([-1, 0, 1, -1, 0, 1, 2, 3], **i32), torch.tensor([0, 3, 8], **i32),
                                         torch.cat([u[1], u[0]]), torch.tensor([1.4, 0.9], device=cuda),
                                         None if probs is None else torch.cat([probs[1], probs[0]]))
        for slot, j, a in ((0, 0, 0), (2, 1, 3)):
            kept = counts[j].item()
            want = rows[a + path[a + 1:a + kept].long()].tolist() + [nxt[j].item()]
            assert out[slots.index(slot)].tolist() == want and pd.lens[slot] == lens[slot] + kept
        assert pd.lens[1] == lens[1] and pd.tok[1] == tok[1] and pd.cache.lens.tolist() == pd.lens


def test_verify_refuses(dec, cuda):
    from e2e_decoder import PagedDecoder
    d, _ = dec
    pd = PagedDecoder(d, 2, max_len=40, page_tokens=32)
    pd.prompt([0], [ids(30, 1, cuda)])
    three = ids(3, 2, cuda)
    before = [t.clone() for t in (pd.cache.pages, pd.cache.table, pd.cache.lens, pd.cache.refs)]
    for args, word in ((([1], [three]), "not in use"), (([0], [ids(10, 3, cuda)]), "past 40"), (([0, 0], [three, three]), "different"),
                       (([0], []), "as many"), (([], []), "at least one"), (([0], [three], [[0, 1]]), "parent"),
                       (([0], [three], [[0, 2, 1]]), "parent"), (([0], [three], [[0, -1, 1]]), "parent"), (([2], [three]), "out of range"),
                       (([0], [three], None, [torch.rand(3)]), "uniforms"), (([0], [three], None, [torch.rand(4)], [0.5, 0.5]), "temperature"),
                       (([0], [three], None, None, 0.7), "uniforms"), (([0], [three], None, None, [0.0]), "uniforms"),
                       (([0], [three], None, [torch.rand(4)], 1.0, [torch.rand(4, 3)]), "draft_probs"),
                       (([0], [three], None, [torch.rand(4)], 1.0, [torch.rand(4, TINY["vocab"], dtype=torch.float64)]), "draft_probs")):
        with pytest.raises(ValueError, match=word):
            pd.verify(*args)
    assert all(torch.equal(a, b) for a, b in zip(before, (pd.cache.pages, pd.cache.table, pd.cache.lens, pd.cache.refs))) and pd.lens == [30, 0]
    # no page left: refused before the pass, nothing changed
    small = PagedDecoder(d, 2, max_len=64, n_pages=1, page_tokens=32)
    small.prompt([0], [ids(31, 1, cuda)])
    with pytest.raises(RuntimeError, match="no free pages"):
        small.verify([0], [three])
    assert small.lens == [31, 0] and small.cache.lens.tolist() == [31, 0]
    got = small.verify([0], [three[:0]])
    assert small.lens == [32, 0] and got[0].shape == (1,)
