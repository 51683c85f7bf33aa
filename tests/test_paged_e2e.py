"""The decoder's batched path (packed prompts, 4-bit paged cache, graph-replayed steps) against a float32 decoder over the
exactly dequantized weights whose cache holds the 4-bit values.

Tolerances: the float32 decoder and the kernels differ by fp16 roundings of activations (the single-sequence path meets 2e-2
of the largest logit in test_e2e.py).  A K or V value that differs by a rounding can fall to the next level, a fifteenth
of its group's range; such values are few and their errors average out: 5e-2 of the largest logit."""
import pytest
import torch

from test_e2e import TINY, _dequant_all
from test_paged_kv import q4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(hiplib, cuda):
    from e2e_decoder import SX8Decoder
    d = SX8Decoder(TINY, device=cuda, seed=3, n_distinct=2, max_len=160)
    return d, _dequant_all(d, cuda)


class Ref:
    """One sequence in float32: the cache holds what 4 bits stand for; a first prompt attends its own rows."""

    def __init__(self, dec, W):
        self.d, self.W, self.k, self.v, self.n = dec, W, [None] * 99, [None] * 99, 0

    def run(self, ids):
        d, cfg = self.d, self.d.cfg
        nh, nk, hd, eps = cfg["n_heads"], cfg["n_kv"], cfg["head_dim"], cfg["eps"]
        T, n0 = ids.shape[0], self.n

        def rms(x, w):
            return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.float()

        def rope(x):
            h = hd // 2
            c, s = d.cos[n0:n0 + T][:, None, :], d.sin[n0:n0 + T][:, None, :]
            return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)

        x = self.W["head"][ids].float()
        for li, ly in enumerate(d.layers):
            w = self.W[li]
            h = rms(x, ly.in_norm)
            q = rope(rms((h @ w["q"].T).view(T, nh, hd), ly.q_norm))
            k = rope(rms((h @ w["k"].T).view(T, nk, hd), ly.k_norm))
            v = (h @ w["v"].T).view(T, nk, hd)
            k4, v4 = q4(k.half()).float(), q4(v.half()).float()
            if n0:
                k4, v4 = torch.cat([self.k[li], k4]), torch.cat([self.v[li], v4])
            self.k[li], self.v[li] = k4, v4
            if n0 or T == 1:
                k, v = k4, v4
            L, rep = k.shape[0], nh // nk
            kt = k.repeat_interleave(rep, 1).permute(1, 2, 0).contiguous()
            vh = v.repeat_interleave(rep, 1).permute(1, 0, 2).contiguous()
            s = torch.matmul(q.permute(1, 0, 2).contiguous(), kt) / hd ** 0.5
            s = s.masked_fill(torch.arange(L, device=s.device) > n0 + torch.arange(T, device=s.device)[:, None], float("-inf"))
            a = torch.matmul(torch.softmax(s, -1), vh).permute(1, 0, 2).reshape(T, nh * hd)
            x = x + a @ w["o"].T
            h2 = rms(x, ly.post_norm)
            x = x + (torch.nn.functional.silu(h2 @ w["gate"].T) * (h2 @ w["up"].T)) @ w["down"].T
        self.n += T
        return (rms(x, d.final_norm) @ self.W["head"].T)[-1]


def near(got, want):
    rel = ((got - want).abs().max() / want.abs().max()).item()
    print("logits rel", rel, flush=True)
    assert rel <= 5e-2


def ids(n, seed, cuda):
    return torch.randint(0, TINY["vocab"], (n,), generator=torch.Generator().manual_seed(seed)).to(cuda)


def test_prompts_and_steps(dec, cuda):
    """Packed prompts and steps of three slots of four: logits of every token against the reference fed the same tokens."""
    from e2e_decoder import PagedDecoder
    d, W = dec
    pd = PagedDecoder(d, 4, max_len=100, page_tokens=32)
    prompts, slots = [ids(n, n, cuda) for n in (5, 40, 33)], [2, 0, 3]
    refs = [Ref(d, W) for _ in slots]
    tok = pd.prompt(slots, prompts)
    rows = {s: i for i, s in enumerate(sorted(slots))}
    for s, p, r, t in zip(slots, prompts, refs, tok):
        want = r.run(p)
        near(pd.logits[rows[s]], want)
        assert t == pd.logits[rows[s]].argmax()
    for i in range(6):
        fed = pd.tok.clone()
        nxt = pd.step(use_graph=i != 1)
        for s, r in zip(slots, refs):
            near(pd.logits[s], r.run(fed[s:s + 1]))
            assert nxt[s] == pd.logits[s].argmax()
    pd.cache.check()
    assert pd.cache.lens.tolist() == pd.lens == [46, 0, 11, 39]


def test_shared_prefix_fork_free_compact(dec, cuda):
    """A prefix run once and forked; its slots go on with prompts of their own; one is freed, the pool compacted and the
    slot used again."""
    from e2e_decoder import PagedDecoder
    d, W = dec
    pd = PagedDecoder(d, 3, max_len=128, n_pages=11, page_tokens=32)
    prefix = ids(50, 1, cuda)
    pd.prompt([2], [prefix])
    pd.fork([2, 2], [0, 1])
    shared = pd.cache.table[0, 0].item()
    assert pd.cache.refs[shared] == 3 and pd.cache.table[0, 1] != pd.cache.table[1, 1]
    tails = [ids(9, 2, cuda), ids(20, 3, cuda)]
    pd.prompt([0, 1], tails)
    refs = [Ref(d, W) for _ in range(2)]
    for i in range(2):
        refs[i].run(prefix)
        near(pd.logits[i], refs[i].run(tails[i]))
    for i in range(3):
        fed = pd.tok.clone()
        pd.step()
        for j in range(2):
            near(pd.logits[j], refs[j].run(fed[j:j + 1]))
    pd.free([0])
    pd.compact()
    used = int((pd.cache.refs > 0).sum())
    assert (pd.cache.refs[:used] > 0).all() and pd.cache.table.max() < used
    new = ids(30, 4, cuda)
    pd.prompt([0], [new])
    refs[0] = Ref(d, W)
    near(pd.logits[0], refs[0].run(new))
    for i in range(2):
        fed = pd.tok.clone()
        pd.step()
        for j in range(2):
            near(pd.logits[j], refs[j].run(fed[j:j + 1]))
    pd.cache.check()


def test_long_prompts_after_a_prefix(dec, cuda):
    """Many new tokens behind tokens that the cache holds: the pages' values read back and attended."""
    from e2e_decoder import PagedDecoder
    d, W = dec
    pd = PagedDecoder(d, 3, max_len=160, page_tokens=64)
    refs = [Ref(d, W) for _ in range(2)]
    first, tails = [ids(11, 1, cuda), ids(3, 2, cuda)], [ids(140, 3, cuda), ids(131, 4, cuda)]
    pd.prompt([2, 0], first)
    pd.prompt([2, 0], tails)
    for row, i in ((1, 0), (0, 1)):
        refs[i].run(first[i])
        near(pd.logits[row], refs[i].run(tails[i]))
    fed = pd.tok.clone()
    pd.step()
    near(pd.logits[2], refs[0].run(fed[2:3]))
    pd.cache.check()


def test_generate_batch(dec, cuda):
    """generate_batch: graph and eager steps give the same tokens, with and without a shared prefix."""
    d, _ = dec
    prompts = [ids(n, n, cuda) for n in (7, 30, 1)]
    for prefix in (None, ids(40, 9, cuda)):
        a = d.generate_batch(prompts, 6, prefix=prefix, page_tokens=32)
        assert a.shape == (3, 6) and torch.equal(a, d.generate_batch(prompts, 6, prefix=prefix, page_tokens=32, use_graph=False))


def test_paged_decoder_refuses(dec, cuda):
    from e2e_decoder import PagedDecoder
    d, _ = dec
    with pytest.raises(ValueError):
        PagedDecoder(d, 2, max_len=1000)
    pd = PagedDecoder(d, 2, max_len=40, n_pages=2, page_tokens=32)
    for slots, prompts in (([2], [ids(3, 1, cuda)]), ([0, 0], [ids(3, 1, cuda)] * 2), ([0], [ids(41, 1, cuda)]), ([], []),
                           ([0], [ids(0, 1, cuda)]), ([0, 1], [ids(3, 1, cuda)])):
        with pytest.raises(ValueError):
            pd.prompt(slots, prompts)
    with pytest.raises(RuntimeError, match="no free pages"):
        pd.prompt([0, 1], [ids(40, 1, cuda)] * 2)
    pd.prompt([0], [ids(40, 1, cuda)])
    with pytest.raises(ValueError):
        pd.step()
    for src, dst in (([0], [0]), ([1], [0]), ([0, 0], [1, 1])):
        with pytest.raises(ValueError):
            pd.fork(src, dst)
    with pytest.raises(RuntimeError, match="no free pages"):
        pd.fork([0], [1])
    with pytest.raises(ValueError):
        pd.free([2])
    # a step that would need a page too many is refused before it changes anything
    pd = PagedDecoder(d, 2, max_len=64, n_pages=2, page_tokens=32)
    pd.prompt([0, 1], [ids(31, 1, cuda), ids(32, 2, cuda)])
    state = pd.cache.table.clone(), pd.cache.lens.clone(), pd.cache.pages.clone()
    with pytest.raises(RuntimeError, match="no free pages"):
        pd.step()
    assert all(torch.equal(a, b) for a, b in zip(state, (pd.cache.table, pd.cache.lens, pd.cache.pages)))
    pd.free([1])
    pd.step()
    pd.step()
    pd.cache.check()
    assert pd.cache.lens.tolist() == pd.lens == [33, 0]


def test_generate_batch_refuses(dec, cuda):
    d, _ = dec
    for prompts, n in (([], 3), ([ids(3, 1, cuda)], 0), ([ids(3, 1, cuda)], 500), ([ids(0, 1, cuda)], 2)):
        with pytest.raises(ValueError):
            d.generate_batch(prompts, n)


def test_a_pass_that_fails_midway(dec, cuda, monkeypatch):
    """Where the layers raise, the decoder's lengths are still the cache's: the slot can be freed and used again."""
    from e2e_decoder import PagedDecoder
    d, _ = dec
    pd = PagedDecoder(d, 2, max_len=64, page_tokens=32)
    pd.prompt([0], [ids(9, 1, cuda)])
    with monkeypatch.context() as m:
        m.setattr(pd, "_rows", lambda *a: (_ for _ in ()).throw(MemoryError()))
        with pytest.raises(MemoryError):
            pd.prompt([1], [ids(5, 2, cuda)])
        with pytest.raises(MemoryError):
            pd.step(use_graph=False)
    assert pd.lens == pd.cache.lens.tolist() == [10, 6]
    pd.free([0, 1])
    a = pd.prompt([0, 1], [ids(9, 1, cuda), ids(5, 2, cuda)])
    fresh = PagedDecoder(d, 2, max_len=64, page_tokens=32)
    assert torch.equal(a, fresh.prompt([0, 1], [ids(9, 1, cuda), ids(5, 2, cuda)]))
    assert torch.equal(pd.step(), fresh.step())
