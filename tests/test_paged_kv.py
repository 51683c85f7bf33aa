"""The paged 4-bit KV cache and the attention of packed sequences on the GPU, against plain
implementations in 64 bits.

Tolerances.  Encoding and reading back are exact: the levels are decided exactly, and a value is one rounding of
m + s level.  Attention outputs are rounded once to their type (half a step, finfo.eps / 2 of the value); before that
  attend: scores are sums of 32-bit products (hd terms; relative 2^-24 each, at most hd 2^-24 of sum |q k|), p * s
    carries 22 bits, sums are 32-bit; with |score| <= 64 in powers of two the weights are within 2^-24 * 64 * 4 = 2^-16
    of themselves, so the output within 2^-15 of the largest value it averages: LOOSE = 2^-15 max |v|.
  varlen: the weights are rounded to the type as well: each within eps / 2 of itself, so the average within
    eps / 2 of the average of |v|, at most eps / 2 max |v|, beside the same 2^-15.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
LOOSE = 2.0 ** -15


# ------------------------------------------------------------------------------ plain implementations, 64 bits
def q4(x):
    """The values that rows (..., hd) stand for in 4 bits."""
    g = x.double().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    r = (hi.float() - lo.float()) * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    s = r.clamp(max=65504.0).half().double()
    m = lo.float().clamp(-65504.0, 65504.0).half().double()
    lv = ((g - m) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15) * (s > 0)
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    return torch.where(bad, math.nan, m + s * lv).flatten(-2)


def attention(q, k, v, first, scale=None, causal=True):
    """q (n, nh, d), k / v (l, nk, d) float64: row i sees keys 0 .. first + i (all of them without causal)."""
    n, nh, d = q.shape
    l, nk = k.shape[:2]
    if l == 0 or n == 0:
        return torch.zeros_like(q)
    rep = nh // nk
    kk = k.repeat_interleave(rep, 1).permute(1, 2, 0).contiguous()
    vv = v.repeat_interleave(rep, 1).permute(1, 0, 2).contiguous()
    w = torch.matmul(q.permute(1, 0, 2).contiguous(), kk) * (scale or 1 / math.sqrt(d))
    see = torch.arange(l, device=q.device) <= first + torch.arange(n, device=q.device)[:, None]
    if not causal:
        see = torch.ones_like(see)
    w = w.masked_fill(~see, -math.inf)
    p = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e300))
    # a key that is not seen has no part in the row, whatever it holds
    vz = torch.where(torch.isfinite(vv), vv, 0.0)
    o = torch.matmul(p, vz)
    odd = (~torch.isfinite(vv)).double()
    o = torch.where(torch.matmul((p > 0).double(), odd) > 0, math.nan, o)
    return (o / p.sum(-1, keepdim=True).clamp(min=1e-300)).permute(1, 0, 2)


def close(got, want, dt, top, more=0.0):
    """got within half a step of want, and LOOSE + more of top."""
    half = torch.finfo(dt).eps / 2
    err = (got.double() - want).abs()
    bound = half * want.abs() * (1 + half) + (LOOSE + more) * top + torch.finfo(dt).tiny
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "NaN in other places"
    worst = ((err - bound).masked_fill(nan, -1.0)).max().item() if err.numel() else -1.0
    assert worst <= 0, f"off by {worst} over the bound"


# ------------------------------------------------------------------------------ helpers
def rand(shape, seed, dt, cuda, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt).to(cuda)


def ints(xs, cuda):
    return torch.tensor(list(xs), dtype=torch.int32, device=cuda)


def cum(ns, cuda):
    out = [0]
    for n in ns:
        out.append(out[-1] + n)
    return ints(out, cuda)


def make(cuda, lens, nk=2, hd=128, pt=64, dt=F16, seed=0, layers=1, spare=0, width=None):
    """A cache with slots of these lengths and its K and V rows (the rows that were encoded)."""
    from sx8_paged_kv import PagedKV4
    need = [(n + pt - 1) // pt for n in lens]
    p = PagedKV4(layers, nk, hd, sum(need) + spare, len(lens), width or max(max(need), 1) + 1, pt, device=cuda)
    p.reserve(ints(lens, cuda))
    T = sum(lens)
    k, v = rand((T, nk, hd), seed, dt, cuda), rand((T, nk, hd), seed + 1, dt, cuda, 0.5)
    k[..., 3] += 4
    if T:
        for layer in range(layers):
            p.append(layer, k, v, cum(lens, cuda))
    p.check()
    return p, k, v


def want_attend(q, k, v, lens, new, scale=None):
    """The reference for packed rows: k, v the values that the cache stands for, by slot."""
    out, a, b = [], 0, 0
    for n, ln in zip(new, lens):
        out.append(attention(q[a:a + n].double(), k[b:b + ln], v[b:b + ln], ln - n, scale))
        a, b = a + n, b + ln
    return torch.cat(out) if out else q.double()


# ------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("pt", [32, 128])
def test_append_read_exact(hiplib, cuda, hd, dt, pt):
    """What is read back is the one rounding of what the definition gives, in several calls that end inside blocks."""
    lens, steps = [0, 1, 33, 70, 200], [[0, 1, 31, 5, 130], [0, 0, 1, 64, 1], [0, 0, 1, 1, 69]]
    from sx8_paged_kv import PagedKV4
    p = PagedKV4(1, 3, hd, 32, 5, 8, pt, device=cuda)
    parts = [[] for _ in lens]
    for i, ns in enumerate(steps):
        p.reserve(ints(ns, cuda))
        k, v = rand((sum(ns), 3, hd), 10 * i, dt, cuda), rand((sum(ns), 3, hd), 10 * i + 1, dt, cuda, 0.1)
        p.append(0, k, v, cum(ns, cuda))
        a = 0
        for s, n in enumerate(ns):
            parts[s].append((k[a:a + n], v[a:a + n]))
            a += n
    p.check()
    assert p.lens.tolist() == lens
    k, v = (torch.cat([x[j] for part in parts for x in part]) for j in range(2))
    gk, gv = p.read(0, sum(lens), cum(lens, cuda), dtype=dt)
    assert torch.equal(gk, q4(k).to(dt)) and torch.equal(gv, q4(v).to(dt))
    # the last tokens alone
    ns = [0, 1, 2, 33, 7]
    lk, lv = p.read(0, sum(ns), cum(ns, cuda), dtype=dt)
    at = torch.cat([torch.arange(e - n, e) for n, e in zip(ns, torch.tensor(lens).cumsum(0).tolist())]).to(cuda)
    assert torch.equal(lk, gk[at]) and torch.equal(lv, gv[at])


def test_append_special_values(hiplib, cuda):
    """Constant groups, ties, subnormals, the largest values, NaN and infinities: as the definition says."""
    from sx8_paged_kv import PagedKV4
    for dt in (F16, BF16):
        x = torch.zeros(12, 1, 64, dtype=torch.float64)
        x[0] = 3.25
        x[1, 0] = torch.arange(64) % 31 * 0.5                      # levels and the middles between them
        x[2, 0] = torch.linspace(-65504, 65504, 64, dtype=torch.float64)
        x[3, 0] = torch.arange(64) * 2.0 ** -24
        x[4, 0, 5] = math.nan
        x[5, 0, 63] = math.inf
        x[6, 0, 0] = -math.inf
        x[7, 0] = torch.randn(64, dtype=torch.float64) * 1e-5 + 100
        x[8, 0] = -torch.arange(64) % 16 * 0.0625
        x[9, 0] = torch.randn(64, dtype=torch.float64) * 3e4
        x[10, 0] = torch.randn(64, dtype=torch.float64) * (1e38 if dt is BF16 else 1e4)
        x[11, 0, 0] = 15.0
        x = x.to(dt).to(cuda)
        p = PagedKV4(1, 1, 64, 1, 1, 1, 32, device=cuda)
        p.reserve(ints([12], cuda))
        p.append(0, x, x, cum([12], cuda))
        k, v = p.read(0, 12, cum([12], cuda), dtype=BF16 if dt is BF16 else F16)
        want = q4(x).to(k.dtype)
        assert torch.equal(k.view(torch.int16)[torch.isfinite(want)], want.view(torch.int16)[torch.isfinite(want)])
        assert torch.equal(torch.isnan(k), torch.isnan(want)) and torch.equal(torch.isinf(k), torch.isinf(want))
        assert torch.equal(torch.nan_to_num(k), torch.nan_to_num(v))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_append_near_borders(hiplib, cuda, dt):
    """Values at the middle between two levels and next to it, over groups of every size and offset: the exact level."""
    from sx8_paged_kv import PagedKV4
    n, hd = 4096, 128
    g = torch.Generator().manual_seed(7)
    lo = torch.randn(n, 2, 1, generator=g).double() * 10.0 ** (torch.rand(n, 2, 1, generator=g) * 8 - 5)
    lo = lo.clamp(-6e4, 6e4).to(dt)
    hi = (lo.double() + 10.0 ** (torch.rand(n, 2, 1, generator=g).double() * 8 - 5)).clamp(-6e4, 6e4).to(dt)
    s = ((hi.float() - lo.float()) * torch.tensor(1 / 15, dtype=torch.float32)).half().double()
    m = lo.float().half().double()
    x = (m + (torch.randint(0, 15, (n, 2, 64), generator=g) + 0.5) * s).to(dt)
    step = torch.randint(-1, 2, (n, 2, 64), generator=g, dtype=torch.int16)
    x = (x.view(torch.int16) + step * (x != 0)).view(dt)
    x = torch.minimum(torch.maximum(x, lo), hi)
    x[..., 0], x[..., 63] = lo[..., 0], hi[..., 0]
    k = x.reshape(n, 1, hd).to(cuda)
    v = k.flip(0).contiguous()
    p = PagedKV4(1, 1, hd, n // 64, 1, n // 64, 64, device=cuda)
    p.reserve(ints([n], cuda))
    p.append(0, k, v, cum([n], cuda))
    gk, gv = p.read(0, n, cum([n], cuda), dtype=dt)
    assert torch.equal(gk, q4(k).to(dt)) and torch.equal(gv, q4(v).to(dt))


def test_append_keeps_other_bytes(hiplib, cuda):
    """Bytes of tokens that a call does not bring stay as they are, and so do pages of other slots."""
    p, k, v = make(cuda, [45, 70], pt=64, spare=2)
    before = p.pages.clone()
    bk, bv = p.read(0, 115, cum([45, 70], cuda))
    p.append(0, rand((5, 2, 128), 7, F16, cuda), rand((5, 2, 128), 8, F16, cuda), cum([2, 3], cuda))
    ak, av = p.read(0, 115, cum([45, 70], cuda))
    keep = [i for i in range(115) if not (43 <= i < 45 or 112 <= i < 115)]
    assert torch.equal(ak[keep], bk[keep]) and torch.equal(av[keep], bv[keep])
    assert not torch.equal(ak[43:45], bk[43:45])
    used = p.table[p.table >= 0].unique().long()
    rest = [i for i in range(p.n_pages) if i not in used.tolist()]
    assert torch.equal(p.pages[:, rest], before[:, rest])


def test_append_read_strides_and_alignment(hiplib, cuda):
    """Rows out of a wider tensor, head-major rows, and rows that begin off 16 bytes."""
    from sx8_paged_kv import PagedKV4
    n, nk, hd = 37, 2, 128
    want = rand((n, nk, hd), 3, F16, cuda)
    wide = torch.zeros(n, 3, nk, hd, dtype=F16, device=cuda)
    wide[:, 1] = want
    major = want.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    odd = torch.zeros(n * nk * hd + 1, dtype=F16, device=cuda)[1:].view(n, nk, hd)
    odd.copy_(want)
    one = want[:1].expand(n, nk, hd)
    for x in (wide[:, 1], major, odd, one):
        p = PagedKV4(1, nk, hd, 2, 1, 2, 32, device=cuda)
        p.reserve(ints([n], cuda))
        p.append(0, x, x, cum([n], cuda))
        big = torch.full((n, nk, 2 * hd), 7.0, dtype=F16, device=cuda)
        k, v = p.read(0, n, cum([n], cuda), out=(big[..., :hd], torch.empty_like(want)))
        assert torch.equal(k, q4(x).half()) and torch.equal(v, k)
        assert (big[..., hd:] == 7).all()


# ------------------------------------------------------------------------------ attend
LENS = [0, 1, 31, 32, 33, 64, 500, 1030]


@pytest.mark.parametrize("nh,nk,hd", [(8, 2, 128), (4, 4, 128), (6, 1, 64), (20, 4, 128), (32, 1, 64), (8, 1, 256)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_one_token(hiplib, cuda, nh, nk, hd, dt):
    p, k, v = make(cuda, LENS, nk, hd, 32, dt)
    q = rand((len(LENS), nh, hd), 5, dt, cuda)
    got = p.attend(0, q)
    vv = q4(v)
    new = [1] * len(LENS)
    out, b = [], 0
    for i, ln in enumerate(LENS):
        out.append(attention(q[i:i + 1].double(), q4(k[b:b + ln]), vv[b:b + ln], ln - 1))
        b += ln
    assert new and got.dtype == dt
    close(got, torch.cat(out), dt, vv.abs().max().item())
    assert not got[0].any()                                         # a slot with no token


@pytest.mark.parametrize("hd,pt", [(64, 64), (128, 128), (256, 32)])
def test_attend_many_tokens(hiplib, cuda, hd, pt):
    """Several new tokens a slot, none for some: tiles of 16 rows that end inside tokens, and causal borders."""
    lens, new = [5, 40, 0, 300, 33, 700], [5, 3, 0, 17, 0, 60]
    p, k, v = make(cuda, lens, 2, hd, pt)
    q = rand((sum(new) + 3, 6, hd), 6, F16, cuda)
    out = torch.full_like(q, 9.0)
    got = p.attend(0, q, cum(new, cuda), out=out)
    close(got[:sum(new)], want_attend(q, q4(k), q4(v), lens, new), F16, q4(v).abs().max().item())
    assert (got[sum(new):] == 9).all()                              # rows behind the last sequence


def test_attend_whole_prompts(hiplib, cuda):
    """Every token of a slot as a new one (its first rows see one key)."""
    lens = [130, 1, 515]
    p, k, v = make(cuda, lens, 1, 128, 64)
    q = rand((sum(lens), 3, 128), 8, F16, cuda)
    close(p.attend(0, q, cum(lens, cuda)), want_attend(q, q4(k), q4(v), lens, lens), F16, q4(v).abs().max().item())


def test_attend_long_and_cut(hiplib, cuda):
    """One long slot beside short ones: its blocks are shared by many work-groups and joined."""
    lens = [70000, 3, 900, 1]
    p, k, v = make(cuda, lens, 1, 128, 256)
    for dt, scale in ((F16, None), (BF16, 0.3)):
        q = rand((4, 8, 128), 9, dt, cuda)
        close(p.attend(0, q, scale=scale), want_attend(q, q4(k), q4(v), lens, [1] * 4, scale), dt, q4(v).abs().max().item())
    again = p.attend(0, q, scale=0.3)
    assert torch.equal(again, p.attend(0, q, scale=0.3))


def test_attend_cu_backwards(hiplib, cuda):
    """A cu that names the same rows for many slots: more units than rows allow, still inside the memory."""
    from sx8_paged_kv import PagedKV4
    p = PagedKV4(1, 1, 64, 2, 4096, 1, 32, device=cuda)
    p.reserve(ints([1, 1] + [0] * 4094, cuda))
    q = rand((64, 256, 64), 1, F16, cuda)
    k = rand((64, 1, 64), 1, F16, cuda)
    cu = ints([0, 64] * 2048 + [64], cuda)
    out = p.attend(0, q, cu)
    p.append(0, k, k, cu)
    p.read(0, 64, cu)
    torch.cuda.synchronize()
    assert out.shape == q.shape and p.refs.tolist() == [1, 1]


@pytest.mark.parametrize("n_slots", [64, 65, 300, 4096])
@pytest.mark.parametrize("nk", [1, 9])
def test_attend_many_slots(hiplib, cuda, n_slots, nk):
    """More slots than a wave has lanes, more units than the launch has waves, with and without cu."""
    lens = [(37 * i) % 71 for i in range(n_slots)]
    p, k, v = make(cuda, lens, nk, 64, 32)
    kk, vv = q4(k), q4(v)
    some = [i for i in range(n_slots) if i < 70 or i % 97 == 0 or i > n_slots - 3]
    ends = torch.tensor(lens).cumsum(0).tolist()
    for new in ([1] * n_slots, [(5 * i) % 4 for i in range(n_slots)]):
        q = rand((sum(new), 2 * nk, 64), 3, F16, cuda)
        got = p.attend(0, q, cum(new, cuda))
        if new[0] == 1:
            assert torch.equal(got, p.attend(0, q))
        firsts = torch.tensor([0] + new).cumsum(0).tolist()
        for i in some:
            a, b, e = firsts[i], ends[i], lens[i]
            want = attention(q[a:a + new[i]].double(), kk[b - e:b], vv[b - e:b], e - new[i])
            close(got[a:a + new[i]], want, F16, 4.0)


def test_attend_more_rows_than_tokens(hiplib, cuda):
    """More new rows than the slot has tokens: the first rows see none and give zeros."""
    p, k, v = make(cuda, [2, 40], 2, 64, 32)
    q = rand((9, 2, 64), 4, F16, cuda)
    got = p.attend(0, q, cum([5, 4], cuda))
    want = want_attend(q, q4(k), q4(v), [2, 40], [5, 4])
    close(got, want, F16, q4(v).abs().max().item())
    assert not got[:3].any() and got[3].any()
    before = p.pages.clone()
    rk, _ = p.read(0, 9, cum([5, 4], cuda), out=(torch.full_like(q, 7.0), torch.full_like(q, 7.0)))
    assert not rk[:3].any() and torch.equal(rk[3:5], q4(k[:2]).half())
    p.append(0, q, q, cum([40, 4], cuda)[:1].repeat(3) + ints([0, 5, 9], cuda))
    p.append(0, k[:2], v[:2], ints([0, 2, 2], cuda))
    p.append(0, k[-4:], v[-4:], ints([0, 0, 4], cuda))
    assert torch.equal(p.pages, before)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_query_sizes(hiplib, cuda, dt):
    """Queries from tiny to large (bf16: far past fp16's range) keep their precision."""
    p, k, v = make(cuda, [300] * 6, 1, 64, 64, F16)
    q = rand((6, 2, 64), 4, torch.float32, cuda)
    mags = torch.tensor([1e-6, 1e-3, 1.0, 30.0, 300.0, 0.0], device=cuda)
    if dt is BF16:
        mags = torch.tensor([1e-30, 1e-3, 1.0, 1e6, 1e20, 0.0], device=cuda)
    q = (q * mags[:, None, None]).to(dt)
    for scale, rows in ((0.125, [0, 1, 2, 5]), (0.125 / 64, [3] if dt is F16 else []),
                        (2.0 ** -23, [3] if dt is BF16 else [4]), (2.0 ** -69, [4] if dt is BF16 else [])):
        if rows:
            got = p.attend(0, q, scale=scale)
            want = want_attend(q, q4(k), q4(v), [300] * 6, [1] * 6, scale)
            close(got[rows], want[rows], dt, q4(v).abs().max().item())


@pytest.mark.parametrize("dt,size", [(F16, 65504.0), (F16, 60.0), (F16, 2e-3), (BF16, 3e38), (BF16, 1e6), (BF16, 1e-3)])
def test_attend_value_sizes(hiplib, cuda, dt, size):
    """Values from small ones to the ends of fp16 and far past them keep their precision: scales of every size times weights of
    every size."""
    from sx8_paged_kv import PagedKV4
    n = 100
    p = PagedKV4(1, 1, 64, 4, 1, 4, 32, device=cuda)
    p.reserve(ints([n], cuda))
    k = rand((n, 1, 64), 1, dt, cuda)
    v = (torch.rand(n, 1, 64, generator=torch.Generator().manual_seed(2)) * 2 - 1).to(cuda)
    v[0, 0, 0], v[0, 0, 1] = 1, -1
    v = (v.double() * size).to(dt)
    p.append(0, k, v, cum([n], cuda))
    q = rand((1, 2, 64), 3, dt, cuda) * torch.tensor([1, 40], device=cuda, dtype=dt)[:, None]
    got = p.attend(0, q).double()
    vv = q4(v)
    want = attention(q.double(), q4(k), vv, n - 1)
    want = want.clamp(-torch.finfo(dt).max, torch.finfo(dt).max) if dt is F16 else want
    err = (got - want).abs().max().item()
    assert err <= (torch.finfo(dt).eps / 2 + LOOSE) * vv.abs().max().item()


def test_attend_scales_that_grow(hiplib, cuda):
    """Blocks whose values grow from nothing to fp16's ends and back: the weights' common power of two
    follows them."""
    from sx8_paged_kv import PagedKV4
    sizes = [0.0, 1e-6, 1e-3, 1.0, 100.0, 65504.0, 1.0, 0.0, 30.0]
    n = 32 * len(sizes)
    p = PagedKV4(1, 1, 128, 9, 1, 9, 32, device=cuda)
    p.reserve(ints([n], cuda))
    k, v = rand((n, 1, 128), 1, F16, cuda), torch.zeros(n, 1, 128, dtype=F16, device=cuda)
    for i, size in enumerate(sizes):
        v[32 * i:32 * i + 32] = ((torch.rand(32, 1, 128, generator=torch.Generator().manual_seed(i)) * 2 - 1) * size).half().to(cuda)
    p.append(0, k, v, cum([n], cuda))
    # queries that pick out one block each, and one that sees all
    q = torch.zeros(1, 10, 128, dtype=F16, device=cuda)
    vv = q4(v)
    for i in range(9):
        q[0, i] = k[32 * i + 5, 0] * 4
    got = p.attend(0, q).double()
    want = attention(q.double(), q4(k), vv, n - 1)
    # a row's bound goes by the values that it gives weight: those of its block (others weigh below 2^-50 there)
    w = torch.softmax(torch.matmul(q[0].double(), q4(k)[:, 0].T.contiguous()) / 128 ** 0.5, -1)
    top = (w @ vv[:, 0].abs().amax(-1, keepdim=True)).flatten()
    for i in range(10):
        err = (got[0, i] - want[0, i]).abs().max().item()
        assert err <= (2.0 ** -11 + LOOSE) * max(top[i].item(), want[0, i].abs().max().item()) + 2.0 ** -25, (i, err)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attend_bits_do_not_depend_on_old_bytes(hiplib, cuda, hd):
    """What lies behind a slot's last token in its page does not change a bit of the result."""
    from sx8_paged_kv import PagedKV4
    lens, got = [45, 1, 130], []
    k, v = rand((sum(lens), 2, hd), 1, F16, cuda), rand((sum(lens), 2, hd), 2, F16, cuda)
    q = rand((3, 4, hd), 3, F16, cuda)
    for seed in (0, 1, 2):
        p = PagedKV4(1, 2, hd, 8, 3, 3, 64, device=cuda)
        if seed:
            p.pages.copy_(torch.randint(0, 256, p.pages.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.uint8))
        p.reserve(ints(lens, cuda))
        p.append(0, k, v, cum(lens, cuda))
        got.append(p.attend(0, q))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_attend_not_finite(hiplib, cuda):
    """NaN and infinity reach the rows that see them, and no others; garbage past the last token reaches none."""
    from sx8_paged_kv import PagedKV4
    n, lens = 6, [40, 38]
    p = PagedKV4(1, 2, 128, 4, 2, 2, 32, device=cuda)
    p.pages.fill_(255)                                              # every scale and minimum a NaN
    p.reserve(ints(lens, cuda))
    k, v = rand((78, 2, 128), 1, F16, cuda), rand((78, 2, 128), 2, F16, cuda)
    v[36, 1, 5] = math.nan                                          # slot 0, head 1: rows 2 .. 5 of its six see it
    k[76, 0, 70] = math.inf                                         # slot 1, token 36: rows 4, 5
    p.append(0, k, v, cum(lens, cuda))
    q = rand((2 * n, 4, 128), 3, F16, cuda)
    got = p.attend(0, q, cum([n, n], cuda))
    want = want_attend(q, q4(k), q4(v), lens, [n, n])
    nan = torch.isnan(got)
    assert nan[2:6, 2:, :64].all() and not nan[2:6, 2:, 64:].any()  # the group of dimension 5
    assert not nan[:2].any() and not nan[2:6, :2].any()
    assert nan[10:, :2].all() and not nan[6:10].any() and not nan[10:, 2:].any()
    ok = ~nan
    ref = torch.where(ok, torch.nan_to_num(want), 0.0)
    close(torch.where(ok, got, 0), ref, F16, 4.0)


def test_attend_bad_pages(hiplib, cuda):
    """Page numbers out of range are no tokens for attend, and neither read nor written."""
    p, k, v = make(cuda, [100, 64], 1, 64, 32, spare=1)
    q = rand((2, 2, 64), 3, F16, cuda)
    kk, vv = q4(k), q4(v)
    table = p.table.clone()
    for bad in (-1, p.n_pages, 2 ** 31 - 1, -2 ** 31):
        p.table[0, 1] = bad
        keep = torch.tensor([i for i in range(100) if not 32 <= i < 64], device=cuda)
        want = attention(q[:1].double(), kk[keep], vv[keep], 68)
        close(p.attend(0, q)[:1], want, F16, vv.abs().max().item())
        before = p.pages.clone()
        x = torch.full((100, 1, 64), 5.0, dtype=F16, device=cuda)
        p.append(0, x, x, ints([0, 100, 100], cuda))
        rk, _ = p.read(0, 100, ints([0, 100, 100], cuda))
        assert not rk[32:64].any() and (rk[keep] == 5).all()
        p.pages.copy_(before)
        p.table.copy_(table)
    close(p.attend(0, q), want_attend(q, kk, vv, [100, 64], [1, 1]), F16, vv.abs().max().item())


def test_attend_odd_lengths_of_the_tables(hiplib, cuda):
    """Lengths past the table, below zero and cu that runs past the rows stay inside the memory."""
    p, k, v = make(cuda, [64, 32], 1, 64, 32, width=2)
    p.lens.copy_(ints([1 << 30, -5], cuda))
    q = rand((2, 1, 64), 3, F16, cuda)
    got = p.attend(0, q)
    close(got[:1], attention(q[:1].double(), q4(k[:64]), q4(v[:64]), 63), F16, 4.0)
    assert not got[1].any()
    p.append(0, q, q)
    p.lens.copy_(ints([64, 32], cuda))
    for cu in ([0, 50, -3], [-9, 1, 1 << 30], [5, 2, 1], [0, 2, 0]):
        out = torch.full_like(q, 3.0)
        p.attend(0, q, ints(cu, cuda), out=out)
        p.read(0, 2, ints(cu, cuda))
        assert torch.isfinite(out).all()


# ------------------------------------------------------------------------------ pages
class Pool:
    """The page operations in plain Python."""

    def __init__(self, n_slots, width, n_pages, pt):
        self.rows = [[] for _ in range(n_slots)]
        self.lens, self.refs = [0] * n_slots, [0] * n_pages
        self.width, self.pt = width, pt

    def free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def reserve(self, add):
        need = [-(-(l + a) // self.pt) - (-(-l // self.pt)) for l, a in zip(self.lens, add)]
        for s, (l, a) in enumerate(zip(self.lens, add)):
            if a < 0:
                return (1, s)
            if l + a > self.width * self.pt:
                return (3, s)
        free = self.free_pages()
        if sum(need) > len(free):
            return (2, 0)
        for s, n in enumerate(need):
            for _ in range(n):
                self.rows[s].append(free.pop(0))
                self.refs[self.rows[s][-1]] = 1
            self.lens[s] += add[s]
        return None

    def fork(self, src, dst):
        n = len(self.lens)
        errors = []
        for i, (a, b) in enumerate(zip(src, dst)):
            if not (0 <= a < n and 0 <= b < n):
                errors.append((i, 1))
            elif self.lens[b]:
                errors.append((i, 4))
        if errors:
            return min(errors)[::-1]
        if len(set(dst)) < len(dst) or set(src) & set(dst):
            return (4, 0)
        free = self.free_pages()
        if sum(self.lens[a] % self.pt != 0 for a in src) > len(free):
            return (2, 0)
        copies = []
        for a, b in zip(src, dst):
            full = self.lens[a] // self.pt
            self.rows[b] = self.rows[a][:full]
            for p in self.rows[b]:
                self.refs[p] += 1
            if self.lens[a] % self.pt:
                copies.append((self.rows[a][full], free[0]))
                self.rows[b].append(free.pop(0))
                self.refs[self.rows[b][-1]] = 1
            self.lens[b] = self.lens[a]
        return copies

    def free(self, slots):
        for i, s in enumerate(slots):
            if not 0 <= s < len(self.lens):
                return (1, i)
        for s in set(slots):
            for p in self.rows[s]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = [], 0
        return None

    def compact(self):
        count = sum(r > 0 for r in self.refs)
        movers = [i for i, r in enumerate(self.refs) if r > 0 and i >= count]
        holes = [i for i, r in enumerate(self.refs) if r == 0 and i < count]
        to = dict(zip(movers, holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return list(to.items())

    def table(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]


def same(p, m):
    assert p.table.tolist() == m.table()
    assert p.lens.tolist() == m.lens
    assert p.refs.tolist() == m.refs


@pytest.mark.parametrize("n_slots,width,n_pages,pt,layers", [(6, 5, 17, 32, 1), (40, 9, 150, 64, 3), (1500, 3, 6000, 128, 1),
                                                             (1, 1, 1, 256, 2)])
def test_pages_against_model(hiplib, cuda, n_slots, width, n_pages, pt, layers):
    """A long run of random page operations: tables, lengths, counts, bytes and errors as the plain model has them."""
    import random
    from sx8_paged_kv import PagedKV4
    rng = random.Random(n_slots)
    p = PagedKV4(layers, 1, 64, n_pages, n_slots, width, pt, device=cuda)
    g = torch.Generator(device="cpu").manual_seed(1)
    fill = torch.randint(0, 256, (layers, n_pages, 16), generator=g, dtype=torch.uint8).to(cuda)
    p.pages.copy_(fill.repeat(1, 1, p.page_bytes // 16))
    m = Pool(n_slots, width, n_pages, pt)
    met = set()
    for it in range(60):
        kind = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        before = p.pages.clone()
        moved = []
        if kind == "reserve":
            top = rng.choice([1, pt, 2 * pt, width * pt])
            add = [rng.choice([0, 0, 1, rng.randrange(0, top + 1)]) for _ in range(n_slots)]
            if rng.random() < 0.1:
                add[rng.randrange(n_slots)] = -1
            add = [a if rng.random() < 0.05 else min(a, width * pt - l) for a, l in zip(add, m.lens)]
            p.reserve(ints(add, cuda))
            err = m.reserve(add)
        elif kind == "fork":
            empty = [s for s, l in enumerate(m.lens) if l == 0]
            n = min(len(empty), rng.randrange(0, n_slots + 1))
            dst = rng.sample(empty, n)
            src = [rng.randrange(n_slots) for _ in dst]
            if rng.random() < 0.7:
                full = [s for s in range(n_slots) if s not in dst]
                src = [rng.choice(full) for _ in dst] if full else []
                dst = dst[:len(src)]
            if dst and rng.random() < 0.1:
                src[-1] = rng.choice([-1, n_slots])
            p.fork(ints(src, cuda), ints(dst, cuda))
            err = m.fork(src, dst) if src else None
            if isinstance(err, list):
                moved, err = err, None
        elif kind == "free":
            slots = [rng.randrange(n_slots) for _ in range(rng.randrange(0, n_slots + 1))]
            if slots and rng.random() < 0.1:
                slots[rng.randrange(len(slots))] = n_slots
            p.free(ints(slots, cuda))
            err = m.free(slots)
        else:
            p.compact()
            moved, err = m.compact(), None
        same(p, m)
        assert p.status.tolist() == (list(err) if err else [0, 0]), (kind, err)
        if err:
            met.add(err[0])
            with pytest.raises(RuntimeError, match="paged cache"):
                p.check()
        p.check()
        want = before.clone()
        if moved:
            a, b = (torch.tensor(x, device=cuda) for x in zip(*moved))
            want[:, b] = before[:, a]
        assert torch.equal(p.pages, want)
    assert met or n_slots == 1


def test_fork_names_its_errors(hiplib, cuda):
    p, _, _ = make(cuda, [40, 0, 0, 10], 1, 64, 32, spare=0)
    state = (p.table.clone(), p.lens.clone(), p.refs.clone())
    for src, dst, code in (([0], [3], 4), ([0, 0], [1, 1], 4), ([0, 1], [1, 2], 4), ([0, 9], [1, 2], 1), ([-1], [1], 1),
                           ([0, 3], [1, 2], 2)):
        p.fork(ints(src, cuda), ints(dst, cuda))
        assert p.status.tolist()[0] == code, (src, dst)
        assert all(torch.equal(a, b) for a, b in zip(state, (p.table, p.lens, p.refs)))
        p.status.zero_()


def test_forked_slots_part(hiplib, cuda):
    """Two forks of one slot go on with different tokens; the source and each other stay as they were."""
    from sx8_paged_kv import PagedKV4
    p = PagedKV4(2, 2, 128, 12, 3, 4, 32, device=cuda)
    p.reserve(ints([70, 0, 0], cuda))
    k, v = rand((70, 2, 128), 1, F16, cuda), rand((70, 2, 128), 2, F16, cuda)
    for layer in range(2):
        p.append(layer, k + layer, v, ints([0, 70, 70, 70], cuda))
    p.fork(ints([0, 0], cuda), ints([1, 2], cuda))
    p.reserve(ints([0, 3, 40], cuda))
    nk, nv = rand((43, 2, 128), 3, F16, cuda), rand((43, 2, 128), 4, F16, cuda)
    for layer in range(2):
        p.append(layer, nk + layer, nv, ints([0, 0, 3, 43], cuda))
    p.check()
    assert p.lens.tolist() == [70, 73, 110]
    for layer in range(2):
        gk, _ = p.read(layer, 253, ints([0, 70, 143, 253], cuda))
        a, b = q4(k + layer).half(), q4(nk + layer).half()
        assert torch.equal(gk, torch.cat([a, a, b[:3], a, b[3:]]))
    p.free(ints([0], cuda))
    p.compact()
    gk, _ = p.read(1, 183, ints([0, 0, 73, 183], cuda))
    assert torch.equal(gk, torch.cat([q4(k + 1).half(), q4(nk + 1).half()[:3], q4(k + 1).half(), q4(nk + 1).half()[3:]]))
    q = rand((2, 4, 128), 5, F16, cuda)
    kk, vv = torch.cat([q4(k), q4(nk)[:3]]), torch.cat([q4(v), q4(nv)[:3]])
    close(p.attend(0, q, ints([0, 0, 1, 2], cuda))[:1], attention(q[:1].double(), kk, vv, 72), F16, 4.0)


def test_step_in_a_graph(hiplib, cuda):
    """A captured step (reserve, append, attend) replayed over page borders, with eager work between the replays, equals
    the same steps run eagerly; two captured graphs on two caches do not disturb each other."""
    from sx8_paged_kv import PagedKV4
    lens, steps = [30, 5, 63], 9

    def start():
        p, _, _ = make(cuda, lens, 2, 128, 32, layers=2, spare=6, width=6)
        return p

    x = [tuple(rand((3, h, 128), 100 * i + j, F16, cuda) for j, h in enumerate((4, 2, 2))) for i in range(steps)]
    add = ints([1, 1, 1], cuda)

    def step(p, q, k, v):
        p.reserve(add)
        outs = []
        for layer in range(2):
            p.append(layer, k, v)
            outs.append(p.attend(layer, q))
        return outs

    eager = start()
    want = [[o.clone() for o in step(eager, *x[i])] for i in range(steps)]
    graphs = []
    for _ in range(2):
        p = start()
        bufs = [t.clone() for t in x[0]]
        saved = [t.clone() for t in (p.table, p.lens, p.refs, p.pages)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(p, *bufs)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(p, *bufs)
        for t, s in zip((p.table, p.lens, p.refs, p.pages), saved):
            t.copy_(s)
        graphs.append((p, bufs, g, outs))
    for i in range(steps):
        for p, bufs, g, outs in graphs:
            for b, t in zip(bufs, x[i]):
                b.copy_(t)
            g.replay()
        torch.cuda.synchronize()
        for p, bufs, g, outs in graphs:
            for o, w in zip(outs, want[i]):
                assert torch.equal(o, w), i
        _ = rand((64, 64), i, F16, cuda).sum()
    for p, *_ in graphs:
        p.check()
        assert torch.equal(p.pages, eager.pages) and torch.equal(p.table, eager.table)


def test_pool_past_four_gib(hiplib, cuda):
    """Pages whose bytes lie past 2^32: written, read, attended, forked and moved."""
    from sx8_paged_kv import PagedKV4
    nk, hd, pt = 8, 128, 128
    n_pages = (1 << 32) // PagedKV4._page_bytes(nk, hd, pt) + 40
    p = PagedKV4(1, nk, hd, n_pages, 3, 4, pt, device=cuda)
    p.refs[:n_pages - 8] = 1                                        # all but the last pages are taken
    n = 300
    p.reserve(ints([n, 0, 0], cuda))
    assert p.table[0, 0] == n_pages - 8 and (n_pages - 8) * p.page_bytes > 1 << 32
    k, v = rand((n, nk, hd), 1, F16, cuda), rand((n, nk, hd), 2, F16, cuda)
    p.append(0, k, v, ints([0, n, n, n], cuda))
    p.fork(ints([0], cuda), ints([2], cuda))
    p.check()
    q = rand((2, nk, hd), 3, F16, cuda)
    want = attention(q[:1].double(), q4(k), q4(v), n - 1)
    cu = ints([0, 1, 1, 2], cuda)
    q[1] = q[0]
    got = p.attend(0, q, cu)
    close(got[:1], want, F16, 4.0)
    assert torch.equal(got[0], got[1])
    p.refs[:n_pages - 8] = 0
    p.compact()
    assert p.table.max() == 3 and torch.equal(p.attend(0, q, cu), got)
    rk, _ = p.read(0, 2 * n, ints([0, n, n, 2 * n], cuda))
    assert torch.equal(rk, torch.cat([q4(k).half()] * 2))


def test_varlen_rows_past_four_gib(hiplib, cuda):
    """Keys and values whose offsets pass 2^32 bytes (rows 2 MB apart)."""
    from sx8_paged_kv import attn_varlen
    T, ts = 2100, 1 << 20
    big = torch.zeros(T * ts, dtype=F16, device=cuda)
    k = torch.as_strided(big, (T, 1, 64), (ts, 64, 1))
    v = torch.as_strided(big, (T, 1, 64), (ts, 64, 1), 64)
    k.copy_(rand((T, 1, 64), 1, F16, cuda))
    v.copy_(rand((T, 1, 64), 2, F16, cuda))
    q = rand((5, 2, 64), 3, F16, cuda)
    got = attn_varlen(q, k, v, ints([0, 3, 5], cuda), ints([0, 50, T], cuda))
    close(got, want_varlen(q, k, v, [3, 2], [50, T - 50]), F16, 5.0, 2.0 ** -11)


def test_two_streams(hiplib, cuda):
    """Two caches worked on by two streams at once give what they give one after the other."""
    pools = [make(cuda, [900 + 200 * i, 64], 2, 128, 64, seed=i)[0] for i in range(2)]
    qs = [rand((2, 8, 128), 50 + i, F16, cuda) for i in range(2)]
    want = [p.attend(0, q) for p, q in zip(pools, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pools[i].attend(0, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


# ------------------------------------------------------------------------------ packed prompts
def want_varlen(q, k, v, nq, nkeys, causal=True, scale=None):
    out, a, b = [], 0, 0
    for n, l in zip(nq, nkeys):
        out.append(attention(q[a:a + n].double(), k[b:b + l].double(), v[b:b + l].double(), l - n, scale, causal))
        a, b = a + n, b + l
    return torch.cat(out)


@pytest.mark.parametrize("nh,nk,hd", [(8, 2, 128), (3, 3, 64), (6, 1, 256), (5, 1, 128)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_varlen_lengths(hiplib, cuda, nh, nk, hd, dt):
    """Lengths around the tiles' borders, empty sequences among them."""
    from sx8_paged_kv import attn_varlen
    ns = [1, 0, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 0, 300, 17]
    T = sum(ns)
    q, k, v = (rand((T, h, hd), i, dt, cuda) for i, h in enumerate((nh, nk, nk)))
    cu = cum(ns, cuda)
    got = attn_varlen(q, k, v, cu)
    top = v.abs().max().item()
    close(got, want_varlen(q, k, v, ns, ns), dt, top, torch.finfo(dt).eps / 2)
    full = attn_varlen(q, k, v, cu, causal=False, scale=0.2)
    close(full, want_varlen(q, k, v, ns, ns, False, 0.2), dt, top, torch.finfo(dt).eps / 2)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_varlen_more_keys_or_rows(hiplib, cuda, hd):
    """Keys of earlier tokens in front, sequences without keys, and more rows than keys (the first rows see none)."""
    from sx8_paged_kv import attn_varlen
    nq, nkeys = [5, 130, 1, 40, 7, 200, 0], [70, 400, 1000, 0, 3, 71, 9]
    q = rand((sum(nq) + 2, 4, hd), 1, F16, cuda)
    k, v = rand((sum(nkeys), 2, hd), 2, F16, cuda), rand((sum(nkeys), 2, hd), 3, F16, cuda)
    for causal in (True, False):
        out = torch.full_like(q, 5.0)
        got = attn_varlen(q, k, v, cum(nq, cuda), cum(nkeys, cuda), causal=causal, out=out)
        want = want_varlen(q, k, v, nq, nkeys, causal)
        if causal:
            a = sum(nq[:4])
            assert not got[a:a + 4].any() and not got[sum(nq[:3]):a].any()
        close(got[:sum(nq)], want, F16, v.abs().max().item(), torch.finfo(F16).eps / 2)
        assert (got[sum(nq):] == 5).all()


def test_varlen_long(hiplib, cuda):
    from sx8_paged_kv import attn_varlen
    for dt in (F16, BF16):
        q, k, v = (rand((2500, h, 128), i, dt, cuda) for i, h in enumerate((4, 2, 2)))
        k = k * 3
        got = attn_varlen(q, k, v, cum([2500], cuda))
        close(got, want_varlen(q, k, v, [2500], [2500]), dt, v.abs().max().item(), torch.finfo(dt).eps / 2)
        assert torch.equal(got, attn_varlen(q, k, v, cum([2500], cuda)))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_varlen_many_small_weights(hiplib, cuda, dt):
    """A key with nearly all of the weight and 100000 with 2^-22.7 of it each: each weight is within eps / 2 of itself."""
    from sx8_paged_kv import attn_varlen
    n, s = 100001, 15.76
    q = torch.zeros(1, 1024, 64, dtype=dt, device=cuda)
    k, v = torch.zeros(n, 1, 64, dtype=dt, device=cuda), torch.ones(n, 1, 64, dtype=dt, device=cuda)
    q[..., 0], k[0, 0, 0], v[0] = 8, 2, 0
    got = attn_varlen(q, k, v, cum([1], cuda), cum([n], cuda), scale=s / 16)
    w = (n - 1) * math.exp(-s)
    close(got, torch.full_like(got, w / (1 + w), dtype=torch.float64), dt, 1.0, torch.finfo(dt).eps / 2)


def test_outputs_on_inputs(hiplib, cuda):
    """out on the rows of q; outputs that are each other or K or V are refused."""
    from sx8_paged_kv import attn_varlen
    for nkeys in (300, 6000):                                           # (whole, in parts)
        q, k, v = rand((300, 4, 128), 1, F16, cuda), rand((nkeys, 4, 128), 2, F16, cuda), rand((nkeys, 4, 128), 3, F16, cuda)
        v[7] = math.nan
        cq, ck = cum([300], cuda), cum([nkeys], cuda)
        want = attn_varlen(q, k, v, cq, ck)
        for bad in (k, v):
            if nkeys == 300:
                with pytest.raises(RuntimeError, match="k or v"):
                    attn_varlen(q, k, v, cq, ck, out=bad)
        attn_varlen(q, k, v, cq, ck, out=q)
        assert torch.equal(q.view(torch.int16), want.view(torch.int16))
    p, _, _ = make(cuda, [900, 64], 2, 128, 64)
    q = rand((2, 8, 128), 1, F16, cuda)
    want = p.attend(0, q)
    assert torch.equal(p.attend(0, q, out=q), want)
    x = torch.empty(2, 2, 128, dtype=F16, device=cuda)
    with pytest.raises(RuntimeError, match="share memory"):
        p.read(0, 2, out=(x, x))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_varlen_few_rows_many_keys(hiplib, cuda, hd, dt):
    """Calls whose keys are cut into parts: sequences of very different lengths, rows without keys, empty parts, values that are
    no finite numbers; and the same without a workspace."""
    import _sx8lib as L
    from sx8_paged_kv import attn_varlen
    nq, nkeys = [3, 130, 1, 6, 2], [5000, 900, 0, 4, 2700]
    assert L.lib().sx8_attn_varlen_workspace_bytes(5, sum(nq), sum(nkeys), 4, hd) > 0
    q = rand((sum(nq) + 1, 4, hd), 1, dt, cuda)
    k, v = rand((sum(nkeys), 2, hd), 2, dt, cuda), rand((sum(nkeys), 2, hd), 3, dt, cuda)
    cq, ck = cum(nq, cuda), cum(nkeys, cuda)
    for causal in (True, False):
        got = attn_varlen(q, k, v, cq, ck, causal=causal, out=torch.full_like(q, 5.0))
        close(got[:-1], want_varlen(q, k, v, nq, nkeys, causal), dt, v.abs().max().item(), torch.finfo(dt).eps / 2)
        assert (got[-1] == 5).all()
        one = torch.full_like(q, 5.0)
        L.call("sx8_attn_varlen", q.data_ptr(), k.data_ptr(), v.data_ptr(), one.data_ptr(), cq.data_ptr(), ck.data_ptr(), 5,
               q.shape[0], k.shape[0], 4, 2, hd, 4 * hd, hd, 2 * hd, hd, 2 * hd, hd, 4 * hd, hd, hd ** -0.5, causal,
               int(dt is BF16), None, 0, L.stream(cuda))
        close(one[:-1], want_varlen(q, k, v, nq, nkeys, causal), dt, v.abs().max().item(), torch.finfo(dt).eps / 2)
    v[4998, 1, 5] = math.nan                                       # seen by rows 1 and 2 of the first sequence
    got = attn_varlen(q, k, v, cq, ck)
    nan = torch.isnan(got[:-1])
    assert nan[1:3, 2:, 5].all() and nan.sum() == 4
    vz = v.clone()
    vz[4998, 1, 5] = 0
    want = want_varlen(q, k, vz, nq, nkeys)
    close(torch.where(nan, 0, got[:-1]), torch.where(nan, 0.0, want), dt, vz.abs().max().item(), torch.finfo(dt).eps / 2)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_varlen_not_finite(hiplib, cuda, dt, bad):
    """A value that is no finite number reaches the rows that see it, and no other row or sequence."""
    from sx8_paged_kv import attn_varlen
    ns = [50, 90, 40]
    q, k, v = (rand((180, h, 128), i, dt, cuda) for i, h in enumerate((2, 1, 1)))
    v[75, 0, 9] = bad                                               # sequence 1, token 25
    got = attn_varlen(q, k, v, cum(ns, cuda))
    odd = ~torch.isfinite(got)
    assert odd[75:140, :, 9].all() and odd.sum() == 65 * 2
    vz = v.clone()
    vz[75, 0, 9] = 0
    want = want_varlen(q, k, vz, ns, ns)
    ok = torch.ones_like(odd)
    ok[75:140, :, 9] = False
    close(torch.where(ok, got, 0), torch.where(ok, want, 0.0), dt, v[torch.isfinite(v)].abs().max().item(),
          torch.finfo(dt).eps / 2)
    if math.isinf(bad):
        assert (got[75:140, :, 9] == bad).all()
    k[75, 0, 0] = math.nan
    got = attn_varlen(q, k, vz, cum(ns, cuda))
    assert torch.isnan(got[75:140]).all() and torch.isfinite(got[:75]).all() and torch.isfinite(got[140:]).all()


def test_varlen_strides(hiplib, cuda):
    """One packed qkv tensor, head-major keys, an output inside a wider tensor, rows off 16 bytes, one broadcast key."""
    from sx8_paged_kv import attn_varlen
    ns, hd = [70, 33], 64
    qkv = rand((103, 6, hd), 1, F16, cuda)
    q, k, v = qkv[:, :4], qkv[:, 4:5], qkv[:, 5:]
    wide = torch.full((103, 4, 2 * hd), 3.0, dtype=F16, device=cuda)
    cu = cum(ns, cuda)
    want = want_varlen(q, k, v, ns, ns)
    got = attn_varlen(q, k, v, cu, out=wide[..., :hd])
    close(got, want, F16, 4.0, 2.0 ** -11)
    assert (wide[..., hd:] == 3).all()
    major = v.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    odd = torch.zeros(103 * hd + 3, dtype=F16, device=cuda)[3:].view(103, 1, hd)
    odd.copy_(k)
    assert torch.equal(attn_varlen(q, odd, major, cu), got)
    one = v[:1].expand(103, 1, hd)
    close(attn_varlen(q, k, one, cu), want_varlen(q, k, one, ns, ns), F16, 4.0, 2.0 ** -11)


def test_varlen_odd_cu(hiplib, cuda):
    """cu that runs past the rows, backwards or below zero stays inside the memory."""
    from sx8_paged_kv import attn_varlen
    q, k, v = (rand((40, 2, 64), i, F16, cuda) for i in range(3))
    for cu in ([0, 1 << 30, 5], [-7, 10, 40], [30, 10, 0]):
        out = torch.zeros_like(q)
        assert torch.isfinite(attn_varlen(q, k, v, ints(cu, cuda), out=out)).all()


def test_varlen_in_a_graph_and_streams(hiplib, cuda):
    from sx8_paged_kv import attn_varlen
    ns = [200, 9, 100]
    q, k, v = (rand((309, h, 128), i, F16, cuda) for i, h in enumerate((4, 2, 2)))
    cu = cum(ns, cuda)
    out = torch.empty_like(q)
    want = attn_varlen(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(attn_varlen(q, k, v, cu, out=out), want)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        attn_varlen(q, k, v, cu, out=out)
    for lens in (ns, [100, 109, 100], [0, 1, 308]):
        cu.copy_(cum(lens, cuda))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attn_varlen(q, k, v, cu))


def test_general_path_gives_the_same(hiplib, cuda, monkeypatch):
    """Without the host module every call takes the wrappers' general path: the same results."""
    import _sx8lib
    from sx8_paged_kv import attn_varlen

    def run():
        p, k, v = make(cuda, [40, 0, 70], 2, 128, 32, spare=3, layers=2)
        q = rand((3, 4, 128), 5, F16, cuda)
        outs = [p.attend(1, q), p.attend(0, q, cum([1, 0, 2], cuda), scale=0.2), *p.read(0, 110, cum([40, 0, 70], cuda)),
                *p.read(1, 3, dtype=BF16), attn_varlen(q, k, v, cum([1, 0, 2], cuda), cum([40, 0, 70], cuda), causal=False),
                attn_varlen(k, k, v, cum([40, 0, 70], cuda))]
        p.fork(ints([0], cuda), ints([1], cuda))
        p.free(ints([2], cuda))
        p.compact()
        p.check()
        return outs + [p.table, p.lens, p.refs, p.pages[:, :4]]

    fast = run()
    assert isinstance(_sx8lib.py().varlen, type(len))               # the module is there
    monkeypatch.setattr(_sx8lib, "_py", _sx8lib._NoHostModule())
    for a, b in zip(fast, run()):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------ refusals of the wrappers
def test_wrappers_refuse(hiplib, cuda):
    from sx8_paged_kv import PagedKV4, attn_varlen
    p, k, v = make(cuda, [40], 1, 64, 32)
    q = rand((1, 2, 64), 1, F16, cuda)
    cu = cum([1], cuda)
    for call in (lambda: p.attend(1, q), lambda: p.attend(-1, q), lambda: p.attend(0, q.float()),
                 lambda: p.attend(0, q[..., :32]), lambda: p.attend(0, q, cu.long()), lambda: p.attend(0, q, cum([1, 1], cuda)),
                 lambda: p.attend(0, q.cpu()), lambda: p.attend(0, q, scale=0.0), lambda: p.attend(0, q, scale=math.nan),
                 lambda: p.attend(0, rand((2, 2, 64), 1, F16, cuda)), lambda: p.attend(0, q, out=q.float()),
                 lambda: p.attend(0, q, out=q[:, :1].expand(1, 2, 64)),
                 lambda: p.attend(0, q.expand(1, 2, 64), out=torch.as_strided(q, (1, 2, 64), (128, 8, 1))),
                 lambda: p.append(0, k, v), lambda: p.append(0, k, v[:3], cum([40], cuda)),
                 lambda: p.append(0, k, v.bfloat16(), cum([40], cuda)), lambda: p.read(0, 2),
                 lambda: p.read(0, 1, dtype=torch.float32), lambda: p.reserve(ints([1, 1], cuda)),
                 lambda: p.reserve([1]), lambda: p.fork(ints([0], cuda), ints([1, 2], cuda)),
                 lambda: p.fork(ints([0, 0], cuda), ints([1, 2], cuda)), lambda: p.free(cu.float()),
                 lambda: PagedKV4(1, 1, 96, 4, 1, 4, device=cuda), lambda: PagedKV4(1, 1, 64, 4, 1, 4, 48, device=cuda),
                 lambda: PagedKV4(1, 1, 64, 4, 5000, 4, device=cuda),
                 lambda: PagedKV4(1, 1, 64, 4, 1, 1 << 17, device=cuda),
                 lambda: PagedKV4.from_tensors(p.pages[..., 16:], p.table, p.lens, p.refs, n_kv=1, head_dim=64, page_tokens=32),
                 lambda: PagedKV4.from_tensors(p.pages, p.table.long(), p.lens, p.refs, n_kv=1, head_dim=64, page_tokens=32),
                 lambda: attn_varlen(q, k, v, cu, cum([1, 2], cuda)), lambda: attn_varlen(q, k, v[:2], cu),
                 lambda: attn_varlen(q, k.bfloat16(), v, cu), lambda: attn_varlen(q.float(), k.float(), v.float(), cu),
                 lambda: attn_varlen(rand((1, 3, 64), 1, F16, cuda), rand((1, 2, 64), 1, F16, cuda),
                                     rand((1, 2, 64), 1, F16, cuda), cu),
                 lambda: attn_varlen(q, k, v, cu, scale=-1.0), lambda: attn_varlen(q[0], k, v, cu),
                 lambda: attn_varlen(q, k, v, cu[:1])):
        with pytest.raises(RuntimeError):
            call()
    assert p.attend(0, q[:0], ints([0, 0], cuda)).shape == (0, 2, 64)
    assert attn_varlen(q[:0], k[:0], v[:0], ints([0, 0], cuda)).shape == (0, 2, 64)
