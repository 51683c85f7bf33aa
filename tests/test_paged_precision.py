"""How many bits the attention over the 4-bit pages and the attention of packed prompts keep, against 64 bits: cases that
averages over many tokens hide."""
import math

import pytest
import torch

from test_paged_kv import BF16, F16, attention, cum, ints, q4, rand

pytestmark = pytest.mark.gpu


def rows(shape, seed, cuda):
    """Uniform in (-1, 1), fp16."""
    return (torch.rand(*shape, generator=torch.Generator().manual_seed(seed)) * 2 - 1).half().to(cuda)


def pool(k, v, cuda, slots=1):
    """A cache whose `slots` slots hold these rows each (n, nk, hd)."""
    from sx8_paged_kv import PagedKV4
    n, nk, hd = k.shape
    width = -(-n // 32)
    p = PagedKV4(1, nk, hd, slots * width, slots, width, 32, device=cuda)
    p.reserve(ints([n] * slots, cuda))
    p.append(0, torch.cat([k] * slots), torch.cat([v] * slots), cum([n] * slots, cuda))
    p.check()
    return p


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attend_sums_of_levels_are_not_short(hiplib, cuda, hd):
    """The sum of the levels and the sum of the minima nearly cancel over many tokens, so a sum of levels that always falls
    short shows in the mean error.  A level enters as 2^-20 times itself, aligned as if at 2^-14, and what lies about 25 places
    below the largest product of a block is cut: a product loses half of 2^-19 levels of the block's largest weight, an
    output 2^-20 scales times 32 of those largest weights' sum.  The outputs' own rounding is of either sign: half a step at
    most, a third of its square on average, so four times the root of that over their number."""
    n, nk, rep, new = 4096, 4, 4, 16
    k, v = rand((n, nk, hd), 1, F16, cuda), rows((n, nk, hd), 2, cuda)
    q = rand((new, nk * rep, hd), 3, F16, cuda)
    got, kk, vv = pool(k, v, cuda).attend(0, q, ints([0, new], cuda)).double(), q4(k), q4(v)
    want = attention(q.double(), kk, vv, n - new)
    w = torch.matmul(q.double().permute(1, 0, 2).contiguous(), kk.repeat_interleave(rep, 1).permute(1, 2, 0).contiguous())
    w = (w / hd ** 0.5).masked_fill(torch.arange(n, device=cuda) > n - new + torch.arange(new, device=cuda)[:, None], -math.inf)
    top = torch.softmax(w, -1).unflatten(-1, (-1, 32)).amax(-1).sum(-1).mean().item()
    half = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - 11)
    noise = half.square().mean().sqrt().item() / (3 * want.numel()) ** 0.5
    mean = (got - want).mean().item()
    bound = 2.0 ** -20 * (2 / 15) * 32 * top + 4 * noise
    print("mean error", mean, "bound", bound, flush=True)
    assert abs(mean) <= bound


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_small_query_values(hiplib, cuda, hd, dt):
    """Query values about 2^-19 of their row's largest decide the scores (the keys' level is zero where that one is): they
    enter exactly.  A score is then good to the products' alignment, hd times 2^-19 levels of the largest of these values
    (2^-11), times the scale 2^12 / sqrt(hd): 2^-14 for hd of 256, and an average of values below 1 to twice that."""
    n = 200
    k = torch.randint(0, 16, (n, 1, hd), generator=torch.Generator().manual_seed(1)).half().to(cuda)
    k[..., 0::64], k[..., 1::64] = 0, 15
    v = rows((n, 1, hd), 2, cuda)
    assert torch.equal(q4(k), k.double())
    q = rand((1, 8, hd), 3, torch.float32, cuda).clamp(-4, 4) * 2.0 ** -13
    q = torch.where(q.abs() < 2.0 ** -16, 0.0, q)                   # (bf16's eight bits at 2^-16 are fp16's at 2^-24)
    q[..., 0] = 64
    q = q.to(dt)
    scale = 2.0 ** 12 / hd ** 0.5
    p = pool(k, v, cuda)
    got, want = p.attend(0, q, scale=scale).double(), attention(q.double(), q4(k), q4(v), n - 1, scale)
    err = ((got - want).abs() - torch.finfo(dt).eps / 2 * want.abs()).max().item()
    print("error past half a step", err, flush=True)
    assert err <= 2.0 ** -13


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attend_every_token_of_a_block(hiplib, cuda, hd, dt):
    """32 queries that give 0.4 of their weight to one token of a block each and the rest to a token whose values are zero: the
    weight times the scale needs both of its fp16 numbers (22 bits), for every token of the block, in values whose level and
    minimum nearly cancel.  A weight is within 2^-18 of itself (scores of 58 powers of two), weight times scale within
    2^-22, a product within 2^-18 levels (2 / 15): all of it below 2^-18 of the value and 2^-20 * 3."""
    n = 64
    k, v = torch.zeros(n, 1, hd, dtype=F16, device=cuda), rows((n, 1, hd), 1, cuda)
    k[range(32), 0, range(32)] = 15
    k[40, 0, 40] = 15
    v[40] = 0
    assert torch.equal(q4(k), k.double())
    q = torch.zeros(1, 32, hd, device=cuda)
    q[0, range(32), range(32)] = 39.6 / 15
    q[..., 40] = 40 / 15
    q = q.to(dt)
    got, want = pool(k, v, cuda).attend(0, q, scale=1.0).double(), attention(q.double(), q4(k), q4(v), n - 1, 1.0)
    err = (got - want).abs() - (torch.finfo(dt).eps / 2 + 2.0 ** -18) * want.abs() - 3 * 2.0 ** -20
    print("largest error over the bound", err.max().item(), flush=True)
    assert err.max() <= 0


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("sizes", [(4.0, 2.0 ** -10), (2.0 ** 12, 0.25), (2.0 ** -10, 2.0 ** -10), (64.0, 2.0)])
@pytest.mark.parametrize("mixed", [False, True])
def test_attend_scales_of_groups(hiplib, cuda, dt, sizes, mixed):
    """A head with a group of large and one of small scales (mixed: the first group's scale changes from token to
    token), a key with 0.6 of the weight and 65000 that share the rest: each group keeps its own precision.  The
    largest weight counts at least 2^10, so a token's weight times scale (below 2; a larger one divided by 2^k into 1/16 .. 2) is
    within 2^-25, of either sign: levels' root square sum times that over the sum of the weights, a third of the square on
    average, six times that.  Weights are within 2^-17 of themselves."""
    n, hd = 65000, 128
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randint(0, 16, (n, 1, hd), generator=g).double() for _ in range(2))
    k[:, :, 64:] = 0
    k[..., 0], k[..., 1], k[0] = 0, 15, 0
    k[0, 0, 0] = 15
    v[..., 0::64], v[..., 1::64] = 0, 15
    s = torch.tensor(sizes).double().repeat_interleave(64).expand(n, 1, hd).clone()
    if mixed:
        s[1::3, :, :64] *= 2.0 ** -6 if sizes[0] > 1 else 2.0 ** 6
    k, v = k.half().to(cuda), (v * s).half().to(cuda)
    assert torch.equal(q4(k), k.double()) and torch.equal(q4(v), v.double())
    q = torch.zeros(1, 4, hd)
    q[..., 0] = 10.7 / 15
    q[..., 2:64] = torch.randn(1, 4, 62, generator=g) * 0.01
    q = q.to(dt).to(cuda)
    got, want = pool(k, v, cuda).attend(0, q, scale=1.0).double(), attention(q.double(), k.double(), v.double(), n - 1, 1.0)
    w = torch.matmul(q[0].double(), k[:, 0].double().T.contiguous())
    total = 2.0 ** 10 * torch.exp(w - w.amax(-1, keepdim=True)).sum(-1).min().item()
    for i in range(2):
        a = slice(64 * i, 64 * i + 64)
        unit = max(1.0, s[..., a].max().item() * 8)                 # 2^k at most for scales in 2^(k - 4) .. 2^(k + 1)
        unit = unit if s[..., a].max() >= 2 else 1.0
        more = 6 * 2.0 ** -25 * unit * 15 * n ** 0.5 / 3 ** 0.5 / total + 2.0 ** -17 * v[..., a].max().item()
        err = ((got - want).abs() - torch.finfo(dt).eps / 2 * want.abs())[..., a].max().item()
        print("group", i, "error past half a step", err, "of", more, "mean value", want[..., a].abs().mean().item(), flush=True)
        assert err <= more


@pytest.mark.parametrize("token", [3, 31, 33, 38])
def test_attend_not_finite_with_a_small_weight(hiplib, cuda, token):
    """A value that is no number reaches a row that attends it with a weight of e^-120, in a block that the row sees
    whole (0 .. 31) and in one that ends inside."""
    k, v = torch.zeros(40, 1, 64, dtype=F16, device=cuda), rows((40, 1, 64), 1, cuda)
    k[39, 0, 0] = 15
    v[token, 0, 5] = math.nan
    q = torch.zeros(1, 2, 64, dtype=F16, device=cuda)
    q[..., 0] = 8
    p = pool(k, v, cuda)
    assert torch.isnan(p.attend(0, q, scale=1.0)).all()
    v[token, 0, 5] = 0
    assert torch.isfinite(pool(k, v, cuda).attend(0, q, scale=1.0)).all()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nkeys,at", [(50, 3), (50, 48), (300, 3), (9000, 3), (9000, 8500)])
def test_varlen_not_finite_with_a_small_weight(hiplib, cuda, dt, bad, nkeys, at):
    """A value that is no finite number reaches the rows that attend it with a weight of e^-120 before and behind the key that
    has the rest, in tiles that the rows see whole or in part and in keys cut into parts."""
    from sx8_paged_kv import attn_varlen
    q, k, v = torch.zeros(4, 2, 64, dtype=dt, device=cuda), torch.zeros(nkeys, 1, 64, dtype=dt, device=cuda), rand((nkeys, 1, 64), 1, dt, cuda)
    q[..., 0], k[20, 0, 0], v[at, 0, 7] = 8, 15, bad
    got = attn_varlen(q, k, v, cum([4], cuda), cum([nkeys], cuda), scale=1.0)
    sees = torch.arange(nkeys - 4, nkeys, device=cuda) >= at
    want = torch.full_like(got[..., 7], bad)
    same = torch.isnan(got[..., 7]) if math.isnan(bad) else got[..., 7] == want
    assert same[sees].all() and torch.isfinite(got[~sees]).all()
    got[..., 7] = 0
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dt", [F16, BF16])
def test_append_levels_exactly(hiplib, cuda, dt):
    """Values on the border between two levels and next to it by any amount (bf16: far below what binary64 holds beside the
    minimum) get the level of the definition, decided here in rational numbers."""
    from fractions import Fraction
    tiny = [2.0 ** -e for e in ((20, 40, 60, 100, 126) if dt is BF16 else (12, 14, 20, 24))]
    groups = []
    for lo in (-1.5, -0.5, -7.5, -14.5, -2.5):                       # steps of 1: zero is the border of two levels
        groups.append([lo, lo + 15, 0.0, -0.0] + tiny + [-t for t in tiny])
        groups.append([4 * x for x in groups[-1][:2]] + groups[-1][2:])
    x = torch.zeros(len(groups), 1, 64, dtype=torch.float64)
    for i, g in enumerate(groups):
        x[i, 0, :len(g)] = torch.tensor(g, dtype=torch.float64)
    x = x.to(dt)
    want = torch.zeros(len(groups), 1, 64, dtype=torch.float64)
    for i, row in enumerate(x[:, 0].double().tolist()):
        lo, hi = min(row), max(row)
        s = ((torch.tensor(hi) - torch.tensor(lo)) * torch.tensor(1 / 15)).half().double().item()
        for d, value in enumerate(row):
            t = (Fraction(value) - Fraction(lo)) / Fraction(s)
            want[i, 0, d] = lo + s * min(max(round(t), 0), 15)
    k, _ = pool(x.to(cuda), x.to(cuda), cuda).read(0, len(groups), cum([len(groups)], cuda), dtype=dt)
    _, v = pool(x.to(cuda), x.to(cuda), cuda).read(0, len(groups), cum([len(groups)], cuda), dtype=dt)
    assert torch.equal(k.cpu(), want.to(dt)) and torch.equal(v, k)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("nq,nkeys", [([700], [3000]), ([3, 90], [5000, 2500])])
def test_varlen_near_equal_weights(hiplib, cuda, hd, dt, nq, nkeys):
    """Long rows of nearly equal weights, whose outputs are far smaller than the values: a weight is rounded to the type, within
    eps / 2 of itself, so an output is within eps / 2 of sum p |v| and its own half step, beside 2^-15 of that sum for scores
    and sums in 32 bits; and the roundings are independent, each with a third of its largest square: the root mean square."""
    from sx8_paged_kv import attn_varlen
    q, k, v = (rand((sum(n), h, hd), i, dt, cuda) for i, (n, h) in enumerate(((nq, 4), (nkeys, 2), (nkeys, 2))))
    q = q * 0.1
    got = attn_varlen(q, k, v, cum(nq, cuda), cum(nkeys, cuda)).double()
    half, a, b = torch.finfo(dt).eps / 2, 0, 0
    for n, keys in zip(nq, nkeys):
        qq, kk, vv = q[a:a + n].double(), k[b:b + keys].double(), v[b:b + keys].double()
        want, size = attention(qq, kk, vv, keys - n), attention(qq, kk, vv.abs(), keys - n)
        w = torch.matmul(qq.permute(1, 0, 2).contiguous(), kk.repeat_interleave(2, 1).permute(1, 2, 0).contiguous()) / hd ** 0.5
        w = w.masked_fill(torch.arange(keys, device=cuda) > keys - n + torch.arange(n, device=cuda)[:, None], -math.inf)
        p = torch.softmax(w, -1)
        square = torch.matmul(p.square(), vv.square().repeat_interleave(2, 1).permute(1, 0, 2).contiguous()).permute(1, 0, 2)
        err = got[a:a + n] - want
        over = (err.abs() - half * want.abs() * (1 + half) - (half + 2.0 ** -15) * size - torch.finfo(dt).tiny).max().item()
        rms = err.square().mean().sqrt().item()
        most = half * ((want.square() + square).mean().item() / 3) ** 0.5 * (1 + 4 / (2 * err.numel()) ** 0.5) + 2.0 ** -17 * size.mean().item()
        print("over", over, "rms", rms, "of", most, flush=True)
        assert over <= 0 and rms <= most
        a, b = a + n, b + keys
