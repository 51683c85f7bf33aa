"""How many bits the attention of drafted trees keeps over the 4-bit pages, against 64 bits: the cases of test_paged_precision.py
that averages over many tokens hide, for units of one tile of query rows (up to 48 rows of a KV head) and of two."""
import math

import pytest
import torch

from test_paged_kv import BF16, F16, attention, ints, q4, rand
from test_paged_precision import pool, rows

pytestmark = pytest.mark.gpu


def chain(n, cuda):
    """Masks of a chain of n rows (up to 63)."""
    return torch.tensor([[(2 << i) - 1] for i in range(n)], dtype=torch.int64, device=cuda)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [4, 16])
def test_sums_of_levels_are_not_short(hiplib, cuda, hd, new):
    """The sum of the levels and the sum of the minima nearly cancel over many tokens, so a sum of levels that always falls
    short shows in the mean error: the bound of the same test of `attend`."""
    n, nk, rep = 4096, 4, 4
    k, v = rand((n, nk, hd), 1, F16, cuda), rows((n, nk, hd), 2, cuda)
    q = rand((new, nk * rep, hd), 3, F16, cuda)
    got, kk, vv = pool(k, v, cuda).attend_tree(0, q, chain(new, cuda), ints([0, new], cuda)).double(), q4(k), q4(v)
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
@pytest.mark.parametrize("heads", [8, 64])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_small_query_values(hiplib, cuda, hd, heads, dt):
    """Query values about 2^-19 of their row's largest decide the scores (the keys' level is zero where that one is): they
    enter exactly, and the bound is that of the same test of `attend`."""
    n = 200
    k = torch.randint(0, 16, (n, 1, hd), generator=torch.Generator().manual_seed(1)).half().to(cuda)
    k[..., 0::64], k[..., 1::64] = 0, 15
    v = rows((n, 1, hd), 2, cuda)
    q = rand((1, heads, hd), 3, torch.float32, cuda).clamp(-4, 4) * 2.0 ** -13
    q = torch.where(q.abs() < 2.0 ** -16, 0.0, q)                   # (bf16's eight bits at 2^-16 are fp16's at 2^-24)
    q[..., 0] = 64
    q = q.to(dt)
    scale = 2.0 ** 12 / hd ** 0.5
    got = pool(k, v, cuda).attend_tree(0, q, chain(1, cuda), scale=scale).double()
    want = attention(q.double(), q4(k), q4(v), n - 1, scale)
    err = ((got - want).abs() - torch.finfo(dt).eps / 2 * want.abs()).max().item()
    print("error past half a step", err, flush=True)
    assert err <= 2.0 ** -13


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads", [32, 64])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_every_token_of_a_block(hiplib, cuda, hd, heads, dt):
    """Queries that give 0.4 of their weight to one token of a block each and the rest to a token whose values are zero: the
    weight times the scale needs both of its fp16 numbers, for every token of the block, in values whose level and
    minimum nearly cancel.  A weight is within 2^-18 of itself (scores of 58 powers of two); as two fp16 numbers it is within
    2^-22, and weight times scale within 2^-22 of that again: a product is within 2^-18 + 2^-21 levels (2 / 15), all of it
    below 2^-18 of the value and 2^-20 * 3, as for `attend`."""
    n = 64
    k, v = torch.zeros(n, 1, hd, dtype=F16, device=cuda), rows((n, 1, hd), 1, cuda)
    k[range(32), 0, range(32)] = 15
    k[40, 0, 40] = 15
    v[40] = 0
    q = torch.zeros(1, heads, hd, device=cuda)
    q[0, range(heads), [i % 32 for i in range(heads)]] = 39.6 / 15
    q[..., 40] = 40 / 15
    q = q.to(dt)
    got, want = pool(k, v, cuda).attend_tree(0, q, chain(1, cuda), scale=1.0).double(), attention(q.double(), q4(k), q4(v), n - 1, 1.0)
    err = (got - want).abs() - (torch.finfo(dt).eps / 2 + 2.0 ** -18) * want.abs() - 3 * 2.0 ** -20
    print("largest error over the bound", err.max().item(), flush=True)
    assert err.max() <= 0


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("heads", [4, 64])
@pytest.mark.parametrize("sizes", [(4.0, 2.0 ** -10), (2.0 ** 12, 0.25), (2.0 ** -10, 2.0 ** -10), (64.0, 2.0)])
@pytest.mark.parametrize("mixed", [False, True])
def test_scales_of_groups(hiplib, cuda, dt, heads, sizes, mixed):
    """A head with a group of large and one of small scales (mixed: the first group's scale changes from token to
    token), a key with 0.6 of the weight and 65000 that share the rest: each group keeps its own precision.  The
    largest weight counts at least 2^10.  A token's weight is cut to two fp16 numbers, in all sums alike (2^-24 at most), its
    product with the scale (below 2; a larger one divided by 2^k into 1/16 .. 2) is within 2^-25 twice (the upper halves' product and
    what the lower ones add): 2 + 1 + 1 times 2^-25 at most, independent of each other a root mean square of
    (4 + 1 + 1)^(1/2) = 2.5 times that of one.  Levels' root square sum times that over the sum of the weights, a third of
    the square on average, six times that.  Weights are within 2^-17 of themselves."""
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
    q = torch.zeros(1, heads, hd)
    q[..., 0] = 10.7 / 15
    q[..., 2:64] = torch.randn(1, heads, 62, generator=g) * 0.01
    q = q.to(dt).to(cuda)
    got = pool(k, v, cuda).attend_tree(0, q, chain(1, cuda), scale=1.0).double()
    want = attention(q.double(), k.double(), v.double(), n - 1, 1.0)
    w = torch.matmul(q[0].double(), k[:, 0].double().T.contiguous())
    total = 2.0 ** 10 * torch.exp(w - w.amax(-1, keepdim=True)).sum(-1).min().item()
    for i in range(2):
        a = slice(64 * i, 64 * i + 64)
        unit = max(1.0, s[..., a].max().item() * 8)                 # 2^k at most for scales in 2^(k - 4) .. 2^(k + 1)
        unit = unit if s[..., a].max() >= 2 else 1.0
        more = 6 * 2.5 * 2.0 ** -25 * unit * 15 * n ** 0.5 / 3 ** 0.5 / total + 2.0 ** -17 * v[..., a].max().item()
        err = ((got - want).abs() - torch.finfo(dt).eps / 2 * want.abs())[..., a].max().item()
        print("group", i, "error past half a step", err, "of", more, "mean value", want[..., a].abs().mean().item(), flush=True)
        assert err <= more


@pytest.mark.parametrize("token", [3, 31, 33, 38])
def test_not_finite_with_a_small_weight(hiplib, cuda, token):
    """A value that is no number reaches a row that attends it with a weight of e^-120, in a block that the row sees
    whole (0 .. 31) and in one that ends inside; a row that does not attend it stays clear of it."""
    k, v = torch.zeros(40, 1, 64, dtype=F16, device=cuda), rows((40, 1, 64), 1, cuda)
    k[39, 0, 0] = 15
    v[token, 0, 5] = math.nan
    q = torch.zeros(8, 2, 64, dtype=F16, device=cuda)
    q[..., 0] = 8
    mask = torch.full((8, 1), 255, dtype=torch.int64, device=cuda)  # rows 32 .. 39 are the new ones
    if token >= 32:
        mask[::2] -= 1 << token - 32
    got = pool(k, v, cuda).attend_tree(0, q, mask, ints([0, 8], cuda), scale=1.0)
    assert torch.isnan(got[1::2]).all() and torch.isnan(got[::2]).all() == (token < 32) and torch.isnan(got[::2]).any() == (token < 32)
    v[token, 0, 5] = 0
    assert torch.isfinite(pool(k, v, cuda).attend_tree(0, q, mask, ints([0, 8], cuda), scale=1.0)).all()
