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
