"""What the wrappers over the paged cache and the packed prompts make of tensors that are not what their memory holds."""
import pytest
import torch

from test_paged_kv import F16, cum, ints, make, rand

pytestmark = pytest.mark.gpu


def negated(x):
    """x, held as a view that negates on reading."""
    y = torch._neg_view(-x)
    assert y.is_neg() and torch.equal(y, x)
    return y


def test_views_that_negate(hiplib, cuda):
    """They are read as the values they stand for; as outputs, tables or lengths they are refused."""
    from sx8_paged_kv import PagedKV4, attn_varlen
    p, k, v = make(cuda, [40, 9], 2, 64, 32)
    q = rand((2, 4, 64), 5, F16, cuda)
    cu, cuk = cum([1, 1], cuda), cum([40, 9], cuda)
    assert torch.equal(p.attend(0, negated(q)), p.attend(0, q))
    want = attn_varlen(q, k, v, cu, cuk)
    for args in ((negated(q), k, v), (q, negated(k), v), (q, k, negated(v))):
        assert torch.equal(attn_varlen(*args, cu, cuk), want)
    before = p.pages.clone()
    p.append(0, negated(k), negated(v), cuk)
    assert torch.equal(p.pages, before)
    n = torch._neg_view
    kk = torch.empty(2, 2, 64, dtype=F16, device=cuda)
    for call in (lambda: p.attend(0, q, out=n(torch.empty_like(q))), lambda: attn_varlen(q, k, v, cu, cuk, out=n(torch.empty_like(q))),
                 lambda: p.read(0, 2, out=(n(kk), kk.clone())), lambda: p.attend(0, q, n(-cu)), lambda: attn_varlen(q, k, v, n(-cu), cuk),
                 lambda: p.reserve(n(ints([0, 0], cuda))), lambda: p.free(n(ints([0], cuda))),
                 lambda: PagedKV4.from_tensors(p.pages, n(p.table), p.lens, p.refs, n_kv=2, head_dim=64, page_tokens=32),
                 lambda: PagedKV4.from_tensors(p.pages, p.table, n(p.lens), p.refs, n_kv=2, head_dim=64, page_tokens=32)):
        with pytest.raises(RuntimeError):
            call()
    p.check()
    assert p.lens.tolist() == [40, 9]
