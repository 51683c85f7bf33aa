"""attend_tree gives the same bits every time: slots cut over all work-groups, whatever ran before and on which stream."""
import pytest
import torch

from test_draft import ancestors, flat, trees, words_of
from test_paged_kv import BF16, F16, cum, make, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("hd,heads", [(128, 16), (64, 4), (256, 8)])
def test_attend_tree_repeats(hiplib, cuda, dt, hd, heads):
    lens, new = [9000, 300, 4100], [31, 2, 17]
    p, _, _ = make(cuda, lens, 2, hd, 64)
    q = rand((sum(new), heads, hd), 5, dt, cuda)
    mask, cu = words_of(flat([ancestors(t) for t in trees(new, 1)]), 1).to(cuda), cum(new, cuda)
    want = p.attend_tree(0, q, mask, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = torch.randn(2048, 2048, device=cuda, dtype=F16)
    for i in range(8):
        if i % 2:
            x = (x @ x).clamp(-1, 1)
        with torch.cuda.stream(side if i % 3 == 2 else torch.cuda.current_stream()):
            got = p.attend_tree(0, q, mask, cu)
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
