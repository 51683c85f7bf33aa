"""Refusals of the entry points that say which new rows a cache holds (on the host, before any launch)."""
import pytest

from test_draft_cpu import ODD, VERIFY, X, _call, _err


def with_after(args, name, **more):
    """The arguments with more of them behind `name`."""
    out = {}
    for k, v in args.items():
        out[k] = v
        if k == name:
            out.update(more)
    return out


WITHIN = with_after(VERIFY, "parents", depth=X)


@pytest.mark.parametrize("change,word", [
    ({"depth": ODD}, "aligned"), ({"logits": None}, "null"), ({"V": 0}, "sizes"), ({"dtype": 3}, "dtypes"), ({"u": None}, "random"),
    ({"workspace_bytes": 8}, "workspace"), ({"depth": None, "logits_stride": 99}, "strides")])
def test_verify_within_refuses(hiplib, change, word):
    assert _call(hiplib, "sx8_draft_verify_within", WITHIN, **change) == 1 and word in _err(hiplib)
