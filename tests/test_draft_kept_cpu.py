"""Refusals of the entry points that say which new rows a cache holds (on the host, before any launch)."""
import pytest

from test_draft_cpu import KEEP, ODD, ROPE, VERIFY, X, _call, _err


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


RESERVE = dict(table=X, lens=X, refs=X, add=X, n_slots=2, max_pages=4, n_pages=8, page_tokens=32, status=X, marks=X, workspace=X,
               workspace_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("name,args,change,word", [
    ("sx8_kv4_reserve_marked", RESERVE, {"marks": ODD}, "aligned"), ("sx8_kv4_reserve_marked", RESERVE, {"add": None}, "null"),
    ("sx8_kv4_reserve_marked", RESERVE, {"workspace_bytes": 8}, "workspace"),
    ("sx8_kv4_append_rope_marked", with_after(ROPE, "depth", marks=X), {"marks": ODD}, "aligned"),
    ("sx8_kv4_append_rope_marked", with_after(ROPE, "depth", marks=X), {"rot": 8}, "rot"),
    ("sx8_kv4_append_rope_marked", with_after(ROPE, "depth", marks=X), {"out": X}, "out may not be q"),
    ("sx8_kv4_append_rope_marked", with_after(ROPE, "depth", marks=None), {"eps": -1.0}, "eps"),
    ("sx8_kv4_keep_marked", with_after(KEEP, "status", marks=X), {"marks": ODD}, "aligned"),
    ("sx8_kv4_keep_marked", with_after(KEEP, "status", marks=X), {"path": None}, "null"),
    ("sx8_kv4_keep_marked", with_after(KEEP, "status", marks=None), {"workspace_bytes": 8}, "workspace")])
def test_marked_forms_refuse(hiplib, name, args, change, word):
    assert _call(hiplib, name, args, **change) == 1 and word in _err(hiplib)
