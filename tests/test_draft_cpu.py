"""Drafted tokens without a GPU: how the tree attention's work is cut, which keys a mask lets a row attend, and what the
entry points refuse (on the host, before any launch)."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
REPO = os.path.dirname(HERE)
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
I32, I64, P = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def emul(hiplib):                                                      # (torch's HIP runtime first)
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    out = os.path.join(HERE, "emul", "build", "libsx8_draft_emul.so")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run([HIPCC, "--cuda-host-only", "-O2", "-std=c++17", "-fPIC", "-shared", "-I",
                    os.path.join(REPO, "sx8-quantization_amd", "csrc"), "-o", out,
                    os.path.join(HERE, "emul", "sx8_draft_emul.hip")], check=True, capture_output=True)
    L = ctypes.CDLL(out)
    L.sx8e_tree_pieces.restype = I64
    L.sx8e_tree_pieces.argtypes = [I32, I32, I32, I32, I32, I32, P, P, I32, P, I64]
    L.sx8e_tree_bits.restype = ctypes.c_uint32
    L.sx8e_tree_bits.argtypes = [P, I32, I32, I32]
    return L


def test_tree_bits(emul):
    """Bit i of what a row attends of 32 keys: keys before the new ones, and new ones whose bit is set."""
    rng = random.Random(1)
    for _ in range(3000):
        words = rng.randint(1, 4)
        m = [rng.getrandbits(64) for _ in range(words)]
        first, block = rng.choice([-70, -1, 0, 1, 31, 32, 33, 63, 100, rng.randrange(400)]), rng.randrange(12) * 32
        got = emul.sx8e_tree_bits((ctypes.c_uint64 * words)(*m), words, first, block)
        want = 0
        for i in range(32):
            j = block + i - first
            want |= (1 if j < 0 else j < 64 * words and m[j // 64] >> j % 64 & 1) << i
        assert got == want, (words, first, block)


def test_tree_work_covers_every_block_once(emul):
    """Every block of every unit belongs to one work-group; a work-group has at most one cut piece that begins its share and
    one that ends it; the parts of a cut unit lie in consecutive work-groups, whose number the combine is told."""
    rng = random.Random(7)
    for _ in range(60):
        S, nk, G, cols = rng.choice([1, 2, 9, 70]), rng.choice([1, 3, 8]), rng.choice([1, 4, 5, 32]), rng.choice([16, 32, 64])
        cap, groups = rng.choice([64, 4096, 1 << 17]), rng.choice([256, 512])
        lens = [rng.choice([0, 1, 31, 32, 33, rng.randrange(cap + 1), cap + 9, -3]) for _ in range(S)]
        new = [rng.choice([0, 1, 3, 40, 64]) for _ in range(S)]
        cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        rows = int(cu[-1])
        la, most = np.array(lens, np.int32), 1 << 20
        out = np.zeros((most, 9), np.int64)
        got = emul.sx8e_tree_pieces(S, nk, G, cap, rows, cols, la.ctypes.data, cu.ctypes.data, groups, out.ctypes.data, most)
        assert got <= most
        pieces, seen, cut = out[:got], {}, {}
        for grp, s, unit, b0, b1, nb, place, parts, whole in pieces.tolist():
            assert 0 <= grp < groups and place in (2 * grp, 2 * grp + 1)
            key = (s, unit)
            assert seen.get(key, 0) == b0 < b1 <= nb, "in order, none twice"
            seen[key] = b1
            if not whole:
                cut.setdefault(key, []).append((grp, place, parts))
        places = [pl for c in cut.values() for _, pl, _ in c]
        assert len(places) == len(set(places))
        for c in cut.values():
            assert c[0][2] == len(c) and [g for g, _, _ in c] == list(range(c[0][0], c[0][0] + len(c)))
            assert all(pl == 2 * g for g, pl, _ in c[1:])
        for s in range(S):
            nb = max(1, (min(max(lens[s], 0), cap) + 31) // 32)
            for u in range(nk * -(-new[s] * G // cols)):
                assert seen.pop((s, u)) == nb
        assert not seen


# ------------------------------------------------------------------------------ refusals
def _err(L):
    return L.sx8_last_error().decode()


def _call(L, name, args, **change):
    """The entry point with these arguments (in order), some of them changed; nothing is launched."""
    a = dict(args)
    a.update(change)
    return getattr(L, name)(*a.values())


X, ODD = P(4096), P(4098)
ROPE = dict(pages=X, table=X, lens=X, cu=X, n_slots=2, max_pages=4, n_pages=8, q=X, k=P(8192), v=X, out=P(1 << 20), rows=5, q_ts=256, q_hs=64,
            k_ts=64, k_hs=64, v_ts=64, v_hs=64, o_ts=256, o_hs=64, nh=4, nk=1, hd=64, page_tokens=32, cos_t=X, sin_t=X, table_rows=9,
            rot=64, interleaved=0, depth=X, q_norm=X, k_norm=X, eps=1e-6, in_dtype=0, dtype=0, stream=None)
TREE = dict(pages=X, table=X, lens=X, cu=X, n_slots=2, max_pages=4, n_pages=8, q=X, out=P(1 << 20), rows=5, q_ts=256, q_hs=64, o_ts=256,
            o_hs=64, mask=X, words=1, nh=4, nk=1, hd=64, page_tokens=32, scale=0.1, dtype=0, workspace=X, workspace_bytes=1 << 40,
            stream=None)
KEEP = dict(pages=X, n_layers=1, table=X, lens=X, refs=X, cu=X, path=X, counts=X, rows=5, n_slots=2, max_pages=4, n_pages=8, nk=1, hd=64,
            page_tokens=32, status=X, workspace=X, workspace_bytes=1 << 30, stream=None)
DTREE = dict(parents=X, cu=X, n_slots=2, rows=5, words=1, mask=X, depth=X, stream=None)
VERIFY = dict(logits=X, logits_stride=100, dtype=2, tokens=X, parents=X, cu=X, n_slots=2, rows=5, V=100, u=X, temperature=X, t=0.0,
              probs=X, probs_stride=100, probs_dtype=2, path=X, counts=X, next=X, workspace=X, workspace_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change,word", [
    ({"pages": None}, "null"), ({"q": None}, "null"), ({"k": None}, "null"), ({"out": None}, "null"), ({"hd": 96}, "shape"),
    ({"page_tokens": 48}, "shape"), ({"rows": -1}, "rows"), ({"cu": None}, "rows"), ({"nh": 3, "nk": 2}, "multiple"), ({"nh": 257}, "multiple"),
    ({"q_ts": 252}, "multiples of 8"), ({"k": ODD}, "aligned"), ({"o_ts": 64}, "overlap"), ({"rot": 8}, "rot"), ({"rot": 72}, "rot"),
    ({"rot": 24}, "rot"), ({"cos_t": None}, "tables"), ({"sin_t": ODD}, "tables"), ({"table_rows": 0}, "tables"), ({"in_dtype": 1}, "dtype"),
    ({"dtype": 2}, "dtype"), ({"in_dtype": 3}, "dtype"), ({"depth": ODD}, "aligned"), ({"q_norm": ODD}, "aligned"), ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"out": X}, "out may not be q"), ({"n_slots": 5000}, "sizes")])
def test_append_rope_refuses(hiplib, change, word):
    assert _call(hiplib, "sx8_kv4_append_rope", ROPE, **change) == 1 and word in _err(hiplib)


@pytest.mark.parametrize("change,word", [
    ({"mask": None}, "mask"), ({"mask": P(4100)}, "mask"), ({"words": 0}, "words"), ({"words": 5}, "words"), ({"scale": 0.0}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"workspace": None}, "workspace"), ({"workspace_bytes": 100}, "workspace"), ({"out": X}, "out may not be q"),
    ({"workspace": P(4096 + 16)}, "workspace"), ({"nh": 300}, "multiple"), ({"o_hs": 32}, "overlap"), ({"dtype": 2}, "dtype"), ({"q": ODD}, "aligned"),
    ({"lens": None}, "null"), ({"n_pages": 0}, "sizes")])
def test_attend_tree_refuses(hiplib, change, word):
    assert _call(hiplib, "sx8_kv4_attend_tree", TREE, **change) == 1 and word in _err(hiplib)
    assert hiplib.sx8_kv4_attend_tree_workspace_bytes(96) == -1


@pytest.mark.parametrize("change,word", [
    ({"pages": None}, "pages"), ({"path": None}, "null"), ({"counts": None}, "null"), ({"status": None}, "null"), ({"hd": 32}, "shape"),
    ({"page_tokens": 16}, "page_tokens"), ({"n_layers": 0}, "n_layers"), ({"cu": None}, "rows"), ({"rows": -1}, "rows"), ({"path": ODD}, "aligned"),
    ({"workspace_bytes": 8}, "workspace"), ({"max_pages": 0}, "sizes")])
def test_keep_refuses_on_the_host(hiplib, change, word):
    assert _call(hiplib, "sx8_kv4_keep", KEEP, **change) == 1 and word in _err(hiplib)
    assert hiplib.sx8_kv4_keep_workspace_bytes(0, 5) == hiplib.sx8_kv4_keep_workspace_bytes(5, -1) == -1


@pytest.mark.parametrize("change,word", [
    ({"parents": None}, "null"), ({"cu": None}, "null"), ({"mask": P(4100)}, "aligned"), ({"words": 0}, "words"), ({"words": 5}, "words"),
    ({"n_slots": 0}, "sizes"), ({"rows": -1}, "sizes")])
def test_draft_tree_refuses(hiplib, change, word):
    assert _call(hiplib, "sx8_draft_tree", DTREE, **change) == 1 and word in _err(hiplib)


@pytest.mark.parametrize("change,word", [
    ({"logits": None}, "null"), ({"next": None}, "null"), ({"path": None}, "null"), ({"V": 0}, "sizes"), ({"V": 1 << 29}, "sizes"), ({"V": (1 << 27) + 1}, "sizes"), ({"rows": (1 << 22) + 1}, "sizes"),
    ({"rows": -1}, "sizes"), ({"dtype": 3}, "dtypes"), ({"probs_dtype": -1}, "dtypes"), ({"logits": ODD}, "aligned"), ({"tokens": P(4100)}, "aligned"),
    ({"logits_stride": 99}, "strides"), ({"probs_stride": 99}, "strides"), ({"u": None}, "random"), ({"u": None, "temperature": None, "t": 0.5}, "random"),
    ({"workspace_bytes": 8}, "workspace"), ({"workspace": None}, "workspace")])
def test_verify_refuses(hiplib, change, word):
    assert _call(hiplib, "sx8_draft_verify", VERIFY, **change) == 1 and word in _err(hiplib)


def test_wrappers_refuse_without_a_gpu(hiplib):
    import torch
    import sx8_draft
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        sx8_draft.draft_tree(i32, i32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        sx8_draft.verify_draft(torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64), i32, i32)


def test_waits_around_asm_of_the_tree_attention(tmp_path):
    """As test_asm_waits.py checks the other attention kernels."""
    import _sx8lib as L
    from test_asm_waits import short_waits
    out = tmp_path / "kernel.s"
    flags = [f for f in L.HIP_FLAGS if f != "-shared"]
    subprocess.run([L.HIPCC, *flags, "-S", "--cuda-device-only", "-I" + L.INCLUDE_DIR, "-o", str(out),
                    os.path.join(L.CSRC_DIR, "sx8_kv4_tree.hip")], check=True, capture_output=True, timeout=600)
    found = short_waits(out.read_text())
    assert "#ASMSTART" in out.read_text()
    assert not found, found[:4]
