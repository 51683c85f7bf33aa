"""The paged cache without a GPU: where the format puts its bits, how the attention's work is cut, and what the entry
points refuse (on the host, before any launch)."""
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
    out = os.path.join(HERE, "emul", "build", "libsx8_kv4_emul.so")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.run([HIPCC, "--cuda-host-only", "-O2", "-std=c++17", "-fPIC", "-shared", "-I",
                    os.path.join(REPO, "sx8-quantization_amd", "csrc"), "-o", out,
                    os.path.join(HERE, "emul", "sx8_kv4_emul.hip")], check=True, capture_output=True)
    L = ctypes.CDLL(out)
    L.sx8e_kv4_pieces.restype = L.sx8e_kv4_slot_places.restype = I64
    L.sx8e_kv4_touched.restype = L.sx8e_kv4_touched_most.restype = I64
    L.sx8e_kv4_pieces.argtypes = [I32, I32, I32, I32, I32, P, P, I32, P, I64]
    L.sx8e_kv4_slot_places.argtypes = [I32, I32, I32, I32, I32, P, P, I32]
    L.sx8e_kv4_touched.argtypes = [I32, I32, P]
    L.sx8e_kv4_touched_most.argtypes = [I64, I64, I32]
    return L


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_format_places(emul, hd):
    """Every level has four bits of its own and every parameter two bytes; they fill the block; and they lie as the
    header of include/sx8_paged.h words it."""
    ng, nb = hd // 64, emul.sx8e_kv4_block_bytes(hd)
    bits, used = np.zeros(nb * 8, int), np.zeros(nb, int)
    w = (I32 * 8)()
    for t in range(32):
        for d in range(hd):
            emul.sx8e_kv4_where(hd, t, d, w)
            e = d % 8
            lane, j, wi = (d % 32) // 8 * 16 + t % 16, d // 32, min(hd // 32, 4)
            assert w[0] == t // 16 * 8 * hd + (j // wi * 64 + lane) * wi * 4 + j % wi * 4
            assert w[1] == 4 * (e // 2) + 16 * (e % 2)
            h, e = t % 16 // 4, t // 16 * 4 + t % 4
            assert w[2] == 16 * hd + (d // 16 // 4 * 64 + h * 16 + d % 16) * 16 + d // 16 % 4 * 4
            assert w[3] == 4 * (e // 2) + 16 * (e % 2) and t == 16 * (e // 4) + 4 * h + e % 4
            for at, shift in ((w[0], w[1]), (w[2], w[3])):
                assert at % 4 == 0 and at + 4 <= 32 * hd
                bits[at * 8 + shift:at * 8 + shift + 4] += 1
            if d % 64 == 0:
                g = d // 64
                slot = 2 * (g * 32 + h * 8 + e)
                assert list(w)[4:] == [32 * hd + slot, 33 * hd + 2 * (t * ng + g), 34 * hd + slot, 35 * hd + slot]
                for at in list(w)[4:]:
                    used[at:at + 2] += 1
    assert (bits[:32 * hd * 8] == 1).all() and (used[32 * hd:] == 1).all() and not used[:32 * hd].any()


def _lists(rng):
    S, nk, G = rng.choice([1, 2, 7, 40]), rng.choice([1, 3, 8]), rng.choice([1, 4, 5, 32])
    cap = rng.choice([64, 4096, 1 << 17])
    lens = [rng.choice([0, 1, 31, 32, 33, rng.randrange(cap + 1), cap + 9, -3]) for _ in range(S)]
    if rng.random() < 0.4:
        return S, nk, G, cap, S, lens, None
    new = [rng.choice([0, 1, 3, 40]) for _ in range(S)]
    cu = np.concatenate([[0], np.cumsum(new)])
    return S, nk, G, cap, int(cu[-1]) + rng.choice([0, 2]), lens, cu


def test_work_split_covers_every_block_once(emul):
    """Every block of every unit belongs to one piece; a wave has at most one piece that starts its share and one
    that ends it, so the partial results' places are distinct; the parts of a cut unit lie in consecutive waves, whose
    number is what the combine is told."""
    rng = random.Random(5)
    for it in range(60):
        S, nk, G, cap, rows, lens, cu = _lists(rng)
        log2 = rng.choice([0, 2, 11])
        waves = 1 << log2
        la = np.array(lens, np.int32)
        ca = None if cu is None else np.array(cu, np.int32)
        cp = None if ca is None else ca.ctypes.data
        args = (S, nk, G, cap, rows, la.ctypes.data, cp)
        n = emul.sx8e_kv4_pieces(*args, log2, None, 0)
        out = np.zeros((max(n, 1), 8), np.int64)
        assert emul.sx8e_kv4_pieces(*args, log2, out.ctypes.data, n) == n
        out = out[:n]
        seen, places, total = {}, set(), 0
        parts = {}
        for wave, s, unit, b0, e, nb, place, told in out:
            assert b0 == seen.get((s, unit), (0, None))[0] and b0 < e <= nb
            if b0 > 0:                                              # goes on: the next wave, as its first piece
                assert wave == seen[s, unit][1] + 1 and place % 2 == 0
                parts[s, unit][1] += 1
            else:
                parts[s, unit] = [told, 1]
            seen[s, unit] = (e, wave, nb)
            if not (b0 == 0 and e == nb):
                assert place not in places and 0 <= place < 2 * waves
                places.add(place)
            total += e - b0
        assert all(e == nb for e, _, nb in seen.values())
        sums = [emul.sx8e_kv4_slot_places(*args, s) for s in range(S)]
        assert all(a == b for a, b in parts.values())
        units = len(seen)
        assert total + 3 * units == sum(sums)
        total = sum(sums)
        share = max(1, -(-total // waves))
        assert all(out[:, 0] * share < total)
        for s in range(S):                                          # units as rows and heads say
            new = 1 if cu is None else int(cu[s + 1] - cu[s])
            units = {u for (t, u) in seen if t == s}
            assert units == set(range(nk * -(-new * G // 16)))


def test_touched_blocks(emul):
    """The blocks of a slot's new tokens, and the grid's bound on those of all slots."""
    rng = random.Random(6)
    first = I32()
    for _ in range(300):
        S = rng.choice([1, 3, 20])
        lens = [rng.randrange(0, 200) for _ in range(S)]
        new = [rng.choice([0, 1, 2, 33, 64, 250]) for _ in range(S)]
        total = 0
        for ln, n in zip(lens, new):
            got = emul.sx8e_kv4_touched(ln, n, ctypes.byref(first))
            want = sorted({p // 32 for p in range(ln - n, ln)})
            assert got == len(want) and (not want or first.value == want[0])
            total += got
        assert total <= emul.sx8e_kv4_touched_most(S, sum(new), 1)
    assert emul.sx8e_kv4_touched_most(9, 9, 0) == 9


# ------------------------------------------------------------------------------ refusals
def test_paged_entry_points_refuse(hiplib):
    L = hiplib
    p, odd, null = P(4096), P(4104), P(None)
    err = lambda: L.sx8_last_error().decode()  # noqa: E731
    assert L.sx8_kv4_page_bytes(8, 128, 64) == 8 * 2 * 4608 and L.sx8_kv4_page_bytes(1, 256, 32) == 9216
    for bad in ((0, 128, 64), (257, 128, 64), (8, 96, 64), (8, 128, 48), (8, 128, 512)):
        assert L.sx8_kv4_page_bytes(*bad) == -1
    assert L.sx8_kv4_attend_workspace_bytes(96) == -1 and L.sx8_kv4_attend_workspace_bytes(128) > 0
    assert L.sx8_kv4_pages_workspace_bytes(0, 4) == -1 and L.sx8_kv4_pages_workspace_bytes(4, 0) == -1
    assert L.sx8_kv4_pages_workspace_bytes(4097, 4) == -1
    ws = L.sx8_kv4_attend_workspace_bytes(64)

    def attend(pages=p, table=p, lens=p, cu=null, slots=4, width=8, n_pages=32, q=p, out=p, rows=4, st=(128, 64, 128, 64),
               nh=2, nk=1, hd=64, pt=32, scale=0.1, dt=0, w=p, wb=ws):
        return L.sx8_kv4_attend(pages, table, lens, cu, slots, width, n_pages, q, out, rows, *st, nh, nk, hd, pt, scale, dt,
                                w, wb, null)

    inf, nan = float("inf"), float("nan")
    for kw in (dict(pages=null), dict(table=null), dict(lens=null), dict(q=null), dict(out=null), dict(w=null),
               dict(pages=odd), dict(q=odd), dict(out=odd), dict(w=P(4096 + 128)), dict(wb=ws - 1), dict(slots=0),
               dict(slots=4097, rows=4097), dict(width=0), dict(width=1 << 18), dict(n_pages=0), dict(n_pages=1 << 31),
               dict(rows=3), dict(rows=-1, cu=p), dict(rows=1 << 31, cu=p), dict(st=(4, 64, 128, 64)),
               dict(st=(128, -64, 128, 64)), dict(st=(128, 64, 64, 64)), dict(st=(128, 64, 0, 64)), dict(nh=3, nk=2), dict(nh=0), dict(nk=0), dict(nh=257), dict(hd=96), dict(pt=16),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=inf), dict(scale=nan), dict(dt=2), dict(cu=P(4098))):
        assert attend(**kw) == 1, kw
        assert "sx8_kv4_attend" in err()
    assert attend(rows=0, cu=p, q=null, out=null) == 0              # nothing to do, nothing launched

    def rows_call(fn, k=p, v=p, rows=4, st=(64, 64, 64, 64), dt=0, cu=null):
        return fn(p, p, p, cu, 4, 8, 32, k, v, rows, *st, 1, 64, 32, dt, null)

    for fn in (L.sx8_kv4_append, L.sx8_kv4_read):
        for kw in (dict(k=null), dict(v=null), dict(k=odd), dict(v=odd), dict(rows=5), dict(st=(60, 64, 64, 64)), dict(dt=3)):
            assert rows_call(fn, **kw) == 1, kw
        assert rows_call(fn, rows=0, cu=p) == 0
    assert rows_call(L.sx8_kv4_read, st=(0, 64, 64, 64)) == 1 and "overlap" in err()

    nb = L.sx8_kv4_pages_workspace_bytes(4, 32)

    def reserve(table=p, lens=p, refs=p, add=p, slots=4, width=8, pages=32, pt=32, status=p, w=p, wb=nb):
        return L.sx8_kv4_reserve(table, lens, refs, add, slots, width, pages, pt, status, w, wb, null)

    for kw in (dict(table=null), dict(lens=null), dict(refs=null), dict(add=null), dict(status=null), dict(w=null),
               dict(w=odd), dict(wb=nb - 1), dict(slots=0), dict(width=0), dict(pages=0), dict(pt=48), dict(table=P(4098))):
        assert reserve(**kw) == 1, kw

    def fork(pages=p, layers=2, pb=4608, src=p, dst=p, n=2, w=p, wb=nb, pt=32):
        return L.sx8_kv4_fork(pages, layers, pb, p, p, p, src, dst, n, 4, 8, 32, pt, p, w, wb, null)

    for kw in (dict(pages=null), dict(pages=odd), dict(layers=0), dict(pb=100), dict(pb=0), dict(src=null), dict(dst=null),
               dict(n=-1), dict(n=5), dict(w=null), dict(wb=8), dict(pt=33)):
        assert fork(**kw) == 1, kw
    assert fork(pb=1 << 30, layers=4096) == 3
    assert fork(n=0, src=null, dst=null) == 0
    assert L.sx8_kv4_free(p, p, p, null, 1, 4, 8, 32, p, null) == 1
    assert L.sx8_kv4_free(p, p, p, p, 4097, 4, 8, 32, p, null) == 1
    assert L.sx8_kv4_free(p, p, p, null, 0, 4, 8, 32, p, null) == 0
    assert L.sx8_kv4_compact(null, 1, 4608, p, p, 4, 8, 32, p, nb, null) == 1
    assert L.sx8_kv4_compact(p, 1, 4608, p, p, 4, 8, 32, p, 0, null) == 1


def test_varlen_entry_point_refuses(hiplib):
    L = hiplib
    p, odd, null = P(4096), P(4104), P(None)

    def call(q=p, k=p, v=p, out=p, cq=p, ck=p, n=2, tq=8, tk=8, nh=2, nk=1, hd=64, st=(128, 64, 64, 64, 64, 64, 128, 64),
             scale=0.1, causal=1, dt=0, w=null, wb=0):
        return L.sx8_attn_varlen(q, k, v, out, cq, ck, n, tq, tk, nh, nk, hd, *st, scale, causal, dt, w, wb, null)

    for kw in (dict(q=null), dict(k=null), dict(v=null), dict(out=null), dict(cq=null), dict(ck=null), dict(q=odd),
               dict(k=odd), dict(v=odd), dict(out=odd), dict(cq=P(4098)), dict(n=0), dict(n=4097), dict(tq=-1),
               dict(tk=1 << 31), dict(nh=3, nk=2), dict(nk=0), dict(hd=32), dict(hd=96), dict(scale=0.0),
               dict(scale=float("nan")), dict(dt=2), dict(st=(128, 64, 60, 64, 64, 64, 128, 64)),
               dict(st=(128, 64, 0, 64, 64, 64, 128, 64)), dict(st=(128, 64, 64, 64, 1 << 24, 64, 128, 64)),
               dict(st=(-128, 64, 64, 64, 64, 64, 128, 64)), dict(st=(128, 64, 64, 64, 64, 64, 64, 64))):
        assert call(**kw) == 1, kw
        assert "sx8_attn_varlen" in L.sx8_last_error().decode()
    assert call(tq=(1 << 31) - 300, nh=4096, n=1, st=(128, 64, 64, 64, 64, 64, 4096 * 64, 64)) == 3
    assert call(tq=0, q=null, out=null) == 0
    # few rows and many keys: keys in parts, and a workspace that is given has to hold them
    need = L.sx8_attn_varlen_workspace_bytes(2, 8, 9000, 2, 64)
    assert need > 0 and L.sx8_attn_varlen_workspace_bytes(2, 8, 100, 2, 64) == 0
    assert L.sx8_attn_varlen_workspace_bytes(1, 1 << 20, 1 << 20, 32, 128) == 0
    assert L.sx8_attn_varlen_workspace_bytes(0, 8, 8, 2, 64) == -1
    assert call(tk=9000, w=p, wb=need - 1) == 1 and "workspace" in L.sx8_last_error().decode()
    assert call(tk=9000, w=P(4096 + 128), wb=need) == 1
