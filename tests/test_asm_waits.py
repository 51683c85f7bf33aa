"""Wait states around inline assembly, in the compiler's output: the compiler keeps them between instructions that it writes
itself and does not look into asm blocks.  For gfx950: two states between a VALU result and an MFMA that reads it, one between
a transcendental's result and a VALU instruction that reads it, five between a scalar register that the VALU wrote and
a memory access that reads it, one between m0 and the load to LDS that uses it, 19 at most between an MFMA's result and an
instruction that reads or overwrites it."""
import os
import re
import subprocess

import pytest

import _sx8lib as L

TRANS = ("v_exp_", "v_rcp_", "v_log_", "v_rsq_", "v_sqrt_", "v_sin_", "v_cos_")


def regs(op):
    m = re.match(r"^-?\|?([vsa])(?:(\d+)|\[(\d+):(\d+)\])", op)
    if not m:
        return {"m0"} if op == "m0" else set()
    a, b = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {m[1] + str(i) for i in range(int(a), int(b) + 1)}


def short_waits(text):
    """(kernel, what, writer, reader) of every access that comes too early, along the listing, labels included."""
    found, kernel, in_asm, clock, past = [], "", False, 0, []
    for line in text.splitlines():
        if "#ASMSTART" in line or "#ASMEND" in line:
            in_asm = "#ASMSTART" in line
            continue
        m = re.match(r"^(_Z\w+):", line)
        if m:
            kernel, past = m[1], []
        code = "" if line.lstrip().startswith(";") else line.split(";")[0].strip()
        if not code or code.startswith(".") or code.endswith(":"):
            continue
        name, _, rest = code.partition(" ")
        ops = [o.strip() for o in re.split(r",(?![^\[]*\])", rest)]
        if name == "s_nop":
            clock += int(ops[0], 0) + 1
            continue
        to_lds = name.startswith("buffer_load") and code.endswith(" lds")
        stores = to_lds or name.startswith(("buffer_store", "global_store", "flat_store", "ds_write", "s_cbranch", "s_wait"))
        reads = set().union(*(regs(w) for o in ops[0 if stores else 1:] for w in o.split())) if ops else set()
        if to_lds:
            reads |= {"m0"}
        writes = set() if stores or not ops else regs(ops[0])
        for wname, wrote, w_asm, at in past[-24:]:
            gap, hit = clock - at - 1, wrote & reads
            if in_asm and wname.startswith("v_mfma") and wrote & (reads | writes) and gap < 19:
                found.append((kernel, "result", wname, code))
            if not hit or not (in_asm or w_asm):
                continue
            valu = wname.startswith("v_") and not wname.startswith("v_mfma")
            if valu and name.startswith("v_mfma") and gap < 2:
                found.append((kernel, "mfma", wname, code))
            if wname.startswith(TRANS) and name.startswith("v_") and gap < 1:
                found.append((kernel, "trans", wname, code))
            if valu and name.startswith(("buffer_", "global_")) and any(r[0] == "s" for r in hit) and gap < 5:
                found.append((kernel, "sgpr", wname, code))
            if "m0" in hit and gap < 1:
                found.append((kernel, "m0", wname, code))
        past = [(n, w - writes, a, at) for n, w, a, at in past[-24:]] + [(name, writes, in_asm, clock)]
        clock += 1
    return found


def test_the_check_sees_short_waits():
    asm = """_Zk:
    v_exp_f32_e32 v1, v2
    ;;#ASMSTART
    v_fma_mixlo_f16 v3, v1, v4, 0
    v_fma_mixhi_f16 v3, v5, v4, 0
    ;;#ASMEND
    v_and_b32_e32 v9, 1, v9
    v_mfma_f32_16x16x32_f16 v[20:23], v[12:15], v[0:3], v[20:23]
    v_readfirstlane_b32 s6, v0
    ;;#ASMSTART
    s_mov_b32 m0, s9
    buffer_load_dwordx4 v7, s[4:7], 0 offen lds
    ;;#ASMEND
"""
    assert [f[1] for f in short_waits(asm)] == ["trans", "mfma", "sgpr", "m0"]
    late = "_Zk:\n v_mfma_f32_16x16x32_f16 v[0:3], v[4:7], v[8:11], 0\n s_nop 3\n ;;#ASMSTART\n v_mov_b32_e32 v2, v20\n ;;#ASMEND\n"
    assert [f[1] for f in short_waits(late)] == ["result"] and short_waits(late.replace("v2,", "v12,")) == []
    mended = asm.replace("    v_fma_mixlo", "    s_nop 0\n    v_fma_mixlo").replace("    v_and_b32", "    s_nop 0\n    v_and_b32")
    mended = mended.replace("    s_mov_b32 m0", "    s_nop 4\n    s_mov_b32 m0").replace("    buffer_load", "    s_nop 0\n    buffer_load")
    assert short_waits(mended) == []


@pytest.mark.parametrize("source", ["sx8_kv4.hip", "sx8_attn_varlen.hip"])
def test_waits_around_asm(source, tmp_path):
    out = tmp_path / "kernel.s"
    flags = [f for f in L.HIP_FLAGS if f != "-shared"] + L.SOURCE_FLAGS.get(source, [])
    subprocess.run([L.HIPCC, *flags, "-S", "--cuda-device-only", "-I" + L.INCLUDE_DIR, "-o", str(out),
                    os.path.join(L.CSRC_DIR, source)], check=True, capture_output=True, timeout=600)
    found = short_waits(out.read_text())
    assert "#ASMSTART" in out.read_text()
    assert not found, found[:4]


def test_asm_names_m0():
    """An asm statement that writes m0 names it among what it overwrites."""
    seen = 0
    for name in sorted(os.listdir(L.CSRC_DIR)):
        text = open(os.path.join(L.CSRC_DIR, name)).read()
        for m in re.finditer(r'asm volatile\((?:[^;"]|"[^"]*")*\);|asm\((?:[^;"]|"[^"]*")*\);', text):
            if re.search(r"s_mov_b32 m0|s_add_u32 m0", m[0]):
                seen += 1
                assert re.search(r':[^:]*"m0"[^:]*\);$', m[0]), (name, m[0])
    assert seen
