"""Wait states that gfx950 leaves to the program, looked for in the built library's code (no GPU).

The compiler keeps them among its own instructions and does not look inside assembly statements: a scalar register that
a vector instruction wrote (v_readfirstlane, v_readlane, a compare) may be read by a vector-memory instruction five wait
states later at the earliest; m0 that a scalar instruction wrote, by a load into LDS one wait state later.  Every
instruction between is one, s_nop n is n + 1."""

import os
import re
import struct
import subprocess

import pytest

from model_amd import build

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 code objects of a library's offload bundles."""
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + n].decode()
            p += 24 + n
            if "gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + len(MAGIC))


SCALARS = re.compile(r"\b(?:s(\d+)\b|s\[(\d+):(\d+)\]|(vcc)\b|(m0)\b)")
VECTOR_MEMORY = ("global_", "buffer_", "flat_", "scratch_")


def scalars(text):
    out = set()
    for one, lo, hi, vcc, m0 in SCALARS.findall(text):
        if one:
            out.add(int(one))
        elif lo:
            out.update(range(int(lo), int(hi) + 1))
        else:
            out.add(vcc or m0)
    return out


def hazards(lines):
    """The instructions of a listing that read a scalar register too early."""
    by_vector, m0, now = {}, None, 0  # register: the wait states before the instruction behind its write
    for line in lines:
        text = line.split("//")[0].split(";")[0].strip()
        if not text or text.endswith(":") or text.startswith("."):
            continue
        op, _, rest = text.partition(" ")
        parts = [x.strip() for x in rest.split(",")]
        if op.startswith(VECTOR_MEMORY):
            early = [r for r in scalars(rest) if now - by_vector.get(r, -9) < 5]
            if early:
                yield text, early
            if "_lds" in op and m0 is not None and now - m0 < 1:
                yield text, ["m0"]
        now += int(parts[0], 0) + 1 if op == "s_nop" else 1
        if op.startswith("v_"):
            # the results come first: of compares, carries and divisions a second one may be scalar
            wrote = scalars(parts[0]) if parts else set()
            if len(parts) > 1 and re.match(r"v_(add_co|sub_co|subrev_co|addc_co|subb_co|subbrev_co|div_scale|mad_u64|mad_i64)", op):
                wrote |= scalars(parts[1])
            if op.startswith("v_cmp") and (op.endswith("_e32") or not wrote):
                wrote.add("vcc")
            for r in wrote:
                by_vector[r] = now
        elif op.startswith("s_") and parts:
            for r in scalars(parts[0]):
                by_vector.pop(r, None)
                if r == "m0":
                    m0 = now


@pytest.mark.parametrize("listing,count", [
    (["v_readfirstlane_b32 s4, v1", "global_load_lds_dwordx4 v2, s[4:5]"], 1),
    (["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_nop 0", "global_load_lds_dwordx4 v2, s[4:5]"], 1),
    (["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_nop 2", "global_load_lds_dwordx4 v2, s[4:5]"], 1),
    (["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_nop 3", "global_load_lds_dwordx4 v2, s[4:5]"], 0),
    (["v_readfirstlane_b32 s5, v1", "s_mov_b32 m0, s9", "s_mov_b64 s[8:9], s[4:5]",
      "global_load_lds_dwordx4 v2, s[8:9]"], 0),
    (["s_mov_b32 m0, s9", "global_load_lds_dwordx4 v2, s[8:9]"], 1),
    (["v_cmp_gt_u32_e64 s[6:7], v1, v2", "s_nop 1", "global_load_dword v3, v2, s[6:7]"], 1),
    (["v_readlane_b32 s3, v1, 2", "buffer_load_dword v1, v2, s[8:11], s3 offen"], 1),
])
def test_the_search_itself(listing, count):
    assert len(list(hazards(listing))) == count


@pytest.mark.timeout(300)
def test_built_code_keeps_the_wait_states(tmp_path):
    if not os.path.exists(build.LIB):
        build.build()
    objdump = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.hipcc()))), "llvm", "bin", "llvm-objdump")
    if not os.path.exists(objdump):
        objdump = "/opt/rocm/llvm/bin/llvm-objdump"
    with open(build.LIB, "rb") as f:
        objects = list(code_objects(f.read()))
    assert len(objects) >= 10  # a source file each
    loads, found = 0, []
    for i, code in enumerate(objects):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        r = subprocess.run([objdump, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], capture_output=True,
                           text=True, check=True)
        path.unlink()
        lines = r.stdout.splitlines()
        loads += sum("global_load_lds_dwordx4" in x for x in lines)
        found += list(hazards(lines))
    assert loads > 0
    assert not found, f"{len(found)} reads too early, of {loads} loads into LDS: {found[:3]}"
