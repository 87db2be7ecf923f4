"""Loads into LDS take their LDS address from M0, and a load directly behind an
instruction that writes M0 may still use the old one: one wait state belongs
between them.  The compiler keeps it for its own builtins; for loads written as
inline assembly it sees no hazard, so the machine code is checked."""

import os
import re
import shutil
import subprocess

import pytest

from flashlite_amd import build

OBJDUMP = os.path.join(build.ROCM, "llvm", "bin", "llvm-objdump")
_LINE = re.compile(r"\s+([a-z]\w+)\s*([^/]*)")


def unwaited(listing):
    """(loads into LDS, those directly behind a write of M0) of a listing."""
    loads, bad, before = 0, [], None
    for line in listing.splitlines():
        m = _LINE.match(line)
        if m is None:
            before = before if not line.endswith(">:") else None
            continue
        op, args = m.group(1), m.group(2).strip()
        if op.startswith("global_load_lds") or (op.startswith("buffer_load") and
                                                re.search(r"\blds$", args)):
            loads += 1
            if before is not None:
                bad.append(f"{before}; {op} {args}")
        writes = re.match(r"m0\b", args) and not op.startswith(("s_cmp", "v_cmp"))
        before = f"{op} {args}" if writes else None
    return loads, bad


def code_objects(library, folder):
    """The library's gfx950 code objects, unpacked into `folder`."""
    copy = shutil.copy(library, folder)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, stdout=subprocess.DEVNULL)
    return sorted(os.path.join(folder, f) for f in os.listdir(folder) if f.endswith(build.ARCH))


@pytest.mark.parametrize("text, bad", [
    ("\ts_mov_b32 m0, s4\n\tglobal_load_lds_dwordx4 v[0:1], off", 1),
    ("\ts_add_i32 m0, s2, 0x400\n\tbuffer_load_dwordx4 v3, s[0:3], 0 offen lds", 1),
    ("\ts_mov_b32 m0, s4\n\ts_nop 0\n\tglobal_load_lds_dword v[0:1], off", 0),
    ("\ts_mov_b32 m0, s4\n\tv_mov_b32 v1, v2\n\tbuffer_load_dwordx4 v3, s[0:3], 0 offen lds", 0),
    ("\ts_mov_b32 m0, s4\n\tbuffer_load_dwordx4 v[4:7], v3, s[0:3], 0 offen", 0),
])
def test_listing(text, bad):
    assert len(unwaited(text)[1]) == bad


@pytest.mark.parametrize("name", [build.LIB_NAME, build.DIAG_LIB_NAME])
def test_loads_into_lds_wait_for_m0(name, tmp_path):
    library = os.path.join(build.PKG_DIR, name)
    if not os.path.exists(OBJDUMP) or not os.path.exists(library):
        pytest.skip("needs llvm-objdump and the built library")
    total = 0
    for code in code_objects(library, str(tmp_path)):
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", code],
                                 check=True, capture_output=True, text=True).stdout
        loads, bad = unwaited(listing)
        total += loads
        assert not bad, f"{os.path.basename(code)}: {len(bad)} of {loads}, first {bad[0]}"
    assert total > 100
