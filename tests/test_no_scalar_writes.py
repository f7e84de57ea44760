"""Nothing here writes memory through the scalar data cache: no source (kernels, inline assembly, the interpreter's tables) names
such an instruction, and the gfx950 assembly of every kernel holds none.  tools/gfxsim therefore models none either: a listing
that had one would end in its "instruction not modelled" instead of running."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCALAR_WRITE = re.compile(r"\bs_(?:(?:buffer_|scratch_)?(?:store|atomic)_|dcache_(?:wb|discard))\w*")
SOURCES = (".hip", ".h", ".inc", ".c", ".cpp", ".py", ".sh", ".s")


def _found(path):
    with open(path, errors="replace") as f:
        return ["%s:%d: %s" % (os.path.relpath(path, ROOT), n, m.group(0)) for n, line in enumerate(f, 1) for m in [SCALAR_WRITE.search(line)] if m]


def test_pattern():
    for family in ("store", "buffer_store", "scratch_store", "atomic", "buffer_atomic"):
        assert SCALAR_WRITE.search("\ts_%s_x" % family)
    for other in ("s_load_dwordx4 s[0:3], s[4:5], 0x0", "s_buffer_load_dword s0, s[4:7], 0x0", "s_dcache_inv", "global_store_dword v[0:1], v2, off",
                  "buffer_store_dword v0, off, s[0:3], 0", "ds_add_u32 v0, v1", "global_atomic_add v[0:1], v2, off"):
        assert not SCALAR_WRITE.search(other)


def test_no_source_names_one():
    bad = []
    for top in ("bench.py", "__graft_entry__.py", "include", "oracle", "sharpziplib_amd", "tests", "tools"):
        top = os.path.join(ROOT, top)
        files = [top] if os.path.isfile(top) else [os.path.join(d, f) for d, sub, names in os.walk(top) if "_build" not in d.split(os.sep) for f in names]
        for f in files:
            if f.endswith(SOURCES) or os.path.basename(f) == "Makefile":
                bad += _found(f)
    assert not bad, bad


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc") and shutil.which("hipcc") is None, reason="hipcc is needed for the device assembly")
@pytest.mark.parametrize("lab", [False, True], ids=["product", "lab"])
def test_no_kernel_holds_one(lab):
    code = "import sys; sys.path.insert(0, %r); from gfxsim import harness as H; H.build(); print(H.BUILD, *H.KERNEL_UNITS)" % os.path.join(ROOT, "tools")
    env = dict(os.environ, GFXSIM_LAB="1" if lab else "")          # (which library is built is settled when the harness is imported)
    build, *units = subprocess.check_output([sys.executable, "-c", code], env=env, text=True).splitlines()[-1].split()
    bad = []
    for u in units:
        bad += _found(os.path.join(build, u + ".s"))
    assert units and not bad, bad
