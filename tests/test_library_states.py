"""What a process sees of the native libraries as they come and go: nothing
built yet, built while the process runs, older than the package, built from
other sources.  Each case runs in a process of its own on a copy of the package,
where building means putting this checkout's libraries in place (or compiling,
where it has none)."""

from __future__ import annotations

import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from flux_b200 import build as flux_build

ROOT = Path(__file__).resolve().parents[1]

# Makes `g.build()` of the copy take this checkout's libraries instead of compiling.
BUILD = f"""
import shutil, sys
from pathlib import Path
import torch
import __graft_entry__ as g

built = [Path(p) for p in {[str(flux_build.LIBRARY), str(flux_build.TORCH_LIBRARY)]!r}]

def build():
    import flux_b200.build as b
    if all(p.exists() for p in built):
        def place(verbose=False):
            b.LIB_DIR.mkdir(exist_ok=True)
            for p in built:
                shutil.copy2(p, b.LIB_DIR / (p.name + ".new"))
                (b.LIB_DIR / (p.name + ".new")).replace(b.LIB_DIR / p.name)
            b._native.SOURCES_PATH.write_text(b._native.sources_digest())
            return b.TORCH_LIBRARY
        b.build_torch_classes = place
    g.build("no reference checkout")

def reserve():
    from flux_b200 import operators as ops
    i32, i64 = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    ops.cache_sequences_reserve_native(i32, i64, i32[0], i64, i64, 16)

def refused(message):
    try:
        reserve()
    except RuntimeError as error:
        assert message in str(error), error
    else:
        raise AssertionError("not refused")
"""


@pytest.fixture
def copy(tmp_path):
    """The package without anything built."""
    for name in ("flux_b200", "flux", "include"):
        shutil.copytree(ROOT / name, tmp_path / name, ignore=shutil.ignore_patterns("_build", "_lib", "__pycache__"))
    shutil.copy2(ROOT / "__graft_entry__.py", tmp_path)
    return tmp_path


def run(copy, code):
    result = subprocess.run([sys.executable, "-c", BUILD + code], cwd=copy, capture_output=True, text=True, timeout=900)
    assert result.returncode == 0, result.stderr[-3000:]


def test_first_build_in_the_process_that_uses_it(copy):
    """Nothing built: the package imports and refuses; after the build it works, in the same process."""
    run(copy, """
from flux_b200 import operators as ops
assert not ops.native_paged_cache_is_available() and not ops.native_logits_process_is_available()
refused("is not built")
build()
assert ops.native_paged_cache_is_available() and ops.native_logits_process_is_available()
refused("CUDA tensors are required")
""")


def test_first_build_by_itself(copy):
    """The documented command in a clean checkout."""
    run(copy, """
build()
refused("CUDA tensors are required")
torch.classes.flux.NativeSmolLM2Decode
""")


def test_operators_are_registered_by_the_import(copy):
    run(copy, "build()")
    run(copy, """
import flux_b200
torch.ops.flux.paged_gqa_decode_attention
torch.ops.flux.logits_process
""")


def older(copy):
    """Libraries from before some entry points were added."""
    lib = copy / "flux_b200" / "_lib"
    lib.mkdir()
    for name, symbol in (("libfluxb200", "fx_last_error"), ("libfluxb200_torch", "flux_torch")):
        source = copy / f"{name}.c"
        source.write_text(f'const char* {symbol}(void) {{ return ""; }}\n')
        subprocess.run(["cc", "-shared", "-fPIC", str(source), "-o", str(lib / f"{name}.so")], check=True)


def test_older_libraries_are_refused_and_rebuilt(copy):
    """The package imports beside libraries that lack entry points, says so, and works once they are rebuilt."""
    older(copy)
    run(copy, """
import flux_b200
from flux_b200 import _native
from flux_b200 import operators as ops
assert not ops.native_paged_cache_is_available() and not flux_b200.is_available()
assert isinstance(_native.load_error(), _native.NativeLibraryUnavailable)
refused("older build")
build()
refused("CUDA tensors are required")
assert _native.load_error() is None
""")


def test_older_libraries_are_replaced_by_the_build_alone(copy):
    older(copy)
    run(copy, """
import flux
build()
refused("CUDA tensors are required")
torch.classes.flux.NativeSmolLM2Decode
""")


def test_an_older_torch_library_beside_a_new_one(copy):
    """As left by a build that ended between the two."""
    older(copy)
    run(copy, """
import flux_b200.build as b
if built[0].exists():
    shutil.copy2(built[0], str(b.LIBRARY) + ".new")
    Path(str(b.LIBRARY) + ".new").replace(b.LIBRARY)
else:
    b.build()
from flux_b200 import operators as ops
assert ops.native_rmsnorm_is_available() and not ops.native_paged_cache_is_available()
refused("older")
build()
refused("CUDA tensors are required")
""")


def test_a_build_from_other_sources_is_not_loaded_by_the_import(copy):
    """Complete libraries of sources that have changed since: the rebuild's code is what the process goes on with."""
    run(copy, "build()")
    source = copy / "flux_b200" / "csrc" / "logits.cu"
    source.write_text(source.read_text() + "\n")
    run(copy, """
import flux_b200, os
from flux_b200 import _native
old = os.stat(_native.LIBRARY_PATH).st_ino
assert not _native.torch_classes_loaded
build()
mapped = [line.split() for line in open("/proc/self/maps") if line.rstrip().endswith("libfluxb200.so")]
assert mapped and {int(fields[4]) for fields in mapped} == {os.stat(_native.LIBRARY_PATH).st_ino} != {old}
refused("CUDA tensors are required")
""")
    run(copy, """
import flux_b200
from flux_b200 import _native
assert _native.torch_classes_loaded  # the record follows the build
""")
