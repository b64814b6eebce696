"""The host side of the paged-cache and logits entry points, compiled without
optimisation and with traps on division by zero, overflow and bad shifts.  The
calls run in a process that sees no GPU: each gets as far as its launch, which
fails there, and reports that."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "flux_b200" / "csrc"
NVCC = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"

pytestmark = pytest.mark.skipif(not Path(NVCC).exists(), reason="needs nvcc")


def compile_library(out: Path, sources: list[Path]) -> Path:
    host = ["-fPIC", "-O0", "-fsanitize=integer-divide-by-zero", "-fsanitize=signed-integer-overflow", "-fsanitize=shift",
            "-fsanitize-undefined-trap-on-error"]
    subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "--expt-relaxed-constexpr", "-O0",
                    "-Xcicc", "-O0", "-Xptxas", "-O0", *(f"-Xcompiler={flag}" for flag in host), "-I", str(ROOT / "include"),
                    "-I", str(CSRC), "-shared", "-cudart", "static", "-o", str(out), *map(str, sources)], check=True)
    return out


@pytest.fixture(scope="module")
def library(tmp_path_factory):
    return compile_library(tmp_path_factory.mktemp("host") / "host.so",
                           [CSRC / "paged_cache.cu", CSRC / "logits.cu", CSRC / "capi.cu"])


CHILD = """
import ctypes, itertools, sys
sys.path.insert(0, {root!r})
from flux_b200 import _native

lib = ctypes.CDLL({library!r})
FAKE = 0x100000  # never dereferenced: nothing can be launched here
SIZE = [4, 2, 2]


def call(name, *args):
    f = getattr(lib, name)
    f.restype, f.argtypes = _native.SIGNATURES[name]
    status = f(*args)
    lib.fx_last_error.restype = ctypes.c_char_p
    assert status == _native.FX_ERR_CUDA, (name, args, status, lib.fx_last_error())


def pool(dtype, dim, pages=5, kv_heads=2, page_size=16, layers=3):
    p = _native.Pages()
    p.keys, p.values, p.dtype = FAKE, 2 * FAKE, dtype
    p.layers, p.pages, p.kv_heads, p.page_size, p.head_dim = layers, pages, kv_heads, page_size, dim
    page = kv_heads * page_size * dim
    for i, s in enumerate((pages * page, page, page_size * dim, dim)):
        p.key_strides[i] = p.value_strides[i] = s
    return ctypes.byref(p)

"""


def run(library, code):
    """In a process of its own, without a GPU."""
    result = subprocess.run([sys.executable, "-c", CHILD.format(root=str(ROOT), library=str(library)) + code],
                            env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, capture_output=True, text=True, timeout=300)
    assert result.returncode == 0, f"exit {result.returncode}: {result.stderr[-2000:]}"


def test_write_of_every_head_size(library):
    """Down to 8 dims, half of which is less than a 16-byte piece of 16-bit elements."""
    run(library, """
for (rows, pages), dim, tokens in itertools.product([(0, 0), (0, 1), (0, 2), (1, 1), (2, 2)], range(8, 257, 8),
                                                    [1, 3, 1000, 200000]):
    heads = 6 if tokens < 200000 else 1
    call("fx_paged_qkv_rope_cache", FAKE, rows, (heads + 4) * dim, tokens, heads, FAKE, dim, FAKE, dim, 50,
         pool(pages, dim), FAKE, tokens, 4, 4, FAKE, None, FAKE, None)
""")


def test_page_operations_of_every_page_size(library):
    run(library, """
for dtype, dim, page_size, layers, count in itertools.product([0, 1, 2], [8, 40, 64, 256], [1, 7, 16, 65536], [1, 30],
                                                              [1, 700, 10 ** 6]):
    p = pool(dtype, dim, page_size=page_size, layers=layers, pages=1000)
    call("fx_cache_pages_copy", p, FAKE, FAKE, count, None)
    if count == 1:
        call("fx_cache_sequences_fork", p, FAKE, 9, 4, 4, FAKE, FAKE, FAKE, FAKE, count, FAKE, FAKE, None)
        if page_size < 65536:
            call("fx_cache_pages_compact", p, FAKE, 9, 4, 4, FAKE, FAKE, FAKE, None)
    call("fx_cache_sequences_reserve", FAKE, 9, 4, 4, FAKE, FAKE, 1000, page_size, FAKE, FAKE, count, FAKE, FAKE, None)
    call("fx_cache_sequences_free", FAKE, 9, 4, 4, FAKE, FAKE, 1000, FAKE, count, None)
""")


def test_logits_of_every_shape(library):
    run(library, """
for dtype, rows, vocab, history in itertools.product([0, 1, 2], [1, 2, 147, 148, 149, 300, 10000], [1, 31, 32, 2049, 49152,
                                                     100277], [0, 1, 8191, 8192, 32767, 32768, 10 ** 6]):
    tokens = FAKE if history else None
    call("fx_logits_process", FAKE, dtype, rows, vocab, vocab, tokens, history, history, tokens, tokens, tokens, None, 0,
         None, 0, FAKE, vocab, None)
""")
