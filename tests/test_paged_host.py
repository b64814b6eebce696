"""The host side of the paged-cache and logits entry points, and the split of
paged attention's tiles (``csrc/paged_attention.cuh``), compiled without
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
    out.parent.mkdir(parents=True, exist_ok=True)
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


# The functions that the kernels themselves call.
SPLIT = r"""
#include "paged_attention.cuh"
using namespace fx;
namespace {
PagedAttend arguments(const int64_t* lengths, int batch, int kv_heads, int capacity) {
    PagedAttend a{};
    a.lengths = lengths;
    a.batch = batch;
    a.kv_heads = kv_heads;
    a.capacity = capacity;
    return a;
}
}
extern "C" {
int tiles32(int rows) { return paged_tiles<32>(rows); }
int tiles64(int rows) { return paged_tiles<64>(rows); }
int tiles128(int rows) { return paged_tiles<128>(rows); }
int first(int64_t i, int total, int ctas) { return paged_first(i, total, ctas); }
int owner(int64_t t, int total, int ctas) { return paged_owner(t, total, ctas); }
int rows_left(int tile_row, int offset, int rows) { return PagedRow::at(0, tile_row, offset, rows, true).rows; }
int64_t grid64(int batch, int kv_heads, int capacity) { return paged_grid<64>(arguments(nullptr, batch, kv_heads, capacity), 148, 3); }
unsigned quotient(int64_t d, unsigned n) { return FastDivide::by(d).quotient(n); }
// Tiles that CTA i of `ctas` walks: (sequence, head, tile, rows) of each; returns how many.
int walk64(const int64_t* lengths, int batch, int kv_heads, int capacity, int total, int ctas, int i, int* out, int room) {
    const PagedAttend a = arguments(lengths, batch, kv_heads, capacity);
    PagedStart start = paged_locate<64>(a, 0, paged_first(i, total, ctas));
    start.left = paged_first(i + int64_t{1}, total, ctas) - paged_first(i, total, ctas);
    PagedCursor<64> at;
    at.begin(start);
    int n = 0;
    for (; at.left > 0 && n < room; ++n) {
        out[4 * n] = at.b;
        out[4 * n + 1] = at.head;
        out[4 * n + 2] = at.tile;
        out[4 * n + 3] = at.piece();
        at.next(a);
    }
    return at.left > 0 ? -1 : n;
}
}
"""

SPLIT_CHILD = """
import random
for f in ("first", "owner"):
    getattr(lib, f).argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int]
lib.grid64.restype = ctypes.c_int64
lib.quotient.argtypes, lib.quotient.restype = [ctypes.c_int64, ctypes.c_uint], ctypes.c_uint
"""


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    folder = tmp_path_factory.mktemp("split")
    (folder / "split.cu").write_text(SPLIT)
    return compile_library(folder / "split.so", [folder / "split.cu"])


def test_tiles_of_up_to_the_most_rows(split):
    """A table may hold 2^31 - 1 rows, whose last tile ends behind them."""
    run(split, SPLIT_CHILD + """
TOP = 2 ** 31 - 1
for tile in (32, 64, 128):
    tiles = getattr(lib, f"tiles{tile}")
    for rows in [0, 1, tile - 1, tile, tile + 1, 5 * tile, 5 * tile + 1, 2147483616, *range(TOP - 130, TOP + 1)]:
        assert tiles(rows) == max(1, -(-rows // tile)), (tile, rows)
        last = (tiles(rows) - 1) * tile
        for offset in (0, 1, tile - 1, tile + 31):
            assert lib.rows_left(last, offset, rows) == rows - last - offset
for capacity in (1, 64, 65, 2147483616, TOP):
    assert lib.grid64(1, 1, capacity) == min(444, -(-capacity // 64))
assert lib.grid64(200, 3, TOP) == 444
""")


def test_every_tile_belongs_to_one_cta(split):
    run(split, SPLIT_CHILD + """
rng = random.Random(4)
for case in range(80):
    batch, kv_heads = rng.randint(1, 40), rng.randint(1, 8)
    lengths = [rng.choice([-1, 0, 1, 64, 65, rng.randint(0, 300), rng.randint(0, 5000), 2 ** 40]) for _ in range(batch)]
    capacity = rng.choice([1, 64, 3000, 10000])
    tiles = [max(1, -(-min(max(n, 0), capacity) // 64)) for n in lengths]
    total = sum(tiles) * kv_heads
    ctas = min(total, rng.choice([1, 7, 148, 444, 512]))
    line = [(b, h, t) for b in range(batch) for h in range(kv_heads) for t in range(tiles[b])]
    walked, sizes = [], []
    for i in range(ctas):
        out = (ctypes.c_int * (4 * total))()
        n = lib.walk64((ctypes.c_int64 * batch)(*lengths), batch, kv_heads, capacity, total, ctas, i, out, total)
        assert n > 0
        for k in range(n):
            b, h, t, piece = out[4 * k:4 * k + 4]
            assert piece == min(tiles[b] - t, n - k)  # of this unit and of this CTA
            assert lib.owner(len(walked), total, ctas) == i
            walked.append((b, h, t))
        sizes.append(n)
    assert walked == line and max(sizes) - min(sizes) <= 1
""")


def test_the_split_of_the_most_tiles(split):
    run(split, SPLIT_CHILD + """
TOP = 2 ** 31 - 1
for total in (TOP, TOP - 1, 2 ** 30):
    for ctas in (1, 3, 148, 444, 512):
        assert lib.first(0, total, ctas) == 0 and lib.first(ctas, total, ctas) == total
        for i in range(ctas):
            first, last = lib.first(i, total, ctas), lib.first(i + 1, total, ctas)
            assert first < last and lib.owner(first, total, ctas) == lib.owner(last - 1, total, ctas) == i
""")


def test_quotients_are_exact(split):
    run(split, SPLIT_CHILD + """
rng = random.Random(9)
for d in [*range(1, 100), *(2 ** k for k in range(17)), *(rng.randint(1, 65536) for _ in range(200)), 65535, 2 ** 31 - 1]:
    for n in [0, 1, d - 1, d, 2 ** 31 - 1, 2 ** 31 - 2, *(rng.randrange(2 ** 31) for _ in range(50))]:
        assert lib.quotient(d, n) == n // d
""")
