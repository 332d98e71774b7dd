"""The loader gives pages of a mapped file back (madvise MADV_DONTNEED) once a converted or gathered slice has been read.  Where the range
reaches behind the mapping, pages of somebody else — a heap, a library's data — read as zeros from then on, without any error.
CPU: the range arithmetic (csrc/file_pages.h).  GPU: what the loader hands to madvise, seen by a stand-in for it."""
import ctypes as C
import json
import os
import struct
import subprocess
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    d = tmp_path_factory.mktemp("pages")
    (d / "shim.cpp").write_text('#include "file_pages.h"\nextern "C" void rows(size_t at, size_t size, size_t cols, size_t r0, size_t r1, size_t page,'
                                'size_t n, size_t* out) { AxFileRange r = ax_file_rows(at, size, cols, r0, r1, page, n); out[0] = r.first; out[1] = r.last; }')
    so = str(d / "shim.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-I", os.path.join(ROOT, "atlas_b200", "csrc"), str(d / "shim.cpp"), "-o", so], check=True)
    L = C.CDLL(so)
    L.rows.argtypes = [C.c_size_t] * 7 + [C.POINTER(C.c_size_t)]

    def call(*a):
        out = (C.c_size_t * 2)()
        L.rows(*a, out)
        return out[0], out[1]
    return call


def test_rows_of_a_file_stay_within_it(rows):
    n = 100_000
    # a 16-bit tensor that ends with the file: 64 rows of 128, from byte 83 616
    assert rows(n - 64 * 128 * 2, 2, 128, 0, 64, 4096, n) == (81920, n)
    assert rows(n - 64 * 128 * 2, 2, 128, 32, 64, 4096, n) == (90112, n)
    assert rows(4096, 4, 10, 0, 3, 4096, n) == (4096, 4096 + 120)
    assert rows(5000, 4, 10, 2, 2, 4096, n) == (4096, 5080)
    # numbers that do not fit the file are cut to it
    assert rows(n - 100, 4, 128, 0, 64, 4096, n) == (98304, n)
    assert rows(n + 9000, 4, 128, 0, 64, 4096, n) == (n, n)


MADVISE = r"""
#define _GNU_SOURCE
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <sys/mman.h>
/* Ranges that start in a mapped .safetensors file: written down, not carried out. */
int madvise(void* p, size_t n, int advice) {
    (void)advice;
    FILE* maps = fopen("/proc/self/maps", "r");
    char line[4096];
    unsigned long a, b, at = (unsigned long)p;
    while (maps && fgets(line, sizeof line, maps))
        if (sscanf(line, "%lx-%lx", &a, &b) == 2 && at >= a && at < b && strstr(line, ".safetensors")) {
            FILE* out = fopen(getenv("MADVISE_LOG"), "a");
            fprintf(out, "%ld\n", (long)(b - (at + n)));
            fclose(out);
        }
    if (maps) fclose(maps);
    return 0;
}
"""

LOAD = r"""
import sys
import atlas_b200 as ab
ab.load_model_from_safetensors(sys.argv[1], ab.ModelConfig(256, 64, 1, 4, 2, 128, 64, 10000.0, 1e-5), kv_dtype=ab.F32)
"""


@pytest.mark.gpu
def test_the_loader_gives_no_pages_back_that_are_not_the_files(tmp_path):
    """An F16 file whose last tensor is one of the converted ones."""
    shapes = {"norm.weight": (64,), "tok_embeddings.weight": (256, 64)}
    for name, shape in (("input_layernorm", (64,)), ("post_attention_layernorm", (64,)), ("self_attn.q_proj", (64, 64)), ("self_attn.k_proj", (32, 64)),
                        ("self_attn.v_proj", (32, 64)), ("self_attn.o_proj", (64, 64)), ("mlp.gate_proj", (128, 64)), ("mlp.up_proj", (128, 64)),
                        ("mlp.down_proj", (64, 128))):
        shapes["layers.0.%s.weight" % name] = shape
    entries, blob = {}, b""
    for name, shape in shapes.items():
        raw = np.ones(shape, np.float16).tobytes()
        entries[name] = {"dtype": "F16", "shape": list(shape), "data_offsets": [len(blob), len(blob) + len(raw)]}
        blob += raw
    path = str(tmp_path / "half.safetensors")
    text = json.dumps(entries)
    with open(path, "wb") as f:
        f.write(struct.pack("<Q", len(text)) + text.encode() + blob)
    (tmp_path / "madvise.c").write_text(MADVISE)
    so, log = str(tmp_path / "madvise.so"), str(tmp_path / "log")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(tmp_path / "madvise.c"), "-o", so], check=True)
    env = dict(os.environ, LD_PRELOAD=so, MADVISE_LOG=log, PYTHONPATH=ROOT)
    r = subprocess.run([sys.executable, "-c", LOAD, path], env=env, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0, r.stderr[-2000:]
    left = [int(x) for x in open(log).read().split()]          # bytes between the end of each range and the end of the mapping
    assert len(left) == len(shapes) and min(left) >= 0, left
