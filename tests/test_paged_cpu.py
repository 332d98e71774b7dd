"""CPU: the index arithmetic of the four-bit paged cache (csrc/paged_index.h compiled with the host compiler) and the refusals of the
packed serving calls — arguments are checked before a device is looked for, so every refusal can be seen without one."""
import ctypes as C
import itertools
import os
import subprocess

import numpy as np
import pytest

import atlas_b200 as ab
from atlas_b200 import _ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SHIM = """
#include "paged_index.h"
extern "C" {
long long tile_bytes(int n, int p, int k, int hd, int g) { AxP4Shape s = { n, p, k, hd, g }; return ax_p4_tile_bytes(s); }
long long pool_bytes(int n, int p, int k, int hd, int g) { AxP4Shape s = { n, p, k, hd, g }; return (long long)ax_p4_pool_bytes(s); }
long long tile_at(int n, int p, int k, int hd, int g, int page, int head, int off) { AxP4Shape s = { n, p, k, hd, g }; return (long long)ax_p4_tile_at(s, page, head, off); }
int plane(int hd, int g) { AxP4Shape s = { 1, 16, 1, hd, g }; return ax_p4_plane_bytes(s); }
int k_word(int hd, int g, int r, int d) { AxP4Shape s = { 1, 16, 1, hd, g }; return ax_p4_k_word(s, r, d); }
int v_half(int hd, int g, int r, int d) { AxP4Shape s = { 1, 16, 1, hd, g }; return ax_p4_v_half(s, r, d); }
int scale_at(int hd, int g, int r, int gr) { AxP4Shape s = { 1, 16, 1, hd, g }; return ax_p4_scale(s, r, gr); }
int col(int r) { return ax_p4_col(r); }
}
"""


@pytest.fixture(scope="module")
def idx(tmp_path_factory):
    d = tmp_path_factory.mktemp("idx")
    (d / "shim.cpp").write_text(SHIM)
    so = str(d / "shim.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I", os.path.join(ROOT, "atlas_b200", "csrc"), str(d / "shim.cpp"), "-o", so], check=True)
    L = C.CDLL(so)
    for f in ("tile_bytes", "pool_bytes", "tile_at"):
        getattr(L, f).restype = C.c_longlong
    return L


@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_every_number_of_a_tile_has_a_place_of_its_own(idx, hd, group):
    plane = idx.plane(hd, group)
    assert plane == 16 * hd // 2
    words = {idx.k_word(hd, group, r, d) for r in range(16) for d in range(0, hd, 8)}
    assert words == set(range(plane // 4))
    halves = {idx.v_half(hd, group, r, d) for r in range(16) for d in range(0, hd, 4)}
    assert halves == set(range(plane // 2))
    scales = {idx.scale_at(hd, group, r, g) for r in range(16) for g in range(hd // group)}
    assert scales == set(range(16 * (hd // group)))
    assert idx.tile_bytes(1, 16, 1, hd, group) == 2 * plane + 2 * 2 * len(scales)
    assert idx.tile_bytes(1, 16, 1, hd, group) % 16 == 0          # a tile is one bulk copy


@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_lanes_find_their_operands(idx, hd, group):
    """What the product's lanes assume: lane 4g + t reads hd / 32 consecutive K words of column 8nt + g whose groups follow one another,
    and V words whose halves are rows 8nt + t and 8nt + 4 + t."""
    w = hd // 32
    for r in range(16):
        col = idx.col(r)
        nt, g, t = r // 8, (r // 4) % 2, r % 4
        assert col == 8 * nt + 2 * t + g                                   # column 2t + b of block nt is row 8nt + 4b + t
        for d in range(0, hd, 8):
            word = idx.k_word(hd, group, r, d)
            assert word // (4 * w) == col
            lane_t, i = (word // w) % 4, word % w
            assert i // (group // 32) == d // group and lane_t == (d % group) // (group // 4)
        for d in range(0, hd, 4):
            half = idx.v_half(hd, group, r, d)
            assert half % 2 == g and (half // 2 // w) % 4 == t and half // 2 // (32 * w) == nt
            assert (half // 2) % w == (d // group) * (group // 32) + ((d % group) % (group // 8)) // 4


@pytest.mark.parametrize("hd", [64, 128])
def test_groups_of_64_keep_a_threads_two_k_words_together(idx, hd):
    """The pair that is written as one 8-byte word."""
    for r in range(16):
        for d in range(0, hd, 16):
            w = idx.k_word(hd, 64, r, d)
            assert w % 2 == 0 and idx.k_word(hd, 64, r, d + 8) == w + 1


def test_numbers_are_rounded_half_away_from_zero():
    """|y| + (1/2 − 2^-25) + 2^23 with the second sum cut off, in f32, next to every border below 8."""
    f = np.float32
    for k in range(8):
        for c in (f(k), f(k + 0.5)):
            y = c
            for _ in range(4):
                y = np.nextafter(y, f(-1))
            for _ in range(9):
                if 0 <= y < 7.5:
                    s = f(y) + f(0.49999997)
                    assert np.floor(np.float64(s)) == np.floor(np.float64(y) + 0.5), y
                y = np.nextafter(y, f(100))


def test_tiles_stay_inside_the_pool(idx):
    for n, p, k, hd, g in itertools.product((1, 3), (16, 48, 128), (1, 5), (64, 128), (32, 64)):
        size, total = idx.tile_bytes(n, p, k, hd, g), idx.pool_bytes(n, p, k, hd, g)
        at = sorted({idx.tile_at(n, p, k, hd, g, page, h, off) for page in range(n) for h in range(k) for off in range(p)})
        assert at == list(range(0, total, size))
    # a pool of 300 GB: offsets beyond 32 bits
    n, p, k = 8_000_000, 16, 16
    assert idx.tile_at(n, p, k, 128, 32, n - 1, k - 1, 15) == idx.pool_bytes(n, p, k, 128, 32) - 2304 == n * k * 2304 - 2304


def test_reciprocal_of_the_page_size_is_exact():
    """slot / page_size as the kernels take it: (slot / 16) · ceil(2^36 / (page_size / 16)) >> 36, at the borders of every page size."""
    for d in range(1, 513):
        inv = -(-(1 << 36) // d)
        top = (1 << 27) - 1
        q = np.unique(np.concatenate([np.arange(0, 50), np.arange(top // d - 50, top // d + 1)]))
        for n in np.concatenate([q * d, q * d + d - 1, [top]]):
            n = int(min(max(n, 0), top))
            assert (n * inv) >> 36 == n // d and n * inv < 1 << 64


def test_argument_structs_have_the_c_layout(tmp_path):
    """Sizes and the offset of the last member, from the header with the host compiler."""
    src = tmp_path / "sizes.c"
    src.write_text('#include "atlas_kernels.h"\n#include <stdio.h>\nint main(void) {'
                   'printf("%zu %zu %zu %zu %zu %zu %zu %zu", sizeof(atlasx_page_plan_args), offsetof(atlasx_page_plan_args, n_tokens),'
                   'sizeof(atlasx_pagedkv_rows), offsetof(atlasx_pagedkv_rows, n), sizeof(atlasx_pagedkv_attn_args), offsetof(atlasx_pagedkv_attn_args, scale),'
                   'sizeof(atlasx_prompt_args), offsetof(atlasx_prompt_args, scale)); return 0; }')
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    for i, f in enumerate((_ffi.PAGE_PLAN, _ffi.PAGED_ROWS, _ffi.PAGED_ATTN, _ffi.PROMPT)):
        assert f.size - 4 == got[2 * i + 1] and f.size <= got[2 * i] < f.size + 8


# ── refusals ─────────────────────────────────────────────────────────────────────
P = 1 << 20      # a pointer that is never followed: every call below is refused before it runs


def refused(rc, text):
    msg = _ffi.lib().atlasx_last_error().decode()
    assert rc == -1 and text in msg, (rc, msg)


def packed(layout, args):
    """The argument struct as the library gets it (None: a null pointer)."""
    return layout.pack(*(0 if v is None else v for v in args.values()))


PLAN = dict(cached=P, fresh=P, free=P, table=P, cu=P, lens=P, slots=P, pos=P, status=P, batch=4, n_free=8, page_size=16, n_pages=8, width=4,
            n_tokens=4)


@pytest.mark.parametrize("change,text", [
    (dict(cached=None), "null argument"), (dict(status=None), "null argument"), (dict(slots=None), "null argument"),
    (dict(free=None), "null argument"), (dict(batch=0), "batch"), (dict(batch=4097), "batch"), (dict(page_size=0), "page_size"),
    (dict(n_pages=1 << 30, page_size=16), "2^31"), (dict(width=0), "column"), (dict(n_tokens=-1), "negative"), (dict(n_tokens=1 << 30), "too many"),
    (dict(n_free=-1), "negative"), ({}, "ctx is null")])
def test_plan_refusals(change, text):
    refused(_ffi.lib().atlasx_page_plan(None, packed(_ffi.PAGE_PLAN, dict(PLAN, **change))), text)


@pytest.mark.parametrize("shape,text", [
    ((0, 16, 1, 64, 32), "positive"), ((4, 16, 0, 64, 32), "positive"), ((4, 8, 1, 64, 32), "multiple of 16"),
    ((4, 24, 1, 64, 32), "multiple of 16"), ((4, 8208, 1, 64, 32), "8192"), ((1 << 27, 16, 1, 64, 32), "2^31"), ((4, 16, 1, 96, 32), "head_dim"),
    ((4, 16, 1, 128, 16), "group"), ((4, 16, 1, 128, 128), "group"), ((4, 16, 1, 128, 32), "ctx is null")])
def test_cache_refusals(shape, text):
    h = C.c_void_p()
    refused(_ffi.lib().atlasx_pagedkv_create(None, *shape, C.byref(h)), text)
    if "ctx" not in text:
        assert _ffi.lib().atlasx_pagedkv_bytes(*shape) == 0
    else:
        assert _ffi.lib().atlasx_pagedkv_bytes(*shape) == 4 * 2304


ROWS = dict(k=P, v=P, slots=P, kt=128, kh=128, vt=128, vh=128, dtype=1, n=3)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(n=-1), "negative"), (dict(n=1 << 30), "too many"), (dict(k=None), "null"), (dict(slots=None), "null"), (dict(k=P + 2), "16-byte"),
    (dict(kt=129), "16-byte"), (dict(vh=4), "16-byte"), (dict(dtype=0, kt=130), "16-byte"), ({}, "ctx or cache is null")])
def test_append_refusals(change, text):
    refused(_ffi.lib().atlasx_pagedkv_append(None, None, packed(_ffi.PAGED_ROWS, dict(ROWS, **change))), text)


READ = dict(ctx=None, kv=None, slots=P, n=3, dtype=0, k=P, v=P)


@pytest.mark.parametrize("change,text", [(dict(dtype=3), "dtype"), (dict(n=-2), "negative"), (dict(v=None), "null"), (dict(v=P + 4), "16-byte"),
                                         ({}, "ctx or cache is null")])
def test_read_refusals(change, text):
    refused(_ffi.lib().atlasx_pagedkv_read(*dict(READ, **change).values()), text)


DEC = dict(q=P, out=P, table=P, lens=P, ws=None, wsn=0, n_heads=8, width=4, batch=2, window=0, scale=0.1)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null"), (dict(lens=None), "null"), (dict(batch=0), "batch"), (dict(batch=5000), "batch"), (dict(n_heads=0), "n_heads"),
    (dict(width=0), "column"), (dict(window=-1), "window"), (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"),
    (dict(q=P + 8), "16-byte"), ({}, "ctx or cache is null")])
def test_decode_refusals(change, text):
    refused(_ffi.lib().atlasx_pagedkv_decode_attention(None, None, packed(_ffi.PAGED_ATTN, dict(DEC, **change))), text)


PROMPT = dict(q=P, k=P, v=P, out=P, qt=512, qh=128, kt=256, kh=128, vt=256, vh=128, ot=512, oh=128, cu_q=P, cu_k=P, dtype=1, batch=2,
              n_q=10, n_k=10, n_heads=4, n_kv=2, hd=128, window=0, scale=0.1)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=0), "dtype"), (dict(batch=0), "batch"), (dict(batch=4097), "batch"), (dict(n_q=-1), "negative"), (dict(n_heads=3), "multiple"),
    (dict(n_kv=0), "multiple"), (dict(hd=96), "head_dim"), (dict(window=-5), "window"), (dict(scale=float("nan")), "finite"),
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(cu_k=None), "null"), (dict(q=P + 2), "16-byte"), (dict(kt=257), "16-byte"),
    (dict(vt=-256), "negative"), (dict(kh=0), "zero"), (dict(qt=0), "zero"), (dict(n_q=1 << 30), "too many"), (dict(oh=64), "overlap"), (dict(ot=0), "overlap"), ({}, "ctx is null")])
def test_prompt_refusals(change, text):
    refused(_ffi.lib().atlasx_prompt_attention(None, packed(_ffi.PROMPT, dict(PROMPT, **change))), text)


class FakeContext:
    device, handle = 0, None


def arr(shape, dtype, strides=None, device=0):
    c = FakeContext()
    c.device = device
    return ab.DeviceArray(c, P, shape, dtype, strides)


def test_python_refuses_arrays_that_do_not_fit():
    q, k = arr((5, 4, 64), ab.BF16), arr((7, 2, 64), ab.BF16)
    cu = arr((3,), ab.I32)
    good = dict(q=q, k=k, v=k, out=q, cu_q=cu, cu_k=cu)
    for change, text in [(dict(q=arr((5, 4, 64), ab.F32)), "bf16 or f16"), (dict(k=arr((7, 2, 128), ab.BF16)), r"k must be"),
                         (dict(v=arr((6, 2, 64), ab.BF16)), "same rows"), (dict(v=arr((7, 2, 64), ab.F16)), "same type"),
                         (dict(out=arr((5, 4, 64), ab.BF16, (512, 64, 2))), "unit stride"), (dict(cu_k=arr((4,), ab.I32)), "shape"),
                         (dict(cu_q=arr((3,), ab.F32)), "int32"), (dict(q=arr((20, 64), ab.BF16)), "dimensions"),
                         (dict(k=arr((7, 2, 64), ab.BF16, device=1)), "device"), (dict(q=7), "not a device array"),
                         (dict(cu_q=arr((3,), ab.I32, (2,))), "contiguous"), (dict(window_size=1 << 40), "out of range")]:
        with pytest.raises(ab.AtlasError, match=text):
            ab.prompt_attention(**dict(good, **change))
    b = arr((4,), ab.I32)
    plan = dict(cached=b, fresh=b, free_pages=b, table=arr((4, 3), ab.I32), cu=arr((5,), ab.I32), lens=b, slots=b, pos=b, status=arr((3,), ab.I32),
                page_size=16, n_pages=4)
    for change, text in [(dict(cu=b), "cu must have shape"), (dict(table=arr((3, 3), ab.I32)), "table must"), (dict(status=b), "status"),
                         (dict(table=arr((4, 3), ab.I32, (1, 4))), "contiguous"), (dict(pos=arr((5,), ab.I32)), "pos"),
                         (dict(lens=arr((4,), ab.F32)), "int32")]:
        with pytest.raises(ab.AtlasError, match=text):
            ab.page_plan(**dict(plan, **change))


def test_torch_tensors_on_the_host_are_refused():
    torch = pytest.importorskip("torch")
    x = torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ab.AtlasError, match="not on device 0"):
        ab.prompt_attention(x, x, x, x, cu, cu)


def test_device_array_strides():
    a = arr((3, 4, 8), ab.F32)
    assert a.strides == (32, 8, 1)
    assert a.columns(8, (3, 2, 8), (32, 8, 1)).ptr == P + 32
    assert np.dtype(np.uint16).itemsize * 8 == 16


def test_device_array_views_stay_within_their_array():
    a = arr((3, 4, 8), ab.F32)                                        # elements 0..95
    assert a.columns(95, (1, 1, 1), (1, 1, 1)).ptr == P + 4 * 95
    assert a.columns(88, (3, 8), (-40, 1)).ptr == P + 4 * 88          # backwards, 8..95
    assert a.columns(96, (0, 8), (8, 1)).shape == (0, 8)              # an empty view reaches nothing
    part = a.columns(8, (3, 2, 8), (32, 8, 1))                        # 0..79 of its own
    assert part.columns(72, (8,), (1,)).ptr == P + 4 * 80
    for view, first, shape, strides in [(a, 96, (1,), (1,)), (a, -1, (1,), (1,)), (a, 8, (3, 4, 8), (32, 8, 1)), (a, 79, (3, 8), (-40, 1)),
                                        (part, 80, (1,), (1,)), (part, 72, (9,), (1,)), (arr((0, 8), ab.F32), 0, (1,), (1,))]:
        with pytest.raises(ab.AtlasError, match="leaves an array"):
            view.columns(first, shape, strides)
    for shape, strides in [((3, 4), (1,)), ((-1, 4), (4, 1))]:
        with pytest.raises(ab.AtlasError, match="a view needs"):
            a.columns(0, shape, strides)


@pytest.mark.parametrize("unit,text", [(-1, "unit"), (0, "head_dim 64")])
def test_selftest_refusals(unit, text):
    refused(_ffi.lib().atlasx_pagedkv_selftest_wait_expiry(None, None, packed(_ffi.PAGED_ATTN, DEC), unit), text)


def test_plan_refuses_outputs_that_overlap():
    """No device is asked: the context is memory of zeros, which a refusal never looks into."""
    ctx = C.create_string_buffer(1 << 16)
    q = 1 << 12
    apart = dict(PLAN, **{n: P + q * i for i, n in enumerate(("cached", "fresh", "free", "table", "cu", "lens", "slots", "pos", "status"))})
    call = lambda **change: _ffi.lib().atlasx_page_plan(C.addressof(ctx), packed(_ffi.PAGE_PLAN, dict(apart, **change)))      # noqa: E731
    for out in ("table", "cu", "lens", "slots", "pos", "status"):
        for other in ("cached", "fresh", "free"):
            refused(call(**{out: apart[other]}), "overlaps an input")
        refused(call(**{out: apart["cached"] + 12}), "overlaps an input")                   # the last request's number
    refused(call(cu=apart["fresh"] - 16), "overlaps an input")                              # five numbers: the last is fresh[0]
    refused(call(table=apart["fresh"] - 60), "overlaps an input")
    refused(call(slots=apart["pos"]), "outputs overlap")
    refused(call(status=apart["table"] + 4 * 15), "outputs overlap")
    if not ab.cuda_available():                                                             # nothing to refuse: a device is asked for
        for fine in ({}, dict(fresh=apart["cached"]), dict(cu=apart["fresh"] - 20), dict(lens=apart["cached"] + 16), dict(table=apart["fresh"] - 64)):
            assert call(**fine) == -2, fine


def test_strides_that_are_never_taken_may_be_anything():
    """Of a single row, of a single head.  Nothing is refused: a device is asked for, or the context is missed."""
    for change in (dict(n=1, kt=129, vt=1), dict(n=1, kt=0, vt=-3)):
        refused(_ffi.lib().atlasx_pagedkv_append(None, None, packed(_ffi.PAGED_ROWS, dict(ROWS, **change))), "ctx or cache is null")
    for change in (dict(n_q=1, qt=1, ot=3), dict(n_q=1, qt=0, ot=-8), dict(n_k=1, kt=0, vt=5), dict(n_k=0, k=None, v=None, kt=0, vt=1, kh=0, vh=-3),
                   dict(n_heads=1, n_kv=1, qh=0, kh=3, vh=-1, oh=7)):
        refused(_ffi.lib().atlasx_prompt_attention(None, packed(_ffi.PROMPT, dict(PROMPT, **change))), "ctx is null")


@pytest.mark.parametrize("ot,oh,fine", [(512, 128, True), (128, 1280, True), (496, 128, False), (384, 128, False), (128, 1272, False), (256, 128, False), (128, 128, False),
                                        (1 << 40, 1 << 40, False)])
def test_rows_of_out_must_not_meet(ot, oh, fine):
    """Ten rows of four heads of 128."""
    refused(_ffi.lib().atlasx_prompt_attention(None, packed(_ffi.PROMPT, dict(PROMPT, ot=ot, oh=oh))), "ctx is null" if fine else "overlap")


def test_arrays_of_another_device_are_refused_without_a_context():
    """The default context, on device 0, takes the call: arrays that are all on device 1 do not move it there."""
    one = lambda shape, dtype: arr(shape, dtype, device=1)                    # noqa: E731
    b = one((4,), ab.I32)
    with pytest.raises(ab.AtlasError, match="cached is not on device 0"):
        ab.page_plan(b, b, b, one((4, 3), ab.I32), one((5,), ab.I32), b, b, b, one((3,), ab.I32), page_size=16, n_pages=4)
    q, cu = one((5, 4, 64), ab.BF16), one((3,), ab.I32)
    with pytest.raises(ab.AtlasError, match="q is not on device 0"):
        ab.prompt_attention(q, q, q, q, cu, cu)


@pytest.mark.parametrize("place", range(5))
def test_a_cache_of_more_than_a_c_int_is_refused(place):
    """Not cut to its low 32 bits."""
    shape = [4, 16, 1, 128, 32]
    with pytest.raises(ab.AtlasError, match="ctx is null"):
        ab.PagedKvCache(*shape, ctx=FakeContext())
    shape[place] += 1 << 32
    with pytest.raises(ab.AtlasError, match="out of range"):
        ab.PagedKvCache(*shape, ctx=FakeContext())


# ── the kernels' own arithmetic ──────────────────────────────────────────────────
@pytest.fixture(scope="module")
def arith(tmp_path_factory):
    """Rounding and slot arithmetic as the kernels have them (csrc/paged_index.h), compiled for the host."""
    d = tmp_path_factory.mktemp("arith")
    (d / "shim.cpp").write_text('#include "paged_index.h"\nextern "C" {\n'
                                'int number(float y) { volatile float s = y + ax_p4_half(y); return (int)s; }\n'
                                'unsigned long long inverse(int p) { return ax_p4_page_inverse(p); }\n'
                                'int page_of(int slot, unsigned long long inv) { return ax_p4_page_of(slot, inv); }\n}\n')
    so = str(d / "shim.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-I", os.path.join(ROOT, "atlas_b200", "csrc"), str(d / "shim.cpp"), "-o", so], check=True)
    L = C.CDLL(so)
    L.number.argtypes, L.inverse.restype, L.page_of.argtypes = [C.c_float], C.c_ulonglong, [C.c_int, C.c_ulonglong]
    return L


def test_the_kernels_round_half_away_from_zero(arith):
    """Next to every half and whole number below 8, on both sides of zero."""
    f = np.float32
    for k in range(8):
        for c in (f(k), f(k + 0.5)):
            y = c
            for _ in range(4):
                y = np.nextafter(y, f(-1))
            for _ in range(9):
                if abs(y) < 7.5:
                    want = int(np.copysign(np.floor(abs(np.float64(y)) + 0.5), y))
                    assert arith.number(float(y)) == want and arith.number(float(-y)) == -want, y
                y = np.nextafter(y, f(100))
    for y in (1e-45, 1e-38, 1e-20, 0.0):
        assert arith.number(y) == arith.number(-y) == 0


def test_the_kernels_find_a_slots_page(arith):
    for p in range(16, 8193, 16):
        inv = arith.inverse(p)
        top = (1 << 31) - 1
        n = top // p
        for page in {0, 1, 2, n // 3, n // 2, n - 2, n - 1}:
            for off in (0, 1, 15, 16, p - 1):
                slot = page * p + off
                if 0 <= slot <= top and off < p:
                    assert arith.page_of(slot, inv) == page, (p, slot)
        assert arith.page_of(top, inv) == top // p
