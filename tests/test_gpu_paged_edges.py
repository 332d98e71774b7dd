"""GPU: the packed serving step where it can go wrong — waits that run out, indices outside the pool, extreme values, lengths and windows —
against plain implementations in 64 bits.  Helpers and tolerances are those of test_gpu_paged.py unless a test derives its own."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import orc
from test_gpu_paged import Cache, bf16, check_decode, decode_by_hand, down, held, prompt_by_hand, prompt_case, rows, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ab():
    import atlas_b200
    return atlas_b200


# ── decode attention: a wait that runs out ───────────────────────────────────────
@pytest.mark.parametrize("lens,n_kv,nh", [([9000], 1, 4), ([3000, 1, 2999, 64], 2, 16), ([40] * 3000, 2, 2), ([200, 17] * 30, 4, 4)])
def test_a_decode_call_whose_wait_ran_out_leaves_its_workspace_good(ab, lens, n_kv, nh):
    """The copy of one unit never comes, at many places of the work: the call ends with an error status, all counters are back at zero, and the
    next call with the same workspace gives what one with a fresh workspace gives."""
    from atlas_b200 import _ffi
    rng = np.random.default_rng(len(lens))
    c = Cache(ab, rng, lens, n_kv, 64, 32, 16)
    q = rng.standard_normal((len(lens), nh, 64)).astype(np.float32)
    want = check_decode(ab, c, nh, 0.125, 0, q=q, workspace=c.kv.workspace())
    ws = c.kv.workspace()
    ctx = c.kv.ctx
    qd, out = up(ab, q, ab.F32), up(ab, q, ab.F32)
    table, n = ab.DeviceArray.from_host(c.table, ab.I32), ab.DeviceArray.from_host(lens, ab.I32)
    args = _ffi.PAGED_ATTN.pack(qd.ptr, out.ptr, table.ptr, n.ptr, ws.ptr, 4 * ws.shape[0], nh, c.table.shape[1], len(lens), 0, 0.125)
    tiles = sum(-(-m // 16) for m in lens) * n_kv
    units = tiles if tiles <= ctx.sm_count * 3 * 4 else sum(-(-(-(-m // 16)) // 2) for m in lens) * n_kv
    places = sorted({0, 1, units - 1, units - 2} | set(rng.integers(0, units, 10).tolist()))
    for unit in places:
        _ffi.check(_ffi.lib().atlasx_pagedkv_selftest_wait_expiry(ctx.handle, c.kv._h, args, int(unit)))
        code = C.c_int(0)
        assert _ffi.lib().atlasx_ctx_poll_device_error(ctx.handle, C.byref(code)) == -5 and code.value == 741
        assert not ws.download()[:3 * ctx.sm_count].any(), unit
        assert np.array_equal(check_decode(ab, c, nh, 0.125, 0, q=q, workspace=ws), want), unit
    # a unit that is not there: nothing is lost
    _ffi.check(_ffi.lib().atlasx_pagedkv_selftest_wait_expiry(ctx.handle, c.kv._h, args, units))
    assert ctx.poll_device_error() == 0 and np.array_equal(out.download(), want)


# ── indices that name nothing ────────────────────────────────────────────────────
def test_bad_slots_and_pages_do_not_stop_a_model(ab):
    """They are reported by poll_device_error, and the model on the same context goes on."""
    import helpers
    w = helpers.synth_weights(helpers.SMALL_SWA, seed=8)
    m = helpers.cuda_model(dict(helpers.SMALL_SWA), w, helpers.SMALL_SWA_LAYERS, kv_dtype=ab.F32)
    want = m.forward_one_gpu(7)
    m.reset()
    kv = ab.PagedKvCache(2, 16, 1, 64)
    x = up(ab, np.ones((1, 1, 64)), ab.F32)
    one = ab.DeviceArray.from_host([1], ab.I32)
    kv.append(x, x, ab.DeviceArray.from_host([32], ab.I32))
    assert np.array_equal(m.forward_one_gpu(7), want)
    with pytest.raises(ab.AtlasError, match="slot"):
        kv.ctx.poll_device_error()
    kv.decode_attention(x, up(ab, np.ones((1, 1, 64)), ab.F32), ab.DeviceArray.from_host([[2]], ab.I32), one, 0.1)
    m.reset()
    assert np.array_equal(m.forward_one_gpu(7), want)
    # a wait that ran out is reported first, and does stop the model; the index error beside it is still there afterwards
    from atlas_b200 import _ffi
    code = C.c_int(0)
    _ffi.check(_ffi.lib().atlasx_comm_selftest_wait_expiry(kv.ctx.handle, C.byref(code), 1))
    with pytest.raises(ab.AtlasError, match="bounded device-side wait"):
        m.forward_one_gpu(7)
    with pytest.raises(ab.AtlasError, match="bounded device-side wait"):
        kv.ctx.poll_device_error()
    with pytest.raises(ab.AtlasError, match="page outside"):
        kv.ctx.poll_device_error()
    assert kv.ctx.poll_device_error() == 0
    m.reset()
    assert np.array_equal(m.forward_one_gpu(7), want)


# ── decode attention: values of very different size ──────────────────────────────
class Held(Cache):
    """A cache of given rows: request i has lens[i] rows of its own, one behind the other, in pages of `page`."""

    def __init__(self, ab, lens, k, v, group, page=16):
        self.ab, self.lens, self.page = ab, lens, page
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need)
        self.table = np.full((len(lens), max(need)), -1)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = np.arange(at, at + m)
            at += m
        full = lambda x: np.concatenate([x, np.zeros((self.n_pages * page - len(x),) + x.shape[1:], x.dtype)])      # noqa: E731
        k, v = full(np.asarray(k, np.float32)), full(np.asarray(v, np.float32))
        self.kv = ab.PagedKvCache(self.n_pages, page, k.shape[1], k.shape[2], group=group)
        self.kv.append(up(ab, k, ab.F32), up(ab, v, ab.F32), ab.DeviceArray.from_host(np.arange(len(k)), ab.I32))
        self.k, self.v = held(k, group), held(v, group)


@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-8, 1e-12, 1e-20])
def test_rows_and_groups_of_zeros_beside_small_values(ab, hd, group, size):
    """A group of zeros says nothing about the size of the others: V of any size beside zero rows (padding, a first token) and beside a
    group of zeros is as accurate as without them (the tolerance has no term for them: 7 · scale ≤ 1.01 · max|v| holds for every group
    that is not zero)."""
    rng = np.random.default_rng(17)
    n = 100
    k, v = rows(rng, n, 2, hd), size * rows(rng, n, 2, hd)
    v[[0, 5, 40, 41, 99]] = 0
    v[20:30, :, :group] = 0
    k[7] = 0
    c = Held(ab, [n], k, v, group)
    check_decode(ab, c, 4, 1 / math.sqrt(hd), 0, rng=rng)
    check_decode(ab, c, 4, 1 / math.sqrt(hd), 3, rng=rng)
    c = Held(ab, [40], k[:40], 0 * v[:40], group)                          # nothing but zeros
    assert not check_decode(ab, c, 4, 0.1, 0, rng=rng).any()


@pytest.mark.parametrize("window", [0, 5_000_000])
def test_tiny_values_over_many_rows(ab, window):
    """2^24 rows (2048 times one page of 8192) with V near 1e-30: the sum of the probabilities stays finite.  The softmax over repeated rows is that
    over the page; a window of w rows sees its last w mod 8192 rows once more than the others.  Tolerance: as for all decode calls, and 2^-112 for values
    below 2^-80, times 2 for the scale's rounding and the products' sums."""
    rng = np.random.default_rng(23)
    page, times = 8192, 2048
    k, v = rows(rng, page, 1, 64), 1e-30 * rows(rng, page, 1, 64)
    c = Held(ab, [page], k, v, 32, page)
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    q[0, 0] = 0                                                              # all rows alike: the largest sum
    out = up(ab, np.full(q.shape, 7.0), ab.F32)
    c.kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(np.zeros((1, times)), ab.I32),
                          ab.DeviceArray.from_host([page * times], ab.I32), 0.125, window)
    n = window or page * times
    count = np.full(page, n // page)
    count[page - n % page:] += 1 if n % page else 0
    for h in range(2):
        a = c.k[:, 0] @ q[0, h].astype(np.float64) * 0.125
        p = np.exp(a - a.max()) * count
        p /= p.sum()
        e = (2.0 ** -16 + 2.0 ** -18) * 0.125 * (np.abs(c.k[:, 0]) @ np.abs(q[0, h].astype(np.float64))).max()
        tol = (2 * e + 2.0 ** -12) * (p @ np.abs(c.v[:, 0])) + 2.0 ** -111
        assert np.all(np.abs(out.download()[0, h] - p @ c.v[:, 0]) <= tol)


# ── capture on the context's stream, with nothing but the driver ─────────────────
class Graph:
    """What was called inside `with Graph(ctx)`, replayed on the context's stream or another one (cuStreamBeginCapture: the calls behind
    cudaStreamBeginCapture and its family)."""

    def __init__(self, ctx, mode=0):
        self.cu, self.s, self.mode = C.CDLL("libcuda.so.1"), C.c_void_p(ctx.stream), mode      # 0 global, 1 thread-local, 2 relaxed
        self.exec = C.c_void_p()

    def ok(self, rc):
        assert rc == 0, "driver error %d" % rc

    def __enter__(self):
        self.ok(self.cu.cuStreamBeginCapture_v2(self.s, self.mode))
        return self

    def __exit__(self, kind, *_):
        g = C.c_void_p()
        rc = self.cu.cuStreamEndCapture(self.s, C.byref(g))
        if kind is None:
            self.ok(rc)
            self.ok(self.cu.cuGraphInstantiateWithFlags(C.byref(self.exec), g, C.c_ulonglong(0)))
        if g:
            self.cu.cuGraphDestroy(g)

    def replay(self, stream=None):
        self.ok(self.cu.cuGraphLaunch(self.exec, C.c_void_p(stream) if stream else self.s))

    def close(self):
        if self.exec:
            self.ok(self.cu.cuGraphExecDestroy(self.exec))
            self.exec = C.c_void_p()

    def free_bytes(self):
        a, b = C.c_size_t(), C.c_size_t()
        self.ok(self.cu.cuMemGetInfo_v2(C.byref(a), C.byref(b)))
        return a.value


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_a_step_is_captured_while_objects_are_freed(ab, mode):
    """plan → append → decode captured with arrays of this module; arrays, caches, vectors and matrices that nothing refers to any more go
    while the capture runs.  The capture holds, the graph follows the lengths, and the memory is free afterwards."""
    rng = np.random.default_rng(61)
    b, nh, n_kv, hd, page, n_pages, width = 3, 4, 2, 128, 16, 60, 16
    kv = ab.PagedKvCache(n_pages, page, n_kv, hd)
    ctx = kv.ctx
    i32 = lambda x: ab.DeviceArray.from_host(x, ab.I32)                       # noqa: E731
    order = rng.permutation(n_pages)
    lens = np.array([100, 16, 47])
    table_np = np.full((b, width), -1)
    at = 0
    for i, n in enumerate(lens):
        m = -(-n // page)
        table_np[i, :m] = order[at:at + m]
        at += m
    k0, v0 = rows(rng, n_pages * page, n_kv, hd), rows(rng, n_pages * page, n_kv, hd)
    kv.append(up(ab, k0, ab.F32), up(ab, v0, ab.F32), i32(np.arange(n_pages * page)))
    kh, vh = held(k0, 32), held(v0, 32)
    table, free, cached, fresh = i32(table_np), i32(order[at:]), i32(lens), i32([1, 1, 1])
    cu, now, slots, pos, status = (i32(np.zeros(n)) for n in (b + 1, b, b, b, 3))
    k, v, q, out = (up(ab, np.zeros((b, h, hd)), ab.F32) for h in (n_kv, n_kv, nh, nh))
    kn, vn, qn = rows(rng, b, n_kv, hd), rows(rng, b, n_kv, hd), rng.standard_normal((b, nh, hd)).astype(np.float32)
    for d, x in ((k, kn), (v, vn), (q, qn)):
        ctx.upload(d.ptr, x)
    gone = [ab.DeviceArray.empty((1 << 28,), ab.F32), ab.PagedKvCache(4096, 64, 8, 128), ab.GpuVec.zeros(1 << 26),
            ab.GpuMatrix.upload(np.zeros((512, 512)), 512, 512), ab.GpuKvCache(4096, 8, 128)]
    # run once outside: kernels are loaded by their first launch
    ab.page_plan(cached, fresh, free, table, cu, now, slots, pos, status, page_size=page, n_pages=n_pages)
    kv.append(k, v, slots)
    kv.decode_attention(q, out, table, now, 0.09)
    ctx.sync()
    g = Graph(ctx, mode)
    before = g.free_bytes()
    with g:
        gone.pop()
        ab.page_plan(cached, fresh, free, table, cu, now, slots, pos, status, page_size=page, n_pages=n_pages)
        gone.clear()
        kv.append(k, v, slots)
        kv.decode_attention(q, out, table, now, 0.09)
        assert g.free_bytes() < before + (1 << 20)                           # kept
    for _ in range(3):
        ctx.upload(out.ptr, np.zeros((b, nh, hd), np.float32))
        g.replay()
        got = out.download()
        assert status.download().tolist()[1:] == [0, 0]
        sl = slots.download()
        kh[sl], vh[sl] = held(kn, 32), held(vn, 32)
        c = Cache.__new__(Cache)
        c.page, c.table, c.k, c.v = page, table.download(), kh, vh
        want, tol = decode_by_hand(c, qn, 0.09, 0, (lens + 1).tolist())
        assert np.all(np.abs(got - want) <= tol)
        used = int(status.download()[0])
        ctx.upload(free.ptr, np.roll(free.download(), -used))
        lens = lens + 1
        ctx.upload(cached.ptr, lens.astype(np.int32))
        kn, vn, qn = rows(rng, b, n_kv, hd), rows(rng, b, n_kv, hd), rng.standard_normal((b, nh, hd)).astype(np.float32)
        for d, x in ((k, kn), (v, vn), (q, qn)):
            ctx.upload(d.ptr, x)
    ctx.sync()
    assert g.free_bytes() > before + (1 << 30)
    g.close()
    assert ctx.poll_device_error() == 0


# ── prompt attention ─────────────────────────────────────────────────────────────
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh", [2, 3])
def test_windows_wider_than_the_prompts(ab, hd, nh):
    """They hide nothing, up to the largest one, with more queries than keys (negative positions) too: bit for bit the result without one."""
    lq, lk = [300, 20, 9, 150, 140], [170, 3, 0, 150, 400]
    want = prompt_case(ab, lq, lk, nh, 1, hd, 0, "BF16", np.random.default_rng(71))
    for window in (400, sum(lk) - 1, sum(lk), 1 << 30, (1 << 31) - 300, (1 << 31) - 1):
        assert np.array_equal(prompt_case(ab, lq, lk, nh, 1, hd, window, "BF16", np.random.default_rng(71)), want), window


@pytest.mark.parametrize("hd", [64, 128])
def test_a_score_of_minus_infinity_weighs_nothing_where_a_row_is_taken_again(ab, hd):
    """Key 0 scores −inf with every query, value 5 has a NaN in column 7: that column is NaN, the others are the softmax over the other keys;
    query 0 sees nothing but key 0: 0 / 0."""
    rng = np.random.default_rng(72)
    n = 150
    q, k, v = (bf16(rng.standard_normal((n, 1, hd)).astype(np.float32)) for _ in range(3))
    q[..., 0] = 1.0
    k[0] = 0
    want, tol = prompt_by_hand(q[1:], k[1:], v[1:], [0, n - 1], [0, n - 1], 0.1, 0, False)      # key 0 left out
    k[0, 0, 0] = -np.inf
    v[5, 0, 7] = np.nan
    out = ab.DeviceArray.empty((n, 1, hd), ab.BF16)
    cu = ab.DeviceArray.from_host([0, n], ab.I32)
    ab.prompt_attention(*(up(ab, t, ab.BF16) for t in (q, k, v)), out, cu, cu, 0.1)
    got = down(ab, out)
    assert np.isnan(got[0]).all() and np.isnan(got[5:, 0, 7]).all()
    fine = np.abs(got[1:] - want) <= tol
    assert fine[:4].all() and np.delete(fine, 7, axis=2).all()
    assert ab.Context.default().poll_device_error() == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_many_small_probabilities_in_f16(ab, hd):
    """One key with a score of 0 and value 0, 2^17 with probabilities of 2^-26 each and value 1: together they are 2^-9 of the row and more than
    that of the output.  Half a step of an f16 number per probability (they are powers of two: none) and of the output."""
    n = (1 << 17) + 1
    q, k, v = np.zeros((1, 1, hd)), np.zeros((n, 1, hd)), np.ones((n, 1, hd))
    q[..., 0] = 1
    k[1:, 0, 0] = -26
    v[0] = 0
    out = ab.DeviceArray.empty((1, 1, hd), ab.F16)
    ab.prompt_attention(*(up(ab, t, ab.F16) for t in (q, k, v)), out, ab.DeviceArray.from_host([0, 1], ab.I32), ab.DeviceArray.from_host([0, n], ab.I32),
                        math.log(2.0))
    want = 2.0 ** -9 / (1 + 2.0 ** -9)
    # ln 2 · log2 e in f32 is off by at most 2^-23 of itself, 26 of it as an exponent by 2^-18
    assert np.all(np.abs(down(ab, out) - want) <= want * (2.0 ** -11 + 2.0 ** -16))


def test_rows_taken_again_do_not_run_out_the_waits_of_others(ab, monkeypatch):
    """A NaN in the first value: every row is taken again, an item's rows for longer than a wait may take.  The limit is set low here so that a
    prompt of 8192 is long enough; with the 10 seconds there are it takes half a million rows."""
    monkeypatch.setenv("ATLASX_PROMPT_SHORT_WAITS", "1")
    ctx = ab.Context(0)
    n, nh, hd = 8192, 5, 64
    rng = np.random.default_rng(73)
    q, k, v = (bf16(rng.standard_normal((n, nh, hd)).astype(np.float32)) for _ in range(3))
    ds = [ab.DeviceArray.from_host(orc.f32_to_bf16_rne(x).reshape(x.shape), ab.BF16, ctx) for x in (q, k, v)]
    out, cu = ab.DeviceArray.empty((n, nh, hd), ab.BF16, ctx), ab.DeviceArray.from_host([0, n], ab.I32, ctx)
    ab.prompt_attention(*ds, out, cu, cu, 0.1, ctx=ctx)
    assert ctx.poll_device_error() == 0
    some = [0, 1, 127, 128, 3000, 8191]                                     # as in every call, and with no wait expired
    got = down(ab, out)[some]
    for i, r in enumerate(some):
        want, tol = prompt_by_hand(q[r:r + 1], k[:r + 1], v[:r + 1], [0, 1], [0, r + 1], 0.1, 0, False)
        assert np.all(np.abs(got[i] - want[0]) <= tol[0])
    v[0] = np.nan
    ctx.upload(ds[2].ptr, orc.f32_to_bf16_rne(v))
    ab.prompt_attention(*ds, out, cu, cu, 0.1, ctx=ctx)
    assert ctx.poll_device_error() == 0
    assert np.isnan(down(ab, out)).all()
    del ds, out, cu
    ctx.close()


# ── single rows and heads with strides of their own ──────────────────────────────
def test_a_single_row_and_a_single_head_of_odd_buffers(ab):
    rng = np.random.default_rng(74)
    hd = 64
    buf = bf16(rng.standard_normal(1000).astype(np.float32))
    b = up(ab, buf, ab.BF16)
    row = lambda at, h: buf[at:at + h * hd].reshape(1, h, hd)                # noqa: E731
    q, k, v = b.columns(8, (1, 2, hd), (333, hd, 1)), b.columns(200, (1, 1, hd), (77, 5, 1)), b.columns(304, (1, 1, hd), (1, 3, 1))
    out = up(ab, np.full((1, 2, hd), 7.0), ab.BF16)
    cu = ab.DeviceArray.from_host([0, 1], ab.I32)
    ab.prompt_attention(q, k, v, out.columns(0, (1, 2, hd), (31, hd, 1)), cu, cu, 0.1)
    assert np.array_equal(down(ab, out), np.repeat(row(304, 1), 2, axis=1))            # one key: its value
    kv = ab.PagedKvCache(1, 16, 1, hd)
    slot = ab.DeviceArray.from_host([3], ab.I32)
    kv.append(k, v, slot)
    ko, vo = ab.DeviceArray.empty((1, 1, hd), ab.F32), ab.DeviceArray.empty((1, 1, hd), ab.F32)
    kv.read(slot, ko, vo)
    assert np.array_equal(ko.download(), held(row(200, 1), 32).astype(np.float32)) and np.array_equal(vo.download(), held(row(304, 1), 32).astype(np.float32))
    # many rows of one head: only the head stride is free
    n = 7
    k = b.columns(16, (n, 1, hd), (72, 1, 1))
    sd = ab.DeviceArray.from_host(np.arange(n), ab.I32)
    kv.append(k, k, sd)
    ko, vo = ab.DeviceArray.empty((n, 1, hd), ab.F32), ab.DeviceArray.empty((n, 1, hd), ab.F32)
    kv.read(sd, ko, vo)
    want = np.stack([buf[16 + 72 * i:16 + 72 * i + hd] for i in range(n)]).reshape(n, 1, hd)
    assert np.array_equal(ko.download(), held(want, 32).astype(np.float32))


def test_values_next_to_halves_are_rounded_away_from_zero(ab):
    """A scale of 1 (a 7 in every group) and values next to every half and whole number, both signs."""
    f = np.float32
    y = [c for k in range(7) for c in (f(k), f(k + 0.5))]
    y = y + [np.nextafter(c, f(-9)) for c in y] + [np.nextafter(c, f(9)) for c in y]
    y = np.array(y + [-c for c in y], np.float32)
    x = np.zeros((-(-len(y) // 31), 1, 64), np.float32)
    for i, c in enumerate(y):
        x[i // 31, 0, 1 + i % 31] = c
    x[..., 0] = x[..., 32] = 7
    n = len(x)
    kv = ab.PagedKvCache(1, 16, 1, 64)
    sd = ab.DeviceArray.from_host(np.arange(n), ab.I32)
    kv.append(up(ab, x, ab.F32), up(ab, x, ab.F32), sd)
    ko, vo = ab.DeviceArray.empty((n, 1, 64), ab.F32), ab.DeviceArray.empty((n, 1, 64), ab.F32)
    kv.read(sd, ko, vo)
    want = np.copysign(np.floor(np.abs(x.astype(np.float64)) + 0.5), x)
    assert np.array_equal(ko.download(), want) and np.array_equal(vo.download(), want)


# ── decode attention: how accurate its parts are ─────────────────────────────────
@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_a_single_cached_row_comes_back_to_21_bits(ab, hd, group):
    """One row: the output is that row.  p · scale is rounded to f32 (2^-24), split into f16 parts (2^-22 of itself; the lo part's own smallest half step
    is 2^-25 where the row's largest p · scale is 2^7), the two products are added, divided by p (2^-24 each): |Δo| ≤ 2^-21·|v| +
    2^-32·1.01·max|v|.  Parts of eight bits would leave 2^-17."""
    rng = np.random.default_rng(81)
    b = 500
    k, v = rows(rng, b, 1, hd), rows(rng, b, 1, hd) * np.exp2(rng.integers(-30, 31, (b, 1, 1)))
    c = Held(ab, [1] * b, np.repeat(k, 16, 0), np.repeat(v, 16, 0), group)      # a page each
    q = rng.standard_normal((b, 2, hd)).astype(np.float32)
    out = up(ab, 0 * q, ab.F32)
    c.kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(np.arange(b).reshape(b, 1), ab.I32), ab.DeviceArray.from_host([1] * b, ab.I32), 0.1)
    want = np.repeat(c.v[::16], 2, 1)
    tol = 2.0 ** -21 * np.abs(want) + 2.0 ** -32 * 1.01 * np.abs(want).max(2, keepdims=True)
    err = np.abs(out.download() - want)
    assert np.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
def test_scores_are_good_to_20_bits(ab, hd, group):
    """Two rows with values 7u and −7u: the output is 7u·tanh((s1 − s2) / 2).  Queries have one number, so a score is one product: scale · log2 e
    is rounded twice, its product with the query once, the query's parts are good to 2^-22, the scale of K, the power of two's way back and the
    difference from the reference round once more: at most 2^-22 + 6·2^-24 < 2^-21 of |s|, and of the reference, which is within 22 of the
    larger s in log2 units (15 and the 7 below): 2^-24 · (|s| + 22).  exp2 is good to 2^-22.  |Δo| ≤ 7u · (½ · (|s1| + |s2|) · 2^-20 + 2^-19); parts of
    eight bits would leave 2^-17·|s|."""
    rng = np.random.default_rng(82)
    b, nh = 700, 4
    k = rows(rng, 2 * b, 1, hd)
    v = np.ones((2 * b, 1, hd), np.float32)
    v[1::2] = -1
    k16, v16 = np.zeros((16 * b, 1, hd), np.float32), np.zeros((16 * b, 1, hd), np.float32)
    for j in range(2):
        k16[j::16], v16[j::16] = k[j::2], v[j::2]
    c = Held(ab, [2] * b, k16, v16, group)
    q = np.zeros((b, nh, hd), np.float32)
    at = rng.integers(0, hd, (b, nh))
    np.put_along_axis(q, at[..., None], rng.uniform(1, 8, (b, nh, 1)).astype(np.float32), 2)
    out = up(ab, 0 * q, ab.F32)
    c.kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(np.arange(b).reshape(b, 1), ab.I32), ab.DeviceArray.from_host([2] * b, ab.I32), 0.7)
    s = [np.einsum("bhd,bd->bh", q.astype(np.float64), c.k[j::16, 0]) * float(np.float32(0.7)) for j in range(2)]
    unit = c.v[0, 0, 0]
    want = unit * np.tanh((s[0] - s[1]) / 2)
    tol = unit * (0.5 * (np.abs(s[0]) + np.abs(s[1])) * 2.0 ** -20 + 2.0 ** -19)
    err = np.abs(out.download() - want[..., None]).max(2)
    assert np.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("n,nh,n_kv", [(300, 1, 1), (700, 4, 2), (5000, 16, 8)])
def test_a_prompt_call_whose_wait_ran_out_leaves_everything_usable(ab, monkeypatch, n, nh, n_kv):
    """The copy of one K tile never comes.  The call ends with an error status, the other items' rows are right, and the next call on the
    same context (tensor memory and all) is too."""
    ctx_of = lambda v: (monkeypatch.setenv("ATLASX_PROMPT_SHORT_WAITS", v), ab.Context(0))[1]      # noqa: E731
    rng = np.random.default_rng(91)
    hd = 64
    q, k, v = (bf16(rng.standard_normal((n, h, hd)).astype(np.float32)) for h in (nh, n_kv, n_kv))
    results = []
    for mode in ("2", "1"):
        ctx = ctx_of(mode)
        ds = [ab.DeviceArray.from_host(orc.f32_to_bf16_rne(x).reshape(x.shape), ab.BF16, ctx) for x in (q, k, v)]
        out, cu = ab.DeviceArray.from_host(np.zeros((n, nh, hd)), ab.BF16, ctx), ab.DeviceArray.from_host([0, n], ab.I32, ctx)
        for _ in range(2):
            ab.prompt_attention(*ds, out, cu, cu, 0.1, ctx=ctx)
            if mode == "2":
                code = C.c_int(0)
                from atlas_b200 import _ffi
                assert _ffi.lib().atlasx_ctx_poll_device_error(ctx.handle, C.byref(code)) == -5 and 721 <= code.value <= 735
            else:
                assert ctx.poll_device_error() == 0
        results.append(down(ab, out))
        del ds, out, cu
        ctx.close()
    broken, fine = results
    some = [0, 1, 127, 255, n - 1]
    for r in some:
        want, tol = prompt_by_hand(q[r:r + 1], k[:r + 1], v[:r + 1], [0, 1], [0, r + 1], 0.1, 0, False)
        assert np.all(np.abs(fine[r] - want[0]) <= tol[0])
    # an item is 256 rows of a head or 128 of two: the lost one, and those that its CTA had taken over, were not written
    same = (broken == fine).all(2)
    assert (same | (broken == 0).all(2)).all() and not same.all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("where", ["q", "k"])
def test_a_nan_score_makes_its_rows_nan_and_no_others(ab, hd, where):
    """In a query: that row of that head.  In a key: the rows that see it, within the window and their sequence, of all heads that share it."""
    rng = np.random.default_rng(92)
    lens, nh, window = [200, 300], 4, 70
    n = sum(lens)
    q, k, v = (bf16(rng.standard_normal((n, h, hd)).astype(np.float32)) for h in (nh, 2, 2))
    cu = np.array([0, 200, 500])
    want, tol = prompt_by_hand(q, k, v, cu, cu, 0.1, window, False)
    nan = np.zeros((n, nh), bool)
    if where == "q":
        q[250, 2, 5] = np.nan
        nan[250, 2] = True
    else:
        k[260, 1, 5] = np.nan
        nan[260:330, 2:] = True
    out = up(ab, np.full(q.shape, 7.0), ab.BF16)
    c = ab.DeviceArray.from_host(cu, ab.I32)
    ab.prompt_attention(*(up(ab, t, ab.BF16) for t in (q, k, v)), out, c, c, 0.1, window)
    got = down(ab, out)
    assert np.isnan(got[nan]).all()
    assert np.all(np.abs(got - want)[~nan] <= tol[~nan])


def test_a_nan_in_an_early_key_of_a_long_prompt(ab):
    """Nothing but NaN, written as fast as anything else: row by row, 40 000 rows of 8 heads would take many seconds."""
    torch = pytest.importorskip("torch")
    n, nh, hd = 40000, 8, 64
    rng = np.random.default_rng(93)
    x = bf16(rng.standard_normal((n, nh, hd)).astype(np.float32))
    qd, vd = up(ab, x, ab.BF16), up(ab, x, ab.BF16)
    kd = [up(ab, x, ab.BF16), None]
    x[3] = np.nan
    kd[1] = up(ab, x, ab.BF16)
    out, cu = ab.DeviceArray.empty((n, nh, hd), ab.BF16), ab.DeviceArray.from_host([0, n], ab.I32)
    ctx = ab.Context.default()
    s = torch.cuda.ExternalStream(ctx.stream)
    ms = []
    for k in kd + kd:
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record(s)
        ab.prompt_attention(qd, k, vd, out, cu, cu, 0.1)
        b.record(s)
        ctx.sync()
        ms.append(a.elapsed_time(b))
    got = down(ab, out)
    assert np.isnan(got[3:]).all() and np.isfinite(got[:3]).all()
    assert ms[3] < 3 * ms[2], ms


# ── offsets that pass 32 bits ────────────────────────────────────────────────────
def test_a_cache_of_more_than_4_gib(ab):
    """65 536 pages of 64 rows and 8 heads (4.8 GB): rows in the first and the last pages, through append, read and decode attention."""
    rng = np.random.default_rng(95)
    n_pages, page, n_kv, hd = 65536, 64, 8, 128
    kv = ab.PagedKvCache(n_pages, page, n_kv, hd)
    assert kv.bytes > 1 << 32
    pages = np.array([n_pages - 1, 0, n_pages - 2, 1, 59652, 59653])          # byte 2^32 lies in page 58 254
    n = len(pages) * page
    k, v = rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
    slots = (pages[:, None] * page + np.arange(page)).ravel()
    sd = ab.DeviceArray.from_host(slots, ab.I32)
    kv.append(up(ab, k, ab.F32), up(ab, v, ab.F32), sd)
    ko, vo = ab.DeviceArray.empty((n, n_kv, hd), ab.F32), ab.DeviceArray.empty((n, n_kv, hd), ab.F32)
    kv.read(sd, ko, vo)
    assert np.array_equal(ko.download(), held(k, 32).astype(np.float32)) and np.array_equal(vo.download(), held(v, 32).astype(np.float32))
    c = Cache.__new__(Cache)
    c.page, c.table, c.k, c.v = page, np.arange(6).reshape(1, 6), held(k, 32), held(v, 32)
    q = rng.standard_normal((1, 16, hd)).astype(np.float32)
    out = up(ab, 0 * q, ab.F32)
    kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(pages.reshape(1, 6), ab.I32), ab.DeviceArray.from_host([n - 5], ab.I32), 0.09)
    want, tol = decode_by_hand(c, q, 0.09, 0, [n - 5])
    assert np.all(np.abs(out.download() - want) <= tol)
    assert kv.ctx.poll_device_error() == 0


@pytest.mark.parametrize("hd,nh", [(128, 32), (64, 33)])
def test_prompt_rows_behind_2_31_elements(ab, hd, nh):
    """A sequence at the end of buffers of 2^31 and more elements each; the rows before it belong to no sequence."""
    rng = np.random.default_rng(96)
    n, m = (1 << 31) // (nh * hd) + 400, 300
    ctx = ab.Context.default()
    x = [bf16(rng.standard_normal((m, nh, hd)).astype(np.float32)) for _ in range(3)]
    big = [ab.DeviceArray.empty((n, nh, hd), ab.BF16) for _ in range(4)]
    first = n - m
    at = 2 * first * nh * hd
    assert first * nh * hd > 1 << 31
    for d, y in zip(big, x):
        ctx.upload(d.ptr + at, orc.f32_to_bf16_rne(y))
    cu = ab.DeviceArray.from_host([first, n], ab.I32)
    ab.prompt_attention(*big, cu, cu, 0.1)
    got = orc.bf16_to_f32(ctx.download(big[3].ptr + at, (m * nh * hd,), np.uint16)).reshape(m, nh, hd)
    want, tol = prompt_by_hand(*x, [0, m], [0, m], 0.1, 0, False)
    assert np.all(np.abs(got - want) <= tol)
    # and the row form there
    x[2][0] = np.nan
    ctx.upload(big[2].ptr + at, orc.f32_to_bf16_rne(x[2]))
    ab.prompt_attention(*big, cu, cu, 0.1, window_size=m - 1)
    got = orc.bf16_to_f32(ctx.download(big[3].ptr + at, (m * nh * hd,), np.uint16)).reshape(m, nh, hd)
    assert np.isnan(got[:m - 1]).all() and np.all(np.abs(got[m - 1] - prompt_by_hand(x[0][m - 1:], x[1][1:], x[2][1:], [0, 1], [0, m - 1], 0.1, 0, False)[0][0])
                                                  <= prompt_by_hand(x[0][m - 1:], x[1][1:], x[2][1:], [0, 1], [0, m - 1], 0.1, 0, False)[1][0])
    assert ctx.poll_device_error() == 0
