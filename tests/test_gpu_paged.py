"""GPU: the packed serving step — block tables, four-bit paged cache, decode attention over it and packed prompt attention — against
plain implementations in 64 bits.

Tolerances, from the arithmetic (u16 = half a step of the 16-bit type: 2^-8 bf16, 2^-11 f16):
  * plan, four-bit values: equal.
  * decode attention: queries and probabilities are split into 16-bit hi + lo parts (error at most 2^-16 of the value each), sums are f32.  A score is
    off by at most e = (2^-16 + 2^-18)·scale·Σ|q·k|, a probability by 2e of itself (its own and the normaliser's), the product by
    2^-16 more, f32 sums by 2^-18 at these lengths:  |Δo| ≤ (2·max e + 2^-15)·Σ p|v|.  The parts of p·(scale of V) are f16 numbers whose
    smallest step is 2^-24 where the row's largest is at least 2^7, so every row may be off by 2^-32 of the largest, times a number of
    at most 7; the largest number of a group is 7 (a scale rounded up leaves it at least 6.97), so 7·scale ≤ 1.01·max|v|:
    |Δo| ≤ … + rows·2^-32·1.01·max_j (p_j·max|v_j|).
  * prompt attention: products of 16-bit numbers are exact in f32, so a score is off by e = 2^-18·scale·Σ|q·k|; a probability is
    rounded to the 16-bit type (u16 of itself; in f16 at least 2^-25 of the row's largest) and the output once more:
    |Δo| ≤ u16·|o| + (u16 + 2·max e + 2^-16)·Σ p|v| + 2^-25·Σ|v| / l for f16, l ≥ 1 the normaliser.
"""
import math

import numpy as np
import pytest

from oracle import orc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ab():
    import atlas_b200
    return atlas_b200


def bf16(x):
    """Rounded to bf16, as f32."""
    return orc.bf16_to_f32(orc.f32_to_bf16_rne(np.ascontiguousarray(x, np.float32))).reshape(np.shape(x))


def up(ab, x, dtype):
    x = np.asarray(x)
    if dtype == ab.BF16:
        return ab.DeviceArray.from_host(orc.f32_to_bf16_rne(np.ascontiguousarray(x, np.float32)).reshape(x.shape), dtype)
    return ab.DeviceArray.from_host(x, dtype)


def down(ab, a):
    x = a.download()
    return orc.bf16_to_f32(x.ravel()).reshape(x.shape) if a.dtype == ab.BF16 else x.astype(np.float32) if a.dtype == ab.F16 else x


def held(x, group):
    """The values the four-bit format holds for f32 rows [..., hd]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    with np.errstate(all="ignore"):
        top = np.abs(g).max(-1)
        s = bf16((top / np.float32(7)).astype(np.float32))
        s = np.where(s < 2.0 ** -126, np.float32(1), s).astype(np.float32)
        y = (g * (np.float32(1) / s)[..., None]).astype(np.float64)
        n = np.clip(np.copysign(np.floor(np.abs(y) + 0.5), y), -7, 7)
        v = n * s[..., None].astype(np.float64)
    v[~np.isfinite(top)] = np.nan
    return v.reshape(x.shape)


def rows(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32)
    x[..., 3] *= 6
    return x


# ── plan ─────────────────────────────────────────────────────────────────────────
def plan_by_hand(cached, fresh, free, table, page, n_pages, n_tokens):
    table = table.copy()
    cu, slots, pos, at = [0], [], [], 0
    for b, (c, n) in enumerate(zip(cached, fresh)):
        for j in range(-(-c // page), -(-(c + n) // page)):
            table[b, j] = free[at]
            at += 1
        for p in range(c, c + n):
            g = table[b, p // page]
            slots.append(g * page + p % page if 0 <= g < n_pages else -1)
            pos.append(p)
        cu.append(cu[-1] + n)
    pad = n_tokens - len(slots)
    return table, np.array(cu), np.array(cached) + fresh, np.array(slots + [-1] * pad), np.array(pos + [-1] * pad), at


def call_plan(ab, cached, fresh, free, table, page, n_pages, n_tokens):
    b = len(cached)
    d = [ab.DeviceArray.from_host(x, ab.I32) for x in (cached, fresh, free, table)]
    o = [ab.DeviceArray.from_host(np.full(n, 77), ab.I32) for n in (b + 1, b, n_tokens, n_tokens, 3)]
    ab.page_plan(*d, *o, page_size=page, n_pages=n_pages)
    return [d[3].download()] + [x.download() for x in o]


@pytest.mark.parametrize("batch,cached_max,fresh_max,page,pad", [
    (1, 0, 1, 16, 0), (1, 5000, 1, 16, 3), (3, 40, 40, 16, 0), (7, 100, 0, 32, 2), (33, 300, 5, 48, 1), (256, 70, 9, 16, 0),
    (257, 1000, 40, 64, 100), (1000, 3, 3, 1, 0), (4096, 20, 2, 16, 5), (2, 10, 9000, 128, 0)])
def test_plan(ab, batch, cached_max, fresh_max, page, pad):
    rng = np.random.default_rng(batch + page)
    cached, fresh = rng.integers(0, cached_max + 1, batch), rng.integers(0, fresh_max + 1, batch)
    width = -(-(cached_max + fresh_max + 1) // page) + 1
    need = int((-(-(cached + fresh) // page)).sum())
    n_pages = need + 9
    order = rng.permutation(n_pages)
    table = rng.integers(-5, 0, (batch, width))
    at = 0
    for b in range(batch):
        m = -(-int(cached[b]) // page)
        table[b, :m] = order[at:at + m]
        at += m
    free = order[at:]
    n_tokens = int(fresh.sum()) + pad
    want = plan_by_hand(cached, fresh, free, table, page, n_pages, n_tokens)
    got = call_plan(ab, cached, fresh, free, table, page, n_pages, n_tokens)
    for g, w, name in zip(got, want, ("table", "cu", "lens", "slots", "pos")):
        assert np.array_equal(g, w), name
    assert got[5].tolist() == [want[5], 0, 0]


@pytest.mark.parametrize("what", ["short", "negative", "wide", "tokens", "long"])
def test_plan_that_cannot_be_made_changes_nothing(ab, what):
    cached, fresh, free = np.array([16, 3, 0]), np.array([1, 20, 16]), np.array([5, 6, 7])
    table, n = np.array([[0, -1], [1, -1], [-1, -1]]), 37
    if what == "short":
        free = free[:2]
    if what == "negative":
        cached[1] = -1
    if what == "wide":
        fresh[0] = 17
    if what == "tokens":
        n = 36
    if what == "long":                                                   # 2^31 rows and more
        cached[1], fresh[1] = 1 << 30, 1 << 30
    got = call_plan(ab, cached, fresh, free, table, 16, 8, n)
    assert np.array_equal(got[0], table)
    assert not got[1].any() and not got[2].any() and (got[3] == -1).all() and (got[4] == -1).all()
    assert got[5].tolist() == ([0, 1, 0] if what == "short" else [0, 0, 1])


def test_plan_pages_outside_the_pool_give_no_slots(ab):
    got = call_plan(ab, np.array([16]), np.array([17]), np.array([8, 2]), np.array([[0, -1, -1]]), 16, 8, 17)
    assert got[0].tolist() == [[0, 8, 2]]
    assert got[3].tolist() == [-1] * 16 + [32] and got[4].tolist() == list(range(16, 33))


# ── four-bit cache ───────────────────────────────────────────────────────────────
@pytest.mark.parametrize("dtype_name", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("hd,group,n_kv,page,n", [(64, 32, 1, 16, 1), (64, 64, 3, 48, 40), (128, 32, 8, 16, 77), (128, 64, 2, 128, 300)])
def test_rows_come_back_as_the_format_holds_them(ab, dtype_name, hd, group, n_kv, page, n):
    dtype = getattr(ab, dtype_name)
    rng = np.random.default_rng(n)
    n_pages = -(-n // page) + 2
    kv = ab.PagedKvCache(n_pages, page, n_kv, hd, group=group)
    cast = {"F32": lambda x: x, "BF16": bf16, "F16": lambda x: x.astype(np.float16).astype(np.float32)}[dtype_name]
    k, v = cast(rows(rng, n, n_kv, hd)), cast(rows(rng, n, n_kv, hd))
    slots = rng.permutation(n_pages * page)[:n]
    # k and v as column ranges of one buffer, as a fused product leaves them
    both = up(ab, np.concatenate([k.reshape(n, -1), v.reshape(n, -1)], 1), dtype)
    w = n_kv * hd
    kd, vd = both.columns(0, (n, n_kv, hd), (2 * w, hd, 1)), both.columns(w, (n, n_kv, hd), (2 * w, hd, 1))
    sd = ab.DeviceArray.from_host(slots, ab.I32)
    kv.append(kd, vd, sd)
    for out_name in ("F32", "BF16", "F16"):
        od = getattr(ab, out_name)
        ko, vo = ab.DeviceArray.empty((n, n_kv, hd), od), ab.DeviceArray.empty((n, n_kv, hd), od)
        kv.read(sd, ko, vo)
        cast_out = {"F32": lambda x: x, "BF16": bf16, "F16": lambda x: x.astype(np.float16).astype(np.float32)}[out_name]
        for got, x in ((ko, k), (vo, v)):
            assert np.array_equal(down(ab, got), cast_out(held(x, group).astype(np.float32)))
    assert kv.ctx.poll_device_error() == 0


def test_heads_may_be_strided(ab):
    """[heads, rows, hd] buffers: the head stride is the large one."""
    rng = np.random.default_rng(3)
    n, n_kv, hd = 21, 4, 64
    k = rows(rng, n_kv, n, hd)
    kd = up(ab, k, ab.F32)
    view = kd.columns(0, (n, n_kv, hd), (hd, n * hd, 1))
    kv = ab.PagedKvCache(2, 16, n_kv, hd)
    sd = ab.DeviceArray.from_host(np.arange(n), ab.I32)
    kv.append(view, view, sd)
    ko, vo = ab.DeviceArray.empty((n, n_kv, hd), ab.F32), ab.DeviceArray.empty((n, n_kv, hd), ab.F32)
    kv.read(sd, ko, vo)
    want = held(k.transpose(1, 0, 2), 32).astype(np.float32)
    assert np.array_equal(ko.download(), want) and np.array_equal(vo.download(), want)


def test_special_values(ab):
    """Zeros, numbers next to the ends of the range, NaN and infinities stay within their group."""
    hd, group = 128, 32
    x = np.ones((8, 1, hd), np.float32)
    x[0] = 0
    x[1, 0, :32] = 1e-45
    x[2, 0, :32] = 3.4e38
    x[3, 0, 40] = np.nan
    x[4, 0, 70] = np.inf
    x[5, 0, 127] = -np.inf
    x[6, 0, :32] = np.linspace(-7, 7, 32)
    x[7, 0, :32] = 1.2e-38
    kv = ab.PagedKvCache(1, 16, 1, hd, group=group)
    sd = ab.DeviceArray.from_host(np.arange(8), ab.I32)
    kv.append(up(ab, x, ab.F32), up(ab, x, ab.F32), sd)
    ko, vo = ab.DeviceArray.empty((8, 1, hd), ab.F32), ab.DeviceArray.empty((8, 1, hd), ab.F32)
    kv.read(sd, ko, vo)
    want = held(x, group).astype(np.float32)
    assert np.isnan(want[3, 0, 32:64]).all() and np.isfinite(want[3, 0, :32]).all()
    for got in (ko, vo):
        assert np.array_equal(got.download(), want, equal_nan=True)


def test_absent_rows_and_slots_behind_the_pool(ab):
    rng = np.random.default_rng(4)
    kv = ab.PagedKvCache(2, 16, 2, 64)
    k = rows(rng, 4, 2, 64)
    kv.append(up(ab, k, ab.F32), up(ab, k, ab.F32), ab.DeviceArray.from_host([5, -1, 9, -7], ab.I32))
    assert kv.ctx.poll_device_error() == 0
    all_slots = ab.DeviceArray.from_host(np.arange(-1, 33), ab.I32)
    ko, vo = ab.DeviceArray.empty((34, 2, 64), ab.F32), ab.DeviceArray.empty((34, 2, 64), ab.F32)
    kv.read(all_slots, ko, vo)
    with pytest.raises(ab.AtlasError, match="slot"):
        kv.ctx.poll_device_error()
    got = ko.download()
    assert not got[0].any() and not got[33].any()                       # slots −1 and 32
    want = held(k, 32).astype(np.float32)
    assert np.array_equal(got[1 + 5], want[0]) and np.array_equal(got[1 + 9], want[2])
    # a page never written holds (0 − 8)·0: zeros of either sign
    assert not got[1 + 20].any()
    before = ko.download()
    kv.append(up(ab, k, ab.F32), up(ab, k, ab.F32), ab.DeviceArray.from_host([32, 1 << 30, -1, 2147483647], ab.I32))
    with pytest.raises(ab.AtlasError, match="slot"):
        kv.ctx.poll_device_error()
    kv.read(ab.DeviceArray.from_host(np.arange(-1, 32), ab.I32), ab.DeviceArray.empty((33, 2, 64), ab.F32), ab.DeviceArray.empty((33, 2, 64), ab.F32))
    kv.read(all_slots, ko, vo)
    with pytest.raises(ab.AtlasError, match="slot"):
        kv.ctx.poll_device_error()
    assert np.array_equal(ko.download(), before)
    assert kv.ctx.poll_device_error() == 0


# ── decode attention ─────────────────────────────────────────────────────────────
class Cache:
    """A filled cache and what it holds."""

    def __init__(self, ab, rng, lens, n_kv, hd, group, page, spare=2, width=0):
        self.ab, self.lens, self.page = ab, lens, page
        need = [-(-n // page) for n in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max(max(need), 1, width)), -1)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        n = self.n_pages * page
        k, v = rows(rng, n, n_kv, hd), rows(rng, n, n_kv, hd)
        self.kv = ab.PagedKvCache(self.n_pages, page, n_kv, hd, group=group)
        self.kv.append(up(ab, k, ab.F32), up(ab, v, ab.F32), ab.DeviceArray.from_host(np.arange(n), ab.I32))
        self.k, self.v = held(k, group), held(v, group)

    def rows_of(self, b, lo, hi):
        t = np.arange(lo, hi)
        s = self.table[b, t // self.page] * self.page + t % self.page
        return self.k[s], self.v[s]


def decode_by_hand(c, q, scale, window, lens):
    b, nh, hd = q.shape
    n_kv = c.k.shape[1]
    out, tol = np.zeros((b, nh, hd)), np.zeros((b, nh, hd))
    for i in range(b):
        n = max(0, min(lens[i], c.table.shape[1] * c.page))
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        k, v = c.rows_of(i, lo, n)
        for h in range(nh):
            kh = h // (nh // n_kv)
            a = (k[:, kh] @ q[i, h].astype(np.float64)) * scale
            e = (2.0 ** -16 + 2.0 ** -18) * abs(scale) * (np.abs(k[:, kh]) @ np.abs(q[i, h].astype(np.float64))).max()
            p = np.exp(a - a.max())
            p /= p.sum()
            out[i, h] = p @ v[:, kh]
            tol[i, h] = (2 * e + 2.0 ** -15) * (p @ np.abs(v[:, kh])) + (n - lo) * 2.0 ** -32 * 1.01 * (p * np.abs(v[:, kh]).max(1)).max()
    return out, tol + 1e-30


def check_decode(ab, c, nh, scale, window, lens=None, workspace=None, q=None, rng=None):
    lens = c.lens if lens is None else lens
    hd = c.kv.head_dim
    q = (rng or np.random.default_rng(9)).standard_normal((len(lens), nh, hd)).astype(np.float32) if q is None else q
    out = up(ab, np.full(q.shape, 7.0), ab.F32)
    c.kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(c.table, ab.I32), ab.DeviceArray.from_host(lens, ab.I32), scale, window,
                          workspace)
    got = out.download()
    want, tol = decode_by_hand(c, q, scale, window, lens)
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    return got


@pytest.mark.parametrize("hd,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("nh,n_kv", [(1, 1), (8, 8), (8, 2), (6, 2), (8, 1), (9, 1), (24, 2)])
def test_decode_heads(ab, hd, group, nh, n_kv):
    rng = np.random.default_rng(nh * 10 + n_kv)
    c = Cache(ab, rng, [37, 1, 130], n_kv, hd, group, 16)
    check_decode(ab, c, nh, 1 / math.sqrt(hd), 0, rng=rng)


@pytest.mark.parametrize("page", [16, 32, 48, 128])
@pytest.mark.parametrize("window", [0, 1, 15, 16, 17, 100])
def test_decode_lengths_pages_windows(ab, page, window):
    rng = np.random.default_rng(page + window)
    c = Cache(ab, rng, [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 127, 128, 129, 200, 0], 2, 128, 32, page)
    check_decode(ab, c, 4, 1 / math.sqrt(128), window, rng=rng)
    assert c.kv.ctx.poll_device_error() == 0


@pytest.mark.parametrize("lens,n_kv,nh", [([5000], 1, 4), ([9001], 4, 4), ([3000, 1, 2999, 64], 2, 16), ([700] * 40, 2, 2), ([3] * 300, 1, 3)])
@pytest.mark.parametrize("window", [0, 1025])
def test_decode_long_and_many(ab, lens, n_kv, nh, window):
    rng = np.random.default_rng(len(lens))
    c = Cache(ab, rng, lens, n_kv, 64, 32, 32)
    check_decode(ab, c, nh, 0.2, window, rng=rng)


def test_decode_of_the_largest_batch(ab):
    rng = np.random.default_rng(41)
    lens = rng.integers(0, 20, 4096).tolist()
    c = Cache(ab, rng, lens, 1, 64, 32, 16)
    check_decode(ab, c, 1, 0.125, 0, rng=rng)


def test_decode_requests_may_share_pages(ab):
    rng = np.random.default_rng(42)
    c = Cache(ab, rng, [64, 80, 33], 2, 128, 64, 16)
    c.table[1, :4] = c.table[0, :4]                                         # a common prefix
    c.table[2, :2] = c.table[0, 0]                                          # the same page twice
    check_decode(ab, c, 6, 0.1, 0, rng=rng)


def test_decode_takes_the_lengths_as_they_are(ab):
    """Lengths beyond the table are cut to it, negative ones are empty; a wide table costs nothing but its columns."""
    rng = np.random.default_rng(5)
    c = Cache(ab, rng, [64, 64, 20], 1, 64, 32, 32, width=2)
    check_decode(ab, c, 2, 0.125, 0, lens=[1000, -3, 20], rng=rng)
    c = Cache(ab, rng, [64, 3], 1, 64, 32, 16, width=900)
    check_decode(ab, c, 2, 0.125, 0, rng=rng)


def test_decode_scores_of_any_size(ab):
    """Scores far apart, equal and zero scale."""
    rng = np.random.default_rng(6)
    c = Cache(ab, rng, [300, 40], 2, 128, 32, 16)
    q = rng.standard_normal((2, 4, 128)).astype(np.float32)
    check_decode(ab, c, 4, 0.0, 0, q=q)
    check_decode(ab, c, 4, -0.1, 0, q=q)
    check_decode(ab, c, 4, 3.0, 0, q=q)
    check_decode(ab, c, 4, 0.1, 0, q=0 * q)


def test_decode_does_not_read_what_is_hidden(ab):
    """NaN and infinities behind the length, before the window and in foreign pages stay where they are; in sight they show."""
    rng = np.random.default_rng(7)
    c = Cache(ab, rng, [50, 33], 1, 128, 32, 16)
    x = np.full((1, 1, 128), np.nan, np.float32)

    def poison(b, t):
        s = c.table[b, t // 16] * 16 + t % 16
        c.kv.append(up(ab, x, ab.F32), up(ab, x, ab.F32), ab.DeviceArray.from_host([s], ab.I32))
    for t in (50, 55, 63, 0, 9):
        poison(0, t)
    poison(1, 47)
    check_decode(ab, c, 4, 0.1, 40, rng=rng)
    poison(1, 32)
    out = ab.DeviceArray.empty((2, 4, 128), ab.F32)
    c.kv.decode_attention(up(ab, rng.standard_normal((2, 4, 128)), ab.F32), out, ab.DeviceArray.from_host(c.table, ab.I32),
                          ab.DeviceArray.from_host(c.lens, ab.I32), 0.1, 40)
    got = out.download()
    assert np.isfinite(got[0]).all() and np.isnan(got[1]).all()


def test_decode_pages_outside_the_pool_are_left_out(ab):
    rng = np.random.default_rng(8)
    c = Cache(ab, rng, [48, 16], 1, 64, 32, 16)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    good = c.table.copy()
    for bad in (-1, c.n_pages, 2147483647, -2147483648):
        c.table = good.copy()
        c.table[0, 1] = bad
        c.table[1, 0] = bad
        out = ab.DeviceArray.empty((2, 2, 64), ab.F32)
        c.kv.decode_attention(up(ab, q, ab.F32), out, ab.DeviceArray.from_host(c.table, ab.I32), ab.DeviceArray.from_host([48, 16], ab.I32), 0.1)
        with pytest.raises(ab.AtlasError, match="page outside"):
            c.kv.ctx.poll_device_error()
        got = out.download()
        c.table = np.stack([good[0][[0, 2, 1]], good[1]])                    # the two pages that are left, side by side
        want, tol = decode_by_hand(c, q, 0.1, 0, [32, 0])
        assert np.all(np.abs(got - want) <= tol)


def test_decode_repeats_bit_for_bit(ab):
    rng = np.random.default_rng(10)
    c = Cache(ab, rng, [4000, 1, 777, 2000], 2, 128, 32, 16)
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    a = check_decode(ab, c, 8, 0.09, 0, q=q)
    for _ in range(3):
        assert np.array_equal(a, check_decode(ab, c, 8, 0.09, 0, q=q, workspace=c.kv.workspace()))


# ── prompt attention ─────────────────────────────────────────────────────────────
def prompt_by_hand(q, k, v, cu_q, cu_k, scale, window, f16):
    u = 2.0 ** -11 if f16 else 2.0 ** -8
    nh, n_kv, hd = q.shape[1], k.shape[1], q.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(len(cu_q) - 1):
        lq, lk = cu_q[b + 1] - cu_q[b], cu_k[b + 1] - cu_k[b]
        if lq <= 0:
            continue
        i, j = np.arange(lq)[:, None] + lk - lq, np.arange(max(lk, 0))[None, :]
        seen = (j <= i) & ((i - j < window) if window else True)
        any_ = seen.any(1) if lk > 0 else np.zeros(lq, bool)
        for h in range(nh):
            kh = h // (nh // n_kv)
            x, y, z = (t.astype(np.float64) for t in (q[cu_q[b]:cu_q[b + 1], h], k[cu_k[b]:cu_k[b + 1], kh], v[cu_k[b]:cu_k[b + 1], kh]))
            if lk <= 0:
                continue
            a = np.where(seen, x @ y.T * scale, -np.inf)
            e = 2.0 ** -18 * abs(scale) * (np.where(seen, np.abs(x) @ np.abs(y).T, 0)).max(1, keepdims=True)
            m = np.where(any_, a.max(1, initial=-np.inf), 0)[:, None]
            p = np.exp(a - m)
            l = np.where(any_[:, None], p.sum(1, keepdims=True), 1)
            o = (p / l) @ z
            out[cu_q[b]:cu_q[b + 1], h] = o
            t = u * np.abs(o) + (u + 2 * e + 2.0 ** -16) * ((p / l) @ np.abs(z)) * (1 + u)
            if f16:
                t = t + 2.0 ** -24 * (seen @ np.abs(z)) / l
            tol[cu_q[b]:cu_q[b + 1], h] = t
    return out, tol + 1e-30


def prompt_case(ab, lq, lk, nh, n_kv, hd, window, dtype_name, rng, fused=False, scale=None):
    dtype = getattr(ab, dtype_name)
    cast = bf16 if dtype_name == "BF16" else (lambda x: x.astype(np.float16).astype(np.float32))
    cu_q, cu_k = np.concatenate([[0], np.cumsum(lq)]), np.concatenate([[0], np.cumsum(lk)])
    q, k, v = cast(rng.standard_normal((cu_q[-1], nh, hd)).astype(np.float32)), cast(rows(rng, cu_k[-1], n_kv, hd)), cast(rows(rng, cu_k[-1], n_kv, hd))
    if fused:
        w = [nh * hd, n_kv * hd, n_kv * hd]
        buf = up(ab, np.concatenate([x.reshape(len(x), -1) for x in (q, k, v)], 1), dtype)
        ds, at = [], 0
        for x, n in zip((q, k, v), w):
            ds.append(buf.columns(at, x.shape, (sum(w), hd, 1)))
            at += n
    else:
        ds = [up(ab, x, dtype) for x in (q, k, v)]
    out = up(ab, np.full(q.shape, 7.0), dtype)
    scale = 1 / math.sqrt(hd) if scale is None else scale
    ab.prompt_attention(*ds, out, ab.DeviceArray.from_host(cu_q, ab.I32), ab.DeviceArray.from_host(cu_k, ab.I32), scale, window)
    want, tol = prompt_by_hand(q, k, v, cu_q, cu_k, scale, window, dtype_name == "F16")
    got = down(ab, out)
    err = np.abs(got - want) / tol
    assert np.all(err <= 1), (float(err.max()), np.argwhere(err > 1)[:5])
    assert ab.Context.default().poll_device_error() == 0
    return got


@pytest.mark.parametrize("dtype_name", ["BF16", "F16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300])
def test_prompt_lengths(ab, dtype_name, hd, n):
    prompt_case(ab, [n], [n], 2, 1, hd, 0, dtype_name, np.random.default_rng(n), fused=n % 2 == 1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 128, 129, 200, 1000])
def test_prompt_windows(ab, hd, window):
    prompt_case(ab, [300, 1, 130], [300, 1, 130], 2, 2, hd, window, "BF16", np.random.default_rng(window))
    prompt_case(ab, [64, 129], [400, 258], 2, 1, hd, window, "F16", np.random.default_rng(window))


@pytest.mark.parametrize("nh,n_kv", [(1, 1), (4, 4), (8, 2), (6, 2), (8, 1), (5, 5), (12, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_heads(ab, nh, n_kv, hd):
    rng = np.random.default_rng(nh)
    prompt_case(ab, [70, 3, 140], [70, 3, 140], nh, n_kv, hd, 0, "BF16", rng, fused=True)


@pytest.mark.parametrize("dtype_name", ["BF16", "F16"])
def test_prompt_packs(ab, dtype_name):
    """Empty sequences, prefixes that are cached already, more queries than keys (the first see nothing), no keys at all."""
    rng = np.random.default_rng(12)
    prompt_case(ab, [0, 5, 0, 200, 1, 40, 7], [0, 5, 0, 200, 300, 517, 7], 4, 2, 128, 0, dtype_name, rng)
    prompt_case(ab, [300, 20, 9, 4], [170, 3, 0, 4], 2, 1, 128, 0, dtype_name, rng)
    prompt_case(ab, [300, 20, 9, 4], [170, 3, 0, 4], 2, 1, 64, 50, dtype_name, rng)
    prompt_case(ab, [3] * 200, [3] * 200, 2, 2, 64, 0, dtype_name, rng)
    prompt_case(ab, [0, 3, 0], [0, 0, 0], 2, 2, 64, 0, dtype_name, rng)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_long(ab, hd):
    prompt_case(ab, [1500, 700], [1500, 2100], 2, 1, hd, 0, "BF16", np.random.default_rng(2))
    prompt_case(ab, [1500, 700], [1500, 2100], 2, 1, hd, 333, "BF16", np.random.default_rng(2))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_prompt_scales(ab, scale):
    prompt_case(ab, [200, 30], [260, 30], 2, 2, 128, 0, "BF16", np.random.default_rng(3), scale=scale)


def test_prompt_scores_that_grow_along_the_row(ab):
    """The running maximum rises by a lot with nearly every tile: sums and outputs have to be brought down each time."""
    n, hd = 700, 128
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal((n, 1, hd)).astype(np.float32) for _ in range(3))
    q[..., 0] = 8.0
    k[..., 0] = np.arange(n)[:, None] / 4.0
    q, k, v = bf16(q), bf16(k), bf16(v)
    out = ab.DeviceArray.empty((n, 1, hd), ab.BF16)
    cu = ab.DeviceArray.from_host([0, n], ab.I32)
    for s in (0.088, -0.088):
        ab.prompt_attention(*(up(ab, x, ab.BF16) for x in (q, k, v)), out, cu, cu, s)
        want, tol = prompt_by_hand(q, k, v, [0, n], [0, n], s, 0, False)
        assert np.all(np.abs(down(ab, out) - want) <= tol)


def poisoned(ab, hd, lens, total, bad, window, value):
    """Outputs with `value` in K and V at the rows `bad`; what they would be without, in 64 bits, and how far off the format lets them
    be (a row that is taken again because its tile held the value rounds differently, within the same bound).  Rows from lens' sum
    to total are padding."""
    rng = np.random.default_rng(5)
    nh = 2
    q, k, v = (bf16(rng.standard_normal((total, nh, hd)).astype(np.float32)) for _ in range(3))
    cu = np.concatenate([[0], np.cumsum(lens)])
    want, tol = prompt_by_hand(q, k, v, cu, cu, 0.1, window, False)
    k[bad] = value
    v[bad] = value
    out = up(ab, np.full(q.shape, 7.0), ab.BF16)
    cu = ab.DeviceArray.from_host(cu, ab.I32)
    ab.prompt_attention(*(up(ab, t, ab.BF16) for t in (q, k, v)), out, cu, cu, 0.1, window)
    got = down(ab, out)
    with np.errstate(invalid="ignore"):
        return got, np.abs(got - want) <= tol


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_hidden_rows_do_not_reach_a_query(ab, hd, value):
    # a row in the middle of the second sequence: the queries before it, and the other sequences, do not see it
    lens, first = [130, 300, 40], 130
    got, fine = poisoned(ab, hd, lens, 470, [first + 150], 0, value)
    assert fine[:first + 150].all() and fine[430:].all()
    # a query that sees it: NaN as soon as a score is NaN or +inf (inf · q has either sign: q·k is NaN for mixed signs)
    assert np.isnan(got[first + 150:430]).all()
    # with a window the queries far behind it do not see it either
    got, fine = poisoned(ab, hd, lens, 470, [first + 20], 30, value)
    assert fine[np.r_[0:first + 20, first + 50:470]].all() and np.isnan(got[first + 20:first + 50]).all()
    # padding behind the last sequence, never written
    got, fine = poisoned(ab, hd, lens, 500, list(range(470, 500)), 0, value)
    assert fine[:470].all() and (got[470:] == 7).all()


def test_prompt_outputs_may_be_strided(ab):
    rng = np.random.default_rng(6)
    n, nh, hd = 90, 2, 64
    q = bf16(rng.standard_normal((n, nh, hd)).astype(np.float32))
    qd = up(ab, q, ab.BF16)
    buf = up(ab, np.full((n, 3 * nh * hd), 7.0), ab.BF16)
    cu = ab.DeviceArray.from_host([0, n], ab.I32)
    ab.prompt_attention(qd, qd, qd, buf.columns(nh * hd, (n, nh, hd), (3 * nh * hd, hd, 1)), cu, cu, 0.1)
    want, tol = prompt_by_hand(q, q, q, [0, n], [0, n], 0.1, 0, False)
    got = down(ab, buf).reshape(n, 3, nh, hd)
    assert np.all(np.abs(got[:, 1] - want) <= tol) and (got[:, [0, 2]] == 7).all()
    # heads outermost: [heads, rows, hd]
    flat = up(ab, np.ascontiguousarray(q.transpose(1, 0, 2)), ab.BF16)
    view = flat.columns(0, (n, nh, hd), (hd, n * hd, 1))
    out = up(ab, np.zeros((nh, n, hd)), ab.BF16)
    ab.prompt_attention(view, view, view, out.columns(0, (n, nh, hd), (hd, n * hd, 1)), cu, cu, 0.1)
    assert np.all(np.abs(down(ab, out).transpose(1, 0, 2) - want) <= tol)


def test_prompt_of_the_largest_batch(ab):
    rng = np.random.default_rng(43)
    lens = rng.integers(0, 4, 4096).tolist()
    prompt_case(ab, lens, lens, 1, 1, 64, 0, "BF16", rng)


def test_prompt_prefix_arrays_are_cut_to_the_buffers(ab):
    """Numbers outside the buffers and decreasing ones: no row is read or written that is not there."""
    rng = np.random.default_rng(44)
    q = bf16(rng.standard_normal((40, 2, 64)).astype(np.float32))
    buf = up(ab, np.full((80, 2, 64), 7.0), ab.BF16)
    qd, out = up(ab, q, ab.BF16), buf.columns(20 * 128, (40, 2, 64), (128, 64, 1))
    for cu_q, cu_k in (([-5, 30, 1000], [-1000, 30, 70]), ([0, 40, 10], [0, 40, 40]), ([2147483647, -2147483648, 7], [0, 0, 0])):
        ab.prompt_attention(qd, qd, qd, out, ab.DeviceArray.from_host(cu_q, ab.I32), ab.DeviceArray.from_host(cu_k, ab.I32), 0.1)
        got = down(ab, buf)
        assert (got[:20] == 7).all() and (got[60:] == 7).all()
    assert ab.Context.default().poll_device_error() == 0
    ab.prompt_attention(qd, qd, qd, out, ab.DeviceArray.from_host([-5, 30, 1000], ab.I32), ab.DeviceArray.from_host([-1000, 30, 70], ab.I32), 0.1)
    want, tol = prompt_by_hand(q, q, q, [0, 30, 40], [0, 30, 40], 0.1, 0, False)
    assert np.all(np.abs(down(ab, buf)[20:60] - want) <= tol)


def test_prompt_rows_outside_every_sequence_stay(ab):
    rng = np.random.default_rng(7)
    q = bf16(rng.standard_normal((60, 1, 64)).astype(np.float32))
    qd, out = up(ab, q, ab.BF16), up(ab, np.full((60, 1, 64), 7.0), ab.BF16)
    cu = ab.DeviceArray.from_host([5, 25, 25, 40], ab.I32)
    ab.prompt_attention(qd, qd, qd, out, cu, cu, 0.1)
    want, tol = prompt_by_hand(q, q, q, [5, 25, 25, 40], [5, 25, 25, 40], 0.1, 0, False)
    got = down(ab, out)
    assert (got[:5] == 7).all() and (got[40:] == 7).all() and np.all(np.abs(got - want)[5:40] <= tol[5:40])


# ── the step as a whole ──────────────────────────────────────────────────────────
def test_a_prompt_and_the_tokens_after_it(ab):
    """Two prompts are planned, stored and attended, then five decode steps with lengths of their own; a later prompt reads its cached
    prefix back.  Everything the cache holds is known, so every output has its value in 64 bits."""
    rng = np.random.default_rng(21)
    nh, n_kv, hd, page, n_pages, width, group = 4, 2, 128, 16, 40, 12, 32
    kv = ab.PagedKvCache(n_pages, page, n_kv, hd, group=group)
    i32 = lambda x: ab.DeviceArray.from_host(x, ab.I32)                   # noqa: E731
    free = rng.permutation(n_pages)
    table = i32(np.full((2, width), -1))
    lens_now, stored = [0, 0], [[np.zeros((0, n_kv, hd))] * 2 for _ in range(2)]
    scale = 1 / math.sqrt(hd)

    def step(fresh, free):
        n = sum(fresh)
        cu, lens, slots, pos, status = (i32(np.zeros(m)) for m in (3, 2, n + 1, n + 1, 3))      # one padding row
        ab.page_plan(i32(lens_now), i32(fresh), i32(free), table, cu, lens, slots, pos, status, page_size=page, n_pages=n_pages)
        k, v = bf16(rows(rng, n + 1, n_kv, hd)), bf16(rows(rng, n + 1, n_kv, hd))
        kv.append(up(ab, k, ab.BF16), up(ab, v, ab.BF16), slots)
        taken, missing, bad = status.download()
        assert missing == bad == 0
        at = 0
        for b, m in enumerate(fresh):
            stored[b] = [np.concatenate([old, held(x[at:at + m], group)]) for old, x in zip(stored[b], (k, v))]
            lens_now[b] += m
            at += m
        assert lens.download().tolist() == lens_now
        return free[taken:], cu, lens, slots, k, v

    free, cu, lens, slots, k, v = step([37, 90], free)
    q = bf16(rng.standard_normal((128, nh, hd)).astype(np.float32))
    out = up(ab, np.full(q.shape, 7.0), ab.BF16)
    ab.prompt_attention(up(ab, q, ab.BF16), up(ab, k, ab.BF16), up(ab, v, ab.BF16), out, cu, cu, scale)
    want, tol = prompt_by_hand(q, k, v, [0, 37, 127], [0, 37, 127], scale, 0, False)
    got = down(ab, out)
    assert np.all(np.abs(got - want)[:127] <= tol[:127]) and (got[127] == 7).all()
    for _ in range(5):
        free, cu, lens, slots, k, v = step([1, 1], free)
        c = Cache.__new__(Cache)
        c.page, c.table = 1, np.arange(2 * 400).reshape(2, 400)
        c.k, c.v = (np.concatenate([np.concatenate([stored[b][i], np.zeros((400 - lens_now[b], n_kv, hd))]) for b in range(2)]) for i in (0, 1))
        q = rng.standard_normal((2, nh, hd)).astype(np.float32)
        out = ab.DeviceArray.empty((2, nh, hd), ab.F32)
        kv.decode_attention(up(ab, q, ab.F32), out, table, lens, scale)
        want, tol = decode_by_hand(c, q, scale, 0, lens_now)
        assert np.all(np.abs(out.download() - want) <= tol)
    # the second request goes on with a prompt of 30: its prefix comes back out of the cache
    had = lens_now[1]
    free, cu, lens, slots, k, v = step([0, 30], free)
    t = table.download()[1]
    all_slots = i32([t[p // page] * page + p % page for p in range(had + 30)])
    ko, vo = ab.DeviceArray.empty((had + 30, n_kv, hd), ab.BF16), ab.DeviceArray.empty((had + 30, n_kv, hd), ab.BF16)
    kv.read(all_slots, ko, vo)
    kb, vb = bf16(stored[1][0]), bf16(stored[1][1])
    assert np.array_equal(down(ab, ko), kb) and np.array_equal(down(ab, vo), vb)
    q = bf16(rng.standard_normal((30, nh, hd)).astype(np.float32))
    out = ab.DeviceArray.empty((30, nh, hd), ab.BF16)
    ab.prompt_attention(up(ab, q, ab.BF16), ko, vo, out, i32([0, 30]), i32([0, had + 30]), scale)
    want, tol = prompt_by_hand(q, kb, vb, [0, 30], [0, had + 30], scale, 0, False)
    assert np.all(np.abs(down(ab, out) - want) <= tol)
    assert kv.ctx.poll_device_error() == 0


def test_a_captured_step_follows_the_lengths(ab):
    """plan → append → decode captured once on the context's stream, replayed with other lengths, rows and queries; two graphs with
    workspaces of their own replayed on two streams at once."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(30)
    nh, n_kv, hd, page, n_pages, width, b = 8, 2, 128, 16, 64, 20, 3
    kv = ab.PagedKvCache(n_pages, page, n_kv, hd)
    ctx = kv.ctx
    dev = torch.device("cuda", ctx.device)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=dev)       # noqa: E731
    order = rng.permutation(n_pages)
    lens0 = np.array([200, 17, 90])
    table_np = np.full((b, width), -1)
    at = 0
    for i, n in enumerate(lens0):
        m = -(-n // page)
        table_np[i, :m] = order[at:at + m]
        at += m
    table, free = i32(table_np), i32(order[at:])
    k0, v0 = rows(rng, n_pages * page, n_kv, hd), rows(rng, n_pages * page, n_kv, hd)
    cached, fresh = i32(lens0), i32([1, 1, 1])
    cu, lens, slots, pos, status = i32(np.zeros(b + 1)), i32(np.zeros(b)), i32(np.zeros(b)), i32(np.zeros(b)), i32(np.zeros(3))
    k, v, q = (torch.zeros(b, m, hd, device=dev) for m in (n_kv, n_kv, nh))
    outs = [torch.zeros(b, nh, hd, device=dev) for _ in range(2)]
    spaces = [torch.zeros((kv.workspace_bytes + 3) // 4, dtype=torch.int32, device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    kv.append(up(ab, k0, ab.F32), up(ab, v0, ab.F32), ab.DeviceArray.from_host(np.arange(n_pages * page), ab.I32))
    ctx.sync()
    s = torch.cuda.ExternalStream(ctx.stream, device=dev)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
            if i == 0:
                ab.page_plan(cached, fresh, free, table, cu, lens, slots, pos, status, page_size=page, n_pages=n_pages, ctx=ctx)
                kv.append(k, v, slots)
            kv.decode_attention(q, outs[i], table, lens, 0.09, 0, spaces[i])
        graphs.append(g)
    kh, vh = held(k0, 32), held(v0, 32)
    for step in range(3):
        kn, vn, qn = rows(rng, b, n_kv, hd), rows(rng, b, n_kv, hd), rng.standard_normal((b, nh, hd)).astype(np.float32)
        for d, x in ((k, kn), (v, vn), (q, qn)):
            d.copy_(torch.from_numpy(x))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graphs[0].replay()
        torch.cuda.synchronize()
        assert status.cpu().tolist()[1:] == [0, 0]
        sl = slots.cpu().numpy()
        kh[sl], vh[sl] = held(kn, 32), held(vn, 32)
        c = Cache.__new__(Cache)
        c.page, c.table, c.k, c.v = page, table.cpu().numpy(), kh, vh
        want, tol = decode_by_hand(c, qn, 0.09, 0, (lens0 + 1).tolist())
        assert np.all(np.abs(outs[0].cpu().numpy() - want) <= tol)
        # both graphs' attention, one on a stream of its own (graph 1 reads what graph 0's last replay left)
        other = torch.cuda.Stream(device=dev)
        with torch.cuda.stream(other):
            graphs[1].replay()
        with torch.cuda.stream(s):
            graphs[0].replay()
        torch.cuda.synchronize()
        assert np.array_equal(outs[0].cpu().numpy(), outs[1].cpu().numpy())
        used = int(status.cpu()[0])
        free.copy_(torch.cat([free[used:], free[:used]]))
        lens0 = lens0 + 1
        cached.copy_(i32(lens0))
        torch.cuda.synchronize()
    del graphs


def test_a_captured_prompt_follows_the_arrays(ab):
    """Prompt attention captured once, replayed with other rows and other sequence boundaries."""
    torch = pytest.importorskip("torch")
    ctx = ab.Context.default()
    dev = torch.device("cuda", ctx.device)
    s = torch.cuda.ExternalStream(ctx.stream, device=dev)
    n, nh, n_kv, hd = 300, 4, 2, 128
    q, k, v = (torch.zeros(n, m, hd, dtype=torch.bfloat16, device=dev) for m in (nh, n_kv, n_kv))
    out = torch.zeros_like(q)
    cu = torch.zeros(4, dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s, capture_error_mode="thread_local"):
        ab.prompt_attention(q, k, v, out, cu, cu, 0.09)
    rng = np.random.default_rng(51)
    for bounds in ([0, 300, 300, 300], [0, 1, 140, 290], [0, 0, 0, 0], [0, 128, 256, 300]):
        x = [bf16(rng.standard_normal(tuple(t.shape)).astype(np.float32)) for t in (q, k, v)]
        for t, y in zip((q, k, v), x):
            t.copy_(torch.from_numpy(y))
        out.fill_(7.0)
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        want, tol = prompt_by_hand(*x, bounds, bounds, 0.09, 0, False)
        got = out.float().cpu().numpy()
        assert np.all(np.abs(got - want)[:bounds[-1]] <= tol[:bounds[-1]]) and (got[bounds[-1]:] == 7).all()
    assert ctx.poll_device_error() == 0
    del g


def test_two_contexts_do_not_meet(ab):
    """A cache of one context is refused by another; each context's stream carries its own calls."""
    other = ab.Context(0)
    kv = ab.PagedKvCache(2, 16, 1, 64)
    from atlas_b200 import _ffi
    d = ab.DeviceArray.from_host(np.zeros(64), ab.F32)
    i = ab.DeviceArray.from_host([0], ab.I32)
    attn = lambda w, n: _ffi.PAGED_ATTN.pack(d.ptr, d.ptr, i.ptr, i.ptr, w, n, 1, 1, 1, 0, 0.1)      # noqa: E731
    rc = _ffi.lib().atlasx_pagedkv_decode_attention(other.handle, kv._h, attn(0, 0))
    assert rc == -1 and b"another context" in _ffi.lib().atlasx_last_error()
    rc = _ffi.lib().atlasx_pagedkv_append(other.handle, kv._h, _ffi.PAGED_ROWS.pack(d.ptr, d.ptr, i.ptr, 64, 64, 64, 64, 0, 1))
    assert rc == -1 and b"another context" in _ffi.lib().atlasx_last_error()
    rc = _ffi.lib().atlasx_pagedkv_decode_attention(kv.ctx.handle, kv._h, attn(d.ptr, 8))
    assert rc == -1 and b"workspace" in _ffi.lib().atlasx_last_error()
    with pytest.raises(ab.AtlasError, match="multiple"):
        ab.PagedKvCache(2, 16, 2, 64).decode_attention(ab.DeviceArray.empty((1, 3, 64), ab.F32), ab.DeviceArray.empty((1, 3, 64), ab.F32),
                                                       ab.DeviceArray.from_host([[0]], ab.I32), i, 0.1)
    other.close()
