"""The cache in 8 bits: written, read back and attended to, against float64 by the layout's definition."""
import numpy as np
import pytest

from plain import cache_q8_plain as P

pytestmark = pytest.mark.gpu

# half a step of a rounding, relative to the value
HALF = {"bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
# query heads, key heads, channels, tokens of a page
SHAPES = [(8, 4, 256, 16), (4, 2, 128, 32), (12, 12, 64, 16), (20, 4, 96, 48), (32, 1, 128, 64), (5, 5, 80, 16), (34, 2, 40, 16), (3, 1, 7, 16),
          (18, 1, 192, 128), (6, 3, 200, 16), (32, 2, 256, 16)]


@pytest.fixture(scope="module")
def rt():
    from zse_amd.runtime.device import Runtime
    return Runtime.get()


def up(rt, x, dtype):
    from zse_amd.weights.safetensors import f32_to_bf16_bits
    x = np.ascontiguousarray(x, np.float32)
    return rt.upload(f32_to_bf16_bits(x), "bfloat16") if dtype == "bfloat16" else rt.upload(x)


def rounded(x, dtype):
    """x as the activations' type holds it, in float32."""
    from zse_amd.weights.safetensors import bf16_bits_to_f32, f32_to_bf16_bits
    x = np.ascontiguousarray(x, np.float32)
    return bf16_bits_to_f32(f32_to_bf16_bits(x)).reshape(x.shape) if dtype == "bfloat16" else x


def device_cache(rt, c):
    return rt.upload(c.k), rt.upload(c.v), rt.upload(c.scales)


def random_cache(rng, pages, nkv, hd, bs, form):
    """Every byte of the cache is what a random head leaves there, padding included."""
    c = P.Cache(pages, nkv, hd, bs, form)
    for x in (c.k, c.v):
        b = rng.integers(0, 256, x.shape).astype(np.uint8)
        b[b == 0x80] = 1
        x[...] = np.where(b & 127 == 127, b & 0x80 | 5, b) if form else b
    c.scales[...] = np.exp(rng.standard_normal(c.scales.shape) * 0.4) / P.TOP[form]
    return c


def tables(rng, lens, bs, width):
    need = [-(-n // bs) for n in lens]
    ids = list(1 + rng.permutation(sum(need)))
    table = np.full((len(lens), width), -1, np.int32)
    for r, n in enumerate(need):
        table[r, :n] = [ids.pop() for _ in range(n)]
    return table, sum(need) + 1


# ------------------------------------------------------------------ written
def write(rt, dtype, cache, rows, positions, slots, inv_freq, rotary, nh, planes=None, ld=None, in_place=False, tokens=None):
    k = rt.kernels(dtype)
    T, width = len(positions), (nh + 2 * cache.nkv) * cache.hd
    ld = ld or width
    held = np.zeros((T, ld), np.float32)
    held[:, :width] = rows
    X = up(rt, held, dtype)
    Q = X if in_place else up(rt, np.full((T, nh * cache.hd), 7.0), dtype)
    KC, VC, SC = device_cache(rt, cache)
    PL = rt.upload(planes) if planes is not None else None
    POS, SL = rt.upload(np.asarray(positions, np.int32)), rt.upload(np.asarray(slots, np.int32)) if slots is not None else None
    F = rt.upload(np.asarray(inv_freq, np.float32)) if rotary else None
    k.zk_rope_cache_write_q8(X.ptr, ld, PL.ptr if PL else None, len(planes) if PL else 0, Q.ptr, ld if in_place else nh * cache.hd, POS.ptr,
                             SL.ptr if SL else None, F.ptr if F else None, rotary, KC.ptr, VC.ptr, SC.ptr, T, nh, cache.nkv, cache.hd,
                             cache.bs, cache.pages, cache.form, rt.stream)
    got = P.Cache(cache.pages, cache.nkv, cache.hd, cache.bs, cache.form)
    got.k, got.v, got.scales = rt.download(KC), rt.download(VC), rt.download(SC)
    return rt.download_f32(Q)[:, :nh * cache.hd], got


def check_written(before, got, q, x, positions, slots, inv_freq, rotary, nh, dtype):
    """x: the rows in float64 as the kernel reads them."""
    nkv, hd, form = before.nkv, before.hd, before.form
    T = len(positions)
    x = x.reshape(T, nh + 2 * nkv, hd)
    turned = P.rotate(x[:, :nh + nkv], positions, inv_freq, rotary)
    # a turned value is off by roundings of its two products, of sine and cosine (two steps each) and of the sum: eight half steps
    # of 32 bits of |a| + |b|, and |a| + |b| is at most twice the larger of the pair's two results, which is at most the head's largest
    off = 8 * 2.0 ** -24 * 2
    near = np.abs(turned).max(axis=-1, keepdims=True) * off
    want_q = turned[:, :nh].reshape(T, -1)
    tol = HALF[dtype] * np.abs(want_q) * 1.01 + np.repeat(near[:, :nh, 0], hd, axis=1)
    assert (np.abs(q - want_q) <= tol).all()
    seen = np.zeros(before.scales.shape, bool)
    for t in range(T):
        if slots is None or slots[t] < 0 or slots[t] // before.bs >= before.pages:
            continue
        page, at = divmod(int(slots[t]), before.bs)
        for h in range(nkv):
            for values, row in ((False, turned[t, nh + h]), (True, x[t, nh + nkv + h])):
                seen[page, h, int(values), at] = True
                scale = np.abs(row).max() / P.TOP[form]
                held = np.float64(got.scales[page, h, int(values), at])
                assert abs(held - scale) <= scale * (off + 2.0 ** -23), (t, h, values)
                codes = P.numbers(got.codes_at(page, h, at, values), form)
                assert np.isfinite(codes).all() and (np.abs(codes).max() == P.TOP[form] or scale == 0)
                err = np.abs(codes * held - row)
                # half a step of the codes, and what the value before the rounding is off by: the row's error and three roundings
                assert (err <= P.half_step(row, held, form) * (1 + 2.0 ** -18) + np.abs(row).max() * (off + 2.0 ** -21)).all(), (t, h, values)
    assert np.array_equal(got.scales[~seen], before.scales[~seen])
    for p, h, s, at in np.argwhere(~seen):
        assert np.array_equal(got.codes_at(p, h, at, bool(s)), before.codes_at(p, h, at, bool(s))), (p, h, s, at)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("nh,nkv,hd,bs", SHAPES)
def test_written(rt, nh, nkv, hd, bs, form, dtype):
    """Portions that begin inside a piece and inside a group of four, and end so; single tokens; tokens that are not stored."""
    rng = np.random.default_rng(hd + form)
    lens, new = [37, 21, 90, 1, 50], [37, 6, 23, 1, 1]
    table, pages = tables(rng, lens, bs, 8)
    before = random_cache(rng, pages, nkv, hd, bs, form)
    positions = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)])
    slots = np.concatenate([table[r, np.arange(n - m, n) // bs] * bs + np.arange(n - m, n) % bs for r, (n, m) in enumerate(zip(lens, new))])
    slots[[3, 40]] = -1
    slots[5] = pages * bs + 3
    positions[3] = -1
    T = len(positions)
    rotary = hd // 2 * 2
    inv_freq = (10000.0 ** (-np.arange(rotary // 2) * 2.0 / rotary)).astype(np.float32)
    rows = rounded(rng.standard_normal((T, (nh + 2 * nkv) * hd)) * np.exp(rng.standard_normal((T, 1))), dtype)
    q, got = write(rt, dtype, before, rows, positions, slots, inv_freq, rotary, nh)
    check_written(before, got, q, rows.astype(np.float64), positions, slots, inv_freq, rotary, nh, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("what", ["part", "none", "in_place", "stride", "sums", "queries", "no_slots", "far", "one", "many"])
def test_written_otherwise(rt, what, dtype):
    rng = np.random.default_rng(len(what))
    nh, nkv, hd, bs, form = 6, 0 if what == "queries" else 2, 136, 16, 1
    T = {"one": 1, "many": 3000}.get(what, 45)
    pages = T // bs + 2
    before = random_cache(rng, pages, max(nkv, 1), hd, bs, form)
    before.nkv = nkv
    rotary = {"part": 34, "none": 0}.get(what, hd)
    inv_freq = (10000.0 ** (-np.arange(rotary // 2) * 2.0 / max(rotary, 1))).astype(np.float32)
    positions = np.arange(T) + (1000000 if what == "far" else 3)
    slots = None if what in ("queries", "no_slots") else bs + 5 + np.arange(T)
    rows = rounded(rng.standard_normal((T, (nh + 2 * nkv) * hd)), dtype)
    planes = None
    if what == "sums":
        planes = rng.standard_normal((3, T, rows.shape[1])).astype(np.float32)
        rows = rounded(planes[0] + planes[1] + planes[2], dtype)
    q, got = write(rt, dtype, before, rows, positions, slots, inv_freq, rotary, nh, planes=planes, in_place=what == "in_place",
                   ld=rows.shape[1] + 3 if what in ("stride", "in_place") else None)
    if what == "queries":
        before.nkv = 1
        assert np.array_equal(got.k, before.k) and np.array_equal(got.scales, before.scales)
        want = P.rotate(rows.astype(np.float64).reshape(T, nh, hd), positions, inv_freq, rotary).reshape(T, -1)
        assert np.abs(q - want).max() <= np.abs(want).max() * (HALF[dtype] + 2.0 ** -19)
        return
    check_written(before, got, q, rows.astype(np.float64), positions, slots, inv_freq, rotary, nh, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hd,rotary", [(64, 8), (64, 48), (96, 64), (256, 64), (256, 248), (40, 16), (72, 10)])
@pytest.mark.parametrize("planes", [0, 1, 2, 4, 5, 6, 7])
def test_written_from_planes_and_turned_in_part(rt, planes, hd, rotary, dtype):
    """The planes of a split product in the order of their numbers; heads of which a part turns, in fours of channels and not."""
    rng = np.random.default_rng(planes + rotary)
    nh, nkv, bs, form, T = 5, 2, 16, planes % 2, 11
    before = random_cache(rng, 4, nkv, hd, bs, form)
    inv_freq = (10000.0 ** (-np.arange(rotary // 2) * 2.0 / rotary)).astype(np.float32)
    positions, slots = np.arange(T) + 900, np.concatenate([21 + np.arange(9), [40, 60]])
    parts = rng.standard_normal((max(planes, 1), T, (nh + 2 * nkv) * hd)).astype(np.float32)
    rows = parts[0]
    for x in parts[1:]:
        rows = rows + x
    rows = rounded(rows, dtype)
    q, got = write(rt, dtype, before, rows, positions, slots, inv_freq, rotary, nh, planes=parts if planes else None)
    check_written(before, got, q, rows.astype(np.float64), positions, slots, inv_freq, rotary, nh, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", [0, 1])
def test_written_from_zeros_and_what_is_not_finite(rt, form, dtype):
    rng = np.random.default_rng(2)
    nh, nkv, hd, bs, T = 2, 3, 72, 16, 6
    before = random_cache(rng, 3, nkv, hd, bs, form)
    rows = rounded(rng.standard_normal((T, (nh + 2 * nkv) * hd)), dtype)
    x = rows.reshape(T, -1, hd)
    x[0, nh:] = 0.0
    x[1, nh:] *= 2.0 ** -110
    x[2, nh + 1, 11], x[2, nh + nkv + 1, 70] = np.inf, -np.inf
    x[3, nh + 2, 71], x[3, nh + nkv, 0] = np.nan, np.nan
    x[4, nh:] = rounded(x[4, nh:] * 2.0 ** 120, dtype)
    x[5, nh:] = rounded(x[5, nh:] * 2.0 ** -90, dtype)
    slots = 16 + np.arange(T)
    _, got = write(rt, dtype, before, rows, np.zeros(T, int), slots, np.zeros(hd // 2), hd, nh)
    for t in range(T):
        for h in range(nkv):
            for values in (False, True):
                row, s = x[t, nh + h + nkv * values].astype(np.float64), got.scales[1, h, int(values), t]
                codes = got.codes_at(1, h, t, values)
                if t < 2:
                    assert s == 0 and not codes.any()
                elif not np.isfinite(row).all():
                    assert np.isnan(s) and not codes.any()
                else:
                    assert (np.abs(P.numbers(codes, form) * np.float64(s) - row) <= P.half_step(row, np.float64(s), form) * 1.001 +
                            np.abs(row).max() * 2.0 ** -20).all()


# ------------------------------------------------------------------ read back
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("nh,nkv,hd,bs", SHAPES)
def test_read(rt, nh, nkv, hd, bs, form, dtype):
    """Bit for bit, transposed and in rows; pages that nobody sees, and slots behind the last token, whatever lies there."""
    rng = np.random.default_rng(hd + form)
    lens, new = [1, 40, 97, 0, 128, 200], [1, 40, 30, 0, 1, 17]
    width = -(-256 // bs)
    table, pages = tables(rng, lens, bs, width)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    for r, n in enumerate(lens):
        if n % bs:
            page = table[r, n // bs]
            c.scales[page, :, :, n % bs:] = np.nan
            for t in range(n % bs, bs):
                for h in range(nkv):
                    for values in (False, True):
                        c.put(page, h, t, values, 127, np.nan)
    table[4, 0] = -1
    table[5, 1] = pages
    k = rt.kernels(dtype)
    KC, VC, SC = device_cache(rt, c)
    TBL, CL = rt.upload(table), rt.upload(np.array(lens, np.int32))
    for window in (0, 1, 33):
        for starts in (True, False):
            n_new = new if starts else [1] * len(lens)
            QS = rt.upload(np.cumsum([0] + n_new).astype(np.int32)) if starts else None
            for transposed in (0, 1):
                shape = (pages, nkv, hd, bs) if transposed else (pages, nkv, bs, hd)
                K, V = up(rt, np.full((pages, nkv, bs, hd), 3.0), dtype), up(rt, np.full(shape, 3.0), dtype)
                k.zk_cache_read_q8(KC.ptr, VC.ptr, SC.ptr, TBL.ptr, width, QS.ptr if QS else None, CL.ptr, K.ptr, V.ptr, len(lens), 200, window,
                                   nkv, hd, bs, pages, transposed, form, rt.stream)
                want = np.full((2, pages, nkv, bs, hd), 3.0, np.float32)
                for r, n in enumerate(lens):
                    first = max(0, n - n_new[r] + 1 - window) // bs if window else 0
                    for j in range(first, -(-n // bs)):
                        if not 0 <= table[r, j] < pages:
                            continue
                        want[:, table[r, j]] = 0.0
                        for t in range(min(bs, n - j * bs)):
                            for h in range(nkv):
                                for values in (0, 1):
                                    want[values, table[r, j], h, t] = c.row(table[r, j], h, t, bool(values)).astype(np.float32)
                got_v = rt.download_f32(V)
                assert np.array_equal(rt.download_f32(K), rounded(want[0], dtype)), (window, starts)
                assert np.array_equal(got_v.swapaxes(2, 3) if transposed else got_v, rounded(want[1], dtype)), (window, starts)


# ------------------------------------------------------------------ attended to
def attend(rt, dtype, c, q, table, lens, max_ctx, nh, scale, cap, window, q_stride=None, table_dev=None):
    k = rt.kernels(dtype)
    R, width = table.shape
    q_stride = q_stride or nh * c.hd
    held = np.zeros((R, q_stride), np.float32)
    held[:, :nh * c.hd] = q.reshape(R, -1)
    Q, TBL, CL = up(rt, held, dtype), rt.upload(table), rt.upload(np.asarray(lens, np.int32))
    KC, VC, SC = device_cache(rt, c)
    room = k.zk_attention_q8_workspace(R, nh, c.hd, max_ctx, width * c.bs)
    WS = rt.upload(np.full((room // 4 + 64,), np.nan, np.float32))
    OUT = up(rt, np.full((R + 1, nh * c.hd), 5.0), dtype)
    k.zk_attention_q8(Q.ptr, q_stride, KC.ptr, VC.ptr, SC.ptr, TBL.ptr, width, CL.ptr, OUT.ptr, R, max_ctx, nh, c.nkv, c.hd, c.bs, c.pages,
                      scale, cap, window, c.form, WS.ptr, room, rt.stream)
    got = rt.download_f32(OUT)
    assert (got[R] == 5.0).all()
    assert np.isnan(rt.download(WS)[-(-room // 4):]).all()
    return got[:R].reshape(R, nh, c.hd)


def check_attended(c, got, q, table, lens, nh, scale, cap, window, dtype):
    for r, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        keys, values = c.rows(table[r], first, n, False), c.rows(table[r], first, n, True)
        want, spread, most = P.attention(q[r].astype(np.float64), keys, values, scale, cap)
        # a score is off by hd roundings of its sum of |q| |k|, and by four of its own factors; the weights by twice that, by the
        # rounding of a weight to the activations' type and by those of exp and of a sum of n
        score = most * (c.hd + 8) * 2.0 ** -24 + (cap or 0.0) * 2.0 ** -20
        # and a weight below the smallest normal number of 32 bits may be zero, which takes up to 2^-126 of a value each
        tol = spread * (2 * score + HALF[dtype] + (n + 64) * 2.0 ** -23) + np.abs(want) * HALF[dtype] * 1.01
        tol = tol + (np.nanmax(np.abs(values)) * n * 2.0 ** -126 if np.isfinite(values).any() else 0.0)
        assert np.isfinite(got[r]).all() and (np.abs(got[r] - want) <= tol).all(), (r, n, np.abs(got[r] - want).max(), tol.min())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("form", [0, 1])
@pytest.mark.parametrize("nh,nkv,hd,bs", SHAPES)
def test_attended(rt, nh, nkv, hd, bs, form, dtype):
    rng = np.random.default_rng(hd + form)
    lens = [0, 1, 15, 16, 17, 33, 128, 129, 300, 513]
    table, pages = tables(rng, lens, bs, -(-640 // bs))
    c = random_cache(rng, pages, nkv, hd, bs, form)
    # whatever lies behind the last token: codes that are not numbers, scales that are not, and infinite ones
    for r, n in enumerate(lens):
        for t in range(n % bs, bs if n % bs else 0):
            for h in range(nkv):
                for values in (False, True):
                    c.put(table[r, n // bs], h, t, values, 255 if t % 2 else 127, np.inf if t % 3 else np.nan)
    q = rounded(rng.standard_normal((len(lens), nh, hd)) * 2, dtype)
    for cap, window in ((0.0, 0), (50.0, 0), (5.0, 100), (0.0, 1), (0.0, 300)):
        got = attend(rt, dtype, c, q, table, lens, 513, nh, hd ** -0.5, cap, window)
        check_attended(c, got, q, table, lens, nh, hd ** -0.5, cap, window, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("what", ["holes", "bad_pages", "none", "stride", "max_ctx", "no_ctx", "big_scores", "all_equal", "nan_key"])
def test_attended_otherwise(rt, what, dtype):
    rng = np.random.default_rng(len(what))
    nh, nkv, hd, bs, form = 8, 2, 64, 32, 1
    lens = [70, 500, 33, 200]
    table, pages = tables(rng, lens, bs, 20)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    q = rounded(rng.standard_normal((4, nh, hd)), dtype)
    scale, max_ctx, stride = 0.125, 512, None
    if what == "holes":
        table[1, [0, 3, 4, 5, 6, 15]] = -1
        table[2, :] = -1
    if what == "bad_pages":
        table[1, [1, 2]] = [pages, 2 ** 31 - 1]
        table[0, 0] = -2 ** 31
    if what == "none":
        lens = [0, 0, 0, 0]
    if what == "stride":
        stride = nh * hd + 5
    if what == "max_ctx":
        max_ctx = 40
    if what == "no_ctx":
        max_ctx, table = 0, table[:, :0]
    if what == "big_scores":
        scale = 50.0
    if what == "all_equal":
        q[:] = 0
    if what == "nan_key":
        c.scales[table[3, 2], 1, 0, 7] = np.nan
    got = attend(rt, dtype, c, q, table, lens, max_ctx, nh, scale, 0.0, 0, q_stride=stride)
    if what == "nan_key":
        assert np.isnan(got[3, nh // 2:]).all() and np.isfinite(got[3, :nh // 2]).all()
        c.scales[table[3, 2], 1, 0, 7] = 1.0
        lens, got = lens[:3], got[:3]
    if what in ("max_ctx", "no_ctx"):
        lens = [min(n, max_ctx) for n in lens]
    check_attended(c, got, q, table, lens, nh, scale, 0.0, 0, dtype)


@pytest.mark.parametrize("dtype,width", [("bfloat16", 300), ("bfloat16", 2000), ("bfloat16", 9000), ("float32", 2000)])
def test_wide_tables(rt, dtype, width):
    """The cut of the keys follows from the width of the table: long contexts in all of its forms, and rows that do not know of each other."""
    rng = np.random.default_rng(width)
    nh, nkv, hd, bs, form = 4, 2, 64, 16, 0
    lens = [4700, 31, 2049, 1024]
    table, pages = tables(rng, lens, bs, width)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    q = rounded(rng.standard_normal((4, nh, hd)) * 2, dtype)
    for window in (0, 1500):
        got = attend(rt, dtype, c, q, table, lens, 4700, nh, 0.125, 0.0, window)
        check_attended(c, got, q, table, lens, nh, 0.125, 0.0, window, dtype)
        alone = attend(rt, dtype, c, q[2:3], table[2:3], lens[2:3], 2304, nh, 0.125, 0.0, window)
        assert np.array_equal(alone[0], got[2])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 4, 128), (34, 2, 256)])
def test_captured_and_on_two_streams(rt, nh, nkv, hd, dtype):
    """A token written, attended to and its pages read back, recorded into two graphs that share a workspace and replayed in turn with other
    tokens, lengths and slots, eager calls on the default stream in between: the bits of the eager calls every time."""
    rng = np.random.default_rng(hd)
    k = rt.kernels(dtype)
    bs, form, R, width = 16, 0, 3, 40
    lens = [600, 17, 300]
    table, pages = tables(rng, [640] * R, bs, width)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    row = (nh + 2 * nkv) * hd
    inv = rt.upload((10000.0 ** (-np.arange(hd // 2) * 2.0 / hd)).astype(np.float32))
    TBL = rt.upload(table)
    WS = rt.zeros((k.zk_attention_q8_workspace(R, nh, hd, 640, width * bs) // 4 + 1,), "float32")

    class State:
        def __init__(self):
            self.cache = device_cache(rt, c)
            self.X, self.Q, self.OUT = (rt.zeros((R, n), dtype) for n in (row, nh * hd, nh * hd))
            self.POS, self.SL, self.CL = (rt.zeros((R,), "int32") for _ in range(3))
            self.K, self.V = rt.zeros((pages, nkv, bs, hd), dtype), rt.zeros((pages, nkv, hd, bs), dtype)

        def fill(self, i):
            r = np.random.default_rng(i)
            x = rounded(r.standard_normal((R, row)), dtype)
            ctx = np.array([n + i for n in lens], np.int32)
            slots = np.array([table[j, (n - 1) // bs] * bs + (n - 1) % bs for j, n in enumerate(ctx)], np.int32)
            from zse_amd.weights.safetensors import f32_to_bf16_bits
            rt.copy_h2d(self.X.ptr, f32_to_bf16_bits(x) if dtype == "bfloat16" else x)
            for t, a in ((self.POS, ctx - 1), (self.SL, slots), (self.CL, ctx)):
                rt.copy_h2d(t.ptr, a.astype(np.int32))

        def run(self, stream):
            kc, vc, sc = self.cache
            k.zk_rope_cache_write_q8(self.X.ptr, row, None, 0, self.Q.ptr, nh * hd, self.POS.ptr, self.SL.ptr, inv.ptr, hd, kc.ptr, vc.ptr, sc.ptr,
                                     R, nh, nkv, hd, bs, pages, form, stream)
            k.zk_attention_q8(self.Q.ptr, nh * hd, kc.ptr, vc.ptr, sc.ptr, TBL.ptr, width, self.CL.ptr, self.OUT.ptr, R, 640, nh, nkv, hd, bs, pages,
                              0.1, 0.0, 0, form, WS.ptr, WS.nbytes, stream)
            k.zk_cache_read_q8(kc.ptr, vc.ptr, sc.ptr, TBL.ptr, width, None, self.CL.ptr, self.K.ptr, self.V.ptr, R, 640, 33, nkv, hd, bs, pages, 1,
                               form, stream)

        def results(self):
            return [rt.download(t) for t in (*self.cache, self.Q, self.OUT, self.K, self.V)]

    a, b, eager = State(), State(), State()
    graphs = []
    for s in (a, b):
        s.fill(0)
        s.run(rt.stream)                  # once outside: what a first call sets up is not recorded
        rt.sync()
        rt.capture_begin()
        try:
            s.run(rt.stream)
        finally:
            graphs.append(rt.capture_end())
    eager.fill(0)
    eager.run(None)
    rt._check(rt.lib.zrt_device_sync(), "device sync")
    for i in range(1, 5):
        for s, g in ((a, graphs[0]), (b, graphs[1])):
            s.fill(i)
            rt.graph_launch(g)
        rt.sync()
        eager.fill(i)
        eager.run(None)
        rt._check(rt.lib.zrt_device_sync(), "device sync")
        want = eager.results()
        for s in (a, b):
            assert all(np.array_equal(x, y) for x, y in zip(s.results(), want)), i
    for g in graphs:
        rt.graph_destroy(g)


@pytest.mark.parametrize("nkv,bs", [(2, 16), (1, 64)])
def test_more_than_64_requests(rt, nkv, bs):
    """Pages numbered through 150 requests, most of them short, some empty; windows; the attention of all of them."""
    rng = np.random.default_rng(bs)
    nh, hd, form, dtype = 4, 64, 1, "bfloat16"
    k = rt.kernels(dtype)
    lens = [int(n) for n in rng.integers(0, 90, 150)]
    lens[::7] = [0] * len(lens[::7])
    new = [int(rng.integers(0, n + 1)) for n in lens]
    table, pages = tables(rng, lens, bs, 8)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    KC, VC, SC = device_cache(rt, c)
    TBL, CL, QS = rt.upload(table), rt.upload(np.array(lens, np.int32)), rt.upload(np.cumsum([0] + new).astype(np.int32))
    for window in (0, 20):
        K, V = up(rt, np.full((pages, nkv, bs, hd), 3.0), dtype), up(rt, np.full((pages, nkv, bs, hd), 3.0), dtype)
        k.zk_cache_read_q8(KC.ptr, VC.ptr, SC.ptr, TBL.ptr, 8, QS.ptr, CL.ptr, K.ptr, V.ptr, len(lens), 96, window, nkv, hd, bs, pages, 0, form,
                           rt.stream)
        want = np.full((2, pages, nkv, bs, hd), 3.0, np.float32)
        for r, n in enumerate(lens):
            for j in range(max(0, n - new[r] + 1 - window) // bs if window else 0, -(-n // bs)):
                want[:, table[r, j]] = 0.0
                for t in range(min(bs, n - j * bs)):
                    for h in range(nkv):
                        for values in (0, 1):
                            want[values, table[r, j], h, t] = c.row(table[r, j], h, t, bool(values)).astype(np.float32)
        assert np.array_equal(rt.download_f32(K), rounded(want[0], dtype)) and np.array_equal(rt.download_f32(V), rounded(want[1], dtype)), window
        q = rounded(rng.standard_normal((len(lens), nh, hd)), dtype)
        got = attend(rt, dtype, c, q, table, lens, 96, nh, 0.125, 0.0, window)
        check_attended(c, got, q, table, lens, nh, 0.125, 0.0, window, dtype)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 300, 511, 512])
def test_windows_as_long_as_everything(rt, window):
    """A window that hides nothing, up to the largest number: the bits of none."""
    rng = np.random.default_rng(0)
    nh, nkv, hd, bs, form, dtype = 4, 2, 64, 16, 0, "float32"
    k = rt.kernels(dtype)
    lens, new = [500, 1, 0, 40], [7, 1, 0, 40]
    table, pages = tables(rng, lens, bs, 32)
    c = random_cache(rng, pages, nkv, hd, bs, form)
    q = rounded(rng.standard_normal((4, nh, hd)), dtype)
    assert np.array_equal(*(attend(rt, dtype, c, q, table, lens, 512, nh, 0.125, 0.0, w) for w in (0, window)))
    KC, VC, SC = device_cache(rt, c)
    TBL, CL, QS = rt.upload(table), rt.upload(np.array(lens, np.int32)), rt.upload(np.cumsum([0] + new).astype(np.int32))
    got = []
    for w in (0, window):
        K, V = up(rt, np.full((pages, nkv, bs, hd), 3.0), dtype), up(rt, np.full((pages, nkv, bs, hd), 3.0), dtype)
        k.zk_cache_read_q8(KC.ptr, VC.ptr, SC.ptr, TBL.ptr, 32, QS.ptr, CL.ptr, K.ptr, V.ptr, 4, 512, w, nkv, hd, bs, pages, 0, form, rt.stream)
        got.append((rt.download(K), rt.download(V)))
    assert all(np.array_equal(x, y) for x, y in zip(*got))


def test_offsets_past_32_bits(rt):
    """A page whose codes lie more than 4 GiB behind the first."""
    nkv, hd, bs, form, nh = 32, 256, 128, 0, 32
    k = rt.kernels("bfloat16")
    pages = (5 << 30) // (nkv * hd * bs)
    page = pages - 1
    assert page * nkv * hd * bs > 2 ** 32
    rng = np.random.default_rng(0)
    KC, VC, SC = (rt.zeros((n,), "float32") for n in (pages * nkv * hd * bs // 4,) * 2 + (pages * nkv * 2 * bs,))
    rows = rounded(rng.standard_normal((3, (nh + 2 * nkv) * hd)), "bfloat16")
    X, Q = up(rt, rows, "bfloat16"), rt.zeros((3, nh * hd), "bfloat16")
    TBL, CL = rt.upload(np.array([[page]], np.int32)), rt.upload(np.array([3], np.int32))
    POS, SL = rt.upload(np.arange(3, dtype=np.int32)), rt.upload((page * bs + np.arange(3)).astype(np.int32))
    k.zk_rope_cache_write_q8(X.ptr, rows.shape[1], None, 0, Q.ptr, nh * hd, POS.ptr, SL.ptr, None, 0, KC.ptr, VC.ptr, SC.ptr, 3, nh, nkv, hd, bs,
                             pages, form, rt.stream)
    WS = rt.zeros((k.zk_attention_q8_workspace(1, nh, hd, 3, bs) // 4 + 1,), "float32")
    OUT = rt.zeros((1, nh * hd), "bfloat16")
    k.zk_attention_q8(Q.ptr + 2 * nh * hd * 2, nh * hd, KC.ptr, VC.ptr, SC.ptr, TBL.ptr, 1, CL.ptr, OUT.ptr, 1, 3, nh, nkv, hd, bs, pages, 1 / 16,
                      0.0, 0, form, WS.ptr, WS.nbytes, rt.stream)
    from zse_amd.runtime.device import Tensor
    before, c = P.Cache(1, nkv, hd, bs, form), P.Cache(1, nkv, hd, bs, form)
    c.k[...], c.v[...] = (rt.download(Tensor(t.ptr + page * nkv * hd * bs, c.k.shape, "uint8", t)) for t in (KC, VC))
    c.scales[...] = rt.download(Tensor(SC.ptr + page * nkv * 2 * bs * 4, c.scales.shape, "float32", SC))
    check_written(before, c, rt.download_f32(Q), rows.astype(np.float64), np.arange(3), np.arange(3), np.zeros(0), 0, nh, "bfloat16")
    x = rounded(rows[2:, :nh * hd], "bfloat16").reshape(1, nh, hd)
    check_attended(c, rt.download_f32(OUT).reshape(1, nh, hd), x, np.zeros((1, 1), np.int32), [3], nh, 1 / 16, 0.0, 0, "bfloat16")
    del KC, VC, SC
