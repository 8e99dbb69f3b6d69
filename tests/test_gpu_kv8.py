"""The paged 8-bit K/V cache: append, read-back and attention against 64-bit numpy
(kv8_ref.py), and a serving loop of them together with the sampling operators."""
import numpy as np
import pytest

import gemma_hip as gh
import kv8_ref as ref
from kv8_ref import U

pytestmark = pytest.mark.gpu
EPS = 1e-6


def tables_of(rng, seqs, per, pages):
    return rng.permutation(pages)[:seqs * per].reshape(seqs, per).astype(np.uint32)


def packed_rows(rng, total, nq, H, D):
    qkv = rng.standard_normal((total, (nq + 2 * H) * D)).astype(np.float32)
    qn, kn = (1 + 0.1 * rng.standard_normal((2, D))).astype(np.float32)
    return qkv, qn, kn


def expected_rows(qkv, qn, kn, rows, past, nq, H, D, rot, k_eq_v, theta):
    x = qkv.astype(np.float64).reshape(len(qkv), nq + 2 * H, D)
    pos = np.concatenate([p + np.arange(r) for r, p in zip(rows, past)]) if len(rows) else np.zeros(0)
    raw = ref.rms(x, EPS)
    q = ref.rope(raw[:, :nq] * qn.astype(np.float64), pos, rot, theta)
    k = ref.rope(raw[:, nq:nq + H] * kn.astype(np.float64), pos, rot, theta)
    v = raw[:, nq:nq + H] if k_eq_v else raw[:, nq + H:]
    return q, k, v


def run_append(ctx, cache, dev, rng, rows, past, tables, nq, rot, k_eq_v=False, theta=10000.0, change=None):
    H, D = cache.H, cache.D
    total = sum(rows)
    qkv, qn, kn = packed_rows(rng, total, nq, H, D)
    if change is not None:
        change(qkv)
    with np.errstate(all="ignore"):
        q, k, v = expected_rows(qkv, qn, kn, rows, past, nq, H, D, rot, k_eq_v, theta)
        at = 0
        for b, n in enumerate(rows):
            if n:
                cache.append(0, tables[b], past[b], k[at:at + n])
                cache.append(1, tables[b], past[b], v[at:at + n])
            at += n
    X, QN, KN, QO = ctx.upload(qkv), ctx.upload(qn), ctx.upload(kn), ctx.alloc(total * nq * D * 4)
    w = (nq + 2 * H) * D
    ctx.kv8_append(dev.cache, dev.batch(rows, past, tables), X.ptr, X.ptr + 4 * nq * D,
                   None if k_eq_v else X.ptr + 4 * (nq + H) * D, w, w, QN, KN, QO, nq, rot, k_eq_v, theta, EPS)
    got = QO.read(np.float32).reshape(total, nq, D)
    # inverse rms: a tree of 16 sums, quotient, root; two products with it; the angle's rounding and
    # the turn's three: 24 half steps of what is turned
    raw = ref.rms(qkv.astype(np.float64).reshape(total, -1, D)[:, :nq], EPS) * qn.astype(np.float64)
    size = np.abs(raw)
    h = rot // 2
    size[..., :h] = size[..., h:rot] = np.abs(raw[..., :h]) + np.abs(raw[..., h:rot])
    if change is None:
        assert np.all(np.abs(got - q) <= 24 * U * size)
    return got


def check_cache(cache, dev, tables, rows, past):
    """Codes and scales of every token that the sequences hold."""
    for which, (codes, scales) in enumerate(zip(dev.codes(), dev.scales())):
        wrong = 0
        for b, n in enumerate(rows):
            for t in range(past[b] + n):
                at = cache.place(tables[b], t)
                if at is None:
                    continue
                p, w = at
                s = cache.scales[which][p, :, w // 16]
                assert np.array_equal(scales[p, :, w // 16], s, equal_nan=True), (which, b, t)
                ok = ~np.isnan(s)
                d = np.abs(codes[p, ok, w].astype(int) - cache.codes[which][p, ok, w])
                assert d.max(initial=0) <= 1
                wrong += int(d.sum())
        assert wrong <= cache.near, (which, wrong, cache.near)


SHAPES = [  # heads, kv heads, head dim, rotated dims, page
    (16, 8, 256, 256, 16), (16, 8, 256, 64, 64), (4, 4, 64, 32, 32), (12, 4, 96, 96, 128), (8, 1, 128, 0, 16),
    (8, 2, 512, 128, 256), (3, 1, 16, 2, 16), (5, 1, 400, 400, 32), (2, 2, 272, 68, 16), (2, 1, 512, 512, 32),
]


@pytest.mark.parametrize("nq,H,D,rot,page", SHAPES)
def test_append_ragged_batches_and_growing_blocks(gpu, nq, H, D, rot, page):
    rng = np.random.default_rng(D + page)
    seqs, per = 4, 3 + 160 // page
    cache = ref.Cache(seqs * per + 3, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, seqs, per, cache.P)
    past = [0, 0, 0, 0]
    # a token, an empty sequence, a block's end and a prompt; then more into the same blocks
    for rows in ([1, 0, 16, 37], [3, 1, 1, 9], [1, 17, 2, 0], [20, 1, 31, 5]):
        run_append(gpu, cache, dev, rng, rows, past, tables, nq, rot)
        check_cache(cache, dev, tables, rows, past)
        past = [p + r for p, r in zip(past, rows)]
    # cut back and written again: the scale of a block that keeps tokens stays
    past = [p - c for p, c in zip(past, (2, 5, 17, 3))]
    rows = [1, 6, 18, 2]
    run_append(gpu, cache, dev, rng, rows, past, tables, nq, rot)
    check_cache(cache, dev, tables, rows, past)
    assert cache.near < 20


def test_append_error_stays_under_a_step(gpu):
    # rows that grow by doublings raise the scale again and again: under one step in all
    H, D, page = 2, 64, 16
    rng = np.random.default_rng(4)
    cache = ref.Cache(1, page, H, D)
    dev = ref.Device(gpu, cache)
    table = np.zeros((1, 1), np.uint32)
    values = []
    for t in range(16):
        kn = np.full(D, 2.0 ** (t - 8), np.float32)
        x = rng.standard_normal((1, 3 * H * D)).astype(np.float32)
        values.append(ref.rms(x.astype(np.float64).reshape(3 * H, D)[H:2 * H], EPS) * kn)
        X, N = gpu.upload(x), gpu.upload(kn)
        gpu.kv8_append(dev.cache, dev.batch([1], [t], table), None, X.ptr + 4 * H * D, X.ptr + 8 * H * D, 0, 3 * H * D,
                       None, N, None, 0, 0, False, 10000.0, EPS)
    s = dev.scales()[0][0, :, 0]
    got = dev.codes()[0][0] * s[:, None, None]  # [head][token][dim]
    assert np.all(np.abs(got - np.stack(values, 1)) < s[:, None, None])
    assert np.all(s * 127 >= np.abs(np.stack(values, 1)).max((1, 2))) and np.all(s * 63.5 < np.abs(np.stack(values, 1)).max((1, 2)))


@pytest.mark.parametrize("position", [100000, 4000000000])
def test_append_far_positions(gpu, position):
    # (the table's first entries have no page: only the last is used)
    H, D, page = 1, 128, 256
    rng = np.random.default_rng(9)
    cache = ref.Cache(2, page, H, D)
    dev = ref.Device(gpu, cache)
    per = position // page + 2
    table = np.full((1, per), 0xffffffff, np.uint32)
    table[0, position // page], table[0, position // page + 1] = 1, 0
    nq = 2
    qkv, qn, kn = packed_rows(rng, 3, nq, H, D)
    X, QN, KN, QO = gpu.upload(qkv), gpu.upload(qn), gpu.upload(kn), gpu.alloc(3 * nq * D * 4)
    w = (nq + 2 * H) * D
    gpu.kv8_append(dev.cache, dev.batch([3], [position], table), X.ptr, X.ptr + 4 * nq * D, X.ptr + 4 * (nq + H) * D, w, w,
                   QN, KN, QO, nq, D, False, 10000.0, EPS)
    q, k, v = expected_rows(qkv, qn, kn, [3], [position], nq, H, D, D, False, 10000.0)
    # angles in 64 bits: off by 4 half steps of the angle, a turn's arc
    arc = position * 4 * 2.0 ** -53
    assert np.abs(QO.read(np.float32).reshape(3, nq, D) - q).max() <= 5 * 24 * U + 5 * arc
    K, V = gpu.alloc(3 * D * 4), gpu.alloc(3 * D * 4)
    gpu.kv8_read(dev.cache, dev.batch([3], [position], table), K, V)
    for got, want, which in ((K, k, 0), (V, v, 1)):
        got = got.read(np.float32).reshape(3, 1, D)
        s = dev.scales()[which][[1] * 3 if position % page < page - 2 else [1, 0, 0], 0,
                                [(position + i) % page // 16 for i in range(3)]]
        assert np.all(np.abs(got - want) <= s[:, None, None] * 0.5 + 5 * arc)


def test_append_without_queries_and_in_place(gpu):
    H, D, page, nq = 2, 128, 32, 4
    rng = np.random.default_rng(3)
    tables = np.array([[2, 0]], np.uint32)
    q = rng.standard_normal((5, nq * D)).astype(np.float32)
    kv = rng.standard_normal((5, 2 * H * D + 7)).astype(np.float32)  # a stride of its own
    n = np.ones(D, np.float32)
    out = []
    for with_q in (True, False):
        cache = ref.Cache(3, page, H, D)
        dev = ref.Device(gpu, cache)
        Q, KV, N = gpu.upload(q), gpu.upload(kv), gpu.upload(n)
        gpu.kv8_append(dev.cache, dev.batch([5], [3], tables), Q if with_q else None, KV, KV.ptr + 4 * H * D, nq * D if with_q else 0,
                       2 * H * D + 7, N if with_q else None, N, Q if with_q else None, nq if with_q else 0, 64, False, 500.0, EPS)
        out.append(dev.codes() + dev.scales())
        if with_q:
            want = ref.rope(ref.rms(q.astype(np.float64).reshape(5, nq, D), EPS), 3 + np.arange(5), 64, 500.0)
            assert np.abs(Q.read(np.float32).reshape(5, nq, D) - want).max() <= 2 * 24 * U * np.abs(want).max()
    assert all(np.array_equal(a, b) for a, b in zip(*out))


def test_append_zero_nan_and_infinite_rows(gpu):
    H, D, page, nq = 1, 64, 16, 2
    rng = np.random.default_rng(8)
    cache = ref.Cache(4, page, H, D)
    dev = ref.Device(gpu, cache)
    tables = np.array([[3, 1], [0, 2]], np.uint32)
    k = slice(nq * D, (nq + H) * D)

    def zeros(x):
        x[:] = 0

    def broken(x):
        x[1, k.start + 5] = np.nan
        x[6, k.start + 9] = np.inf

    run_append(gpu, cache, dev, rng, [2, 3], [0, 0], tables, nq, 32, change=zeros)
    check_cache(cache, dev, tables, [2, 3], [0, 0])
    assert not dev.scales()[0][[3, 0], 0, 0].any()
    run_append(gpu, cache, dev, rng, [4, 5], [2, 3], tables, nq, 32, change=broken)
    check_cache(cache, dev, tables, [4, 5], [2, 3])
    assert np.isnan(dev.scales()[0][[3, 0], 0, 0]).all() and np.isfinite(dev.scales()[1]).all()
    # still NaN with a good row behind, good again from the block's first token on
    run_append(gpu, cache, dev, rng, [1, 1], [6, 8], tables, nq, 32)
    assert np.isnan(dev.scales()[0][[3, 0], 0, 0]).all()
    run_append(gpu, cache, dev, rng, [3, 17], [0, 0], tables, nq, 32)
    check_cache(cache, dev, tables, [3, 17], [0, 0])


def test_rows_without_a_page_and_rows_of_no_sequence(gpu):
    H, D, page, nq = 2, 64, 16, 2
    rng = np.random.default_rng(5)
    cache = ref.Cache(3, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    before = dev.codes() + dev.scales()
    # sequence 0: second page absent; 1: runs past its table; entries beyond the cache
    tables = np.array([[0, 3], [0xffffffff, 2]], np.uint32)
    rows, past = [20, 10], [0, 30]
    run_append(gpu, cache, dev, rng, rows, past, tables, nq, 64)
    check_cache(cache, dev, tables, rows, past)
    after = dev.codes() + dev.scales()
    for i in range(4):  # page 1 belongs to no one; page 2 got two tokens, at 14 and 15
        assert np.array_equal(before[i][1], after[i][1])
    K, V = (gpu.upload(np.full((33, H * D), 7.0, np.float32)) for _ in "kv")
    gpu.kv8_read(dev.cache, dev.batch(rows, past, tables, num_rows=33), K, V)
    for which, got in enumerate((K, V)):
        got = got.read(np.float32).reshape(33, H, D)
        want = np.concatenate([cache.rows(which, tables[b], past[b], rows[b])[0] for b in range(2)])
        assert np.abs(got[:30] - want).max() <= np.abs(cache.scales[which]).max() * (cache.near > 0)
        assert np.all(got[30:] == 7.0)
    # bounds that are too small for the rows: the rest is not touched
    K2 = gpu.upload(np.full((33, H * D), 7.0, np.float32))
    gpu.kv8_read(dev.cache, dev.batch(rows, past, tables, num_rows=25, max_rows=18), K2, None)
    got2, got = K2.read(np.float32).reshape(33, -1), K.read(np.float32).reshape(33, -1)
    untouched = [18, 19] + list(range(25, 33))
    assert np.all(got2[untouched] == 7.0)
    rest = [i for i in range(25) if i not in untouched]
    assert np.array_equal(got2[rest], got[rest])


# ---- attention -------------------------------------------------------------------------------
def run_attn(gpu, dev, rows, past, tables, q, scale, window, max_kv=0, **bounds):
    nq, D = q.shape[1:]
    b = dev.batch(rows, past, tables, **bounds)
    Q = gpu.upload(q)
    O = gpu.upload(np.full(q.shape, 5.0, np.float32))
    n = gpu.kv8_attn_workspace(dev.cache, b, nq, window, max_kv)
    W = gpu.alloc(n) if n else None
    gpu.kv8_attn(dev.cache, b, Q, O, nq, scale, window, max_kv, W, n)
    return O.read(np.float32).reshape(q.shape)


def run_many(gpu, dev, rows, past, tables, q, scale, window, max_kv=0, **bounds):
    """The same as the head of a batch with room for many more rows: the kernel of many columns."""
    room = np.full((q.shape[0] + 10000 // q.shape[1], *q.shape[1:]), np.nan, np.float32)
    room[:len(q)] = q
    many = dict(num_rows=len(room), max_rows=len(room)) if not bounds else bounds
    got = run_attn(gpu, dev, rows, past, tables, room, scale, window, max_kv, **many)
    assert np.all(got[len(q):] == 5.0)
    return got[:len(q)]


def run_stream(gpu, dev, rows, past, tables, q, scale, window, max_kv=0, **bounds):
    """The same with tables that have room for 96 MB of codes: loads that pass by the caches."""
    c = dev.c
    tokens = (96 << 20) // (2 * c.D * c.H * len(rows)) + 64
    wide = np.full((len(rows), max(tables.shape[1], tokens // c.page + 1)), 0xffffffff, np.uint32)
    wide[:, :tables.shape[1]] = tables
    return run_attn(gpu, dev, rows, past, wide, q, scale, window, max_kv, **bounds)


RUNS = pytest.mark.parametrize("run", [run_attn, run_many, run_stream])
ATTN = [  # nq, H, D, page, rows, past, window, scale
    (16, 8, 256, 16, [1], [543], 0, 1.0),
    (16, 8, 256, 32, [1, 1, 1, 1, 0, 1], [0, 15, 16, 700, 40, 129], 0, 0.0625),
    (16, 8, 256, 64, [5, 1, 9, 2], [90, 31, 0, 300], 0, 0.0625),
    (16, 8, 256, 64, [70], [0], 0, 0.0625),
    (16, 8, 256, 16, [33, 40], [100, 5], 24, 0.0625),
    (8, 8, 64, 32, [1, 3], [200, 77], 0, 0.125),
    (12, 4, 96, 128, [7, 20, 1], [3, 50, 260], 0, 0.1),
    (12, 4, 96, 16, [7, 20, 1], [3, 50, 260], 1, 0.1),
    (8, 1, 128, 64, [3, 1], [500, 2], 100, 0.0884),
    (8, 2, 512, 32, [1, 6], [333, 60], 0, 0.0442),
    (8, 2, 512, 256, [40], [17], 33, 1.0),
    (40, 2, 16, 16, [1, 2], [70, 0], 0, 0.25),
    (5, 1, 400, 32, [2, 30], [64, 1], 0, 0.05),
    (3, 1, 272, 16, [1], [0], 0, 0.06),
    (4, 4, 256, 16, [1], [2500], 0, 0.0625),
    (8, 8, 64, 16, [1] * 70, [(37 * i) % 90 for i in range(70)], 0, 0.125),
]


@pytest.mark.parametrize("nq,H,D,page,rows,past,window,scale", ATTN)
@RUNS
def test_attention(gpu, run, nq, H, D, page, rows, past, window, scale):
    rng = np.random.default_rng(nq * D + page + window)
    per = max(-(-(p + r) // page) for p, r in zip(past, rows)) + 1
    cache = ref.Cache(len(rows) * per + 2, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    want, bound = ref.attention(cache, rows, past, tables, q, scale, window)
    for max_kv in (0, max(p + r for p, r in zip(past, rows)), 1):  # (a plan for less than there is computes the same)
        got = run(gpu, dev, rows, past, tables, q, scale, window, max_kv)
        assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())


@RUNS
def test_attention_scales_far_apart_and_zero_blocks(gpu, run):
    # V blocks whose scales differ by 2^40: small probabilities times large values count
    nq, H, D, page = 4, 2, 128, 16
    rng = np.random.default_rng(12)
    cache = ref.Cache(12, page, H, D, rng)
    cache.scales[1] = 2.0 ** rng.integers(-30, 11, cache.scales[1].shape)
    cache.scales[1][3] = 0
    cache.codes[1][3] = 0
    cache.scales[0][4] = 0
    cache.codes[0][4] = 0
    dev = ref.Device(gpu, cache)
    tables = np.arange(12, dtype=np.uint32)[None]
    q = rng.standard_normal((1, nq, D)).astype(np.float32) * 0.3
    want, bound = ref.attention(cache, [1], [180], tables, q, 0.1, 0)
    got = run(gpu, dev, [1], [180], tables, q, 0.1, 0)
    assert np.all(np.abs(got - want) <= bound)


@RUNS
def test_attention_of_the_smallest_scales(gpu, run):
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(19)
    cache = ref.Cache(12, page, H, D, rng)
    cache.scales[1][:] = 2.0 ** -126
    dev = ref.Device(gpu, cache)
    tables = np.arange(12, dtype=np.uint32)[None]
    q = rng.standard_normal((2, nq, D)).astype(np.float32)
    want, bound = ref.attention(cache, [2], [180], tables, q, 0.3, 0)
    got = run(gpu, dev, [2], [180], tables, q, 0.3, 0)
    # (sums below f32's normal range: half a step of 2^-149 a wave, a split and the quotient, 12 at most)
    assert np.all(np.abs(got - want) <= bound + 6 * 2.0 ** -149)


@RUNS
def test_attention_masked_places_may_hold_anything(gpu, run):
    # NaN, infinite and huge scales behind a sequence's last token, in front of its window and in
    # pages of others change nothing; pages that are absent are as masked
    nq, H, D, page = 4, 2, 64, 32
    rng = np.random.default_rng(21)
    cache = ref.Cache(8, page, H, D, rng)
    tables = np.array([[5, 2, 7, 1], [0, 0xffffffff, 3, 6]], np.uint32)
    rows, past, window = [2, 3], [70, 85], 30
    q = rng.standard_normal((5, nq, D)).astype(np.float32)
    want, bound = ref.attention(cache, rows, past, tables, q, 0.2, window)
    for which in (0, 1):
        s = cache.scales[which]
        s[4] = np.nan                      # no one's
        s[5], s[0] = np.inf, np.nan        # in front of both windows (tokens 0 .. 31)
        s[1], s[6] = np.nan, np.inf        # behind both ends
        s[7, :, 1] = 2.0 ** 120            # tokens 80 .. 95 of the first sequence
    dev = ref.Device(gpu, cache)
    got = run(gpu, dev, rows, past, tables, q, 0.2, window)
    assert np.all(np.abs(got - want) <= bound)


@RUNS
def test_attention_rows_that_see_nothing(gpu, run):
    nq, H, D, page = 2, 1, 64, 16
    rng = np.random.default_rng(2)
    cache = ref.Cache(2, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    q = rng.standard_normal((4, nq, D)).astype(np.float32)
    tables = np.array([[0xffffffff, 0xffffffff], [9, 1]], np.uint32)
    # first: no page at all; second: window 2 at tokens 40, 41, past the table
    got = run(gpu, dev, [2, 2], [0, 40], tables, q, 1.0, 2)
    assert not got.any()
    # rows of no sequence and rows over the bounds keep what they have
    got = run(gpu, dev, [2], [3], np.array([[1, 0]], np.uint32), q, 1.0, 0, num_rows=4)
    assert np.all(got[2:] == 5.0) and not np.any(got[:2] == 5.0)
    got = run(gpu, dev, [4], [3], np.array([[1, 0]], np.uint32), q, 1.0, 0, max_rows=1)
    assert np.all(got[1:] == 5.0)
    got = run(gpu, dev, [0, 0], [3, 1], np.array([[1, 0], [0, 1]], np.uint32), q, 1.0, 0, num_rows=4, max_rows=4)
    assert np.all(got == 5.0)


@RUNS
def test_attention_queries_of_any_size(gpu, run):
    # rows of zeros, tiny, huge and broken queries next to ordinary ones
    nq, H, D, page = 2, 1, 128, 16
    rng = np.random.default_rng(6)
    cache = ref.Cache(4, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = np.arange(4, dtype=np.uint32)[None]
    q = rng.standard_normal((6, nq, D)).astype(np.float32)
    q[1] = 0
    q[2] *= 1e-30
    q[3] *= 1e4
    q[4, 0, 3] = np.nan
    q[4, 1, 5] = np.inf
    want, bound = ref.attention(cache, [6], [50], tables, np.nan_to_num(q, posinf=0), 0.05, 0)
    got = run(gpu, dev, [6], [50], tables, q, 0.05, 0)
    assert np.isnan(got[4]).all()
    fine = [0, 1, 2, 3, 5]
    assert np.all(np.abs(got - want)[fine] <= bound[fine])


@RUNS
def test_attention_nan_block_spoils_its_rows_only(gpu, run):
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(16)
    cache = ref.Cache(8, page, H, D, rng)
    tables = np.arange(8, dtype=np.uint32).reshape(2, 4)
    q = rng.standard_normal((2, nq, D)).astype(np.float32)
    want, bound = ref.attention(cache, [1, 1], [60, 60], tables, q, 0.2, 0)
    cache.scales[0][2, 1] = np.nan
    dev = ref.Device(gpu, cache)
    got = run(gpu, dev, [1, 1], [60, 60], tables, q, 0.2, 0)
    assert np.isnan(got[0, 2:]).all()
    assert np.all(np.abs(got - want)[0, :2] <= bound[0, :2]) and np.all(np.abs(got - want)[1] <= bound[1])


@pytest.mark.parametrize("nq,H,D,page,rows,past,window,scale", [
    (8, 8, 64, 64, [1100], [0], 0, 0.125),
    (8, 8, 64, 16, [1100], [40], 100, 0.125),
    (8, 4, 48, 32, [600, 3, 0, 700], [0, 500, 7, 33], 0, 0.15),
    (16, 2, 272, 32, [1030], [5], 0, 0.06),
])
def test_attention_of_long_prompts(gpu, nq, H, D, page, rows, past, window, scale):
    rng = np.random.default_rng(D + window)
    per = max(-(-(p + r) // page) for p, r in zip(past, rows))
    cache = ref.Cache(len(rows) * per, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    got = run_attn(gpu, dev, rows, past, tables, q, scale, window)
    assert gpu.kv8_attn_workspace(dev.cache, dev.batch(rows, past, tables), nq, window, 0) == 0
    # (every seventh row: a batch of its own to the formula)
    at = 0
    for b, n in enumerate(rows):
        for i in list(range(0, n, 7)) + [n - 1] * (n > 0):
            want, bound = ref.attention(cache, [1], [past[b] + i], tables[b:b + 1], q[at + i:at + i + 1], scale, window)
            assert np.all(np.abs(got[at + i:at + i + 1] - want) <= bound), (b, i)
        at += n


@pytest.mark.parametrize("rows,past", [([1, 3], [700, 90]), ([1100], [0])])
def test_attention_in_place(gpu, rows, past):
    nq, H, D, page = 8, 8, 64, 32
    rng = np.random.default_rng(8)
    per = max(-(-(p + r) // page) for p, r in zip(past, rows))
    cache = ref.Cache(len(rows) * per, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    want = run_attn(gpu, dev, rows, past, tables, q, 0.125, 0)
    b = dev.batch(rows, past, tables)
    n = gpu.kv8_attn_workspace(dev.cache, b, nq, 0, 0)
    X, W = gpu.upload(q), gpu.alloc(max(n, 16))
    gpu.kv8_attn(dev.cache, b, X, X, nq, 0.125, 0, 0, W, n)
    assert np.array_equal(X.read(np.float32).reshape(q.shape), want)


def test_attention_repeats_and_replays(gpu):
    # the same bits every time, also from two graphs that share the workspace
    nq, H, D, page = 16, 8, 256, 32
    rng = np.random.default_rng(7)
    cache = ref.Cache(80, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, 2, 40, 80)
    q = [rng.standard_normal((2, nq, D)).astype(np.float32) for _ in range(2)]
    b = dev.batch([1, 1], [1200, 333], tables)
    n = gpu.kv8_attn_workspace(dev.cache, b, nq, 0, 1201)
    assert n > 0
    W = gpu.alloc(n)
    Q = [gpu.upload(x) for x in q]
    O = [gpu.alloc(x.nbytes) for x in q]
    eager = []
    for x, o in zip(Q, O):
        gpu.kv8_attn(dev.cache, b, x, o, nq, 0.0625, 0, 1201, W, n)
        eager.append(o.read(np.float32))
    graphs = []
    for x, o in zip(Q, O):
        gpu.graph_begin()
        gpu.kv8_attn(dev.cache, b, x, o, nq, 0.0625, 0, 1201, W, n)
        graphs.append(gpu.graph_end())
    for turn in range(4):
        for g in graphs:
            gpu.graph_launch(g)
        for o, e in zip(O, eager):
            assert np.array_equal(o.read(np.float32), e)
            gpu.fill_u32(o, 0, e.size)
        gpu.sync()
    for g in graphs:
        gpu.graph_destroy(g)


# ---- all together ----------------------------------------------------------------------------
def test_serving_loop(gpu):
    """Prompts, then drafted tokens appended, attended, turned into probabilities and verified;
    rejected tokens are cut back and their places written again."""
    nq, H, D, page, V, n = 4, 2, 64, 16, 500, 3
    rng = np.random.default_rng(31)
    seqs = 3
    cache = ref.Cache(40, page, H, D)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, seqs, 8, cache.P)
    past = [0, 0, 0]
    rows = [21, 1, 16]
    head = rng.standard_normal((nq * D, V)).astype(np.float32)
    for turn in range(5):
        q = run_append(gpu, cache, dev, rng, rows, past, tables, nq, 32)
        check_cache(cache, dev, tables, rows, past)
        cache.codes, cache.scales = dev.codes(), dev.scales()  # (a border case is not counted twice)
        want, bound = ref.attention(cache, rows, past, tables, q, 0.125, 0)
        got = run_attn(gpu, dev, rows, past, tables, q, 0.125, 0)
        assert np.all(np.abs(got - want) <= bound)
        if turn:
            logits = (got.reshape(seqs * (n + 1), -1) @ head).astype(np.float32)
            L, S = gpu.upload(logits), gpu.logit_probs_workspace(len(logits), V)
            P, W = gpu.alloc(logits.nbytes), gpu.alloc(S)
            gpu.logit_probs(L, P, len(logits), V, V, 30.0, 0.7, W, S)
            p = P.read(np.float32).reshape(seqs, n + 1, V)
            pw, pb = ref.probabilities(logits, 30.0, 0.7)
            assert np.all(np.abs(p.reshape(-1, V) - pw) <= pb * pw + 1e-37)
            d = p[:, :n] * rng.uniform(0.5, 1.5, (seqs, n, V)).astype(np.float32)
            d = (d / d.sum(-1, keepdims=True)).astype(np.float32)
            tokens = d.argmax(-1).astype(np.uint32)
            u, pick = rng.random((seqs, n), np.float32), rng.random(seqs, np.float32)
            T, A = gpu.alloc(seqs * (n + 1) * 4), gpu.alloc(seqs * 4)
            S = gpu.spec_verify_workspace(seqs, V)
            W, D_, K, U_, I = gpu.alloc(S), gpu.upload(d), gpu.upload(tokens), gpu.upload(u), gpu.upload(pick)
            gpu.spec_verify(P, D_, K, None, U_, I, T, A, seqs, n, V, W, S)
            out, accepted = ref.verify(p, d, tokens, [n] * seqs, u, pick)
            assert np.array_equal(T.read(np.uint32).reshape(seqs, n + 1), out)
            assert np.array_equal(A.read(np.uint32), accepted)
            past = [x + 1 + int(a) for x, a in zip(past, accepted)]  # the last token and the kept drafts stay
        else:
            past = [x + r for x, r in zip(past, rows)]
        rows = [n + 1] * seqs


def test_captured_step_with_sequences_that_grow(gpu):
    """One recorded step (append, attention, probabilities, verification), replayed while the lengths,
    rows and numbers in its arrays change, against the same calls made directly on a second cache."""
    nq, H, D, page, V, n, seqs = 4, 2, 64, 16, 301, 2, 3
    rng = np.random.default_rng(43)
    T = seqs * (n + 1)
    tables = tables_of(rng, seqs, 4, 12)
    w = (nq + 2 * H) * D
    sides = []
    for _ in range(2):
        dev = ref.Device(gpu, ref.Cache(12, page, H, D))
        b = dev.batch([n + 1] * seqs, [0] * seqs, tables)
        B = dict(dev=dev, b=b, X=gpu.alloc(T * w * 4), N=gpu.upload(np.ones(D, np.float32)), Q=gpu.alloc(T * nq * D * 4),
                 O=gpu.alloc(T * nq * D * 4), L=gpu.alloc(T * V * 4), P=gpu.alloc(T * V * 4), K=gpu.alloc(seqs * n * 4),
                 ND=gpu.alloc(seqs * 4), U=gpu.alloc(seqs * n * 4), I=gpu.alloc(seqs * 4), T=gpu.alloc(T * 4), A=gpu.alloc(seqs * 4))
        B["sizes"] = sizes = (gpu.kv8_attn_workspace(dev.cache, b, nq, 0, 4 * page), gpu.logit_probs_workspace(T, V),
                              gpu.spec_verify_workspace(seqs, V))
        B["W"] = [gpu.alloc(max(x, 16)) for x in sizes]
        sides.append(B)

    def step(B):
        gpu.kv8_append(B["dev"].cache, B["b"], B["X"].ptr, B["X"].ptr + 4 * nq * D, B["X"].ptr + 4 * (nq + H) * D, w, w,
                       B["N"], B["N"], B["Q"], nq, D, False, 10000.0, EPS)
        gpu.kv8_attn(B["dev"].cache, B["b"], B["Q"], B["O"], nq, 0.125, 0, 4 * page, B["W"][0], B["sizes"][0])
        gpu.logit_probs(B["L"], B["P"], T, V, V, 30.0, 1.0, B["W"][1], B["sizes"][1])
        gpu.spec_verify(B["P"], None, B["K"], B["ND"], B["U"], B["I"], B["T"], B["A"], seqs, n, V, B["W"][2], B["sizes"][2])

    gpu.graph_begin()
    step(sides[0])
    graph = gpu.graph_end()
    past = np.array([0, 5, 14], np.uint32)
    for turn in range(5):
        x = rng.standard_normal((T, w)).astype(np.float32)
        logits = rng.standard_normal((T, V)).astype(np.float32) * 4
        tokens, drafts = rng.integers(0, V, (seqs, n)).astype(np.uint32), rng.integers(0, n + 1, seqs).astype(np.uint32)
        u, pick = rng.random((seqs, n), np.float32) * 0.1, rng.random(seqs, np.float32)
        for B in sides:
            for name, a in (("X", x), ("L", logits), ("K", tokens), ("ND", drafts), ("U", u), ("I", pick)):
                B[name].write(a)
            B["b"].held[1].write(past)
        gpu.graph_launch(graph)
        step(sides[1])
        gpu.sync()
        for name in ("Q", "O", "P", "T", "A"):
            one, two = (B[name].read(np.uint32) for B in sides)
            assert np.array_equal(one, two), (turn, name)
        for one, two in zip(*(B["dev"].codes() + B["dev"].scales() for B in sides)):
            assert np.array_equal(one, two)
        past += 1 + sides[0]["A"].read(np.uint32)
        for B in sides:  # nothing is left over from one turn for the next
            for name in ("O", "P", "T"):
                gpu.fill_u32(B[name], 0x7fc00000, B[name].nbytes // 4)
    gpu.graph_destroy(graph)
