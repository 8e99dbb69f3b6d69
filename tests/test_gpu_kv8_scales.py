"""Paged 8-bit attention where the scales of a cache's values lie far apart: what a row's result
loses is measured by the weights that the row itself sees."""
import numpy as np
import pytest

import kv8_ref as ref
from kv8_ref import U
from test_gpu_kv8 import RUNS, run_attn, tables_of

pytestmark = pytest.mark.gpu


def attention(cache, rows, past, tables, q, scale, window=0, only=None):
    """kv8_ref.attention's result, with a bound that takes nothing from outside a row: its terms of
    the formula, and for the halves of a weight p * scale(V) the unit of the row's own largest one.
    That is at least 2^10 units (many columns; 2^14 with few), and of each weight half the last step of
    an f16, 2^-25 units, may be lost, times a code of up to 127.  A result below f32's normal range
    is off by half a step, 2^-150.
    """
    out, bound, at = np.zeros_like(q, np.float64), np.zeros_like(q, np.float64), 0
    G = q.shape[1] // cache.H
    for b, n in enumerate(rows):
        k, has = cache.rows(0, tables[b], 0, past[b] + n)
        v, _ = cache.rows(1, tables[b], 0, past[b] + n)
        vs = np.zeros((past[b] + n, cache.H))
        for t in range(past[b] + n):
            place = cache.place(tables[b], t)
            if place is not None:
                vs[t] = cache.scales[1][place[0], :, place[1] // 16]
        token = np.arange(past[b] + n)
        for i in range(n):
            if only is not None and (at + i) not in only:
                continue
            t = past[b] + i
            seen = has & (token <= t)
            if window:
                seen &= token > t - window
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                kk, vv = k[seen, h // G], v[seen, h // G]
                s = scale * (kk @ q[at + i, h].astype(np.float64))
                d = s - s.max()
                p = np.exp(d)
                p /= p.sum()
                rel = 8 * U * (np.abs(s) + np.abs(s).max()) + 4 * U * np.abs(d) + (8 + len(p) / 4 + 64) * U
                out[at + i, h] = p @ vv
                bound[at + i, h] = (p * rel) @ np.abs(vv) + (p @ rel) * np.abs(out[at + i, h])
                bound[at + i, h] += len(p) * 127 * (p * vs[seen, h // G]).max() * 2.0 ** -35 + 2.0 ** -150
        at += n
    return out, bound


def check(got, want, bound, rows=None):
    off = np.abs(got - want) > bound
    if rows is not None:
        off = off[rows]
    assert not off.any(), (int(off.sum()), float((np.abs(got - want) / np.maximum(bound, 1e-300)).max()))


@pytest.mark.parametrize("low,high", [(-4, 10), (-4, 16), (-4, 24), (-4, 40), (-4, 120), (-100, 20), (-126, -60)])
@RUNS
def test_a_block_that_only_later_rows_see(gpu, run, low, high):
    # tokens 0 .. 15 in a block of small values, from 16 on in one of large ones: the row at token 15 sees the first alone
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(100 + high)
    cache = ref.Cache(2, page, H, D, rng)
    cache.scales[1][0], cache.scales[1][1] = 2.0 ** low, 2.0 ** high
    dev = ref.Device(gpu, cache)
    tables = np.array([[0, 1]], np.uint32)
    q = rng.standard_normal((4, nq, D)).astype(np.float32)
    want, bound = attention(cache, [4], [14], tables, q, 0.2)
    assert np.all(np.abs(want[:2]).max(-1) > 2.0 ** low)
    check(run(gpu, dev, [4], [14], tables, q, 0.2, 0), want, bound)


@pytest.mark.parametrize("low,high", [(-4, 20), (-4, 40), (-30, 90)])
@RUNS
def test_a_block_that_only_earlier_rows_see(gpu, run, low, high):
    # large values that leave the window of the tile's later rows
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(200 + high)
    cache = ref.Cache(4, page, H, D, rng)
    cache.scales[1][:] = 2.0 ** low
    cache.scales[1][1] = 2.0 ** high
    dev = ref.Device(gpu, cache)
    tables = np.array([[0, 1, 2, 3]], np.uint32)
    q = rng.standard_normal((4, nq, D)).astype(np.float32)
    want, bound = attention(cache, [4], [50], tables, q, 0.2, 20)  # windows from tokens 31 .. 34 on
    check(run(gpu, dev, [4], [50], tables, q, 0.2, 20), want, bound)


def with_low_scores(gpu, blocks, low, tokens, drop, small, large, seed):
    """A cache of one key head whose blocks `low` have scores that are lower by `drop` (nats) and values
    of scale `large`; the others' is `small`."""
    nq, D, page = 2, 64, 16
    rng = np.random.default_rng(seed)
    cache = ref.Cache(blocks, page, 1, D, rng)
    cache.scales[0][:] = 2.0 ** -5
    cache.codes[0][:] = rng.integers(-2, 3, cache.codes[0].shape)
    cache.codes[0][low] = -127
    cache.scales[1][:] = small
    cache.scales[1][low] = large
    dev = ref.Device(gpu, cache)
    q = (1 + 0.01 * rng.standard_normal((1, nq, D))).astype(np.float32)
    return cache, dev, np.arange(blocks, dtype=np.uint32)[None], q, drop / (D * 127 / 32), [1], [tokens - 1]


@pytest.mark.parametrize("drop,small,large", [
    (20, 2.0 ** -4, 2.0 ** 30),      # 2^-29 of weight times values 2^34 times as large
    (60, 2.0 ** -4, 2.0 ** 40),      # values that are lost by right
    (97, 2.0 ** -20, 2.0 ** 118),    # probabilities below f32's range: of weight all the same
    (97, 0.0, 2.0 ** 20),            # nothing but those
    (97, 0.0, 2.0 ** 100),
    (30, 2.0 ** -126, 2.0 ** -90),
])
@pytest.mark.parametrize("low", [[0], [5], [0, 1, 2], [3, 9, 10]])
@RUNS
def test_large_values_of_small_probability(gpu, run, low, drop, small, large):
    cache, dev, tables, q, scale, rows, past = with_low_scores(gpu, 12, low, 185, drop, small, large, 7)
    want, bound = attention(cache, rows, past, tables, q, scale)
    check(run(gpu, dev, rows, past, tables, q, scale, 0), want, bound)


@pytest.mark.parametrize("drop,small,large", [(20, 2.0 ** -4, 2.0 ** 30), (97, 2.0 ** -20, 2.0 ** 118), (97, 0.0, 2.0 ** 60)])
def test_parts_with_units_of_their_own(gpu, drop, small, large):
    # the large values all lie in one of the parts that a long sequence is split into
    cache, dev, tables, q, scale, rows, past = with_low_scores(gpu, 260, list(range(100, 108)), 4150, drop, small, large, 8)
    b = dev.batch(rows, past, tables)
    assert gpu.kv8_attn_workspace(dev.cache, b, q.shape[1], 0, 0) > 0
    want, bound = attention(cache, rows, past, tables, q, scale)
    check(run_attn(gpu, dev, rows, past, tables, q, scale, 0), want, bound)


@pytest.mark.parametrize("size,scale_k,scale", [(1e-36, 2.0 ** 112, 1.0), (1e-40, 2.0 ** 125, 1.0), (1e-30, 2.0 ** 60, 1e11),
                                                (1e30, 2.0 ** -104, 1.0), (1e25, 2.0 ** -126, 1e12), (1e-30, 2.0 ** 126, 1e-9)])
@RUNS
def test_queries_and_keys_of_sizes_far_apart(gpu, run, size, scale_k, scale):
    # scores of ordinary size, from factors at the ends of the range of f32
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(int(np.log2(scale_k)) + 300)
    cache = ref.Cache(12, page, H, D, rng)
    cache.scales[0][:] = scale_k * 2.0 ** -rng.integers(0, 3, cache.scales[0].shape)
    cache.scales[0][7], cache.codes[0][7] = 0, 0
    dev = ref.Device(gpu, cache)
    tables = np.arange(12, dtype=np.uint32)[None]
    q = (rng.standard_normal((2, nq, D)) * size).astype(np.float32)
    unit = size * scale_k * scale
    scale = np.float32(scale * min(1.0, 0.01 / unit))  # (scores of a few units)
    want, bound = attention(cache, [2], [150], tables, q, float(scale))
    check(run(gpu, dev, [2], [150], tables, q, float(scale), 0), want, bound)


@RUNS
def test_rows_of_sizes_far_apart_in_one_tile(gpu, run):
    # the first row's scores are ordinary under key scales of 2^100, the second's under those of 2^-40
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(77)
    cache = ref.Cache(12, page, H, D, rng)
    for row, scale_k in enumerate((2.0 ** 100, 2.0 ** -40)):
        cache.scales[0][:] = scale_k
        dev = ref.Device(gpu, cache)
        q = rng.standard_normal((2, nq, D)).astype(np.float32) * np.array([[[1e-33]], [[1e9]]], np.float32)
        want, bound = attention(cache, [2], [150], np.arange(12, dtype=np.uint32)[None], q, 1.0, only={row})
        got = run(gpu, dev, [2], [150], np.arange(12, dtype=np.uint32)[None], q, 1.0, 0)
        check(got, want, bound, [row])


@pytest.mark.parametrize("size", [1.0, 1e9, 1e30])
def test_parts_of_scores_past_all_units(gpu, size):
    # equal scores of any size are an average of the values, also of values near f32's end
    nq, D, page = 2, 64, 16
    rng = np.random.default_rng(11)
    cache = ref.Cache(260, page, 1, D, rng)
    cache.codes[0][:], cache.scales[0][:], cache.scales[1][:] = 1, 1.0, 2.0 ** 110
    cache.codes[1][:] = rng.integers(100, 128, cache.codes[1].shape)
    dev = ref.Device(gpu, cache)
    tables = np.arange(260, dtype=np.uint32)[None]
    q = np.full((1, nq, D), size, np.float32)
    b = dev.batch([1], [4149], tables)
    assert gpu.kv8_attn_workspace(dev.cache, b, nq, 0, 0) > 0
    got = run_attn(gpu, dev, [1], [4149], tables, q, 1.0, 0)
    values = cache.rows(1, tables[0], 0, 4150)[0][:, 0]
    # (weights are equal up to the exponentials' 4 half steps and the sums' n / 4 + 64, as above)
    assert np.all(np.abs(got[0] - values.mean(0)) <= 2 * (4 + 8 + 4150 / 4 + 64) * U * values.mean(0))


@pytest.mark.parametrize("D", [64, 256])
def test_a_prompt_with_blocks_far_apart(gpu, D):
    # causal rows over values of every size: each row as precise as its own
    nq, H, page, n = 8, 8, 32, 1100
    rng = np.random.default_rng(17 + D)
    cache = ref.Cache(-(-n // page), page, H, D, rng)
    cache.scales[1][:] = 2.0 ** rng.integers(-60, -50, cache.scales[1].shape)
    cache.scales[1][10:] *= 2.0 ** 30
    cache.scales[1][20:, ::2] *= 2.0 ** 40
    dev = ref.Device(gpu, cache)
    tables = np.arange(cache.P, dtype=np.uint32)[None]
    q = rng.standard_normal((n, nq, D)).astype(np.float32)
    assert gpu.kv8_attn_workspace(dev.cache, dev.batch([n], [0], tables), nq, 0, 0) == 0
    some = sorted(set(range(0, n, 61)) | {318, 319, 320, 321, 638, 639, 640, 641, n - 1})
    want, bound = attention(cache, [n], [0], tables, q, 0.1, only=set(some))
    check(run_attn(gpu, dev, [n], [0], tables, q, 0.1, 0), want, bound, some)
