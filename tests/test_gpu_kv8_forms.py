"""Forms of the paged 8-bit calls that a user of the interface can reach: values taken from raw
keys, heads between the kernels' widths, and attention kernels by the plan that takes them
(kv8_forms.py names the cases; test_serving_forms.py holds the plan to them)."""
import numpy as np
import pytest

import gemma_hip as gh
import kv8_ref as ref
from kv8_forms import PROMPTS, STREAMS
from kv8_ref import U
from test_gpu_kv8 import EPS, check_cache, packed_rows, run_append, run_attn, tables_of

pytestmark = pytest.mark.gpu


# ---- append ----------------------------------------------------------------------------------
@pytest.mark.parametrize("nq,H,D,rot,page", [(16, 8, 256, 256, 16), (4, 4, 64, 32, 32), (12, 4, 96, 96, 128), (8, 2, 512, 128, 32),
                                             (8, 1, 128, 0, 16), (6, 2, 144, 144, 32), (4, 2, 192, 48, 16)])
def test_append_values_from_raw_keys(gpu, nq, H, D, rot, page):
    rng = np.random.default_rng(D + rot)
    per = 2 + 80 // page
    cache = ref.Cache(3 * per + 1, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, 3, per, cache.P)
    past = [0, 0, 0]
    for rows in ([1, 0, 21], [5, 3, 1], [1, 16, 30]):
        run_append(gpu, cache, dev, rng, rows, past, tables, nq, rot, k_eq_v=True)
        check_cache(cache, dev, tables, rows, past)
        past = [p + r for p, r in zip(past, rows)]
    assert cache.near < 20


def test_append_values_from_raw_keys_take_no_values(gpu):
    # V_in is not read: the same bits with an array of NaN there
    nq, H, D, page = 4, 2, 128, 16
    rng = np.random.default_rng(40)
    qkv, qn, kn = packed_rows(rng, 9, nq, H, D)
    w, out = (nq + 2 * H) * D, []
    for v in (None, np.nan):
        cache = ref.Cache(2, page, H, D)
        dev = ref.Device(gpu, cache)
        qkv[:, (nq + H) * D:] = 0 if v is None else v
        X, QN, KN, QO = gpu.upload(qkv), gpu.upload(qn), gpu.upload(kn), gpu.alloc(9 * nq * D * 4)
        gpu.kv8_append(dev.cache, dev.batch([9], [4], np.array([[1, 0]], np.uint32)), X.ptr, X.ptr + 4 * nq * D,
                       None if v is None else X.ptr + 4 * (nq + H) * D, w, w, QN, KN, QO, nq, D, True, 10000.0, EPS)
        out.append([QO.read(np.float32)] + dev.codes() + dev.scales())
    assert all(np.array_equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("nq,H,D,rot,page", [(6, 2, 144, 144, 32), (4, 2, 192, 48, 16), (3, 1, 240, 240, 64), (2, 2, 208, 0, 128)])
def test_append_heads_between_the_widths(gpu, nq, H, D, rot, page):
    rng = np.random.default_rng(D)
    per = 3 + 128 // page
    cache = ref.Cache(3 * per, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, 3, per, cache.P)
    past = [0, 7, 0]
    for rows in ([1, 9, 37], [18, 0, 3], [2, 1, 16]):
        run_append(gpu, cache, dev, rng, rows, past, tables, nq, rot)
        check_cache(cache, dev, tables, rows, past)
        past = [p + r for p, r in zip(past, rows)]
    assert cache.near < 20


# ---- attention -------------------------------------------------------------------------------
@pytest.mark.parametrize("nq,H,D,page,rows,past,window,max_pages,kernel", STREAMS)
def test_attention_of_codes_by_the_caches(gpu, nq, H, D, page, rows, past, window, max_pages, kernel):
    rng = np.random.default_rng(D + window % 1000)
    per = max(-(-(p + r) // page) for p, r in zip(past, rows)) + 1
    cache = ref.Cache(len(rows) * per + 2, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = np.full((len(rows), max_pages), 0xffffffff, np.uint32)
    tables[:, :per] = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    want, bound = ref.attention(cache, rows, past, tables[:, :per], q, 0.1, window)
    got = run_attn(gpu, dev, rows, past, tables, q, 0.1, window)
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())


@pytest.mark.parametrize("nq,H,D,page,rows,past,window,bounds,kernel", PROMPTS)
def test_attention_of_prompts_by_bounds(gpu, nq, H, D, page, rows, past, window, bounds, kernel):
    """bounds: num_rows and max_rows as the host gives them, also below what seq_start says: rows past
    them are not touched."""
    rng = np.random.default_rng(D + rows[0])
    per = max(-(-(p + r) // page) for p, r in zip(past, rows))
    cache = ref.Cache(len(rows) * per, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    got = run_attn(gpu, dev, rows, past, tables, q, 0.1, window, num_rows=bounds[0], max_rows=bounds[1])
    at = 0
    for b, n in enumerate(rows):
        live = max(0, min(n, bounds[1], bounds[0] - at))
        for i in sorted(set(list(range(0, live, 23)) + [live - 1])) if live else []:
            want, bound = ref.attention(cache, [1], [past[b] + i], tables[b:b + 1], q[at + i:at + i + 1], 0.1, window)
            assert np.all(np.abs(got[at + i:at + i + 1] - want) <= bound), (b, i)
        assert np.all(got[at + live:at + n] == 5.0), b
        at += n


# ---- a cache of more than 4 GiB --------------------------------------------------------------
def test_pages_past_32_bits_of_bytes(gpu):
    """Codes of 4.3 GiB each of keys and values, of which only the last pages and the first are named, against the
    same calls on a small cache: the same bits."""
    nq, H, D, page = 8, 4, 512, 64
    pages = (1 << 32) // (page * H * D) + 2000
    rng = np.random.default_rng(77)
    rows, past = [70, 3], [0, 0]
    qkv, qn, kn = packed_rows(rng, sum(rows), nq, H, D)
    w, sides = (nq + 2 * H) * D, []
    for n, names in ((4, [3, 0, 2, 1]), (pages, [pages - 1, 0, pages - 2, pages - 1000])):
        tables = np.array([[names[0], names[1]], [names[2], names[3]]], np.uint32)
        c = gh.Kv8Cache(None, None, None, None, n, page, H, D)
        codes, scales = gh.lib().gh_kv8_code_bytes(c), gh.lib().gh_kv8_scale_bytes(c)
        assert codes == n * page * H * D and (n == 4 or codes > 1 << 32)
        held = [gpu.alloc(b) for b in (codes, codes, scales, scales)]
        c.k, c.v, c.k_scale, c.v_scale = (h.ptr for h in held)
        start, P, T = (gpu.upload(np.asarray(a, np.uint32)) for a in (np.concatenate([[0], np.cumsum(rows)]), past, tables))
        b = gh.Kv8Batch(start.ptr, P.ptr, T.ptr, 2, 2, sum(rows), max(rows))
        X, QN, KN, Q = gpu.upload(qkv), gpu.upload(qn), gpu.upload(kn), gpu.alloc(sum(rows) * nq * D * 4)
        gpu.kv8_append(c, b, X.ptr, X.ptr + 4 * nq * D, X.ptr + 4 * (nq + H) * D, w, w, QN, KN, Q, nq, D, False, 10000.0, EPS)
        K, V, O = (gpu.alloc(sum(rows) * h * D * 4) for h in (H, H, nq))
        gpu.kv8_read(c, b, K, V)
        size = gpu.kv8_attn_workspace(c, b, nq, 0, 70)
        W = gpu.alloc(max(size, 16))
        gpu.kv8_attn(c, b, Q, O, nq, 0.0442, 0, 70, W, size)
        sides.append([x.read(np.uint32) for x in (Q, K, V, O)])
        for h in held:
            h.free()
    for one, two in zip(*sides):
        assert np.array_equal(one, two)
    assert np.isfinite(sides[0][3].view(np.float32)).all()
