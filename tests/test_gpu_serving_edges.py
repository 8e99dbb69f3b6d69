"""Calls of the batched serving operators that their documentation allows at its edges: addresses of
any element, many query heads of one key head, pages that sequences share, tables without an end."""
import numpy as np
import pytest

import kv8_ref as ref
from test_gpu_kv8 import RUNS, run_attn, tables_of
from test_gpu_sample import drafted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_off,v_off", [(4, 0), (0, 8), (12, 4)])
def test_read_to_any_address(gpu, k_off, v_off):
    H, D, page = 2, 48, 32
    rng = np.random.default_rng(k_off + v_off)
    cache = ref.Cache(5, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    rows, past, tables = [19, 4], [7, 30], np.array([[4, 1], [0, 2]], np.uint32)
    K, V = (gpu.upload(np.full(23 * H * D + 16, 7.0, np.float32)) for _ in "kv")
    gpu.kv8_read(dev.cache, dev.batch(rows, past, tables), K.ptr + k_off, V.ptr + v_off)
    for which, buffer, off in ((0, K, k_off), (1, V, v_off)):
        got = buffer.read(np.float32)
        want = np.concatenate([cache.rows(which, tables[b], past[b], rows[b])[0] for b in range(2)]).reshape(-1)
        at = off // 4
        assert np.array_equal(got[at:at + want.size], want.astype(np.float32))
        assert np.all(got[:at] == 7.0) and np.all(got[at + want.size:] == 7.0)


@pytest.mark.parametrize("nq,H,D,rows,past,window", [(64, 1, 64, [2, 1], [40, 300], 0), (64, 1, 64, [260], [0], 0),
                                                     (70, 2, 96, [1, 5], [90, 3], 11), (70, 2, 96, [150], [20], 33),
                                                     (33, 1, 256, [280], [1], 0)])
@RUNS
def test_attention_of_many_heads_on_one(gpu, run, nq, H, D, rows, past, window):
    # more query heads a key head than a tile has columns
    page = 32
    rng = np.random.default_rng(nq + rows[0])
    per = max(-(-(p + r) // page) for p, r in zip(past, rows))
    cache = ref.Cache(len(rows) * per, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = tables_of(rng, len(rows), per, cache.P)
    q = rng.standard_normal((sum(rows), nq, D)).astype(np.float32)
    got = run(gpu, dev, rows, past, tables, q, 0.1, window)
    at = 0
    for b, n in enumerate(rows):
        for i in sorted(set(range(0, n, 37)) | {n - 1}):
            want, bound = ref.attention(cache, [1], [past[b] + i], tables[b:b + 1], q[at + i:at + i + 1], 0.1, window)
            assert np.all(np.abs(got[at + i:at + i + 1] - want) <= bound), (b, i)
        at += n


@RUNS
def test_attention_over_shared_pages(gpu, run):
    # two sequences with the same first pages, a page twice in one table
    nq, H, D, page = 4, 2, 64, 32
    rng = np.random.default_rng(3)
    cache = ref.Cache(6, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = np.array([[2, 4, 1, 0], [2, 4, 5, 4]], np.uint32)
    q = rng.standard_normal((3, nq, D)).astype(np.float32)
    rows, past = [1, 2], [70, 110]
    want, bound = ref.attention(cache, rows, past, tables, q, 0.1, 0)
    assert np.all(np.abs(run(gpu, dev, rows, past, tables, q, 0.1, 0) - want) <= bound)


def test_attention_with_scales_of_either_sign_and_none(gpu):
    nq, H, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(14)
    cache = ref.Cache(9, page, H, D, rng)
    dev = ref.Device(gpu, cache)
    tables = np.arange(9, dtype=np.uint32)[None]
    q = rng.standard_normal((2, nq, D)).astype(np.float32)
    for scale in (-0.2, 0.0, 1e-30):
        want, bound = ref.attention(cache, [2], [140], tables, q, scale, 0)
        assert np.all(np.abs(run_attn(gpu, dev, [2], [140], tables, q, scale, 0) - want) <= bound), scale


@pytest.mark.parametrize("offset", [4, 8, 12])
def test_verification_of_rows_at_any_address(gpu, offset):
    B, n, V = 5, 2, 8192
    rng = np.random.default_rng(offset)
    p, q, tokens = drafted(rng, B, n, V, 0.5)
    u, pick = rng.random((B, n), np.float32), rng.random(B, np.float32)
    T, D = gpu.alloc(p.nbytes + 16), gpu.alloc(q.nbytes + 16)
    T.write(p, offset)
    D.write(q, offset)
    K, U, I = gpu.upload(tokens), gpu.upload(u), gpu.upload(pick)
    O, A = gpu.alloc(B * (n + 1) * 4), gpu.alloc(B * 4)
    size = gpu.spec_verify_workspace(B, V)
    W = gpu.alloc(size)
    gpu.spec_verify(T.ptr + offset, D.ptr + offset, K, None, U, I, O, A, B, n, V, W, size)
    want = ref.verify(p, q, tokens, [n] * B, u, pick)
    assert np.array_equal(O.read(np.uint32).reshape(B, n + 1), want[0]) and np.array_equal(A.read(np.uint32), want[1])
