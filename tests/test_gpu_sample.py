"""Probabilities from logits and the verification of drafted tokens against 64-bit
numpy (kv8_ref.py)."""
import numpy as np
import pytest

import kv8_ref as ref

pytestmark = pytest.mark.gpu


def run_probs(gpu, x, cap, temperature, stride=None, vocab=None, offset=0, in_place=False):
    rows, width = x.shape
    stride, vocab = stride or width, vocab or width
    X = gpu.alloc(x.nbytes + 64)
    X.write(x, offset)
    P = X if in_place else gpu.upload(np.full(x.size + 16, 3.0, np.float32))
    n = gpu.logit_probs_workspace(rows, vocab)
    W = gpu.alloc(n)
    gpu.logit_probs(X.ptr + offset, P.ptr + offset, rows, vocab, stride, cap, temperature, W, n)
    return P.read(np.float32, x.size, offset).reshape(x.shape)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 262144), (3, 4095), (5, 4097), (2, 50001), (7, 8192), (40, 1003)])
@pytest.mark.parametrize("cap,temperature", [(0.0, 1.0), (30.0, 0.8), (5.0, 0.1)])
def test_probabilities(gpu, rows, vocab, cap, temperature):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    want, bound = ref.probabilities(x, cap, temperature)
    for in_place in (False, True):
        got = run_probs(gpu, x, cap, temperature, in_place=in_place)
        # (below 2^-126 a step is not relative any more)
        assert np.all(np.abs(got - want) <= bound * want + 2.0 ** -126)


def test_probabilities_rows_in_a_wider_matrix(gpu):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 1000)).astype(np.float32)
    for vocab, offset in ((996, 0), (997, 0), (996, 4), (1, 8)):
        want, bound = ref.probabilities(x[:, :vocab], 0.0, 1.0)
        got = run_probs(gpu, x, 0.0, 1.0, stride=1000, vocab=vocab, offset=offset)
        assert np.all(np.abs(got[:, :vocab] - want) <= bound * want + 2.0 ** -126)
        assert np.all(got[:2, vocab:] == 3.0)  # what lies between the rows


@pytest.mark.parametrize("cap", [0.0, 30.0, 0.5])
def test_probabilities_of_masked_and_broken_rows(gpu, cap):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((6, 9001)).astype(np.float32)
    x[0] = -np.inf
    x[1, rng.random(9001) < 0.999] = -np.inf
    x[2] = -np.inf
    x[2, 8000] = -3.4e38
    x[3, 77] = np.nan
    x[4, 5000] = np.inf
    x[5] = np.finfo(np.float32).min
    got = run_probs(gpu, x, cap, 1.0)
    assert not got[0].any() and np.isnan(got[3]).all()
    assert got[2, 8000] == 1 and got[2].sum() == 1
    assert np.allclose(got[5], 1 / 9001, rtol=1e-5)
    want, bound = ref.probabilities(x[[1]], cap, 1.0)
    assert np.all(np.abs(got[1] - want[0]) <= bound[0] * want[0] + 2.0 ** -126)
    if cap:
        want, bound = ref.probabilities(x[[4]], cap, 1.0)
        assert np.all(np.abs(got[4] - want[0]) <= bound[0] * want[0] + 2.0 ** -126)
    else:
        assert np.isnan(got[4]).all()


# ---- verification ----------------------------------------------------------------------------
def run_verify(gpu, target, draft, tokens, n_draft, u, pick):
    B, rows, V = target.shape
    up = lambda a, t: None if a is None else gpu.upload(np.asarray(a, t))  # noqa: E731
    T, D, K, N, U, I = (up(target, np.float32), up(draft, np.float32), up(tokens, np.uint32), up(n_draft, np.uint32),
                        up(u, np.float32), up(pick, np.float32))
    O, A = gpu.alloc(B * rows * 4), gpu.alloc(B * 4)
    n = gpu.spec_verify_workspace(B, V)
    W = gpu.alloc(n)
    gpu.spec_verify(T, D, K, N, U, I, O, A, B, rows - 1, V, W, n)
    return O.read(np.uint32).reshape(B, rows), A.read(np.uint32)


def softmax(x):
    e = np.exp(x - x.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def drafted(rng, B, n, V, noise):
    z = rng.standard_normal((B, n + 1, V)) * 2
    p, q = softmax(z), softmax(z[:, :n] + noise * rng.standard_normal((B, n, V)))
    tokens = np.array([[rng.choice(V, p=q[b, i].astype(np.float64) / q[b, i].astype(np.float64).sum()) for i in range(n)]
                       for b in range(B)], np.uint32).reshape(B, n)
    return p, q, tokens


@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (3, 2, 7), (16, 5, 4096), (9, 4, 4099), (5, 3, 50000), (2, 4, 262144), (4, 70, 33)])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verification(gpu, B, n, V, with_draft):
    rng = np.random.default_rng(V + n)
    p, q, tokens = drafted(rng, B, n, V, 0.6)
    draft = q if with_draft else None
    for turn in range(3):
        n_draft = None if turn == 0 else rng.integers(0, n + 2, B)  # (more than there are counts as all)
        u, pick = rng.random((B, n), np.float32), rng.random(B, np.float32)
        if turn == 2:
            u[:] = 0
        want = ref.verify(p, draft, tokens, [n] * B if n_draft is None else n_draft, u, pick)
        got = run_verify(gpu, p, draft, tokens, n_draft, u, pick)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verification_without_drafts(gpu):
    rng = np.random.default_rng(3)
    p = softmax(rng.standard_normal((4, 1, 9000)))
    pick = np.array([0.0, 0.25, 0.999, np.float32(1) - np.float32(2) ** -24], np.float32)
    got = run_verify(gpu, p, None, None, None, None, pick)
    want = ref.verify(p, None, np.zeros((4, 0)), [0] * 4, None, pick)
    assert np.array_equal(got[0], want[0]) and not got[1].any()


def test_verification_at_the_borders(gpu):
    V = 5000
    p = np.zeros((8, 2, V), np.float32)
    q = np.zeros((8, 1, V), np.float32)
    tokens = np.zeros((8, 1), np.uint32)
    u = np.full((8, 1), 0.5, np.float32)
    pick = np.full(8, 0.5, np.float32)
    p[0, 0, [10, 20]], q[0, 0, [10, 20]], tokens[0] = 0.5, 0.5, 10   # the same rows: kept (0.25 < 0.5)
    p[0, 1, [4094, 4097]] = 0.5                                    # pick 0.5 of 1: the sum at 4094 is not over it
    p[1, 0, 30], q[1, 0, 40], tokens[1] = 1.0, 1.0, 40              # certain of another: rejected, 30
    p[2, 0, [1, 2]], q[2, 0, [1, 2]], tokens[2] = 0.25, 0.5, 1      # 0.25 < 0.25 is false; nothing left over: the target itself
    p[3, 0, 3], q[3, 0, 3], tokens[3] = 1.0, 1.0, V                 # a token that is none
    p[4, 1], tokens[4], u[4], p[4, 0, 0], q[4, 0, 0] = 0, 0, 0, 1, 1  # kept, and then nothing to draw
    p[5, 0, 7], p[5, 0, 8], q[5, 0, 9], tokens[5], pick[5] = 0.5, 0.5, 1.0, 9, 1.5  # a share past the end: the last
    p[6, 0, 7], p[6, 0, 8], q[6, 0, 9], tokens[6], pick[6] = 0.5, np.nan, 1.0, 9, np.nan  # NaN weighs nothing, and is share 0
    p[7, 0, 7], q[7, 0, 9], tokens[7] = np.inf, 1.0, 9              # an infinite sum
    got, accepted = run_verify(gpu, p, q, tokens, None, u, pick)
    none = ref.NONE
    assert got.tolist() == [[10, 4097], [30, none], [2, none], [3, none], [0, none], [8, none], [7, none], [none, none]]
    assert accepted.tolist() == [1, 0, 0, 0, 1, 0, 0, 0]
