"""A compressed model, its scores and answers drawn from them: the operators as the algorithms use them, captured, on streams, from threads."""
import math
import pickle
import threading

import numpy as np
import pytest
import scipy.sparse as sp
import torch

from test_gpu_ops import GRID, gen, quantised_reference, random_mxfp4, sample_reference, values_of  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def data():
    from recpack_amd.synth import powerlaw_csr

    return powerlaw_csr(700, 333, 0.03, seed=11).to_scipy()


@pytest.fixture(scope="module")
def ease(data):
    from recpack_amd import EASE

    return EASE(l2=30.0).fit(data)


@pytest.fixture(scope="module")
def small(ease):
    return ease.compress(profiles=True)


def full_scores(X, S):
    return np.asarray(X @ S)


def test_compress_is_the_quantised_model(ease, small, data):
    B = ease._model.dense_download().astype(np.float64)
    S = small.similarity_matrix_.toarray()
    np.testing.assert_array_equal(S, quantised_reference(B)[2])
    np.testing.assert_array_equal(values_of(small._columns), quantised_reference(B.T)[2])
    assert small.nbytes < 2 * 333 * (11 * 17 + 16)
    # the largest step is 2 of 8 (values 4 and 6 below the power of two 8), rounded to the nearest; past 6 the value is cut: 2 of 8 at most
    nb = -(-333 // 32)
    pad = np.zeros((333, nb * 32))
    pad[:, :333] = np.abs(B)
    top = np.repeat(pad.reshape(333, nb, 32).max(-1), 32, axis=1)[:, :333]
    assert (np.abs(S - B) <= top * 0.25 + 1e-300).all()


def test_fit_is_ease_then_compress(small, data):
    from recpack_amd import CompressedEASE

    c = CompressedEASE(l2=30.0).fit(data)
    assert (c.similarity_matrix_ != small.similarity_matrix_).nnz == 0
    with pytest.raises(ValueError, match="profiles=True"):
        c.profile_scores(np.zeros((1, 333)))


def test_scores_and_predict(small, data):
    S = small.similarity_matrix_.toarray()
    want = full_scores(data, S)
    bound = 2 * (np.diff(data.indptr)[:, None] + 1) * 2.0 ** -24 * full_scores(data, np.abs(S)) + 1e-30
    got = small.scores(data).double().cpu().numpy()
    assert (np.abs(got - want) <= bound).all()
    P = small.predict(data)
    assert P.shape == data.shape and (np.abs(P.toarray() - want) <= bound).all()
    w = np.random.default_rng(3).random(data.nnz).astype(np.float32)
    Xw = sp.csr_matrix((w.astype(np.float64), data.indices, data.indptr), shape=data.shape)
    got = small.scores(data, weights=w, exclude_history=True).cpu().numpy()
    mask = data.toarray() != 0
    assert np.isneginf(got[mask]).all()
    assert (np.abs(got.astype(np.float64) - full_scores(Xw, S))[~mask] <= bound[~mask]).all()


def test_predict_topk(small, data):
    s = small.scores(data, exclude_history=True).cpu().numpy()
    got = small.predict_topk(data, 20, exclude_history=True, exclude_items=[1, 2, 3])
    s[:, [1, 2, 3]] = -np.inf
    for u in range(data.shape[0]):
        x = np.where(s[u] == 0, -np.inf, s[u])
        order = np.argsort(-x, kind="stable")[:20]
        order = np.sort(order[x[order] > -np.inf])
        row = got.indices[got.indptr[u]:got.indptr[u + 1]]
        np.testing.assert_array_equal(row, order)
        np.testing.assert_array_equal(got.data[got.indptr[u]:got.indptr[u + 1]], s[u][order].astype(np.float64))
    with pytest.raises(ValueError, match="1024"):
        from recpack_amd import CompressedEASE

        big = CompressedEASE()
        big.n_items_, big._rows, big._columns = 5000, random_mxfp4(__import__("recpack_amd").ops, 5000, 5000, 1), None
        big.predict_topk(sp.csr_matrix((2, 5000)), 2000)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 7, 300])
def test_profile_scores(small, dtype, m):
    P = torch.randn(m, 333, generator=gen(m)).to(dtype)
    W = values_of(small._columns)  # rows: items that are scored
    want = P.double().numpy() @ W.T
    got = small.profile_scores(P, dtype=torch.float32)
    bound = 8 * math.sqrt(3 * 333) * 2.0 ** -23 * (np.abs(P.double().numpy()) @ np.abs(W).T) + 1e-30
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


def check_draws(items, probs, scores, u, temperature, top_p, min_p, K):
    rows = scores.shape[0]
    want = sample_reference(scores.astype(np.float64), u.astype(np.float64), np.full(rows, np.float64(np.float32(temperature))), np.full(rows, K), np.full(rows, np.float64(np.float32(top_p))),
                            np.full(rows, np.float64(np.float32(min_p))))
    np.testing.assert_array_equal(items, want[0])
    np.testing.assert_allclose(probs, want[1], rtol=2.0 ** -24 + 1e-9)


@pytest.mark.parametrize("n,K,temperature,top_p,min_p", [(1, 0, 0.05, 0.9, 0.0), (10, 50, 0.02, 1.0, 0.001), (5, 333, 0.0, 1.0, 0.0)])
def test_compressed_predict_sample(small, data, n, K, temperature, top_p, min_p):
    u = np.random.default_rng(5).random((data.shape[0], n), dtype=np.float32)
    s = small.scores(data, exclude_history=True).cpu().numpy()
    items, probs = small.predict_sample(data, n, K, temperature, top_p, min_p, exclude_history=True, u=u)
    check_draws(items, probs, np.where(s == 0, -np.inf, s), u, temperature, top_p, min_p, K)
    again = small.predict_sample(data, n, K, temperature, top_p, min_p, exclude_history=True, seed=9)
    once = small.predict_sample(data, n, K, temperature, top_p, min_p, exclude_history=True, seed=9)
    np.testing.assert_array_equal(again[0], once[0])


def test_predict_sample_of_every_algorithm(ease, data):
    from recpack_amd import ItemKNN, TARSItemKNN, TimedInteractions

    knn = ItemKNN(K=30).fit(data)
    coo = data.tocoo()
    log = TimedInteractions(coo.row, coo.col, np.random.default_rng(1).integers(1, 10 ** 6, data.nnz), data.shape)
    tars = TARSItemKNN(K=30, fit_decay=1e-6, predict_decay=1e-6, similarity="cosine").fit(log)
    u = np.random.default_rng(2).random((data.shape[0], 6), dtype=np.float32)
    for algo, X in ((ease, data), (knn, data), (tars, log)):
        top = algo.predict_topk(X, 40, exclude_history=True)
        items, probs = algo.predict_sample(X, 6, K=40, temperature=0.1, top_p=0.95, exclude_history=True, u=u)
        dense = np.full(data.shape, -np.inf)
        rows = np.repeat(np.arange(data.shape[0]), np.diff(top.indptr))
        dense[rows, top.indices] = top.data
        check_draws(items, probs, dense, u, 0.1, 0.95, 0.0, 40)
        best, _ = algo.predict_sample(X, 6, K=40, temperature=0.0, exclude_history=True)
        for r in range(0, data.shape[0], 50):
            order = np.argsort(-dense[r], kind="stable")[:6]
            order = order[dense[r][order] > -np.inf]
            np.testing.assert_array_equal(best[r][:len(order)], order)
            assert (best[r][len(order):] == -1).all()
    with pytest.raises(ValueError, match="1 <= K"):
        knn.predict_sample(data, 2, K=0)
    with pytest.raises(ValueError, match="n = 0"):
        knn.predict_sample(data, 0)
    with pytest.raises(ValueError, match="u has shape"):
        knn.predict_sample(data, 2, u=np.zeros((3, 3)))
    with pytest.raises(ValueError):
        knn.predict_sample(data, 2, exclude_items=[])


def test_no_users(ease, small):
    empty = sp.csr_matrix((0, 333))
    assert small.predict_topk(empty, 5).shape == (0, 333)
    assert tuple(small.scores(empty).shape) == (0, 333)
    for algo in (small, ease):
        items, probs = algo.predict_sample(empty, 3, K=10)
        assert items.shape == probs.shape == (0, 3)
    # users without a history, among others
    X = sp.csr_matrix((np.ones(3), ([1, 1, 3], [0, 5, 7])), shape=(5, 333))
    for algo in (small, ease):
        items, probs = algo.predict_sample(X, 2, K=10, seed=1)
        assert (items[[0, 2, 4]] == -1).all() and (probs[[0, 2, 4]] == 0).all() and (items[[1, 3]] >= 0).all()


def test_pickle(small, data):
    other = pickle.loads(pickle.dumps(small))
    assert torch.equal(other.scores(data), small.scores(data))
    assert torch.equal(other.profile_scores(np.ones((2, 333))), small.profile_scores(np.ones((2, 333))))
    assert other.get_params() == small.get_params()


def test_compress_refusals(ease):
    from recpack_amd import CompressedEASE, ItemKNN

    with pytest.raises(Exception):
        CompressedEASE().predict(sp.csr_matrix((1, 333)))
    with pytest.raises(ValueError, match="items"):
        ease.compress().scores(sp.csr_matrix((1, 5)))
    knn = ItemKNN(K=3).fit(sp.csr_matrix(np.eye(5) + np.eye(5, k=1)))
    with pytest.raises(ValueError, match="dense model"):
        CompressedEASE()._compress(knn._model)


# ---- captured, on streams, from threads -------------------------------------------------------------------------------------------------------

def chain(ops, ctx, B, indptr, indices, u):
    """Compress, score, draw; and the dense product beside it."""
    rows = ops.mxfp4_quantize(ctx, B)
    s = ops.mxfp4_scores(ctx, indptr, indices, rows, exclude_history=True)
    one = ops.sample(ctx, s, u[:, :1].contiguous(), temperature=0.5, top_p=0.9)
    slate = ops.sample(ctx, s, u, temperature=0.5, top_k=100)
    cols = ops.mxfp4_quantize(ctx, B, transpose=True)
    dense = ops.mxfp4_gemm_nt(ctx, B[:70], cols)
    back = ops.mxfp4_dequantize(ctx, rows)
    return [s, *one, *slate, dense, back]


def chain_inputs(n, seed):
    g = gen(seed)
    B = torch.randn(n, n, generator=g) * 0.1
    counts = torch.randint(0, 40, (23,), generator=g)
    indptr = torch.zeros(24, dtype=torch.int32)
    indptr[1:] = counts.cumsum(0)
    indices = torch.randint(0, n, (int(indptr[-1]),), generator=g, dtype=torch.int32)
    return [t.cuda() for t in (B, indptr, indices, torch.rand(23, 8, generator=g))]


@pytest.mark.parametrize("n", [400, 3001])
def test_captured_and_replayed(n):
    from recpack_amd import get_context, ops

    ctx = get_context(0)
    inputs = chain_inputs(n, 1)
    eager = [t.clone() for t in chain(ops, ctx, *inputs)]
    graphs = []
    for _ in range(2):  # two graphs of the same calls: each has its own scratch memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = chain(ops, ctx, *inputs)
        graphs.append((g, out))
    for turn in range(3):
        inputs[0].mul_(1.5 if turn else 1.0)
        inputs[3].copy_(torch.rand(23, 8, generator=gen(50 + turn)))
        if turn == 0:
            inputs[3].copy_(chain_inputs(n, 1)[3])
        want = chain(ops, ctx, *inputs) if turn else eager
        for t in graphs[0][1] + graphs[1][1]:
            t.zero_()
        graphs[0][0].replay()
        junk = torch.full((1 << 20,), float("nan"), device="cuda").sum()  # the program's own work in between
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)
        assert junk.isnan()


def test_on_another_stream():
    from recpack_amd import get_context, ops

    ctx = get_context(0)
    want = [t.clone() for t in chain(ops, ctx, *chain_inputs(1500, 2))]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        inputs = chain_inputs(1500, 2)
        for t in inputs:  # produced late on this stream, nothing waited for on the host
            t.copy_(t + 0)
        out = chain(ops, ctx, *inputs)
    stream.synchronize()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


def test_from_threads():
    from recpack_amd import get_context, ops

    ctx = get_context(0)
    want = {s: [t.clone() for t in chain(ops, ctx, *chain_inputs(900, s))] for s in (1, 2, 3)}
    wrong = []

    def work(seed):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            inputs = chain_inputs(900, seed)
            for _ in range(10):
                out = chain(ops, ctx, *inputs)
        stream.synchronize()
        if not all(torch.equal(a, b) for a, b in zip(out, want[seed])):
            wrong.append(seed)

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
