"""The 4-bit and sampling operators where rounding decides: far tails of wide rows, exact products in every tile shape, sums that must not depend on the batch."""
import decimal
import math

import numpy as np
import pytest
import torch

from test_gpu_ops import check_sample, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from recpack_amd import get_context

    return get_context(0)


@pytest.fixture(scope="module")
def ops():
    from recpack_amd import ops

    return ops


# ---- sampling: one best score and a flat tail far below ---------------------------------------------------------------------------------

def tail_draw(width, at, below, u, top_p=1.0, top_k=0):
    """The draw from a best score at index `at` and width - 1 equal ones `below` it, in 60 decimal digits: (index, probability)."""
    with decimal.localcontext(decimal.Context(prec=60)):
        D = decimal.Decimal
        m = (-D(below)).exp()
        n = min(top_k or width, width)  # kept ranks: the best one and n - 1 of the tail
        if top_p < 1:
            n = min(n, max(1, 1 + math.ceil((D(top_p) * (1 + (n - 1) * m) - 1) / m)))
        kept = 1 + (n - 1) * m
        want = (D(u) * kept - 1) / m
        if want < 0:
            return at, float(1 / kept)
        # a draw within a hundredth of a candidate from the border between two says nothing (a mass is right to 2^-32 of itself, 2^25 of them to 2^-7)
        assert D("0.01") < want % 1 < D("0.99"), want % 1
        k = int(want)
        return (k if k < at else k + 1), float(m / kept)


TAILS = [(100_000, 26.0, 1.0), (100_000, 13.0, 0.5), (30_001, 24.5, 1.0), (2 ** 20 + 1, 28.0, 1.0), (2 ** 20 + 1, 30.0, 1.0)]


@pytest.mark.parametrize("width,below,temperature", TAILS)
@pytest.mark.parametrize("rows", [1, 12, 64])
def test_sample_from_a_far_tail(ctx, ops, width, below, temperature, rows):
    """A tail of 1e-7 of the mass, an item of which has 1e-12: drawn by uniforms next to 1, with the item's own probability."""
    at = width // 3
    x = torch.full((width,), -below)
    x[at] = 0.0
    us = [1 - 2.0 ** -24, 1 - 2.0 ** -23, 1 - 3 * 2.0 ** -24, 0.5]
    x, u = x.cuda().expand(rows, width).contiguous(), torch.tensor([us[r % 4] for r in range(rows)]).view(rows, 1).cuda()
    for setting in (dict(), dict(top_p=1 - 2.0 ** -23), dict(top_k=width - 5), dict(min_p=1e-14)):
        idx, prob, n = ops.sample(ctx, x, u, temperature=temperature, **setting)
        want = [tail_draw(width, at, below / temperature, us[r % 4], setting.get("top_p", 1.0), setting.get("top_k", 0)) for r in range(min(rows, 4))]
        assert idx.view(-1).tolist() == [want[r % 4][0] for r in range(rows)]
        # the masses' sum is right to 2^-31, a mass to 2^-45; one rounding to float32
        np.testing.assert_allclose(prob.view(-1).double().cpu().numpy(), [want[r % 4][1] for r in range(rows)], rtol=2.0 ** -24 + 2.0 ** -30)
        assert (n == 1).all()
    idx, prob, _ = ops.sample(ctx, x, u, temperature=temperature, min_p=1e-9)  # (the tail is below it)
    assert (idx == at).all() and (prob == 1).all()


def test_sample_from_the_tail_of_a_very_wide_row(ctx, ops):
    """2^25 items 25.75 below the best one have 2.2e-4 of the mass together."""
    width, below, at = 2 ** 25 + 7, 25.75, 12_345
    x = torch.full((1, width), -below, device="cuda")
    x[0, at] = 0.0
    for u in (0.25, 1 - 2.0 ** -12 + 2.0 ** -14, 1 - 2.0 ** -13, 1 - 2.0 ** -24):
        for setting in (dict(), dict(top_p=1 - 2.0 ** -14), dict(top_k=2 ** 24)):
            idx, prob, _ = ops.sample(ctx, x, torch.tensor([[u]], device="cuda"), **setting)
            want = tail_draw(width, at, below, u, setting.get("top_p", 1.0), setting.get("top_k", 0))
            assert int(idx) == want[0]
            assert abs(float(prob) - want[1]) <= want[1] * (2.0 ** -24 + 2.0 ** -30)


@pytest.mark.parametrize("below", [5.0, 18.0, 23.0, 40.0])
def test_sample_from_a_tail_of_different_scores(ctx, ops, below):
    """The same with a tail of different scores, in extended precision: index and probability."""
    width = 100_000
    x = torch.randn(1, width, generator=gen(3)) - below
    x[0, 77] = 0.0
    order = np.argsort(-x[0].double().numpy(), kind="stable")
    m = np.exp(x[0].numpy().astype(np.longdouble)[order])
    c = np.cumsum(m)
    for u in (0.1, 0.9, 1 - 2.0 ** -12, 1 - 2.0 ** -20, 1 - 2.0 ** -23, 1 - 2.0 ** -24):
        k = int(np.searchsorted(c, np.longdouble(u) * c[-1], side="right"))
        idx, prob, _ = ops.sample(ctx, x.cuda(), torch.tensor([[u]], device="cuda"))
        assert int(idx) == order[k]
        assert abs(float(prob) - float(m[k] / c[-1])) <= float(m[k] / c[-1]) * (2.0 ** -24 + 2.0 ** -30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("top_k", [0, 3000])
def test_sample_alone_and_among_others(ctx, ops, dtype, top_k):
    """Few rows (slices of them) and many (a workgroup each): the same draws, bit for bit."""
    x = (torch.randn(70, 30_001, generator=gen(1)) * 4).to(dtype).cuda()
    u = torch.rand(70, 1, generator=gen(2)).cuda()
    for setting in (dict(), dict(temperature=0.3, top_p=0.9), dict(temperature=2.0, min_p=0.003)):
        many = ops.sample(ctx, x, u, top_k=top_k, **setting)
        for part in (slice(0, 1), slice(5, 25)):
            for a, b in zip(many, ops.sample(ctx, x[part], u[part], top_k=top_k, **setting)):
                assert torch.equal(a[part], b)


@pytest.mark.parametrize("rows", [3, 70])
def test_sample_min_p_on_a_border(ctx, ops, rows):
    """Scores whose mass is min_p, a step above and a step below it, in bins on either side of an octave's end."""
    width = 25_000
    for octaves in (1, 3, 31, 32, 40):
        x = torch.full((rows, width), -70.0)
        x[:, 5] = 0.0
        edge = np.float32(-octaves * math.log(2))
        for i, v in enumerate((np.nextafter(edge, np.float32(0)), edge, np.nextafter(edge, np.float32(-99)), edge * np.float32(1.004), edge * np.float32(0.996))):
            x[:, 100 + 50 * i] = float(v)
        u = torch.linspace(0, 1, rows).view(rows, 1) * (1 - 2.0 ** -24)
        check_sample(ctx, ops, x, u, min_p=2.0 ** -octaves)
        check_sample(ctx, ops, x, u, min_p=float(np.nextafter(np.float32(2.0 ** -octaves), np.float32(0))))


# ---- scores: the same bits alone and in any batch -----------------------------------------------------------------------------------------

def wide_mxfp4(ops, rows, cols, seed, lo, hi):
    nb = -(-cols // 32)
    codes = torch.randint(0, 256, (rows, nb * 16), generator=gen(seed), dtype=torch.uint8)
    if cols % 2:
        codes[:, cols // 2] &= 15
    codes[:, (cols + 1) // 2:] = 0
    return ops.MXFP4(codes.cuda(), torch.randint(lo, hi, (rows, nb), generator=gen(seed + 1), dtype=torch.uint8).cuda(), cols)


def batch_of(histories, times):
    """CSR of the given histories, one after the other, `times` times."""
    counts = torch.tensor([len(h) for h in histories] * times)
    indptr = torch.zeros(len(counts) + 1, dtype=torch.int32)
    indptr[1:] = counts.cumsum(0)
    return indptr.cuda(), torch.cat([torch.cat(histories)] * times).cuda()


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("items,times", [(2500, 700), (4101, 500), (12_300, 250)])
@pytest.mark.parametrize("lo,hi", [(117, 126), (0, 8), (3, 200)])
def test_scores_do_not_depend_on_the_batch(ctx, ops, weighted, items, times, lo, hi):
    """Few users (four waves to a tile of columns) and many (one): sums of many entries, bit for bit; within the bound of float32 sums."""
    w = wide_mxfp4(ops, items, items, items, lo, hi)
    sizes = [1, 3, 37, 64, 65, 133, 300, 9]
    histories = [torch.randint(0, items, (n,), generator=gen(n), dtype=torch.int32) for n in sizes]
    histories[3][::7] = -1  # (entries that count nothing move the others together)
    indptr, indices = batch_of(histories, times)
    one = torch.randn(sum(sizes), generator=gen(5)).cuda() if weighted else None
    kw = dict(exclude_history=True) if items == 2500 else {}
    got = ops.mxfp4_scores(ctx, indptr, indices, w, weights=None if one is None else one.repeat(times), **kw)
    few_ptr, few_indices = batch_of(histories, 1)
    few = ops.mxfp4_scores(ctx, few_ptr, few_indices, w, weights=one, **kw)
    assert torch.equal(got.view(times, len(sizes), items)[[0, 1, times - 1]].contiguous(), few.expand(3, -1, -1).contiguous())
    at = 0
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
    for u, h in enumerate(histories):
        part = None if one is None else one[at:at + len(h)]
        alone = ops.mxfp4_scores(ctx, torch.tensor([0, len(h)], dtype=torch.int32).cuda(), h.cuda(), w, weights=part, **kw)
        assert torch.equal(alone[0], few[u])
        h, f = h.long(), torch.ones(len(h), dtype=torch.float64) if part is None else part.double().cpu()
        h, f = h[h >= 0], f[h >= 0]
        codes = w.codes.cpu()[h].long()
        V = torch.stack((lut[codes & 15], lut[codes >> 4]), -1).view(len(h), -1) * torch.exp2(w.scales.cpu()[h].double() - 127).repeat_interleave(32, 1)
        want, size = (f[:, None] * V).sum(0)[:items], (f[:, None] * V).abs().sum(0)[:items]
        # n adds (and products), each off by at most half a step of at most the sum of the magnitudes (or of float32's least number)
        bound = (len(h) + 1) * (2.0 ** -23 * size + 2.0 ** -149)
        gone = torch.isneginf(alone[0].cpu())
        assert bool((((alone[0].double().cpu() - want).abs() <= bound) | gone).all())
        assert int(gone.sum()) == (len(set(h.tolist())) if kw else 0)
        at += sizes[u]


# ---- products: the documented limits -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,dtype", [(1, torch.float32), (2, torch.bfloat16), (4, torch.float32), (5, torch.float16)])
def test_product_with_the_most_rows_of_w(ctx, ops, m, dtype):
    """N = 2^28, more workgroups of 16 rows than a launch takes: the rows at the ends and where the launches meet are those of a small product."""
    n, k = 2 ** 28, 32
    w = ops.MXFP4.empty(n, k, "cuda")
    w.codes.random_(generator=torch.Generator(device="cuda").manual_seed(m))
    w.scales.random_(120, 127, generator=torch.Generator(device="cuda").manual_seed(9))
    a = torch.randn(m, k, generator=gen(m)).to(dtype).cuda()
    got = ops.mxfp4_gemm_nt(ctx, a, w)
    at = torch.tensor([0, 1, 63, 2 ** 26 + 5, 2 ** 27 - 1, 2 ** 27, 2 ** 27 + 17, 2 ** 28 - 17, 2 ** 28 - 16, 2 ** 28 - 1], device="cuda")
    few = ops.mxfp4_dequantize(ctx, ops.MXFP4(w.codes[at].contiguous(), w.scales[at].contiguous(), k)).double()
    want, size = a.double() @ few.t(), a.double().abs() @ few.t().abs()
    # 32 products in three planes at most, a step (2^-23) of the magnitudes' sum each at most; one rounding
    assert bool(((got[:, at].double() - want).abs() <= 96 * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs()).all())
    for part in got.view(-1).split(2 ** 28):
        assert bool(part.isfinite().all())


def normal_mxfp4(ops, n, k, seed, scale=127):
    w = wide_mxfp4(ops, n, k, seed, 0, 1)
    w.scales.fill_(scale)
    return w


@pytest.mark.parametrize("m,n,k", [(40, 5003, 5000), (300, 9001, 700), (9, 2000, 9000)])
def test_product_f16_rows_beside_a_wide_one(ctx, ops, m, n, k):
    """Rows of W beside one whose scales lie more than 2^36 apart: their sums are the same bits as without it; that row's are right."""
    a = torch.randn(m, k, generator=gen(m)).half().cuda()
    w = normal_mxfp4(ops, n, k, 4)
    rows = [3, 16, 700, 702, 703, n - 1]
    w.codes[rows, :16] = 0  # (a block of zeros: it takes any scale without a change)
    without = ops.mxfp4_gemm_nt(ctx, a, w, dtype=torch.float32)
    w.codes[rows, 0] = 0x21  # 0.5 and 1.0, once 2^-40 of the others
    w.scales[rows, 0] = 127 - 40
    with_them = ops.mxfp4_gemm_nt(ctx, a, w, dtype=torch.float32)
    others = [r for r in range(n) if r not in rows]
    assert torch.equal(with_them[:, others], without[:, others])
    few = ops.mxfp4_dequantize(ctx, ops.MXFP4(w.codes[rows].contiguous(), w.scales[rows].contiguous(), k)).double()
    want, size = a.double() @ few.t(), a.double().abs() @ few.t().abs()
    assert bool(((with_them[:, rows].double() - want).abs() <= 8 * math.sqrt(2 * k) * 2.0 ** -23 * size).all())
    # a row of A that meets nothing but the small block: exact
    one = torch.zeros(m, k)
    one[:, 0], one[:, 1] = torch.arange(m) + 1.0, 0.25
    got = ops.mxfp4_gemm_nt(ctx, one.half().cuda(), w, dtype=torch.float32)[:, rows].cpu()
    assert torch.equal(got, ((one[:, :1] * 0.5 + 0.25) * 2.0 ** -40).expand(-1, len(rows)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(2, 64, 64), (16, 64, 64), (40, 5000, 5000)])
def test_product_from_the_least_to_the_largest_number(ctx, ops, dtype, m, n, k):
    """One element per row of A, of every power of two, against 1 and 2^100: exact; below 2^-110 a float32 element may lose the bits under 2^-133."""
    i = torch.arange(m)
    for scale in (127, 227):
        w = normal_mxfp4(ops, n, k, 1, scale)
        w.codes.zero_()
        w.codes[i, i // 2] = torch.where(i % 2 == 0, 2, 32).to(torch.uint8).cuda()  # 1.0 on the diagonal
        a = torch.zeros(m, k, dtype=dtype, device="cuda")
        g = gen(m + scale)
        for e in range(-149, 128):
            v = (torch.randint(1 << 23, 1 << 24, (m,), generator=g).double() * 2.0 ** (e - 23)).to(dtype)
            if not bool(v.isfinite().all()):
                continue
            a[i, i] = v.cuda()
            got = ops.mxfp4_gemm_nt(ctx, a, w, dtype=torch.float32).diagonal()[:m].cpu()
            want = (v.double() * 2.0 ** (scale - 127)).float()
            if dtype == torch.float32 and e < -110:
                assert bool(((got.double() - want.double()).abs() <= 2.0 ** (-133 + scale - 127)).all())
            else:
                assert torch.equal(got, want)


EVERY_TILE = [
    (torch.float32, 1, 3000, 2048), (torch.float32, 4, 5003, 7001), (torch.bfloat16, 2, 2001, 4100), (torch.float16, 1, 3000, 5000),  # few rows
    (torch.float32, 97, 1999, 2003), (torch.bfloat16, 64, 1000, 1000), (torch.float16, 33, 2000, 2000),                              # one launch
    (torch.float32, 9, 2000, 5001), (torch.float16, 16, 20001, 5000), (torch.bfloat16, 16, 2001, 4200),                              # 16 x 64, K in parts
    (torch.bfloat16, 33, 3001, 6000), (torch.float16, 64, 999, 9000), (torch.float32, 40, 4001, 4096), (torch.float32, 64, 9000, 9000),  # 64 x 64
    (torch.bfloat16, 130, 20001, 8100), (torch.float32, 200, 9001, 4000), (torch.float16, 300, 8001, 8001),                          # 128 x 128, K in parts
    (torch.bfloat16, 1100, 8010, 200), (torch.float16, 1100, 8010, 330), (torch.float32, 1100, 8010, 130),                           # 128 x 256
    (torch.bfloat16, 2050, 8200, 257), (torch.float16, 2050, 8200, 90),                                                              # 256 x 256
    (torch.bfloat16, 1500, 12001, 4200), (torch.float16, 2001, 12000, 4200), (torch.float32, 1500, 12001, 4200), (torch.float16, 300, 30001, 4300),  # the last round in parts
    ("mxfp4", 20, 700, 9000), ("mxfp4", 30, 40001, 3000), ("mxfp4", 90, 1501, 17000), ("mxfp4", 200, 1999, 5000), ("mxfp4", 600, 3001, 1000), ("mxfp4", 1000, 8000, 3000),
    ("mxfp4", 4000, 4200, 300), ("mxfp4", 1500, 12003, 8300)]


@pytest.mark.parametrize("dtype,m,n,k", EVERY_TILE)
def test_product_is_exact_in_every_tile(ctx, ops, dtype, m, n, k):
    """One element per row of A: C holds its products with a column of W, bit for bit.  (A plane of A left out, a fragment or a part of K in
    another's place or added twice changes nearly all of them; the bounds of sums over K would let a lost third plane pass.)"""
    g = gen(m + n + k)
    at = torch.randint(0, k, (m,), generator=g)
    at[0], at[-1] = 0, k - 1
    if m > 40:
        at[1:40] = torch.arange(k - 40, k - 1)
    i = torch.arange(m)
    w = wide_mxfp4(ops, n, k, n + k, 110, 146)  # (within 2^36: f16 in one pass)
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6], device="cuda")
    sign = torch.randint(0, 2, (m,), generator=g) * 2.0 - 1

    def column(q, rows, cols):  # the values at (rows, cols), one column for each
        byte = q.codes[rows, cols // 2].long()
        return lut[torch.where(cols % 2 == 0, byte & 15, byte >> 4)] * torch.exp2(q.scales[rows, cols // 32].float() - 127)

    if dtype == "mxfp4":
        a = wide_mxfp4(ops, m, k, m, 100, 150)
        a.codes.zero_()
        a.codes[i, at // 2] = (torch.randint(1, 8, (m,), generator=g) << (at % 2 * 4)).to(torch.uint8).cuda()
        v = column(a, i.cuda(), at.cuda())
    else:
        bits = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}[dtype]
        v = (torch.randint(1 << (bits - 1), 1 << bits, (m,), generator=g) | (0x8001 if bits == 24 else 1)).double() * torch.exp2(torch.randint(-14, 5, (m,), generator=g).double() + 1 - bits) * sign
        a = torch.zeros(m, k, dtype=dtype)
        a[i, at] = v.to(dtype)
        assert torch.equal(a[i, at].double(), v)
        if dtype == torch.float32:
            w.codes.copy_(torch.tensor([1, 2, 4, 6, 9, 10, 12, 14], dtype=torch.uint8, device="cuda")[w.codes.long() & 7] * 17)  # powers of two
            w.codes[:, (k + 1) // 2:] = 0
            if k % 2:
                w.codes[:, k // 2] &= 15
            # two planes of bf16 do not hold any of these elements
            high = (v.float().view(torch.int32) & -65536).view(torch.float32)
            rest = ((v.float() - high).view(torch.int32) & -65536).view(torch.float32)
            assert bool((high + rest != v.float()).all())
        a, v = a.cuda(), v.float().cuda()
    want = v[:, None] * column(w, torch.arange(n, device="cuda")[None, :], at.cuda()[:, None].expand(m, n))
    assert int((want != 0).sum()) > m * n // 2
    assert torch.equal(ops.mxfp4_gemm_nt(ctx, a, w, dtype=torch.float32), want)


# ---- the compressed model's inputs -------------------------------------------------------------------------------------------------------------

def test_scores_of_every_sparse_format():
    import scipy.sparse as sp

    from recpack_amd import EASE
    from recpack_amd.synth import powerlaw_csr

    X = powerlaw_csr(90, 90, 0.1, seed=3).to_scipy()
    model = EASE(l2=10.0).fit(X).compress()
    want = model.scores(X, exclude_history=True)
    for kind in ("csc", "coo", "lil"):
        assert torch.allclose(model.scores(X.asformat(kind), exclude_history=True), want, rtol=1e-5, atol=1e-6)  # (entries of a row in another order)
    assert torch.equal(model.scores(sp.csr_array(X), exclude_history=True), want)
    with pytest.raises(ValueError, match="CSR"):
        model.scores(X.tocsc(), weights=np.ones(X.nnz))


# ---- calls that other tests do not make ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,width", [(1, 100_000), (3, 30_001), (20, 30_001), (70, 5_000)])
@pytest.mark.parametrize("top_k", [0, 2000])
def test_draws_from_long_prefixes_captured(ctx, ops, rows, width, top_k):
    """Every form of the whole-row draw in a graph, replayed on other scores, settings and uniforms."""
    x, u = torch.empty(rows, width, device="cuda"), torch.empty(rows, 1, device="cuda")
    t, p, m = (torch.empty(rows, device="cuda") for _ in range(3))

    def fill(turn):
        g = gen(turn)
        x.copy_(torch.randn(rows, width, generator=g) * (1 + 5 * turn))
        if turn == 2:
            x[0] = -math.inf  # (a row without candidates, after rows with some)
        for v, lo, size in ((u, 0.0, 1.0), (t, 0.3, 1.0), (p, 0.5, 0.5), (m, 0.0, 1e-3)):
            v.copy_(torch.rand(v.shape, generator=g) * size + lo)
        u.clamp_(max=1 - 2.0 ** -24)

    def call():
        return ops.sample(ctx, x, u, temperature=t, top_k=top_k, top_p=p, min_p=m)

    fill(0)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn in range(5):
        fill(turn)
        want = [v.clone() for v in call()]
        for v in out:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_scores_captured_with_other_histories(ctx, ops):
    """Row pointers are read when the graph runs: shorter, longer and empty histories in the same buffers."""
    items, users, room = 3000, 40, 4000
    w = wide_mxfp4(ops, items, items, 1, 117, 126)
    indptr, indices, weights = torch.zeros(users + 1, dtype=torch.int32, device="cuda"), torch.zeros(room, dtype=torch.int32, device="cuda"), torch.zeros(room, device="cuda")

    def call():
        return [ops.mxfp4_scores(ctx, indptr, indices, w, exclude_history=True), ops.mxfp4_scores(ctx, indptr, indices, w, weights=weights, dtype=torch.bfloat16)]

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn in range(4):
        g = gen(turn)
        counts = torch.randint(0, (1, 30, 100, 2)[turn], (users,), generator=g)
        indptr[1:] = counts.cumsum(0).cuda()
        indices.copy_(torch.randint(0, items, (room,), generator=g, dtype=torch.int32))
        weights.copy_(torch.randn(room, generator=g))
        want = [v.clone() for v in call()]
        for v in out:
            v.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_scores_without_entries(ctx, ops):
    w = wide_mxfp4(ops, 700, 700, 2, 117, 126)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    keep = torch.arange(700, device="cuda") % 3 > 0
    for weights in (None, torch.zeros(0, device="cuda")):
        got = ops.mxfp4_scores(ctx, torch.zeros(6, dtype=torch.int32, device="cuda"), none, w, weights=weights, exclude_history=True, item_keep=keep)
        assert bool((got[:, keep] == 0).all()) and bool(torch.isneginf(got[:, ~keep]).all())


def test_products_on_two_streams_at_once(ctx, ops):
    """Two products of different plans and the draws of long prefixes under way together: each has its own scratch memory."""
    w = wide_mxfp4(ops, 9000, 5000, 3, 117, 126)
    a = [torch.randn(m, 5000, generator=gen(m)).cuda() for m in (60, 300)]
    x, u = torch.randn(4, 60_000, generator=gen(9)).cuda(), torch.rand(4, 1, generator=gen(8)).cuda()
    calls = [lambda: ops.mxfp4_gemm_nt(ctx, a[0], w), lambda: ops.mxfp4_gemm_nt(ctx, a[1].half(), w), lambda: ops.sample(ctx, x, u, top_p=0.9)[0]]
    want = [c().clone() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for _ in range(5):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
    torch.cuda.synchronize()
    for i, v in enumerate(got):
        assert torch.equal(v, want[i % len(calls)])
