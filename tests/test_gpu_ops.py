"""4-bit (MXFP4) matrices, their products and sampling (recpack_amd.ops) against plain implementations in 64 bits."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


@pytest.fixture(scope="module")
def ctx():
    from recpack_amd import get_context

    return get_context(0)


@pytest.fixture(scope="module")
def ops():
    from recpack_amd import ops

    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- the format, by its definition -----------------------------------------------------------------------------------------------------

def quantised_reference(x):
    """(codes, scale bytes, values) of the rows of a float64 array."""
    rows, cols = x.shape
    nb = -(-cols // 32)
    v = np.zeros((rows, nb * 32))
    v[:, :cols] = x
    v = v.reshape(rows, nb, 32)
    top = np.abs(v).max(-1)
    bad = ~np.isfinite(v).all(-1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where((top > 0) & ~bad, np.frexp(np.where(bad, 1.0, top))[1] - 1 - 2, -127)
    e = np.clip(e, -127, 127)
    with np.errstate(invalid="ignore"):
        a = np.abs(v) / np.exp2(e)[..., None]
    a = np.where(bad[..., None], 0.0, a)
    at = np.zeros(a.shape, dtype=np.uint8)
    for i, border in enumerate((.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # half way: to the even mantissa
        at += (a >= border) if i % 2 else (a > border)
    code = np.where(bad[..., None], 0, at | (np.signbit(v) << 3)).astype(np.uint8)
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    values = np.where(bad[..., None], np.nan, np.copysign(GRID[at], v) * np.exp2(e)[..., None])
    code = code.reshape(rows, -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte, values.reshape(rows, -1)[:, :cols]


def values_of(m):
    codes, scales = m.codes.cpu().numpy(), m.scales.cpu().numpy().astype(np.float64)
    out = np.empty((codes.shape[0], codes.shape[1] * 2))
    for side, c in ((0, codes & 15), (1, codes >> 4)):
        out[:, side::2] = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    out *= np.repeat(np.where(scales == 255, np.nan, np.exp2(scales - 127)), 32, axis=1)
    return out[:, :m.cols]


def rows_with_edges(rows, cols, dtype, seed):
    x = torch.randn(rows, cols, generator=gen(seed)) * torch.exp2(torch.randint(-20, 12, (rows, cols), generator=gen(seed + 1)).float() * (torch.rand(rows, 1, generator=gen(seed + 2)) < 0.5))
    x = x.to(dtype)
    flat = x.view(-1)
    special = [0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 8.0, -2.5, torch.finfo(dtype).max, torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 4]
    for i, v in enumerate(special):
        if i * 7 < flat.numel():
            flat[i * 7] = v
    if rows > 2:
        x[1] = 0
    if rows > 4 and cols > 40:
        x[3, 5], x[3, 37], x[4, cols - 1] = math.nan, math.inf, -math.inf
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 33), (3, 31), (5, 64), (33, 77), (70, 300), (257, 65), (520, 129), (31, 2050)])
def test_quantise_and_read_back(ctx, ops, dtype, transpose, rows, cols):
    x = rows_with_edges(rows, cols, dtype, rows * 131 + cols)
    ref = x.double().numpy()
    codes, byte, values = quantised_reference(ref.T if transpose else ref)
    q = ops.mxfp4_quantize(ctx, x.cuda(), transpose=transpose)
    assert q.shape == ((cols, rows) if transpose else (rows, cols))
    np.testing.assert_array_equal(q.scales.cpu().numpy(), byte)
    np.testing.assert_array_equal(q.codes.cpu().numpy(), codes)
    with np.errstate(over="ignore"):
        expected = torch.from_numpy(values)
    for out_type in TYPES:
        got = ops.mxfp4_dequantize(ctx, q, dtype=out_type).cpu()
        # float32 holds every value exactly, so the one rounding is that of the float64 value
        torch.testing.assert_close(got, expected.float().to(out_type), rtol=0, atol=0, equal_nan=True)


def test_quantise_strides_and_given_outputs(ctx, ops):
    big = torch.randn(40, 211, generator=gen(3)).cuda()
    x = big[3:, 5:142]  # rows start at odd elements
    want = quantised_reference(x.double().cpu().numpy())
    buf = torch.full((50, 96), 7, dtype=torch.uint8, device="cuda")
    sc = torch.full((50, 9), 9, dtype=torch.uint8, device="cuda")
    out = ops.MXFP4(buf[:37, :80], sc[:37, :5], 137)
    assert ops.mxfp4_quantize(ctx, x, out=out) is out
    np.testing.assert_array_equal(out.codes.cpu().numpy(), want[0])
    np.testing.assert_array_equal(out.scales.cpu().numpy(), want[1])
    assert (buf[37:] == 7).all() and (buf[:, 80:] == 7).all() and (sc[37:] == 9).all() and (sc[:, 5:] == 9).all()
    # a transposed view takes the other kernel, an expanded one is copied
    for y in (big.t(), big[:1].expand(6, 211), big[:, ::2], big[:0], big[:, :0]):
        q = ops.mxfp4_quantize(ctx, y)
        np.testing.assert_array_equal(q.codes.cpu().numpy(), quantised_reference(y.double().cpu().numpy())[0] if y.numel() else q.codes.cpu().numpy())
        assert q.shape == tuple(y.shape)
    room = torch.full((37, 200), 5.0, device="cuda")
    ops.mxfp4_dequantize(ctx, out, out=room[:, 20:157])
    np.testing.assert_array_equal(room[:, 20:157].double().cpu().numpy(), want[2])
    assert (room[:, :20] == 5).all() and (room[:, 157:] == 5).all()


def test_foreign_scales_read_back(ctx, ops):
    """Every scale byte and code: the smallest are subnormal, the largest overflow to infinity."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, 256)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).repeat(1, 16)
    m = ops.MXFP4(codes.cuda(), scales.cuda(), 512)
    want = torch.from_numpy(values_of(m)).float()
    for t in TYPES:
        torch.testing.assert_close(ops.mxfp4_dequantize(ctx, m, dtype=t).cpu(), want.to(t), rtol=0, atol=0, equal_nan=True)


# ---- product ---------------------------------------------------------------------------------------------------------------------------

def random_mxfp4(ops, rows, cols, seed, pad_rows=0):
    nb = -(-cols // 32)
    codes = torch.randint(0, 256, (rows, nb * 16), generator=gen(seed), dtype=torch.uint8)
    if cols % 2:
        codes[:, cols // 2] &= 15
    codes[:, (cols + 1) // 2:] = 0
    scales = torch.randint(117, 126, (rows, nb), generator=gen(seed + 1), dtype=torch.uint8)
    return ops.MXFP4(codes.cuda(), scales.cuda(), cols)


def product_bound(a, w, terms, out, out_type):
    """Sums in float32: every one of the partial sums is off by at most one step (2^-23; a matrix instruction may truncate) of at most
    sum |a w|, and these errors are independent in sign: 8 sqrt(terms) of them are a bound in practice; then one rounding."""
    return 8 * math.sqrt(terms) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T) + torch.finfo(out_type).eps / 2 * np.abs(out) + torch.finfo(out_type).tiny


SIZES = [(1, 1, 1), (1, 17, 33), (2, 100, 1000), (4, 65, 129), (5, 64, 128), (16, 500, 257), (17, 33, 500), (64, 64, 64), (65, 130, 1030), (128, 257, 96), (257, 129, 300),
         (300, 1000, 2003), (1, 3000, 2048), (3, 2001, 4100)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_dense(ctx, ops, dtype, m, n, k):
    a = torch.randn(m, k, generator=gen(m * 7 + n)).to(dtype)
    w = random_mxfp4(ops, n, k, n * 3 + k)
    A, W = a.double().numpy(), values_of(w)
    want = A @ W.T
    for out_type in TYPES if (m, n, k) == (65, 130, 1030) else [dtype]:
        got = ops.mxfp4_gemm_nt(ctx, a.cuda(), w, dtype=out_type)
        assert got.dtype == out_type
        planes = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[dtype]
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= product_bound(A, W, planes * k, want, out_type)).all(), err.max()


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_4bit(ctx, ops, m, n, k):
    a = torch.randn(m, k, generator=gen(m * 7 + n))
    qa, w = ops.mxfp4_quantize(ctx, a.cuda()), random_mxfp4(ops, n, k, n * 3 + k)
    A, W = values_of(qa), values_of(w)
    for out_type in (torch.float32, torch.bfloat16):
        got = ops.mxfp4_gemm_nt(ctx, qa, w, dtype=out_type)
        want = A @ W.T
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= product_bound(A, W, k, want, out_type)).all(), err.max()


def test_product_f32_is_more_than_bf16(ctx, ops):
    """Every bit of a float32 operand counts: one significant element per row, the result is that element exactly."""
    a = torch.zeros(64, 96)
    a[torch.arange(64), torch.arange(64)] = torch.randn(64, generator=gen(5)) * 1e3
    top = torch.finfo(torch.float32).max
    a[7, 7], a[8, 8], a[9, 9], a[10, 10] = top, 1.2345679e-30, -top, 65504.0
    codes = torch.zeros(64, 48, dtype=torch.uint8)
    i = torch.arange(64)
    codes[i, i // 2] = torch.where(i % 2 == 0, 2, 32).to(torch.uint8)  # 1.0 on the diagonal
    w = ops.MXFP4(codes.cuda(), torch.full((64, 3), 127, dtype=torch.uint8, device="cuda"), 96)
    got = ops.mxfp4_gemm_nt(ctx, a.cuda(), w).cpu()
    torch.testing.assert_close(got.diagonal(), a.diagonal(), rtol=0, atol=0)
    half = a.clamp(-65504, 65504).half()
    torch.testing.assert_close(ops.mxfp4_gemm_nt(ctx, half.cuda(), w).cpu().diagonal(), half.diagonal(), rtol=0, atol=0)


def test_product_not_finite(ctx, ops):
    a = torch.randn(40, 100, generator=gen(1))
    a[3, 9], a[5, 50], a[6, 0] = math.inf, math.nan, -math.inf
    w = random_mxfp4(ops, 70, 100, 8)
    w.scales[11, 2] = 255
    A, W = a.double().numpy(), values_of(w)
    with np.errstate(invalid="ignore"):
        want = A @ W.T
    for dtype in TYPES:
        got = ops.mxfp4_gemm_nt(ctx, a.to(dtype).cuda(), w).double().cpu().numpy()
        for r in range(40):
            for v in (np.isnan, np.isposinf, np.isneginf):
                np.testing.assert_array_equal(v(got[r]), v(want[r]))
    qa = ops.mxfp4_quantize(ctx, a.cuda())
    got = ops.mxfp4_gemm_nt(ctx, qa, w).cpu()
    assert got[[3, 5, 6]].isnan().all() and got[:, 11].isnan().all()
    keep = [r for r in range(40) if r not in (3, 5, 6)]
    assert got[keep][:, [c for c in range(70) if c != 11]].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(40, 5000, 5000), (300, 9001, 700), (700, 6003, 1000)])
def test_product_scales_far_apart(ctx, ops, dtype, m, n, k):
    """Rows of W whose blocks differ by 2^35 .. 2^200, rows of A that meet only the small ones; zero blocks and NaN blocks among them."""
    g = gen(m)
    w = random_mxfp4(ops, n, k, 2)
    w.scales.fill_(130)
    for row, block, scale in ((3, 2, 130 - 35), (7, 3, 130 - 36), (9, 3, 130 - 37), (20, 1, 60), (1000, 5, 254 - 2), (1001, 5, 0), (n - 1, 3, 90), (n - 2, 7, 0)):
        w.scales[row, block] = scale
    w.codes[1001, 5 * 16:6 * 16] = 0  # (a block of zeros)
    w.scales[2000, 4] = 255
    a = torch.randn(m, k, generator=g)
    for r in range(8):  # row r of A: nothing but block r
        a[r] = 0
        a[r, r * 32:r * 32 + 32] = torch.randn(32, generator=g)
    a = a.to(dtype).cuda()
    W = values_gpu(ops, ctx, w)
    A = a.double()
    got = ops.mxfp4_gemm_nt(ctx, a, w, dtype=torch.float32).double()
    W[2000, 128:160] = math.nan
    want, size = A @ W.t(), A.abs() @ W.abs().t()
    # (a block of 6 x 2^125 times a standard normal number passes float32's largest, 2^128: such sums are no numbers in any order)
    fits = ~(size >= 2.0 ** 127)
    assert torch.equal(got.isnan() & fits, want.isnan()) and bool(got[:, 2000].isnan().all()) and int((~fits).sum()) <= m
    terms = k * {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[dtype]
    bound = 8 * math.sqrt(terms) * 2.0 ** -23 * size + torch.finfo(torch.float32).tiny
    assert bool((((got - want).abs() <= bound) | want.isnan() | ~fits).all())


def test_product_not_finite_large(ctx, ops):
    a = torch.randn(40, 5000, generator=gen(1))
    a[3, 9], a[5, 50], a[6, 0] = math.inf, math.nan, -math.inf
    w = random_mxfp4(ops, 5000, 5000, 8)
    w.scales[11, 2] = 255
    for dtype in TYPES:
        x = a.to(dtype).cuda()
        got, want = ops.mxfp4_gemm_nt(ctx, x, w), x.double() @ values_gpu(ops, ctx, w).t()
        want[:, 11] = math.nan
        for v in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(v(got), v(want))


def test_product_strides(ctx, ops):
    big = torch.randn(90, 301, generator=gen(2)).cuda()
    a = big[1:78, 3:204]
    w = random_mxfp4(ops, 45, 201, 4)
    room = torch.full((77, 100), 3.0, device="cuda")
    ops.mxfp4_gemm_nt(ctx, a, w, out=room[:, 11:56])
    A, W = a.double().cpu().numpy(), values_of(w)
    want = A @ W.T
    assert (np.abs(room[:, 11:56].double().cpu().numpy() - want) <= product_bound(A, W, 3 * 201, want, torch.float32)).all()
    assert (room[:, :11] == 3).all() and (room[:, 56:] == 3).all()
    for shape in ((0, 201), (5, 201)):
        got = ops.mxfp4_gemm_nt(ctx, torch.zeros(shape, device="cuda"), w)
        assert got.shape == (shape[0], 45) and (got == 0).all()
    none = ops.mxfp4_gemm_nt(ctx, torch.zeros(4, 0, device="cuda"), ops.mxfp4_quantize(ctx, torch.zeros(6, 0, device="cuda")))
    assert none.shape == (4, 6) and (none == 0).all()  # an empty sum


# ---- scores of histories -----------------------------------------------------------------------------------------------------------------

def histories(users, items, mean, seed):
    g = gen(seed)
    n = torch.randint(0, 2 * mean + 1, (users,), generator=g)
    n[0] = 0
    if users > 2:
        n[2] = min(4 * mean + 70, 3 * items)
    indptr = torch.zeros(users + 1, dtype=torch.int32)
    indptr[1:] = n.cumsum(0)
    indices = torch.randint(0, items, (int(indptr[-1]),), generator=g, dtype=torch.int32)  # repeats among them
    return indptr, indices


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("users,items,mean", [(1, 1, 1), (3, 31, 3), (5, 33, 20), (7, 500, 40), (20, 2049, 60), (4, 6000, 100)])
def test_scores(ctx, ops, dtype, weighted, users, items, mean):
    indptr, indices = histories(users, items, mean, users + items)
    w = random_mxfp4(ops, items, items, items)
    weights = torch.randn(indices.numel(), generator=gen(9)) if weighted else None
    keep = torch.rand(items, generator=gen(10)) < 0.8
    W = values_of(w)
    X = np.zeros((users, items))
    absX = np.zeros((users, items))
    rows = np.repeat(np.arange(users), np.diff(indptr.numpy()))
    f = np.ones(len(indices)) if weights is None else weights.double().numpy()
    np.add.at(X, (rows, indices.numpy()), f)
    np.add.at(absX, (rows, indices.numpy()), np.abs(f))
    want = X @ W
    # n adds (and products) in float32, each off by at most half a step of at most the sum of the magnitudes, then one rounding
    n = np.diff(indptr.numpy())[:, None] + 1
    bound = 2 * n * 2.0 ** -24 * (absX @ np.abs(W)) + torch.finfo(dtype).eps / 2 * np.abs(want) + torch.finfo(dtype).tiny
    args = (ctx, indptr.cuda(), indices.cuda(), w, None if weights is None else weights.cuda())
    got = ops.mxfp4_scores(*args, dtype=dtype)
    assert got.dtype == dtype and got.shape == (users, items)
    assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()
    masked = ops.mxfp4_scores(*args, exclude_history=True, item_keep=keep.cuda(), dtype=dtype).cpu()
    gone = torch.zeros(users, items, dtype=torch.bool)
    gone[torch.from_numpy(rows), indices.long()] = True
    gone |= ~keep
    assert (masked[gone] == -math.inf).all()
    torch.testing.assert_close(masked[~gone], got.cpu()[~gone], rtol=0, atol=0)


def test_scores_bad_entries_and_rectangles(ctx, ops):
    """Entries outside the matrix count nothing, a row pointer beyond the entries reads none of them."""
    w = random_mxfp4(ops, 50, 333, 1)
    W = values_of(w)
    indptr = torch.tensor([0, 4, 4, 7, 900, 2, -5, 3], dtype=torch.int32)
    indices = torch.tensor([3, 50, -1, 7, 2147483647, 9, -2147483648, 11], dtype=torch.int32)
    room = torch.full((7, 400), 5.0, device="cuda")
    got = ops.mxfp4_scores(ctx, indptr.cuda(), indices.cuda(), w, out=room[:, 9:342]).double().cpu().numpy()
    rows = [[3, 7], [], [9], [11], [], [], [3]]
    for u, r in enumerate(rows):
        np.testing.assert_allclose(got[u], W[r].sum(0) if r else np.zeros(333), rtol=0, atol=4 * 2.0 ** -24 * np.abs(W).max() * 4)
    assert (room[:, :9] == 5).all() and (room[:, 342:] == 5).all()
    assert ops.mxfp4_scores(ctx, indptr[:1].cuda(), indices[:0].cuda(), w).shape == (0, 333)
    none = ops.MXFP4(torch.zeros(0, 176, dtype=torch.uint8, device="cuda"), torch.zeros(0, 11, dtype=torch.uint8, device="cuda"), 333)
    assert (ops.mxfp4_scores(ctx, indptr[:3].cuda(), indices.cuda(), none) == 0).all()


# ---- sampling ----------------------------------------------------------------------------------------------------------------------------

def sample_reference(scores, u, temperature, top_k, top_p, min_p, lengths=None, ids=None):
    """The definition, row by row, in float64 (settings: one per row)."""
    rows, width = scores.shape
    items, probs = np.full(u.shape, -1, np.int64), np.zeros(u.shape)
    for r in range(rows):
        x = scores[r] if lengths is None else scores[r, :max(0, min(int(lengths[r]), width))]
        there = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
        there = there[np.argsort(-x[there], kind="stable")][:int(top_k[r]) or None]
        if not there.size:
            continue
        t = float(temperature[r])
        val = x[there]

        def masses(v):
            with np.errstate(invalid="ignore", over="ignore"):
                return np.exp(np.where(v == v[0], 0.0, (v - v[0]) / t))

        if t > 0:
            p = masses(val)
            n = len(p)
            if top_p[r] < 1:
                n = 1 + int(np.searchsorted(np.cumsum(p), float(top_p[r]) * p.sum()))
            n = min(n, len(p), int((p >= float(min_p[r])).sum()))
            there, val = there[:n], val[:n]
        for d in range(min(u.shape[1], len(there))):
            k = 0
            if t > 0:
                p = masses(val)
                c = np.cumsum(p)
                uu = min(max(float(np.nan_to_num(u[r, d], nan=0.0)), 0.0), 1 - 2.0 ** -24)
                k = min(int(np.searchsorted(c, uu * c[-1], side="right")), len(p) - 1)
                probs[r, d] = p[k] / c[-1]
            else:
                probs[r, d] = 1.0
            items[r, d] = there[k] if ids is None else ids[r, there[k]]
            there, val = np.delete(there, k), np.delete(val, k)
    return items, probs, (items >= 0).sum(1)


def check_sample(ctx, ops, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lengths=None, ids=None, top_k_per_row=None):
    rows = x.shape[0]
    cuda = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v  # noqa: E731
    got = ops.sample(ctx, cuda(x), cuda(u), cuda(temperature), top_k, cuda(top_p), cuda(min_p), lengths=cuda(lengths), ids=cuda(ids), top_k_per_row=cuda(top_k_per_row))
    per_row = lambda v: v.double().numpy() if isinstance(v, torch.Tensor) else np.full(rows, np.float64(np.float32(v)))  # noqa: E731
    k = np.full(rows, top_k) if top_k_per_row is None else np.where(top_k_per_row.numpy() > 0, np.minimum(top_k_per_row.numpy(), top_k), top_k)
    want = sample_reference(x.double().cpu().numpy(), u.double().cpu().numpy(), per_row(temperature), k, per_row(top_p), per_row(min_p),
                            None if lengths is None else lengths.cpu().numpy(), None if ids is None else ids.cpu().numpy())
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[2].cpu().numpy(), want[2])
    # float64 sums of at most 2^20 masses, one rounding to float32
    np.testing.assert_allclose(got[1].double().cpu().numpy(), want[1], rtol=2.0 ** -24 + 1e-9, atol=2.0 ** -149)
    return got


WIDTHS = [1, 2, 63, 200, 256, 257, 1000, 1024, 1025, 2500, 20011]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_sample_one(ctx, ops, dtype, width):
    rows = 37
    g = gen(width)
    x = (torch.randn(rows, width, generator=g) * 2).to(dtype)
    x[torch.rand(rows, width, generator=g) < 0.1] = -math.inf
    x[4] = -math.inf
    if width > 1:
        x[5, 1:] = -math.inf
        x[6, 0] = math.nan
    u = torch.rand(rows, 1, generator=g)
    t, p, m = torch.rand(rows, generator=g) * 2 + 0.05, torch.rand(rows, generator=g), torch.rand(rows, generator=g) * 0.1
    check_sample(ctx, ops, x, u)
    check_sample(ctx, ops, x, u, temperature=t, top_p=p)
    check_sample(ctx, ops, x, u, temperature=t, min_p=m)
    check_sample(ctx, ops, x, u, temperature=0.7, top_p=0.9, min_p=0.01)
    check_sample(ctx, ops, x, u, temperature=t, top_p=p, top_k=50)
    check_sample(ctx, ops, x, u, temperature=t, top_p=p, top_k=2000)
    check_sample(ctx, ops, x, u, temperature=0.0, top_p=0.5)
    check_sample(ctx, ops, x, u, temperature=0.0, top_k=3)
    lengths = torch.randint(-2, width + 3, (rows,), generator=g, dtype=torch.int32)
    ids = torch.randint(0, 2 ** 31 - 1, (rows, width), generator=g, dtype=torch.int32)
    check_sample(ctx, ops, x, u, temperature=t, top_p=0.8, lengths=lengths, ids=ids)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,top_k,draws", [(1, 0, 3), (5, 0, 5), (5, 3, 8), (200, 0, 20), (256, 0, 256), (257, 100, 40), (1000, 0, 30), (1024, 0, 200), (3000, 50, 20), (3000, 256, 60),
                                               (3000, 257, 20), (20011, 200, 20), (20011, 1000, 10), (5000, 1024, 1024)])
def test_sample_slates(ctx, ops, dtype, width, top_k, draws):
    rows = 9
    g = gen(width + draws)
    x = (torch.randn(rows, width, generator=g) * 2).to(dtype)
    x[torch.rand(rows, width, generator=g) < 0.1] = -math.inf
    u = torch.rand(rows, draws, generator=g)
    t, p = torch.rand(rows, generator=g) + 0.3, torch.rand(rows, generator=g) * 0.5 + 0.5
    check_sample(ctx, ops, x, u, temperature=t, top_k=top_k)
    check_sample(ctx, ops, x, u, temperature=t, top_k=top_k, top_p=p, min_p=0.001)
    check_sample(ctx, ops, x, u, temperature=0.001, top_k=top_k)  # everything but the best underflows: relative to the best one left
    check_sample(ctx, ops, x, u, temperature=0.0, top_k=top_k)
    if top_k:
        check_sample(ctx, ops, x, u, temperature=t, top_k=top_k, top_k_per_row=torch.randint(-1, top_k + 5, (rows,), generator=g, dtype=torch.int32))


@pytest.mark.parametrize("width", [300, 1100, 9000, 50001])
def test_sample_ties_and_extremes(ctx, ops, width):
    """Rows of equal scores, of two scores, of the type's lowest value, of infinities; uniforms at the ends and on borders."""
    low = torch.finfo(torch.float32).min
    g = gen(width)
    x = torch.stack([torch.zeros(width), torch.full((width,), low), torch.full((width,), -7.25), (torch.arange(width) % 2).float(),
                     torch.where(torch.arange(width) % 3 == 0, low, 0.5), torch.where(torch.arange(width) % 5 == 0, math.inf, 1.0),
                     torch.where(torch.arange(width) % 2 == 0, -0.0, 0.0), torch.randint(0, 3, (width,), generator=g).float(),
                     torch.linspace(-5, 5, width), torch.linspace(5, -5, width), torch.where(torch.arange(width) == width // 2, 1e30, torch.randn(width, generator=g)),
                     torch.full((width,), math.nan)])
    rows = x.shape[0]
    for uu in (0.0, 0.5, 0.25, 1 - 2.0 ** -24, 1.0, -1.0, math.nan, 0.3):
        u = torch.full((rows, 1), uu)
        check_sample(ctx, ops, x, u)
        check_sample(ctx, ops, x, u, top_p=0.5)
        check_sample(ctx, ops, x, u, top_k=1000, temperature=2.0)
        check_sample(ctx, ops, x, u, top_k=1056, top_p=0.75)
        check_sample(ctx, ops, x, u, min_p=1.0)
        check_sample(ctx, ops, x, u, top_p=0.0)
    check_sample(ctx, ops, x, torch.rand(rows, 10, generator=g), top_k=40)
    check_sample(ctx, ops, x.bfloat16(), torch.rand(rows, 10, generator=g), top_k=1000, top_p=0.5)
    check_sample(ctx, ops, x, torch.rand(rows, 1, generator=g), temperature=1e-30)
    check_sample(ctx, ops, x, torch.rand(rows, 1, generator=g), temperature=1e30)
    check_sample(ctx, ops, x, torch.rand(rows, 1, generator=g), temperature=0.0)


@pytest.mark.parametrize("width,top_k", [(2, 0), (5, 0), (64, 0), (65, 0), (200, 0), (256, 0), (257, 0), (500, 0), (513, 0), (1024, 0), (3000, 120), (3000, 400), (3000, 1000), (40000, 1000)])
@pytest.mark.parametrize("apart", [1, 2, 64, 10 ** 6])
def test_sample_close_scores(ctx, ops, width, top_k, apart):
    """Scores that share their leading bits: some neighbours, some groups, all of them; equal ones among them."""
    g = gen(width + apart)
    step = torch.arange(width) // max(1, min(apart, width)) * 100.0  # groups of `apart` scores within some ulps of each other
    x = (1000.0 + step).float()
    x = (x.view(torch.int32) + torch.randint(0, 256, (6, width), generator=g, dtype=torch.int32)).view(torch.float32)
    x = torch.stack([row[torch.randperm(width, generator=g)] for row in x])
    x[1::2] *= -1
    n = min(top_k or width, 64)
    check_sample(ctx, ops, x, torch.zeros(6, n), temperature=0.0, top_k=top_k)
    check_sample(ctx, ops, x, torch.rand(6, n, generator=g), temperature=0.05, top_k=top_k, top_p=0.9)


@pytest.mark.parametrize("rows,width", [(1, 30001), (3, 40000), (12, 30001), (63, 20001), (64, 30001), (70, 1500), (2, 20000), (300, 2050)])
@pytest.mark.parametrize("top_k", [0, 1025, 5000])
def test_sample_whole_rows(ctx, ops, rows, width, top_k):
    """One draw from a long prefix: few wide rows over many workgroups, otherwise a workgroup to a row; rows without candidates among them."""
    g = gen(rows + width + top_k)
    x = torch.randn(rows, width, generator=g) * 2
    x[torch.rand(rows, width, generator=g) < 0.1] = -math.inf
    if rows > 2:
        x[1] = math.nan
        x[2, 7:] = -math.inf
    u = torch.rand(rows, 1, generator=g)
    k = min(top_k, width)
    check_sample(ctx, ops, x, u, temperature=0.8, top_k=k, top_p=0.9, min_p=0.001)
    check_sample(ctx, ops, x, u, temperature=torch.rand(rows, generator=g) + 0.3, top_k=k)
    check_sample(ctx, ops, x.half(), u, temperature=0.0, top_k=k)
    check_sample(ctx, ops, torch.round(x), u, temperature=1.0, top_k=k, top_p=0.5)  # thousands of equal scores


def test_sample_far_below(ctx, ops):
    """Candidates far below the best one: by value in one coarse bin, drawn after the rest is gone."""
    x = torch.cat([torch.tensor([[50.0, 49.0]]), torch.randn(1, 30000, generator=gen(0)) - 400], 1)
    check_sample(ctx, ops, x.repeat(5, 1), torch.rand(5, 12, generator=gen(1)), top_k=500)
    check_sample(ctx, ops, x.repeat(5, 1), torch.rand(5, 1, generator=gen(1)), top_k=20000, top_p=0.999)
    check_sample(ctx, ops, x, torch.tensor([[0.999]]), temperature=300.0)


def test_sample_many_rows_is_the_distribution(ctx, ops):
    """Frequencies follow the masses: 200 000 draws, each of 40 items within 6 standard deviations."""
    n, width = 200_000, 40
    x = torch.randn(1, width, generator=gen(4))
    u = torch.rand(n, 1, generator=gen(5))
    got = ops.sample(ctx, x.cuda().expand(n, width), u.cuda())[0].cpu().view(-1)
    p = torch.softmax(x.double().view(-1), 0)
    seen = torch.bincount(got.long(), minlength=width).double()
    assert (torch.abs(seen - n * p) <= 6 * torch.sqrt(n * p * (1 - p))).all()


def test_sample_strides_and_empty(ctx, ops):
    big = torch.randn(20, 3000, generator=gen(6))
    u = torch.rand(20, 9, generator=gen(7))
    check_sample(ctx, ops, big[2:11, 7:2100], u[2:11, 3:5], top_k=30)
    check_sample(ctx, ops, big.t()[:50, :20], u[:1, :3].expand(50, 3), top_k=10)
    for width in (0, 5):
        idx, prob, nnz = ops.sample(ctx, torch.zeros(0, width, device="cuda"), torch.zeros(0, 2, device="cuda"))
        assert idx.shape == (0, 2) and nnz.shape == (0,)
    idx, prob, nnz = ops.sample(ctx, torch.zeros(3, 0, device="cuda"), torch.zeros(3, 2, device="cuda"))
    assert (idx == -1).all() and (prob == 0).all() and (nnz == 0).all()


# ---- products in every tile shape: large enough for the plans that fill the card ------------------------------------------------------------

def values_gpu(ops, ctx, m):
    """float64 values on the GPU, by the format (the codes' table and 2^(s - 127))."""
    lut = torch.from_numpy(np.concatenate([GRID, -GRID])).cuda()
    c = torch.stack((m.codes & 15, m.codes >> 4), -1).view(m.shape[0], -1).long()
    return (lut[c] * torch.exp2(m.scales.double() - 127).repeat_interleave(32, 1))[:, :m.cols]


@pytest.mark.parametrize("dtype,m,n,k", [
    (torch.bfloat16, 1100, 8010, 200), (torch.float16, 1100, 8010, 330), (torch.float32, 1100, 8010, 130),  # 128 x 256 tiles
    (torch.bfloat16, 2050, 8200, 257), (torch.float16, 2050, 8200, 90),                                     # 256 x 256
    (torch.bfloat16, 130, 20001, 8100), (torch.float32, 200, 9001, 4000),                                   # 128 x 128, K in parts
    (torch.bfloat16, 33, 3001, 6000), (torch.float16, 64, 999, 9000), (torch.float32, 9, 2000, 5001), (torch.float32, 4, 5003, 7001),
    ("mxfp4", 4000, 4200, 300), ("mxfp4", 600, 3001, 1000), ("mxfp4", 200, 1999, 5000), ("mxfp4", 20, 700, 9000),
    ("mxfp4", 20, 40001, 3000), ("mxfp4", 300, 8001, 2000), ("mxfp4", 1000, 8000, 3000), ("mxfp4", 500, 3001, 5000), ("mxfp4", 90, 1501, 17000),
    (torch.bfloat16, 1500, 12001, 4200), (torch.float16, 2001, 12000, 4200), (torch.float32, 1500, 12001, 4200), ("mxfp4", 1500, 12003, 8300),  # the last round in parts
    (torch.bfloat16, 300, 30002, 4200), (torch.float16, 300, 30001, 4300), (torch.float32, 300, 30001, 4200), ("mxfp4", 700, 30001, 8300),
    (torch.bfloat16, 16, 2001, 4200), (torch.float16, 300, 5003, 1000), (torch.float32, 40, 4001, 4096), (torch.bfloat16, 500, 1001, 3999)])
def test_product_large(ctx, ops, dtype, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a = torch.randn(m, k, device="cuda", generator=g)
    w = random_mxfp4(ops, n, k, 3)
    if dtype == "mxfp4":
        a = ops.mxfp4_quantize(ctx, a)
        A, terms, out_type = values_gpu(ops, ctx, a), k, torch.float32
    else:
        a = a.to(dtype)
        A, terms, out_type = a.double(), k * {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}[dtype], dtype
    W = values_gpu(ops, ctx, w)
    got = ops.mxfp4_gemm_nt(ctx, a, w)
    want = A @ W.t()
    bound = 8 * math.sqrt(terms) * 2.0 ** -23 * (A.abs() @ W.abs().t()) + torch.finfo(out_type).eps / 2 * want.abs() + torch.finfo(out_type).tiny
    assert got.dtype == out_type
    assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(got, ops.mxfp4_gemm_nt(ctx, a, w))  # no part of K is added in another order


# ---- what is left alone, what is huge ---------------------------------------------------------------------------------------------------------

def framed(rows, cols, dtype, value=7):
    """An output inside a larger buffer, and a check that the frame around it is as it was."""
    big = torch.full((rows + 2, cols + 5), value, dtype=dtype, device="cuda")
    out = big[1:-1, 3:-2]

    def untouched():
        frame = torch.ones_like(big, dtype=torch.bool)
        frame[1:-1, 3:-2] = False
        return bool((big[frame] == value).all())

    return out, untouched


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_around_an_output_is_written(ctx, ops, dtype):
    g = gen(4)
    w = random_mxfp4(ops, 333, 333, 5)
    for rows in (1, 3, 17, 70):
        out, untouched = framed(rows, 333, dtype)
        assert torch.equal(ops.mxfp4_gemm_nt(ctx, torch.randn(rows, 333, generator=g).cuda(), w, out=out).contiguous(), out) and untouched()
        indptr = torch.arange(rows + 1, dtype=torch.int32).cuda() * 3
        indices = torch.randint(0, 333, (rows * 3,), generator=g, dtype=torch.int32).cuda()
        for weights in (None, torch.rand(rows * 3, generator=g).cuda()):
            out, untouched = framed(rows, 333, dtype)
            ops.mxfp4_scores(ctx, indptr, indices, w, weights=weights, out=out)
            assert untouched() and not (out == 7).all()
    out, untouched = framed(333, 333, dtype)
    ops.mxfp4_dequantize(ctx, w, out=out)
    assert untouched()
    # the codes of a matrix inside a larger one
    codes, scales = torch.full((12, 32 * 16), 9, dtype=torch.uint8, device="cuda"), torch.full((12, 32), 9, dtype=torch.uint8, device="cuda")
    m = ops.MXFP4(codes[1:-1, 16:16 * 5], scales[1:-1, 2:6], 100)
    x = torch.randn(10, 100, generator=g).to(dtype).cuda()
    for transpose in (False, True):
        codes.fill_(9), scales.fill_(9)
        ops.mxfp4_quantize(ctx, x.t().contiguous() if transpose else x, transpose=transpose, out=m)
        np.testing.assert_array_equal(values_of(m), quantised_reference(x.double().cpu().numpy())[2])
        assert int((codes == 9).sum()) >= 12 * 32 * 16 - 10 * 64 and bool((codes[:, :16] == 9).all()) and bool((codes[:, 80:] == 9).all())
        assert bool((codes[0] == 9).all()) and bool((codes[-1] == 9).all()) and bool((scales[:, 6:] == 9).all()) and bool((scales[0] == 9).all())


@pytest.mark.parametrize("m,n,k", [(0, 5, 7), (5, 0, 7), (5, 7, 0), (1, 7, 0), (40, 70, 0)])
def test_empty_products(ctx, ops, m, n, k):
    w = ops.mxfp4_quantize(ctx, torch.ones(n, k, device="cuda"))
    for a in (torch.ones(m, k, device="cuda"), ops.mxfp4_quantize(ctx, torch.ones(m, k, device="cuda"))):
        got = ops.mxfp4_gemm_nt(ctx, a, w, out=torch.full((m, n), 3.0, device="cuda"))
        assert got.shape == (m, n) and bool((got == 0).all())


@pytest.mark.parametrize("m", [1, 4, 40])
def test_product_of_the_largest_scale(ctx, ops, m):
    """6 x 2^127 in a row's last block is no number of float32 (quantising makes no scale that large): the row's sums are not finite, the others'
    are not touched.  Infinite in one pass over float32; with A in bf16 planes 1 = 1 + 0 + 0, and 0 times infinity is NaN."""
    w = ops.mxfp4_quantize(ctx, torch.ones(6, 70, device="cuda"))
    w.scales[2, 2], w.codes[2, 32] = 254, 0x07
    got = ops.mxfp4_gemm_nt(ctx, torch.ones(m, 70, device="cuda"), w)
    assert not bool(got[:, 2].isfinite().any()) and bool((got[:, [0, 1, 3, 4, 5]] == 70).all())
    assert m > 4 or bool(got[:, 2].isinf().all())


def test_offsets_past_32_bits(ctx, ops):
    """Inputs and outputs of more than 2^32 bytes (2^31 elements): the last rows are those of the last rows alone."""
    rows, cols = 70001, 33001
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    last = x[-5:].clone()
    q, ql = ops.mxfp4_quantize(ctx, x), ops.mxfp4_quantize(ctx, last)
    assert torch.equal(q.codes[-5:], ql.codes) and torch.equal(q.scales[-5:], ql.scales)
    t = ops.mxfp4_quantize(ctx, x, transpose=True)
    part = ops.mxfp4_quantize(ctx, x[69984:].contiguous(), transpose=True)  # (a multiple of 32 rows in front)
    assert torch.equal(t.codes[:, 69984 // 2:], part.codes) and torch.equal(t.scales[:, 69984 // 32:], part.scales)
    back = ops.mxfp4_dequantize(ctx, q, dtype=torch.float16)
    assert torch.equal(back[-5:], ops.mxfp4_dequantize(ctx, ql, dtype=torch.float16))
    del t, part, back
    u = torch.rand(rows, 4, device="cuda")
    for k in (20, 0):
        n = 4 if k else 1
        got, want = ops.sample(ctx, x, u[:, :n], top_k=k), ops.sample(ctx, last, u[-5:, :n], top_k=k)
        assert all(torch.equal(a[-5:], b) for a, b in zip(got, want))
    indptr = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    indices = torch.arange(rows, dtype=torch.int32, device="cuda")
    out = ops.mxfp4_scores(ctx, indptr, indices, q, dtype=torch.float16)  # (every history is one row of the matrix)
    assert torch.equal(out[-5:], ops.mxfp4_dequantize(ctx, ql, dtype=torch.float16))
    del out
    w = ops.mxfp4_quantize(ctx, torch.randn(40000, 96, device="cuda"))
    a = torch.randn(60001, 96, device="cuda", dtype=torch.float16)
    got = ops.mxfp4_gemm_nt(ctx, a, w)
    assert got.numel() > 2 ** 31 and torch.equal(got[-3:], ops.mxfp4_gemm_nt(ctx, a[-300:], w)[-3:])


def test_codes_past_4_gib(ctx, ops):
    n = 100000
    w = ops.MXFP4.empty(n, n, "cuda")
    w.codes.random_(generator=torch.Generator(device="cuda").manual_seed(2))
    w.scales.random_(120, 130, generator=torch.Generator(device="cuda").manual_seed(3))
    at = torch.tensor([n - 1, 5, n - 2, 99998 - 1], dtype=torch.int32, device="cuda")
    few = ops.MXFP4(w.codes[at.long()].contiguous(), w.scales[at.long()].contiguous(), n)
    rows = ops.mxfp4_dequantize(ctx, few).double()
    got = ops.mxfp4_scores(ctx, torch.tensor([0, 4, 5], dtype=torch.int32, device="cuda"), torch.cat([at, at[:1]]), w)
    assert torch.equal(got[1].double(), rows[0])
    assert bool(((got[0].double() - rows.sum(0)).abs() <= 4 * 2.0 ** -23 * rows.abs().sum(0)).all())
    a = torch.randn(2, n, device="cuda")
    want = a.double() @ rows.t()
    got = ops.mxfp4_gemm_nt(ctx, a, w)[:, at.long()].double()
    assert bool(((got - want).abs() <= 8 * math.sqrt(n) * 2.0 ** -23 * (a.double().abs() @ rows.abs().t())).all())
