"""Refusals of the 4-bit and sampling operators: every argument is checked before the device is touched (no GPU is needed)."""
import ctypes as C

import pytest
import torch

from recpack_amd import _lib, ops

P = 0x10000  # an address that is never read: the calls below are refused before


def refused(name, args, message, code=_lib.RPHIP_EINVAL):
    lib = _lib.load_library()
    assert getattr(lib, name)(*args) == code
    text = lib.rphip_last_error().decode()
    assert message in text, text


def quantize(rows=4, cols=64, x=P, x_type=0, ldx=64, transpose=0, codes=P, ldc=32, scales=P, lds=2):
    return [None, None, rows, cols, x, x_type, ldx, transpose, codes, ldc, scales, lds]


@pytest.mark.parametrize("change,message", [
    (dict(x_type=3), "element type"), (dict(x_type=-1), "element type"), (dict(rows=-1), "no matrix size"), (dict(cols=2 ** 31), "no matrix size"),
    (dict(codes=None), "NULL codes"), (dict(scales=None), "NULL codes"), (dict(codes=P + 8), "multiples of 16"), (dict(ldc=40), "multiples of 16"),
    (dict(ldc=16), "too small"), (dict(lds=1), "too small"), (dict(x=None), "x is NULL"), (dict(x=P + 2), "not aligned"), (dict(ldx=63), "ldx"), (dict(), "ctx is NULL")])
def test_quantize_refuses(change, message):
    refused("rphip_mxfp4_quantize", quantize(**change), message)


def test_quantize_transpose_limit():
    refused("rphip_mxfp4_quantize", quantize(rows=32, cols=2 ** 28 + 1, ldx=2 ** 28 + 1, transpose=1, ldc=16, lds=1), "2^28", _lib.RPHIP_ELIMIT)


def dequantize(rows=4, cols=64, codes=P, ldc=32, scales=P, lds=2, out=P, out_type=0, ldo=64):
    return [None, None, rows, cols, codes, ldc, scales, lds, out, out_type, ldo]


@pytest.mark.parametrize("change,message", [(dict(out_type=7), "element type"), (dict(codes=None), "NULL codes"), (dict(ldc=16), "too small"), (dict(out=None), "out is NULL"),
                                            (dict(out=P + 1), "not aligned"), (dict(ldo=60), "ld_out"), (dict(), "ctx is NULL")])
def test_dequantize_refuses(change, message):
    refused("rphip_mxfp4_dequantize", dequantize(**change), message)


def gemm(m=4, n=8, k=64, a=P, a_type=0, lda=64, asc=None, ldas=0, w=P, ldw=32, ws=P, ldws=2, c=P, c_type=0, ldc=8, work=P, size=1 << 30):
    return [None, None, m, n, k, a, a_type, lda, asc, ldas, w, ldw, ws, ldws, c, c_type, ldc, work, size]


@pytest.mark.parametrize("change,message", [
    (dict(m=-1), "mxfp4_gemm_nt"), (dict(a_type=4), "of A"), (dict(c_type=3), "of C"), (dict(w=None), "NULL codes"), (dict(ldw=16), "too small"),
    (dict(a_type=3, lda=32), "NULL codes"), (dict(a_type=3, lda=16, asc=P, ldas=2), "too small"), (dict(c=None), "NULL argument"), (dict(a=None), "NULL argument"),
    (dict(lda=63), "lda < K"), (dict(a=P + 2), "lda < K"), (dict(ldc=7), "ldc < N"), (dict(), "ctx is NULL")])
def test_gemm_refuses(change, message):
    refused("rphip_mxfp4_gemm_nt", gemm(**change), message)


def test_gemm_limits():
    refused("rphip_mxfp4_gemm_nt", gemm(m=65535 * 16 + 1), "rows of A", _lib.RPHIP_ELIMIT)
    refused("rphip_mxfp4_gemm_nt", gemm(n=2 ** 28 + 1, ldc=2 ** 28 + 1), "rows of W", _lib.RPHIP_ELIMIT)
    refused("rphip_mxfp4_gemm_nt_workspace", [None, 1, 1, 1, 0, C.byref(C.c_int64())], "NULL argument")


def scores(users=3, nnz=5, indptr=P, indices=P, weights=None, rows=64, cols=64, codes=P, ldc=32, scales=P, lds=2, exclude=0, keep=None, out=P, out_type=0, ldo=64):
    return [None, None, users, nnz, indptr, indices, weights, rows, cols, codes, ldc, scales, lds, exclude, keep, out, out_type, ldo]


@pytest.mark.parametrize("change,message", [
    (dict(out_type=3), "element type"), (dict(users=-1), "users"), (dict(nnz=2 ** 31), "entries"), (dict(codes=P + 4), "multiples of 16"), (dict(lds=1), "too small"),
    (dict(exclude=1, rows=63), "square"), (dict(indptr=None), "NULL argument"), (dict(indices=None), "NULL argument"), (dict(out=None), "NULL argument"), (dict(out=P + 2), "not aligned"),
    (dict(ldo=63), "ld_out"), (dict(), "ctx is NULL")])
def test_scores_refuses(change, message):
    refused("rphip_mxfp4_scores", scores(**change), message)


def sample(rows=2, width=10, scores=P, type=0, ld=10, lengths=None, ids=None, ld_ids=0, draws=1, u=P, ldu=1, params=True, idx=P, prob=P, nnz=P, **setting):
    p = _lib.SampleParams(setting.get("temperature", 1.0), setting.get("top_p", 1.0), setting.get("min_p", 0.0), setting.get("top_k", 0), None, None, None, setting.get("top_k_dev"))
    return [None, None, rows, width, scores, type, ld, lengths, ids, ld_ids, draws, u, ldu, C.byref(p) if params else None, idx, prob, nnz, None, 0]


@pytest.mark.parametrize("change,message", [
    (dict(params=False), "params"), (dict(type=3), "element type"), (dict(rows=-1), "rows of"), (dict(width=2 ** 30 + 1, ld=2 ** 31), "rows of"), (dict(draws=0), "draws"), (dict(draws=2 ** 30 + 1, ldu=2 ** 31), "draws"),
    (dict(ld=9), "leading dimension"), (dict(ids=P, ld_ids=9), "leading dimension"), (dict(draws=2, ldu=1), "leading dimension"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"), (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"),
    (dict(min_p=-0.1), "min_p"), (dict(top_k=-1), "top_k"), (dict(top_k_dev=P), "bound"), (dict(idx=None), "NULL argument"), (dict(u=None), "NULL argument"),
    (dict(scores=None), "NULL argument"), (dict(scores=P + 1), "not aligned"), (dict(), "ctx is NULL")])
def test_sample_refuses(change, message):
    refused("rphip_sample", sample(**change), message)


def test_sample_limit():
    refused("rphip_sample", sample(width=5000, ld=5000, draws=2, ldu=2), "1024", _lib.RPHIP_ELIMIT)
    refused("rphip_sample", sample(width=5000, ld=5000, draws=2, ldu=2, top_k=1025), "1024", _lib.RPHIP_ELIMIT)
    refused("rphip_sample", sample(width=5000, ld=5000, draws=2, ldu=2, top_k=1024), "ctx is NULL")


class FakeContext:
    device, handle, lib = 0, None, None


def test_tensors_are_checked():
    ctx, x = FakeContext(), torch.zeros(4, 64)
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    m = ops.MXFP4(codes, scales, 64)
    assert m.shape == (4, 64) and m.nbytes == 4 * 34
    for call in (lambda: ops.mxfp4_quantize(ctx, x), lambda: ops.mxfp4_dequantize(ctx, m), lambda: ops.mxfp4_gemm_nt(ctx, x, m), lambda: ops.sample(ctx, x, x[:, :1])):
        with pytest.raises(ValueError, match="cpu"):  # the wrong device
            call()
    with pytest.raises(TypeError):
        ops.mxfp4_quantize(ctx, [[1.0]])
    for bad in ((codes.int(), scales, 64), (codes, scales, 65), (codes, scales[:3], 64), (codes[:, :16], scales, 64), (codes, scales.t().contiguous().t(), 64),
                (torch.zeros(4, 40, dtype=torch.uint8)[:, :32], scales, 64), (torch.zeros(4, 48, dtype=torch.uint8)[:, 8:40], scales, 64)):
        with pytest.raises(ValueError):
            ops.MXFP4(*bad)


class OnTheHost:
    """A context whose device is the tensors' own (-1: none), for checks that come after the device's."""

    device, handle, lib = -1, None, None


def test_gradients_are_refused():
    ctx, x, w = OnTheHost(), torch.zeros(4, 64, requires_grad=True), torch.zeros(5, requires_grad=True)
    plain, m = torch.zeros(4, 64), ops.MXFP4(torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8), 64)
    indptr, indices = torch.tensor([0, 2, 5], dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
    calls = [("x", lambda: ops.mxfp4_quantize(ctx, x)), ("x", lambda: ops.mxfp4_quantize(ctx, x * 2)), ("a", lambda: ops.mxfp4_gemm_nt(ctx, x, m)),
             ("weights", lambda: ops.mxfp4_scores(ctx, indptr, indices, m, weights=w)), ("scores", lambda: ops.sample(ctx, x, plain[:, :1])),
             ("temperature", lambda: ops.sample(ctx, plain, plain[:, :1], temperature=w[:4])), ("out", lambda: ops.mxfp4_dequantize(ctx, m, out=torch.zeros(64, 64, requires_grad=True)))]
    for name, call in calls:
        with pytest.raises(ValueError, match=f"^{name} requires a gradient"):
            call()
    with torch.no_grad():  # (past the check: the stand-in has no library)
        with pytest.raises(Exception) as e:
            ops.mxfp4_quantize(ctx, x)
        assert "gradient" not in str(e.value)


class Recorder:
    """Stands in for the library: notes what it is asked for, and refuses it."""

    def __init__(self):
        self.asked = []

    def rphip_sample_workspace(self, handle, rows, width, draws, top_k, size):
        self.asked.append(top_k)
        return _lib.RPHIP_EINVAL


@pytest.mark.parametrize("top_k,passed", [(0, 0), (7, 7), (2**31 - 1, 2**31 - 1), (2**32 + 5, 2**31 - 1), (10**30, 2**31 - 1), (-1, -1), (5 - 2**32, -1)])
def test_top_k_of_more_than_32_bits(top_k, passed):
    ctx = OnTheHost()
    ctx.lib = Recorder()
    with pytest.raises(_lib.RecpackHipError):
        ops.sample(ctx, torch.zeros(4, 64), torch.zeros(4, 1), top_k=top_k)
    assert ctx.lib.asked == [passed]


def test_what_is_no_tensor_is_a_type_error():
    ctx, m = OnTheHost(), ops.MXFP4(torch.zeros(64, 32, dtype=torch.uint8), torch.zeros(64, 2, dtype=torch.uint8), 64)
    indptr, indices = torch.tensor([0, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for name, call in (("indices", lambda: ops.mxfp4_scores(ctx, indptr, [0], m)), ("item_keep", lambda: ops.mxfp4_scores(ctx, indptr, indices, m, item_keep=[1] * 64)),
                       ("weights", lambda: ops.mxfp4_scores(ctx, indptr, indices, m, weights=[1.0])), ("indptr", lambda: ops.mxfp4_scores(ctx, [0, 1], indices, m)),
                       ("codes", lambda: ops.MXFP4([0], m.scales, 64)), ("u", lambda: ops.sample(ctx, torch.zeros(1, 4), [[0.5]]))):
        with pytest.raises(TypeError, match=f"^{name}: a torch tensor"):
            call()
