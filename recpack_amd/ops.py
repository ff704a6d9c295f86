"""Operators on torch CUDA tensors: 4-bit (MXFP4) matrices, their products, and sampling from scores (include/recpack_hip.h, last section).

Every function takes the :class:`recpack_amd._lib.Context` of the tensors' device first and runs on torch's current stream of that
device; nothing is copied to the host or waited for, so the calls can be captured into a graph.  Outputs may be given (``out=``);
otherwise they are allocated.  There is no backward pass: a fitted model is compressed and answered from, not trained through
(tensors that require a gradient are refused while gradients are recorded).
"""
from __future__ import annotations

import ctypes as C

import torch

from recpack_amd import _lib

BLOCK = 32  # elements that share a scale
SLATE_MAX = 1024  # candidates (top_k, or the width) up to which several items can be drawn without replacement
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MXFP4 = 3


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _stream(ctx):
    return torch.cuda.current_stream(ctx.device).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # (the same value without a Stream object: a microsecond of a small call)

    def _stream(ctx):  # noqa: F811
        return torch._C._cuda_getCurrentRawStream(ctx.device)


def _on(ctx, name, t):
    """``t`` is a tensor on the context's GPU that nobody expects a gradient of."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: a torch tensor is expected, got {type(t).__name__}")
    if t.get_device() != ctx.device:
        raise ValueError(f"{name} is on {t.device}, the context on cuda:{ctx.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and there is no backward pass: detach it, or call under torch.no_grad()")


def _type_of(name, dtype):
    code = _TYPES.get(dtype)
    if code is None:
        raise TypeError(f"{name}: float32, float16 or bfloat16 expected, got {dtype}")
    return code


def _rows_ok(t):
    """Rows are contiguous and do not overlap."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    return (s1 == 1 or cols <= 1) and (s0 >= cols or rows <= 1)


def _matrix(name, t):
    """A two-dimensional tensor whose rows are contiguous (copied if they are not), and its leading dimension."""
    if t.dim() != 2:
        raise ValueError(f"{name}: two dimensions expected, got {tuple(t.shape)}")
    if t.is_contiguous():  # (the usual case first: a small call is as long as its checks)
        return t, t.size(1)
    if not _rows_ok(t):
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 and t.stride(0) > t.shape[1] else t.shape[1]


def _output(ctx, out, rows, cols, dtype, near):
    """The given output, checked, or a new one on the device of the tensor ``near``; with its leading dimension and element type."""
    if out is None:
        code = _type_of("dtype", dtype)
        return near.new_empty((rows, cols), dtype=dtype), cols or 1, code
    _on(ctx, "out", out)
    code = _type_of("out", out.dtype)
    if tuple(out.shape) != (rows, cols):
        raise ValueError(f"out: {(rows, cols)} expected, got {tuple(out.shape)}")
    if not _rows_ok(out):
        raise ValueError("out: rows must be contiguous and must not overlap")
    return out, max(out.stride(0) if rows > 1 else 0, cols, 1), code


def _scratch(size, near):
    """Scratch memory of a call: torch's allocator keeps it with the stream, and with the graph a call is captured into."""
    return near.new_empty(size, dtype=torch.uint8) if size else None


class MXFP4:
    """A quantised matrix: ``codes`` uint8 [rows, 16 * blocks], ``scales`` uint8 [rows, blocks], ``cols`` (blocks = ceil(cols / 32)).

    Two elements of a row share a byte, the even one in the low nibble; 32 share a scale byte s, which stands for 2^(s - 127) (255: the
    block is NaN).  Codes beyond the last column are 0."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        blocks = -(-int(cols) // BLOCK)
        for name, t, width in (("codes", codes, blocks * 16), ("scales", scales, blocks)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name}: a torch tensor is expected, got {type(t).__name__}")
            if t.dtype != torch.uint8 or t.dim() != 2 or t.shape[1] != width:
                raise ValueError(f"{name}: uint8 [rows, {width}] expected for {cols} columns, got {t.dtype} {tuple(t.shape)}")
            if not _rows_ok(t):
                raise ValueError(f"{name}: rows must be contiguous and must not overlap")
        if codes.shape[0] != scales.shape[0]:
            raise ValueError(f"{codes.shape[0]} rows of codes, {scales.shape[0]} of scales")
        if codes.get_device() != scales.get_device():
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        if codes.numel() and (codes.data_ptr() % 16 or (codes.shape[0] > 1 and codes.stride(0) % 16)):
            raise ValueError("codes: the rows must start at multiples of 16 bytes")
        self.codes, self.scales, self.cols = codes, scales, int(cols)

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "MXFP4":
        """Room for a matrix.  (The rows of one beyond a MB start at cache lines: the products read them by lines.)"""
        blocks = -(-cols // BLOCK)
        width = blocks * 16
        line = -(-width // 128) * 128 if rows * width > 1 << 20 else width
        codes = torch.empty((rows, line), dtype=torch.uint8, device=device)
        m = cls.__new__(cls)
        m.codes, m.cols = codes[:, :width] if line != width else codes, cols
        m.scales = codes.new_empty((rows, blocks))
        return m

    @property
    def shape(self):
        return (self.codes.shape[0], self.cols)

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def _args(self):
        c, s = self.codes, self.scales
        rows, width = c.shape
        if rows > 1 and width:
            return c.data_ptr(), c.stride(0), s.data_ptr(), s.stride(0)
        return c.data_ptr(), width, s.data_ptr(), s.size(1)


def mxfp4_quantize(ctx, x: torch.Tensor, transpose: bool = False, out: MXFP4 | None = None) -> MXFP4:
    """The rows of ``x`` (with ``transpose`` its columns: the result is that of ``x.T``) in MXFP4 (rphip_mxfp4_quantize)."""
    _on(ctx, "x", x)
    code = _type_of("x", x.dtype)
    if not x.is_contiguous() and x.dim() == 2 and x.shape[0] > 1 and x.shape[1] > 1 and x.stride(0) == 1 and x.stride(1) >= x.shape[0]:
        x, transpose = x.t(), not transpose  # a transposed view: its columns are contiguous
    x, ldx = _matrix("x", x)
    m, n = x.shape
    rows, cols = (n, m) if transpose else (m, n)
    if out is None:
        out = MXFP4.empty(rows, cols, x.device)
    elif out.shape != (rows, cols):
        raise ValueError(f"out: {(rows, cols)} expected, got {out.shape}")
    else:
        _on(ctx, "out", out.codes)
    codes, ldc, scales, lds = out._args()
    _lib.check(ctx.lib.rphip_mxfp4_quantize(ctx.handle, _stream(ctx), m, n, x.data_ptr(), code, ldx, 1 if transpose else 0, codes, ldc, scales, lds))
    return out


def mxfp4_dequantize(ctx, m: MXFP4, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of a quantised matrix (exact in float32; rounded once otherwise)."""
    _on(ctx, "m", m.codes)
    rows = m.codes.size(0)
    out, ldo, code = _output(ctx, out, rows, m.cols, dtype, m.codes)
    codes, ldc, scales, lds = m._args()
    _lib.check(ctx.lib.rphip_mxfp4_dequantize(ctx.handle, _stream(ctx), rows, m.cols, codes, ldc, scales, lds, out.data_ptr(), code, ldo))
    return out


def mxfp4_gemm_nt(ctx, a, w: MXFP4, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ w.T`` with a quantised ``w`` [N, K] and ``a`` [M, K] a float32 / float16 / bfloat16 tensor (its products are exact; of float32
    elements below 2^-110 the bits under 2^-133 may be left out) or itself :class:`MXFP4`.  Sums in float32; the result in ``dtype`` (default: that of ``a``, float32 for MXFP4)."""
    _on(ctx, "w", w.codes)
    if isinstance(a, MXFP4):
        _on(ctx, "a", a.codes)
        a_ptr, lda, a_scales, ldas = a._args()
        a_type, keep = _MXFP4, a
        dtype = dtype or torch.float32
    else:
        _on(ctx, "a", a)
        a_type = _type_of("a", a.dtype)
        keep, lda = _matrix("a", a)
        a_ptr, a_scales, ldas = keep.data_ptr(), None, 0
        dtype = dtype or a.dtype
    (m, k), n = a.shape, w.codes.shape[0]
    if k != w.cols:
        raise ValueError(f"a {(m, k)} and w {w.shape}: the second dimensions must be equal")
    out, ldo, code = _output(ctx, out, m, n, dtype, w.codes)
    size = C.c_int64()
    _lib.check(ctx.lib.rphip_mxfp4_gemm_nt_workspace(ctx.handle, m, n, k, a_type, C.byref(size)))
    ws = _scratch(size.value, w.codes)
    wc, ldw, wsc, ldws = w._args()
    _lib.check(ctx.lib.rphip_mxfp4_gemm_nt(ctx.handle, _stream(ctx), m, n, k, a_ptr, a_type, lda, a_scales, ldas, wc, ldw, wsc, ldws, out.data_ptr(), code, ldo, _ptr(ws),
                                           size.value))
    return out


def _vector(ctx, name, t, n, dtype):
    _on(ctx, name, t)
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: {dtype} [{n}] expected, got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def mxfp4_scores(ctx, indptr: torch.Tensor, indices: torch.Tensor, w: MXFP4, weights: torch.Tensor | None = None, exclude_history: bool = False,
                 item_keep: torch.Tensor | None = None, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """Scores of histories against a quantised item-item matrix (rphip_mxfp4_scores): row u is the sum of ``weights[e] * w[indices[e]]`` over
    the entries e of the CSR row u (int32 ``indptr`` / ``indices``).  ``exclude_history``: the history's items get -inf; ``item_keep`` (bool or
    uint8 [cols]): items with 0 get -inf."""
    _on(ctx, "w", w.codes)
    _on(ctx, "indptr", indptr)
    _on(ctx, "indices", indices)
    if indptr.dim() != 1 or indptr.shape[0] < 1:
        raise ValueError(f"indptr: one dimension of users + 1 expected, got {tuple(indptr.shape)}")
    users, nnz = indptr.shape[0] - 1, indices.numel()
    indptr, indices = _vector(ctx, "indptr", indptr, users + 1, torch.int32), _vector(ctx, "indices", indices, nnz, torch.int32)
    if weights is not None:
        weights = _vector(ctx, "weights", weights, nnz, torch.float32)
    if item_keep is not None:
        _on(ctx, "item_keep", item_keep)
        item_keep = _vector(ctx, "item_keep", item_keep.view(torch.uint8) if item_keep.dtype == torch.bool else item_keep, w.cols, torch.uint8)
    out, ldo, code = _output(ctx, out, users, w.cols, dtype, w.codes)
    codes, ldc, scales, lds = w._args()
    _lib.check(ctx.lib.rphip_mxfp4_scores(ctx.handle, _stream(ctx), users, nnz, indptr.data_ptr(), indices.data_ptr(), _ptr(weights), w.codes.shape[0], w.cols, codes, ldc,
                                          scales, lds, 1 if exclude_history else 0, _ptr(item_keep), out.data_ptr(), code, ldo))
    return out


def sample(ctx, scores: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lengths: torch.Tensor | None = None,
           ids: torch.Tensor | None = None, top_k_per_row: torch.Tensor | None = None):
    """Draw ``u.shape[1]`` items without replacement from every row of ``scores`` (rphip_sample has the definition).

    ``u`` float32 [rows, draws] holds the uniforms.  ``temperature``, ``top_p`` and ``min_p`` are numbers or float32 tensors [rows]; ``top_k`` (0 =
    all) is a number, ``top_k_per_row`` int32 [rows] lowers it per row.  ``lengths`` int32 [rows]: only the first so many scores of a row count;
    ``ids`` int32 [rows, width]: what is returned in place of the index.  Returns (items int32 [rows, draws], -1 where nothing was left;
    their probabilities float32 [rows, draws]; the number drawn int32 [rows])."""
    _on(ctx, "scores", scores)
    _on(ctx, "u", u)
    code = _type_of("scores", scores.dtype)
    scores, ld = _matrix("scores", scores)
    rows, width = scores.shape
    if u.dtype != torch.float32 or u.dim() != 2 or u.shape[0] != rows:
        raise ValueError(f"u: float32 [{rows}, draws] expected, got {u.dtype} {tuple(u.shape)}")
    u, ldu = _matrix("u", u)
    draws = u.shape[1]
    if lengths is not None:
        lengths = _vector(ctx, "lengths", lengths, rows, torch.int32)
    ld_ids = 0
    if ids is not None:
        _on(ctx, "ids", ids)
        if ids.dtype != torch.int32 or tuple(ids.shape) != (rows, width):
            raise ValueError(f"ids: int32 {(rows, width)} expected, got {ids.dtype} {tuple(ids.shape)}")
        ids, ld_ids = _matrix("ids", ids)
    top_k = max(-1, min(int(top_k), 2**31 - 1))  # (the library's argument has 32 bits; beyond the width it means all, below 0 it is refused)
    p = _lib.SampleParams(1.0, 1.0, 0.0, top_k)
    keep = []  # (copies of strided settings live until the call is made)
    for name, v in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if isinstance(v, torch.Tensor):
            v = _vector(ctx, name, v, rows, torch.float32)
            keep.append(v)
            setattr(p, name + "_dev", v.data_ptr())
        else:
            setattr(p, name, float(v))
    if top_k_per_row is not None:
        top_k_per_row = _vector(ctx, "top_k_per_row", top_k_per_row, rows, torch.int32)
        p.top_k_dev = top_k_per_row.data_ptr()
    idx = u.new_empty((rows, draws), dtype=torch.int32)
    prob = u.new_empty((rows, draws))
    nnz = u.new_empty(rows, dtype=torch.int32)
    size = C.c_int64()
    _lib.check(ctx.lib.rphip_sample_workspace(ctx.handle, rows, width, draws, top_k, C.byref(size)))
    ws = _scratch(size.value, scores)
    _lib.check(ctx.lib.rphip_sample(ctx.handle, _stream(ctx), rows, width, scores.data_ptr(), code, ld, _ptr(lengths), _ptr(ids), ld_ids, draws, u.data_ptr(), ldu,
                                    C.byref(p), idx.data_ptr(), prob.data_ptr(), nnz.data_ptr(), _ptr(ws), size.value))
    return idx, prob, nnz
