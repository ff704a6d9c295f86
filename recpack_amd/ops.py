"""Operators on torch CUDA tensors: 4-bit (MXFP4) matrices, their products, and sampling from scores (include/recpack_hip.h, last section).

Every function takes the :class:`recpack_amd._lib.Context` of the tensors' device first and runs on torch's current stream of that
device; nothing is copied to the host or waited for, so the calls can be captured into a graph.  Outputs may be given (``out=``);
otherwise they are allocated.  There is no backward pass: a fitted model is compressed and answered from, not trained through.
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
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _stream(ctx):
    return C.c_void_p(torch.cuda.current_stream(ctx.device).cuda_stream)


def _on(ctx, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name}: a torch tensor is expected, got {type(t).__name__}")
        if not t.is_cuda or t.device.index != ctx.device:
            raise ValueError(f"{name} is on {t.device}, the context on cuda:{ctx.device}")


def _floating(name, t):
    if t.dtype not in _TYPES:
        raise TypeError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")


def _matrix(name, t):
    """A two-dimensional tensor whose rows are contiguous (copied if they are not), and its leading dimension."""
    if t.dim() != 2:
        raise ValueError(f"{name}: two dimensions expected, got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t, max(t.stride(0) if t.shape[0] > 1 else 0, t.shape[1])


def _output(name, out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device), max(shape[1], 1)
    if tuple(out.shape) != tuple(shape) or (dtype is not None and out.dtype != dtype):
        raise ValueError(f"{name}: {tuple(shape)} of {dtype} expected, got {tuple(out.shape)} of {out.dtype}")
    if out.shape[1] > 1 and out.stride(1) != 1 or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError(f"{name}: rows must be contiguous and must not overlap")
    return out, max(out.stride(0) if out.shape[0] > 1 else 0, out.shape[1], 1)


class MXFP4:
    """A quantised matrix: ``codes`` uint8 [rows, 16 * blocks], ``scales`` uint8 [rows, blocks], ``cols`` (blocks = ceil(cols / 32)).

    Two elements of a row share a byte, the even one in the low nibble; 32 share a scale byte s, which stands for 2^(s - 127) (255: the
    block is NaN).  Codes beyond the last column are 0."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int):
        blocks = -(-int(cols) // BLOCK)
        for name, t, width in (("codes", codes, blocks * 16), ("scales", scales, blocks)):
            if t.dtype != torch.uint8 or t.dim() != 2 or t.shape[1] != width:
                raise ValueError(f"{name}: uint8 [rows, {width}] expected for {cols} columns, got {t.dtype} {tuple(t.shape)}")
            if t.shape[1] > 1 and t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
                raise ValueError(f"{name}: rows must be contiguous and must not overlap")
        if codes.shape[0] != scales.shape[0]:
            raise ValueError(f"{codes.shape[0]} rows of codes, {scales.shape[0]} of scales")
        if codes.numel() and (codes.data_ptr() % 16 or (codes.shape[0] > 1 and codes.stride(0) % 16)):
            raise ValueError("codes: the rows must start at multiples of 16 bytes")
        self.codes, self.scales, self.cols = codes, scales, int(cols)

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
        ldc, lds = (t.stride(0) if t.numel() and t.shape[0] > 1 else t.shape[1] for t in (self.codes, self.scales))
        return _ptr(self.codes), ldc, _ptr(self.scales), lds


def mxfp4_quantize(ctx, x: torch.Tensor, transpose: bool = False, out: MXFP4 | None = None) -> MXFP4:
    """The rows of ``x`` (with ``transpose`` its columns: the result is that of ``x.T``) in MXFP4 (rphip_mxfp4_quantize)."""
    _on(ctx, x=x)
    _floating("x", x)
    if x.dim() == 2 and x.shape[0] > 1 and x.shape[1] > 1 and x.stride(0) == 1 and x.stride(1) >= x.shape[0]:
        x, transpose = x.t(), not transpose  # a transposed view: its columns are contiguous
    x, ldx = _matrix("x", x)
    rows, cols = (x.shape[1], x.shape[0]) if transpose else x.shape
    blocks = -(-cols // BLOCK)
    if out is None:
        # (rows of more than a cache line start at one: the products read them by lines)
        width = blocks * 16
        codes = torch.empty(rows, -(-width // 128) * 128 if width > 128 else width, dtype=torch.uint8, device=x.device)
        out = MXFP4(codes[:, :width], torch.empty(rows, blocks, dtype=torch.uint8, device=x.device), cols)
    elif out.shape != (rows, cols):
        raise ValueError(f"out: {(rows, cols)} expected, got {out.shape}")
    _on(ctx, codes=out.codes, scales=out.scales)
    codes, ldc, scales, lds = out._args()
    _lib.check(ctx.lib.rphip_mxfp4_quantize(ctx.handle, _stream(ctx), x.shape[0], x.shape[1], _ptr(x), _TYPES[x.dtype], ldx, 1 if transpose else 0, codes, ldc, scales, lds))
    return out


def mxfp4_dequantize(ctx, m: MXFP4, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of a quantised matrix (exact in float32; rounded once otherwise)."""
    _on(ctx, codes=m.codes, scales=m.scales, out=out)
    dtype = out.dtype if out is not None else dtype
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    out, ldo = _output("out", out, m.shape, dtype, m.device)
    codes, ldc, scales, lds = m._args()
    _lib.check(ctx.lib.rphip_mxfp4_dequantize(ctx.handle, _stream(ctx), m.shape[0], m.cols, codes, ldc, scales, lds, _ptr(out), _TYPES[dtype], ldo))
    return out


def mxfp4_gemm_nt(ctx, a, w: MXFP4, dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ w.T`` with a quantised ``w`` [N, K] and ``a`` [M, K] a float32 / float16 / bfloat16 tensor (its products are exact) or itself
    :class:`MXFP4`.  Sums in float32; the result in ``dtype`` (default: that of ``a``, float32 for MXFP4)."""
    _on(ctx, w=w.codes, w_scales=w.scales, out=out)
    if isinstance(a, MXFP4):
        _on(ctx, a=a.codes, a_scales=a.scales)
        a_ptr, lda, a_scales, ldas = a._args()
        a_type, device = _MXFP4, a.device
        keep = a
        dtype = dtype or torch.float32
    else:
        _on(ctx, a=a)
        _floating("a", a)
        keep, lda = _matrix("a", a)
        a_ptr, a_scales, ldas, a_type, device = _ptr(keep), None, 0, _TYPES[a.dtype], a.device
        dtype = dtype or a.dtype
    if a.shape[1] != w.cols:
        raise ValueError(f"a {tuple(a.shape)} and w {w.shape}: the second dimensions must be equal")
    dtype = out.dtype if out is not None else dtype
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    m, k = a.shape
    out, ldo = _output("out", out, (m, w.shape[0]), dtype, device)
    size = C.c_int64()
    _lib.check(ctx.lib.rphip_mxfp4_gemm_nt_workspace(ctx.handle, m, w.shape[0], k, a_type, C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=device) if size.value else None
    wc, ldw, wsc, ldws = w._args()
    _lib.check(ctx.lib.rphip_mxfp4_gemm_nt(ctx.handle, _stream(ctx), m, w.shape[0], k, a_ptr, a_type, lda, a_scales, ldas, wc, ldw, wsc, ldws, _ptr(out), _TYPES[dtype],
                                           ldo, _ptr(ws), size.value))
    return out


def _vector(name, t, n, dtype):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name}: {dtype} [{n}] expected, got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def mxfp4_scores(ctx, indptr: torch.Tensor, indices: torch.Tensor, w: MXFP4, weights: torch.Tensor | None = None, exclude_history: bool = False,
                 item_keep: torch.Tensor | None = None, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """Scores of histories against a quantised item-item matrix (rphip_mxfp4_scores): row u is the sum of ``weights[e] * w[indices[e]]`` over
    the entries e of the CSR row u (int32 ``indptr`` / ``indices``).  ``exclude_history``: the history's items get -inf; ``item_keep`` (bool or
    uint8 [cols]): items with 0 get -inf."""
    _on(ctx, indptr=indptr, indices=indices, w=w.codes, w_scales=w.scales, weights=weights, item_keep=item_keep, out=out)
    if indptr.dim() != 1 or indptr.shape[0] < 1:
        raise ValueError(f"indptr: one dimension of users + 1 expected, got {tuple(indptr.shape)}")
    users, nnz = indptr.shape[0] - 1, indices.numel()
    indptr, indices = _vector("indptr", indptr, users + 1, torch.int32), _vector("indices", indices, nnz, torch.int32)
    if weights is not None:
        weights = _vector("weights", weights, nnz, torch.float32)
    if item_keep is not None:
        item_keep = _vector("item_keep", item_keep.view(torch.uint8) if item_keep.dtype == torch.bool else item_keep, w.cols, torch.uint8)
    dtype = out.dtype if out is not None else dtype
    if dtype not in _TYPES:
        raise TypeError(f"dtype: float32, float16 or bfloat16 expected, got {dtype}")
    out, ldo = _output("out", out, (users, w.cols), dtype, w.device)
    codes, ldc, scales, lds = w._args()
    _lib.check(ctx.lib.rphip_mxfp4_scores(ctx.handle, _stream(ctx), users, nnz, _ptr(indptr), _ptr(indices), _ptr(weights), w.shape[0], w.cols, codes, ldc, scales, lds,
                                          1 if exclude_history else 0, _ptr(item_keep), _ptr(out), _TYPES[dtype], ldo))
    return out


def sample(ctx, scores: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lengths: torch.Tensor | None = None,
           ids: torch.Tensor | None = None, top_k_per_row: torch.Tensor | None = None):
    """Draw ``u.shape[1]`` items without replacement from every row of ``scores`` (rphip_sample has the definition).

    ``u`` float32 [rows, draws] holds the uniforms.  ``temperature``, ``top_p`` and ``min_p`` are numbers or float32 tensors [rows]; ``top_k`` (0 =
    all) is a number, ``top_k_per_row`` int32 [rows] lowers it per row.  ``lengths`` int32 [rows]: only the first so many scores of a row count;
    ``ids`` int32 [rows, width]: what is returned in place of the index.  Returns (items int32 [rows, draws], -1 where nothing was left;
    their probabilities float32 [rows, draws]; the number drawn int32 [rows])."""
    _on(ctx, scores=scores, u=u, lengths=lengths, ids=ids, top_k_per_row=top_k_per_row)
    _floating("scores", scores)
    scores, ld = _matrix("scores", scores)
    rows, width = scores.shape
    if u.dtype != torch.float32 or u.dim() != 2 or u.shape[0] != rows:
        raise ValueError(f"u: float32 [{rows}, draws] expected, got {u.dtype} {tuple(u.shape)}")
    u, ldu = _matrix("u", u)
    draws = u.shape[1]
    if lengths is not None:
        lengths = _vector("lengths", lengths, rows, torch.int32)
    ld_ids = 0
    if ids is not None:
        if ids.dtype != torch.int32 or tuple(ids.shape) != (rows, width):
            raise ValueError(f"ids: int32 {(rows, width)} expected, got {ids.dtype} {tuple(ids.shape)}")
        ids, ld_ids = _matrix("ids", ids)
    p = _lib.SampleParams(1.0, 1.0, 0.0, int(top_k))
    keep = []
    for name, v in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)):
        if isinstance(v, torch.Tensor):
            _on(ctx, **{name: v})
            v = _vector(name, v, rows, torch.float32)
            keep.append(v)
            setattr(p, name + "_dev", v.data_ptr())
        else:
            setattr(p, name, float(v))
    if top_k_per_row is not None:
        top_k_per_row = _vector("top_k_per_row", top_k_per_row, rows, torch.int32)
        p.top_k_dev = top_k_per_row.data_ptr()
    idx = torch.empty(rows, draws, dtype=torch.int32, device=scores.device)
    prob = torch.empty(rows, draws, dtype=torch.float32, device=scores.device)
    nnz = torch.empty(rows, dtype=torch.int32, device=scores.device)
    size = C.c_int64()
    _lib.check(ctx.lib.rphip_sample_workspace(ctx.handle, rows, width, draws, int(top_k), C.byref(size)))
    ws = torch.empty(size.value, dtype=torch.uint8, device=scores.device) if size.value else None
    _lib.check(ctx.lib.rphip_sample(ctx.handle, _stream(ctx), rows, width, _ptr(scores), _TYPES[scores.dtype], ld, _ptr(lengths), _ptr(ids), ld_ids, draws, _ptr(u), ldu,
                                    C.byref(p), _ptr(idx), _ptr(prob), _ptr(nnz), _ptr(ws), size.value))
    return idx, prob, nnz
