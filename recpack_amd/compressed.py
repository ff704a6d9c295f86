"""``CompressedEASE``: an EASE model held in 4 bits per similarity (MXFP4), and what it answers with.

The item-item matrix of :class:`recpack_amd.EASE` takes 4 bytes per pair of items (40 GB at 100 000 items); quantised by blocks of 32 it
takes 17/32 byte (5.3 GB).  The scores are those of the quantised matrix, exactly summed in float32; how far they are from the full
model's is the quantisation's doing: a similarity is off by less than a quarter of the largest in its block of 32, and by 12 % of their
root mean square where they are spread as a normal distribution is.  On two synthetic power-law matrices (3000 and 8000 items) 94 to 96 % of the
full model's 10 and 100 best items are among the compressed one's, and the scores are off by 8 % of their root mean square.  The reference has no counterpart: its ``similarity_matrix_`` is a float64 CSR (recpack/algorithms/ease.py:92).
"""
from __future__ import annotations

import numpy as np
import scipy.sparse as sp

from recpack_amd import _lib
from recpack_amd.algorithms import EASE, Algorithm, draw_uniforms, get_context, item_mask

CHUNK_BYTES = 1 << 30  # scores of a chunk of users on the device


def entries_by_row(X, in_order: bool):
    """Row pointers and column indices of the stored entries of a sparse matrix, by rows, none of them joined; ``in_order``: as they stand, which
    is by rows in a CSR matrix only."""
    if X.format == "csr":
        return X.indptr, X.indices[:X.indptr[-1]]
    if in_order:
        raise ValueError(f"weights go with the stored entries of a CSR matrix, X is {X.format}")
    coo = X.tocoo()
    indptr = np.zeros(X.shape[0] + 1, dtype=np.int64)
    np.cumsum(np.bincount(coo.row, minlength=X.shape[0]), out=indptr[1:])
    return indptr, coo.col[np.argsort(coo.row, kind="stable")]


class CompressedEASE(Algorithm):
    """EASE (recpack/algorithms/ease.py:19-109) whose fitted matrix is kept in MXFP4 (:mod:`recpack_amd.ops`) instead of float32.

    Same constructor arguments as :class:`EASE`, and ``profiles``: also keep the matrix quantised along the other axis, for
    :meth:`profile_scores` (as much memory again).  ``fit`` fits EASE, quantises and lets the float32 matrix go; ``EASE.compress()`` makes one
    from a model that is already fitted."""

    def __init__(self, l2=1e3, alpha=0, density=None, profiles=False):
        super().__init__()
        self.l2 = l2
        self.alpha = alpha
        self.density = density
        self.profiles = profiles

    # ---- the model --------------------------------------------------------------------------------------------------------------------
    def _fit(self, X: sp.csr_matrix):
        ease = EASE(self.l2, self.alpha, self.density)
        ease._fit(X)
        try:
            self._compress(ease._model)
        finally:
            ease._model.close()

    def _compress(self, model: "_lib.Model"):
        import torch

        from recpack_amd import ops

        ctx = model.ctx
        if model.kind != _lib.RPHIP_MODEL_DENSE or model.dense_layout()["n_local"] != model.n_items or model.dense_layout()["panel"]:
            raise ValueError("only a whole dense model can be compressed")
        ptr, n, ld = model.dense_device_ptr()
        ctx.sync()  # (B is written on the context's stream, read on torch's)
        B = torch.as_tensor(_lib._DevBytes(ptr, ld * n * 4), device=f"cuda:{ctx.device}").view(torch.float32).view(n, ld)[:, :n]
        self._rows = ops.mxfp4_quantize(ctx, B)
        self._columns = ops.mxfp4_quantize(ctx, B, transpose=True) if self.profiles else None
        torch.cuda.current_stream(ctx.device).synchronize()  # (the caller may let B go)
        self._host = None
        self.n_items_ = n

    def __getstate__(self):
        state = dict(super().__getstate__() if hasattr(super(), "__getstate__") else self.__dict__)
        rows, columns = state.pop("_rows", None), state.pop("_columns", None)
        if rows is not None:
            state["_host"] = [None if m is None else (m.codes.cpu().numpy(), m.scales.cpu().numpy()) for m in (rows, columns)]
        return state

    def __setstate__(self, state):
        if hasattr(super(), "__setstate__"):
            super().__setstate__(state)
        else:
            self.__dict__.update(state)

    def _matrices(self):
        """(rows, columns) on the device; an unpickled model is uploaded on its first use."""
        if getattr(self, "_rows", None) is None:
            host = getattr(self, "_host", None)
            if host is not None:
                self._columns = self._upload(host[1])
                self._rows = self._upload(host[0])  # (the last one: it says that both are there, also to another thread)
                self._host = None
            elif getattr(self, "_rows", None) is None:
                raise AttributeError("CompressedEASE is not fitted")
        return self._rows, self._columns

    def _upload(self, arrays):
        import torch

        from recpack_amd import ops

        if arrays is None:
            return None
        m = ops.MXFP4.empty(arrays[0].shape[0], self.n_items_, f"cuda:{get_context().device}")
        m.codes.copy_(torch.from_numpy(arrays[0]))
        m.scales.copy_(torch.from_numpy(arrays[1]))
        return m

    def _check_fit_complete(self):
        if getattr(self, "_rows", None) is None and getattr(self, "_host", None) is None:
            raise AttributeError("CompressedEASE is not fitted")

    @property
    def similarity_matrix_(self) -> sp.csr_matrix:
        """The quantised similarities as a float64 CSR (made anew on every access)."""
        from recpack_amd import ops

        self._check_fit_complete()
        return sp.csr_matrix(ops.mxfp4_dequantize(get_context(), self._matrices()[0]).cpu().numpy().astype(np.float64))

    @property
    def nbytes(self) -> int:
        return sum(m.nbytes for m in self._matrices() if m is not None)

    # ---- answers ----------------------------------------------------------------------------------------------------------------------
    def scores(self, X: sp.csr_matrix, exclude_history: bool = False, item_keep=None, weights=None, dtype=None, out=None):
        """Scores of histories as a torch tensor [users, items] on the GPU: X @ similarity_matrix_ (base.py:248) with the stored entries of the
        sparse ``X`` counted once each (repeated ones as often as they stand), or ``weights`` (CSR only: one number per stored entry, in its order)
        times.  ``exclude_history`` / ``item_keep``: those items get -inf."""
        import torch

        from recpack_amd import ops

        rows, _ = self._matrices()
        if not sp.issparse(X):
            raise TypeError(f"X: a scipy sparse matrix is expected, got {type(X).__name__}")
        if X.shape[1] != self.n_items_:
            raise ValueError(f"X has {X.shape[1]} items, the model {self.n_items_}")
        indptr, indices = entries_by_row(X, weights is not None)
        ctx = get_context()
        device = f"cuda:{ctx.device}"

        def put(a, t):
            return torch.from_numpy(np.ascontiguousarray(a, dtype=t)).to(device)

        if len(indices) > np.iinfo(np.int32).max:
            raise ValueError("more than 2^31 stored entries: pass the users in parts")
        keep = None if item_keep is None else put(np.asarray(item_keep) != 0, np.uint8)
        w = None if weights is None else put(weights, np.float32)
        return ops.mxfp4_scores(ctx, put(indptr, np.int32), put(indices, np.int32), rows, weights=w, exclude_history=exclude_history, item_keep=keep,
                                dtype=dtype or torch.float32, out=out)

    def profile_scores(self, profiles, dtype=None):
        """Scores of dense, real-valued user profiles [m, items] (numpy or torch; float32, float16 or bfloat16): profiles @ similarity_matrix_
        with the matrix quantised along its first axis (``profiles=True``), on the matrix cores.  What predict of a dense model refuses
        (valued prediction matrices) - decayed, averaged or folded-in profiles.  Returns a torch tensor on the GPU."""
        import torch

        from recpack_amd import ops

        _, columns = self._matrices()
        if columns is None:
            raise ValueError("profile_scores needs CompressedEASE(..., profiles=True)")
        ctx = get_context()
        P = profiles if isinstance(profiles, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(profiles, dtype=np.float32))
        return ops.mxfp4_gemm_nt(ctx, P.to(f"cuda:{ctx.device}"), columns, dtype=dtype)

    def _chunks(self, X):
        per = max(1, CHUNK_BYTES // (4 * max(self.n_items_, 1)))
        for u0 in range(0, X.shape[0], per):
            yield u0, X[u0:u0 + per]

    def _predict(self, X: sp.csr_matrix) -> sp.csr_matrix:
        parts = [sp.csr_matrix(self.scores(part).cpu().numpy().astype(np.float64)) for _, part in self._chunks(X)]
        return sp.vstack(parts, format="csr") if parts else sp.csr_matrix(X.shape)

    def _candidates(self, part, exclude_history, keep):
        """Scores with everything that cannot be recommended at -inf: masked items, and zeros (predict does not store them)."""
        s = self.scores(part, exclude_history=exclude_history, item_keep=keep)
        return s.masked_fill_(s == 0, -np.inf)

    def predict_topk(self, X, K: int, exclude_history: bool = False, exclude_items=None, select_items=None) -> sp.csr_matrix:
        """The K best scores per user, as ``ItemSimilarityMatrixAlgorithm.predict_topk`` returns them (K <= 1024; a small catalogue's number of items
        takes a larger K's place)."""
        import torch

        from recpack_amd import ops

        self._check_fit_complete()
        X = self._transform_predict_input(X)
        K = min(int(K), max(1, self.n_items_))
        if K > ops.SLATE_MAX:
            raise ValueError(f"predict_topk of a compressed model takes K <= {ops.SLATE_MAX}, got {K}")
        keep = item_mask(X, exclude_items, select_items)
        parts = []
        for _, part in self._chunks(X):
            s = self._candidates(part, exclude_history, keep)
            idx, _, n = ops.sample(get_context(), s, torch.zeros(s.shape[0], K, device=s.device), temperature=0.0, top_k=K)
            val = s.gather(1, idx.clamp(min=0).long()).cpu().numpy().astype(np.float64)
            idx, n = idx.cpu().numpy(), n.cpu().numpy()
            mask = np.arange(K)[None, :] < n[:, None]
            indptr = np.zeros(len(n) + 1, dtype=np.int64)
            np.cumsum(n, out=indptr[1:])
            m = sp.csr_matrix((val[mask], idx[mask], indptr), shape=part.shape)
            m.sort_indices()
            parts.append(m)
        return sp.vstack(parts, format="csr") if parts else sp.csr_matrix(X.shape)

    def predict_sample(self, X, n: int = 1, K: int = 0, temperature: float = 1.0, top_p: float = 1.0, min_p: float = 0.0, exclude_history: bool = False, exclude_items=None,
                       select_items=None, u=None, seed=None):
        """``n`` items drawn without replacement from every user's scores: ``ItemSimilarityMatrixAlgorithm.predict_sample`` with the whole
        catalogue as candidates (``K`` = 0, n = 1) or the best ``K`` <= 1024."""
        import torch

        from recpack_amd import ops

        self._check_fit_complete()
        X = self._transform_predict_input(X)
        keep = item_mask(X, exclude_items, select_items)
        u = draw_uniforms(u, seed, X.shape[0], n)
        items, probs = np.full(u.shape, -1, np.int32), np.zeros(u.shape, np.float32)
        for u0, part in self._chunks(X):
            s = self._candidates(part, exclude_history, keep)
            uu = torch.from_numpy(u[u0:u0 + s.shape[0]]).to(s.device)
            idx, p, _ = ops.sample(get_context(), s, uu, temperature=temperature, top_k=int(K), top_p=top_p, min_p=min_p)
            items[u0:u0 + s.shape[0]], probs[u0:u0 + s.shape[0]] = idx.cpu().numpy(), p.cpu().numpy()
        return items, probs
