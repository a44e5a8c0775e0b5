"""Training on a mined sample matrix (sc_trainer_*, sc_lr_*, sc_sample): what
GentleAdaboost::Train does with the descriptors a Miner leaves on the GPU
(GentleAdaboost.cpp:11-231), on torch device tensors.

    miner.mine_batch_device(frames, capacity, samples)    # [n, n_patches, 32]
    tr = Trainer()
    rows, _ = tr.sample(log_weight, u)                    # the roulette wheel
    loss, dw, db = tr.loss(samples, w, target, b, rows=rows[0])
    score = tr.response(samples, w, b, residual=score, alpha=1 / k, beta=1 - 1 / k)
"""
from __future__ import annotations

import ctypes

from . import SurfCascadeError, _check, load_library  # noqa: F401

_ACT = {"none": 0, "sigmoid": 1}
_RES = {None: 0, "none": 0, "row": 1, "full": 2}


class _Samples(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("n_patches", ctypes.c_int32),
                ("n", ctypes.c_int64), ("ld", ctypes.c_int64), ("rows", ctypes.c_void_p),
                ("n_rows", ctypes.c_int64)]


class _WeakBank(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int32), ("h", ctypes.c_int32), ("patch", ctypes.c_void_p),
                ("w", ctypes.c_void_p), ("b", ctypes.c_void_p)]


class _SampleParams(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_double), ("top_k", ctypes.c_int32),
                ("top_p", ctypes.c_double), ("min_p", ctypes.c_double)]


class Trainer:
    """Launches the training kernels of one GPU (sc_trainer).  Calls are
    asynchronous and ordered like torch operations: they run on torch's current
    stream of the trainer's device, allocate their results and workspaces from
    torch, and can be captured into a graph.  Tensors live on the trainer's
    device; a layout the C ABI does not take is refused, not copied.  One
    trainer is not thread-safe.

    samples: [n, n_patches, 32] float32, float16 or bfloat16, each sample's
    descriptors contiguous (any stride between samples).  w: float32
    [m, 32] or [m, h, 32]; b: None or float32 [m] or [m, h].  patch: None or
    int32 [m]; rows: None or int32 [r].  A row or patch number out of range is
    absent (include/surfcascade.h)."""

    def __init__(self, device: int = 0):
        import torch
        self._torch = torch
        self._dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self._L = load_library()
        self.device = int(device)
        self._dev = torch.device("cuda", self.device)
        h = ctypes.c_void_p()
        _check(self._L.sc_trainer_create(self.device, ctypes.byref(h)))
        self._h = h.value
        self._on = None  # the raw stream it launches on, once set
        self._raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)

    def close(self):
        if getattr(self, "_h", None):
            self._L.sc_trainer_destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()

    def synchronize(self):
        _check(self._L.sc_trainer_synchronize(self._h))

    # -- operands ------------------------------------------------------------
    def _follow(self):
        """Launch on torch's current stream of this device (a trainer that
        changes streams waits for its earlier work, sc_trainer_set_stream)."""
        if self._h is None:
            raise ValueError("the trainer is closed")
        s = self._raw(self.device) if self._raw is not None \
            else self._torch.cuda.current_stream(self.device).cuda_stream
        if s != self._on:
            _check(self._L.sc_trainer_set_stream(self._h, s or None, 0))
            self._on = s

    def _need(self, t, dtype, shape, what):
        """A contiguous tensor of this type and shape on this device."""
        if t.dtype != dtype or t.get_device() != self.device:
            raise ValueError("%s must be a %s tensor on cuda:%d (got %s on %s)"
                             % (what, dtype, self.device, t.dtype, t.device))
        if tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError("%s must be contiguous, of shape %s (got %s, strides %s)"
                             % (what, shape, tuple(t.shape), t.stride()))
        return t.data_ptr()

    def _rowwise(self, t, dtype, r, cols, what):
        """[r, cols] (or [r, m, h], cols = m*h) values, each row contiguous ->
        (pointer, stride between rows)."""
        if t.dtype != dtype or t.get_device() != self.device:
            raise ValueError("%s must be a %s tensor on cuda:%d (got %s on %s)"
                             % (what, dtype, self.device, t.dtype, t.device))
        n, step = 1, 1
        for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if size != 1 and stride != step:
                raise ValueError("each row of %s must be contiguous (strides %s)" % (what, t.stride()))
            step *= size
            n *= size
        if t.dim() < 2 or t.shape[0] != r or n != cols:
            raise ValueError("%s must have %d rows of %d values (got %s)" % (what, r, cols, tuple(t.shape)))
        ld = t.stride(0)
        if r > 1 and cols > 0 and ld < cols:
            raise ValueError("rows of %s overlap (strides %s)" % (what, t.stride()))
        return t.data_ptr(), max(ld, cols)

    def _operands(self, samples, w, b, patch, rows):
        torch = self._torch
        if samples.dtype not in self._dtypes or samples.get_device() != self.device:
            raise ValueError("samples must be float32, float16 or bfloat16 on cuda:%d (got %s on %s)"
                             % (self.device, samples.dtype, samples.device))
        if samples.dim() != 3 or samples.shape[2] != 32:
            raise ValueError("samples must be [n, n_patches, 32] (got %s)" % (tuple(samples.shape),))
        n, p, _ = samples.shape
        s0, s1, s2 = samples.stride()
        if s2 != 1 or (p > 1 and s1 != 32) or (n > 1 and s0 < 32 * p):
            raise ValueError("each sample's descriptors must be contiguous (strides %s)" % (samples.stride(),))
        if w.dim() not in (2, 3) or w.shape[-1] != 32:
            raise ValueError("w must be [m, 32] or [m, h, 32] (got %s)" % (tuple(w.shape),))
        sets = tuple(w.shape[:-1])  # (m,) or (m, h)
        m, h = sets[0], (sets[1] if len(sets) == 2 else 1)
        x = _Samples(samples.data_ptr(), self._dtypes[samples.dtype], p, n, max(s0, 32 * p), None, 0)
        r = n
        if rows is not None:
            r = rows.numel()
            x.rows = self._need(rows, torch.int32, (r,), "rows") or 1  # (an empty tensor has no address)
            x.n_rows = r
        k = _WeakBank(m, h, None if patch is None else self._need(patch, torch.int32, (m,), "patch") or None,
                      self._need(w, torch.float32, sets + (32,), "w"),
                      None if b is None else self._need(b, torch.float32, sets, "b") or None)
        if patch is None and m > p:
            raise ValueError("%d weak learners, %d patches and no patch numbers" % (m, p))
        return x, k, r, sets, m * h

    def _empty(self, shape, dtype=None):
        return self._torch.empty(shape, dtype=dtype or self._torch.float32, device=self._dev)

    def _workspace(self, bytes_):
        return self._torch.empty(bytes_, dtype=self._torch.uint8, device=self._dev) if bytes_ else None

    @staticmethod
    def _ptr(t):
        return None if t is None else t.data_ptr()

    # -- weak learners -------------------------------------------------------
    def response(self, samples, w, b=None, patch=None, rows=None, activation="sigmoid", alpha=1.0,
                 residual=None, beta=1.0, out=None):
        """alpha * act(x . w + b) + beta * residual for every row and learner
        -> float32 [r, m] or [r, m, h] (sc_lr_response).  residual: None, one
        value per row [r], or one per result; out may be that residual."""
        self._follow()
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        res, kind, res_ld = None, 0, 0
        if residual is not None and residual.dim() == 1:
            kind, res_ld = 1, 1
            if residual.shape[0] != r or residual.dtype != self._torch.float32 \
                    or residual.get_device() != self.device or (r > 1 and residual.stride(0) < 1):
                raise ValueError("residual must be float32 [%d] on cuda:%d" % (r, self.device))
            res, res_ld = residual.data_ptr(), max(residual.stride(0), 1)
        elif residual is not None:
            kind = 2
            res, res_ld = self._rowwise(residual, self._torch.float32, r, cols, "residual")
        if out is None:
            out = self._empty((r,) + sets)
            y, y_ld = out.data_ptr(), cols
        else:
            y, y_ld = self._rowwise(out, self._torch.float32, r, cols, "out")
        _check(self._L.sc_lr_response(self._h, ctypes.byref(x), ctypes.byref(k), _ACT[activation], alpha,
                                      res, kind, res_ld, beta, y, y_ld))
        return out

    def response_grad(self, samples, w, grad_out, b=None, patch=None, rows=None, activation="sigmoid",
                      alpha=1.0, residual=None, beta=1.0):
        """Backward pass of `response` for grad_out ([r, m] or [r, m, h]) ->
        (dw like w, db [m] or [m, h], dres or None) (sc_lr_response_grad).
        residual: None or "none", "row" or "full", the residual's kind."""
        self._follow()
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        dy, dy_ld = self._rowwise(grad_out, self._torch.float32, r, cols, "grad_out")
        kind = _RES[residual]
        dw, db = self._empty(sets + (32,)), self._empty(sets)
        dres = self._empty((r,) if kind == 1 else (r,) + sets) if kind else None
        ws, ws_bytes = self._lr_workspace(x, k)
        _check(self._L.sc_lr_response_grad(self._h, ctypes.byref(x), ctypes.byref(k), _ACT[activation], alpha,
                                           dy, dy_ld, dw.data_ptr(), db.data_ptr(), kind, beta,
                                           self._ptr(dres), 1 if kind == 1 else cols, self._ptr(ws), ws_bytes))
        return dw, db, dres

    def loss(self, samples, w, target, b=None, weight=None, patch=None, rows=None):
        """Weighted logistic loss of every learner with its gradient ->
        (loss [m] or [m, h], dw like w, db) (sc_lr_loss).  target and weight:
        float32 [n], by sample; a sample of weight 0 is not looked at."""
        self._follow()
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        n = samples.shape[0]
        t = self._need(target, self._torch.float32, (n,), "target")
        c = None if weight is None else self._need(weight, self._torch.float32, (n,), "weight") or None
        loss, dw, db = self._empty(sets), self._empty(sets + (32,)), self._empty(sets)
        ws, ws_bytes = self._lr_workspace(x, k)
        _check(self._L.sc_lr_loss(self._h, ctypes.byref(x), ctypes.byref(k), t, c, loss.data_ptr(),
                                  dw.data_ptr(), db.data_ptr(), self._ptr(ws), ws_bytes))
        return loss, dw, db

    def _lr_workspace(self, x, k):
        size = ctypes.c_size_t()
        _check(self._L.sc_lr_workspace(ctypes.byref(x), ctypes.byref(k), ctypes.byref(size)))
        return self._workspace(size.value), size.value

    # -- draws ---------------------------------------------------------------
    def sample(self, scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lens=None):
        """Draws places from each row of scores (log-weights, [v] or [b, v]
        float32, float16 or bfloat16) by the random numbers u (float64 [s] or
        [b, s], in [0, 1)) -> (index int32 like u, kept int32 [b])
        (sc_sample).  lens: int32 [b], the length of each row."""
        torch = self._torch
        self._follow()
        if scores.dtype not in self._dtypes or scores.get_device() != self.device:
            raise ValueError("scores must be float32, float16 or bfloat16 on cuda:%d (got %s on %s)"
                             % (self.device, scores.dtype, scores.device))
        if scores.dim() not in (1, 2) or u.dim() != scores.dim():
            raise ValueError("scores [v] with u [s], or scores [b, v] with u [b, s] (got %s and %s)"
                             % (tuple(scores.shape), tuple(u.shape)))
        s2 = scores if scores.dim() == 2 else scores[None]
        u2 = u if u.dim() == 2 else u[None]
        b, v = s2.shape
        s = u2.shape[1]
        sc, ld = self._rowwise(s2, scores.dtype, b, v, "scores")
        up, u_ld = self._rowwise(u2, torch.float64, b, s, "u")
        ln = None if lens is None else self._need(lens, torch.int32, (b,), "lens") or None
        index, kept = self._empty(tuple(u.shape), torch.int32), self._empty((b,), torch.int32)
        prm = _SampleParams(temperature, top_k, top_p, min_p)
        size = ctypes.c_size_t()
        _check(self._L.sc_sample_workspace(b, v, s, ctypes.byref(size)))
        ws = self._workspace(size.value)
        _check(self._L.sc_sample(self._h, sc, self._dtypes[scores.dtype], b, v, ld, ln, ctypes.byref(prm), up, s,
                                 u_ld, index.data_ptr(), s, kept.data_ptr(), self._ptr(ws), size.value))
        return index, kept

    # -- models --------------------------------------------------------------
    def bank(self, weak_classifiers):
        """(w [m, 32], b [m], patch [m]) of trained weak classifiers
        (LogisticRegression objects, a StageClassifier's list): their bias
        input folded in, b = w[32] * bias (LogisticRegression.cpp:60-64)."""
        torch = self._torch
        weak = list(weak_classifiers)
        w = torch.tensor([[float(v) for v in k.w[:32]] for k in weak], dtype=torch.float32).reshape(len(weak), 32)
        b = torch.tensor([float(k.w[32]) * k.bias for k in weak], dtype=torch.float64).float()
        patch = torch.tensor([k.patch_index for k in weak], dtype=torch.int32)
        return w.to(self._dev), b.to(self._dev), patch.to(self._dev)
