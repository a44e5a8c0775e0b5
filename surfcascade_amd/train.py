"""Training on a mined sample matrix (sc_trainer_*, sc_lr_*, sc_sample): what
GentleAdaboost::Train does with the descriptors a Miner leaves on the GPU
(GentleAdaboost.cpp:11-231), on torch device tensors.

    miner.mine_batch_device(frames, capacity, samples)    # [n, n_patches, 32]
    tr = Trainer()
    rows, _ = tr.sample(log_weight, u)                    # the roulette wheel
    loss, dw, db = tr.loss(samples, w, target, b, rows=rows)
    score = tr.response(samples, w, b, residual=score, alpha=1 / k, beta=1 - 1 / k)
"""
from __future__ import annotations

import ctypes

from . import _check, _SampleParams, _Samples, _WeakBank, load_library

class UnknownName(KeyError, ValueError):
    """An activation or kind of residual that does not exist: refused as a wrong
    value, and as the missing key it is."""

    def __str__(self):
        return ValueError.__str__(self)


class _Names(dict):
    def __missing__(self, name):
        raise UnknownName("%s must be one of %s (got %r)" % (self.what, ", ".join(map(repr, self)), name))


_ACT = _Names(none=0, sigmoid=1)
_ACT.what = "activation"
_RES = _Names({None: 0, "none": 0, "row": 1, "full": 2})
_RES.what = "residual"


class Trainer:
    """Launches the training kernels of one GPU (sc_trainer).  Calls are
    asynchronous and ordered like torch operations: they run on torch's current
    stream of the trainer's device, allocate their results from torch, and can be
    captured into a graph (workspaces: the trainer's own, a captured call's the
    graph's).  Tensors live on the trainer's
    device; a layout the C ABI does not take is refused, not copied.  One
    trainer is not thread-safe.

    samples: [n, n_patches, 32] float32, float16 or bfloat16, each sample's
    descriptors contiguous (any stride between samples).  w: float32
    [m, 32] or [m, h, 32]; b: None or float32 [m] or [m, h].  patch: None or
    int32 [m]; rows: None or int32 [r].  A row or patch number out of range is
    absent (include/surfcascade.h).

    Results carry no autograd history: `response_grad` and `loss` return the
    gradients, and operands that ask for one are refused (detach them, or call
    under torch.no_grad()), as are operands with a forward-mode tangent."""

    def __init__(self, device: int = 0):
        import torch
        self._torch = torch
        self._dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self._L = load_library()
        self.device = int(device)
        self._dev = torch.device("cuda", self.device)
        self._f32, self._f64, self._i32 = torch.float32, torch.float64, torch.int32
        self._like = torch.empty_like
        self._fwd = torch.autograd.forward_ad
        self._ws = None
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
        s = self._raw(self.device) if self._raw is not None \
            else self._torch.cuda.current_stream(self.device).cuda_stream
        if s != self._on:
            if self._h is None:
                raise ValueError("the trainer is closed")
            _check(self._L.sc_trainer_set_stream(self._h, s or None, 0))
            self._on = s

    def _need(self, t, dtype, shape, what):
        """The address of a contiguous tensor of this type and shape on this
        device (an empty one: any device address)."""
        if t.dtype is not dtype or t.get_device() != self.device:
            raise ValueError("%s must be a %s tensor on cuda:%d (got %s on %s)"
                             % (what, dtype, self.device, t.dtype, t.device))
        if t.shape != shape or not t.is_contiguous():
            raise ValueError("%s must be contiguous, of shape %s (got %s, strides %s)"
                             % (what, shape, tuple(t.shape), t.stride()))
        return t.data_ptr()

    def _rowwise(self, t, dtype, r, cols, what):
        """[r, cols] (or [r, m, h], cols = m*h) values, each row contiguous ->
        (pointer, stride between rows)."""
        if t.dtype is not dtype or t.get_device() != self.device:
            raise ValueError("%s must be a %s tensor on cuda:%d (got %s on %s)"
                             % (what, dtype, self.device, t.dtype, t.device))
        shape = t.shape
        if len(shape) < 2 or shape[0] != r or t.numel() != r * cols:
            raise ValueError("%s must have %d rows of %d values (got %s)" % (what, r, cols, tuple(shape)))
        if t.is_contiguous():
            return t.data_ptr(), cols
        stride, step = t.stride(), 1
        for k in range(len(shape) - 1, 0, -1):
            if shape[k] != 1 and stride[k] != step:
                raise ValueError("each row of %s must be contiguous (strides %s)" % (what, stride))
            step *= shape[k]
        if r > 1 and stride[0] < cols:
            raise ValueError("rows of %s overlap (strides %s)" % (what, stride))
        return t.data_ptr(), max(stride[0], cols)

    def _no_grad(self, *wanted):
        """wanted: the operands' requires_grad"""
        if any(wanted) and self._torch.is_grad_enabled():
            raise ValueError("results carry no autograd history: detach the operands (response_grad and loss "
                             "return gradients)")

    def _no_tangents(self, *operands):
        """Of forward-mode differentiation (no_grad leaves it on)."""
        if any(t is not None and self._fwd.unpack_dual(t).tangent is not None for t in operands):
            raise ValueError("results carry no forward-mode tangents: detach the operands")

    def _operands(self, samples, w, b, patch, rows):
        f32, i32 = self._f32, self._i32
        if w.requires_grad or samples.requires_grad or (b is not None and b.requires_grad):
            self._no_grad(True)
        if self._fwd._current_level >= 0:
            self._no_tangents(samples, w, b)
        dtype = self._dtypes.get(samples.dtype)
        if dtype is None or samples.get_device() != self.device:
            raise ValueError("samples must be float32, float16 or bfloat16 on cuda:%d (got %s on %s)"
                             % (self.device, samples.dtype, samples.device))
        shape, sets = samples.shape, w.shape[:-1]  # sets: (m,) or (m, h)
        if len(shape) != 3 or shape[2] != 32:
            raise ValueError("samples must be [n, n_patches, 32] (got %s)" % (tuple(shape),))
        if not 1 <= len(sets) <= 2 or w.shape[-1] != 32:
            raise ValueError("w must be [m, 32] or [m, h, 32] (got %s)" % (tuple(w.shape),))
        n, p, _ = shape
        ld = 32 * p
        if not samples.is_contiguous():
            s0, s1, s2 = samples.stride()
            if s2 != 1 or (p > 1 and s1 != 32) or (n > 1 and s0 < ld):
                raise ValueError("each sample's descriptors must be contiguous (strides %s)" % (samples.stride(),))
            ld = max(s0, ld)
        m, h = sets if len(sets) == 2 else (sets[0], 1)
        r, at = n, None
        if rows is not None:
            r = rows.numel()
            at = self._need(rows, i32, (r,), "rows") or 1  # (an empty tensor has no address)
        if patch is not None:
            patch = self._need(patch, i32, (m,), "patch") or None
        elif m > p:
            raise ValueError("%d weak learners, %d patches and no patch numbers" % (m, p))
        x = _Samples(samples.data_ptr(), dtype, p, n, ld, at, r)
        k = _WeakBank(m, h, patch, self._need(w, f32, sets + (32,), "w"),
                      None if b is None else self._need(b, f32, sets, "b") or None)
        return x, k, r, sets, m * h

    def _workspace(self, rc, bytes_):
        """After a call that brought no workspace: True when it has to be made
        again with the one now in self._ws, of bytes_() bytes.  A captured call
        needs memory of its graph's own (the trainer's own is shared by its
        other calls), which torch's allocator hands out under a capture."""
        if rc == 0:
            return False
        if rc == -1:
            with self._torch.cuda.device(self._dev):
                n = bytes_() if self._torch.cuda.is_current_stream_capturing() else 0
                if n:
                    self._ws = self._torch.empty(n, dtype=self._torch.uint8, device=self._dev)
                    return True
        _check(rc)
        return False

    # -- weak learners -------------------------------------------------------
    def response(self, samples, w, b=None, patch=None, rows=None, activation="sigmoid", alpha=1.0,
                 residual=None, beta=1.0, out=None):
        """alpha * act(x . w + b) + beta * residual for every row and learner
        -> float32 [r, m] or [r, m, h] (sc_lr_response).  residual: None, one
        value per row [r], or one per result; out may be the latter, and
        overlaps no other operand (it counts as written in place)."""
        self._follow()
        act = _ACT[activation]
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        res, kind, res_ld = None, 0, 0
        if residual is not None:
            self._no_grad(residual.requires_grad)
            if self._fwd._current_level >= 0:
                self._no_tangents(residual)
            if residual.dim() == 1:
                kind, res_ld = 1, residual.stride(0)
                if residual.shape[0] != r or residual.dtype is not self._f32 \
                        or residual.get_device() != self.device or (r > 1 and res_ld < 1):
                    raise ValueError("residual must be float32 [%d] on cuda:%d" % (r, self.device))
                res, res_ld = residual.data_ptr(), max(res_ld, 1)
            else:
                kind = 2
                res, res_ld = self._rowwise(residual, self._f32, r, cols, "residual")
        if out is None:
            out = w.new_empty((r,) + sets)
            y, y_ld = out.data_ptr(), cols
        else:
            self._no_grad(out.requires_grad)
            if self._fwd._current_level >= 0:
                self._no_tangents(out)
            y, y_ld = self._rowwise(out, self._f32, r, cols, "out")
            if not out.is_inference():  # (what autograd saved of it is no longer that)
                self._torch.autograd.graph.increment_version(out)
        rc = self._L.sc_lr_response(self._h, x, k, act, alpha, res, kind, res_ld, beta, y, y_ld)
        if rc:
            _check(rc)
        return out

    def response_grad(self, samples, w, grad_out, b=None, patch=None, rows=None, activation="sigmoid",
                      alpha=1.0, residual=None, beta=1.0):
        """Backward pass of `response` for grad_out ([r, m] or [r, m, h]) ->
        (dw like w, db [m] or [m, h], dres or None) (sc_lr_response_grad).
        residual: None or "none", "row" or "full", the residual's kind."""
        self._follow()
        act, kind = _ACT[activation], _RES[residual]
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        self._no_grad(grad_out.requires_grad)
        if self._fwd._current_level >= 0:
            self._no_tangents(grad_out)
        dy, dy_ld = self._rowwise(grad_out, self._f32, r, cols, "grad_out")
        dw, db, dres, dr = self._like(w), w.new_empty(sets) if b is None else self._like(b), None, None
        if kind:
            dres = w.new_empty((r,) if kind == 1 else (r,) + sets)
            dr = dres.data_ptr()

        def call(ws, ws_bytes):
            return self._L.sc_lr_response_grad(self._h, x, k, act, alpha, dy, dy_ld, dw.data_ptr(),
                                               db.data_ptr(), kind, beta, dr, 1 if kind == 1 else cols, ws, ws_bytes)

        if self._workspace(call(None, 0), lambda: self._lr_bytes(x, k)):
            _check(call(self._ws.data_ptr(), self._ws.numel()))
            self._ws = None
        return dw, db, dres

    def loss(self, samples, w, target, b=None, weight=None, patch=None, rows=None):
        """Weighted logistic loss of every learner with its gradient ->
        (loss [m] or [m, h], dw like w, db) (sc_lr_loss).  target and weight:
        float32 [n], by sample; a sample of weight 0 is not looked at."""
        self._follow()
        x, k, r, sets, cols = self._operands(samples, w, b, patch, rows)
        self._no_grad(target.requires_grad, weight is not None and weight.requires_grad)
        if self._fwd._current_level >= 0:
            self._no_tangents(target, weight)
        n = samples.shape[0]
        t = self._need(target, self._f32, (n,), "target")
        c = None if weight is None else self._need(weight, self._f32, (n,), "weight") or None
        db, dw = w.new_empty(sets) if b is None else self._like(b), self._like(w)
        loss = self._like(db)

        def call(ws, ws_bytes):
            return self._L.sc_lr_loss(self._h, x, k, t, c, loss.data_ptr(), dw.data_ptr(), db.data_ptr(), ws, ws_bytes)

        if self._workspace(call(None, 0), lambda: self._lr_bytes(x, k)):
            _check(call(self._ws.data_ptr(), self._ws.numel()))
            self._ws = None
        return loss, dw, db

    def _lr_bytes(self, x, k):
        size = ctypes.c_size_t()
        _check(self._L.sc_lr_workspace(x, k, size))
        return size.value

    # -- draws ---------------------------------------------------------------
    def sample(self, scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lens=None):
        """Draws places from each row of scores (log-weights, [v] or [b, v]
        float32, float16 or bfloat16) by the random numbers u (float64 [s] or
        [b, s], in [0, 1)) -> (index int32 like u, kept int32 [b])
        (sc_sample).  lens: int32 [b], the length of each row."""
        self._follow()
        self._no_grad(scores.requires_grad)
        if self._fwd._current_level >= 0:
            self._no_tangents(scores)
        dtype, dim = self._dtypes.get(scores.dtype), scores.dim()
        if dtype is None or scores.get_device() != self.device:
            raise ValueError("scores must be float32, float16 or bfloat16 on cuda:%d (got %s on %s)"
                             % (self.device, scores.dtype, scores.device))
        if not 1 <= dim <= 2 or u.dim() != dim:
            raise ValueError("scores [v] with u [s], or scores [b, v] with u [b, s] (got %s and %s)"
                             % (tuple(scores.shape), tuple(u.shape)))
        shape = u.shape
        if dim == 1:
            scores, u = scores[None], u[None]
        b, v = scores.shape
        s = u.shape[1]
        sc, ld = self._rowwise(scores, scores.dtype, b, v, "scores")
        up, u_ld = self._rowwise(u, self._f64, b, s, "u")
        ln = None if lens is None else self._need(lens, self._i32, (b,), "lens") or None
        index = u.new_empty(shape, dtype=self._i32)
        kept = index.new_empty(b)
        most = 2**31 - 1  # (a C int; the library refuses rows that long, and such a top_k keeps all)
        prm = _SampleParams(temperature, max(-1, min(top_k, most)), top_p, min_p)
        if v > most or s > most or b > most:
            raise ValueError("more than 2^31 - 1 rows, scores or draws")

        def call(ws, ws_bytes):
            return self._L.sc_sample(self._h, sc, dtype, b, v, ld, ln, prm, up, s, u_ld, index.data_ptr(), s,
                                     kept.data_ptr(), ws, ws_bytes)

        if self._workspace(call(None, 0), lambda: self._sample_bytes(b, v, s)):
            _check(call(self._ws.data_ptr(), self._ws.numel()))
            self._ws = None
        return index, kept

    def _sample_bytes(self, b, v, s):
        size = ctypes.c_size_t()
        _check(self._L.sc_sample_workspace(b, v, s, size))
        return size.value

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
