"""Operators on token ids, logits and pairs of answers, as torch calls on one MI355X (C-ABI: include/mlease_operators.h).

They stand beside the trainer's own, which do not call them: a lookup of rows by id with a scaling (``HipScorer.score_rows`` sums a
row's coefficients, this gives each id's row), and its gradient by sorted ids, the log-likelihood of a token among many classes with
its gradient (``HipAdmmEngine.test_loglik_sums`` has two), and the logistic loss with weight and offset on the margins of pairs.

    ops = HipOperators(device=0)
    x = ops.embedding_lookup(table, ids, scale=math.sqrt(width))
    ...                                                     # the caller's own layers
    logp, stats = ops.token_loglik(logits, target)
    r = ops.preference_loss(logp, ref_logp, seq_ptr, beta=0.1, scale=1.0 / pairs, mask=mask)
    dlogits = ops.token_loglik_gradient(logits, target, stats, r.grad, out=logits)
    ...
    ops.embedding_gradient(dx, ids, n_rows, scale=math.sqrt(width), out=table_grad, accumulate=True)

Gradients are calls of their own, as everywhere in this package: nothing records them. A tensor that automatic differentiation
follows is refused, since its gradient would be missing without a word; layers recorded by torch meet these calls at
`logits.detach()` and take the gradient from there with `logits.backward(dlogits)`. Every call enqueues its work on torch's
current stream of the device and returns; it allocates its outputs and workspace from torch on that stream, so that it can be
captured into a graph and made from several threads and streams. Tensors that were written on another stream need the caller's
event, as for any torch operation. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

from .hip_engine import load_library

# every entry point include/mlease_operators.h declares
OPERATOR_SYMBOLS = [
    "mlx_embedding_lookup", "mlx_embedding_gradient_workspace", "mlx_embedding_gradient", "mlx_token_loglik_workspace", "mlx_token_loglik",
    "mlx_token_loglik_gradient", "mlx_preference_loss_workspace", "mlx_preference_loss",
]

PreferenceResult = namedtuple("PreferenceResult", "loss pair_loss margin ratio grad")


def load_operators():
    """The HIP library with the operators' argument types declared."""
    L = load_library()
    if not getattr(L, "_operators_declared", False):
        vp, i32, i64, f32, sz = C.c_void_p, C.c_int32, C.c_int64, C.c_float, C.c_size_t
        psz = C.POINTER(sz)
        L.mlx_embedding_lookup.argtypes = [i32, vp, i32, vp, i64, i64, i64, i32, vp, i64, f32, vp, i64]
        L.mlx_embedding_gradient_workspace.argtypes = [i64, i64, i64, psz]
        L.mlx_embedding_gradient.argtypes = [i32, vp, i32, vp, i64, i32, vp, i64, f32, i32, i32, vp, i64, i64, i64, vp, sz]
        L.mlx_token_loglik_workspace.argtypes = [i64, i64, psz]
        L.mlx_token_loglik.argtypes = [i32, vp, i32, vp, i64, i64, i64, i32, vp, vp, vp, vp, sz]
        L.mlx_token_loglik_gradient.argtypes = [i32, vp, i32, vp, i64, i64, i64, i32, vp, vp, vp, vp, i64]
        L.mlx_preference_loss_workspace.argtypes = [i64, i64, psz]
        L.mlx_preference_loss.argtypes = [i32, vp, vp, vp, i64, vp, i64, f32, f32, f32, i32, vp, vp, vp, vp, vp, vp, vp, vp, vp, sz]
        L._operators_declared = True
    return L


class HipOperators:
    """The operators on one device. Arguments that a call cannot take raise ValueError (wrong tensors) or RuntimeError (the library's checks)."""

    def __init__(self, device: int = 0):
        import torch

        self.L = load_operators()
        if not torch.cuda.is_available():
            raise RuntimeError("no HIP device visible: the MI355X path has no CPU fallback")
        if not 0 <= int(device) < torch.cuda.device_count():
            raise RuntimeError("device %d out of range (%d devices)" % (device, torch.cuda.device_count()))
        self.device = int(device)
        self._setup(torch)

    def _setup(self, torch):
        self._torch = torch
        self._at = torch.device("cuda", self.device)
        self._types = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
        self._id_types = {torch.int32: 0, torch.int64: 1}
        self._f32 = torch.float32
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)       # the stream's handle without the object around it: 2 us of a call
        self._forward = torch.autograd.forward_ad
        at, device = self._at, self.device
        self._stream = (lambda: raw(device)) if raw else (lambda: torch.cuda.current_stream(at).cuda_stream)

    # -- checks -----------------------------------------------------------------------------------
    def _as_stored(self, t, what):
        """Nothing records these calls: what came back for a tensor that automatic differentiation follows would silently lack its gradient."""
        if t.requires_grad and self._torch.is_grad_enabled():
            raise ValueError("%s requires a gradient, which these calls do not record: pass it detached (gradients are calls of their own)" % what)
        if self._forward._current_level >= 0 and self._forward.unpack_dual(t).tangent is not None:
            raise ValueError("%s carries a forward-mode tangent, which these calls do not follow" % what)
        if t.is_neg():
            raise ValueError("%s is a view that torch negates when it is read: pass its resolve_neg()" % what)

    def _matrix(self, t, what):
        """(pointer, ld) of a 2-D tensor of this device whose rows are contiguous."""
        if t.dim() != 2 or t.dtype not in self._types:
            raise ValueError("%s must be a matrix of float32, bfloat16 or float16, not %d-dimensional %s" % (what, t.dim(), t.dtype))
        if t.device != self._at:
            raise ValueError("%s is on %s, these operators are on %s" % (what, t.device, self._at))
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError("the rows of %s must be contiguous (strides %s)" % (what, tuple(t.stride())))
        if t.requires_grad or self._forward._current_level >= 0 or t.is_neg():
            self._as_stored(t, what)
        return t.data_ptr(), t.stride(0)

    def _vector(self, t, what, n, dtype):
        if t.requires_grad or self._forward._current_level >= 0 or t.is_neg():
            self._as_stored(t, what)
        if t.dtype is dtype and t.dim() == 1 and t.numel() == n and t.device == self._at and t.is_contiguous():
            return t.data_ptr()
        if t.dim() != 1 or t.shape[0] != n or t.dtype != dtype:
            raise ValueError("%s must be a vector of %d %s, not %s %s" % (what, n, dtype, tuple(t.shape), t.dtype))
        if t.device != self._at:
            raise ValueError("%s is on %s, these operators are on %s" % (what, t.device, self._at))
        raise ValueError("%s must be contiguous" % what)

    def _ids(self, t, what, n=None):
        """(pointer, type) of a vector of ids."""
        if t.dim() != 1 or t.dtype not in self._id_types or (n is not None and t.shape[0] != n):
            raise ValueError("%s must be a vector of %sint32 or int64, not %s %s" % (what, "" if n is None else "%d " % n, tuple(t.shape), t.dtype))
        if t.device != self._at:
            raise ValueError("%s is on %s, these operators are on %s" % (what, t.device, self._at))
        if not t.is_contiguous():
            raise ValueError("%s must be contiguous" % what)
        return t.data_ptr(), self._id_types[t.dtype]

    def _output(self, out, shape, dtype):
        """(tensor, pointer, ld) of a new matrix, or of the caller's."""
        if out is None:
            out = self._torch.empty(shape, dtype=dtype, device=self._at)
            return out, out.data_ptr(), shape[1]
        if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
            raise ValueError("out must be %s %s, not %s %s" % (tuple(shape), dtype, tuple(out.shape), out.dtype))
        p, ld = self._matrix(out, "out")
        return out, p, ld

    def _workspace(self, query, *sizes):
        need = C.c_size_t()
        self._ck(query(*sizes, C.byref(need)))
        if not need.value:
            return None, None, 0
        w = self._torch.empty(need.value, dtype=self._torch.uint8, device=self._at)      # torch's blocks are aligned to 512 bytes
        return w, w.data_ptr(), need.value

    def _ck(self, rc, written=None):
        """written: the caller's tensor that a call's kernels write; torch is told, so that a graph that kept it for a backward pass notices."""
        if written is not None and rc in (0, -2):        # (-2: some of the launches may have been made)
            self._torch.autograd.graph.increment_version(written)
        if rc != 0:
            raise RuntimeError("mlease_hip error %d: %s" % (rc, self.L.mlx_last_error(None).decode()))

    # -- lookup -----------------------------------------------------------------------------------
    def embedding_lookup(self, table, ids, scale: float = 1.0, out=None):
        """out[t] = scale * table[ids[t]]; ids outside the table (-1) give rows of zeros. table [rows, width], ids [n] int32 / int64."""
        tp, ld = self._matrix(table, "table")
        ip, it = self._ids(ids, "ids")
        rows, width = table.shape
        n = ids.shape[0]
        given = out
        out, op, ldo = self._output(out, (n, width), table.dtype)
        self._ck(self.L.mlx_embedding_lookup(self.device, self._stream(), self._types[table.dtype], tp, rows, width, ld, it, ip, n, scale, op, ldo), given)
        return out

    def embedding_gradient(self, grad_out, ids, n_rows: int, scale: float = 1.0, out=None, accumulate: bool = False, dtype=None):
        """grad[v] = scale * (sum of the rows of grad_out whose id is v), [n_rows, width], in grad_out's type or float32 (dtype, or out's).
        accumulate: added to `out`, whose other rows are not touched. The same inputs give the same bits."""
        gp, ldg = self._matrix(grad_out, "grad_out")
        n, width = grad_out.shape
        ip, it = self._ids(ids, "ids", n)
        if accumulate and out is None:
            raise ValueError("accumulate needs out, the gradient to add to")
        dtype = dtype or (grad_out.dtype if out is None else out.dtype)
        if dtype not in self._types:
            raise ValueError("grad must be of grad_out's type or float32, not %s" % dtype)
        given = out
        out, op, ldo = self._output(out, (n_rows, width), dtype)
        keep, wp, wb = self._workspace(self.L.mlx_embedding_gradient_workspace, n_rows, width, n)
        self._ck(self.L.mlx_embedding_gradient(self.device, self._stream(), self._types[grad_out.dtype], gp, ldg, it, ip, n, scale, bool(accumulate),
                                               self._types[dtype], op, n_rows, width, ldo, wp, wb), given)
        return out

    # -- log-likelihood ---------------------------------------------------------------------------
    def token_loglik(self, logits, target):
        """logp[t] = logits[t, target[t]] - log sum exp logits[t] (float32), and stats [n, 2] for token_loglik_gradient. A target outside
        the classes (-1) is absent: logp 0, and its row is not read."""
        lp, ld = self._matrix(logits, "logits")
        n, classes = logits.shape
        ip, it = self._ids(target, "target", n)
        logp, stats = self._torch.empty(n, dtype=self._f32, device=self._at), self._torch.empty((n, 2), dtype=self._f32, device=self._at)
        keep, wp, wb = self._workspace(self.L.mlx_token_loglik_workspace, n, classes)
        self._ck(self.L.mlx_token_loglik(self.device, self._stream(), self._types[logits.dtype], lp, n, classes, ld, it, ip, logp.data_ptr(), stats.data_ptr(), wp, wb))
        return logp, stats

    def token_loglik_gradient(self, logits, target, stats, grad_logp, out=None):
        """dlogits[t, j] = grad_logp[t] * ([j == target[t]] - softmax(logits[t])[j]) in logits' type; out may be logits itself."""
        lp, ld = self._matrix(logits, "logits")
        n, classes = logits.shape
        ip, it = self._ids(target, "target", n)
        gp = self._vector(grad_logp, "grad_logp", n, self._f32)
        if tuple(stats.shape) != (n, 2) or not stats.is_contiguous():
            raise ValueError("stats must be what token_loglik gave for these logits, [%d, 2]" % n)
        sp = self._vector(stats.view(-1), "stats", 2 * n, self._f32)
        given = out
        out, op, ldo = self._output(out, (n, classes), logits.dtype)
        self._ck(self.L.mlx_token_loglik_gradient(self.device, self._stream(), self._types[logits.dtype], lp, n, classes, ld, it, ip, sp, gp, op, ldo), given)
        return out

    # -- preference -------------------------------------------------------------------------------
    def preference_loss(self, logp, ref_logp, seq_ptr, beta: float = 0.1, smoothing: float = 0.0, scale: float = 1.0, mask=None, weight=None, offset=None,
                        mean: bool = False, grad: bool = True):
        """Loss and gradient of pairs of packed sequences: sequence s holds the tokens seq_ptr[s] .. seq_ptr[s + 1] (ascending: where they descend grad is
        unspecified), the first half of the sequences are the preferred ones. beta, smoothing and scale are taken as 32-bit numbers. logp, ref_logp (or None) [n] float32, seq_ptr [2 pairs + 1] int64, mask (or None) [n] bool / uint8, weight, offset
        (or None) [pairs] float32. Returns loss = sum of scale * weight * pair_loss, pair_loss, margin [pairs], ratio [2 pairs] and grad [n]
        (None where grad=False)."""
        torch, f32 = self._torch, self._f32
        if seq_ptr.dim() != 1 or seq_ptr.shape[0] % 2 != 1:
            raise ValueError("seq_ptr must be a vector of 2 * pairs + 1 int64, not %s" % (tuple(seq_ptr.shape),))
        n, pairs = logp.numel(), (seq_ptr.shape[0] - 1) // 2
        lp, qp = self._vector(logp, "logp", n, f32), self._vector(seq_ptr, "seq_ptr", 2 * pairs + 1, torch.int64)
        rp = None if ref_logp is None else self._vector(ref_logp, "ref_logp", n, f32)
        mp = None if mask is None else self._vector(mask, "mask", n, torch.uint8 if mask.dtype == torch.uint8 else torch.bool)
        wp = None if weight is None else self._vector(weight, "weight", pairs, f32)
        fp = None if offset is None else self._vector(offset, "offset", pairs, f32)
        # The pairs' values in one block (tensors of their own, not views: each can be written and kept without the others), the loss and the gradient in
        # theirs, since programs keep them. The workspace is enough for any number of tokens, as the header says: no need to ask.
        empty, at, kb = torch.empty, self._at, 16384 + 8 * pairs
        ratio, pair_loss, margin = torch.unsafe_split_with_sizes(empty(4 * pairs, dtype=f32, device=at), (2 * pairs, pairs, pairs))
        loss, keep = logp.new_empty(()), empty(kb, dtype=torch.uint8, device=at)
        g = empty(n, dtype=f32, device=at) if grad else None
        p = ratio.data_ptr()
        self._ck(self.L.mlx_preference_loss(self.device, self._stream(), lp, rp, n, qp, pairs, beta, smoothing, scale, bool(mean), mp, wp, fp, loss.data_ptr(),
                                            p + 8 * pairs, p + 12 * pairs, p, None if g is None else g.data_ptr(), keep.data_ptr(), kb))
        return PreferenceResult(loss, pair_loss, margin, ratio, g)
