"""Learned query adapters: retrieval that learns from feedback while the stored rows stay as they are.

Every tenant -- a (workspace, knowledge base) pair, the WHERE of ``PGVector.query`` (``pgvector.py:577-580``) -- may have
a low-rank adapter that moves its query embeddings, beside one projection all tenants share.  No reference counterpart:
the reference sends every embedding to the search as the embedding service returns it.

* ``QueryAdapters``    -- the weights; ``apply`` (one call for the waiting requests of all tenants), ``backward``, and
                          ``feedback_gradients``, which runs a whole training step's gradients
* ``preference_loss``  -- loss and gradient of pairs (preferred row, rejected row); ``HvsIndex.preference_loss`` reads
                          the rows of a table in place
* ``clip_grad_norm``   -- the global norm over many gradients, and the clipped gradients

Data are torch tensors on one GPU, of which ``data_ptr()`` is used; the work is queued on torch's current stream of that
GPU and the calls return without waiting.  Scratch memory comes from torch's allocator, call by call, so calls on several
streams do not meet in it and a call captured into a HIP graph owns what it uses.  No autograd graph is recorded: gradients
are what ``backward`` and ``preference_loss`` return.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import _lib
from ._lib import DTYPE_CODE, HvsAdaptersStruct, HvsPreferenceStruct, HvsTensorStruct, check, load_library

_CODE_OF = {torch.float32: _lib.HVS_F32, torch.float16: _lib.HVS_F16, torch.bfloat16: _lib.HVS_BF16}


def _dtype_code(t) -> int:
    code = _CODE_OF.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported tensor dtype {t.dtype}")
    return code


def _need_tensor(name: str, t, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name} must live on {'a GPU' if device is None else device}, not on {t.device}")


def _rows(name: str, t, width: int, dtype, device, n: Optional[int] = None):
    """A [n, width] tensor whose rows are contiguous and do not overlap -> (tensor, row pitch in elements)."""
    if (type(t) is torch.Tensor and t.dtype is dtype and t.dim() == 2 and t.is_contiguous() and t.device == device and t.shape[1] == width
            and (n is None or t.shape[0] == n)):
        return t, width
    _need_tensor(name, t, device)
    if t.dim() != 2 or t.shape[1] != width or (n is not None and t.shape[0] != n):
        raise ValueError(f"{name} must be [{'n' if n is None else n}, {width}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape[0] <= 1:
        return (t if t.stride(1) == 1 or width == 1 else t.contiguous()), width
    if (t.stride(1) != 1 and width > 1) or t.stride(0) < width:
        t = t.contiguous()
    return t, t.stride(0)


def _out_rows(name: str, t, n: int, width: int, dtype, device):
    """The same for a tensor that is written: it is taken as it is or refused."""
    _need_tensor(name, t, device)
    if tuple(t.shape) != (n, width) or t.dtype != dtype:
        raise ValueError(f"{name} must be [{n}, {width}] of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    if n and ((width > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < width)):
        raise ValueError(f"the rows of {name} must be contiguous and apart")
    return t, (t.stride(0) if n > 1 else width)


def _numbers(name: str, values, n: Optional[int], dtype, device):
    """Whole numbers, one per row or pair, on the GPU."""
    if (type(values) is torch.Tensor and values.dtype is dtype and values.dim() == 1 and values.is_contiguous() and values.device == device
            and (n is None or values.shape[0] == n)):
        return values
    if not isinstance(values, torch.Tensor):
        values = np.ascontiguousarray(values)
        values = torch.as_tensor(values if values.size else values.astype(np.int64), device=device)  # (an empty list has no type)
    _need_tensor(name, values, device)
    if values.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be whole numbers (int32 or int64), got {values.dtype}")
    if values.dim() != 1 or (n is not None and len(values) != n):
        raise ValueError(f"{name} must hold {'one dimension' if n is None else n} entries, got {tuple(values.shape)}")
    if values.dtype != dtype:
        if dtype == torch.int32:  # what does not fit stays what it is: negative, or past the last adapter
            values = values.clamp(-1, 0x7FFFFFFF)
        values = values.to(dtype)
    return values.contiguous()


def _scratch(nbytes: int, device):
    """Scratch memory and its address; None where none is needed."""
    if not nbytes:
        return None, None
    t = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return t, t.data_ptr()


def _stream(device) -> int:
    """torch's current stream of a GPU (the raw handle: building a Stream object costs more than a small launch)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


@functools.lru_cache(maxsize=4096)
def _adapters_workspace(code: int, d_in: int, d_out: int, rank: int, n_adapters: int, n: int, max_ld: int, backward: int) -> int:
    need = ctypes.c_uint64(0)
    st = HvsAdaptersStruct(None, None, None, None, code, d_in, d_out, rank, n_adapters)
    check(load_library().hvs_adapters_workspace(ctypes.byref(st), n, max_ld, backward, ctypes.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _preference_workspace(nq: int, pairs: int, dim: int) -> int:
    need = ctypes.c_uint64(0)
    st = HvsPreferenceStruct(n_queries=nq, n_pairs=pairs, query_dtype=_lib.HVS_F32, beta=1.0, label_smoothing=0.0)
    check(load_library().hvs_preference_workspace(ctypes.byref(st), dim, ctypes.byref(need)))
    return need.value


class FeedbackGradients(NamedTuple):
    """What ``QueryAdapters.feedback_gradients`` returns: device tensors."""

    loss: object     # [pairs]
    margin: object   # [pairs]
    grad_a: object   # [adapters, rank, d_in], clipped
    grad_b: object   # [adapters, d_out, rank], clipped
    norm: object     # [] global norm before clipping


class QueryAdapters:
    """``y = W x + scale[c] * B[c] (A[c] x)`` for a row ``x`` with adapter code ``c``; ``W x`` alone for ``c < 0``.

    ``projection`` [d_out, d_in], ``a`` [adapters, rank, d_in], ``b`` [adapters, d_out, rank]: contiguous tensors of one
    dtype (float32, float16 or bfloat16) on one GPU; ``scale`` [adapters] float32.  The object keeps the tensors it is
    given: a training loop that changes them in place changes the adapters, and another tensor like the old one may take its
    place.  For float16 and bfloat16, sums are held in fp32
    and every output is rounded once; ``A[c] x`` is kept in fp32 on its way into ``B[c]``.  An infinite element of a row stays
    with that row, a weight that is not finite with its tenant's rows (an infinite ``B`` of a 16-bit type may give NaN where
    the formula gives an infinity: it meets ``A[c] x`` in two parts).
    """

    def __init__(self, projection, a, b, scale):
        _need_tensor("projection", projection)
        device = projection.device
        for name, t, dim in (("projection", projection, 2), ("a", a, 3), ("b", b, 3), ("scale", scale, 1)):
            _need_tensor(name, t, device)
            if t.dim() != dim or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous with {dim} dimensions")
            if t.dtype != (torch.float32 if name == "scale" else projection.dtype):
                raise ValueError(f"{name} must be {torch.float32 if name == 'scale' else projection.dtype}, got {t.dtype}")
        self._code = _dtype_code(projection)
        self.d_out, self.d_in = projection.shape
        self.n_adapters, self.rank = a.shape[0], a.shape[1]
        if a.shape[2] != self.d_in:
            raise ValueError(f"a must be [adapters, rank, {self.d_in}], got {tuple(a.shape)}")
        if tuple(b.shape) != (self.n_adapters, self.d_out, self.rank):
            raise ValueError(f"b must be [{self.n_adapters}, {self.d_out}, {self.rank}], got {tuple(b.shape)}")
        if len(scale) != self.n_adapters:
            raise ValueError(f"scale must hold {self.n_adapters} entries, got {len(scale)}")
        for what, v, most in (("d_in", self.d_in, _lib.HVS_MAX_ADAPTER_DIM), ("d_out", self.d_out, _lib.HVS_MAX_ADAPTER_DIM),
                              ("rank", self.rank, _lib.HVS_MAX_ADAPTER_RANK), ("adapters", self.n_adapters, _lib.HVS_MAX_ADAPTERS)):
            if not 1 <= v <= most:
                raise ValueError(f"{what} must be in [1, {most}], got {v}")
        self.device, self.dtype = device, projection.dtype
        self._lib = load_library()
        self._like = dict(projection=projection.shape, a=a.shape, b=b.shape, scale=scale.shape)
        self.projection, self.a, self.b, self.scale = projection, a, b, scale
        self._hold()

    @classmethod
    def create(cls, dim: int, n_adapters: int, rank: int = 16, dtype: str = "f32", device: int = 0, scale: float = 1.0, seed: int = 0) -> "QueryAdapters":
        """Adapters that change nothing yet: ``W`` the identity, ``B`` zero, ``A`` random (normal, 1 / sqrt(dim)), so that the
        first gradient reaches ``B``."""
        if dtype not in DTYPE_CODE:
            raise ValueError(f"dtype must be one of {sorted(DTYPE_CODE)}, got {dtype!r}")
        t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        dev = torch.device("cuda", int(device))
        gen = torch.Generator().manual_seed(int(seed))
        a = (torch.randn(n_adapters, rank, dim, generator=gen) / math.sqrt(dim)).to(dev, t)
        return cls(torch.eye(dim, dtype=t, device=dev), a, torch.zeros(n_adapters, dim, rank, dtype=t, device=dev),
                   torch.full((n_adapters,), float(scale), dtype=torch.float32, device=dev))

    def __setattr__(self, name, value):
        """Another weight takes the place of the old one if it is like it."""
        if name in self.__dict__.get("_like", ()):
            self._check_weight(name, value)
        super().__setattr__(name, value)

    def _check_weight(self, name: str, t) -> None:
        dtype = torch.float32 if name == "scale" else self.dtype
        _need_tensor(name, t, self.device)
        if t.shape != self._like[name] or t.dtype != dtype or not t.is_contiguous():
            raise ValueError(f"{name} must stay a contiguous {tuple(self._like[name])} tensor of {dtype}, got {tuple(t.shape)} of {t.dtype}; "
                             "make another QueryAdapters for other weights")

    def _hold(self) -> None:
        """Checks the weights and holds on to their memory, so that what the kernels read is there whatever becomes of the tensors."""
        weights = self.projection, self.a, self.b, self.scale
        for name, t in zip(self._like, weights):
            self._check_weight(name, t)
        where = tuple(t.data_ptr() for t in weights)
        self._held = where, HvsAdaptersStruct(*where, self._code, self.d_in, self.d_out, self.rank, self.n_adapters), [t.detach() for t in weights]

    def _struct(self, scale=None) -> HvsAdaptersStruct:
        """The weights as the library takes them."""
        if (self.projection.data_ptr(), self.a.data_ptr(), self.b.data_ptr(), self.scale.data_ptr()) != self._held[0]:
            self._hold()  # other memory: a weight was replaced (``ad.a = ...``, ``ad.a.data = ...``)
        where, struct, _ = self._held
        if scale is None:
            return struct
        return HvsAdaptersStruct(*where[:3], scale.data_ptr(), self._code, self.d_in, self.d_out, self.rank, self.n_adapters)

    def _workspace(self, n: int, max_ld: int, backward: int):
        size = _adapters_workspace(self._code, self.d_in, self.d_out, self.rank, self.n_adapters, n, max_ld, backward)
        ws, ptr = _scratch(size, self.device)
        return ws, ptr, size

    def apply(self, x, codes, out=None, return_hidden: bool = False):
        """``x`` [n, d_in] and one adapter code per row -> [n, d_out]; every row may use another adapter.

        A torch tensor of the adapters' dtype gives a torch tensor (``out``, when given); with ``return_hidden`` also the
        float32 [n, rank] values ``A[c] x`` that ``backward`` takes.  A numpy array (float32, from an embedding service)
        gives a float32 numpy array, rounded to the adapters' dtype on its way in.  A code past the last adapter makes its row NaN.  ``out`` must not overlap ``x``
        (columns of one wide tensor do not) or the weights."""
        if not isinstance(x, torch.Tensor):
            if out is not None or return_hidden:
                raise ValueError("out and return_hidden need device tensors")
            x = np.ascontiguousarray(x, dtype=np.float32)
            y = self.apply(torch.from_numpy(x).to(self.device, self.dtype), codes)
            return y.to(torch.float32).cpu().numpy()
        x, ld_x = _rows("x", x, self.d_in, self.dtype, self.device)
        n = x.shape[0]
        codes = _numbers("codes", codes, n, torch.int32, self.device)
        if out is None:
            out, ld_out = x.new_empty(n, self.d_out), self.d_out
        else:
            out, ld_out = _out_rows("out", out, n, self.d_out, self.dtype, self.device)
        hidden = torch.empty((n, self.rank), dtype=torch.float32, device=self.device) if return_hidden else None
        if n:
            ws, ws_ptr, size = self._workspace(n, max(ld_x, ld_out), 0)
            check(self._lib.hvs_adapters_apply(self.device.index, _stream(self.device), ctypes.byref(self._struct()), x.data_ptr(), ld_x, codes.data_ptr(), n,
                                               out.data_ptr(), ld_out, hidden.data_ptr() if return_hidden else None, ws_ptr, size))
        return (out, hidden) if return_hidden else out

    def backward(self, grad, x, codes, hidden, input_grad: bool = True):
        """Gradients of ``apply`` for ``grad`` [n, d_out], the gradient of its output; ``hidden`` is what ``apply`` returned.

        -> ``(grad_x, grad_a, grad_b)``: grad_x [n, d_in] in the adapters' dtype (None without ``input_grad``), grad_a and
        grad_b float32 in the shapes of ``a`` and ``b``, zero for adapters no row uses.  The projection is frozen.  The same
        call gives the same bits."""
        return self._backward(grad, x, codes, hidden, input_grad, None)

    def _backward(self, grad, x, codes, hidden, input_grad, scale):
        """``backward`` with another ``scale`` in place of the adapters' (None: theirs)."""
        x, ld_x = _rows("x", x, self.d_in, self.dtype, self.device)
        n = x.shape[0]
        grad, ld_grad = _rows("grad", grad, self.d_out, self.dtype, self.device, n)
        codes = _numbers("codes", codes, n, torch.int32, self.device)
        hidden, _ = _rows("hidden", hidden, self.rank, torch.float32, self.device, n)
        hidden = hidden.contiguous()
        grad_x = x.new_empty(n, self.d_in) if input_grad else None
        grad_a = torch.empty(self.a.shape, dtype=torch.float32, device=self.device)
        grad_b = torch.empty(self.b.shape, dtype=torch.float32, device=self.device)
        ws, ws_ptr, size = self._workspace(n, max(ld_x, ld_grad), 1)
        check(self._lib.hvs_adapters_backward(self.device.index, _stream(self.device), ctypes.byref(self._struct(scale)), grad.data_ptr(), ld_grad,
                                              x.data_ptr(), ld_x, codes.data_ptr(), hidden.data_ptr(), n, grad_x.data_ptr() if input_grad and n else None, self.d_in,
                                              grad_a.data_ptr(), grad_b.data_ptr(), ws_ptr, size))
        return grad_x, grad_a, grad_b

    def feedback_gradients(self, table, x, codes, chosen, rejected, offsets, beta: float = 20.0, label_smoothing: float = 0.0,
                           weights=None, max_norm: float = math.inf) -> FeedbackGradients:
        """The gradients of one training step on rated answers: adapt the queries ``x``, take the preference loss of their
        pairs of rows of ``table`` (an ``HvsIndex``, or a tensor of rows) against the unadapted projection ``W x`` as the
        reference policy, go back to the adapters and clip.  Apply them with any optimizer, in place.

        For float16 adapters the loss's gradient is taken in float32 and goes back multiplied by a power of two that puts its
        largest element below 2^14, which ``scale`` takes out again: the mean over many pairs has elements far below what
        float16 holds."""
        y, hidden = self.apply(x, codes, return_hidden=True)
        reference = self.apply(x, torch.full((len(y),), -1, dtype=torch.int32, device=self.device))
        half = self.dtype is torch.float16
        if half:
            y, reference = y.float(), reference.float()
        args = dict(reference=reference, beta=beta, label_smoothing=label_smoothing, weights=weights)
        if isinstance(table, torch.Tensor):
            loss, margin, grad = preference_loss(y, table, chosen, rejected, offsets, **args)
        else:
            loss, margin, grad = table.preference_loss(y, chosen, rejected, offsets, **args)
        scale = None
        if half:
            # (of the finite ones: a query with a code past the last adapter has none, and adds nothing; max_norm inf scales nothing)
            largest = clip_grad_norm([grad.nan_to_num(0.0, 0.0, 0.0)], math.inf, norm_type=math.inf).clamp_(min=2.0**-100)
            unit = (largest / torch.frexp(largest).mantissa).mul_(2.0**-14)  # exact: the power of two above it, over 2^14
            grad = torch.div(grad, unit, out=torch.empty(grad.shape, dtype=torch.float16, device=self.device))
            scale = self.scale * unit
        _, grad_a, grad_b = self._backward(grad, x, codes, hidden, False, scale)
        norm = clip_grad_norm([grad_a, grad_b], max_norm)
        return FeedbackGradients(loss, margin, grad_a, grad_b, norm)


def _preference(queries, dim, chosen, rejected, offsets, reference, beta, label_smoothing, weights, launch):
    """The part ``preference_loss`` and ``HvsIndex.preference_loss`` share; ``launch(struct, stream, workspace, size)``."""
    _need_tensor("queries", queries)
    device = queries.device
    code = _dtype_code(queries)
    queries, ld = _rows("queries", queries, dim, queries.dtype, device)
    nq = queries.shape[0]
    offsets = _numbers("offsets", offsets, nq + 1, torch.int64, device)
    chosen = _numbers("chosen", chosen, None, torch.int64, device)
    pairs = len(chosen)
    rejected = _numbers("rejected", rejected, pairs, torch.int64, device)
    ld_ref = 0
    if reference is not None:
        reference, ld_ref = _rows("reference", reference, dim, queries.dtype, device, nq)
    if weights is not None:
        _need_tensor("weights", weights, device)
        if weights.dtype != torch.float32 or tuple(weights.shape) != (pairs,):
            raise ValueError(f"weights must hold {pairs} float32 entries")
        weights = weights.contiguous()
    loss = torch.empty(pairs, dtype=torch.float32, device=device)
    margin = torch.empty(pairs, dtype=torch.float32, device=device)
    grad = queries.new_empty(nq, dim)
    st = HvsPreferenceStruct(queries.data_ptr(), ld, None if reference is None else reference.data_ptr(), ld_ref, offsets.data_ptr(), chosen.data_ptr(),
                             rejected.data_ptr(), None if weights is None else weights.data_ptr(), loss.data_ptr(), margin.data_ptr(),
                             grad.data_ptr(), dim, nq, pairs, code, float(beta), float(label_smoothing))
    size = _preference_workspace(nq, pairs, dim)
    ws, ws_ptr = _scratch(size, device)
    check(launch(ctypes.byref(st), _stream(device), ws_ptr, size))
    return loss, margin, grad


def preference_loss(queries, rows, chosen, rejected, offsets, reference=None, beta: float = 20.0, label_smoothing: float = 0.0, weights=None):
    """Preference loss of pairs of rows and its gradient for the queries, in one pass over the rows.

    ``queries`` [nq, dim]; ``rows`` [n, dim]; pairs ``offsets[i] .. offsets[i + 1]`` (``offsets`` [nq + 1], ascending)
    belong to query i, and pairs outside all of them are left out; ``chosen`` / ``rejected`` are row positions.  With a
    policy that picks rows by softmax(beta cos(query, row)),
    ``margin = (cos(q, chosen) - cos(q, rejected)) - (cos(q0, chosen) - cos(q0, rejected))`` for the reference policy's
    queries q0 (``reference`` [nq, dim]; None: without that term) is the paired log ratio over beta, and
    ``loss = -(1 - s) log sigmoid(beta margin) - s log sigmoid(-beta margin)`` with ``s = label_smoothing`` in [0, 0.5].

    -> ``(loss [pairs], margin [pairs], grad [nq, dim])``: grad, in the queries' dtype, is the gradient of
    ``sum(weights * loss)``; without ``weights`` of the mean (whose elements fall below what float16 holds as pairs grow: take
    float32 queries, or larger weights).  A pair with a negative position is left out (loss and margin
    0); one with a position past the last row is NaN and makes its query's gradient NaN."""
    _need_tensor("queries", queries)
    _need_tensor("rows", rows, queries.device)
    if rows.dim() != 2:
        raise ValueError(f"rows must be [n, dim], got {tuple(rows.shape)}")
    code = _dtype_code(rows)
    rows, ld = _rows("rows", rows, rows.shape[1], rows.dtype, rows.device)
    return _preference(queries, rows.shape[1], chosen, rejected, offsets, reference, beta, label_smoothing, weights,
                       lambda st, stream, ws, size: load_library().hvs_preference_loss(rows.device.index, stream, st, rows.data_ptr(), code, rows.shape[1],
                                                                                       ld, rows.shape[0], ws, size))


def clip_grad_norm(grads: Sequence, max_norm: float, norm_type: float = 2.0, out: Optional[Sequence] = None):
    """Scale all of ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` and return ``norm``, a float32 device scalar.

    ``norm`` is the 2-norm over every element of every tensor (``norm_type`` 2; squares summed in double precision), or the
    largest absolute value (``math.inf``).  The tensors are contiguous, of float32, float16 or bfloat16 in any mix, on one
    GPU, at least one; they are scaled in place, or into ``out`` (tensors of the same shapes and dtypes).  ``max_norm`` inf
    scales nothing.  A NaN anywhere makes the norm and every element NaN."""
    grads = list(grads)
    if not grads:
        raise ValueError("clip_grad_norm needs at least one tensor")
    if norm_type not in (2, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type!r}")
    outs = grads if out is None else list(out)
    if len(outs) != len(grads):
        raise ValueError(f"out holds {len(outs)} tensors for {len(grads)}")
    _need_tensor("grads[0]", grads[0])
    device = grads[0].device
    entries = []
    for i, (g, o) in enumerate(zip(grads, outs)):
        if not isinstance(g, torch.Tensor) or g.device != device:
            _need_tensor(f"grads[{i}]", g, device)
        if not g.is_contiguous():
            raise ValueError(f"grads[{i}] must be contiguous")
        if o is not g:
            if not isinstance(o, torch.Tensor) or o.device != device:
                _need_tensor(f"out[{i}]", o, device)
            if o.shape != g.shape or o.dtype != g.dtype or not o.is_contiguous():
                raise ValueError(f"out[{i}] must be contiguous, {tuple(g.shape)} of {g.dtype}")
        entries.append((g.data_ptr(), o.data_ptr(), g.numel(), _dtype_code(g)))
    table = (HvsTensorStruct * len(entries))(*entries)
    lib = load_library()
    norm = torch.empty((), dtype=torch.float32, device=device)
    need = ctypes.c_uint64(0)
    check(lib.hvs_clip_workspace(table, len(grads), ctypes.byref(need)))
    ws, ws_ptr = _scratch(need.value, device)
    check(lib.hvs_clip_grad_norm(device.index, _stream(device), table, len(grads), float(max_norm), int(norm_type == math.inf), norm.data_ptr(), ws_ptr,
                                 need.value))
    return norm


__all__ = ["QueryAdapters", "FeedbackGradients", "preference_loss", "clip_grad_norm"]
