"""Smooth losses whose scores come in rows, one softmax per row: terms for classifiers, re-rankers and routers.

They stand beside ``LogisticLoss`` and ``SquaredDistance`` (one score per sample) and honour the same surface,
``value_and_gradient(u, out=None) -> (f(u), grad)``, so ``Composed(loss, A)``, ``SlicedSeparableSum`` and every iteration of the
package take them: ``u`` is then a :class:`HIPVector` holding the rows one after another.  They also take the scores as a 2-D torch
tensor on the device (Float32, Float64, bfloat16 or Float16; rows any distance apart), as a training program has them, and
``value_and_gradient_async`` leaves the value on the device, so that nothing waits.

A loss runs on its context's stream.  Called under another current torch stream, it waits for that stream's work and that
stream waits for the loss.  One host thread per context at a time; a graph is recorded with ``Context.capture_begin`` (with ``out``
and ``value`` given: nothing can be allocated while recording) and works on the loss's own buffers: keep the loss as long as the graph."""
import ctypes as C

import numpy as np

from . import _lib
from ._lib import PG_BF16, PG_F16, PG_F32, PG_F64, ProxGradError
from .device import HIPVector, get_context


_torch_module = None
_DTYPES = {}


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch

        _DTYPES.update({torch.float32: PG_F32, torch.float64: PG_F64, torch.bfloat16: PG_BF16, torch.float16: PG_F16})
        _torch_module = torch
    return _torch_module


def _dtype_code(dt):
    _torch()
    return _DTYPES.get(dt)


def _as_tensor(x, name):
    """x as a torch tensor, wherever it lives"""
    torch = _torch()
    if isinstance(x, HIPVector):
        return x.torch()
    if isinstance(x, torch.Tensor):
        return x
    return torch.from_numpy(np.ascontiguousarray(x))


def _rows_of(x, name, shape, kinds, convert):
    """x checked against ``shape`` and brought to one of ``kinds`` (else to ``convert``), last axis dense"""
    t = _as_tensor(x, name)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype not in kinds:
        if t.is_floating_point() != convert.is_floating_point or t.is_complex():
            raise TypeError(f"{name} has element type {t.dtype}")
        t = t.to(convert)
    if t.dim() and t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _common_device(tensors, ctx):
    """the context: given, or that of the device the tensors live on"""
    devices = {t.device.index for t in tensors if t is not None and t.is_cuda}
    if len(devices) > 1:
        raise ValueError("the loss's tensors live on different devices")
    if ctx is None:
        ctx = get_context(devices.pop() if devices else None)
    elif devices and devices != {ctx.device}:
        raise ValueError("the loss's tensors live on another device than its context")
    return ctx


def _raw_stream(device):
    """the current torch stream's handle (every call looks: torch's own accessor makes a Stream object each time)"""
    torch = _torch()
    fast = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return fast(device) if fast is not None else torch.cuda.current_stream(device).cuda_stream


def _stream_of(ctx):
    torch = _torch()
    return torch.cuda.ExternalStream(ctx.stream, device=ctx.torch_device) if ctx.stream else torch.cuda.default_stream(ctx.torch_device)


def _settle(ctx, tensors):
    """a new loss's tensors: what the current stream still does to them comes before the context's later work, and their memory
    is not handed out again while the context uses it"""
    with _Ordered(ctx):
        pass
    if _raw_stream(ctx.device) != ctx.stream:
        for v in tensors:
            if v is not None and v.numel():
                v.record_stream(_stream_of(ctx))


class _Ordered:
    """the call's kernels run on the context's stream: between the current torch stream's past and its future"""

    __slots__ = ("ctx", "cur", "ext")

    def __init__(self, ctx):
        self.ctx = ctx

    def __enter__(self):
        torch = _torch()
        ctx = self.ctx
        self.cur = None
        if ctx.capturing:
            return
        if _raw_stream(ctx.device) != ctx.stream:
            cur = torch.cuda.current_stream(ctx.torch_device)
            with torch.cuda.device(ctx.device):
                if torch.cuda.is_current_stream_capturing():
                    raise ProxGradError("a torch graph is being recorded: record with Context.capture_begin instead",
                                        code=_lib.PG_ERR_UNSUPPORTED)
                self.cur, self.ext = cur, _stream_of(ctx)
                self.ext.wait_stream(cur)

    def __exit__(self, *exc):
        if self.cur is not None:
            with _torch().cuda.device(self.ctx.device):
                self.cur.wait_stream(self.ext)


class _RowLoss:
    """Checks of the scores and of ``out``, shared by the row losses; a subclass has ``rows``, ``classes``, ``ctx``, ``_evaluate``."""

    is_generalized_quadratic = False

    def _open(self, ctx, *tensors):
        self.ctx = _common_device(tensors, ctx)
        if self.ctx.capturing:
            raise ProxGradError("device allocation during stream capture: make the loss before")
        return self.ctx.torch_device

    def _locate(self, u, name):
        """(pointer, row distance, dtype code) of scores or gradients"""
        n, v = self.rows, self.classes
        if isinstance(u, HIPVector):
            if u.n != n * v:
                raise ValueError(f"{name} must hold {n} x {v} scores, got {u.n}")
            if u.ctx.device != self.ctx.device:
                raise ValueError(f"{name} lives on another device than the loss")
            if u.ctx.stream != self.ctx.stream:
                raise ValueError(f"{name} belongs to a context on another stream than the loss's")
            return u.ptr, max(v, 1), u.pg_dtype
        code = _dtype_code(getattr(u, "dtype", None))
        if code is None:
            raise TypeError(f"{name} must be a HIPVector or a Float32, Float64, bfloat16 or Float16 torch tensor")
        if u.get_device() != self.ctx.device:  # -1 on the host
            raise ValueError(f"{name} must live on the loss's device {self.ctx.device}")
        shape = u.shape
        if len(shape) == 2 and shape[0] == n and shape[1] == v:
            ld, step = u.stride()
            if v > 1 and step != 1:
                raise ValueError(f"the scores of a row of {name} must be adjacent (stride 1)")
            if n <= 1:
                ld = max(v, 1)
            elif ld < v:
                raise ValueError(f"the rows of {name} overlap")
            return u.data_ptr(), ld, code
        if len(shape) == 1 and shape[0] == n * v and (n * v == 0 or u.stride(0) == 1):
            return u.data_ptr(), max(v, 1), code
        raise ValueError(f"{name} must have shape ({n}, {v}), got {tuple(shape)}")

    def _like(self, u):
        if isinstance(u, HIPVector):
            return u.similar()
        if self.ctx.capturing:
            raise ProxGradError("device allocation during stream capture: give out and value")
        return _torch().empty(u.shape, dtype=u.dtype, device=u.device)

    def _place(self, u, out):
        """arguments of the entry point for scores ``u`` and gradient ``out`` (made if None)"""
        up, uld, code = self._locate(u, "u")
        if out is None:
            out = self._like(u)
        op, old, ocode = self._locate(out, "out")
        if ocode != code:
            raise TypeError("out must have the scores' element type")
        if self.rows and self.classes and not (op == up and (old == uld or self.rows == 1)):
            size = 8 if code == PG_F64 else (4 if code == PG_F32 else 2)
            reach = ((self.rows - 1) * uld + self.classes) * size, ((self.rows - 1) * old + self.classes) * size
            if op < up + reach[0] and up < op + reach[1]:
                gap = ((op - up) % (uld * size)) if uld == old else 0  # side by side in one buffer is fine
                if not (uld == old and self.classes * size <= gap <= (uld - self.classes) * size):
                    raise ValueError("out overlaps u: it may be u itself or apart from it")
        return out, (up, uld, op, old, code)

    def value_and_gradient(self, u, out=None):
        """(f(u), grad f(u)); waits for the value.  ``out``: where the gradient goes (may be ``u`` itself)"""
        out, where = self._place(u, out)
        f = C.c_double()
        with _Ordered(self.ctx):
            self._evaluate(where, None, C.byref(f))
        return (u.dtype.type(f.value) if isinstance(u, HIPVector) else f.value), out

    def value_and_gradient_async(self, u, out=None, value=None):
        """The same without waiting: the value is a one-element torch tensor on the device (Float32; Float64 for Float64 scores)"""
        torch = _torch()
        out, where = self._place(u, out)
        vdt = torch.float64 if where[4] == PG_F64 else torch.float32
        if value is None:
            if self.ctx.capturing:
                raise ProxGradError("device allocation during stream capture: give out and value")
            value = torch.empty((), dtype=vdt, device=self.ctx.torch_device)
        elif value.numel() != 1 or value.dtype != vdt or not value.is_cuda or value.device.index != self.ctx.device:
            raise ValueError(f"value must be a one-element {vdt} tensor on the loss's device")
        if _raw_stream(self.ctx.device) == self.ctx.stream:
            self._evaluate(where, value.data_ptr(), None)
        else:
            with _Ordered(self.ctx):
                self._evaluate(where, value.data_ptr(), None)
        return value, out

    def __call__(self, u):
        scratch = getattr(self, "_scratch", None)
        if scratch is None or type(scratch) is not type(u) or scratch.dtype != u.dtype:
            scratch = self._scratch = self._like(u)
        return self.value_and_gradient(u, out=scratch)[0]


class DistillationLoss(_RowLoss):
    """Distillation from a teacher's top logits (include/proxgrad_hip_rows.h: pg_distill_value_and_gradient).

    ``teacher_logits`` (rows x top) at classes ``teacher_index`` (rows x top; -1: no entry), temperature T, per-row ``weights``:

        f(u) = lam sum_n w_n KL(p_n || softmax(u_n / T)) + label_lam sum_n w_n (log sum exp u_n - u_n[y_n])

    p is the softmax of the listed logits / T; with ``teacher_lse`` -- log sum exp of ALL the teacher's logits / T per row -- it is the
    teacher's own probability, and the classes outside the list count as one more class (then f is not convex).  ``labels``: -1 = none.
    The usual factor T^2 is the caller's: ``lam=T**2``.  Rows of weight 0 are not read.  Tensors on the device are used where
    they are, later changes included (a copy of those whose last axis is not dense or whose type is none of Float32, Float64 --
    logits bfloat16 and Float16 too --, int32, int64); host arrays are checked and uploaded.  An index or label that is out of range on the
    device makes the value and that row's gradient NaN."""

    def __init__(self, teacher_logits, teacher_index, n_classes, *, temperature=1.0, lam=1.0, teacher_lse=None, weights=None,
                 labels=None, label_lam=0.0, ctx=None):
        torch = _torch()
        t = _as_tensor(teacher_logits, "teacher_logits")
        if t.dim() != 2:
            raise ValueError("teacher_logits must be a (rows, top) array")
        self.rows, top = int(t.shape[0]), int(t.shape[1])
        self.classes = int(n_classes)
        if not 0 <= self.classes <= 1 << 24:
            raise ValueError("n_classes must be between 0 and 2^24")
        if top > 1024:
            raise ValueError("at most 1024 listed logits per row")
        self.temperature, self.lam, self.label_lam = float(temperature), float(lam), float(label_lam)
        if not (self.temperature > 0 and np.isfinite(self.temperature)):
            raise ValueError("temperature must be positive and finite")
        if not (self.lam >= 0 and self.label_lam >= 0 and np.isfinite(self.lam) and np.isfinite(self.label_lam)):
            raise ValueError("lam and label_lam must be nonnegative and finite")
        if labels is None and self.label_lam:
            raise ValueError("label_lam without labels")
        reals, ints = (torch.float32, torch.float64), (torch.int32, torch.int64)
        t = _rows_of(t, "teacher_logits", (self.rows, top), (*reals, torch.bfloat16, torch.float16), torch.float32)
        index = _rows_of(teacher_index, "teacher_index", (self.rows, top), ints, torch.int64)
        lse = None if teacher_lse is None else _rows_of(teacher_lse, "teacher_lse", (self.rows,), reals, torch.float32)
        weights = None if weights is None else _rows_of(weights, "weights", (self.rows,), reals, torch.float32)
        labels = None if labels is None else _rows_of(labels, "labels", (self.rows,), ints, torch.int64)
        for name, v in (("teacher_index", index), ("labels", labels)):
            if v is not None and not v.is_cuda and v.numel() and not (int(v.min()) >= -1 and int(v.max()) < self.classes):
                raise ValueError(f"{name} must lie between -1 and n_classes - 1")
        if weights is not None and not weights.is_cuda and weights.numel() and not bool((weights >= 0).all()):
            raise ValueError("weights must be nonnegative")
        self.is_convex = lse is None
        dev = self._open(ctx, t, index, lse, weights, labels)
        self._keep = t, index, lse, weights, labels = [None if v is None else v.to(dev) for v in (t, index, lse, weights, labels)]
        _settle(self.ctx, self._keep)
        ptr = lambda v: None if v is None else v.data_ptr()  # noqa: E731
        bits = lambda v: 64 if v is not None and v.dtype == torch.int64 else 32  # noqa: E731
        code = lambda v: PG_F32 if v is None else _dtype_code(v.dtype)  # noqa: E731
        self._d = _lib.pg_distill(rows=self.rows, classes=self.classes, top=top, teacher=ptr(t),
                                  teacher_ld=t.stride(0) if self.rows > 1 else top, index=ptr(index),
                                  index_ld=index.stride(0) if self.rows > 1 else top, teacher_lse=ptr(lse), weights=ptr(weights),
                                  labels=ptr(labels), teacher_dtype=code(t), index_bits=bits(index), lse_dtype=code(lse),
                                  weights_dtype=code(weights), label_bits=bits(labels), temperature=self.temperature, lam=self.lam,
                                  label_lam=self.label_lam)
        self._dref = C.byref(self._d)
        self._entry = _lib.load().pg_distill_value_and_gradient

    def _evaluate(self, where, value, f_out):
        up, uld, op, old, code = where
        status = self._entry(self.ctx.handle, self._dref, code, up, uld, op, old, value, f_out)
        if status:
            _lib.check(status)


def _balance_tiles(tokens, experts, offsets, num_cu):
    """(rows of (begin, end, group, part), tokens of a tile, whether each group is one tile): an evaluation in pieces of one group each.

    Small groups take a workgroup each and one launch; 64 tokens of 64 experts take 7.4 us that way and 9.9 in tiles, 64 of 256 experts 14.0
    and 14.2.  Else a tile is four waves' work, at least a step of theirs: four tiles per compute unit (131072 x 256: 94 us; two 103,
    eight 95), no fewer than 16 tokens in one (256 x 256: 14.4 us; 32 tokens 18.7, 64 tokens 27.4)."""
    offsets = np.asarray(offsets, np.int64)
    lengths = np.diff(offsets)
    longest = int(lengths.max(initial=0))
    whole = longest * experts <= 4096
    size = max(1, longest) if whole else max(16, -(-tokens // (4 * num_cu)))
    parts = -(-lengths // size)
    group = np.repeat(np.arange(len(lengths)), parts)
    part = np.arange(len(group)) - np.repeat(np.cumsum(parts) - parts, parts)
    begin = offsets[:-1][group] + lengths[group] * part // np.maximum(parts[group], 1)
    end = offsets[:-1][group] + lengths[group] * (part + 1) // np.maximum(parts[group], 1)
    part[parts[group] == 1] = -1
    behind = np.arange(offsets[-1], tokens, max(size, 16))  # tokens behind the last group
    tiles = np.stack([np.concatenate([begin, behind]), np.concatenate([end, np.minimum(behind + max(size, 16), tokens)]),
                      np.concatenate([group, np.full(len(behind), -1)]), np.concatenate([part, np.zeros(len(behind), np.int64)])], axis=1)
    return tiles, size, whole


class BalanceLoss(_RowLoss):
    """Balance of a router's experts (include/proxgrad_hip_rows.h: pg_balance_value_and_gradient).

    The scores are a router's (tokens x n_experts), p their softmax per token; a token chooses its ``k`` highest scores (the lowest
    index first among equal ones; never -inf), or what ``chosen`` (tokens x k; -1: none) says.  Per group g of tokens -- all of them, or
    ``offsets[g] .. offsets[g + 1]``, a sequence each, empty ones allowed -- with c_e the choices of expert e and n the unmasked tokens:

        f(u) = lam sum_g n_experts / (k n_g^2) sum_e c_ge sum_t p_te

    lam per group at perfect balance.  The gradient holds the counts fixed, so f is smooth between changes of the choices only,
    and not convex.  ``mask``: False = the token counts for nothing and its gradient is zero, as behind the last group.  After an
    evaluation ``counts`` (groups x n_experts, int32, on the device) holds the c of that evaluation: one tensor, overwritten by the next."""

    is_convex = False

    def __init__(self, tokens, n_experts, k, *, offsets=None, mask=None, chosen=None, lam=1.0, ctx=None):
        torch = _torch()
        self.rows, self.classes, self.k, self.lam = int(tokens), int(n_experts), int(k), float(lam)
        if not 0 <= self.rows < 1 << 31:
            raise ValueError("tokens must be between 0 and 2^31 - 1")
        if not 1 <= self.classes <= 1024:
            raise ValueError("n_experts must be between 1 and 1024")
        if not 1 <= self.k <= self.classes:
            raise ValueError("k must be between 1 and n_experts")
        if not (self.lam >= 0 and np.isfinite(self.lam)):
            raise ValueError("lam must be nonnegative and finite")
        if offsets is None:
            offsets = [0, self.rows]
        else:
            offsets = np.asarray(offsets.cpu() if isinstance(offsets, torch.Tensor) else offsets)
            if offsets.ndim != 1 or offsets.size < 1:
                raise ValueError("offsets must be a list of at least one position")
            if offsets.dtype.kind not in "iu":
                raise TypeError("offsets must be integers")
            offsets = [int(o) for o in offsets]
            if offsets[0] != 0 or offsets[-1] > self.rows or any(a > b for a, b in zip(offsets, offsets[1:])):
                raise ValueError("offsets must start at 0, never fall, and end at most at the number of tokens")
        if mask is not None:
            mask = _as_tensor(mask, "mask")
            if tuple(mask.shape) != (self.rows,):
                raise ValueError(f"mask must have shape ({self.rows},)")
            if mask.dtype not in (torch.bool, torch.uint8):
                raise TypeError("mask must be boolean")
            mask = mask.contiguous()
        if chosen is not None:
            chosen = _rows_of(chosen, "chosen", (self.rows, self.k), (torch.int32, torch.int64), torch.int64)
            if not chosen.is_cuda and chosen.numel() and not (int(chosen.min()) >= -1 and int(chosen.max()) < self.classes):
                raise ValueError("chosen must lie between -1 and n_experts - 1")
        dev = self._open(ctx, mask, chosen)
        groups = len(offsets) - 1
        tiles, size, whole = _balance_tiles(self.rows, self.classes, offsets, self.ctx.device_info()["compute_units"])
        even = offsets == [0, self.rows]  # one group: its tiles need no list
        ntiles = -(-self.rows // size) if even else len(tiles)
        last_part = ntiles - 1 if even else int(tiles[:, 3].max(initial=0))
        packed = np.empty((len(tiles), 3), np.int64)  # pg_balance_tile: two int64, two int32
        packed[:, :2] = tiles[:, :2]
        packed[:, 2] = (tiles[:, 2] & 0xFFFFFFFF) | (tiles[:, 3] << 32)
        tiles_d = None if even else torch.from_numpy(packed).to(dev)
        mask, chosen = (None if v is None else v.to(dev) for v in (mask, chosen))
        self._counts = torch.zeros(groups, self.classes, dtype=torch.int32, device=dev)
        copies = min(16, 1 + max(last_part, 0) // 16)  # some sixteen tiles to an accumulator
        state = torch.zeros(4 + (0 if whole else 2 * groups * copies * (self.classes + 2)), dtype=torch.int32, device=dev)
        self._keep = tiles_d, mask, chosen, state
        _settle(self.ctx, (*self._keep, self._counts))
        ptr = lambda v: None if v is None else v.data_ptr()  # noqa: E731
        self._b = _lib.pg_balance(tokens=self.rows, groups=groups, ntiles=ntiles, tile_tokens=size, tiles=ptr(tiles_d), mask=ptr(mask), chosen=ptr(chosen),
                                  chosen_ld=0 if chosen is None else (chosen.stride(0) if self.rows > 1 else self.k), counts=ptr(self._counts),
                                  state=ptr(state), experts=self.classes, k=self.k,
                                  chosen_bits=64 if chosen is not None and chosen.dtype == torch.int64 else 32, whole=whole, copies=copies, lam=self.lam)
        self._bref = C.byref(self._b)
        self._entry = _lib.load().pg_balance_value_and_gradient

    @property
    def counts(self):
        return self._counts

    def _evaluate(self, where, value, f_out):
        up, uld, op, old, code = where
        status = self._entry(self.ctx.handle, self._bref, code, up, uld, op, old, value, f_out)
        if status:
            _lib.check(status)
