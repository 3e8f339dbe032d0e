"""The operators of a training step on torch tensors (include/ccsm_train_ops.h, in libccsm_train): products with bias, activation and residual,
embedding lookup, and activations kept in 8 bits, each with the gradients that a training step needs.

    y, z = linear(x, w, b, residual, activation="gelu", keep_preact=True)
    dx, dw, db = linear_backward(dy, x, w, z, activation="gelu")          # x and z may be checkpoint8(x, ...) and checkpoint8(z, ...)
    y = embedding(ids, table, scale=2.0);   dtable = embedding_backward(dy, ids, len(table), scale=2.0)
    c = checkpoint8(x, "int8");             x_hat = c.values()

What torch.nn does for the reference here: nn.Embedding (ccsmeth/models.py:35, 91), nn.Linear and the activation behind it
(ccsmeth/utils/attention.py:34-36, 69), autograd's saved tensors (ccsmeth/train_multigpu.py:283-312).

Tensors are float32, float16 or bfloat16 on one GPU, one type per call.  Work is enqueued on `stream` (a torch.cuda.Stream; default: torch's
current stream of the tensors' device) and nothing waits for the GPU; calls can be captured into a graph.  Row-strided views are taken as
they are, other layouts are copied.  There is no autograd: gradients are calls, as in Trainer.forward_backward; inputs that require a
gradient are refused while grad mode is on, and those with a forward-mode tangent.  There is no CPU path.
"""
import ctypes as C
import struct

from . import _lib
from . import train as _train

EXPORTS = ("ccsm_train_ops_last_error", "ccsm_train_linear_workspace", "ccsm_train_linear_forward", "ccsm_train_linear_backward_workspace",
           "ccsm_train_linear_backward", "ccsm_train_linear_way", "ccsm_train_linear_backward_way", "ccsm_train_embedding_forward", "ccsm_train_embedding_backward_workspace",
           "ccsm_train_embedding_backward", "ccsm_train_act8_pack", "ccsm_train_act8_unpack")
ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "sigmoid": 3, "gelu": 4, "silu": 5}
CODES = {"int8": 1, "e4m3": 2}


class Saved(C.Structure):
    _fields_ = [("data", C.c_void_p), ("ld", C.c_int64), ("code", C.c_int32), ("scales", C.c_void_p), ("lds", C.c_int64)]


class Linear(C.Structure):
    _fields_ = [("type", C.c_int32), ("activation", C.c_int32), ("rows", C.c_int64), ("inner", C.c_int32), ("outer", C.c_int32),
                ("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p), ("ldw", C.c_int64), ("bias", C.c_void_p),
                ("residual", C.c_void_p), ("ldr", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64), ("preact", C.c_void_p), ("ldp", C.c_int64)]


class LinearGrad(C.Structure):
    _fields_ = [("type", C.c_int32), ("activation", C.c_int32), ("rows", C.c_int64), ("inner", C.c_int32), ("outer", C.c_int32),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("x", Saved), ("w", C.c_void_p), ("ldw", C.c_int64), ("preact", Saved),
                ("dx", C.c_void_p), ("lddx", C.c_int64), ("dw", C.c_void_p), ("lddw", C.c_int64), ("dbias", C.c_void_p)]


# the two structures as bytes (the header's layout): one pack call is a third of what filling a ctypes structure costs per call
_LINEAR = struct.Struct("@iiqiiPqPqPPqPqPq")
_GRAD = struct.Struct("@iiqiiPqPqiPqPqPqiPqPqPqP")
_SAVED = struct.Struct("@PqiPq")
assert _LINEAR.size == C.sizeof(Linear) and _GRAD.size == C.sizeof(LinearGrad) and _SAVED.size == C.sizeof(Saved)
_NONE = (0, 0, 0, 0, 0)

_ops = None


def load():
    global _ops
    if _ops is not None:
        return _ops
    lib = _train.load()
    vp, ci, cl, cf, cs = C.c_void_p, C.c_int, C.c_int64, C.c_float, C.c_size_t
    lib.ccsm_train_ops_last_error.restype = C.c_char_p
    lib.ccsm_train_linear_workspace.argtypes = [vp]
    lib.ccsm_train_linear_workspace.restype = cs
    lib.ccsm_train_linear_forward.argtypes = [ci, vp, vp, cs, vp]
    lib.ccsm_train_linear_backward_workspace.argtypes = [vp]
    lib.ccsm_train_linear_backward_workspace.restype = cs
    lib.ccsm_train_linear_backward.argtypes = [ci, vp, vp, cs, vp]
    lib.ccsm_train_linear_way.argtypes = lib.ccsm_train_linear_backward_way.argtypes = [vp, vp]
    lib.ccsm_train_embedding_forward.argtypes = [ci, ci, ci, cl, vp, cl, C.c_int32, vp, cl, cf, vp, cl, vp]
    lib.ccsm_train_embedding_backward_workspace.argtypes = [ci, cl, cl, C.c_int32]
    lib.ccsm_train_embedding_backward_workspace.restype = cs
    lib.ccsm_train_embedding_backward.argtypes = [ci, ci, ci, cl, vp, cl, C.c_int32, vp, cl, cf, vp, cl, vp, cs, vp]
    lib.ccsm_train_act8_pack.argtypes = [ci, ci, ci, cl, C.c_int32, vp, cl, vp, cl, vp, cl, vp]
    lib.ccsm_train_act8_unpack.argtypes = [ci, ci, cl, C.c_int32, vp, vp, cl, vp]
    _ops = lib
    return lib


def _check(status):
    if status != _lib.OK:
        raise _lib.CcsmError(status, load().ccsm_train_ops_last_error().decode())


def _types():
    import torch
    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}, {torch.uint8: 0, torch.int32: 1, torch.int64: 2}


_TYPE = _ID = _torch = _Tensor = _forward = None


def _init():
    global _TYPE, _ID, _torch, _Tensor, _forward
    if _torch is None:
        import torch
        import torch.autograd.forward_ad as _forward
        _TYPE, _ID = _types()
        _torch, _Tensor = torch, torch.Tensor
    return _torch


def _tensor(t, name, dtype=None, device=None):
    torch = _torch
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor" % name)
    if t.dtype not in _TYPE:
        raise ValueError("%s must be float32, float16 or bfloat16, not %s" % (name, t.dtype))
    if dtype is not None and t.dtype is not dtype:
        raise ValueError("%s is %s, the call's type is %s" % (name, t.dtype, dtype))
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient: these calls are not seen by autograd (use torch.no_grad() and the *_backward calls)" % name)
    if _dual() and _forward.unpack_dual(t).tangent is not None:
        raise ValueError("%s has a forward-mode tangent: these calls are not seen by autograd" % name)
    return t


def _dual():
    """whether tensors may have forward-mode tangents (a dual level is entered)"""
    return getattr(_forward, "_current_level", 0) >= 0


def _on_gpu(t, name):
    if not t.is_cuda:
        raise ValueError("%s must be on a GPU: there is no CPU path" % name)


# A call of one token is bound by the host (10 us, of which the launch is 3): the two checks below see in a few attributes that nothing is wrong, and
# leave it to the ones above to say what is.
def _lead(t, name):
    """the type and the device's number of a call's first tensor"""
    if type(t) is not _Tensor or t.dtype not in _TYPE or t.requires_grad or not t.is_cuda or _dual():
        _tensor(t, name)
        _on_gpu(t, name)
    return t.dtype, t.get_device()


def _same(t, name, dtype, at, lead):
    """t, of the call's type and on its device"""
    if type(t) is _Tensor and t.dtype is dtype and t.get_device() == at and not t.requires_grad and not _dual():
        return t
    return _tensor(t, name, dtype, lead.device)


def _rows(t):
    """(tensor whose rows are contiguous, its row stride): t as it is, or a copy"""
    if t.is_contiguous() and t.dim() and not t.is_neg():
        return t, t.shape[-1]
    t = t.resolve_neg()                                    # (the imaginary part of a conjugate: its memory holds the other sign)
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.dim() else t.reshape(1, 1)
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1))


def _elsewhere(call, stream, device, given, *args, **kw):
    """call(*args, **kw) with `stream` as the current stream: what it allocates belongs to that stream, and the tensors that it was given are kept for it until
    its work is done."""
    torch = _torch
    if not isinstance(stream, torch.cuda.Stream):
        raise TypeError("stream must be a torch.cuda.Stream")
    if stream.device != device:
        raise ValueError("stream belongs to %s, the tensors to %s" % (stream.device, device))
    with torch.cuda.stream(stream):
        out = call(*args, **kw)
        for t in given:
            if isinstance(t, Checkpoint8):
                t.codes.record_stream(stream)
                t.scales.record_stream(stream)
            elif t is not None:
                t.record_stream(stream)
    return out


def _raw_stream(at):
    return _torch._C._cuda_getCurrentRawStream(at)


def _scratch(n, lead):
    return lead.new_empty(n, dtype=_torch.uint8) if n else None


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _activation(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation must be one of %s, not %r" % (", ".join(ACTIVATIONS), name))
    return ACTIVATIONS[name]


def _library():
    if _ops is None or _torch is None:
        _init()
        load()
    return _ops


def _out(out, shape, dtype, device, name):
    if out.shape != shape or out.dtype is not dtype or out.device != device:
        raise ValueError("%s must be a %s tensor of shape %s on %s" % (name, dtype, tuple(shape), device))
    if out.dim() > 1 and not out.is_contiguous() and (out.dim() != 2 or out.stride(1) != 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1]) or \
            out.dim() == 1 and out.numel() > 1 and out.stride(0) != 1:
        raise ValueError("%s must have contiguous rows" % name)
    if out.is_neg():
        raise ValueError("%s is a view with its sign turned" % name)
    return out


class Checkpoint8:
    """An activation in 8 bits (layout: include/ccsm_train_ops.h): `codes` (rows, width rounded up to 32) and `scales` (rows, width / 32 rounded up),
    uint8; `shape` and `dtype` of the tensor it was made of; `code` "int8" or "e4m3"."""

    def __init__(self, codes, scales, shape, dtype, code):
        torch = _init()
        shape = tuple(int(n) for n in shape)
        if code not in CODES:
            raise ValueError("code must be one of %s, not %r" % (", ".join(CODES), code))
        if dtype not in _TYPE:
            raise ValueError("dtype must be float32, float16 or bfloat16, not %s" % dtype)
        if not shape or shape[-1] < 1:
            raise ValueError("a checkpoint has at least one column")
        rows = 1
        for n in shape[:-1]:
            rows *= n
        blocks = -(-shape[-1] // 32)
        for t, cols, name in ((codes, 32 * blocks, "codes"), (scales, blocks, "scales")):
            if t.dtype is not torch.uint8 or tuple(t.shape) != (rows, cols) or not t.is_contiguous():
                raise ValueError("%s must be a contiguous uint8 tensor of shape %s" % (name, (rows, cols)))
        if codes.device != scales.device:
            raise ValueError("codes and scales are on different devices")
        self.codes, self.scales, self.shape, self.dtype, self.code = codes, scales, torch.Size(shape), dtype, code

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def _saved(self):
        blocks = (self.shape[-1] + 31) // 32
        return self.codes.data_ptr(), 32 * blocks, CODES[self.code], self.scales.data_ptr(), blocks

    def values(self, dtype=None, *, out=None, stream=None):
        """The values that the codes stand for, as a tensor of `dtype` (default: the type it was made of, which holds them exactly)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _TYPE:
            raise ValueError("dtype must be float32, float16 or bfloat16, not %s" % dtype)
        lib = _library()
        codes, shape = self.codes, self.shape
        _on_gpu(codes, "the checkpoint")
        if stream is not None:
            return _elsewhere(self.values, stream, self.device, (self, out), dtype, out=out)
        if out is None:
            y, width = codes.new_empty(shape, dtype=dtype), shape[-1]
            ldy = width
        else:
            y, width = _out(_tensor(out, "out"), shape, dtype, self.device, "out"), shape[-1]
            ldy = _rows(y)[1]
        at = codes.get_device()
        _check(lib.ccsm_train_act8_unpack(at, _TYPE[dtype], codes.shape[0], width, _SAVED.pack(*self._saved()), y.data_ptr(), ldy, _raw_stream(at)))
        return y


def checkpoint8(x, code="int8", *, stream=None):
    """x (..., width) -> Checkpoint8: blocks of 32 values of a row share a power of two; "int8" keeps 127 even steps either side of zero (bounded
    activations, normalised inputs), "e4m3" three bits behind the leading one (long-tailed ones)."""
    lib = _library()
    if code not in CODES:
        raise ValueError("code must be one of %s, not %r" % (", ".join(CODES), code))
    t, at = _lead(x, "x")
    shape = x.shape
    if not shape or shape[-1] < 1:
        raise ValueError("x must have at least one column")
    if stream is not None:
        return _elsewhere(checkpoint8, stream, x.device, (x,), x, code)
    x2, ldx = _rows(x)
    width = shape[-1]
    rows, blocks, u8 = x.numel() // width, (width + 31) // 32, _torch.uint8
    codes, scales = x.new_empty((rows, 32 * blocks), dtype=u8), x.new_empty((rows, blocks), dtype=u8)
    _check(lib.ccsm_train_act8_pack(at, _TYPE[t], CODES[code], rows, width, x2.data_ptr(), ldx, codes.data_ptr(), 32 * blocks, scales.data_ptr(), blocks, _raw_stream(at)))
    c = Checkpoint8.__new__(Checkpoint8)                    # (what __init__ checks holds here)
    c.codes, c.scales, c.shape, c.dtype, c.code = codes, scales, shape, t, code
    return c


def linear(x, weight, bias=None, residual=None, activation="none", keep_preact=False, *, out=None, stream=None):
    """y = act(x weight^T + bias) + residual; x (..., inner), weight (outer, inner), bias (outer), residual and y (..., outer).
    keep_preact: -> (y, z) with z = x weight^T + bias as linear_backward takes it.  out: where y goes; it may be the residual and shares no memory with
    the other tensors."""
    lib = _library()
    act = _activation(activation)
    t, at = _lead(x, "x")
    _same(weight, "weight", t, at, x)
    given, both = x.shape, weight.shape
    if len(both) != 2 or not given or given[-1] != both[1]:
        raise ValueError("x must be (..., inner) and weight (outer, inner): got %s and %s" % (tuple(given), tuple(both)))
    outer, inner = both
    if inner < 1 or outer < 1:
        raise ValueError("weight has no rows or no columns")
    shape = given[:-1] + (outer,)
    if bias is not None and _same(bias, "bias", t, at, x).shape != (outer,):
        raise ValueError("bias must be (%d,)" % outer)
    if residual is not None and _same(residual, "residual", t, at, x).shape != shape:
        raise ValueError("residual must be %s" % (tuple(shape),))
    if stream is not None:
        return _elsewhere(linear, stream, x.device, (x, weight, bias, residual, out), x, weight, bias, residual, activation, keep_preact, out=out)
    y, ldy = (x.new_empty(shape), outer) if out is None else _rows(_out(_tensor(out, "out"), shape, t, x.device, "out"))
    z = x.new_empty(shape) if keep_preact else None
    x2, ldx = _rows(x)
    w2, ldw = _rows(weight)
    b1 = None if bias is None else bias.resolve_neg().contiguous()
    r2, ldr = (None, 0) if residual is None else _rows(residual)
    p = _LINEAR.pack(_TYPE[t], act, x.numel() // inner, inner, outer, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(b1), _ptr(r2), ldr, y.data_ptr(), ldy, _ptr(z), outer)
    need = lib.ccsm_train_linear_workspace(p)
    ws = _scratch(need, x)
    _check(lib.ccsm_train_linear_forward(at, p, _ptr(ws), need, _raw_stream(at)))
    if out is not None:
        y = out
    return (y, z) if keep_preact else y


def linear_backward(dy, x, weight, preact=None, activation="none", *, need_dx=True, need_dw=True, need_db=True, stream=None):
    """The gradients of y = act(x weight^T + bias) (+ residual, whose gradient is dy itself): (dx, dw, db), None for what is not needed.
    Large 16-bit products with an activation take dy act'(preact) rounded to the type: their dx and dw carry two roundings (include/ccsm_train_ops.h).
    dy (..., outer); x (..., inner) and preact (..., outer) are tensors or Checkpoint8s; preact only where there is an activation."""
    lib = _library()
    act = _activation(activation)
    t, at = _lead(dy, "dy")
    _same(weight, "weight", t, at, dy)
    given, both = dy.shape, weight.shape
    if len(both) != 2 or not given or given[-1] != both[0]:
        raise ValueError("dy must be (..., outer) and weight (outer, inner): got %s and %s" % (tuple(given), tuple(both)))
    outer, inner = both
    lead = given[:-1]
    if inner < 1 or outer < 1:
        raise ValueError("weight has no rows or no columns")
    if act and preact is None:
        raise ValueError("preact is needed for the slope of %s" % activation)

    def saved(v, cols, name):
        if v is None:
            return _NONE, None
        if v.shape != lead + (cols,):
            raise ValueError("%s must be %s, not %s" % (name, tuple(lead) + (cols,), tuple(v.shape)))
        if isinstance(v, Checkpoint8):
            if v.codes.get_device() != at:
                raise ValueError("%s is on %s, not on %s" % (name, v.device, dy.device))
            if v.dtype is not t:
                raise ValueError("%s was made of %s, the call's type is %s" % (name, v.dtype, t))
            return v._saved(), None
        v2, ld = _rows(_same(v, name, t, at, dy))
        return (v2.data_ptr(), ld, 0, 0, 0), v2

    if need_dw and x is None:
        raise ValueError("x is needed for dw")
    if stream is not None:
        return _elsewhere(linear_backward, stream, dy.device, (dy, x, weight, preact), dy, x, weight, preact, activation, need_dx=need_dx, need_dw=need_dw, need_db=need_db)
    xs, _x = saved(x if need_dw else None, inner, "x")
    zs, _z = saved(preact if act else None, outer, "preact")
    dx = dy.new_empty(lead + (inner,)) if need_dx else None
    dw = dy.new_empty((outer, inner)) if need_dw else None
    db = dy.new_empty(outer) if need_db else None
    d2, ldd = _rows(dy)
    w2, ldw = _rows(weight)
    p = _GRAD.pack(_TYPE[t], act, dy.numel() // outer, inner, outer, d2.data_ptr(), ldd, *xs, w2.data_ptr(), ldw, *zs, _ptr(dx), inner, _ptr(dw), inner, _ptr(db))
    need = lib.ccsm_train_linear_backward_workspace(p)
    ws = _scratch(need, dy)
    _check(lib.ccsm_train_linear_backward(at, p, _ptr(ws), need, _raw_stream(at)))
    return dx, dw, db


def _ids(ids, at, lead):
    if not isinstance(ids, _Tensor) or ids.dtype not in _ID:
        raise ValueError("ids must be a uint8, int32 or int64 tensor")
    if ids.get_device() != at:
        raise ValueError("ids are on %s, not on %s" % (ids.device, lead.device))
    return ids.contiguous()


def embedding(ids, table, scale=1.0, *, out=None, stream=None):
    """y (*ids.shape, width) = scale * table[ids].  Ids outside [0, len(table)), padding of -1 for instance, give a row of zeros."""
    lib = _library()
    t, at = _lead(table, "table")
    both = table.shape
    if len(both) != 2 or both[0] < 1 or both[1] < 1:
        raise ValueError("table must be (rows, width)")
    if stream is not None:
        return _elsewhere(embedding, stream, table.device, (ids, table, out), ids, table, scale, out=out)
    i = _ids(ids, at, table)
    rows, width = both
    shape = ids.shape + (width,)
    y, ldy = (table.new_empty(shape), width) if out is None else _rows(_out(_tensor(out, "out"), shape, t, table.device, "out"))
    t2, ldt = _rows(table)
    _check(lib.ccsm_train_embedding_forward(at, _TYPE[t], _ID[i.dtype], i.numel(), i.data_ptr(), rows, width, t2.data_ptr(), ldt, float(scale), y.data_ptr(), ldy, _raw_stream(at)))
    return y if out is None else out


def embedding_backward(dy, ids, rows, scale=1.0, *, out=None, stream=None):
    """The gradient of embedding()'s table, (rows, width) in dy's type: row v = scale * the sum of dy's rows whose id is v, zero where there is none.
    A row's sum has one order, that of its tokens: the same inputs give the same bits."""
    lib = _library()
    t, at = _lead(dy, "dy")
    rows = int(rows)
    if rows < 1:
        raise ValueError("rows must be at least 1")
    given = dy.shape
    if not given or given[-1] < 1 or not hasattr(ids, "shape") or given[:-1] != ids.shape:
        raise ValueError("dy must be (*ids.shape, width)")
    if stream is not None:
        return _elsewhere(embedding_backward, stream, dy.device, (dy, ids, out), dy, ids, rows, scale, out=out)
    width = given[-1]
    i = _ids(ids, at, dy)
    dt, ldt = (dy.new_empty((rows, width)), width) if out is None else _rows(_out(_tensor(out, "out"), _torch.Size((rows, width)), t, dy.device, "out"))
    d2, ldd = _rows(dy)
    kind, n = _TYPE[t], i.numel()
    need = lib.ccsm_train_embedding_backward_workspace(kind, n, rows, width)
    ws = _scratch(need, dy)
    _check(lib.ccsm_train_embedding_backward(at, kind, _ID[i.dtype], n, i.data_ptr(), rows, width, d2.data_ptr(), ldd, float(scale), dt.data_ptr(), ldt, _ptr(ws), need, _raw_stream(at)))
    return dt if out is None else out
