"""Products with weights held in 4 bits: the codes, scales and zero points of quant_weight's quantizers, packed into the
layout that the matrix-core kernels read (include/mq.h, mq_w4 / mq_linear4), and the products on them.

  pack_weight(w, wq_bits, datatype, group_size)      quantize a weight [N, K] (or experts [E, N, K]) and pack it
  pack_codes(q, scale, zp, wq_bits, datatype, ...)   pack what _int_quant_meta / _fp_quant_meta returned
  packed_linear(x, weight, bias)                     x W^T + bias, any number of rows; backward: dx, db
  packed_expert_linear(x, weight, counts, bias)      the same with rows sorted by expert; backward: dx, db
  PackedLinear                                       nn.Linear's place in a model (quant_model(..., packed=True))

W = scale * (q - zero point), per group of input channels; the weight is frozen (no gradient for codes or scales).
Activations are float16 or bfloat16 (below 2^116: sums over code values come before the scales), sums float32, results
rounded once.  The reference keeps such codes beside the weight
(_LinearDump, quant_weight.py:876-914) and multiplies by the dequantized float16 weight; there is no CPU compute path.
"""
import ctypes
import warnings
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib
from .fused import TABLE_LISTS, lut_values, require_device

INT_ASYM, INT_SYM, TABLE, FP4 = 0, 1, 2, 3   # mq_w4_kind
_XDTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


class _W4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("params", ctypes.c_void_p), ("norm", ctypes.c_void_p),
                ("experts", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64), ("group", ctypes.c_int64),
                ("kind", ctypes.c_int32), ("reserved", ctypes.c_int32), ("values", ctypes.c_float * 16)]


_bound = None


def _bind():
    """libmq.so with the signatures of the 4-bit entry points set."""
    global _bound
    if _bound is None:
        L = _lib.lib()
        vp, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_size_t
        pw = ctypes.POINTER(_W4)
        L.mq_w4_data_bytes.restype, L.mq_w4_data_bytes.argtypes = sz, [i64, i64, i64]
        L.mq_w4_params_bytes.restype, L.mq_w4_params_bytes.argtypes = sz, [pw]
        L.mq_w4_pack.restype, L.mq_w4_pack.argtypes = ctypes.c_int, [pw, vp, vp, vp, vp]
        L.mq_w4_unpack.restype, L.mq_w4_unpack.argtypes = ctypes.c_int, [pw, vp, vp]
        L.mq_linear4_workspace_bytes.restype, L.mq_linear4_workspace_bytes.argtypes = sz, [pw, i32, i64, i32, i32, i32]
        L.mq_linear4.restype, L.mq_linear4.argtypes = ctypes.c_int, [pw, vp, i32, i64, i64, vp, vp, vp, vp, sz, vp]
        L.mq_linear4_grad.restype, L.mq_linear4_grad.argtypes = ctypes.c_int, [pw, vp, i32, i64, i64, vp, vp, vp, vp, sz, vp]
        _bound = L
    return _bound


def table_order(values):
    """The sixteen entries of a 3- / 4-bit value list by code: 0 and the positive values, then (from entry 9) the
    negative ones; an eighth value of one sign stands in entry 8."""
    pos, neg = sorted(v for v in values if v > 0), sorted((v for v in values if v < 0), reverse=True)
    if len(pos) > 8 or len(neg) > 8 or len(pos) + len(neg) > 15:
        raise ValueError("a 4-bit table holds at most 16 values")
    out = [0.0] * 16
    out[1:1 + len(pos[:7])] = pos[:7]
    out[9:9 + len(neg[:7])] = neg[:7]
    if len(pos) + len(neg) == 15:
        out[8] = (pos + neg)[7] if len(pos) == 8 else neg[7]
    return out


def _kind_of(wq_bits, datatype):
    """-> (mq_w4_kind, table by code | None); the refusals of quant_datatype for names it does not know
    (quant_weight.py:553-556)."""
    from .quant_weight import _KNOWN_TABLES
    if not isinstance(datatype, str):
        raise ValueError(f"unexpected data type {datatype!r}.")
    if datatype.startswith("int"):
        if wq_bits not in (2, 3, 4):
            raise ValueError(f"packed weights hold 2-, 3- or 4-bit integers, not {wq_bits}-bit")
        return (INT_ASYM if "asym" in datatype else INT_SYM), None
    if wq_bits not in (3, 4):
        raise ValueError(f"packed weights hold 3- or 4-bit tables, not {wq_bits}-bit")
    if datatype not in _KNOWN_TABLES[wq_bits]:
        raise ValueError(f"unexpected data type {datatype}.")
    if datatype == "fp4":
        return FP4, None
    return TABLE, table_order(TABLE_LISTS[datatype] if datatype in TABLE_LISTS else lut_values(datatype))


def _check_integers(q, kind):
    """Refuses integers that four bits of the kind do not hold (the library keeps them within its range, mq_w4_pack)."""
    low, high = (0, 15) if kind == INT_ASYM else (-7, 7)
    lo, hi = torch.aminmax(q.view(torch.uint8 if kind == INT_ASYM else torch.int8))
    if int(lo) < low or int(hi) > high:
        raise ValueError(f"codes from {int(lo)} to {int(hi)}: {low} to {high} can be packed")


def _check_values(q, c, norm, params):
    """Refuses values that the table of c, into which q has been packed, does not hold (they became 0): unpacked with scales
    of one, the codes have to be q."""
    ones, out = torch.full_like(params, 0x3C00), torch.empty_like(q)
    c.params, c.norm = ones.data_ptr(), norm.data_ptr()
    with torch.cuda.device(q.device):
        _lib.check(_bind().mq_w4_unpack(ctypes.byref(c), out.data_ptr(), torch.cuda.current_stream().cuda_stream))
    if bool((out != q).any()):
        raise ValueError("codes that are not values of the table")


def _group(group_size):
    """quant_weight.py:241-255: > 0 per group, -1 per tensor, everything else per row."""
    if group_size is None or (group_size <= 0 and group_size != -1):
        return 0
    return int(group_size)


class PackedWeight:
    """A weight [N, K], or a stack of experts [E, N, K], held in 4 bits on a ROCm device.

    data, params, norm: what the kernels read (include/mq.h, mq_w4), all integer tensors, so that no module-wide change
    of dtype touches them.  experts: E, or None for a single weight."""

    def __init__(self, data, params, norm, experts, n, k, group_size, wq_bits, datatype):
        """Takes the three tensors as they are; their sizes have to be what pack_codes made for this weight."""
        self.data, self.params, self.norm = data, params, norm
        self.experts, self.n, self.k = experts, int(n), int(k)
        self.group_size, self.wq_bits, self.datatype = _group(group_size), wq_bits, datatype
        self._describe()

    def _describe(self):
        kind, values = _kind_of(self.wq_bits, self.datatype)
        L = _bind()
        s = _W4(experts=self.experts or 1, n=self.n, k=self.k, group=max(self.group_size, 0), kind=kind)
        if values is not None:
            s.values[:] = values
        for t, dtype, nbytes in ((self.data, torch.int32, L.mq_w4_data_bytes(self.experts or 1, self.n, self.k)),
                                 (self.params, torch.int16, L.mq_w4_params_bytes(ctypes.byref(s))),
                                 (self.norm, torch.int32, 4 * (self.experts or 1))):
            if t.dtype != dtype or t.numel() * t.element_size() != nbytes or not nbytes or not t.is_contiguous() \
                    or t.device != self.data.device:
                raise ValueError(f"not the tensors of a packed weight: {t.dtype} {tuple(t.shape)} on {t.device}")
        self._c = s
        self._ref = ctypes.byref(s)
        self._at = None   # the addresses that _c holds
        self._need = {}   # workspace bytes by (dtype, rows, aligned, counted, grad)

    def _taken(self):
        """The description for a call, with the addresses that the tensors have now: `t.data = other` and their like keep
        the tensor object and give its old memory back."""
        at = (self.data.data_ptr(), self.params.data_ptr(), self.norm.data_ptr())
        if at != self._at:
            self._describe()
            self._c.data, self._c.params, self._c.norm = at
            self._at = at
        return self._ref

    def _versions(self):
        """How often each tensor has been written in place (tensors of inference mode do not say)."""
        try:
            return self.data._version, self.params._version, self.norm._version
        except RuntimeError:
            return None

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_c", "_ref", "_at", "_need")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._describe()

    @property
    def device(self):
        return self.data.device

    @property
    def shape(self):
        return torch.Size((self.n, self.k) if self.experts is None else (self.experts, self.n, self.k))

    def to(self, device):
        """The same weight on another ROCm device."""
        return PackedWeight(self.data.to(device), self.params.to(device), self.norm.to(device), self.experts, self.n, self.k,
                            self.group_size, self.wq_bits, self.datatype)

    def _operands(self):
        """The weight as the registered operators take it."""
        return (self.data, self.params, self.norm), (self.experts or 0, self.n, self.k, self.group_size, self.wq_bits, self.datatype)

    @torch.no_grad()
    def dequantize(self):
        """The float16 weight, with the bits that _int_quant_meta / _fp_quant_meta return for it, but for the sign of zero
        (a code has none): those of quant_int, quant_int_asym and quant_datatype too, except for a table with one scale per
        tensor, which quant_datatype computes in float32 (quant_weight.py:562-575)."""
        if _recorded(self.data):
            tensors, form = self._operands()
            return torch.ops.quantization_amd.packed_dequantize(*tensors, *form)
        return _dequantize(self)

    def __repr__(self):
        g = {0: "per row", -1: "per tensor"}.get(self.group_size, f"groups of {self.group_size}")
        return f"PackedWeight({tuple(self.shape)}, {self.wq_bits}-bit {self.datatype}, {g}, {self.device})"


def _dequantize(weight):
    out = torch.empty(weight.shape, dtype=torch.float16, device=weight.device)
    with torch.cuda.device(weight.device):
        _lib.check(_bind().mq_w4_unpack(weight._taken(), out.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out


@torch.no_grad()
def pack_codes(q, scale, zp=None, wq_bits: int = 4, datatype: str = "int4", group_size=None) -> PackedWeight:
    """Pack codes and parameters as _int_quant_meta / _fp_quant_meta return them (quant_weight.py:717-872).

    q: int8 / uint8 codes (integers: 0 .. 15 with zero points, -7 .. 7 without) or float16 table values, [N, K] or
    [N, G, group_size]; scale (and, for asymmetric integers, zp): float16, [N, G] per group, [N] per row, [] per tensor.
    With a leading dimension E on all of them: a stack of experts.  Groups are multiples of 32 that divide K; rows may have
    any length.  Codes that the format does not hold raise ValueError (which waits for the device)."""
    return _pack(q, scale, zp, wq_bits, datatype, group_size, True)


def _pack(q, scale, zp, wq_bits, datatype, group_size, check):
    if _compiling() or _tracing() or get_proxy_mode() is not None:
        raise RuntimeError("packing a weight cannot be recorded: pack it beforehand")
    kind, values = _kind_of(wq_bits, datatype)
    g = _group(group_size)
    experts = scale.dim() - (2 if g > 0 else 0 if g == -1 else 1)
    if experts not in (0, 1):
        raise ValueError(f"scale: {tuple(scale.shape)} is no shape of scales for group_size {group_size}")
    lead = tuple(scale.shape[:experts])
    if q.dim() == experts + 3 and g > 0:
        q = q.flatten(-2)
    if q.dim() != experts + 2 or tuple(q.shape[:experts]) != lead:
        raise ValueError(f"codes {tuple(q.shape)} and scales {tuple(scale.shape)} do not belong together")
    n, k = q.shape[-2:]
    if min(q.shape) < 1:
        raise ValueError(f"an empty weight {tuple(q.shape)} cannot be packed")
    if g > 0 and k % g:
        raise RuntimeError(f"shape '[{n}, {k // g}, {g}]' is invalid for input of size {n * k}")
    if g > 0 and g % 32:
        raise ValueError(f"packed weights have groups of a multiple of 32 input channels, not {g}")
    want = lead + ((n, k // g) if g > 0 else () if g == -1 else (n,))
    if (zp is not None) != (kind == INT_ASYM):
        raise ValueError(f"{datatype}: a zero point goes with asymmetric integers, and only with them")
    for name, t in (("scale", scale), ("zp", zp)):
        if t is not None and (tuple(t.shape) != want or t.dtype != torch.float16):
            raise ValueError(f"{name}: float16 {want} wanted, got {t.dtype} {tuple(t.shape)}")
    if q.dtype not in ((torch.float16,) if kind >= TABLE else (torch.int8, torch.uint8)):
        raise ValueError(f"codes of {datatype} cannot be {q.dtype}")
    q = require_device(q).contiguous()
    if check and kind < TABLE:
        _check_integers(q, kind)
    dev = q.device

    def rows(t):   # one scale per row at least
        t = t.to(dev)
        if g == -1:
            t = t.reshape(lead + (1,)).expand(lead + (n,))
        return t.contiguous()

    scale, zp = rows(scale), None if zp is None else rows(zp)
    L = _bind()
    e = lead[0] if experts else 1
    c = _W4(experts=e, n=n, k=k, group=max(g, 0), kind=kind)
    if values is not None:
        c.values[:] = values
    nbytes, pbytes = L.mq_w4_data_bytes(e, n, k), L.mq_w4_params_bytes(ctypes.byref(c))
    if not nbytes or not pbytes:
        raise ValueError(f"a weight of {tuple(q.shape)} is beyond what can be packed")
    # a power of two that brings the largest |weight| below 2^15 and above 2^13 (gradient of float16 activations)
    top = scale.reshape(e, -1).abs().amax(1).float()
    reach = 15 + zp.reshape(e, -1).abs().amax(1).float() if zp is not None else 16.0
    exponent = torch.frexp(top * reach).exponent
    ok = torch.isfinite(top * reach) & (top > 0)
    norm = (127 + torch.where(ok, 15 - exponent, torch.zeros_like(exponent))) << 23   # the bits of 2^(15 - exponent)
    data = torch.empty(nbytes // 4, dtype=torch.int32, device=dev)
    params = torch.empty(pbytes // 2, dtype=torch.int16, device=dev)
    c.data, c.params = data.data_ptr(), params.data_ptr()
    with torch.cuda.device(dev):
        _lib.check(L.mq_w4_pack(ctypes.byref(c), q.data_ptr(), scale.data_ptr(), None if zp is None else zp.data_ptr(),
                                torch.cuda.current_stream().cuda_stream))
    norm = norm.to(torch.int32)
    if check and kind >= TABLE:
        _check_values(q, c, norm, params)
    return PackedWeight(data, params, norm, lead[0] if experts else None, n, k, group_size, wq_bits,
                        datatype)


@torch.no_grad()
def pack_weight(w, wq_bits: int = 4, datatype: str = "int4", group_size=None) -> PackedWeight:
    """Quantize a weight [N, K] or a stack of experts [E, N, K] with the quantizers of quant_weight and pack the result."""
    from .quant_weight import _fp_quant_meta, _int_quant_meta
    kind, _ = _kind_of(wq_bits, datatype)
    if w.dim() not in (2, 3):
        raise ValueError(f"a weight [N, K] or [E, N, K] is wanted, got {tuple(w.shape)}")
    if min(w.shape) < 1:
        raise ValueError(f"an empty weight {tuple(w.shape)} cannot be packed")
    g = _group(group_size)
    if g > 0 and w.shape[-1] % g == 0 and g % 32:
        raise ValueError(f"packed weights have groups of a multiple of 32 input channels, not {g}")

    def meta(m):
        if kind >= TABLE:
            _, q, scale = _fp_quant_meta(m, wq_bits=wq_bits, datatype=datatype, group_size=group_size)
            return q, scale, None
        _, q, scale, zp = _int_quant_meta(m, wq_bits=wq_bits, asym=kind == INT_ASYM, group_size=group_size)
        return q, scale, zp

    w = require_device(w)
    if w.dim() == 2:
        q, scale, zp = meta(w)
    elif g == -1:   # one scale per expert
        parts = [meta(m) for m in w]
        q, scale = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
        zp = torch.stack([p[2] for p in parts]) if kind == INT_ASYM else None
    else:
        e, n, k = w.shape
        q, scale, zp = meta(w.reshape(e * n, k))
        q, scale = q.reshape(e, n, k), scale.reshape((e, n) + tuple(scale.shape[1:]))
        zp = None if zp is None else zp.reshape(scale.shape)
    return _pack(q, scale, zp, wq_bits, datatype, group_size, False)


def _rows_of(t):
    """A 2-D tensor as (tensor, elements from row to row) with neighbouring columns side by side."""
    rows, cols = t.shape
    if t.is_contiguous() or rows == 1 and (cols == 1 or t.stride(1) == 1):
        return t, cols
    if cols > 1 and t.stride(1) != 1 or 0 < t.stride(0) < cols:
        return t.contiguous(), cols
    return t, t.stride(0)


def _on_device(call, t, *args):
    """call(t, *args) with t's device as the current one."""
    index = t.get_device()
    if index == torch._C._cuda_getDevice():
        return call(t, *args, index)
    with torch.cuda.device(index):
        return call(t, *args, index)


def _workspace(weight, t, code, at, rows, ld, counts, grad):
    """-> (tensor | None, its address, bytes).  Of this call alone: a captured graph keeps it in its own pool, and calls on
    other streams have their own."""
    key = (code, rows, at % 16 == 0 and (ld % 8 == 0 and ld <= 1 << 23 or rows == 1), counts is not None, grad)
    need = weight._need.get(key)
    if need is None:
        if len(weight._need) >= 4096:
            weight._need.clear()
        need = weight._need[key] = _bound.mq_linear4_workspace_bytes(weight._ref, *key)
    if not need:
        return None, None, 0
    ws = torch.empty(need, dtype=torch.uint8, device=t.device)
    return ws, ws.data_ptr(), need


def _address(t):
    """For the library, to which 0 says that there is none."""
    at = None if t is None else t.data_ptr()
    if at == 0:
        raise RuntimeError("a tensor without memory of its own")
    return at


def _forward(x, weight, bias, counts, index):
    L = _bound or _bind()
    (rows, k), code = x.shape, _XDTYPES[x.dtype]
    y = x.new_empty((rows, weight.n))
    if rows:
        ref = weight._taken()
        x, ld = (x, k) if x.is_contiguous() else _rows_of(x)
        at = x.data_ptr()
        ws, wp, need = _workspace(weight, x, code, at, rows, ld, counts, 0)
        rc = L.mq_linear4(ref, at, code, rows, ld, _address(bias), _address(counts), y.data_ptr(), wp, need,
                          torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _lib.check(rc)
    return y


def _backward(dy, weight, counts, want_x, want_bias, index):
    L = _bound or _bind()
    rows, n = dy.shape
    dx = dy.new_empty((rows, weight.k)) if want_x else None
    db = dy.new_empty((n,) if weight.experts is None else (weight.experts, n)) if want_bias else None
    if not rows:
        return dx, None if db is None else db.zero_()
    ref = weight._taken()
    dy, ld = _rows_of(dy)
    at, code = dy.data_ptr(), _XDTYPES[dy.dtype]
    ws, wp, need = _workspace(weight, dy, code, at, rows, ld, counts, want_x + 2 * want_bias)
    rc = L.mq_linear4_grad(ref, at, code, rows, ld, _address(counts),
                           None if dx is None else dx.data_ptr(), None if db is None else db.data_ptr(), wp, need,
                           torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)
    return dx, db


# ---- where someone records or interprets torch's operators -------------------------------------------------
# The calls above hand addresses to the library, which nothing in torch sees: a recorder would keep the allocation of the
# result alone and replay that.  So wherever one is at work the same calls run as operators of torch's own.
_PLAIN = {torch.Tensor, nn.Parameter, type(None)}
_compiling, _tracing, _modes = torch.compiler.is_dynamo_compiling, torch._C._is_tracing, torch._C._len_torch_dispatch_stack


def _recorded(x, bias=None, counts=None):
    """True under torch.compile, torch.jit.trace, a dispatch mode (make_fx, torch.export, fake tensors) or for tensors of
    another class."""
    return (_compiling() or _tracing() or _modes() or type(x) not in _PLAIN or type(bias) not in _PLAIN
            or type(counts) not in _PLAIN)


@torch.library.custom_op("quantization_amd::packed_product", mutates_args=(), device_types="cuda")
def _product_op(x: torch.Tensor, data: torch.Tensor, params: torch.Tensor, norm: torch.Tensor, bias: Optional[torch.Tensor],
                counts: Optional[torch.Tensor], experts: int, n: int, k: int, group_size: int, wq_bits: int,
                datatype: str) -> torch.Tensor:
    weight = PackedWeight(data, params, norm, experts or None, n, k, group_size, wq_bits, datatype)
    _no_tangents(x, bias)
    bias, counts = _check_operands(x, weight, bias), _check_rows(x, weight, counts)
    if x.dim() != 2:
        raise ValueError(f"rows [R, {k}] are wanted, got {tuple(x.shape)}")
    return _on_device(_forward, x, weight, bias, counts)


@_product_op.register_fake
def _(x, data, params, norm, bias, counts, experts, n, k, group_size, wq_bits, datatype):
    return x.new_empty((x.shape[0], n))


@torch.library.custom_op("quantization_amd::packed_product_grad", mutates_args=(), device_types="cuda")
def _gradient_op(dy: torch.Tensor, data: torch.Tensor, params: torch.Tensor, norm: torch.Tensor,
                 counts: Optional[torch.Tensor], experts: int, n: int, k: int, group_size: int, wq_bits: int, datatype: str,
                 want_x: bool, want_bias: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """What is not wanted comes back empty."""
    _no_tangents(dy)
    weight = PackedWeight(data, params, norm, experts or None, n, k, group_size, wq_bits, datatype)
    if dy.dtype not in _XDTYPES or dy.dim() != 2 or dy.shape[1] != n or dy.device != data.device:
        raise ValueError(f"a gradient {dy.dtype} {tuple(dy.shape)} on {dy.device} does not fit a weight {tuple(weight.shape)}")
    dx, db = None, None
    if want_x or want_bias:
        dx, db = _on_device(_backward, dy, weight, _check_rows(dy, weight, counts), want_x, want_bias)
    return dy.new_empty(0) if dx is None else dx, dy.new_empty(0) if db is None else db


@_gradient_op.register_fake
def _(dy, data, params, norm, counts, experts, n, k, group_size, wq_bits, datatype, want_x, want_bias):
    db = ((experts, n) if experts else (n,)) if want_bias else (0,)
    return dy.new_empty((dy.shape[0], k) if want_x else (0,)), dy.new_empty(db)


def _product_op_setup(ctx, inputs, output):
    x, data, params, norm, bias, counts, *form = inputs
    ctx.save_for_backward(data, params, norm, counts)
    ctx.form = form


def _product_op_backward(ctx, dy):
    want_x, want_bias = ctx.needs_input_grad[0], ctx.needs_input_grad[4]
    dx, db = torch.ops.quantization_amd.packed_product_grad(dy, *ctx.saved_tensors, *ctx.form, want_x, want_bias)
    return (dx if want_x else None, None, None, None, db if want_bias else None) + (None,) * 7


_product_op.register_autograd(_product_op_backward, setup_context=_product_op_setup)


@torch.library.custom_op("quantization_amd::packed_dequantize", mutates_args=(), device_types="cuda")
def _dequantize_op(data: torch.Tensor, params: torch.Tensor, norm: torch.Tensor, experts: int, n: int, k: int,
                   group_size: int, wq_bits: int, datatype: str) -> torch.Tensor:
    return _dequantize(PackedWeight(data, params, norm, experts or None, n, k, group_size, wq_bits, datatype))


@_dequantize_op.register_fake
def _(data, params, norm, experts, n, k, group_size, wq_bits, datatype):
    return data.new_empty((experts, n, k) if experts else (n, k), dtype=torch.float16)


def _product(x, weight, bias, counts):
    if _recorded(x, bias, counts):
        tensors, form = weight._operands()
        return torch.ops.quantization_amd.packed_product(x, *tensors, bias, counts, *form)
    return _on_device(_forward, x, weight, bias, counts)


def _gradient(dy, weight, counts, want_x, want_bias):
    if _recorded(dy, None, counts):
        tensors, form = weight._operands()
        dx, db = torch.ops.quantization_amd.packed_product_grad(dy, *tensors, counts, *form, want_x, want_bias)
        return dx if want_x else None, db if want_bias else None
    return _on_device(_backward, dy, weight, counts, want_x, want_bias)


def _solid(t):
    """t in memory: tangents may be zeros without any."""
    return torch.zeros(t.shape, dtype=t.dtype, device=t.device) if t._is_zerotensor() else t


def _no_tangents(*tensors):
    """The operators have no forward-mode formula; torch would drop the tangents without a word."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("forward-mode differentiation goes through packed_linear and packed_expert_linear")


class _PackedProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bias, weight, counts):
        # (the weight's tensors are not saved: hooks that move what is saved would carry the whole weight to and fro)
        ctx.weight, ctx.versions = weight, weight._versions()
        ctx.save_for_backward(counts)
        if forward_ad._current_level >= 0:
            ctx.save_for_forward(counts)
            return _product(x, weight, bias, counts)
        return _on_device(_forward, x, weight, bias, counts)   # (_run has seen that nobody records it)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        counts, = ctx.saved_tensors
        want_x, want_bias = ctx.needs_input_grad[:2]
        if want_x and ctx.weight._versions() != ctx.versions:
            raise RuntimeError("the packed weight has been written in place since the forward pass: its gradient would be "
                               "that of another weight")
        dy, tangent = (dy, None) if forward_ad._current_level < 0 else forward_ad.unpack_dual(dy)
        dx, db = _gradient(dy, ctx.weight, counts, want_x, want_bias)
        if tangent is not None:   # (linear in dy)
            tx, tb = _gradient(_solid(tangent), ctx.weight, counts, want_x, want_bias)
            dx, db = (None if v is None else forward_ad.make_dual(v, t) for v, t in ((dx, tx), (db, tb)))
        return dx, db, None, None

    @staticmethod
    def jvp(ctx, dx, dbias, *_):
        """Linear in x and the bias: the tangent is the product of the tangents."""
        counts, = ctx.saved_tensors
        return _run(_solid(dx), ctx.weight, None if dbias is None else _solid(dbias).contiguous(), counts)


def _check_operands(x, weight, bias):
    if not isinstance(weight, PackedWeight):
        raise TypeError(f"a PackedWeight is wanted, got {type(weight).__name__}")
    if not x.is_cuda:
        raise RuntimeError("packed products expect ROCm device tensors; no CPU fallback exists")
    if x.dtype not in _XDTYPES:
        raise ValueError(f"float16 or bfloat16 activations are wanted, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] != weight.k:
        raise ValueError(f"activations {tuple(x.shape)} do not fit a weight {tuple(weight.shape)}")
    if x.get_device() != weight.data.get_device():
        raise ValueError(f"activations on {x.device}, weight on {weight.device}")
    if bias is not None:
        want = (weight.n,) if weight.experts is None else (weight.experts, weight.n)
        if tuple(bias.shape) != want or bias.dtype != x.dtype or bias.device != x.device:
            raise ValueError(f"bias: {x.dtype} {want} on {x.device} wanted, got {bias.dtype} {tuple(bias.shape)} on "
                             f"{bias.device}")
        bias = bias.contiguous()
    return bias


def _check_rows(x, weight, counts):
    """The counts of experts' rows as the library reads them; None for a single weight."""
    if weight.experts is None:
        if counts is not None:
            raise ValueError("counts go with a stack of experts")
        return None
    if not isinstance(counts, torch.Tensor) or counts.dtype not in (torch.int32, torch.int64) \
            or tuple(counts.shape) != (weight.experts,) or counts.device != x.device:
        raise ValueError(f"counts: int32 or int64 [{weight.experts}] on {x.device} wanted")
    if counts.dtype == torch.int64:
        counts = counts.clamp(0, x.shape[0]).to(torch.int32)
    return counts.contiguous()


def _run(x, weight, bias, counts):
    forwards = forward_ad._current_level >= 0
    if not forwards and _recorded(x, bias, counts):
        return _product(x, weight, bias, counts)   # (the operator knows its gradient)
    if forwards or torch.is_grad_enabled() and (x.requires_grad or bias is not None and bias.requires_grad):
        return _PackedProduct.apply(x, bias, weight, counts)
    return _on_device(_forward, x, weight, bias, counts)


def packed_linear(x, weight: PackedWeight, bias=None):
    """x [..., K] -> x W^T + bias [..., N], in x's dtype (float16 / bfloat16).

    One row reads the weight at memory speed, many rows run on the matrix cores; the values of the codes enter the
    products exactly and the scales are applied in float32.  Differentiable in x and bias (once)."""
    bias = _check_operands(x, weight, bias)
    if weight.experts is not None:
        raise ValueError("a stack of experts goes through packed_expert_linear")
    if x.dim() == 2:
        return _run(x, weight, bias, None)
    return _run(x.reshape(-1, weight.k), weight, bias, None).reshape(x.shape[:-1] + (weight.n,))


def packed_expert_linear(x, weight: PackedWeight, counts, bias=None):
    """x [R, K], rows sorted by expert -> [R, N] with row r times the weight (plus the bias row) of its expert.

    counts: int32 or int64 [E] on x's device, the number of rows of each expert; it is never read by the host, so a
    call can be captured and replayed with other counts.  Rows behind the last expert's come back as zeros; counts that
    add up to more than R are cut off there.  Differentiable in x and bias (once)."""
    bias = _check_operands(x, weight, bias)
    if weight.experts is None:
        raise ValueError("a single weight goes through packed_linear")
    if x.dim() != 2:
        raise ValueError(f"rows [R, {weight.k}] are wanted, got {tuple(x.shape)}")
    return _run(x, weight, bias, _check_rows(x, weight, counts))


_BUFFERS = {"weight_data": "data", "weight_params": "params", "weight_norm": "norm"}   # of PackedLinear: its PackedWeight's


class PackedLinear(nn.Module):
    """A Linear whose weight is held in 4 bits: quantizes src.weight with pack_weight; the bias stays a parameter."""

    _packed = None   # the PackedWeight of the present buffers, once one has been asked for

    def __init__(self, src: nn.Linear, wq_bits: int = 4, datatype: str = "int4", group_size=None):
        super().__init__()
        self.in_features, self.out_features = src.in_features, src.out_features
        p = pack_weight(src.weight.data, wq_bits, datatype, group_size)
        self._form = (p.experts, p.n, p.k, p.group_size, p.wq_bits, p.datatype)
        for name, of in _BUFFERS.items():
            self.register_buffer(name, getattr(p, of))
        self.bias = None if src.bias is None else nn.Parameter(src.bias.detach().to(p.device),
                                                               requires_grad=src.bias.requires_grad)

    @property
    def packed(self) -> PackedWeight:
        """The weight that the buffers hold (moved, loaded or assigned ones are taken up)."""
        p = self._packed
        if p is None or p.data is not self.weight_data or p.params is not self.weight_params or p.norm is not self.weight_norm:
            p = self._packed = PackedWeight(self.weight_data, self.weight_params, self.weight_norm, *self._form)
        return p

    # Wherever buffers are exchanged the PackedWeight goes with them: it would keep the old ones' memory.
    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if name in _BUFFERS:
            self._packed = None

    def _apply(self, fn, recurse=True):
        self._packed = None
        return super()._apply(fn, recurse)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_packed"}

    def __setstate__(self, state):
        old = state.pop("_packed", None)   # modules saved before _form was kept
        if old is not None:
            state["_form"] = (old.experts, old.n, old.k, old.group_size, old.wq_bits, old.datatype)
        super().__setstate__(state)

    # A state dict says what its codes mean: the buffers of two formats may have the same sizes.
    def _format(self):
        _, n, k, group, bits, datatype = self._form
        kind, values = _kind_of(bits, datatype)
        name = {INT_ASYM: "asymmetric integers", INT_SYM: "symmetric integers", FP4: "fp4"}.get(kind) or \
            "table " + " ".join(f"{v:g}" for v in values)
        rows = group <= 0 or group == k and k % 128 == 0    # (one group: the same parameters)
        return f"{n} x {k}, {name}, {'one scale per row' if rows else f'groups of {group}'}"

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "weight_format"] = torch.tensor(list(self._format().encode()), dtype=torch.uint8)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        key = prefix + "weight_format"
        text = state_dict.get(key)
        if text is not None and not text.is_meta:
            theirs = bytes(text.to(torch.uint8).tolist()).decode(errors="replace")
            if theirs != self._format():   # nothing of it is taken over
                error_msgs.append(f"{key}: the format of the state dict's weight is \"{theirs}\", this module's "
                                  f"\"{self._format()}\"")
                return
        elif text is None and prefix + "weight_data" in state_dict:
            warnings.warn(f"{key} is missing: a weight of another format would be decoded wrongly", stacklevel=2)
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        if key in unexpected_keys:
            unexpected_keys.remove(key)

    def forward(self, x):
        return packed_linear(x, self.packed, self.bias)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, {self.packed}"
