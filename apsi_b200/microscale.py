"""Microscaled 4-bit floating point on the device: quantise, dequantise, multiply, and multiply by expert.

``"mxfp4"``: e2m1 codes with a power-of-two scale per 32 values along a row.  ``"nvfp4"``: e2m1 codes with an e4m3 scale
per 16 values and one float32 scale for the whole tensor.  Both are what the tensor cores of an sm_100 GPU multiply as
they are: a product of two ``MxTensor`` never expands its codes.  The reference has minifloats with a scale
per row or tensor only (``precision.quantize``, apsi/precision.py:205-246).

    w = quantize(W, "nvfp4")                       # [N, K] weight, or [E, N, K]: one per expert
    y = linear(x, w)                               # x quantised on the way in, or an MxTensor
    q = quantize(x, "nvfp4", rows=r.rows, offsets=r.offsets)      # rows of x in expert order (experts.route)
    z = linear_grouped(q, w)                       # group e of the rows times w[e]

Everything runs on the current stream of the operands' device and allocates outputs only; an argument that does not fit raises
``LowbitError`` before anything is launched.  Row indices and group offsets live on the device and are checked there: one out
of range is not followed and sets ``DEVERR_BAD_INDEX`` (``kernels.device_errors``).
"""
import torch

from . import _lib
from ._lib import DT_BF16, DT_F16, DT_F32, LB_E_ARG, LB_E_DEVICE, LowbitError, MICROSCALED_FMT, MX_MAX_GROUPS, MX_PARTIALS

__all__ = ["MxTensor", "quantize", "dequantize", "pack", "plain_scales", "linear", "linear_grouped"]

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}
_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(_lib.load(), name)
    return f


def _err(msg):
    return LowbitError(LB_E_ARG, msg)


def _cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise LowbitError(LB_E_DEVICE, f"{name} must be a CUDA tensor (the B200 path has no CPU fallback)")
    return t


def _launch(dev, name, *args):
    """One call of the library on ``dev``'s current stream (the last argument)."""
    if dev.index == torch.cuda.current_device():
        rc = _fn(name)(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = _fn(name)(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _lib.check(rc)


def _format(fmt):
    f = MICROSCALED_FMT.get(fmt)
    if f is None:
        raise _err(f"'{fmt}' is not a microscaled format {sorted(MICROSCALED_FMT)}")
    return f


def _row_bytes(K):
    return (K + 31) // 32 * 16


def _scale_bytes(fmt, R, K, G, per):
    """lb_mx_scale_bytes, without the call."""
    blocks = (R + 127) // 128 if not G else G * ((per + 127) // 128) if per else R // 128 + min(G, R)
    return blocks * ((K + 255) // 256) * (2 if fmt == "mxfp4" else 4) * 512


def _ptr(t):
    return None if t is None else t.data_ptr()


class MxTensor:
    """Microscaled rows: ``fmt``; ``shape`` ([R, K], or [E, N, K] for one matrix per expert); ``codes`` uint8
    [rows, row bytes]; ``scales`` uint8, in the tensor cores' order (``plain_scales`` gives rows); ``tensor_scale``
    float32 [1] (nvfp4; else None); ``offsets`` int32 [G + 1] when the rows are ragged groups (else None)."""
    __slots__ = ("fmt", "shape", "codes", "scales", "tensor_scale", "offsets")

    def __init__(self, fmt, shape, codes, scales, tensor_scale=None, offsets=None):
        self.fmt, self.shape, self.codes, self.scales = fmt, shape, codes, scales
        self.tensor_scale, self.offsets = tensor_scale, offsets

    @property
    def device(self):
        return self.codes.device

    @property
    def rows(self):
        return self.shape[0] if len(self.shape) == 2 else self.shape[0] * self.shape[1]

    def _groups(self):
        """(G, per) as the library takes them."""
        if self.offsets is not None:
            return self.offsets.numel() - 1, 0
        return (0, 0) if len(self.shape) == 2 else (self.shape[0], self.shape[1])

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def dequantize(self, dtype=torch.float32):
        return dequantize(self, dtype)

    def __repr__(self):
        return f"MxTensor({self.fmt}, {list(self.shape)}, {self.device})"


def _index(t, name, dev):
    if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
        raise _err(f"{name} must be a contiguous int32 vector on {dev}")
    return t


def _tensor_scale(fmt, t, dev):
    if fmt != "nvfp4":
        if t is not None:
            raise _err(f"{fmt} has no tensor scale")
        return None
    if t is None or isinstance(t, torch.Tensor):
        if t is not None and (t.device != dev or t.dtype != torch.float32 or t.numel() != 1):
            raise _err(f"tensor_scale must be one float32 value on {dev}")
        return t
    if not 0.0 < float(t) < float("inf"):
        raise _err(f"tensor_scale must be positive and finite, got {t}")
    return torch.full((1,), float(t), dtype=torch.float32, device=dev)


def quantize(x, fmt, tensor_scale=None, rows=None, offsets=None):
    """The rows of ``x`` [R, K] (float32, bfloat16 or float16; any row stride) in a microscaled format; [E, N, K]
    (contiguous) gives one matrix per expert.

    ``tensor_scale`` (nvfp4): a positive number or a float32 tensor of one; by default the smallest power of two that keeps
    every block scale in range, found in a pass over x.  ``rows`` (int32): quantise x[rows] instead, in that order.
    ``offsets`` (int32 [G + 1]): the (chosen) rows are groups [offsets[e], offsets[e + 1]), for ``linear_grouped``."""
    f = _format(fmt)
    _cuda(x, "x")
    dt = _DT.get(x.dtype)
    if dt is None:
        raise _err(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    dev, shape = x.device, tuple(x.shape)
    G = per = 0
    if len(shape) == 3:
        if not x.is_contiguous() or rows is not None or offsets is not None:
            raise _err("one matrix per expert [E, N, K] must be contiguous, with neither rows nor offsets")
        G, per, K = shape
        if not 0 < G <= MX_MAX_GROUPS:
            raise _err(f"at most {MX_MAX_GROUPS} experts, got {G}")
        R_in, ldx = G * per, K
    elif len(shape) == 2:
        R_in, K = shape
        ldx = x.stride(0) if R_in > 1 else max(K, 1)
    else:
        raise _err(f"x must be [R, K] or [E, N, K], got {list(shape)}")
    if K == 0 or x.stride(-1) != 1 and K > 1:
        raise _err("the values of a row must be next to each other, and at least one")
    R = R_in
    if rows is not None:
        R = _index(rows, "rows", dev).numel()
        shape = (R, K)
    if offsets is not None:
        G = _index(offsets, "offsets", dev).numel() - 1
        if not 0 < G <= MX_MAX_GROUPS:
            raise _err(f"offsets must hold 2 to {MX_MAX_GROUPS + 1} values, got {G + 1}")
    t = _tensor_scale(fmt, tensor_scale, dev)
    auto = None
    if t is None and f == _lib.FMT_NVFP4:
        auto = torch.empty((1 + MX_PARTIALS,), dtype=torch.float32, device=dev)
        if R == 0:
            auto[0] = 1.0
    codes = torch.empty((R, _row_bytes(K)), dtype=torch.uint8, device=dev)
    scales = torch.empty((_scale_bytes(fmt, R, K, G, per),), dtype=torch.uint8, device=dev)
    _launch(dev, "lb_mx_quant", f, x.data_ptr(), dt, R_in, K, ldx, _ptr(rows), R, _ptr(offsets), G, per, _ptr(t), _ptr(auto),
            codes.data_ptr(), scales.data_ptr())
    return MxTensor(fmt, shape, codes, scales, t if auto is None else auto[:1], offsets)


def dequantize(q, dtype=torch.float32):
    """The values of an ``MxTensor`` in float32, bfloat16 or float16 (rows that lie in no group are not written)."""
    dt = _DT.get(dtype)
    if dt is None:
        raise _err(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    G, per = q._groups()
    K, dev = q.shape[-1], q.codes.device
    out = torch.empty(q.shape, dtype=dtype, device=dev)
    _launch(dev, "lb_mx_dequant", MICROSCALED_FMT[q.fmt], q.codes.data_ptr(), q.scales.data_ptr(), _ptr(q.tensor_scale), q.rows, K,
            _ptr(q.offsets), G, per, out.data_ptr(), dt, K)
    return out


def pack(codes, scales, K, fmt, tensor_scale=None):
    """An ``MxTensor`` from a checkpoint's arrays: ``codes`` uint8 [N, >= ceil(K / 2)] (even element in the low bits) or
    [E, N, ...], ``scales`` [N, >= blocks] or [E, N, ...]: uint8, or the float8 type whose bytes they are."""
    f = _format(fmt)
    _cuda(codes, "codes")
    dev, lead = codes.device, tuple(codes.shape[:-1])
    if codes.dtype != torch.uint8 or len(lead) not in (1, 2) or 0 in lead:
        raise _err("codes must be uint8 [N, bytes] or [E, N, bytes]")
    if not isinstance(scales, torch.Tensor) or scales.device != dev or scales.element_size() != 1 or tuple(scales.shape[:-1]) != lead:
        raise _err(f"scales must be one byte per block, {list(lead)} rows of them, on {dev}")
    nb = -(-K // _BLOCK[fmt])
    if K <= 0 or codes.shape[-1] < (K + 1) // 2 or scales.shape[-1] < nb:
        raise _err(f"K = {K} needs {(K + 1) // 2} code bytes and {nb} scales a row")
    if len(lead) == 2 and lead[0] > MX_MAX_GROUPS:
        raise _err(f"at most {MX_MAX_GROUPS} experts, got {lead[0]}")
    G, N = (1, lead[0]) if len(lead) == 1 else lead
    rb = _row_bytes(K)
    flat = codes.reshape(G * N, codes.shape[-1])
    if K % 32 or flat.shape[1] != rb or not flat.is_contiguous() or flat.data_ptr() % 16:
        full = torch.zeros((G * N, rb), dtype=torch.uint8, device=dev)
        full[:, :(K + 1) // 2] = flat[:, :(K + 1) // 2]
        if K % 2:
            full[:, K // 2] &= 15
        flat = full
    s = scales.view(torch.uint8).reshape(G * N, -1)[:, :nb].contiguous()
    atoms = torch.empty((_scale_bytes(fmt, N * G, K, G if len(lead) == 2 else 0, N if len(lead) == 2 else 0),),
                        dtype=torch.uint8, device=dev)
    _launch(dev, "lb_mx_scales", f, s.data_ptr(), nb, G, N, K, atoms.data_ptr(), 1)
    t = _tensor_scale(fmt, 1.0 if tensor_scale is None and fmt == "nvfp4" else tensor_scale, dev)
    return MxTensor(fmt, lead + (K,), flat, atoms, t)


def plain_scales(q):
    """The scale bytes of an ``MxTensor`` in rows: uint8 [..., rows, blocks] (not for ragged groups)."""
    if q.offsets is not None:
        raise _err("ragged groups have no plain scales: quantise without offsets")
    G, N = (1, q.shape[0]) if len(q.shape) == 2 else q.shape[:2]
    K, nb = q.shape[-1], -(-q.shape[-1] // _BLOCK[q.fmt])
    out = torch.empty((*q.shape[:-1], nb), dtype=torch.uint8, device=q.device)
    if out.numel():
        _launch(q.device, "lb_mx_scales", MICROSCALED_FMT[q.fmt], out.data_ptr(), nb, G, N, K, q.scales.data_ptr(), 0)
    return out


def _output(out, M, N, dev, accumulate):
    if out is None:
        if accumulate:
            raise _err("accumulate needs an output tensor")
        return torch.empty((M, N), dtype=torch.bfloat16, device=dev), N
    if not isinstance(out, torch.Tensor) or out.device != dev or out.dtype != torch.bfloat16:
        raise _err(f"out must be a bfloat16 tensor on {dev}")
    if out.dim() != 2 or out.shape[0] != M or out.shape[1] != N or (out.stride(1) != 1 and N > 1):
        raise _err(f"out must be [{M}, {N}] with unit column stride")
    ld = out.stride(0) if M > 1 else N
    if ld < N:
        raise _err("the rows of out overlap")
    return out, ld


def _bias(bias, n, dev):
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.device != dev or bias.dtype != torch.bfloat16
                             or bias.numel() != n or not bias.is_contiguous()):
        raise _err(f"bias must be a contiguous bfloat16 tensor of {n} values on {dev}")
    return bias


def linear(x, w, bias=None, out=None, accumulate=False, tensor_scale=None):
    """y = x . w^T (+ bias) (+ out if accumulate), bfloat16 [M, N], float32 accumulation, over the values the codes stand for.

    ``w``: an ``MxTensor`` [N, K].  ``x``: an ``MxTensor`` [M, K] of the same format, or float values [..., K], which
    are quantised to it first (nvfp4: with ``tensor_scale``, else the one ``quantize`` finds); y then has x's leading sizes."""
    if not isinstance(w, MxTensor) or len(w.shape) != 2 or w.offsets is not None:
        raise _err("w must be an MxTensor [N, K]")
    lead = None
    if not isinstance(x, MxTensor):
        _cuda(x, "x")
        lead = x.shape[:-1]
        x = quantize(x.reshape(-1, x.shape[-1]), w.fmt, tensor_scale)
    if x.fmt != w.fmt or len(x.shape) != 2 or x.offsets is not None or x.shape[1] != w.shape[1] or x.device != w.device:
        raise _err(f"x must be {w.fmt} [M, {w.shape[1]}] in one group on {w.device}, got {x}")
    (M, K), N, dev = x.shape, w.shape[0], w.codes.device
    y, ld = _output(out, M, N, dev, accumulate)
    _launch(dev, "lb_mx_linear", MICROSCALED_FMT[w.fmt], x.codes.data_ptr(), x.scales.data_ptr(), _ptr(x.tensor_scale), M, K,
            w.codes.data_ptr(), w.scales.data_ptr(), _ptr(w.tensor_scale), N, _ptr(_bias(bias, N, dev)), 1 if accumulate else 0,
            y.data_ptr(), ld)
    return y if lead is None or out is not None else y.view(*lead, N)


def linear_grouped(x, w, bias=None, out=None, accumulate=False):
    """y[r] = x[r] . w[e]^T (+ bias[e]) for the rows r of group e: bfloat16 [R, N].

    ``x``: an ``MxTensor`` [R, K] quantised with ``offsets`` of E groups; ``w``: [E, N, K] of the same format; ``bias``
    [E, N].  Rows that lie in no group are not written."""
    if not isinstance(w, MxTensor) or len(w.shape) != 3:
        raise _err("w must be an MxTensor [E, N, K]")
    E, N, K = w.shape
    if (not isinstance(x, MxTensor) or x.fmt != w.fmt or x.offsets is None or x.shape[1] != K or x.device != w.device
            or x.offsets.numel() != E + 1):
        raise _err(f"x must be an MxTensor {w.fmt} [R, {K}] on {w.device} quantised with the offsets of {E} groups, got {x}")
    M, dev = x.shape[0], w.codes.device
    y, ld = _output(out, M, N, dev, accumulate)
    _launch(dev, "lb_mx_linear_grouped", MICROSCALED_FMT[w.fmt], x.codes.data_ptr(), x.scales.data_ptr(), _ptr(x.tensor_scale), M, K,
            x.offsets.data_ptr(), E, w.codes.data_ptr(), w.scales.data_ptr(), _ptr(w.tensor_scale), N, _ptr(_bias(bias, E * N, dev)),
            1 if accumulate else 0, y.data_ptr(), ld)
    return y
