"""Drop-in replacement for spikingbrain_cpu/quant.py on B200 (sm_100a).

Same public surface as the reference module: ``FORMATS``, ``quantize_per_channel``,
``Int8Linear(weight, bias, block=128)``, ``DynamicInt8Linear(weight, bias)``, the float formats
and ``make_linear(fmt, weight, bias=None)`` (quant.py:22-111).  Modules take the weight the
loader hands them (a CPU bf16/fp32 tensor, loader.py:49), quantise and pack it on the current
CUDA device once, and own the device buffers.  ``forward`` returns fp32 like the reference.

The ``int8`` and ``int8-dyn`` formats run only through libsbq.so (hand-written sm_100a kernels);
there is no CPU or PyTorch fallback for them.  A CPU input tensor is copied to the device, run
there and the result copied back, so the modules also work inside the reference's CPU model
loop; device inputs stay on the device with no host synchronisation.
"""

from __future__ import annotations

import ctypes

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib as L

FORMATS = ("float32", "bfloat16", "float16", "int8", "int8-dyn")
# 4-bit weights with one bf16 scale per group of 32, 64 or 128 input features (no reference counterpart):
# accepted by make_linear beside the reference's formats
INT4_FORMATS = ("int4-g32", "int4-g64", "int4-g128")
INT4_GROUPS = (32, 64, 128)

_DTYPE_CODE = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_ELEM = {torch.float32: 4, torch.float16: 2, torch.bfloat16: 2}


def _device(device=None) -> torch.device:
    if device is not None:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("int8 formats run on a CUDA device, got " + str(device))
        return device
    if not torch.cuda.is_available():
        raise RuntimeError("the int8 formats need a CUDA device (B200, sm_100a); none is available")
    return torch.device("cuda", torch.cuda.current_device())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _written(t: torch.Tensor) -> torch.Tensor:
    """t, after a kernel wrote to its address: counted as a change in place, as torch's own operations count theirs (a kept
    SharedInputGroup result, or a tensor saved for a gradient, goes by that count)."""
    torch._C._increment_version((t,))
    return t


def _ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def pack_weight(weight: torch.Tensor, device=None, rowsum: bool = False):
    """Quantise an [n, k] float weight per output channel on the device (quant.py:25-29) and pack it.

    Returns ``(packed, scale, rowsum)``: the packed int8 tiles (flat int8 tensor), the fp32
    per-row scales and, if asked for, the int32 row sums used by the int8-dyn epilogue.
    """
    dev = _device(device)
    if weight.dim() != 2:
        raise ValueError("weight must be 2-D [out_features, in_features], got shape %s" % (tuple(weight.shape),))
    w = weight.detach()
    if w.dtype not in _DTYPE_CODE:
        w = w.float()
    w = w.to(dev)
    if w.stride(1) != 1 or w.stride(0) < w.shape[1]:
        w = w.contiguous()
    n, k = w.shape
    packed = torch.empty(L.packed_bytes(n, k), dtype=torch.int8, device=dev)
    scale = torch.empty(n, dtype=torch.float32, device=dev)
    rs = torch.empty(n, dtype=torch.int32, device=dev) if rowsum else None
    L.call("sbq_quantize_pack", _ptr(w), _DTYPE_CODE[w.dtype], n, k, w.stride(0), _ptr(packed), _ptr(scale),
           _ptr(rs), _stream(dev))
    return packed, scale, rs


def pack_int8(q: torch.Tensor, device=None, rowsum: bool = False):
    """Pack an already-quantised int8 [n, k] weight (e.g. a ``qweight`` from a state dict)."""
    dev = _device(device)
    if q.dim() != 2 or q.dtype != torch.int8:
        raise ValueError("qweight must be a 2-D int8 tensor")
    q = q.to(dev).contiguous()
    n, k = q.shape
    packed = torch.empty(L.packed_bytes(n, k), dtype=torch.int8, device=dev)
    rs = torch.empty(n, dtype=torch.int32, device=dev) if rowsum else None
    L.call("sbq_pack_int8", _ptr(q), n, k, k, _ptr(packed), _ptr(rs), _stream(dev))
    return packed, rs


def unpack_int8(packed: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """Packed tiles -> row-major int8 [n, k] on the same device."""
    q = torch.empty(n, k, dtype=torch.int8, device=packed.device)
    L.call("sbq_unpack_int8", _ptr(packed), n, k, _ptr(q), k, _stream(packed.device))
    return q


def quantize_per_channel(weight: torch.Tensor, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """quant.py:25-29 computed on the device: ``(q int8 [n, k], scale fp32 [n])``, bit-identical."""
    packed, scale, _ = pack_weight(weight, device)
    return unpack_int8(packed, *weight.shape), scale


def _workspace(m: int, k: int, x_dtype: torch.dtype, device: torch.device):
    """(workspace tensor or None, bytes) for the int8 format's fp32 prefill path (sbq_linear_w8_ws):
    the bf16 high / low parts of x, taken from torch's caching allocator (no device sync)."""
    nbytes = int(L.load().sbq_linear_w8_workspace_bytes(m, k, _DTYPE_CODE[x_dtype]))
    if nbytes == 0:
        return None, 0
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def _prepare_x(x: torch.Tensor, k: int, device: torch.device):
    """Flatten x to [m, k'] on the device with 16-byte aligned rows; k' is k rounded up to 16."""
    if x.shape[-1] != k:
        raise ValueError("input feature size %d does not match the weight's %d" % (x.shape[-1], k))
    on_host = x.device.type != "cuda"
    xd = x.to(device, non_blocking=True) if on_host or x.device != device else x
    if xd.dtype not in _DTYPE_CODE:
        xd = xd.float()
    x2 = xd.reshape(-1, k)
    k16 = (k + 15) // 16 * 16
    if k16 != k:
        x2 = F.pad(x2, (0, k16 - k))
    elif (x2.stride(-1) != 1 or (x2.stride(0) * _ELEM[x2.dtype]) % 16 or x2.data_ptr() % 16) and x2.shape[0] > 0:
        x2 = x2.contiguous()
    return x2, k16, on_host


class _PackedLinear(nn.Module):
    """Common state handling: device-packed weight, reference-compatible state dict keys."""

    def _init_packed(self, weight: torch.Tensor, bias: torch.Tensor | None, device, rowsum: bool):
        dev = _device(device)
        packed, scale, rs = pack_weight(weight, dev, rowsum=rowsum)
        self.out_features, self.in_features = int(weight.shape[0]), int(weight.shape[1])
        self.register_buffer("packed", packed, persistent=False)
        self.register_buffer("scale", scale)
        if rowsum:
            self.register_buffer("rowsum", rs, persistent=False)
        else:
            self.rowsum = None
        self.bias = None if bias is None else nn.Parameter(bias.detach().float().to(dev), requires_grad=False)

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scale: torch.Tensor, rowsum: torch.Tensor | None, out_features: int,
                    in_features: int, bias: torch.Tensor | None = None, **attrs):
        """A module around weights already quantised and packed on the device (e.g. by
        ``loader.StreamingPacker``); the buffers are adopted, not copied."""
        if packed.numel() != L.packed_bytes(out_features, in_features) or scale.numel() != out_features:
            raise ValueError("packed buffers do not match a [%d, %d] weight" % (out_features, in_features))
        mod = cls.__new__(cls)
        nn.Module.__init__(mod)
        mod.out_features, mod.in_features = int(out_features), int(in_features)
        mod.register_buffer("packed", packed, persistent=False)
        mod.register_buffer("scale", scale)
        if rowsum is not None:
            mod.register_buffer("rowsum", rowsum, persistent=False)
        else:
            mod.rowsum = None
        dev = scale.device
        mod.bias = None if bias is None else nn.Parameter(bias.detach().float().to(dev), requires_grad=False)
        for k_, v in attrs.items():
            setattr(mod, k_, v)
        return mod

    @property
    def qweight(self) -> torch.Tensor:
        """Row-major int8 [out, in] view of the packed weight (the reference's ``qweight`` buffer)."""
        return unpack_int8(self.packed, self.out_features, self.in_features)

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "qweight"] = self.qweight

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        key = prefix + "qweight"
        q = state_dict.get(key)
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)
        if key in unexpected_keys:
            unexpected_keys.remove(key)
        if q is None:
            if strict:
                missing_keys.append(key)
            return
        if tuple(q.shape) != (self.out_features, self.in_features):
            error_msgs.append("size mismatch for %s: %s != %s" % (key, tuple(q.shape),
                                                                  (self.out_features, self.in_features)))
            return
        packed, rs = pack_int8(q, self.packed.device, rowsum=self.rowsum is not None)
        self.packed.copy_(packed)
        if rs is not None:
            self.rowsum.copy_(rs)

    def extra_repr(self) -> str:
        return "in_features=%d, out_features=%d, bias=%s" % (self.in_features, self.out_features, self.bias is not None)


class Int8Linear(_PackedLinear):
    """Format ``int8``: symmetric per-output-channel int8 weight, fp32 scale epilogue (quant.py:32-53).

    ``block`` is accepted for signature compatibility; the device kernels do not dequantise the
    weight into fp32 blocks.  ``out_dtype`` may be set to ``torch.float16`` for the fp16-output
    prefill configuration; the default matches the reference (fp32).
    """

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, block: int = 128, device=None):
        super().__init__()
        self._init_packed(weight, bias, device, rowsum=False)
        self.block = block
        self.out_dtype = torch.float32

    def forward_into(self, x2: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """Low-level device call: x2 [m, k'] (k' = in_features rounded up to 16, 16-byte aligned rows)
        into ``out`` [m, out_features] (fp32 or fp16, unit column stride, any row stride)."""
        m, n = x2.shape[0], self.out_features
        if out.shape != (m, n) or out.stride(1) != 1 or out.dtype not in (torch.float32, torch.float16):
            raise ValueError("output must be an fp32/fp16 [%d, %d] view with unit column stride" % (m, n))
        if m > 0:
            ws, ws_bytes = _workspace(m, x2.shape[1], x2.dtype, out.device)
            L.call("sbq_linear_w8_ws", _ptr(x2), _DTYPE_CODE[x2.dtype], x2.stride(0), _ptr(self.packed),
                   _ptr(self.scale), _ptr(self.bias), m, n, x2.shape[1], _ptr(out),
                   L.F32 if out.dtype == torch.float32 else L.F16, out.stride(0), _ptr(ws), ws_bytes,
                   _stream(out.device))
        return _written(out)

    def gemv_job(self, x2: torch.Tensor, out: torch.Tensor) -> L.GemvJob:
        """This projection as one job of a grouped decode launch (see ``gemv_group``)."""
        return L.GemvJob(x2.data_ptr(), x2.stride(0), self.packed.data_ptr(), self.scale.data_ptr(), None, None,
                         None if self.bias is None else self.bias.data_ptr(), self.out_features, x2.shape[1],
                         out.data_ptr(), L.F32 if out.dtype == torch.float32 else L.F16, out.stride(0))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        dev = self.scale.device
        x2, _, on_host = _prepare_x(x, self.in_features, dev)
        out = torch.empty(x2.shape[0], self.out_features, dtype=self.out_dtype, device=dev)
        self.forward_into(x2, out)
        out = out.reshape(*shape[:-1], self.out_features)
        return out.to("cpu") if on_host else out


def gemv_group(jobs, x_dtype: torch.dtype, m: int, device: torch.device, n_ready: int = 0) -> None:
    """Run several decode projections (``Int8Linear.gemv_job`` / ``FusedGatedMLP.gateup_job``) in one
    launch: up to 8 jobs, all with ``m`` <= 16 rows of x of dtype ``x_dtype``.  The first ``n_ready``
    jobs read inputs written two or more launches back and run without waiting for the previous
    launch (sbq_gemv_w8_group_ready: the previous kernel must be a grouped GEMV launch)."""
    arr = (L.GemvJob * len(jobs))(*jobs)
    if n_ready:
        L.call("sbq_gemv_w8_group_ready", arr, len(jobs), n_ready, _DTYPE_CODE[x_dtype], m, _stream(device))
    else:
        L.call("sbq_gemv_w8_group", arr, len(jobs), _DTYPE_CODE[x_dtype], m, _stream(device))


class DynamicInt8Linear(_PackedLinear):
    """Format ``int8-dyn`` (quant.py:56-66): activations quantised at run time, int8 x int8 -> int32.

    ``mode="per_tensor"`` (default) reproduces the reference bit for bit: fbgemm's per-tensor
    uint8 quantisation with a zero point, int32 accumulation and the fp32 epilogue.
    ``mode="per_token"`` is the symmetric per-row variant (no reference counterpart).
    """

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, mode: str = "per_tensor", device=None):
        super().__init__()
        if mode not in ("per_tensor", "per_token"):
            raise ValueError("unknown activation quantisation mode " + mode)
        self._init_packed(weight, bias, device, rowsum=True)
        self.mode = mode

    @property
    def _mode_code(self) -> int:
        return L.ACT_PER_TENSOR if self.mode == "per_tensor" else L.ACT_PER_TOKEN

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        shape = x.shape
        dev = self.scale.device
        x2, k16, on_host = _prepare_x(x, self.in_features, dev)
        m, n = x2.shape[0], self.out_features
        out = torch.empty(m, n, dtype=torch.float32, device=dev)
        if m > 0:
            lib = L.load()
            ws_bytes = int(lib.sbq_dyn_workspace_bytes(m, k16, self._mode_code))
            ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
            L.call("sbq_linear_dyn", _ptr(x2), _DTYPE_CODE[x2.dtype], x2.stride(0), self._mode_code,
                   _ptr(self.packed), _ptr(self.rowsum), _ptr(self.scale), _ptr(self.bias), m, n, k16, _ptr(out), n,
                   _ptr(ws), ws_bytes, _stream(dev))
        out = out.reshape(*shape[:-1], n)
        return out.to("cpu") if on_host else out

    def forward_stages(self, x: torch.Tensor):
        """The integer stages separately: ``(y, xq, s, zp, acc)`` (per-token: ``(y, xq, s_tok, None, acc)``).

        Runs the two kernels of ``forward`` through their own entry points and also returns the
        quantised activation, its parameters and the int32 accumulators for bit-exact checks.
        """
        dev = self.scale.device
        x2, k16, _ = _prepare_x(x, self.in_features, dev)
        m, n = x2.shape[0], self.out_features
        st = _stream(dev)
        lib = L.load()
        acc = torch.empty(m, n, dtype=torch.int32, device=dev)
        y = torch.empty(m, n, dtype=torch.float32, device=dev)
        if self.mode == "per_tensor":
            xq = torch.empty(m, k16, dtype=torch.uint8, device=dev)
            s = torch.empty(1, dtype=torch.float32, device=dev)
            zp = torch.empty(1, dtype=torch.int32, device=dev)
            ws_bytes = int(lib.sbq_dyn_workspace_bytes(m, k16, L.ACT_PER_TENSOR))
            ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
            L.call("sbq_quant_act_per_tensor", _ptr(x2), _DTYPE_CODE[x2.dtype], x2.stride(0), m, k16, _ptr(xq),
                   _ptr(s), _ptr(zp), _ptr(ws), ws_bytes, st)
        else:
            xq = torch.empty(m, k16, dtype=torch.int8, device=dev)
            s = torch.empty(m, dtype=torch.float32, device=dev)
            zp = None
            L.call("sbq_quant_act_per_token", _ptr(x2), _DTYPE_CODE[x2.dtype], x2.stride(0), m, k16, _ptr(xq),
                   _ptr(s), st)
        L.call("sbq_gemm_w8a8", _ptr(xq), self._mode_code, _ptr(self.packed), _ptr(self.rowsum), _ptr(s), _ptr(zp),
               _ptr(self.scale), _ptr(self.bias), m, n, k16, _ptr(y), n, _ptr(acc), st)
        return y, xq[:, :self.in_features], s, zp, acc


# ---- format int4: 4-bit weights with group scales ------------------------------------------------

def _check_group(group: int) -> int:
    if group not in INT4_GROUPS:
        raise ValueError("group size must be one of %s, got %s" % (INT4_GROUPS, group))
    return int(group)


def _int4_buffers(n: int, k: int, group: int, dev: torch.device):
    lib = L.load()
    return (torch.empty(int(lib.sbq_w4_packed_bytes(n, k)), dtype=torch.uint8, device=dev),
            torch.empty(int(lib.sbq_w4_scale_bytes(n, k, group)), dtype=torch.uint8, device=dev),
            # fp32 powers of two, held as their bits: a module's .half() or .to(dtype) leaves integer buffers alone
            torch.empty((n + 15) // 16 * 16, dtype=torch.int32, device=dev))


def _check_int4_buffers(n: int, k: int, group: int, packed: torch.Tensor, scales: torch.Tensor,
                        rowmul: torch.Tensor | None = None) -> int:
    """The group size, if the buffers are those of an [n, k] weight on one CUDA device: the kernels read by n, k and group."""
    lib, group = L.load(), _check_group(group)
    bufs = [(packed, int(lib.sbq_w4_packed_bytes(n, k)), torch.uint8), (scales, int(lib.sbq_w4_scale_bytes(n, k, group)), torch.uint8)]
    if rowmul is not None:
        bufs.append((rowmul, (n + 15) // 16 * 16, torch.int32))
    if any(size == 0 or t.numel() != size or t.dtype != dtype or not t.is_contiguous() for t, size, dtype in bufs):
        raise ValueError("packed buffers do not match a [%d, %d] weight in groups of %d" % (n, k, group))
    if any(not t.is_cuda or t.device != packed.device for t, _, _ in bufs):
        raise ValueError("packed buffers must be on one CUDA device")
    return group


def pack_weight_int4(weight: torch.Tensor, group: int = 128, device=None):
    """Quantise an [n, k] float weight per output channel and group of ``group`` inputs on the device, packed.

    ``s = bf16(max(max|w|, 1e-8) / 7)``, ``q = clamp(rint(w / s), -7, 7)``; a group with an infinity or a NaN
    gets the scale NaN.  Returns ``(packed, scales, rowmul)``, the three device buffers the 4-bit kernels read.
    """
    dev = _device(device)
    group = _check_group(group)
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError("weight must be 2-D [out_features, in_features], got shape %s" % (tuple(weight.shape),))
    w = weight.detach()
    if w.dtype not in _DTYPE_CODE:
        w = w.float()
    w = w.to(dev)
    if w.stride(1) != 1 or w.stride(0) < w.shape[1]:
        w = w.contiguous()
    n, k = w.shape
    bufs = _int4_buffers(n, k, group, dev)
    with torch.cuda.device(dev):
        L.call("sbq_w4_quantize_pack", _ptr(w), _DTYPE_CODE[w.dtype], n, k, w.stride(0), group, *map(_ptr, bufs), _stream(dev))
    return bufs


def pack_int4(q: torch.Tensor, scale: torch.Tensor, group: int = 128, device=None):
    """Pack given codes (int8 [n, k], values in [-8, 7]) and bf16 scales [n, ceil(k / group)].

    The scales are taken as they are: they must be finite bf16 (round others yourself, so that the codes
    fit the scales that are stored).  Returns the buffers of ``pack_weight_int4``.
    """
    dev = _device(device)
    group = _check_group(group)
    if q.dim() != 2 or q.dtype != torch.int8 or q.numel() == 0:
        raise ValueError("codes must be a 2-D int8 tensor")
    n, k = q.shape
    if scale.dtype != torch.bfloat16 or tuple(scale.shape) != (n, -(-k // group)):
        raise ValueError("scales must be bf16 [%d, %d], got %s %s" % (n, -(-k // group), scale.dtype, tuple(scale.shape)))
    q, scale = q.to(dev).contiguous(), scale.to(dev).contiguous()
    lo, hi = (int(v) for v in torch.aminmax(q))
    if lo < -8 or hi > 7:
        raise ValueError("codes must lie in [-8, 7], got [%d, %d]" % (lo, hi))
    if not bool(torch.isfinite(scale).all()):
        raise ValueError("scales must be finite")
    bufs = _int4_buffers(n, k, group, dev)
    with torch.cuda.device(dev):
        L.call("sbq_w4_pack", _ptr(q), k, _ptr(scale), scale.shape[1], n, k, group, *map(_ptr, bufs), _stream(dev))
    return bufs


def unpack_int4(packed: torch.Tensor, scales: torch.Tensor, n: int, k: int, group: int):
    """Packed buffers -> ``(q int8 [n, k], scale bf16 [n, ceil(k / group)])`` on the same device."""
    group = _check_int4_buffers(n, k, group, packed, scales)
    dev = packed.device
    q = torch.empty(n, k, dtype=torch.int8, device=dev)
    scale = torch.empty(n, -(-k // group), dtype=torch.bfloat16, device=dev)
    with torch.cuda.device(dev):
        L.call("sbq_w4_unpack", _ptr(packed), _ptr(scales), n, k, group, _ptr(q), k, _ptr(scale), scale.shape[1], _stream(dev))
    return q, scale


def quantize_per_group(weight: torch.Tensor, group: int = 128, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q int8 [n, k], scale bf16 [n, ceil(k / group)])`` of the ``int4`` formats, computed on the device."""
    packed, scales, _ = pack_weight_int4(weight, group, device)
    return unpack_int4(packed, scales, *weight.shape, group)


def _raw_stream(device: torch.device) -> int:
    """The current stream's handle (torch.cuda.current_stream builds an object for it: 2 us of a 9 us call)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _in_place(x: torch.Tensor, k: int, device: torch.device) -> bool:
    """Whether the library takes x [..., k] where it is, as a decode loop passes it."""
    return x.dtype in _DTYPE_CODE and x.dim() > 0 and x.shape[-1] == k and x.device == device and x.is_contiguous() \
        and (x.data_ptr() % 16 == 0 or k % 16 != 0)


class Int4Linear(nn.Module):
    """Formats ``int4-g32`` / ``int4-g64`` / ``int4-g128``: 4-bit weight, one bf16 scale per output channel and
    group of input features; y = x (q * s)^T + b.

    x may be fp32, fp16 or bf16 (fp32 enters the product with 22 bits, the others exactly; elements of fp32 rows,
    and of bf16 rows when there are more than 16, keep an absolute 2^-39 of their row's largest), products are
    summed in fp32, and ``out_dtype`` (fp32 as in the other formats, or fp16 / bf16) is the type of the
    result.  Frozen like every format here: no gradient and no forward-mode tangent flows through it.  State dicts hold ``qweight``
    (int8 codes [n, k]) and ``scale`` (bf16 [n, ceil(k / group)]); both are copies of the packed weight, so
    writing into them does not change it (load a state dict, or pack anew).
    """

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, group: int = 128, device=None):
        super().__init__()
        self._adopt(pack_weight_int4(weight, group, device), weight.shape, bias, group)

    def _adopt(self, bufs, shape, bias, group: int) -> None:
        packed, scales, rowmul = bufs
        self.out_features, self.in_features, self.group = int(shape[0]), int(shape[1]), int(group)
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError("bias must have shape (%d,), got %s" % (self.out_features, tuple(bias.shape)))
        self.register_buffer("packed", packed, persistent=False)
        self.register_buffer("scales", scales, persistent=False)
        self.register_buffer("rowmul", rowmul, persistent=False)
        self.bias = None if bias is None else nn.Parameter(bias.detach().float().to(packed.device).contiguous(), requires_grad=False)
        self.out_dtype = torch.float32

    @classmethod
    def from_packed(cls, packed: torch.Tensor, scales: torch.Tensor, rowmul: torch.Tensor, out_features: int,
                    in_features: int, bias: torch.Tensor | None = None, group: int = 128):
        """A module around buffers of ``pack_weight_int4`` / ``pack_int4``; they are adopted, not copied."""
        group = _check_int4_buffers(out_features, in_features, group, packed, scales, rowmul)
        mod = cls.__new__(cls)
        nn.Module.__init__(mod)
        mod._adopt((packed, scales, rowmul), (out_features, in_features), bias, group)
        # the products read the weight before they wait for the kernel before them: this one stands between them and a
        # kernel that has just written the buffers
        torch.zeros(1, device=packed.device)
        return mod

    @classmethod
    def from_quantized(cls, q: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, group: int = 128,
                       device=None):
        """A module of given codes (int8 [n, k] in [-8, 7]) and bf16 scales [n, ceil(k / group)]."""
        return cls.from_packed(*pack_int4(q, scale, group, device), q.shape[0], q.shape[1], bias, group)

    @property
    def qweight(self) -> torch.Tensor:
        """The codes, int8 [out, in] (a copy)."""
        return unpack_int4(self.packed, self.scales, self.out_features, self.in_features, self.group)[0]

    @property
    def scale(self) -> torch.Tensor:
        """The group scales, bf16 [out, ceil(in / group)] (a copy)."""
        return unpack_int4(self.packed, self.scales, self.out_features, self.in_features, self.group)[1]

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "qweight"], destination[prefix + "scale"] = unpack_int4(
            self.packed, self.scales, self.out_features, self.in_features, self.group)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        keys = (prefix + "qweight", prefix + "scale")
        q, scale = (state_dict.get(key) for key in keys)
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)
        for key in keys:
            if key in unexpected_keys:
                unexpected_keys.remove(key)
        if q is None or scale is None:
            if strict:
                missing_keys.extend(key for key, v in zip(keys, (q, scale)) if v is None)
            return
        want = ((self.out_features, self.in_features), (self.out_features, -(-self.in_features // self.group)))
        if (tuple(q.shape), tuple(scale.shape)) != want:
            error_msgs.append("size mismatch for %s: %s, %s != %s, %s" % (prefix + "qweight / scale", tuple(q.shape),
                                                                          tuple(scale.shape), *want))
            return
        try:
            bufs = pack_int4(q, scale, self.group, self.packed.device)
        except ValueError as e:
            error_msgs.append("%s: %s" % (prefix + "qweight / scale", e))
            return
        for dst, src in zip((self.packed, self.scales, self.rowmul), bufs):
            dst.copy_(src)

    def forward_into(self, x2: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        """Low-level device call: x2 [m, in_features] (16-byte aligned rows if in_features is a multiple of 16)
        into ``out`` [m, out_features] (fp32, fp16 or bf16, unit column stride, any row stride)."""
        m, n = x2.shape[0], self.out_features
        if out.shape != (m, n) or (out.stride(1) != 1 and n > 1) or out.dtype not in _DTYPE_CODE:
            raise ValueError("output must be an fp32/fp16/bf16 [%d, %d] view with unit column stride" % (m, n))
        k = self.in_features
        if x2.shape[1] != k or (x2.stride(1) != 1 and k > 1) or x2.dtype not in _DTYPE_CODE:
            raise ValueError("input must be an fp32/fp16/bf16 [m, %d] view with unit column stride" % k)
        dev = self._buffers["packed"].device
        if x2.device != dev or out.device != dev:
            raise ValueError("input and output must be on the weight's device %s" % dev)
        self._run(x2, m, k, x2.stride(0) if m > 1 else k, out, out.stride(0) if m > 1 else n, dev)
        return _written(out)

    def _run(self, x: torch.Tensor, m: int, k: int, ldx: int, out: torch.Tensor, ldy: int, dev: torch.device) -> None:
        if m == 0:
            return
        if dev.index != torch._C._cuda_getDevice():  # the library launches on the current device
            with torch.cuda.device(dev):
                return self._run(x, m, k, ldx, out, ldy, dev)
        b, code, bias = self._buffers, _DTYPE_CODE[x.dtype], self._parameters.get("bias")
        if bias is not None and bias.dtype != torch.float32:  # a module converted with .half() or .to(dtype)
            bias = bias.float()
        ws, ws_bytes = _int4_workspace(m, self.out_features, k, code, 1, dev)
        status = L.load().sbq_linear_w4(
            x.data_ptr(), code, ldx, b["packed"].data_ptr(), b["scales"].data_ptr(), b["rowmul"].data_ptr(), self.group,
            None if bias is None else bias.data_ptr(), m, self.out_features, k, out.data_ptr(), _DTYPE_CODE[out.dtype], ldy,
            None if ws is None else ws.data_ptr(), ws_bytes, _raw_stream(dev))
        if status:
            L.check(status, "sbq_linear_w4")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        k, n, dev = self.in_features, self.out_features, self._buffers["packed"].device
        if _in_place(x, k, dev):
            out = torch.empty(*x.shape[:-1], n, dtype=self.out_dtype, device=dev)  # 0.9 us less than new_empty
            self._run(x, x.numel() // k, k, k, out, n, dev)
            return out
        x2, on_host = _int4_rows(x, k, dev)
        out = self.forward_into(x2, torch.empty(x2.shape[0], n, dtype=self.out_dtype, device=dev))
        out = out.view(*x.shape[:-1], n)
        return out.to("cpu") if on_host else out

    def extra_repr(self) -> str:
        return "in_features=%d, out_features=%d, bias=%s, group=%d" % (self.in_features, self.out_features,
                                                                       self.bias is not None, self.group)


def _int4_rows(x: torch.Tensor, k: int, device: torch.device):
    """x flattened to rows [m, k] as the 4-bit calls take them, and whether it came from the host."""
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError("input feature size %s does not match the weight's %d" % (x.shape[-1] if x.dim() else "()", k))
    on_host = x.device.type != "cuda"
    xd = x if x.device == device else x.to(device, non_blocking=True)
    if xd.dtype not in _DTYPE_CODE:
        xd = xd.float()
    x2 = xd.reshape(-1, k)
    if x2.shape[0] and ((x2.stride(1) != 1 and k > 1) or (x2.shape[0] > 1 and x2.stride(0) < k) or
                        (k % 16 == 0 and (x2.data_ptr() % 16 or (x2.shape[0] > 1 and x2.stride(0) * _ELEM[x2.dtype] % 16)))):
        x2 = x2.contiguous() if x2.data_ptr() % 16 == 0 or not x2.is_contiguous() else x2.clone()
    return x2, on_host


def _int4_workspace(m: int, n: int, k: int, x_code: int, matrices: int, device: torch.device):
    """(tensor or None, bytes) of a 4-bit call's workspace, from torch's caching allocator."""
    if m <= 16 and x_code != L.F32 and k % 16 == 0:
        return None, 0
    nbytes = L.load().sbq_linear_w4_workspace_bytes(m, n, k, x_code, matrices)
    return (torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes) if nbytes else (None, 0)


# ---- float formats (outside the int8 hot path; cuBLAS through torch, fp32 results) ----------

class FP16Linear(nn.Module):
    """Format ``float16`` (quant.py:69-77): fp16 weights, fp32 activations and output."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, device=None):
        super().__init__()
        dev = _device(device)
        self.register_buffer("weight", weight.detach().to(dev, torch.float16).contiguous())
        self.bias = None if bias is None else nn.Parameter(bias.detach().float().to(dev), requires_grad=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        on_host = x.device.type != "cuda"
        xd = x.to(self.weight.device).float()
        out = torch.matmul(xd, self.weight.t().float())
        if self.bias is not None:
            out = out + self.bias
        return out.to("cpu") if on_host else out


class BF16Linear(nn.Module):
    """Format ``bfloat16`` (quant.py:80-87)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, device=None):
        super().__init__()
        dev = _device(device)
        self.register_buffer("weight", weight.detach().to(dev, torch.bfloat16).contiguous())
        self.bias = None if bias is None else nn.Parameter(bias.detach().to(dev, torch.bfloat16), requires_grad=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        on_host = x.device.type != "cuda"
        out = F.linear(x.to(self.weight.device, torch.bfloat16), self.weight, self.bias).float()
        return out.to("cpu") if on_host else out


class FloatLinear(nn.Module):
    """Format ``float32`` (quant.py:90-97)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, device=None):
        super().__init__()
        dev = _device(device)
        self.register_buffer("weight", weight.detach().to(dev, torch.float32).contiguous())
        self.bias = None if bias is None else nn.Parameter(bias.detach().float().to(dev), requires_grad=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        on_host = x.device.type != "cuda"
        out = F.linear(x.to(self.weight.device).float(), self.weight, self.bias)
        return out.to("cpu") if on_host else out


def make_linear(fmt: str, weight: torch.Tensor, bias: torch.Tensor | None = None) -> nn.Module:
    """quant.py:100-111: format string -> module; ``ValueError`` for an unknown format.  Beside the
    reference's formats it takes ``INT4_FORMATS``."""
    if fmt == "float32":
        return FloatLinear(weight, bias)
    if fmt == "bfloat16":
        return BF16Linear(weight, bias)
    if fmt == "float16":
        return FP16Linear(weight, bias)
    if fmt == "int8":
        return Int8Linear(weight, bias)
    if fmt == "int8-dyn":
        return DynamicInt8Linear(weight, bias)
    if fmt in INT4_FORMATS:
        return Int4Linear(weight, bias, group=int(fmt[6:]))
    raise ValueError("unknown weight format " + fmt)
