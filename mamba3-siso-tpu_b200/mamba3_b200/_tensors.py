"""Tensor -> C-ABI plumbing shared by the kernel wrappers."""

from __future__ import annotations

import math
import weakref

import torch
from torch.autograd import forward_ad

from . import _capi as C


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_handle(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def require_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("the Mamba-3 SISO kernels run on CUDA tensors only (no CPU path)")


def io_dtype(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return C.M3_DTYPE_BF16
    if dt == torch.float32:
        return C.M3_DTYPE_F32
    raise ValueError(f"unsupported dtype {dt}; want bfloat16 or float32")


def policy_code(name) -> int:
    key = str(name).strip().lower()  # a name or a layout.DtypePolicy
    if key in ("bf16", "bfloat16", "default"):
        return C.M3_POLICY_BF16
    if key in ("f32", "fp32", "float32", "highest"):
        return C.M3_POLICY_F32
    raise ValueError(f"Unknown dtype policy {name!r}; want 'bf16' or 'f32'")


def f32c(t):
    """fp32, innermost-contiguous (outer strides are passed through)."""
    if t is None:
        return None
    if t.dtype != torch.float32:
        t = t.float()
    if t.dim() and t.stride(-1) != 1:
        t = t.contiguous()
    return t


_F32_CACHE = {}  # id(tensor) -> (weakref to it, its version, fp32 copy); tensors compare elementwise, so no WeakKeyDictionary


def f32dense(t):
    """fp32, dense.  Small tensors that need a conversion (per-head parameters held in bf16)
    are converted once and reused while their version is unchanged, so a decode step does
    not re-convert every layer's biases on every token."""
    if t is None:
        return None
    if t.dtype == torch.float32 and t.is_contiguous():
        return t
    if t.numel() <= (1 << 16) and not t.requires_grad:
        key = id(t)
        hit = _F32_CACHE.get(key)
        if hit is not None and hit[0]() is t and hit[1] == t._version:
            return hit[2]
        c = t.float().contiguous()
        if not (t.is_cuda and torch.cuda.is_current_stream_capturing()):
            _F32_CACHE[key] = (weakref.ref(t, lambda _r, k=key: _F32_CACHE.pop(k, None)), t._version, c)
        return c
    return t.float().contiguous()


def inner_contig(t, dtype):
    if t is None:
        return None
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.stride(-1) != 1:
        t = t.contiguous()
    return t


def st_bln(t) -> C.M3Strides:
    """(B, L, X) with contiguous X."""
    return C.M3Strides(t.stride(0), 0, t.stride(1))


def st_bhlp(t) -> C.M3Strides:
    return C.M3Strides(t.stride(0), t.stride(1), t.stride(2))


def st_blh(t) -> C.M3Strides:
    return C.M3Strides(t.stride(0), t.stride(2), t.stride(1))


def rows2(t, nd):
    """Element strides of the leading ``nd`` axes of ``t`` seen as two: (all but the last,
    the last).  None if the outer ones do not collapse into one stride."""
    if nd == 0:
        return 0, 0
    st = t.stride()
    if nd == 1:
        return 0, st[0]
    if nd == 2:
        return st[0], st[1]
    outer = [ss for ss in zip(t.shape[:nd - 1], st) if ss[0] != 1]
    for (_, st0), (s1, st1) in zip(outer, outer[1:]):
        if st0 != s1 * st1:
            return None
    return (outer[-1][1] if outer else 0), st[nd - 1]


def row_input(t, nd):
    """``t`` with its trailing axis (if any, beyond the ``nd`` leading ones) contiguous and its
    leading axes addressable by two strides, copied only where it is not, and those strides."""
    st = rows2(t, nd) if t.dim() == nd or t.stride(-1) == 1 or t.shape[-1] == 1 else None
    if st is None:
        t = t.detach().contiguous()
        st = rows2(t, nd)
    return t, st


def row_counts(lead):
    """(outer, inner) row counts of a leading shape, as `rows2` splits it."""
    inner = lead[-1] if lead else 1
    outer = 1
    for s in lead[:-1]:
        outer *= s
    if outer * inner > 1 << 30:
        raise ValueError(f"{outer * inner} rows: at most 2^30 are supported")
    return (outer, inner) if inner else (0, 1)


def vocab_of(n, most):
    """A vocabulary that the kernels' ints hold (a wider one would be cut to 32 bits on its way to them)."""
    if not 1 <= n <= most:
        raise ValueError(f"a vocabulary of {n}: from 1 to {most} are supported")
    return n


def require_here(device, *ts):
    """Every given tensor is on the CUDA device ``device``."""
    if device.type != "cuda":
        raise ValueError("the Mamba-3 SISO kernels run on CUDA tensors only (no CPU path)")
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError(f"every tensor must be on {device}, got one on {t.device}")


# the public torch.cuda.current_stream builds a Stream object per call, a tenth of a small call's cost
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def call(fn, args, device):
    """One library call on the current stream of ``device``; raises on a non-zero status."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = fn(args, stream_handle(device))
    else:
        rc = fn(args, _raw_stream(device.index) if _raw_stream else stream_handle(device))
    if rc:
        C.check(rc)


def no_tangent(name, t):
    """Refuses a dual tensor: `torch.autograd.forward_ad` marks it neither by requires_grad nor by its memory,
    and a kernel's result would come without the tangent."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def written(t):
    """Tells autograd that a kernel wrote to the caller's ``t``, so that a backward that saved its old values raises."""
    torch.autograd.graph.increment_version(t)


def _span(t):
    """Bytes from a tensor's first element to past its last."""
    return t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride())))


def apart(a, b) -> bool:
    """Two tensors with contiguous last axes have no byte in common (certainly: apart in memory, or column
    ranges of rows whose distances have a common divisor)."""
    if not a.numel() or not b.numel():
        return True
    d = b.data_ptr() - a.data_ptr()
    if d >= _span(a) or -d >= _span(b):
        return True
    pitch = math.gcd(*(st * t.element_size() for t in (a, b) for n, st in zip(t.shape[:-1], t.stride()) if n > 1))
    return pitch > 0 and a.shape[-1] * a.element_size() <= d % pitch <= pitch - b.shape[-1] * b.element_size()
