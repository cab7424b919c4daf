"""Python host binding of libsdb.so: the reference's op interface over the C ABI.

The reference (stable-diffusion.assembly) exposes its kernels to ggml as
operations on ggml tensors (sources/ops.h:26-62): mul_mat, the gated GELU
after it, conv2d (direct or Winograd), attention, group_norm and norm, each
with the chain of element-wise nodes fused after it (sources/fusion.h).
This module offers the same operations on CUDA tensors (torch is used only to
hold device memory and name a stream), described to the library in ggml's
terms: ne[] dimension 0 fastest, nb[] byte strides.  A torch tensor of shape
(d3, d2, d1, d0) is the ggml tensor ne = [d0, d1, d2, d3].

Errors are raised as SdbError with the library's status and message; a
status of NOT_SUPPORTED means the reference would leave the node to ggml.
There is no CPU fallback: without the built library every call raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
import weakref
from pathlib import Path
from typing import Iterable, Sequence

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "libsdb.so"

TYPE_F32 = 0
TYPE_F16 = 1
STEP_ADD, STEP_MUL, STEP_SILU = 0, 1, 2
MAX_STEPS = 6

OK, NOT_SUPPORTED, INVALID, CUDA_ERROR, OUT_OF_MEMORY, DEVICE_ERROR = range(6)
STATUS_NAMES = ["OK", "NOT_SUPPORTED", "INVALID", "CUDA_ERROR", "OUT_OF_MEMORY", "DEVICE_ERROR"]

# Exported symbols of include/sdb.h, checked by the tests.
EXPORTS = [
    "sdb_mul_mat_supported", "sdb_mul_mat", "sdb_mul_mat_transient", "sdb_mul_mat_gated_supported",
    "sdb_mul_mat_gated",
    "sdb_conv2d_supported", "sdb_conv2d", "sdb_attention_supported", "sdb_attention",
    "sdb_group_norm", "sdb_group_norm_no_alloc", "sdb_norm", "sdb_forget", "sdb_store_stats", "sdb_token_downsampling",
    "sdb_set_tuning", "sdb_get_tuning", "sdb_device_status", "sdb_last_error", "sdb_launch_count",
    "sdb_concat", "sdb_upscale_nearest", "sdb_timestep_embedding", "sdb_euler_cfg_step", "sdb_soft_max",
    "sdb_coarser_tokens", "sdb_euler_ancestral_cfg_step", "sdb_group_norm_stats", "sdb_conv2d_normed",
    "sdb_mul_mat_normed", "sdb_mul_mat_layer_normed", "sdb_mul_mat_gated_layer_normed",
    "sdb_q4_bytes", "sdb_q4_quantize", "sdb_q4_import", "sdb_q4_from_blocks", "sdb_q4_dequantize",
    "sdb_mul_mat_q4_supported", "sdb_mul_mat_q4", "sdb_mul_mat_q4_gated_supported", "sdb_mul_mat_q4_gated",
    "sdb_residual_norm",
]


class SdbError(RuntimeError):
    def __init__(self, status: int, message: str):
        self.status = status
        name = STATUS_NAMES[status] if 0 <= status < len(STATUS_NAMES) else str(status)
        super().__init__(f"{name}: {message}")


class Tensor(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("ne", ctypes.c_int64 * 4), ("nb", ctypes.c_int64 * 4),
                ("data", ctypes.c_void_p)]


class Step(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("operand", ctypes.c_void_p), ("nb", ctypes.c_int64 * 4)]


class NormIn(ctypes.Structure):
    _fields_ = [("stats", ctypes.c_void_p), ("gamma", ctypes.c_void_p), ("beta", ctypes.c_void_p),
                ("groups", ctypes.c_int32), ("silu", ctypes.c_int32)]


class ChainStruct(ctypes.Structure):
    _fields_ = [("count", ctypes.c_int32), ("steps", Step * MAX_STEPS), ("redirect", ctypes.c_void_p),
                ("from_redirect", ctypes.c_int32)]


_lib = None


def load(path: str | os.PathLike | None = None) -> ctypes.CDLL:
    """Loads libsdb.so (built by build.py); raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise SdbError(CUDA_ERROR, f"{p} is not built (run stable-diffusion.assembly_b200/build.py)")
    lib = ctypes.CDLL(str(p))
    T = ctypes.POINTER(Tensor)
    C = ctypes.POINTER(ChainStruct)
    vp = ctypes.c_void_p
    i = ctypes.c_int
    sigs = {
        "sdb_mul_mat_supported": (i, [T, T, T]),
        "sdb_mul_mat": (i, [T, T, T, C, vp]),
        "sdb_mul_mat_transient": (i, [T, T, T, C, vp]),
        "sdb_soft_max": (i, [T, T, ctypes.c_float, vp]),
        "sdb_mul_mat_gated_supported": (i, [T, T, T]),
        "sdb_mul_mat_gated": (i, [T, T, T, C, vp]),
        "sdb_conv2d_supported": (i, [T, T, T, ctypes.POINTER(ctypes.c_int32)]),
        "sdb_conv2d": (i, [T, T, T, ctypes.POINTER(ctypes.c_int32), C, vp]),
        "sdb_attention_supported": (i, [T, T, T, T]),
        "sdb_attention": (i, [T, T, T, T, ctypes.c_float, C, vp]),
        "sdb_group_norm": (i, [T, T, ctypes.c_int32, ctypes.c_float, C, vp]),
        "sdb_group_norm_no_alloc": (i, [T, T, ctypes.c_int32, ctypes.c_float, C, vp]),
        "sdb_norm": (i, [T, T, ctypes.c_float, C, vp]),
        "sdb_forget": (None, [vp, ctypes.c_size_t]),
        "sdb_store_stats": (None, [ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64)]),
        "sdb_token_downsampling": (i, [ctypes.c_int64, ctypes.c_int64]),
        "sdb_set_tuning": (i, [ctypes.c_char_p]),
        "sdb_get_tuning": (i, [ctypes.c_char_p, ctypes.POINTER(ctypes.c_int64)]),
        "sdb_device_status": (ctypes.c_uint, [i]),
        "sdb_last_error": (ctypes.c_char_p, []),
        "sdb_launch_count": (ctypes.c_uint64, []),
        "sdb_concat": (i, [T, T, T, ctypes.c_int32, vp]),
        "sdb_upscale_nearest": (i, [T, T, vp]),
        "sdb_coarser_tokens": (i, [T, T, ctypes.c_int32, vp]),
        "sdb_timestep_embedding": (i, [T, T, ctypes.c_int32, ctypes.c_int32, vp]),
        "sdb_group_norm_stats": (i, [T, ctypes.c_int32, ctypes.c_float, vp, vp]),
        "sdb_conv2d_normed": (i, [T, T, T, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(NormIn), C, vp]),
        "sdb_mul_mat_normed": (i, [T, T, T, ctypes.POINTER(NormIn), C, vp]),
        "sdb_mul_mat_layer_normed": (i, [T, T, T, ctypes.c_float, C, C, vp]),
        "sdb_mul_mat_gated_layer_normed": (i, [T, T, T, ctypes.c_float, C, C, vp]),
        # The structs of these come packed as bytes (_packed, Q4.struct, ...), passed by address.
        "sdb_q4_bytes": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32]),
        "sdb_q4_quantize": (i, [vp, vp, vp]),
        "sdb_q4_import": (i, [vp, vp, vp, vp, vp]),
        "sdb_q4_from_blocks": (i, [vp, ctypes.c_int64, vp, vp]),
        "sdb_q4_dequantize": (i, [vp, vp, vp]),
        "sdb_mul_mat_q4_supported": (i, [vp, vp, vp]),
        "sdb_mul_mat_q4": (i, [vp, vp, vp, vp, vp]),
        "sdb_mul_mat_q4_gated_supported": (i, [vp, vp, vp, vp]),
        "sdb_mul_mat_q4_gated": (i, [vp, vp, vp, vp, ctypes.c_int32, vp, vp]),
        "sdb_residual_norm": (i, [vp, vp, vp, vp, vp, vp]),
        "sdb_euler_cfg_step": (i, [vp, vp, vp, ctypes.c_int64, ctypes.c_float, ctypes.c_float, ctypes.c_float,
                                   ctypes.c_float, vp]),
        "sdb_euler_ancestral_cfg_step": (i, [vp, vp, vp, vp, ctypes.c_int64, ctypes.c_float, ctypes.c_float,
                                             ctypes.c_float, ctypes.c_float, vp]),
    }
    for name, (res, args) in sigs.items():
        f = getattr(lib, name)
        f.restype = res
        f.argtypes = args
    _lib = lib
    return lib


def _check(status: int) -> None:
    if status != OK:
        msg = load().sdb_last_error()
        raise SdbError(status, msg.decode() if msg else "")


# ---------------------------------------------------------------- tensors

def describe(t, ne: Sequence[int] | None = None, nb: Sequence[int] | None = None) -> Tensor:
    """The ggml description of a torch tensor (or an explicit ne / nb view of it)."""
    import torch

    if t.dtype == torch.float32:
        ty, es = TYPE_F32, 4
    elif t.dtype == torch.float16:
        ty, es = TYPE_F16, 2
    else:
        raise SdbError(INVALID, f"unsupported dtype {t.dtype}")
    d = Tensor()
    d.type = ty
    if ne is None:
        shape = list(reversed(t.shape))
        strides = [s * es for s in reversed(t.stride())]
        while len(shape) < 4:
            strides.append(strides[-1] * shape[-1] if shape else es)
            shape.append(1)
        if len(shape) > 4:
            raise SdbError(INVALID, "more than 4 dimensions")
        ne, nb = shape, strides
    for k in range(4):
        d.ne[k] = int(ne[k])
        d.nb[k] = int(nb[k])
    d.data = t.data_ptr()
    return d


def _stream_ptr(stream) -> int:
    import torch

    if stream is None:
        stream = torch.cuda.current_stream()
    return int(stream.cuda_stream)


def _own_strides(t) -> tuple:
    """The element strides of a chain's operand by its own extents, 0 along those of 1."""
    own = [0 if e == 1 else s for e, s in zip(reversed(t.shape), reversed(t.stride()))]
    return tuple((own + [0, 0, 0, 0])[:4])


class Chain:
    """An epilogue chain (sdasm::Epilogue): steps applied in order to each output element.

    add(t) / mul(t): t an FP32 CUDA tensor broadcastable to the output in ggml's
    sense (a dimension of extent 1 is broadcast), or read by explicit element
    strides nb, dimension 0 first; silu().  redirect(r,
    from_redirect) makes the operation write into r (a residual connection).
    """

    def __init__(self):
        # (kind, operand, strides): the operand's own strides as a tuple, explicit ones as a list.
        self.steps: list[tuple[int, object, Sequence[int]]] = []
        self.redirect_tensor = None
        self.from_redirect = False
        self._keep: list = []

    def _operand(self, kind, t, nb):
        import torch

        if t.dtype != torch.float32 or not t.is_cuda:
            raise SdbError(INVALID, "chain operands are FP32 CUDA tensors")
        self.steps.append((kind, t, _own_strides(t) if nb is None else list(nb)))
        return self

    def add(self, t, nb=None):
        return self._operand(STEP_ADD, t, nb)

    def mul(self, t, nb=None):
        return self._operand(STEP_MUL, t, nb)

    def silu(self):
        self.steps.append((STEP_SILU, None, [0, 0, 0, 0]))
        return self

    def redirect(self, t, from_redirect: bool = False):
        self.redirect_tensor = t
        self.from_redirect = from_redirect
        return self

    def struct(self) -> ChainStruct:
        if len(self.steps) > MAX_STEPS:
            raise SdbError(INVALID, "chain longer than 6 steps")
        c = ChainStruct()
        c.count = len(self.steps)
        for i, (kind, t, nb) in enumerate(self.steps):
            c.steps[i].kind = kind
            c.steps[i].operand = t.data_ptr() if t is not None else None
            for k in range(4):
                c.steps[i].nb[k] = nb[k]
        c.redirect = self.redirect_tensor.data_ptr() if self.redirect_tensor is not None else None
        c.from_redirect = 1 if self.from_redirect else 0
        return c


def _chain_ptr(chain: Chain | None):
    if chain is None:
        return None
    return ctypes.pointer(chain.struct())


# ---------------------------------------------------------------- weights

# The library keeps weights packed by address (the reference's store, which
# ggml tells of every write through sdasm_forget).  torch's caching allocator
# hands a freed block's address to the next tensor, so the binding forgets an
# address when a different tensor object shows up there.  A weight changed in
# place must still be forgotten by the caller: forget(w).
_weights: dict[int, weakref.ref] = {}


def _guard_weight(w) -> None:
    ptr = w.data_ptr()
    ref = _weights.get(ptr)
    if ref is not None and ref() is w:
        return
    if ref is not None:
        load().sdb_forget(ctypes.c_void_p(ptr), ctypes.c_size_t(w.numel() * w.element_size()))
    _weights[ptr] = weakref.ref(w)


# ---------------------------------------------------------------- operations

def mul_mat(w, x, out=None, chain: Chain | None = None, stream=None):
    """dst[m][n] = sum_k x[m][k] w[n][k]: w (N, K) FP16/FP32, x (..., K) FP32 -> (..., N)."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(*x.shape[:-1], w.shape[0], dtype=torch.float32, device=x.device)
    _guard_weight(w)
    dw, dx, dy = describe(w), describe(x), describe(out)
    if not lib.sdb_mul_mat_supported(dw, dx, dy):
        raise SdbError(NOT_SUPPORTED, "mul_mat shapes not supported")
    _check(lib.sdb_mul_mat(dw, dx, dy, _chain_ptr(chain), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def mul_mat_transient(w, x, out=None, chain: Chain | None = None, stream=None):
    """mul_mat for a first operand written between calls (packed every call, never kept):
    w (N, K) FP32/FP16, x (..., K) FP32 -> (..., N)."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(*x.shape[:-1], w.shape[0], dtype=torch.float32, device=x.device)
    _check(lib.sdb_mul_mat_transient(describe(w), describe(x), describe(out), _chain_ptr(chain),
                                     ctypes.c_void_p(_stream_ptr(stream))))
    return out


def soft_max(x, scale: float = 1.0, out=None, stream=None):
    """GGML_OP_SOFT_MAX without a mask: softmax(scale * x) along the last dimension (x may be out)."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty_like(x)
    _check(lib.sdb_soft_max(describe(x), describe(out), ctypes.c_float(scale), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def mul_mat_supported(w, x, out) -> bool:
    """Whether sdb_mul_mat takes these operands (under the tuning in effect)."""
    return bool(load().sdb_mul_mat_supported(describe(w), describe(x), describe(out)))


def mul_mat_gated_supported(w, x, out) -> bool:
    """Whether sdb_mul_mat_gated takes these operands (under the tuning in effect)."""
    return bool(load().sdb_mul_mat_gated_supported(describe(w), describe(x), describe(out)))


def mul_mat_gated(w, x, out=None, chain: Chain | None = None, stream=None):
    """GEGLU: y = x w^T (+chain), out = y[..., :N/2] * GELU(y[..., N/2:])."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(*x.shape[:-1], w.shape[0] // 2, dtype=torch.float32, device=x.device)
    _guard_weight(w)
    dw, dx, dy = describe(w), describe(x), describe(out)
    _check(lib.sdb_mul_mat_gated(dw, dx, dy, _chain_ptr(chain), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def conv_out_size(size: int, k: int, s: int, p: int, d: int) -> int:
    return (size + 2 * p - d * (k - 1) - 1) // s + 1


def conv2d(w, x, stride=(1, 1), padding=(0, 0), dilation=(1, 1), out=None, chain: Chain | None = None,
           stream=None):
    """ggml_conv_2d_direct: w (OC, IC, KH, KW), x (N, IC, H, W) FP32 -> (N, OC, OH, OW)."""
    import torch

    lib = load()
    oc, _, kh, kw = w.shape
    n, _, h, wd = x.shape
    oh = conv_out_size(h, kh, stride[1], padding[1], dilation[1])
    ow = conv_out_size(wd, kw, stride[0], padding[0], dilation[0])
    if out is None:
        out = torch.empty(n, oc, oh, ow, dtype=torch.float32, device=x.device)
    params = (ctypes.c_int32 * 6)(stride[0], stride[1], padding[0], padding[1], dilation[0], dilation[1])
    _guard_weight(w)
    dw, dx, dy = describe(w), describe(x), describe(out)
    _check(lib.sdb_conv2d(dw, dx, dy, params, _chain_ptr(chain), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def attention(q, k, v, scale: float, out=None, chain: Chain | None = None, stream=None):
    """FLASH_ATTN_EXT without a mask on token-major tensors.

    q (B, LQ, H*D), k (B, LK, HK*D), v (B, LK, HK*DV) with D / DV given by the
    head counts in `heads` of the views below; returns (B, LQ, H*DV).
    Use attention_heads() for explicit head counts.
    """
    raise NotImplementedError("use attention_heads(q, k, v, heads, kv_heads, scale)")


def attention_heads(q, k, v, heads: int, kv_heads: int, scale: float, out=None, chain: Chain | None = None,
                    stream=None):
    """softmax(scale q k^T) v per head; q (B, LQ, H*D), k/v (B, LK, HK*D) -> (B, LQ, H*DV).

    The ggml views are q [D, LQ, H, B] (head h at byte offset h*D*es of each
    token row), k [D, LK, HK, B], v [DV, LK, HK, B], dst [DV, H, LQ, B].
    """
    import torch

    lib = load()
    b, lq, hd = q.shape
    _, lk, hkd = k.shape
    d = hd // heads
    dv = v.shape[2] // kv_heads
    if out is None:
        out = torch.empty(b, lq, heads * dv, dtype=torch.float32, device=q.device)
    qs, ks, vs = q.element_size(), k.element_size(), v.element_size()
    dq = describe(q, [d, lq, heads, b], [qs, q.stride(1) * qs, d * qs, q.stride(0) * qs])
    dk = describe(k, [d, lk, kv_heads, b], [ks, k.stride(1) * ks, d * ks, k.stride(0) * ks])
    dvv = describe(v, [dv, lk, kv_heads, b], [vs, v.stride(1) * vs, dv * vs, v.stride(0) * vs])
    do = describe(out, [dv, heads, lq, b], [4, dv * 4, out.stride(1) * 4, out.stride(0) * 4])
    if not lib.sdb_attention_supported(dq, dk, dvv, do):
        raise SdbError(NOT_SUPPORTED, "attention shapes not supported")
    _check(lib.sdb_attention(dq, dk, dvv, do, ctypes.c_float(scale), _chain_ptr(chain),
                             ctypes.c_void_p(_stream_ptr(stream))))
    return out


def group_norm(x, groups: int, eps: float, out=None, chain: Chain | None = None, stream=None):
    """GGML_OP_GROUP_NORM over (N, C, H, W): groups of C/groups (rounded up) channels."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty_like(x)
    _check(lib.sdb_group_norm(describe(x), describe(out), groups, ctypes.c_float(eps), _chain_ptr(chain),
                              ctypes.c_void_p(_stream_ptr(stream))))
    return out


def group_norm_no_alloc(x, groups: int, eps: float, out, chain: Chain | None = None, stream=None):
    """group_norm without any device allocation (sdb_group_norm_no_alloc): out must be given."""
    lib = load()
    _check(lib.sdb_group_norm_no_alloc(describe(x), describe(out), groups, ctypes.c_float(eps), _chain_ptr(chain),
                                       ctypes.c_void_p(_stream_ptr(stream))))
    return out


def norm(x, eps: float, out=None, chain: Chain | None = None, stream=None):
    """GGML_OP_NORM: each row (last torch dimension) to mean 0, variance 1."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty_like(x)
    _check(lib.sdb_norm(describe(x), describe(out), ctypes.c_float(eps), _chain_ptr(chain),
                        ctypes.c_void_p(_stream_ptr(stream))))
    return out


def forget(t_or_ptr, size: int | None = None) -> None:
    """Drops packed weights made from the memory of t (sdasm_forget)."""
    lib = load()
    if size is None:
        ptr, size = t_or_ptr.data_ptr(), t_or_ptr.numel() * t_or_ptr.element_size()
    else:
        ptr = t_or_ptr
    lib.sdb_forget(ctypes.c_void_p(ptr), ctypes.c_size_t(size))
    for a in [a for a in _weights if ptr <= a < ptr + size]:
        del _weights[a]


def store_stats() -> tuple[int, int]:
    lib = load()
    e, b = ctypes.c_int64(), ctypes.c_int64()
    lib.sdb_store_stats(ctypes.byref(e), ctypes.byref(b))
    return e.value, b.value


def set_tuning(spec: str) -> None:
    _check(load().sdb_set_tuning(spec.encode()))


def get_tuning(name: str) -> int:
    v = ctypes.c_int64()
    _check(load().sdb_get_tuning(name.encode(), ctypes.byref(v)))
    return v.value


def device_status(clear: bool = True) -> int:
    return int(load().sdb_device_status(1 if clear else 0))


def launch_count() -> int:
    return int(load().sdb_launch_count())


def token_downsampling(width: int, height: int) -> int:
    return int(load().sdb_token_downsampling(width, height))


# ---------------------------------------------------------------- channels-last images

def describe_nhwc(t) -> Tensor:
    """A contiguous (N, H, W, C) FP32 tensor as the ggml image [W, H, C, N] it holds (channels-last strides)."""
    n, h, w, c = t.shape
    es = t.element_size()
    return describe(t, [w, h, c, n], [c * es, w * c * es, es, h * w * c * es])


def conv2d_nhwc(w, x, stride=(1, 1), padding=(0, 0), dilation=(1, 1), out=None, chain: Chain | None = None,
                stream=None, out_nchw: bool = False):
    """ggml_conv_2d_direct on channels-last images: w (OC, IC, KH, KW), x (N, H, W, IC) -> (N, OH, OW, OC),
    or with out_nchw the output channel-major, (N, OC, OH, OW)."""
    import torch

    lib = load()
    oc, _, kh, kw = w.shape
    n, h, wd, _ = x.shape
    oh = conv_out_size(h, kh, stride[1], padding[1], dilation[1])
    ow = conv_out_size(wd, kw, stride[0], padding[0], dilation[0])
    if out is None:
        shape = (n, oc, oh, ow) if out_nchw else (n, oh, ow, oc)
        out = torch.empty(*shape, dtype=torch.float32, device=x.device)
    params = (ctypes.c_int32 * 6)(stride[0], stride[1], padding[0], padding[1], dilation[0], dilation[1])
    _guard_weight(w)
    dy = describe(out) if out_nchw else describe_nhwc(out)
    _check(lib.sdb_conv2d(describe(w), describe_nhwc(x), dy, params, _chain_ptr(chain),
                          ctypes.c_void_p(_stream_ptr(stream))))
    return out


def channel_operand(t):
    """ggml strides of a per-channel operand (C,) for a channels-last image output: broadcast over W, H, N."""
    return [0, 0, 1, 0]


def group_norm_nhwc(x, groups: int, eps: float, out=None, chain: Chain | None = None, stream=None):
    """GGML_OP_GROUP_NORM on a channels-last image (N, H, W, C), C % groups == 0."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty_like(x)
    _check(lib.sdb_group_norm(describe_nhwc(x), describe_nhwc(out), groups, ctypes.c_float(eps), _chain_ptr(chain),
                              ctypes.c_void_p(_stream_ptr(stream))))
    return out


class GroupNormIn:
    """A GroupNorm (+ SiLU) that the next operation applies as it reads its input (sdb_norm_in):
    the statistics of x (group_norm_stats), gamma and beta (C,) or None, groups, SiLU."""

    def __init__(self, stats, groups: int, gamma=None, beta=None, silu: bool = False):
        self.stats, self.groups, self.gamma, self.beta, self.silu = stats, groups, gamma, beta, silu
        self.c = NormIn(stats.data_ptr(), gamma.data_ptr() if gamma is not None else None,
                        beta.data_ptr() if beta is not None else None, groups, 1 if silu else 0)


def group_norm_stats(x, groups: int, eps: float, out=None, stream=None):
    """Mean and 1 / sqrt(variance + eps) per image and group of a channels-last image (N, H, W, C):
    (N, groups, 2) FP32 (sdb_group_norm_stats)."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(x.shape[0], groups, 2, dtype=torch.float32, device=x.device)
    _check(lib.sdb_group_norm_stats(describe_nhwc(x), groups, ctypes.c_float(eps), ctypes.c_void_p(out.data_ptr()),
                                    ctypes.c_void_p(_stream_ptr(stream))))
    return out


def conv2d_nhwc_normed(w, x, norm: GroupNormIn, stride=(1, 1), padding=(0, 0), dilation=(1, 1), out=None,
                       chain: Chain | None = None, stream=None):
    """conv2d_nhwc of GroupNorm(x) [+ SiLU], the normalisation applied as the convolution reads x."""
    import torch

    lib = load()
    oc, _, kh, kw = w.shape
    n, h, wd, _ = x.shape
    oh = conv_out_size(h, kh, stride[1], padding[1], dilation[1])
    ow = conv_out_size(wd, kw, stride[0], padding[0], dilation[0])
    if out is None:
        out = torch.empty(n, oh, ow, oc, dtype=torch.float32, device=x.device)
    params = (ctypes.c_int32 * 6)(stride[0], stride[1], padding[0], padding[1], dilation[0], dilation[1])
    _guard_weight(w)
    _check(lib.sdb_conv2d_normed(describe(w), describe_nhwc(x), describe_nhwc(out), params, ctypes.byref(norm.c),
                                 _chain_ptr(chain), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def mul_mat_normed(w, x, norm: GroupNormIn, out=None, chain: Chain | None = None, stream=None):
    """mul_mat of GroupNorm(x) [+ SiLU]: x (N, P, C), the P positions of each of N images."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(*x.shape[:-1], w.shape[0], dtype=torch.float32, device=x.device)
    _guard_weight(w)
    _check(lib.sdb_mul_mat_normed(describe(w), describe(x), describe(out), ctypes.byref(norm.c), _chain_ptr(chain),
                                  ctypes.c_void_p(_stream_ptr(stream))))
    return out


def mul_mat_layer_normed(w, x, eps: float, norm_chain: Chain | None = None, out=None, chain: Chain | None = None,
                         gated: bool = False, stream=None):
    """mul_mat (or mul_mat_gated) of LayerNorm(x) with its chain (gamma, beta), the normalisation done in
    the linear layer's split of the rows: x (..., K) -> (..., N) (N / 2 gated)."""
    import torch

    lib = load()
    if out is None:
        n = w.shape[0] // 2 if gated else w.shape[0]
        out = torch.empty(*x.shape[:-1], n, dtype=torch.float32, device=x.device)
    _guard_weight(w)
    fn = lib.sdb_mul_mat_gated_layer_normed if gated else lib.sdb_mul_mat_layer_normed
    _check(fn(describe(w), describe(x), describe(out), ctypes.c_float(eps), _chain_ptr(norm_chain), _chain_ptr(chain),
              ctypes.c_void_p(_stream_ptr(stream))))
    return out


def concat_channels_nhwc(a, b, out=None, stream=None):
    """GGML_OP_CONCAT along C of channels-last images (N, H, W, Ca) and (N, H, W, Cb)."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(*a.shape[:3], a.shape[3] + b.shape[3], dtype=torch.float32, device=a.device)
    _check(lib.sdb_concat(describe_nhwc(a), describe_nhwc(b), describe_nhwc(out), 2,
                          ctypes.c_void_p(_stream_ptr(stream))))
    return out


def upscale_nearest_nhwc(x, factor: int = 2, out=None, stream=None):
    """GGML_OP_UPSCALE (nearest) of a channels-last image by an integer factor."""
    import torch

    lib = load()
    n, h, w, c = x.shape
    if out is None:
        out = torch.empty(n, h * factor, w * factor, c, dtype=torch.float32, device=x.device)
    _check(lib.sdb_upscale_nearest(describe_nhwc(x), describe_nhwc(out), ctypes.c_void_p(_stream_ptr(stream))))
    return out


def coarser_tokens(x, width: int, height: int, factor: int, out=None, stream=None):
    """ToDo's keys' and values' tokens: x (N, height * width, C) tokens of a grid, row after row ->
    (N, ceil(height / f) * ceil(width / f), C), every f-th token of every f-th row."""
    import torch

    lib = load()
    n, l, c = x.shape
    if l != width * height:
        raise SdbError(INVALID, "coarser_tokens: the tokens are not the grid's")
    w2, h2 = -(-width // factor), -(-height // factor)
    if out is None:
        out = torch.empty(n, h2 * w2, c, dtype=torch.float32, device=x.device)
    s = [v * 4 for v in x.stride()]
    src = describe(x, [c, width, height, n], [s[2], s[1], s[1] * width, s[0]])
    dst = describe(out, [c, w2, h2, n], [4, 4 * c, 4 * c * w2, 4 * c * w2 * h2])
    _check(lib.sdb_coarser_tokens(src, dst, factor, ctypes.c_void_p(_stream_ptr(stream))))
    return out


def timestep_embedding(t, dim: int, max_period: int = 10000, out=None, stream=None):
    """GGML_OP_TIMESTEP_EMBEDDING: t (N,) FP32 -> (N, dim) = [cos(t f) | sin(t f)]."""
    import torch

    lib = load()
    if out is None:
        out = torch.empty(t.shape[0], dim, dtype=torch.float32, device=t.device)
    _check(lib.sdb_timestep_embedding(describe(t), describe(out), dim, max_period,
                                      ctypes.c_void_p(_stream_ptr(stream))))
    return out


def euler_ancestral_cfg_step(eps, x, x_in, noise, cfg: float, sigma: float, sigma_next: float, c_in_next: float,
                             stream=None):
    """The ancestral Euler step with guidance: x += (sigma_down - sigma) e + sigma_up noise (see sdb.h)."""
    lib = load()
    _check(lib.sdb_euler_ancestral_cfg_step(ctypes.c_void_p(eps.data_ptr()), ctypes.c_void_p(x.data_ptr()),
                                            ctypes.c_void_p(x_in.data_ptr() if x_in is not None else 0),
                                            ctypes.c_void_p(noise.data_ptr()), ctypes.c_int64(x.numel()),
                                            ctypes.c_float(cfg), ctypes.c_float(sigma), ctypes.c_float(sigma_next),
                                            ctypes.c_float(c_in_next), ctypes.c_void_p(_stream_ptr(stream))))


def euler_cfg_step(eps, x, x_in, cfg: float, sigma: float, sigma_next: float, c_in_next: float, stream=None):
    """x += (sigma_next - sigma) (eps_u + cfg (eps_c - eps_u)); x_in[0] = x_in[1] = x c_in_next (eps = [eps_u, eps_c])."""
    lib = load()
    _check(lib.sdb_euler_cfg_step(ctypes.c_void_p(eps.data_ptr()), ctypes.c_void_p(x.data_ptr()),
                                  ctypes.c_void_p(x_in.data_ptr() if x_in is not None else 0),
                                  ctypes.c_int64(x.numel()), ctypes.c_float(cfg), ctypes.c_float(sigma),
                                  ctypes.c_float(sigma_next), ctypes.c_float(c_in_next),
                                  ctypes.c_void_p(_stream_ptr(stream))))


# ---------------------------------------------------------------- 4-bit weights

# A call of a few microseconds should not wait for its description: the structs of the operators below are
# packed into bytes in one step each, and the bytes' address is passed.
_TENSOR = struct.Struct("=i4x4q4qQ")
_STEP = struct.Struct("=i4xQ4q")
_CHAIN_TAIL = struct.Struct("=Qi4x")
_Q4 = struct.Struct("=Q2q2i")
_NORM_FORM = struct.Struct("=ifQQ")
_OPERAND = struct.Struct("=Q4q")
_KEEP_SCALE = struct.Struct("=2f")
_NO_STEP = _STEP.pack(0, 0, 0, 0, 0, 0)
_NO_OPERAND = _OPERAND.pack(0, 0, 0, 0, 0)

GATES = {"gelu": 0, "silu": 1}
NORMS = {"none": 0, "layer": 1, "rms": 2}


def _packed(t, what: str) -> bytes:
    """The sdb_tensor of an FP32 or FP16 CUDA tensor of at most four dimensions, as bytes."""
    shape, stride = t.shape, t.stride()
    es = t.element_size()
    if not t.is_floating_point() or (es != 4 and (es != 2 or str(t.dtype) != "torch.float16")):
        raise SdbError(INVALID, f"{what}: unsupported dtype {t.dtype}")
    ty = TYPE_F32 if es == 4 else TYPE_F16
    nd = len(shape)
    if nd == 2:
        n1, n0 = shape
        s1, s0 = stride
        s1 *= es
        return _TENSOR.pack(ty, n0, n1, 1, 1, s0 * es, s1, s1 * n1, s1 * n1, t.data_ptr())
    if nd == 3:
        n2, n1, n0 = shape
        s2, s1, s0 = stride
        s2 *= es
        return _TENSOR.pack(ty, n0, n1, n2, 1, s0 * es, s1 * es, s2, s2 * n2, t.data_ptr())
    if nd == 0 or nd > 4:
        raise SdbError(INVALID, f"{what}: one to four dimensions")
    ne = [shape[nd - 1 - d] if d < nd else 1 for d in range(4)]
    nb = [stride[nd - 1 - d] * es if d < nd else 0 for d in range(4)]
    return _TENSOR.pack(ty, *ne, *nb, t.data_ptr())


def _chain_tensors(chain: Chain | None) -> tuple:
    """The tensors of a chain: its operands, then its redirect."""
    if chain is None:
        return ()
    found = [t for _, t, _ in chain.steps if t is not None]
    if chain.redirect_tensor is not None:
        found.append(chain.redirect_tensor)
    return tuple(found)


def _check_operand(t, nb, shape, cols: int, rows: int) -> None:
    """Refuses an operand that is not of the output's extents or, read by explicit strides, one that a chain
    would read past its memory's end."""
    if type(nb) is tuple and nb == _own_strides(t):
        d = 0
        for e in reversed(t.shape):
            if e != 1 and e != (cols if d == 0 else shape[-1 - d] if d < len(shape) else 1):
                raise SdbError(INVALID, f"a chain operand of {tuple(t.shape)} for {cols} columns of {tuple(shape)}")
            d += 1
        return
    if min(nb) < 0:
        raise SdbError(INVALID, "a chain operand's strides are not negative")
    last = (cols - 1) * nb[0]
    for d in range(1, len(shape)):
        last += (shape[-1 - d] - 1) * nb[d]
    if rows and last >= t.untyped_storage().nbytes() // 4 - t.storage_offset():
        raise SdbError(INVALID, "a chain operand ends before the output's rows")


def _packed_chain(chain: Chain | None, tensors: tuple, out, cols: int):
    """The sdb_chain of an operation on out's rows, `cols` columns each, as bytes (None: no chain)."""
    if chain is None:
        return None
    shape = out.shape
    steps, r = chain.steps, chain.redirect_tensor
    if r is not None and (r.dtype != out.dtype or r.shape != shape or r.stride() != out.stride()):
        raise SdbError(INVALID, "a chain's redirect has the output's type, extents and strides")
    # A chain that is used again as it was is not described again: the key is all that the checks of operands with
    # their own strides look at.  The memory behind explicit strides is looked at in every call.
    own = True
    places = []
    for kind, t, nb in steps:
        if t is None:
            places.append(kind)
        elif type(nb) is tuple:
            places.append((kind, nb, t.data_ptr(), t.shape, t.stride()))
        else:
            own = False
            places.append((kind, *nb, t.data_ptr()))
    key = (places, cols, shape, None if r is None else r.data_ptr(), chain.from_redirect)
    kept = chain.__dict__.get("_described")
    if own and kept is not None and kept[0] == key:
        return kept[1]
    if len(steps) > MAX_STEPS:
        raise SdbError(INVALID, "chain longer than 6 steps")
    rows = out.numel()
    parts = [struct.pack("=i4x", len(steps))]
    for kind, t, nb in steps:
        if t is not None:
            _check_operand(t, nb, shape, cols, rows)
            own = own and nb == _own_strides(t)
        parts.append(_STEP.pack(kind, t.data_ptr() if t is not None else 0, *nb))
    parts.extend([_NO_STEP] * (MAX_STEPS - len(steps)))
    parts.append(_CHAIN_TAIL.pack(key[3] or 0, 1 if chain.from_redirect else 0))
    packed = b"".join(parts)
    chain._described = (key, packed) if own else None
    return packed


_raw_stream = None  # device index -> the address of its current stream
_raw_device = None  # the current device's index


def _find_raw() -> None:
    """The two lookups a call makes, without the Python objects of torch.cuda.current_stream() (3 of a call's
    8 microseconds on the host) where this torch offers that."""
    global _raw_stream, _raw_device
    import torch

    torch.cuda.init()
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: torch.cuda.current_stream(index).cuda_stream)
    _raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _on(fn, what: str, tensors, stream, *args) -> None:
    """Calls fn(*args, stream) with the tensors' device current, on `stream` or that device's current stream."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index:
            index = -1
    if index < 0:
        raise SdbError(INVALID, f"{what}: the tensors are not on one CUDA device")
    if _raw_stream is None:
        _find_raw()
    if stream is None:
        address = _raw_stream(index)
    elif stream.device.index != index:
        raise SdbError(INVALID, f"{what}: the stream is another device's")
    else:
        address = stream.cuda_stream
    if _raw_device() == index:
        status = fn(*args, address)
    else:
        import torch

        with torch.cuda.device(index):
            status = fn(*args, address)
    if status != OK:
        _check(status)


def _made(stream, device, what: str, make):
    """make()'s new tensor or matrix for a call on `stream`, from that stream's memory: the current stream's
    may still be written by work that has not run yet.  It is not given to others before the stream that is
    current here is done with it either."""
    if stream is None or device.type != "cuda":
        return make()
    import torch

    current = torch.cuda.current_stream(device)
    if stream == current:
        return make()
    if stream.device != current.device:
        raise SdbError(INVALID, f"{what}: the stream is another device's")
    with torch.cuda.stream(stream):
        made = make()
    made.data.record_stream(current)  # a matrix's memory, or the tensor's own
    return made


class Q4:
    """A matrix (n, k) of 4-bit numbers with group scales on the device (sdb_q4): value = d (q - 8), or with
    `minimum` d q + m, an FP16 d (and m) for every `group` numbers of a row.  Made by q4_quantize, q4_import or
    q4_from_blocks; read by mul_mat_q4 and mul_mat_q4_gated."""

    def __init__(self, n: int, k: int, group: int = 32, minimum: bool = False, device=None):
        import torch

        self._form = (k, n, group, 1 if minimum else 0)
        self._size = load().sdb_q4_bytes(*self._form)
        if self._size <= 0:
            raise SdbError(INVALID, f"no 4-bit matrix of {n} x {k} in groups of {group}")
        self.n, self.k, self.group, self.minimum = n, k, group, bool(minimum)
        self.data = torch.empty(self._size, dtype=torch.uint8, device="cuda" if device is None else device)

    @property
    def data(self):
        """The matrix's memory, uint8; another of its size may take its place."""
        return self._data

    @data.setter
    def data(self, t):
        import torch

        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise SdbError(INVALID, "4-bit matrices are on a CUDA device")
        if t.dtype != torch.uint8 or t.shape != (self._size,) or not t.is_contiguous():
            raise SdbError(INVALID, f"a 4-bit matrix's memory is {self._size} dense bytes")
        self._data, self._at = t, None

    @property
    def struct(self) -> bytes:
        """The sdb_q4 of the memory the matrix has now: a copy of a matrix has memory of its own."""
        at = self._data.data_ptr()
        if at != self._at:
            self._packed, self._at = _Q4.pack(at, *self._form), at
        return self._packed

    def values(self, out=None, stream=None):
        """The numbers the matrix stands for, FP32 (n, k) (sdb_q4_dequantize)."""
        import torch

        if out is None:
            device = self.data.device
            out = _made(stream, device, "Q4.values",
                        lambda: torch.empty(self.n, self.k, dtype=torch.float32, device=device))
        _on(load().sdb_q4_dequantize, "Q4.values", (self.data, out), stream, self.struct, _packed(out, "Q4.values"))
        return out


def q4_quantize(w, group: int = 32, minimum: bool = False, stream=None) -> Q4:
    """w (n, k) FP32 or FP16, rows contiguous, quantized to 4 bits (sdb_q4_quantize)."""
    if w.dim() != 2:
        raise SdbError(INVALID, "q4_quantize: a matrix (n, k)")
    q = _made(stream, w.device, "q4_quantize", lambda: Q4(w.shape[0], w.shape[1], group, minimum, w.device))
    _on(load().sdb_q4_quantize, "q4_quantize", (w, q.data), stream, _packed(w, "q4_quantize"), q.struct)
    return q


def q4_import(codes, scales, minima=None, k: int | None = None, group: int = 32, stream=None) -> Q4:
    """From 4-bit numbers: codes (n, (k + 1) // 2) uint8, the even column in a byte's low half; scales and minima
    (n, ceil(k / group)) FP16; k twice the bytes of a row unless given (sdb_q4_import)."""
    import torch

    k = 2 * codes.shape[-1] if k is None else k
    n, groups = codes.shape[0], -(-k // group) if group else 0
    q = _made(stream, codes.device, "q4_import", lambda: Q4(n, k, group, minima is not None, codes.device))
    if codes.dtype != torch.uint8 or codes.shape != (n, (k + 1) // 2) or not codes.is_contiguous():
        raise SdbError(INVALID, "q4_import: codes must be dense uint8 (n, (k + 1) // 2)")
    tensors = [codes, scales, q.data] + ([minima] if minima is not None else [])
    for t in (scales, minima):
        if t is not None and (t.dtype != torch.float16 or t.shape != (n, groups) or not t.is_contiguous()):
            raise SdbError(INVALID, "q4_import: scales and minima must be dense FP16 (n, ceil(k / group))")
    _on(load().sdb_q4_import, "q4_import", tensors, stream, codes.data_ptr(), scales.data_ptr(),
        minima.data_ptr() if minima is not None else None, q.struct)
    return q


def q4_from_blocks(blocks, k: int, minimum: bool = False, stream=None) -> Q4:
    """From ggml's blocks: blocks (n, bytes of a row) uint8, GGML_TYPE_Q4_0 or with `minimum` GGML_TYPE_Q4_1
    (sdb_q4_from_blocks)."""
    import torch

    if blocks.dtype != torch.uint8 or blocks.dim() != 2 or blocks.stride(1) != 1:
        raise SdbError(INVALID, "q4_from_blocks: blocks must be uint8 (n, bytes of a row)")
    if k % 32 != 0 or blocks.shape[1] < k // 32 * (20 if minimum else 18):
        raise SdbError(INVALID, "q4_from_blocks: rows are k / 32 whole blocks")
    q = _made(stream, blocks.device, "q4_from_blocks", lambda: Q4(blocks.shape[0], k, 32, minimum, blocks.device))
    _on(load().sdb_q4_from_blocks, "q4_from_blocks", (blocks, q.data), stream, blocks.data_ptr(), blocks.stride(0),
        q.struct)
    return q


def mul_mat_q4(w: Q4, x, out=None, chain: Chain | None = None, stream=None):
    """dst[m][n] = sum_k x[m][k] value[n][k], then the chain: w a Q4 (N, K), x (..., K) FP32 or FP16 -> (..., N)
    of out's type (x's unless out is given).  For a few rows of x."""
    import torch

    if out is None:
        out = _made(stream, x.device, "mul_mat_q4",
                    lambda: torch.empty(*x.shape[:-1], w.n, dtype=x.dtype, device=x.device))
    extra = _chain_tensors(chain)
    _on((_lib or load()).sdb_mul_mat_q4, "mul_mat_q4", (w.data, x, out, *extra), stream, w.struct,
        _packed(x, "mul_mat_q4"), _packed(out, "mul_mat_q4"), _packed_chain(chain, extra, out, w.n))
    return out


def mul_mat_q4_gated(w: Q4, gate: Q4, x, act: str = "gelu", out=None, chain: Chain | None = None, stream=None):
    """(x W^T) act(x V^T) of two Q4 (N, K), the chain applied to both products as to columns 0..N - 1 and
    N..2N - 1 of one; act "gelu" or "silu"."""
    import torch

    if act not in GATES:
        raise SdbError(INVALID, f"mul_mat_q4_gated: no gate {act!r}")
    if out is None:
        out = _made(stream, x.device, "mul_mat_q4_gated",
                    lambda: torch.empty(*x.shape[:-1], w.n, dtype=x.dtype, device=x.device))
    extra = _chain_tensors(chain)
    _on((_lib or load()).sdb_mul_mat_q4_gated, "mul_mat_q4_gated", (w.data, gate.data, x, out, *extra), stream,
        w.struct, gate.struct, _packed(x, "mul_mat_q4_gated"), _packed(out, "mul_mat_q4_gated"), GATES[act],
        _packed_chain(chain, extra, out, 2 * w.n))
    return out


# ---------------------------------------------------------------- the residual block

class Norm:
    """A row's norm (sdb_norm_form): "layer" or "rms", eps, and weight and bias (C,) FP32 or None."""

    def __init__(self, kind: str, eps: float = 1e-5, weight=None, bias=None):
        if kind not in NORMS:
            raise SdbError(INVALID, f"no norm {kind!r}")
        self.kind, self.eps, self.weight, self.bias = kind, eps, weight, bias
        self.tensors = [t for t in (weight, bias) if t is not None]
        for t in self.tensors:
            if str(t.dtype) != "torch.float32" or t.dim() != 1 or not t.is_contiguous():
                raise SdbError(INVALID, "a norm's weight and bias are dense FP32 (C,)")

    def packed(self, c: int) -> bytes:
        """The sdb_norm_form for rows of c numbers."""
        w = b = 0
        if self.weight is not None:
            w = self.weight.data_ptr()
            if self.weight.numel() != c:
                raise SdbError(INVALID, f"a norm of {self.weight.numel()} numbers for rows of {c}")
        if self.bias is not None:
            b = self.bias.data_ptr()
            if self.bias.numel() != c:
                raise SdbError(INVALID, f"a norm of {self.bias.numel()} numbers for rows of {c}")
        return _NORM_FORM.pack(NORMS[self.kind], self.eps, w, b)


_NO_NORM = _NORM_FORM.pack(0, 0.0, 0, 0)


def _packed_operand(t, shape) -> bytes:
    """An FP32 tensor broadcastable to `shape`, as the bytes of an sdb_operand."""
    if t is None:
        return _NO_OPERAND
    if t.element_size() != 4 or not t.is_floating_point():
        raise SdbError(INVALID, "modulations are FP32")
    nb = [0, 0, 0, 0]
    ts = t.shape
    if len(ts) > len(shape):
        raise SdbError(INVALID, "a modulation has more dimensions than the rows")
    d = 0
    for e, s, n in zip(reversed(ts), reversed(t.stride()), reversed(shape)):
        if e != 1:
            if e != n:
                raise SdbError(INVALID, f"a modulation of {tuple(ts)} for rows of {tuple(shape)}")
            nb[d] = s
        d += 1
    return _OPERAND.pack(t.data_ptr(), *nb)


def residual_norm(x, y, post: Norm | None = None, gate=None, keep: float = 1.0, scale: float = 1.0,
                  pre: Norm | None = None, mul=None, add=None, h=None, out=None, want_h: bool = True,
                  want_out: bool = True, stream=None):
    """h = keep x + scale gate post(y); out = pre(h) (1 + mul) + add.  Returns (h, out).

    x, y (..., C) FP32 or FP16, up to four dimensions, either None; gate, mul and add FP32, broadcastable to
    them.  h is of x's type, out of y's (of the other's where one is None); h may be x, out may be y (the
    update in place).  want_h / want_out False: that one is not made (None).
    """
    ref = x if x is not None else y
    if ref is None:
        raise SdbError(INVALID, "residual_norm: neither x nor y")
    shape = ref.shape
    if not want_h:
        h = None
    elif h is None:
        h = _made(stream, ref.device, "residual_norm", lambda: ref.new_empty(shape))
    if not want_out:
        out = None
    elif out is None:
        out = _made(stream, ref.device, "residual_norm", lambda: (y if y is not None else x).new_empty(shape))
    tensors = [ref]
    for t in (y, h, out, gate, mul, add):
        if t is not None:
            tensors.append(t)
    if post is not None:
        tensors += post.tensors
    if pre is not None:
        tensors += pre.tensors
    c = shape[-1] if len(shape) else 0
    params = b"".join((_KEEP_SCALE.pack(keep, scale),
                       _NO_NORM if post is None else post.packed(c), _NO_NORM if pre is None else pre.packed(c),
                       _NO_OPERAND if gate is None else _packed_operand(gate, shape),
                       _NO_OPERAND if mul is None else _packed_operand(mul, shape),
                       _NO_OPERAND if add is None else _packed_operand(add, shape)))
    what = "residual_norm"
    _on((_lib or load()).sdb_residual_norm, what, tensors, stream,
        _packed(x, what) if x is not None else None, _packed(y, what) if y is not None else None,
        _packed(h, what) if h is not None else None, _packed(out, what) if out is not None else None, params)
    return h, out
