"""Tensor-level wrappers of the C ABI: shape/dtype checks, pointer marshalling, stream.

These are the calls the reference-shaped holders in `iquestrt_b200.kernels` make.  Every
function launches on torch's current CUDA stream, allocates nothing when its outputs
are passed in, and raises on any non-zero return code.  PyTorch is used for device
memory and streams only."""

from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import torch

from . import _lib
from ._lib import (ACT_BF16, ACT_E4M3, ROUTE_SIGMOID, ROUTE_SOFTMAX, TAIL_ATTN, TAIL_MLP,
                   X_BF16_GROUPQ, X_BF16_SPLIT2, X_E4M3_GROUP, X_E4M3_UNSCALED)

E4M3 = torch.float8_e4m3fn

__all__ = ["Scratch", "TailSpec", "linear", "linear_static", "linear_static_status", "qkv_heads",
           "router",
           "moe_gate", "moe_down", "tail",
           "AttnWork", "attn_decode", "EvictWork", "kv_evict", "kv_advance",
           "X_BF16_GROUPQ", "X_BF16_SPLIT2", "X_E4M3_GROUP", "X_E4M3_UNSCALED",
           "TAIL_ATTN", "TAIL_MLP", "ROUTE_SOFTMAX", "ROUTE_SIGMOID", "ACT_E4M3", "ACT_BF16"]


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _need(name, t, dtype, shape=None, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor, got {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


class Scratch:
    """The zero-filled work area the streaming kernels share (split-tile partials, tile
    counters, the CTA ticket and the device status word).  One per stream of calls."""

    def __init__(self, device="cuda"):
        lib = _lib.load()
        self.bytes = int(lib.iq_scratch_bytes())
        self.buf = torch.zeros(self.bytes, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr()
        self.index = self.buf.get_device()

    def status(self, clear: bool = True) -> int:
        """Synchronises the current stream and returns the device status code.  After an
        error the whole work area is zeroed (with `clear`): a launch that gave up may have
        left counters and hand-off words behind."""
        code = C.c_int(0)
        _lib.check("iq_status_read",
                   _lib.load().iq_status_read(self.ptr, C.byref(code), int(clear), _stream()))
        if code.value and clear:
            self.buf.zero_()
        return code.value

    def raise_on_error(self, where: str = "device status") -> None:
        code = self.status()
        if code:
            raise _lib.IqError(where, code)


@dataclass
class TailSpec:
    """Arguments of the all-reduce + residual + RMSNorm epilogue (see `iq_tail_args`).

    `partial` is this rank's bf16 [m,h] rows; for world > 1 it must live in a symmetric
    buffer and `comm` (a `parallel.SymmSlot`) supplies the multicast / peer addresses."""

    kind: int
    partial: torch.Tensor
    residual: torch.Tensor
    w_norm: torch.Tensor
    h_out: torch.Tensor
    norm_out: torch.Tensor
    scale: float = 1.0
    eps: float = 1e-6
    w_first: torch.Tensor | None = None
    norm_fp8: torch.Tensor | None = None
    norm_fp8_scale: torch.Tensor | None = None
    inv_out: torch.Tensor | None = None
    comm: object | None = None
    timeout_ms: int = 2000
    _keep: list = field(default_factory=list, repr=False)

    def to_c(self, status_ptr: int) -> _lib.TailArgs:
        m, h = self.partial.shape
        dev = self.partial.device
        _need("partial", self.partial, torch.bfloat16)
        fp32 = self.residual.dtype == torch.float32
        _need("residual", self.residual, torch.float32 if fp32 else torch.bfloat16, (m, h), dev)
        _need("w_norm", self.w_norm, torch.float32, (h,), dev)
        _need("h_out", self.h_out, torch.float32 if fp32 else torch.bfloat16, (m, h), dev)
        _need("norm_out", self.norm_out, torch.bfloat16, (m, h), dev)
        if self.kind == TAIL_ATTN:
            _need("w_first", self.w_first, torch.float32, (h,), dev)
        if self.norm_fp8 is not None:
            _need("norm_fp8", self.norm_fp8, E4M3, (m, h), dev)
        if self.norm_fp8_scale is not None:
            _need("norm_fp8_scale", self.norm_fp8_scale, torch.float32, (m, h // 128), dev)
        if self.inv_out is not None:
            _need("inv_out", self.inv_out, torch.float32, (m,), dev)
        a = _lib.TailArgs()
        a.kind = self.kind
        a.m, a.h = m, h
        a.partial = self.partial.data_ptr()
        if self.comm is None:
            a.world, a.rank = 1, 0
        else:
            self.comm.fill(a, self.partial)
        a.residual = self.residual.data_ptr()
        a.residual_fp32 = int(fp32)
        a.w_first = _ptr(self.w_first)
        a.w_norm = self.w_norm.data_ptr()
        a.scale, a.eps = float(self.scale), float(self.eps)
        a.h_out = self.h_out.data_ptr()
        a.norm_out = self.norm_out.data_ptr()
        a.norm_fp8 = _ptr(self.norm_fp8)
        a.norm_fp8_scale = _ptr(self.norm_fp8_scale)
        a.inv_out = _ptr(self.inv_out)
        a.status = status_ptr
        a.timeout_ms = int(self.timeout_ms)
        return a


_SCRATCH: dict[int, Scratch] = {}


def default_scratch(device=None) -> Scratch:
    """The per-device scratch the reference-shaped holders share (their calls are ordered
    on one stream, as one captured decode step is)."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    if index is None:
        index = torch.cuda.current_device()
    if index not in _SCRATCH:
        _SCRATCH[index] = Scratch(torch.device("cuda", index))
    return _SCRATCH[index]


def tail(spec: TailSpec, scratch: Scratch, *, pdl: bool = False) -> None:
    """The epilogue on its own: one CTA (`iq_tail`)."""
    a = spec.to_c(scratch.ptr)
    _lib.check("iq_tail", _lib.load().iq_tail(C.byref(a), _stream(), int(pdl)))


def _linear_args(x, w, w_scale, out, x_kind, x_scale, block):
    """Checks the operands of the block-FP8 GEMV and fills the part of `iq_linear_args`
    that `linear` and `linear_static` share."""
    m, k = x.shape
    n = w.shape[0]
    dev = x.device
    _need("w", w, E4M3, (n, k), dev)
    rg, kg = block
    _need("w_scale", w_scale, torch.float32, (n // rg, k // kg), dev)
    if x_kind is None:
        if x.dtype == torch.bfloat16:
            x_kind = X_BF16_GROUPQ
        else:
            x_kind = X_E4M3_GROUP if x_scale is not None else X_E4M3_UNSCALED
    _need("x", x, torch.bfloat16 if x_kind in (X_BF16_GROUPQ, X_BF16_SPLIT2) else E4M3, None, dev)
    if x_kind == X_E4M3_GROUP:
        _need("x_scale", x_scale, torch.float32, (m, k // 128), dev)
    if out is not None:
        _need("out", out, torch.bfloat16, (m, n), dev)
    a = _lib.LinearArgs()
    a.x, a.x_scale, a.x_kind = x.data_ptr(), _ptr(x_scale), x_kind
    a.m, a.k, a.n = m, k, n
    a.w, a.w_scale, a.rg, a.kg = w.data_ptr(), w_scale.data_ptr(), rg, kg
    a.out = _ptr(out)
    return a


def linear(x, w, w_scale, *, scratch: Scratch, out=None, x_kind=None, x_scale=None,
           block=(128, 128), tail: TailSpec | None = None, push=None, out_f32=None,
           pdl: bool = False):
    """`out[m,n] bf16 = x[m,k] @ dequant(w[n,k], w_scale).T` on the streaming GEMV kernel,
    optionally followed in the same launch by `tail` (whose `partial` must be `out`).

    `x` is bf16 (quantised in the kernel per 1x128 group, or split in two e4m3 terms with
    `x_kind=X_BF16_SPLIT2`) or e4m3 (with `x_scale [m,k/128]`, or unscaled).  `push` (a
    `parallel.SymmSlot`) sends the rows to that slot's landing zone on every rank without
    running a tail, for a later `tail(...)` on the same slot.  `out_f32 [m,n]` receives the
    result before its bf16 rounding; with it and no `out` only the fp32 result is written
    (and returned)."""
    only_f32 = out is None and out_f32 is not None and tail is None and push is None
    if out is None and not only_f32:
        out = torch.empty(x.shape[0], w.shape[0], dtype=torch.bfloat16, device=x.device)
    if out_f32 is not None:
        _need("out_f32", out_f32, torch.float32, (x.shape[0], w.shape[0]), x.device)
    a = _linear_args(x, w, w_scale, out, x_kind, x_scale, block)
    a.out_f32 = _ptr(out_f32)
    a.scratch, a.scratch_bytes = scratch.ptr, scratch.bytes
    t = None
    if tail is not None:
        t = tail.to_c(scratch.ptr)
        a.tail = C.pointer(t)
    elif push is not None and push.world > 1 and push.protocol == "push":
        a.push = C.pointer(push.push_args())
    a.pdl = int(pdl)
    _lib.check("iq_linear", _lib.load().iq_linear(C.byref(a), _stream()))
    return out_f32 if only_f32 else out


def qkv_heads(qkv, w_qn, w_kn, cos, sin, slot, q_out, k_cache, v_cache, *, q_heads: int,
              kv_heads: int, rotary_dim: int, eps: float, scratch: Scratch | None = None,
              pdl: bool = False):
    """The attention prologue after the QKV product (`iq_qkv_heads`): `qkv [m, (q_heads +
    2 kv_heads) * D]` fp32 -> `q_out [m, q_heads, D]` bf16 (normalised, roped), k and v
    into rows `slot [m]` (int64) of `k_cache` / `v_cache [capacity, kv_heads, D]` (bf16 or
    e4m3)."""
    m = qkv.shape[0]
    dev = qkv.device
    d = q_out.shape[-1]
    _need("qkv", qkv, torch.float32, (m, (q_heads + 2 * kv_heads) * d), dev)
    _need("w_qn", w_qn, torch.float32, (d,), dev)
    _need("w_kn", w_kn, torch.float32, (d,), dev)
    _need("cos", cos, torch.bfloat16, (m, rotary_dim), dev)
    _need("sin", sin, torch.bfloat16, (m, rotary_dim), dev)
    _need("slot", slot, torch.int64, (m,), dev)
    _need("q_out", q_out, torch.bfloat16, (m, q_heads, d), dev)
    if k_cache.dtype not in (torch.bfloat16, E4M3) or v_cache.dtype != k_cache.dtype:
        raise ValueError("the KV caches must both be bf16 or both e4m3")
    cap = k_cache.shape[0]
    _need("k_cache", k_cache, k_cache.dtype, (cap, kv_heads, d), dev)
    _need("v_cache", v_cache, k_cache.dtype, (cap, kv_heads, d), dev)
    a = _lib.HeadsArgs()
    a.qkv = qkv.data_ptr()
    a.m, a.q_heads, a.kv_heads, a.head_dim, a.rotary_dim = m, q_heads, kv_heads, d, rotary_dim
    a.w_qn, a.w_kn, a.cos, a.sin = w_qn.data_ptr(), w_kn.data_ptr(), cos.data_ptr(), sin.data_ptr()
    a.eps, a.slot, a.q_out = float(eps), slot.data_ptr(), q_out.data_ptr()
    a.k_cache, a.v_cache, a.capacity = k_cache.data_ptr(), v_cache.data_ptr(), cap
    a.kv_kind = ACT_E4M3 if k_cache.dtype == E4M3 else ACT_BF16
    a.status = None if scratch is None else scratch.ptr
    a.pdl = int(pdl)
    _lib.check("iq_qkv_heads", _lib.load().iq_qkv_heads(C.byref(a), _stream()))
    return q_out


def router(x, weight, *, top_k: int, scratch: Scratch, score: int = ROUTE_SOFTMAX, sel=None,
           wt=None, logits=None, pdl: bool = False):
    """Router GEMV + top-k in one launch: returns `(sel int32 [m*top_k], wt fp32 [m*top_k],
    logits fp32 [m,e])`, pairs in ascending expert id per row."""
    m, h = x.shape
    e = weight.shape[0]
    dev = x.device
    _need("x", x, torch.bfloat16, None, dev)
    _need("weight", weight, torch.bfloat16, (e, h), dev)
    if sel is None:
        sel = torch.empty(m * top_k, dtype=torch.int32, device=dev)
    if wt is None:
        wt = torch.empty(m * top_k, dtype=torch.float32, device=dev)
    if logits is None:
        logits = torch.empty(m, e, dtype=torch.float32, device=dev)
    _need("sel", sel, torch.int32, None, dev)
    _need("wt", wt, torch.float32, None, dev)
    _need("logits", logits, torch.float32, (m, e), dev)
    if sel.numel() < m * top_k or wt.numel() < m * top_k:
        raise ValueError("sel/wt must hold m*top_k entries")
    a = _lib.RouterArgs()
    a.x, a.w = x.data_ptr(), weight.data_ptr()
    a.m, a.h, a.e, a.top_k, a.score = m, h, e, top_k, score
    a.sel, a.wt, a.logits = sel.data_ptr(), wt.data_ptr(), logits.data_ptr()
    a.scratch, a.scratch_bytes, a.pdl = scratch.ptr, scratch.bytes, int(pdl)
    _lib.check("iq_router", _lib.load().iq_router(C.byref(a), _stream()))
    return sel, wt, logits


def moe_gate(x_fp8, sel, fc, fc_scale, act, *, m: int, top_k: int, scratch: Scratch,
             x_scale=None, shared_fc=None, shared_fc_scale=None, pdl: bool = False):
    """Gate/Up + SiLU of the routed pairs of the first `m` rows (+ shared experts) into
    `act [m*(top_k+n_shared), i_loc]` (e4m3 unscaled, or bf16).  `x_fp8` is e4m3 (with
    `x_scale`, or unscaled) or bf16 (quantised per 1x128 group inside the kernel)."""
    e, two_i, h = fc.shape
    i_loc = two_i // 2
    dev = fc.device
    _need("fc", fc, E4M3, None, dev)
    _need("fc_scale", fc_scale, torch.float32, (e, two_i // 64, h // 128), dev)
    x_is_bf16 = x_fp8.dtype == torch.bfloat16
    _need("x", x_fp8, torch.bfloat16 if x_is_bf16 else E4M3, None, dev)
    if x_fp8.shape[-1] != h or x_fp8.shape[0] < m:
        raise ValueError(f"x must be [>= {m}, {h}], got {tuple(x_fp8.shape)}")
    _need("sel", sel, torch.int32, None, dev)
    n_shared = 0
    if shared_fc is not None:
        n_shared = 1 if shared_fc.dim() == 2 else shared_fc.shape[0]
        _need("shared_fc", shared_fc, E4M3, None, dev)
        _need("shared_fc_scale", shared_fc_scale, torch.float32, None, dev)
        if shared_fc.numel() != n_shared * two_i * h:
            raise ValueError("shared_fc must have the experts' [2*i_loc, h] shape")
    slots = top_k + n_shared
    if act.dtype not in (E4M3, torch.bfloat16):
        raise ValueError("act must be e4m3 or bf16")
    _need("act", act, act.dtype, None, dev)
    if act.numel() < m * slots * i_loc:
        raise ValueError("act too small")
    if x_scale is not None:
        _need("x_scale", x_scale, torch.float32, None, dev)
    a = _lib.MoeGateArgs()
    if x_is_bf16:
        a.x_bf16 = x_fp8.data_ptr()
    else:
        a.x_fp8, a.x_scale = x_fp8.data_ptr(), _ptr(x_scale)
    a.m, a.h, a.i_loc, a.n_experts, a.top_k, a.n_shared = m, h, i_loc, e, top_k, n_shared
    a.sel, a.fc, a.fc_scale = sel.data_ptr(), fc.data_ptr(), fc_scale.data_ptr()
    a.shared_fc, a.shared_fc_scale = _ptr(shared_fc), _ptr(shared_fc_scale)
    a.act, a.act_kind = act.data_ptr(), ACT_E4M3 if act.dtype == E4M3 else ACT_BF16
    a.scratch, a.scratch_bytes, a.pdl = scratch.ptr, scratch.bytes, int(pdl)
    _lib.check("iq_moe_gate", _lib.load().iq_moe_gate(C.byref(a), _stream()))
    return act


def moe_down(act, sel, wt, proj, proj_scale, out, *, m: int, top_k: int, scratch: Scratch,
             shared_proj=None, shared_proj_scale=None, tail: TailSpec | None = None,
             push=None, pdl: bool = False):
    """Down of the routed pairs (+ shared experts) into `out[:m]` bf16 `[m,h]`, optionally
    followed in the same launch by `tail`; `push` as in `linear`."""
    e, h, i_loc = proj.shape
    dev = proj.device
    _need("proj", proj, E4M3, None, dev)
    _need("proj_scale", proj_scale, torch.float32, (e, h // 128, i_loc // 64), dev)
    _need("sel", sel, torch.int32, None, dev)
    _need("wt", wt, torch.float32, None, dev)
    _need("out", out, torch.bfloat16, None, dev)
    if out.shape[-1] != h or out.shape[0] < m:
        raise ValueError(f"out must be [>= {m}, {h}]")
    n_shared = 0
    if shared_proj is not None:
        n_shared = 1 if shared_proj.dim() == 2 else shared_proj.shape[0]
        _need("shared_proj", shared_proj, E4M3, None, dev)
        _need("shared_proj_scale", shared_proj_scale, torch.float32, None, dev)
    if act.dtype not in (E4M3, torch.bfloat16):
        raise ValueError("act must be e4m3 or bf16")
    _need("act", act, act.dtype, None, dev)
    a = _lib.MoeDownArgs()
    a.act, a.act_kind = act.data_ptr(), ACT_E4M3 if act.dtype == E4M3 else ACT_BF16
    a.m, a.h, a.i_loc, a.n_experts, a.top_k, a.n_shared = m, h, i_loc, e, top_k, n_shared
    a.sel, a.wt = sel.data_ptr(), wt.data_ptr()
    a.proj, a.proj_scale = proj.data_ptr(), proj_scale.data_ptr()
    a.shared_proj, a.shared_proj_scale = _ptr(shared_proj), _ptr(shared_proj_scale)
    a.out = out.data_ptr()
    a.scratch, a.scratch_bytes = scratch.ptr, scratch.bytes
    t = None
    if tail is not None:
        t = tail.to_c(scratch.ptr)
        a.tail = C.pointer(t)
    elif push is not None and push.world > 1 and push.protocol == "push":
        a.push = C.pointer(push.push_args())
    a.pdl = int(pdl)
    _lib.check("iq_moe_down", _lib.load().iq_moe_down(C.byref(a), _stream()))
    return out[:m]


def linear_static(x, w, w_scale, out, *, x_kind=None, x_scale=None, block=(128, 128),
                  pdl: bool = False):
    """`linear` for callers that cannot allocate device memory where they call it (inside a
    host application's stream capture, or with a memory budget spent in full at start-up):
    the kernel's work area is a device array built into the library, so no scratch buffer
    is passed and `out` must be given.  Limits: n, k <= 65536, no fused tail.  All calls on
    a device share that array, so order them on one stream; the first call on a device
    should come before any stream capture.  A device-side error of the call stays readable
    through `linear_static_status` until the next `linear_static` on the device."""
    a = _linear_args(x, w, w_scale, out, x_kind, x_scale, block)
    a.pdl = int(pdl)
    _lib.check("iq_linear_static", _lib.load().iq_linear_static(C.byref(a), _stream()))
    return out


def linear_static_status() -> int:
    """Synchronises the current stream and returns the device status code the last
    `linear_static` call on this device left (0 = none)."""
    code = C.c_int(0)
    _lib.check("iq_linear_static_status",
               _lib.load().iq_linear_static_status(C.byref(code), _stream()))
    return code.value


# ---------------------------------------------------------------------- the paged KV cache
# These calls are a few microseconds of device time each, so their checks read every
# tensor's properties once and the arguments are packed in one go.
_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def _on(index, name, packed):
    """Calls entry point `name` on device `index`'s current stream, with it as the current
    device."""
    fn = getattr(_lib.load(), name)
    if index == torch._C._cuda_getDevice():
        code = fn(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            code = fn(packed, torch._C._cuda_getCurrentRawStream(index))
    if code:
        raise _lib.IqError(name, code)


def _take(name, t, dtype, shape, index):
    """Checks a tensor whose last axis is contiguous; returns its strides."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must have dtype {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors are on "
                         f"{'cpu' if index < 0 else f'cuda:{index}'}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must be contiguous along its last axis")
    return st


def _take_out(name, t, dtype, shape, index):
    """`_take` for a tensor that is written: no two elements at one address."""
    st = _take(name, t, dtype, shape, index)
    if not t.is_contiguous():
        reach = 1
        for size, step in sorted(zip(shape, st), key=lambda x: x[1]):
            if size > 1:
                if step < reach:
                    raise ValueError(f"{name} must not overlap itself (strides {st})")
                reach += step * (size - 1)
    return st


def _cache_pair(k_cache, v_cache, index):
    if not isinstance(k_cache, torch.Tensor) or k_cache.dim() != 3:
        raise ValueError("the KV caches must be [capacity, kv_heads, head_dim] tensors")
    dtype, shape = k_cache.dtype, k_cache.shape
    if dtype is not _BF16 and dtype is not E4M3:
        raise ValueError("the KV caches must both be bf16 or both e4m3")
    return (shape, ACT_E4M3 if dtype is E4M3 else ACT_BF16,
            _take_out("k_cache", k_cache, dtype, shape, index),
            _take_out("v_cache", v_cache, dtype, shape, index))


def _pages(page_table, page_size, batch, index):
    """(stride of the table's rows, pages a row); checks the table and the page size."""
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise ValueError("page_table must be a [batch, pages] tensor")
    shape = page_table.shape
    st = _take("page_table", page_table, _I32, shape, index)
    if shape[0] != batch or shape[1] < 1:
        raise ValueError(f"page_table must be [{batch}, pages >= 1], got {tuple(shape)}")
    if page_size < 1:
        raise ValueError(f"page_size must be at least 1, got {page_size}")
    return st[0], shape[1]


def _gpu(name, index):
    if index < 0:
        raise ValueError(f"{name} must be a CUDA tensor")


def _status(scratch, index):
    """Address of the status word; a kernel that finds an error writes there."""
    if scratch is None:
        return 0
    if scratch.index != index:
        raise ValueError(f"scratch must be on cuda:{index}, got {scratch.buf.device}")
    return scratch.ptr


class AttnWork:
    """The work area of `attn_decode` for given sizes (`rows`: page_size x pages of the page
    table; `weights`: for calls that accumulate weights).  Calls that share one must be
    ordered on one stream, replays of graphs that captured it included."""

    def __init__(self, *, batch: int, q_len: int, q_heads: int, kv_heads: int, head_dim: int,
                 rows: int, weights: bool = False, device="cuda"):
        self.bytes = int(_lib.load().iq_attn_work_bytes(batch, q_len, q_heads, kv_heads, head_dim,
                                                        rows, int(weights)))
        if self.bytes == 0:
            raise ValueError(
                f"unsupported attention shape: batch {batch}, q_len {q_len}, heads {q_heads}/"
                f"{kv_heads}, head_dim {head_dim}, rows {rows} (head_dim a multiple of 16 up to "
                "256, q_len 1..8, batch up to 1024, q_heads a multiple of kv_heads and at most "
                "512 query rows a key/value head)")
        self.buf = torch.empty(self.bytes, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr()
        self.index = self.buf.get_device()


def attn_decode(q, k_cache, v_cache, page_table, lengths, *, page_size: int, scale=None,
                window: int = 0, out=None, lse=None, weights=None, positions=None, seen=None,
                slot=None, work: AttnWork | None = None, scratch: Scratch | None = None, pdl: bool = True):
    """Attention of the last `q_len` tokens of each sequence over its paged KV cache
    (`iq_attn_decode`): `q [batch, q_len, q_heads, D]` bf16 -> `out`, same shape.

    `k_cache` / `v_cache [capacity, kv_heads, D]` are what `qkv_heads` writes (bf16, or e4m3,
    with which each row of q is rounded to 2^-25 of its largest element or finer),
    row j of sequence b being row `page_table[b, j // page_size] * page_size + j % page_size`;
    `lengths [batch]` (int32) counts the rows with the new ones.  New token r sees the rows up
    to its own, the last `window` of them if `window` is not 0: rows of the cache, whose order
    is that of the tokens until `kv_evict` cuts the sequence, so not for such a cache.  A token
    that sees nothing gets zeros, and -inf in `lse [batch, q_len, q_heads]` (fp32, optional).  `scale` defaults
    to D ** -0.5.

    `weights [batch, kv_heads, >= rows]` (fp32) gains each row's softmax weights, summed over
    the query heads of its key/value head and the new tokens; the new tokens' own entries are
    set, and those of `positions` (int32, same shape) to the tokens' positions, `seen [batch]`
    (int32) being the tokens seen so far with the new ones.  With `slot [batch * q_len]` (int64,
    what `kv_advance` wrote) a sequence that had no room for the new tokens (slots of -1) keeps
    its weights and positions; what its rows of `out` hold means nothing.  Without `work` one is allocated
    for the call.  A length or page out of range shows in `scratch`'s status word.  `pdl` lets
    the launch's set-up overlap the kernel before it; nothing is read or written before that
    kernel is done.

    Addresses of q, out and the caches, and their strides, are multiples of 16 bytes."""
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be a tensor [batch, q_len, q_heads, head_dim]")
    shape, index = q.shape, q.get_device()
    batch, q_len, q_heads, d = shape
    qs = _take("q", q, _BF16, shape, index)
    (capacity, kv_heads, kd), kind, ks, vs = _cache_pair(k_cache, v_cache, index)
    if kd != d or kv_heads < 1 or q_heads % kv_heads:
        raise ValueError(f"q {tuple(shape)} does not fit caches of {kv_heads} heads of {kd}")
    ts, pages = _pages(page_table, page_size, batch, index)
    _take("lengths", lengths, _I32, (batch,), index)
    if window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    window = min(window, page_size * pages)      # (more is no window, however much it is)
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=q.device)
    os_ = _take_out("out", out, _BF16, shape, index)
    lse_ptr = w_ptr = pos_ptr = seen_ptr = slot_ptr = w_rows = 0
    ws = ps = (0, 0)
    if lse is not None:
        _take("lse", lse, _F32, shape[:3], index)
        if not lse.is_contiguous():
            raise ValueError("lse must be contiguous")
        lse_ptr = lse.data_ptr()
    if weights is not None:
        if weights.dim() != 3 or weights.shape[2] < page_size * pages:
            raise ValueError(f"weights must be [{batch}, {kv_heads}, >= {page_size * pages}], got "
                             f"{tuple(weights.shape)}")
        w_rows = weights.shape[2]
        ws = _take_out("weights", weights, _F32, (batch, kv_heads, w_rows), index)
        w_ptr = weights.data_ptr()
    if (positions is None) != (seen is None) or (positions is not None and weights is None):
        raise ValueError("positions and seen come together, with weights")
    if positions is not None:
        ps = _take_out("positions", positions, _I32, weights.shape, index)
        _take("seen", seen, _I32, (batch,), index)
        pos_ptr, seen_ptr = positions.data_ptr(), seen.data_ptr()
    if slot is not None:
        if weights is None:
            raise ValueError("slot comes with weights")
        _take("slot", slot, _I64, (batch * q_len,), index)
        slot_ptr = slot.data_ptr()
    _gpu("q", index)
    if work is None:
        work = AttnWork(batch=batch, q_len=q_len, q_heads=q_heads, kv_heads=kv_heads, head_dim=d,
                        rows=page_size * pages, weights=weights is not None, device=q.device)
    elif work.index != index:
        raise ValueError(f"work must be on cuda:{index}, got {work.buf.device}")
    _on(index, "iq_attn_decode", _lib.PACK_ATTN.pack(
        q.data_ptr(), qs[0], qs[1], qs[2], k_cache.data_ptr(), v_cache.data_ptr(),
        ks[0], ks[1], vs[0], vs[1], kind, capacity, page_table.data_ptr(), ts, page_size, pages,
        lengths.data_ptr(), batch, q_len, q_heads, kv_heads, d, window,
        d ** -0.5 if scale is None else scale, out.data_ptr(), os_[0], os_[1], os_[2], lse_ptr,
        w_ptr, ws[0], ws[1], w_rows, pos_ptr, ps[0], ps[1], seen_ptr, slot_ptr, work.ptr, work.bytes,
        _status(scratch, index), int(pdl)))
    return out


class EvictWork:
    """The work area of `kv_evict` for given sizes (`rows`: page_size x pages of the page
    table).  Calls that share one must be ordered on one stream."""

    def __init__(self, *, batch: int, kv_heads: int, rows: int, device="cuda"):
        self.bytes = int(_lib.load().iq_evict_work_bytes(batch, kv_heads, rows))
        if self.bytes == 0:
            raise ValueError(f"unsupported eviction shape: batch {batch}, {kv_heads} heads, {rows} "
                             "rows (batch x heads up to 65535, rows up to 262144)")
        self.buf = torch.empty(self.bytes, dtype=torch.uint8, device=device)
        self.ptr = self.buf.data_ptr()
        self.index = self.buf.get_device()


def kv_evict(k_cache, v_cache, page_table, lengths, weights, positions, seen, *, page_size: int,
             budget: int, lengths_out, keep_first: int = 0, keep_last: int = 0, weights_out=None,
             positions_out=None, work: EvictWork | None = None, scratch: Scratch | None = None,
             pdl: bool = True):
    """Cuts every sequence of more than `budget` rows down to `budget` (`iq_kv_evict`): each
    key/value head keeps its rows of position < `keep_first` or >= `seen - keep_last`, then
    those of the largest accumulated weight (ties to the lower row).

    `weights` (fp32) and `positions` (int32) are `[batch, kv_heads, >= rows]` as `attn_decode`
    keeps them.  Rows that stay below `budget` stay where they are; the others move, in place
    and in ascending order, into the places freed there, with their weights and positions
    (`weights_out` / `positions_out`, by default the inputs themselves).  `lengths_out [batch]`
    (int32, not in the memory of `lengths` or `seen`: layers of a model share the lengths of
    before) gets the new lengths.  Sequences must not share pages.  The rows' order is given up
    with that (`positions` keeps it): a window of `attn_decode` would count the wrong rows."""
    if not isinstance(weights, torch.Tensor) or weights.dim() != 3:
        raise ValueError("weights must be a tensor [batch, kv_heads, rows]")
    shape, index = weights.shape, weights.get_device()
    batch, kv_heads, n = shape
    (capacity, kh, d), kind, ks, vs = _cache_pair(k_cache, v_cache, index)
    ts, pages = _pages(page_table, page_size, batch, index)
    if kh != kv_heads or n < page_size * pages:
        raise ValueError(f"weights must be [{batch}, {kh}, >= {page_size * pages}], got "
                         f"{tuple(shape)}")
    if budget < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
        raise ValueError(f"budget must be at least 1 and hold the protected rows, got {budget} for "
                         f"{keep_first} + {keep_last}")
    weights_out = weights if weights_out is None else weights_out
    positions_out = positions if positions_out is None else positions_out
    ws = _take("weights", weights, _F32, shape, index)
    ps = _take("positions", positions, _I32, shape, index)
    wo = _take_out("weights_out", weights_out, _F32, shape, index)
    po = _take_out("positions_out", positions_out, _I32, shape, index)
    _take("lengths", lengths, _I32, (batch,), index)
    _take("seen", seen, _I32, (batch,), index)
    _take("lengths_out", lengths_out, _I32, (batch,), index)
    n_ptr, out_ptr = lengths.data_ptr(), lengths_out.data_ptr()
    if abs(out_ptr - n_ptr) < 4 * batch:
        raise ValueError("lengths_out must not be lengths")
    _gpu("weights", index)
    if work is None:
        work = EvictWork(batch=batch, kv_heads=kv_heads, rows=page_size * pages,
                         device=weights.device)
    elif work.index != index:
        raise ValueError(f"work must be on cuda:{index}, got {work.buf.device}")
    _on(index, "iq_kv_evict", _lib.PACK_EVICT.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], vs[0], vs[1], kind, capacity,
        page_table.data_ptr(), ts, page_size, pages, n_ptr, seen.data_ptr(), weights.data_ptr(),
        ws[0], ws[1], positions.data_ptr(), ps[0], ps[1], weights_out.data_ptr(), wo[0], wo[1],
        positions_out.data_ptr(), po[0], po[1], out_ptr, batch, kv_heads, d, budget, keep_first,
        keep_last, work.ptr, work.bytes, _status(scratch, index), int(pdl)))
    return lengths_out


def kv_advance(page_table, lengths, seen, slot, pos, *, page_size: int, capacity: int,
               q_len: int = 1, max_positions: int = 0, lengths_out=None, seen_out=None,
               scratch: Scratch | None = None, pdl: bool = True):
    """The cache rows and positions of the next `q_len` tokens of every sequence
    (`iq_kv_advance`), on the device, so that a captured step finds its own rows: `slot` and
    `pos [batch * q_len]` (int64) are what `qkv_heads` and the rotary tables take.  `lengths`
    and `seen [batch]` (int32) grow by `q_len`, in place unless `lengths_out` / `seen_out` are
    given.  A sequence whose pages end before, or whose positions would reach `max_positions`
    (the rows of a rotary table; 0: no limit), gets slots of -1, which `qkv_heads` refuses to
    write, and positions of 0, and stays as it was (with `scratch`'s status word set)."""
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("lengths must be a tensor [batch]")
    shape, index = lengths.shape, lengths.get_device()
    batch = shape[0]
    if not 1 <= q_len <= 8:
        raise ValueError(f"q_len must be 1..8, got {q_len}")
    if batch < 1 or capacity < 1 or max_positions < 0:
        raise ValueError("batch and capacity must be at least 1, max_positions not negative")
    ts, pages = _pages(page_table, page_size, batch, index)
    lengths_out = lengths if lengths_out is None else lengths_out
    seen_out = seen if seen_out is None else seen_out
    _take("lengths", lengths, _I32, shape, index)
    _take("seen", seen, _I32, shape, index)
    _take("lengths_out", lengths_out, _I32, shape, index)
    _take("seen_out", seen_out, _I32, shape, index)
    _take("slot", slot, _I64, (batch * q_len,), index)
    _take("pos", pos, _I64, (batch * q_len,), index)
    _gpu("lengths", index)
    _on(index, "iq_kv_advance", _lib.PACK_ADVANCE.pack(
        page_table.data_ptr(), ts, page_size, pages, capacity, lengths.data_ptr(), seen.data_ptr(),
        lengths_out.data_ptr(), seen_out.data_ptr(), slot.data_ptr(), pos.data_ptr(), batch, q_len,
        max_positions, _status(scratch, index), int(pdl)))
    return slot, pos
