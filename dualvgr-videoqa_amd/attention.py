"""Host side of include/dvgr_attn.h: multi-head attention to an encoder's states of another length, forward and backward --
`cross_attention` on tensors, `CrossAttention` with its projections on `HipLinear`.  The words of a question over the frames of its
video, clips over words, one word of an answer over everything.  No CPU / eager fallback."""
from __future__ import annotations

import ctypes as C
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L_
from .inputs import HipLinear

MAX_HEAD = 128


def _ready(t):
    """`t`, or a copy whose heads start at multiples of 16 bytes."""
    per = 16 // t.element_size()
    if t.stride(3) != 1 or t.stride(2) % per or t.stride(1) % per or t.stride(0) % per or t.data_ptr() & 15:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _view(t):
    return L_.AttnView(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _problem(q, k, v, o, lens, mask, scale, lse):
    B, Lq, H, Dh = q.shape
    return L_.AttnProblem(B, Lq, k.shape[1], H, k.shape[2], Dh, L_.elem_code(q, "cross_attention"), scale, _view(q), _view(k), _view(v), _view(o),
                          lens.data_ptr() if lens is not None else None, mask.data_ptr() if mask is not None else None,
                          mask.stride(0) if mask is not None else 0, lse.data_ptr() if lse is not None else None)


def _forward(q, k, v, lens, mask, scale, want_lse):
    lib = L_.load()
    B, Lq, H, Dh = q.shape
    o = torch.empty(B, Lq, H, Dh, device=q.device, dtype=q.dtype)
    lse = torch.empty(B, H, Lq, device=q.device, dtype=torch.float32) if want_lse else None
    a = _problem(q, k, v, o, lens, mask, scale, lse)
    L_.check(lib.dvgr_attn_check(C.byref(a)), "dvgr_attn_check")
    nbytes = lib.dvgr_attn_forward_workspace_bytes(C.byref(a))
    ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8) if nbytes else None
    here, stream = L_.on(q)
    with here:
        L_.check(lib.dvgr_attn_forward(C.byref(a), ws.data_ptr() if nbytes else None, nbytes, stream), "dvgr_attn_forward")
    return o, lse


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lens, mask, scale):
        L_.note_graph(ctx, torch.cuda.current_stream(q.device).cuda_stream, q, k, v)
        q, k, v = _ready(q), _ready(k), _ready(v)
        o, lse = _forward(q, k, v, lens, mask, scale, True)
        ctx.save_for_backward(q, k, v, o, lse, lens, mask)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        lib = L_.load()
        L_.check_capture(ctx, "cross_attention")
        q, k, v, o, lse, lens, mask = ctx.saved_tensors
        g = _ready(g)
        need_q, need_kv = ctx.needs_input_grad[0], ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        new = lambda t, need: torch.empty(t.shape, device=t.device, dtype=t.dtype) if need else None  # noqa: E731
        gq, gk, gv = new(q, need_q), new(k, need_kv), new(v, need_kv)
        a = _problem(q, k, v, o, lens, mask, ctx.scale, lse)
        none = L_.AttnView(None, 0, 0, 0)
        gr = L_.AttnGrads(_view(g), _view(gq) if need_q else none, _view(gk) if need_kv else none, _view(gv) if need_kv else none)
        nbytes = lib.dvgr_attn_backward_workspace_bytes(C.byref(a))
        ws = torch.empty(nbytes, device=q.device, dtype=torch.uint8)
        here, stream = L_.on(q)
        with here:
            L_.check(lib.dvgr_attn_backward(C.byref(a), C.byref(gr), ws.data_ptr(), nbytes, stream), "dvgr_attn_backward")
        return gq, gk if ctx.needs_input_grad[1] else None, gv if ctx.needs_input_grad[2] else None, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor = None, mask: torch.Tensor = None,
                    scale: float = None) -> torch.Tensor:
    """softmax(scale q k^T) v per head: q (B, Lq, H, Dh), k and v (B, Lk, Hk, Dh) -> (B, Lq, H, Dh).

    fp32, bf16 or fp16; Dh a multiple of 8 up to 128; H a multiple of Hk (query head h reads key head h // (H // Hk)).  Any strides
    (heads that do not start at multiples of 16 bytes are copied first).  Key j of sample b is there if j < lens[b] (integers (B),
    clamped to [0, Lk]) and mask[b, j] (bool (B, Lk)); keys that are not there are never used, NaN included, and get zero gradients.
    A query without keys gives zeros.  scale > 0, default 1 / sqrt(Dh).  Without a gradient wanted (one word at a time, serving)
    nothing is kept for a backward."""
    L_.elem_code(q, "cross_attention")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise RuntimeError(f"cross_attention: q (B, Lq, H, Dh), k and v (B, Lk, Hk, Dh); got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, _, H, Dh = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    if k.dtype != q.dtype or v.dtype != q.dtype or k.device != q.device or v.device != q.device:
        raise RuntimeError("cross_attention: q, k and v have one type and are on one device")
    if Hk < 1 or H < 1 or H % Hk:
        raise RuntimeError(f"cross_attention: the query heads ({H}) are a multiple of the key heads ({Hk})")
    if Dh % 8 or not 8 <= Dh <= MAX_HEAD:
        raise RuntimeError(f"cross_attention: the head size is a multiple of 8 up to {MAX_HEAD}; got {Dh}")
    scale = 1.0 / math.sqrt(Dh) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise RuntimeError(f"cross_attention: scale is a positive number; got {scale}")
    if lens is not None:
        if tuple(lens.shape) != (B,) or lens.device != q.device or lens.dtype not in (torch.int64, torch.int32):
            raise RuntimeError(f"cross_attention: lens is (B) int64 or int32 on q's device; got {tuple(lens.shape)} {lens.dtype} on {lens.device}")
        lens = lens.long().contiguous()
    if mask is not None:
        if tuple(mask.shape) != (B, Lk) or mask.device != q.device or mask.dtype != torch.bool:
            raise RuntimeError(f"cross_attention: mask is (B, Lk) bool on q's device; got {tuple(mask.shape)} {mask.dtype} on {mask.device}")
        if mask.stride(1) != 1:
            mask = mask.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attend.apply(q, k, v, lens, mask, scale)
    return _forward(_ready(q), _ready(k), _ready(v), lens, mask, scale, False)[0]


class CrossAttention(nn.Module):
    """Attention of (B, Lq, module_dim) to an encoder's states (B, Lk, state_dim), with its projections on `HipLinear`.

    `states()` gives the states' keys and values: a program that answers word by word calls it once for a video and passes the pair
    as `kv` from then on.  dtype 'fp32' | 'bf16x3' | 'bf16' as for the unit: the operand format of the projections; with 'bf16' the
    attention takes bf16 tensors too."""

    def __init__(self, module_dim: int = 768, num_heads: int = 8, state_dim: int = None, key_heads: int = None, dtype: str = "fp32"):
        super().__init__()
        if module_dim % num_heads:
            raise ValueError(f"module_dim {module_dim} is not a multiple of num_heads {num_heads}")
        self.num_heads, self.key_heads = int(num_heads), int(key_heads or num_heads)
        self.head_dim = module_dim // num_heads
        if self.num_heads % self.key_heads or self.head_dim % 8 or self.head_dim > MAX_HEAD:
            raise ValueError(f"num_heads is a multiple of key_heads, the head size a multiple of 8 up to {MAX_HEAD}; got {num_heads}, "
                             f"{self.key_heads}, {self.head_dim}")
        self.half = dtype == "bf16"
        self.query = HipLinear(module_dim, module_dim, dtype=dtype)
        self.key_value = HipLinear(state_dim or module_dim, 2 * self.key_heads * self.head_dim, dtype=dtype)
        self.out = HipLinear(module_dim, module_dim, dtype=dtype)

    def states(self, states: torch.Tensor):
        """(B, Lk, state_dim) -> (keys, values), each (B, Lk, key_heads, head_dim): two views of one projection."""
        kv = self.key_value(states)
        if self.half:
            kv = kv.to(torch.bfloat16)
        kv = kv.view(*states.shape[:2], 2, self.key_heads, self.head_dim)
        return kv[:, :, 0], kv[:, :, 1]

    def forward(self, x: torch.Tensor, states: torch.Tensor = None, lens: torch.Tensor = None, mask: torch.Tensor = None, kv=None):
        if (states is None) == (kv is None):
            raise RuntimeError("CrossAttention takes the encoder's states or the keys and values made of them")
        k, v = self.states(states) if kv is None else kv
        q = self.query(x)
        if self.half:
            q = q.to(torch.bfloat16)
        o = cross_attention(q.view(*x.shape[:2], self.num_heads, self.head_dim), k, v, lens, mask)
        return self.out(o.reshape(*x.shape[:2], -1).float())
