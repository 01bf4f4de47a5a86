"""Host side of include/dvgr_attn.h: multi-head attention to an encoder's states of another length, forward and backward --
`cross_attention` on tensors, `CrossAttention` with its projections on `HipLinear`.  The words of a question over the frames of its
video, clips over words, one word of an answer over everything.  No CPU / eager fallback."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib as L_
from .inputs import HipLinear

MAX_HEAD = 128


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor = None, mask: torch.Tensor = None,
                    scale: float = None) -> torch.Tensor:
    """softmax(scale q k^T) v per head: q (B, Lq, H, Dh), k and v (B, Lk, Hk, Dh) -> (B, Lq, H, Dh).

    fp32, bf16 or fp16; Dh a multiple of 8 up to 128; H a multiple of Hk (query head h reads key head h // (H // Hk)).  Any strides
    (heads that do not start at multiples of 16 bytes are copied first).  Key j of sample b is there if j < lens[b] (integers (B),
    clamped to [0, Lk]) and mask[b, j] (bool (B, Lk)); keys that are not there are never used, NaN included, and get zero gradients.
    A query without keys gives zeros.  1e-30 <= scale <= 1e30, default 1 / sqrt(Dh).  Without a gradient wanted (one word at a time, serving)
    nothing is kept for a backward."""
    return L_.torch_ops().cross_attention(q, k, v, lens, mask, scale)


def _fp32(t: torch.Tensor, name: str) -> torch.Tensor:
    """`t` as the projections take it (its gradient comes back in its own type)."""
    if t.dim() != 3 or t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"CrossAttention: {name}: (batch, length, features) in fp32, bf16 or fp16; got {tuple(t.shape)} {t.dtype}")
    return t.float()


class CrossAttention(nn.Module):
    """Attention of (B, Lq, module_dim) to an encoder's states (B, Lk, state_dim), with its projections on `HipLinear`.

    `states()` gives the states' keys and values: a program that answers word by word calls it once for a video and passes the pair
    as `kv` from then on.  dtype 'fp32' | 'bf16x3' | 'bf16' as for the unit: the operand format of the projections; with 'bf16' the
    attention takes bf16 tensors too.  Inputs in fp32, bf16 or fp16 (an embedding's, say); parameters and output are fp32."""

    def __init__(self, module_dim: int = 768, num_heads: int = 8, state_dim: int = None, key_heads: int = None, dtype: str = "fp32"):
        super().__init__()
        if module_dim % num_heads:
            raise ValueError(f"module_dim {module_dim} is not a multiple of num_heads {num_heads}")
        self.num_heads, self.key_heads = int(num_heads), int(key_heads or num_heads)
        self.head_dim = module_dim // num_heads
        if self.num_heads % self.key_heads or self.head_dim % 8 or self.head_dim > MAX_HEAD:
            raise ValueError(f"num_heads is a multiple of key_heads, the head size a multiple of 8 up to {MAX_HEAD}; got {num_heads}, "
                             f"{self.key_heads}, {self.head_dim}")
        self.bf16_attention = dtype == "bf16"
        self.query = HipLinear(module_dim, module_dim, dtype=dtype)
        self.key_value = HipLinear(state_dim or module_dim, 2 * self.key_heads * self.head_dim, dtype=dtype)
        self.out = HipLinear(module_dim, module_dim, dtype=dtype)

    def states(self, states: torch.Tensor):
        """(B, Lk, state_dim) -> (keys, values), each (B, Lk, key_heads, head_dim): two views of one projection."""
        kv = self.key_value(_fp32(states, "the encoder's states"))
        if self.bf16_attention:
            kv = kv.to(torch.bfloat16)
        kv = kv.view(*states.shape[:2], 2, self.key_heads, self.head_dim)
        return kv[:, :, 0], kv[:, :, 1]

    def forward(self, x: torch.Tensor, states: torch.Tensor = None, lens: torch.Tensor = None, mask: torch.Tensor = None, kv=None):
        if (states is None) == (kv is None):
            raise RuntimeError("CrossAttention takes the encoder's states or the keys and values made of them")
        x = _fp32(x, "the input")
        k, v = self.states(states) if kv is None else kv
        q = self.query(x)
        if self.bf16_attention:
            q = q.to(torch.bfloat16)
        o = cross_attention(q.view(*x.shape[:2], self.num_heads, self.head_dim), k, v, lens, mask)
        return self.out(o.reshape(*x.shape[:2], -1).float())
