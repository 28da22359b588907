"""A key / value cache held in 8 bits, and rotary positions as the kernels take them.

``KV8Cache`` holds e4m3 codes with one power-of-two scale per block of tokens and kv head; ``ops.kv8_append`` writes
it, ``ops.kv8_load`` reads it back as bfloat16, ``ops.flash_decode_kv8`` attends over it.  Half the bytes of the bf16
cache of ``runtime.FlashSVDV15DenseKVCache``, for the same number of tokens; ``runtime.FlashSVDV15KV8Cache`` holds one per
layer of a model.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from ._lib import FsvdKv8

BLOCKS = (16, 32, 64, 128)


def made_once(what: str, device, make):
    """What ``make`` puts on a device for later calls to keep.  They may come from any stream, so it is complete when this
    returns; a graph capture would only record how to make it, so there it is refused."""
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} made at the first use, which cannot be captured: make such a call before the capture")
        made = make()
        torch.cuda.current_stream().synchronize()
    return made


@dataclass
class Rotary:
    """``inv_freq``: float64 CUDA tensor [rotary_dim / 2], radians per position; ``interleaved``: pairs (2i, 2i + 1)
    instead of (i, i + rotary_dim / 2); ``scale`` multiplies cos and sin."""

    inv_freq: torch.Tensor
    interleaved: bool = False
    scale: float = 1.0


def rotary(rotary_dim: int, *, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained_len: int = 0,
           low: float = 1.0, high: float = 32.0, interleaved: bool = False, device="cuda") -> Rotary:
    """Frequencies ``theta ** (-2 i / rotary_dim)`` in 64 bits, stretched ``factor`` times for contexts longer than the
    trained one:

    ``"linear"``  every frequency divided by the factor;
    ``"ntk"``     a larger theta: the slowest pair turns ``factor`` times slower, the fastest as it was;
    ``"yarn"``    pairs that turn at least ``high`` times over ``trained_len`` positions stay, those that turn at most
                  ``low`` times are divided by the factor, a linear ramp in the number of turns between them; cos and
                  sin are multiplied by 0.1 ln(factor) + 1.
    """
    R = int(rotary_dim)
    if R < 2 or R % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError(f"unknown rotary scaling {scaling!r} (none, linear, ntk, yarn)")
    if not (factor >= 1.0 and math.isfinite(factor)):
        raise ValueError(f"the factor must be at least 1, got {factor}")
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive, got {theta}")
    theta, scale = float(theta), 1.0
    if scaling == "ntk" and R > 2:
        theta *= float(factor) ** (R / (R - 2))
    f = theta ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if trained_len <= 0 or not high > low:
            raise ValueError("yarn needs trained_len > 0 and high > low")
        keep = ((trained_len * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    return Rotary(f.to(device), interleaved, scale)


class KV8Cache:
    """``k`` / ``v`` [B, Hk, S_max, Dh] float8_e4m3fn codes (a head's tokens lie together: a tile of them is one piece
    of memory), ``k_scale`` / ``v_scale`` [B, Hk, ceil(S_max / block)] float32.  A code stands for code * scale."""

    __slots__ = ("_k", "_v", "_k_scale", "_v_scale", "_block", "index", "struct", "ref")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block: int = 64):
        if k.ndim != 4:
            raise ValueError(f"k must be [B, Hk, S_max, Dh], got {tuple(k.shape)}")
        shape = k.shape
        B, Hk, S, Dh = shape
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block}")
        if Dh != 128 and Dh != 64:
            raise ValueError(f"head_dim {Dh} unsupported (64, 128)")
        if B < 1 or Hk < 1 or S < 1:
            raise ValueError(f"empty cache {tuple(shape)}")
        if v.shape != shape:
            raise ValueError("v shape must match k")
        if k.dtype is not torch.float8_e4m3fn or v.dtype is not torch.float8_e4m3fn:
            raise ValueError("the codes are float8_e4m3fn tensors")
        want = (B, Hk, -(-S // block))
        if k_scale.shape != want or v_scale.shape != want or k_scale.dtype is not torch.float32 or v_scale.dtype is not torch.float32:
            raise ValueError(f"k_scale and v_scale must be float32 {want}, got {k_scale.dtype} {tuple(k_scale.shape)} and "
                             f"{v_scale.dtype} {tuple(v_scale.shape)}")
        index = k.get_device()
        if index < 0 or not (index == v.get_device() == k_scale.get_device() == v_scale.get_device()):
            raise ValueError("the cache is CUDA tensors of one device (there is no CPU path)")
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
            raise ValueError("the cache needs contiguous tensors")
        self._k, self._v, self._k_scale, self._v_scale, self._block, self.index = k, v, k_scale, v_scale, block, index
        self.struct = FsvdKv8(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), B, Hk, S, Dh, block)
        self.ref = C.byref(self.struct)

    # (the tensors cannot be exchanged: `struct` holds their addresses)
    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    k_scale = property(lambda self: self._k_scale)
    v_scale = property(lambda self: self._v_scale)
    block = property(lambda self: self._block)

    @classmethod
    def empty(cls, batch: int, max_len: int, num_kv_heads: int, head_dim: int, *, block: int = 64, device="cuda") -> "KV8Cache":
        """A cache without tokens: zero codes, scales of one."""
        shape = (int(batch), int(num_kv_heads), int(max_len), int(head_dim))
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block}")
        k = torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
        s = torch.ones((*shape[:2], -(-shape[2] // block)), dtype=torch.float32, device=device)
        return cls(k, torch.zeros_like(k.view(torch.uint8)).view(torch.float8_e4m3fn), s, s.clone(), block)

    @property
    def batch(self) -> int:
        return self.k.shape[0]

    @property
    def max_len(self) -> int:
        return self.k.shape[2]

    @property
    def device(self) -> torch.device:
        return self.k.device

    def nbytes(self) -> int:
        return 2 * (self.k.numel() + 4 * self.k_scale.numel())
