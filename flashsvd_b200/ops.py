"""Tensor-level wrappers over the C ABI.

PyTorch is used for device memory and the current CUDA stream only; every function enqueues one
kernel launch through libflashsvd_b200.so on ``torch.cuda.current_stream()`` and does not
synchronise.  Argument errors raise ``ValueError`` before anything is launched, like the
reference wrappers (kernels/mlp/decode/dual_split_triton_pcat_s.py:139-155).
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import FsvdDims, FsvdLayer, LAYER_FIELDS, check


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    if dtype == torch.float32:
        return _lib.DTYPE_F32
    raise ValueError(f"flashsvd_b200 supports bfloat16 and float32 tensors, got {dtype}")


def _is_q4(w) -> bool:
    return hasattr(w, "packed")


def _code(x: torch.Tensor, *factors) -> int:
    """dtype code of a call: the activations' type, or DTYPE_BF16_Q4 when the factors are int4
    tile streams (quant.Q4Factor; all of them must be, and the activations bfloat16)."""
    nq = sum(1 for w in factors if w is not None and _is_q4(w))
    if nq == 0:
        return _dtype_code(x.dtype)
    if nq != sum(1 for w in factors if w is not None) or x.dtype != torch.bfloat16:
        raise ValueError("int4 factors need bfloat16 activations and every factor of the call quantised")
    return _lib.DTYPE_BF16_Q4


def _ptr(t) -> int | None:
    if t is None:
        return None
    if _is_q4(t):
        t = t.packed
    if not t.is_cuda:
        raise ValueError("flashsvd_b200 ops need CUDA tensors (there is no CPU path)")
    if not t.is_contiguous():
        raise ValueError("flashsvd_b200 ops need contiguous tensors")
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def set_launch_config(warps: int = 0, depth: int = 0, grid: int = 0) -> None:
    """Pick the kernel geometry (see fsvd_set_launch_config in include/flashsvd_b200.h)."""
    check(_lib.load().fsvd_set_launch_config(int(warps), int(depth), int(grid)))


def set_wait_limit(sm_clocks: int) -> None:
    """Budget of every device-side wait in SM clocks (see fsvd_set_wait_limit)."""
    check(_lib.load().fsvd_set_wait_limit(int(sm_clocks)))


def launch_count() -> int:
    return int(_lib.load().fsvd_launch_count())


@dataclass
class Workspace:
    """Scratch for the per-op entry points: rank-space partial sums, the SwiGLU activation,
    attention split partials and the grid-barrier words."""

    buf: torch.Tensor
    nbytes: int

    @property
    def ptr(self) -> int:
        return self.buf.data_ptr()

    def status(self) -> int:
        """Blocking read of the device status word; raises if a device-side wait ran out."""
        st = C.c_int(0)
        check(_lib.load().fsvd_workspace_status(self.ptr, C.byref(st)))
        return int(st.value)

    def raw_status(self) -> int:
        """The status word itself (blocking), without the exception."""
        st = C.c_int(0)
        _lib.load().fsvd_workspace_status(self.ptr, C.byref(st))
        return int(st.value)

    def clear_status(self) -> None:
        check(_lib.load().fsvd_workspace_clear_status(self.ptr, _stream()))


def make_dims(*, dtype, B=1, d=8, H=1, Hk=1, Dh=64, I=8, Rq=8, Rk=8, Rv=8, Ro=8, Rg=8, Ru=8,
              Rd=8, S_max=1, vocab=0, n_layers=0, eps=1e-6, rows_are_positions=0) -> FsvdDims:
    """rows_are_positions=1: the B rows are consecutive positions of one sequence (a chunk of its
    prompt) that share cache row 0; cache_seqlens[b] must be first + b."""
    return FsvdDims(_dtype_code(dtype) if isinstance(dtype, torch.dtype) else int(dtype), B, d, H,
                    Hk, Dh, I, Rq, Rk, Rv, Ro, Rg, Ru, Rd, S_max, vocab, n_layers, eps,
                    int(rows_are_positions))


def make_workspace(dims: FsvdDims, device) -> Workspace:
    lib = _lib.load()
    n = int(lib.fsvd_workspace_bytes(C.byref(dims)))
    buf = torch.zeros(n, dtype=torch.uint8, device=device)
    return Workspace(buf, n)


def lowrank_proj(x, v_w, u_w, ws: Workspace, residual=None, out=None):
    """y = (residual +) x @ v_w.T @ u_w.T for x[B, d_in], v_w[R, d_in], u_w[d_out, R]."""
    if x.ndim != 2:
        raise ValueError(f"x must be [B, d_in], got {tuple(x.shape)}")
    B, d_in = x.shape
    if len(v_w.shape) != 2 or v_w.shape[1] != d_in:
        raise ValueError(f"v_w must be [R, {d_in}], got {tuple(v_w.shape)}")
    R = v_w.shape[0]
    if len(u_w.shape) != 2 or u_w.shape[1] != R:
        raise ValueError(f"u_w must be [d_out, {R}], got {tuple(u_w.shape)}")
    d_out = u_w.shape[0]
    if out is None:
        out = torch.empty((B, d_out), dtype=x.dtype, device=x.device)
    check(_lib.load().fsvd_lowrank_proj(
        _ptr(x), _ptr(v_w), _ptr(u_w), _ptr(residual), _ptr(out), B, d_in, R, d_out,
        _code(x, v_w, u_w), ws.ptr, ws.nbytes, _stream()))
    return out


def lift(p, u_w, ws: Workspace, residual=None, out=None):
    """y = (residual +) p @ u_w.T for p[B, R], u_w[d_out, R] (one factor, no rank step)."""
    if p.ndim != 2:
        raise ValueError(f"p must be [B, R], got {tuple(p.shape)}")
    B, R = p.shape
    if len(u_w.shape) != 2 or u_w.shape[1] != R:
        raise ValueError(f"u_w must be [d_out, {R}], got {tuple(u_w.shape)}")
    d_out = u_w.shape[0]
    if out is None:
        out = torch.empty((B, d_out), dtype=p.dtype, device=p.device)
    check(_lib.load().fsvd_lift(_ptr(p), _ptr(u_w), _ptr(residual), _ptr(out), B, R, d_out,
                                _code(p, u_w), ws.ptr, ws.nbytes, _stream()))
    return out


def lowrank_proj_static(x, v_w, u_w, residual=None, out=None):
    """lowrank_proj on the library's built-in scratch (B * R <= 8192): no workspace argument and
    no device allocation inside the call when ``out`` is given.  Calls share one scratch array
    per device and must not overlap in time."""
    if x.ndim != 2:
        raise ValueError(f"x must be [B, d_in], got {tuple(x.shape)}")
    B, d_in = x.shape
    if v_w.ndim != 2 or v_w.shape[1] != d_in:
        raise ValueError(f"v_w must be [R, {d_in}], got {tuple(v_w.shape)}")
    R = v_w.shape[0]
    if u_w.ndim != 2 or u_w.shape[1] != R:
        raise ValueError(f"u_w must be [d_out, {R}], got {tuple(u_w.shape)}")
    d_out = u_w.shape[0]
    if out is None:
        out = torch.empty((B, d_out), dtype=x.dtype, device=x.device)
    check(_lib.load().fsvd_lowrank_proj_static(
        _ptr(x), _ptr(v_w), _ptr(u_w), _ptr(residual), _ptr(out), B, d_in, R, d_out,
        _dtype_code(x.dtype), _stream()))
    return out


def mlp_swiglu_decode(x, gate_u, up_u, down_v, down_u, ws: Workspace, *, upgate_v=None,
                      norm_w=None, eps=1e-6, residual=None, out=None):
    """Fused low-rank SwiGLU MLP for one token per row of x.

    With ``upgate_v`` ([Ru+Rg, d], up rows first) x is the hidden state [B, d]; without it x is
    PCat [B, Ru+Rg] = [p_up | p_gate].  gate_u/up_u are [I, R], down_v [Rd, I], down_u [d, Rd].
    """
    if x.ndim != 2:
        raise ValueError(f"x must be 2-D, got {tuple(x.shape)}")
    B = x.shape[0]
    I, Rg = gate_u.shape
    if tuple(up_u.shape) != tuple(gate_u.shape):
        raise ValueError(f"up_u shape {tuple(up_u.shape)} must match gate_u shape {tuple(gate_u.shape)}")
    Ru = up_u.shape[1]
    if len(down_v.shape) != 2 or down_v.shape[1] != I:
        raise ValueError(f"down_v must be [Rd, {I}], got {tuple(down_v.shape)}")
    Rd = down_v.shape[0]
    if len(down_u.shape) != 2 or down_u.shape[1] != Rd:
        raise ValueError(f"down_u must be [d, {Rd}], got {tuple(down_u.shape)}")
    d = down_u.shape[0]
    if upgate_v is not None:
        if tuple(upgate_v.shape) != (Ru + Rg, d) or x.shape[1] != d:
            raise ValueError(f"upgate_v must be [{Ru + Rg}, {d}] and x [B, {d}]")
    elif x.shape[1] != Ru + Rg:
        raise ValueError(f"PCat must be [B, {Ru + Rg}], got {tuple(x.shape)}")
    if out is None:
        out = torch.empty((B, d), dtype=x.dtype, device=x.device)
    check(_lib.load().fsvd_mlp_swiglu_decode(
        _ptr(x), _ptr(norm_w), float(eps), _ptr(upgate_v), _ptr(gate_u), _ptr(up_u), _ptr(down_v),
        _ptr(down_u), _ptr(residual), _ptr(out), B, d, I, Ru, Rg, Rd,
        _code(x, upgate_v, gate_u, up_u, down_v, down_u), ws.ptr, ws.nbytes, _stream()))
    return out


def qkv_rope_append(x, qkv_v, q_u, k_u, v_u, cos, sin, k_cache, v_cache, cache_seqlens,
                    ws: Workspace, *, num_heads, num_kv_heads, head_dim, ranks, norm_w=None,
                    eps=1e-6, q_out=None):
    """Rank-project, lift, rotate and append the current token; returns the rotated q[B,H,Dh]."""
    B, d = x.shape
    Rq, Rk, Rv = (int(r) for r in ranks)
    if tuple(qkv_v.shape) != (Rq + Rk + Rv, d):
        raise ValueError(f"qkv_v must be [{Rq + Rk + Rv}, {d}], got {tuple(qkv_v.shape)}")
    if tuple(q_u.shape) != (num_heads * head_dim, Rq):
        raise ValueError(f"q_u must be [{num_heads * head_dim}, {Rq}], got {tuple(q_u.shape)}")
    if tuple(k_u.shape) != (num_kv_heads * head_dim, Rk) or tuple(v_u.shape) != (num_kv_heads * head_dim, Rv):
        raise ValueError("k_u / v_u must be [Hk*Dh, Rk] / [Hk*Dh, Rv]")
    if k_cache.ndim != 4 or k_cache.shape[0] < B or tuple(k_cache.shape[2:]) != (num_kv_heads, head_dim):
        raise ValueError(f"k_cache must be [>=B, S, {num_kv_heads}, {head_dim}], got {tuple(k_cache.shape)}")
    if v_cache.shape != k_cache.shape:
        raise ValueError("v_cache shape must match k_cache")
    S_max = k_cache.shape[1]
    if cos.shape[0] < S_max or cos.shape[1] != head_dim // 2 or sin.shape != cos.shape:
        raise ValueError(f"cos/sin must be [>={S_max}, {head_dim // 2}]")
    if cache_seqlens.dtype != torch.int32 or cache_seqlens.numel() < B:
        raise ValueError("cache_seqlens must be int32 [B]")
    if k_cache.shape[0] != B and B > 1:
        raise ValueError("k_cache batch dimension must equal B")
    if q_out is None:
        q_out = torch.empty((B, num_heads, head_dim), dtype=x.dtype, device=x.device)
    check(_lib.load().fsvd_qkv_rope_append(
        _ptr(x), _ptr(norm_w), float(eps), _ptr(qkv_v), _ptr(q_u), _ptr(k_u), _ptr(v_u),
        _ptr(cos), _ptr(sin), _ptr(k_cache), _ptr(v_cache), _ptr(cache_seqlens), _ptr(q_out),
        B, d, num_heads, num_kv_heads, head_dim, Rq, Rk, Rv, S_max, _code(x, qkv_v, q_u, k_u, v_u),
        ws.ptr, ws.nbytes, _stream()))
    return q_out


def flash_decode(q, k_cache, v_cache, cache_seqlens, ws: Workspace, *, seqlen_add=0, scale=0.0,
                 out=None):
    """Split-KV single-query attention over cache positions [0, cache_seqlens[b]+seqlen_add)."""
    if q.ndim != 3:
        raise ValueError(f"q must be [B, H, Dh], got {tuple(q.shape)}")
    B, H, Dh = q.shape
    if k_cache.ndim != 4 or k_cache.shape[3] != Dh or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache / v_cache must be [B, S, Hk, Dh]")
    if k_cache.shape[0] != B:
        raise ValueError("cache batch dimension must equal B")
    S_max, Hk = k_cache.shape[1], k_cache.shape[2]
    if cache_seqlens.dtype != torch.int32 or cache_seqlens.numel() < B:
        raise ValueError("cache_seqlens must be int32 [B]")
    if out is None:
        out = torch.empty_like(q)
    check(_lib.load().fsvd_flash_decode(
        _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(cache_seqlens), int(seqlen_add), _ptr(out),
        B, H, Hk, Dh, S_max, float(scale), _dtype_code(q.dtype), ws.ptr, ws.nbytes, _stream()))
    return out


def make_layer_struct(tensors: dict) -> FsvdLayer:
    layer = FsvdLayer()
    for name in LAYER_FIELDS:
        setattr(layer, name, _ptr(tensors[name]))
    return layer


def decode_layer(dims: FsvdDims, layer: FsvdLayer, cos, sin, cache_seqlens, x_in, x_out,
                 ws: Workspace):
    """One decoder layer for one new token per sequence; x_in/x_out are [B, d] in the model dtype."""
    check(_lib.load().fsvd_decode_layer(
        C.byref(dims), C.byref(layer), _ptr(cos), _ptr(sin), _ptr(cache_seqlens), _ptr(x_in),
        _ptr(x_out), ws.ptr, ws.nbytes, _stream()))
    return x_out


def make_tp_workspace(dims: FsvdDims, device) -> Workspace:
    """Workspace of the tensor-parallel layer (tiled path at every batch size)."""
    n = int(_lib.load().fsvd_tp_workspace_bytes(C.byref(dims)))
    if n == 0:
        check(-2)
    return Workspace(torch.zeros(n, dtype=torch.uint8, device=device), n)


def tp_decode_layer(dims: FsvdDims, layer: FsvdLayer, cos, sin, cache_seqlens, x_in, x_out, exchange, ws: Workspace, *,
                    x_norm_in=None, next_norm_w=None, x_norm_out=None):
    """One decoder layer on this rank's shards; the partial sums of the output projection and of the
    down projection are exchanged with the other ranks inside the kernels (``exchange``: the handle of
    a ``tensor_parallel.PeerExchange``).  x_out is the full layer output, the same on every rank.
    ``x_norm_in``: ln1-normalised x_in the caller already holds; ``next_norm_w`` / ``x_norm_out``: also
    write rmsnorm(x_out) * next_norm_w (the next layer's input norm, or the final norm)."""
    check(_lib.load().fsvd_tp_decode_layer(
        C.byref(dims), C.byref(layer), _ptr(cos), _ptr(sin), _ptr(cache_seqlens), _ptr(x_in), _ptr(x_norm_in),
        _ptr(x_out), _ptr(next_norm_w), _ptr(x_norm_out), exchange, ws.ptr, ws.nbytes, _stream()))
    return x_out


# ---- operators for callers that drive the layers themselves: rotary positions, the 8-bit cache, the next token
def _raw_stream(device: torch.device):
    return torch.cuda.current_stream(device).cuda_stream


class _SameDevice:
    """Makes the device of the tensors current for the launch (nothing to do when it is)."""

    __slots__ = ("index", "was")

    def __init__(self, device: torch.device):
        self.index, self.was = device.index, None

    def __enter__(self):
        now = torch.cuda.current_device()
        if now != self.index:
            self.was = now
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.was is not None:
            torch.cuda.set_device(self.was)


def _want(name: str, t, dtype, device, shape=None, strided: bool = False):
    """Checks one tensor argument; with `strided` only the last two dimensions have to be contiguous."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise ValueError(f"{name}: flashsvd_b200 ops need CUDA tensors (there is no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if strided:
        if t.numel() and (t.stride(-1) != 1 and t.shape[-1] > 1 or t.stride(-2) != t.shape[-1] and t.shape[-2] > 1):
            raise ValueError(f"{name}: heads and dimensions must be contiguous")
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def rope_qk(q, k, positions, inv_freq, *, interleaved=False, scale=1.0, q_out=None, k_out=None):
    """Rotates q[T, H, Dh] and k[T, Hk, Dh] (or None) at positions[T] (int32); returns (q_out, k_out).

    Dimensions [0, 2 * len(inv_freq)) of a head take part: pair i turns by ``position * inv_freq[i]`` (float64, formed
    in 64 bits), pairs are (i, i + len(inv_freq)), or (2i, 2i + 1) with ``interleaved``; cos and sin are multiplied by
    ``scale``; the other dimensions are copied.  bfloat16 or float32; tokens may be strided (slices of a packed
    projection).  q_out / k_out may be q / k themselves when those are contiguous."""
    if q.ndim != 3:
        raise ValueError(f"q must be [T, H, Dh], got {tuple(q.shape)}")
    T, H, Dh = q.shape
    dtype, dev = q.dtype, q.device
    code = _dtype_code(dtype)
    _want("q", q, dtype, dev, strided=True)
    _want("positions", positions, torch.int32, dev, (T,))
    if inv_freq.ndim != 1:
        raise ValueError("inv_freq must be a vector")
    _want("inv_freq", inv_freq, torch.float64, dev)
    Hk = 0
    if k is not None:
        if k.ndim != 3:
            raise ValueError(f"k must be [T, Hk, Dh], got {tuple(k.shape)}")
        Hk = k.shape[1]
        _want("k", k, dtype, dev, (T, Hk, Dh), strided=True)
        k_out = torch.empty((T, Hk, Dh), dtype=dtype, device=dev) if k_out is None else _want("k_out", k_out, dtype, dev, k.shape)
    elif k_out is not None:
        raise ValueError("k_out without k")
    q_out = torch.empty((T, H, Dh), dtype=dtype, device=dev) if q_out is None else _want("q_out", q_out, dtype, dev, q.shape)
    if T == 0:
        return q_out, k_out
    with _SameDevice(dev):
        check(_lib.load().fsvd_rope_qk(
            q.data_ptr(), q.stride(0) if T > 1 else 0, None if k is None else k.data_ptr(), 0 if k is None or T < 2 else k.stride(0),
            positions.data_ptr(), inv_freq.data_ptr(), 2 * inv_freq.shape[0], int(interleaved), float(scale), q_out.data_ptr(),
            None if k is None else k_out.data_ptr(), T, H, Hk, Dh, code, _raw_stream(dev)))
    return q_out, k_out


def make_kv8_workspace(batch, num_heads, num_kv_heads, head_dim, max_len, device) -> Workspace:
    """Scratch of ``kv8_append`` and ``flash_decode_kv8`` for these sizes; launches that share one must be ordered."""
    n = int(_lib.load().fsvd_kv8_workspace_bytes(int(batch), int(num_heads), int(num_kv_heads), int(head_dim), int(max_len)))
    if n == 0:
        raise ValueError(f"no 8-bit cache of these sizes: batch {batch}, heads {num_heads}/{num_kv_heads}, head_dim {head_dim}, "
                         f"max_len {max_len}")
    return Workspace(torch.zeros(n, dtype=torch.uint8, device=device), n)


def _ws_of(ws: Workspace, dev) -> Workspace:
    if ws.buf.device != dev:
        raise ValueError(f"the workspace is on {ws.buf.device}, the call's tensors on {dev}")
    return ws


def kv8_append(k, v, cache, cache_seqlens, ws: Workspace, *, new_lens=None, q=None, rotary=None, q_out=None):
    """Quantises k / v [B, L, Hk, Dh] into ``cache`` (kv8.KV8Cache) at positions cache_seqlens[b] .. + L - 1
    (+ new_lens[b] - 1 with ``new_lens``); with ``rotary`` (kv8.Rotary) the keys, and q [B, L, H, Dh] when given, are
    rotated at their positions first.  Returns the rotated q (rows past new_lens[b] are not written) or None.

    cache_seqlens (int32 [B]) is not advanced.  A token that does not fit the cache is dropped and sets the workspace
    status, as in ``qkv_rope_append``.  Batch and tokens may be strided."""
    st, dev = cache.struct, cache.device
    if k.ndim != 4:
        raise ValueError(f"k must be [B, L, {st.Hk}, {st.Dh}], got {tuple(k.shape)}")
    B, L = k.shape[0], k.shape[1]
    _want("k", k, torch.bfloat16, dev, (st.B, L, st.Hk, st.Dh), strided=True)
    _want("v", v, torch.bfloat16, dev, k.shape, strided=True)
    if v.stride() != k.stride():
        v = v.contiguous()
        k = k.contiguous()
    _want("cache_seqlens", cache_seqlens, torch.int32, dev, (B,))
    if new_lens is not None:
        _want("new_lens", new_lens, torch.int32, dev, (B,))
    H, qs = 0, (0, 0)
    if rotary is not None:
        if rotary.inv_freq.ndim != 1:
            raise ValueError("inv_freq must be a vector")
        _want("inv_freq", rotary.inv_freq, torch.float64, dev)
    if q is not None:
        if rotary is None:
            raise ValueError("q is passed to be rotated: rotary is missing")
        if q.ndim != 4:
            raise ValueError(f"q must be [B, L, H, Dh], got {tuple(q.shape)}")
        H = q.shape[2]
        _want("q", q, torch.bfloat16, dev, (B, L, H, st.Dh), strided=True)
        qs = (q.stride(0), q.stride(1))
        if q_out is None:
            q_out = torch.empty((B, L, H, st.Dh), dtype=torch.bfloat16, device=dev)
        else:
            _want("q_out", q_out, torch.bfloat16, dev, q.shape)
    elif q_out is not None:
        raise ValueError("q_out without q")
    _ws_of(ws, dev)
    if L == 0:
        return q_out
    with _SameDevice(dev):
        check(_lib.load().fsvd_kv8_append(
            cache.ref, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), cache_seqlens.data_ptr(),
            None if new_lens is None else new_lens.data_ptr(), None if q is None else q.data_ptr(), *qs,
            None if q is None else q_out.data_ptr(), None if rotary is None else rotary.inv_freq.data_ptr(),
            0 if rotary is None else 2 * rotary.inv_freq.shape[0], 0 if rotary is None else int(rotary.interleaved),
            1.0 if rotary is None else float(rotary.scale), H, L, ws.ptr, ws.nbytes, _raw_stream(dev)))
    return q_out


def kv8_load(cache, start, length, *, cache_seqlens=None, seqlen_add=0, k_out=None, v_out=None):
    """Positions [start, start + length) of the cache as bfloat16 numbers: (k, v), each [B, Hk, length, Dh].  With
    ``cache_seqlens`` rows from cache_seqlens[b] + seqlen_add on are zeros."""
    st, dev = cache.struct, cache.device
    start, length = int(start), int(length)
    if start < 0 or length < 0 or start + length > st.S_max:
        raise ValueError(f"positions {start} + {length} are outside the cache ({st.S_max})")
    shape = (st.B, st.Hk, length, st.Dh)
    if cache_seqlens is not None:
        _want("cache_seqlens", cache_seqlens, torch.int32, dev, (st.B,))
    k_out = torch.empty(shape, dtype=torch.bfloat16, device=dev) if k_out is None else _want("k_out", k_out, torch.bfloat16, dev, shape)
    v_out = torch.empty(shape, dtype=torch.bfloat16, device=dev) if v_out is None else _want("v_out", v_out, torch.bfloat16, dev, shape)
    if length == 0:
        return k_out, v_out
    with _SameDevice(dev):
        check(_lib.load().fsvd_kv8_load(cache.ref, start, length, None if cache_seqlens is None else cache_seqlens.data_ptr(),
                                        int(seqlen_add), k_out.data_ptr(), v_out.data_ptr(), _raw_stream(dev)))
    return k_out, v_out


def flash_decode_kv8(q, cache, cache_seqlens, ws: Workspace, *, seqlen_add=0, scale=0.0, out=None):
    """``flash_decode`` over an 8-bit cache: q[B, H, Dh] bfloat16 against positions [0, cache_seqlens[b] + seqlen_add),
    scale <= 0 selects 1/sqrt(Dh); a sequence without positions gives zeros."""
    st, dev = cache.struct, cache.device
    if q.ndim != 3:
        raise ValueError(f"q must be [B, H, Dh], got {tuple(q.shape)}")
    H = q.shape[1]
    _want("q", q, torch.bfloat16, dev, (st.B, H, st.Dh))
    _want("cache_seqlens", cache_seqlens, torch.int32, dev, (st.B,))
    out = torch.empty_like(q) if out is None else _want("out", out, torch.bfloat16, dev, q.shape)
    _ws_of(ws, dev)
    with _SameDevice(dev):
        check(_lib.load().fsvd_flash_decode_kv8(cache.ref, q.data_ptr(), cache_seqlens.data_ptr(), int(seqlen_add), out.data_ptr(),
                                                H, float(scale), ws.ptr, ws.nbytes, _raw_stream(dev)))
    return out


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, probs_out=None):
    """One token per row of logits[B, V] (float32 or bfloat16; rows may be strided) from uniforms[B] (float32 in [0, 1)):
    (tokens int32 [B], probs float32 [B]).

    Weights are exp((logit - max) / temperature).  In descending order of the logits (lower index first among equals)
    the first ``top_k`` stay (0: all), of those the ones whose preceding mass is at most ``top_p`` of it (1: all), of
    those the ones with weight >= ``min_p`` (0: all).  The token is the first one in index order whose running mass
    exceeds uniforms[b] of the kept mass; probs is its share.  temperature <= 0 takes the largest logit.  Each setting
    is a number or a tensor with one value per row (float32; top_k int32)."""
    if logits.ndim != 2:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    B, V = logits.shape
    dev = logits.device
    code = _dtype_code(logits.dtype)
    if not logits.is_cuda:
        raise ValueError("logits: flashsvd_b200 ops need CUDA tensors (there is no CPU path)")
    if V < 1:
        raise ValueError("logits of an empty vocabulary")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: a row must be contiguous")
    _want("uniforms", uniforms, torch.float32, dev, (B,))
    ptrs, values = [], []
    for name, x, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if torch.is_tensor(x):
            ptrs.append(_want(name, x, dtype, dev, (B,)).data_ptr())
            values.append(0)
        else:
            ptrs.append(None)
            values.append(int(x) if dtype == torch.int32 else float(x))
    out = torch.empty(B, dtype=torch.int32, device=dev) if out is None else _want("out", out, torch.int32, dev, (B,))
    probs_out = torch.empty(B, dtype=torch.float32, device=dev) if probs_out is None else _want("probs_out", probs_out, torch.float32, dev, (B,))
    if B == 0:
        return out, probs_out
    with _SameDevice(dev):
        check(_lib.load().fsvd_sample(
            logits.data_ptr(), logits.stride(0) if B > 1 else V, code, uniforms.data_ptr(), *ptrs, *values, out.data_ptr(),
            probs_out.data_ptr(), B, V, _raw_stream(dev)))
    return out, probs_out
