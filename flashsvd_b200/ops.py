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
# (These are calls of a few microseconds on the device: the checks are written for their cost.)
_BF16, _F32, _F64, _I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
_lib_handle = None


def _library():
    global _lib_handle
    if _lib_handle is None:
        _lib_handle = _lib.load()
    return _lib_handle


def _raw_stream(index: int) -> int:
    """The current stream of a device as an integer."""
    return torch._C._cuda_getCurrentRawStream(index)


def _launch(index: int, entry, *args) -> None:
    """A call into the library with the tensors' device current; its status."""
    if torch._C._cuda_getDevice() == index:
        status = entry(*args)
    else:
        with torch.cuda.device(index):
            status = entry(*args)
    if status:
        check(status)


def _refuse(name: str, t, dtype, index: int, shape, strided: bool):
    """Says what is wrong with a tensor argument that `_ok` did not take."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise ValueError(f"{name}: flashsvd_b200 ops need CUDA tensors (there is no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on cuda:{index}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    raise ValueError(f"{name}: heads and dimensions must be contiguous" if strided else f"{name} must be contiguous")


def _ok(name: str, t, dtype, index: int, shape=None):
    """A contiguous tensor of this type, device and shape; its address."""
    try:
        if t.dtype is dtype and t.get_device() == index and (shape is None or t.shape == shape) and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:   # (no tensor)
        pass
    _refuse(name, t, dtype, index, shape, False)


def _ok_strided(name: str, t, dtype, index: int, shape):
    """As `_ok`, with any strides in front of the last two dimensions."""
    try:
        fits = t.dtype is dtype and t.get_device() == index and t.shape == shape
    except AttributeError:
        fits = False
    if not fits:
        _refuse(name, t, dtype, index, shape, True)
    if not t.is_contiguous() and t.numel():
        H, D = shape[-2:]
        st = t.stride()
        if (st[-1] != 1 and D > 1) or (st[-2] != D and H > 1):
            _refuse(name, t, dtype, index, shape, True)
    return t.data_ptr()


def _device_of(name: str, t, ndim: int, what: str) -> int:
    """Index of the device of the argument that the others go by."""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise ValueError(f"{name}: flashsvd_b200 ops need CUDA tensors (there is no CPU path)")
    if t.ndim != ndim:
        raise ValueError(f"{name} must be {what}, got {tuple(t.shape)}")
    return t.get_device()


def _room_like(t):
    """A contiguous tensor of the same size."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def rope_qk(q, k, positions, inv_freq, *, interleaved=False, scale=1.0, q_out=None, k_out=None):
    """Rotates q[T, H, Dh] and k[T, Hk, Dh] (or None) at positions[T] (int32); returns (q_out, k_out).

    Dimensions [0, 2 * len(inv_freq)) of a head take part: pair i turns by ``position * inv_freq[i]`` (float64, formed
    in 64 bits), pairs are (i, i + len(inv_freq)), or (2i, 2i + 1) with ``interleaved``; cos and sin are multiplied by
    ``scale``; the other dimensions are copied.  bfloat16 or float32; tokens may be strided (slices of a packed
    projection).  q_out / k_out may be q / k themselves when those are contiguous."""
    index = _device_of("q", q, 3, "[T, H, Dh]")
    shape = q.shape
    T, H, Dh = shape
    dtype = q.dtype
    code = _dtype_code(dtype)
    qp = _ok_strided("q", q, dtype, index, shape)
    pp = _ok("positions", positions, _I32, index, (T,))
    fp = _ok("inv_freq", inv_freq, _F64, index)
    if inv_freq.ndim != 1:
        raise ValueError("inv_freq must be a vector")
    Hk, kp, kop, ks = 0, None, None, 0
    if k is not None:
        if k.ndim != 3:
            raise ValueError(f"k must be [T, Hk, Dh], got {tuple(k.shape)}")
        Hk = k.shape[1]
        kp = _ok_strided("k", k, dtype, index, (T, Hk, Dh))
        if k_out is None:
            k_out = _room_like(k)
            kop = k_out.data_ptr()
        else:
            kop = _ok("k_out", k_out, dtype, index, (T, Hk, Dh))
        ks = k.stride(0) if T > 1 else 0
    elif k_out is not None:
        raise ValueError("k_out without k")
    if q_out is None:
        q_out = _room_like(q)
        qop = q_out.data_ptr()
    else:
        qop = _ok("q_out", q_out, dtype, index, shape)
    if T == 0:
        return q_out, k_out
    _launch(index, _library().fsvd_rope_qk, qp, q.stride(0) if T > 1 else 0, kp, ks, pp, fp, 2 * inv_freq.shape[0],
            1 if interleaved else 0, scale, qop, kop, T, H, Hk, Dh, code, _raw_stream(index))
    return q_out, k_out


def make_kv8_workspace(batch, num_heads, num_kv_heads, head_dim, max_len, device) -> Workspace:
    """Scratch of ``kv8_append`` and ``flash_decode_kv8`` for these sizes, and for all that need no more (as many heads per kv
    head, or fewer); launches that share one must be ordered."""
    n = int(_lib.load().fsvd_kv8_workspace_bytes(int(batch), int(num_heads), int(num_kv_heads), int(head_dim), int(max_len)))
    if n == 0:
        raise ValueError(f"no 8-bit cache of these sizes: batch {batch}, heads {num_heads}/{num_kv_heads}, head_dim {head_dim}, "
                         f"max_len {max_len}")
    return Workspace(torch.zeros(n, dtype=torch.uint8, device=device), n)


def _add(n) -> int:
    n = int(n)
    if not -(1 << 31) <= n < 1 << 31:
        raise ValueError(f"seqlen_add {n} is no 32-bit number")
    return n


def _scratch(ws: Workspace, index: int):
    if ws.buf.get_device() != index:
        raise ValueError(f"the workspace is on {ws.buf.device}, the call's tensors on cuda:{index}")
    return ws.buf.data_ptr()


def kv8_append(k, v, cache, cache_seqlens, ws: Workspace, *, new_lens=None, q=None, rotary=None, q_out=None):
    """Quantises k / v [B, L, Hk, Dh] into ``cache`` (kv8.KV8Cache) at positions cache_seqlens[b] .. + L - 1
    (+ new_lens[b] - 1 with ``new_lens``); with ``rotary`` (kv8.Rotary) the keys, and q [B, L, H, Dh] when given, are
    rotated at their positions first.  Returns the rotated q (rows past new_lens[b] are not written) or None.

    cache_seqlens (int32 [B]) is not advanced.  A token that does not fit the cache is dropped and sets the workspace
    status, as in ``qkv_rope_append``.  Batch and tokens may be strided."""
    st, index = cache.struct, cache.index
    B, Hk, Dh = st.B, st.Hk, st.Dh
    if k.ndim != 4:
        raise ValueError(f"k must be [B, L, {Hk}, {Dh}], got {tuple(k.shape)}")
    L = k.shape[1]
    shape = (B, L, Hk, Dh)
    kp = _ok_strided("k", k, _BF16, index, shape)
    vp = _ok_strided("v", v, _BF16, index, shape)
    kst = k.stride()
    if v.stride() != kst:
        k, v = k.contiguous(), v.contiguous()
        kp, vp, kst = k.data_ptr(), v.data_ptr(), k.stride()
    sp = _ok("cache_seqlens", cache_seqlens, _I32, index, (B,))
    np_ = None if new_lens is None else _ok("new_lens", new_lens, _I32, index, (B,))
    fp, R, inter, scale = None, 0, 0, 1.0
    if rotary is not None:
        f = rotary.inv_freq
        fp = _ok("inv_freq", f, _F64, index)
        if f.ndim != 1:
            raise ValueError("inv_freq must be a vector")
        R, inter, scale = 2 * f.shape[0], 1 if rotary.interleaved else 0, rotary.scale
    H, qp, qop, qs0, qs1 = 0, None, None, 0, 0
    if q is not None:
        if rotary is None:
            raise ValueError("q is passed to be rotated: rotary is missing")
        if q.ndim != 4:
            raise ValueError(f"q must be [B, L, H, Dh], got {tuple(q.shape)}")
        H = q.shape[2]
        qshape = (B, L, H, Dh)
        qp = _ok_strided("q", q, _BF16, index, qshape)
        qs0, qs1 = q.stride()[:2]
        if q_out is None:
            q_out = _room_like(q)
            qop = q_out.data_ptr()
        else:
            qop = _ok("q_out", q_out, _BF16, index, qshape)
    elif q_out is not None:
        raise ValueError("q_out without q")
    wp = _scratch(ws, index)
    if L == 0:
        return q_out
    _launch(index, _library().fsvd_kv8_append, cache.ref, kp, vp, kst[0], kst[1], sp, np_, qp, qs0, qs1, qop, fp, R, inter, scale,
            H, L, wp, ws.nbytes, _raw_stream(index))
    return q_out


def kv8_load(cache, start, length, *, cache_seqlens=None, seqlen_add=0, k_out=None, v_out=None):
    """Positions [start, start + length) of the cache as bfloat16 numbers: (k, v), each [B, Hk, length, Dh].  With
    ``cache_seqlens`` rows from cache_seqlens[b] + seqlen_add on are zeros."""
    st, index = cache.struct, cache.index
    start, length = int(start), int(length)
    if start < 0 or length < 0 or start + length > st.S_max:
        raise ValueError(f"positions {start} + {length} are outside the cache ({st.S_max})")
    shape = (st.B, st.Hk, length, st.Dh)
    sp = None if cache_seqlens is None else _ok("cache_seqlens", cache_seqlens, _I32, index, (st.B,))
    if k_out is None:
        k_out = cache.k.new_empty(shape, dtype=_BF16)
        kp = k_out.data_ptr()
    else:
        kp = _ok("k_out", k_out, _BF16, index, shape)
    if v_out is None:
        v_out = torch.empty_like(k_out)
        vp = v_out.data_ptr()
    else:
        vp = _ok("v_out", v_out, _BF16, index, shape)
    if length == 0:
        return k_out, v_out
    _launch(index, _library().fsvd_kv8_load, cache.ref, start, length, sp, _add(seqlen_add), kp, vp, _raw_stream(index))
    return k_out, v_out


def flash_decode_kv8(q, cache, cache_seqlens, ws: Workspace, *, seqlen_add=0, scale=0.0, out=None):
    """``flash_decode`` over an 8-bit cache: q[B, H, Dh] bfloat16 against positions [0, cache_seqlens[b] + seqlen_add),
    scale <= 0 selects 1/sqrt(Dh); a sequence without positions gives zeros."""
    st, index = cache.struct, cache.index
    if q.ndim != 3:
        raise ValueError(f"q must be [B, H, Dh], got {tuple(q.shape)}")
    H = q.shape[1]
    shape = (st.B, H, st.Dh)
    qp = _ok("q", q, _BF16, index, shape)
    sp = _ok("cache_seqlens", cache_seqlens, _I32, index, (st.B,))
    if out is None:
        out = torch.empty_like(q)
        op = out.data_ptr()
    else:
        op = _ok("out", out, _BF16, index, shape)
    wp = _scratch(ws, index)
    _launch(index, _library().fsvd_flash_decode_kv8, cache.ref, qp, sp, _add(seqlen_add), op, H, scale, wp, ws.nbytes, _raw_stream(index))
    return out


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, probs_out=None):
    """One token per row of logits[B, V] (float32 or bfloat16; rows may be strided) from uniforms[B] (float32 in [0, 1)):
    (tokens int32 [B], probs float32 [B]).

    Weights are exp((logit - max) / temperature).  In descending order of the logits (lower index first among equals)
    the first ``top_k`` stay (0: all), of those the ones whose preceding mass is at most ``top_p`` of it (1: all), of
    those the ones with weight >= ``min_p`` (0: all).  The token is the first one in index order whose running mass
    exceeds uniforms[b] of the kept mass; probs is its share.  temperature <= 0 takes the largest logit (a positive one
    below 2^-64 counts as 2^-64).  Each setting
    is a number or a tensor with one value per row (float32; top_k int32)."""
    index = _device_of("logits", logits, 2, "[B, V]")
    B, V = logits.shape
    code = _dtype_code(logits.dtype)
    if V < 1:
        raise ValueError("logits of an empty vocabulary")
    if V > 1 and logits.stride(1) != 1:
        raise ValueError("logits: a row must be contiguous")
    rows = (B,)
    up = _ok("uniforms", uniforms, _F32, index, rows)
    tp = kp = pp = mp = None
    if torch.is_tensor(temperature):
        tp, temperature = _ok("temperature", temperature, _F32, index, rows), 1.0
    if torch.is_tensor(top_k):
        kp, top_k = _ok("top_k", top_k, _I32, index, rows), 0
    elif top_k > V:
        top_k = 0
    if torch.is_tensor(top_p):
        pp, top_p = _ok("top_p", top_p, _F32, index, rows), 1.0
    if torch.is_tensor(min_p):
        mp, min_p = _ok("min_p", min_p, _F32, index, rows), 0.0
    if out is None:
        out = torch.empty_like(uniforms, dtype=_I32)
        op = out.data_ptr()
    else:
        op = _ok("out", out, _I32, index, rows)
    if probs_out is None:
        probs_out = torch.empty_like(uniforms)
        bp = probs_out.data_ptr()
    else:
        bp = _ok("probs_out", probs_out, _F32, index, rows)
    if B == 0:
        return out, probs_out
    _launch(index, _library().fsvd_sample, logits.data_ptr(), logits.stride(0) if B > 1 else V, code, up, tp, kp, pp, mp, temperature,
            top_k, top_p, min_p, op, bp, B, V, _raw_stream(index))
    return out, probs_out
