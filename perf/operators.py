"""Operators of a decoder that is driven layer by layer, as cases that can be timed and compared: rotary positions,
a key / value cache held in 8 bits (append, read back, attention of one query per sequence) and the choice of the
next token.

A case is a dict of plain values.  ``op`` is one of
  "rope"    q[T, H, Dh] and k[T, Hk, Dh] rotated at positions[T]; ``rot`` of the Dh dimensions take part, in pairs
            (i, i + rot/2) (layout "half") or (2i, 2i + 1) ("interleaved"); ``scaling`` names the frequencies
  "update"  L new tokens per sequence behind ctx - b * step held ones: q and k are rotated, keys and values quantised
            into the cache (e4m3 codes, one power-of-two scale per ``block`` tokens and kv head), the prefix read back
  "attend"  one query per sequence over a cache that holds ctx - b * step tokens
  "sample"  a token per row of logits[B, V] from one uniform number each: temperature, top-k, top-p, min-p
``own`` false computes them in plain torch operations, true through the package's operators.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP = -60          # smallest exponent of a block's scale
_workspaces = {}       # one per set of sizes, as a serving program keeps it


def _case(name, op, **kw):
    return dict(name=name, op=op, **kw)


def listed():
    return [
        # one sequence, one token, one layer: the smallest call there is
        _case("rope_b1", "rope", dtype="bf16", T=1, pos0=517, H=32, Hk=32, Dh=128, rot=128, layout="half", scaling="none",
              packed=False),
        # a prompt chunk far into a long context: grouped heads, half of each head rotated, adjacent pairs, stretched
        # frequencies, q and k still inside the packed projection
        _case("rope_long_gqa", "rope", dtype="bf16", T=8191, pos0=122880, H=64, Hk=8, Dh=128, rot=64, layout="interleaved",
              scaling="yarn", packed=True),
        # the 32-bit mode, odd number of rows
        _case("rope_f32", "rope", dtype="f32", T=509, pos0=0, H=16, Hk=16, Dh=64, rot=64, layout="half", scaling="linear",
              packed=False),
        # a small batch appends one token per sequence, each at a place of its own inside its block
        _case("update_step_b8", "update", B=8, L=1, ctx=190, step=17, H=32, Hk=32, Dh=128, rot=128, layout="half",
              scaling="none", block=64),
        # a whole prompt of odd length into an empty cache
        _case("update_prompt", "update", B=1, L=2041, ctx=0, step=0, H=32, Hk=32, Dh=128, rot=128, layout="half",
              scaling="none", block=64),
        # chunks of four prompts behind what they have already written, grouped heads, small blocks
        _case("update_chunk_gqa", "update", B=4, L=301, ctx=1000, step=37, H=64, Hk=8, Dh=128, rot=64, layout="interleaved",
              scaling="yarn", block=32),
        # one user, a short context: latency
        _case("attend_b1", "attend", B=1, ctx=512, step=0, H=32, Hk=32, Dh=128, block=64),
        # two long documents under a wide grouped-query layer
        _case("attend_long_gqa", "attend", B=2, ctx=131071, step=30011, H=64, Hk=8, Dh=128, block=64),
        # a few dozen sequences at a medium context
        _case("attend_b32", "attend", B=32, ctx=2048, step=0, H=32, Hk=32, Dh=128, block=64),
        # a full server of a small model, every sequence at a length of its own
        _case("attend_b128_ragged", "attend", B=128, ctx=1023, step=6, H=16, Hk=16, Dh=64, block=32),
        # one user, nucleus sampling
        _case("sample_b1", "sample", dtype="f32", B=1, V=32000, temperature=0.8, top_k=0, top_p=0.95, min_p=0.0, mixed=False),
        # a full server with a large vocabulary, settings of its own for every row
        _case("sample_b128_mixed", "sample", dtype="f32", B=128, V=100003, temperature=0.9, top_k=50, top_p=0.9, min_p=0.05,
              mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    G = rng.choice([1, 1, 2, 4, 8])
    Hk = rng.choice([1, 2, 4, 5, 8, 8, 16, 32]) if G > 1 else rng.choice([4, 8, 12, 16, 32, 40])
    return G * Hk, Hk


def draw(rng):
    op = rng.choice(["rope", "rope", "update", "update", "attend", "attend", "attend", "sample", "sample"])
    H, Hk = _heads(rng)
    Dh = rng.choice([64, 128, 128])
    layout, scaling = rng.choice(["half", "half", "interleaved"]), rng.choice(["none", "none", "linear", "yarn"])
    rot = rng.choice([Dh, Dh, Dh // 2, Dh // 4 * 3])
    block = rng.choice([16, 32, 64, 64, 128])
    if op == "rope":
        T = _log_int(rng, 1, 8191 * 72 // (2 * H))
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f32"]), T=T, pos0=_log_int(rng, 1, 131072), H=H, Hk=Hk, Dh=Dh,
                    rot=rot, layout=layout, scaling=scaling, packed=rng.random() < 0.5)
    if op == "update":
        B = _log_int(rng, 1, 32)
        L = rng.choice([1, _log_int(rng, 1, max(1, 4096 // B))])
        ctx = rng.choice([0, _log_int(rng, 1, 4096 // B)])
        step = rng.randrange(0, max(1, ctx // B)) if B > 1 else 0
        return dict(op=op, B=B, L=L, ctx=ctx, step=step, H=H, Hk=Hk, Dh=Dh, rot=rot, layout=layout, scaling=scaling, block=block)
    if op == "attend":
        B = _log_int(rng, 1, 128)
        ctx = _log_int(rng, 1, max(16, min(131072, 500_000_000 // (2 * B * Hk * Dh))))
        step = rng.randrange(0, ctx // B + 1) if B > 1 else 0
        return dict(op=op, B=B, ctx=ctx, step=step, H=H, Hk=Hk, Dh=Dh, block=block)
    return dict(op=op, dtype=rng.choice(["f32", "f32", "bf16"]), B=_log_int(rng, 1, 128), V=_log_int(rng, 300, 180000),
                temperature=round(rng.uniform(0.3, 1.6), 3), top_k=rng.choice([0, 0, _log_int(rng, 1, 1000)]),
                top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.01, 0.3), 3)]),
                mixed=rng.random() < 0.3)


def _lens(c):
    return [c["ctx"] - b * c["step"] for b in range(c["B"])]


def _frequencies(rot, scaling):
    """(radians per position of each pair in 64 bits, factor on cos and sin)."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":   # slow pairs stretched 32 times, fast ones as they are, a ramp between
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return f * keep + f / 32.0 * (1.0 - keep), 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def _codes(x, block):
    """e4m3 codes and scales of x[B, Hk, S, Dh], block by block."""
    B, Hk, S, Dh = x.shape
    nb = -(-S // block)
    pad = torch.zeros(B, Hk, nb * block, Dh, dtype=x.dtype, device=x.device)
    pad[:, :, :S] = x
    scale = _scale(pad.view(B, Hk, nb, block, Dh).abs().amax((3, 4)).float())
    codes = (pad.view(B, Hk, nb, block * Dh).float() / scale[..., None]).to(torch.float8_e4m3fn)
    return codes.view(B, Hk, nb * block, Dh)[:, :, :S].contiguous(), scale


def _scale(amax):
    """The smallest power of two, 2^MIN_EXP at least, with amax <= 448 scale."""
    m, e = torch.frexp(amax)   # amax = m 2^e, 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(amax), torch.where(m > 0.875, e - 8, e - 9).clamp_min(MIN_EXP).float())


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def randn(*size, dtype=torch.bfloat16):
        return torch.randn(*size, device=dev, generator=gen).to(dtype)

    s = {"case": c}
    if c["op"] == "rope":
        dt = torch.float32 if c["dtype"] == "f32" else torch.bfloat16
        T, H, Hk, Dh = c["T"], c["H"], c["Hk"], c["Dh"]
        if c["packed"]:
            qkv = randn(T, H + 2 * Hk, Dh, dtype=dt)
            s.update(q=qkv[:, :H], k=qkv[:, H:H + Hk])
        else:
            s.update(q=randn(T, H, Dh, dtype=dt), k=randn(T, Hk, Dh, dtype=dt))
        s["positions"] = torch.arange(c["pos0"], c["pos0"] + T, device=dev, dtype=torch.int32)
    elif c["op"] == "sample":
        # a few likely tokens above a broad tail, as a language model's last layer gives them
        logits = 2.0 * torch.randn(c["B"], c["V"], device=dev, generator=gen)
        logits += 3.0 * torch.randn(c["B"], c["V"], device=dev, generator=gen).clamp_min(2.5) - 7.5
        s["logits"] = logits if c["dtype"] == "f32" else logits.to(torch.bfloat16)
        s["uniforms"] = torch.rand(c["B"], device=dev, generator=gen)
        row = torch.arange(c["B"], device=dev)
        if c["mixed"]:   # greedy rows, rows without one filter or the other, filters of their own
            s["temperature"] = torch.where(row % 7 == 3, 0.0, c["temperature"] * (1.0 + 0.01 * row)).float()
            s["top_k"] = torch.where(row % 3 == 1, 0, c["top_k"] + row).int()
            s["top_p"] = torch.where(row % 4 == 2, 1.0, c["top_p"]).float()
            s["min_p"] = torch.where(row % 5 == 0, 0.0, c["min_p"]).float()
        else:
            s.update(temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
    else:
        B, H, Hk, Dh, S = c["B"], c["H"], c["Hk"], c["Dh"], c["ctx"] + c.get("L", 0) + 8
        # keys have a few channels that are larger than the others
        lift = torch.where(torch.rand(Hk, 1, Dh, device=dev, generator=gen) < 0.04, 6.0, 1.0).to(torch.bfloat16)
        s["k8"], s["k_scale"] = _codes(randn(B, Hk, S, Dh) * lift, c["block"])
        s["v8"], s["v_scale"] = _codes(randn(B, Hk, S, Dh), c["block"])
        s["lens"] = torch.tensor(_lens(c), device=dev, dtype=torch.int32)
        if c["op"] == "attend":
            s["q"] = randn(B, H, Dh) * 1.5
        else:
            qkv = randn(B, c["L"], H + 2 * Hk, Dh)   # q, k and v stay inside the packed projection
            s.update(q=qkv[:, :, :H], k=qkv[:, :, H:H + Hk], v=qkv[:, :, H + Hk:])
    if "rot" in c:
        f, s["scale"] = _frequencies(c["rot"], c["scaling"])
        s["inv_freq"] = f.to(dev)
    return s


# ---- plain forms
def _rotated(x, positions, s, dtype):
    """x[..., heads, Dh] rotated at positions[...], in `dtype`; the angles of far positions take 64 bits."""
    c = s["case"]
    ang = positions.double()[..., None, None] * s["inv_freq"]
    cos, sin = (s["scale"] * torch.cos(ang)).to(dtype), (s["scale"] * torch.sin(ang)).to(dtype)
    x = x.to(dtype)
    part = x[..., :c["rot"]]
    if c["layout"] == "half":
        a, b = part[..., :c["rot"] // 2], part[..., c["rot"] // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., c["rot"]:]], -1)


def _append(codes, scales, x, lens, block):
    """Quantises x[B, L, Hk, Dh] into codes[B, Hk, S, Dh] / scales[B, Hk, blocks] behind the first lens[b] tokens."""
    B, L, Hk, Dh = x.shape
    S, nb = codes.shape[2], scales.shape[2]
    pos = lens.long()[:, None] + torch.arange(L, device=x.device)
    x = x.float().transpose(1, 2)
    amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    blk = (pos // block)[:, None].expand(B, Hk, L)
    most = torch.zeros_like(scales).scatter_reduce(2, blk, amax, "amax")
    touched = torch.zeros_like(scales, dtype=torch.bool).scatter(2, blk, True)
    held = (torch.arange(nb, device=x.device) * block)[None, None] < lens[:, None, None]
    new = torch.where(held, torch.maximum(scales, _scale(most)), _scale(most))
    new = torch.where(touched, new, scales)
    # tokens that a growing block already holds
    raw, rows = codes.view(torch.uint8), torch.arange(B, device=x.device)[:, None]
    old = ((lens.long() // block * block)[:, None] + torch.arange(block, device=x.device)).clamp_max(S - 1)
    ratio = torch.where(held, scales / new, 1.0).gather(2, (old // block)[:, None].expand(B, Hk, block))
    was = raw[rows, :, old].view(torch.float8_e4m3fn).float() * ratio.transpose(1, 2)[..., None]
    raw[rows, :, old] = was.to(torch.float8_e4m3fn).view(torch.uint8)
    q = x / new.gather(2, blk)[..., None]
    q = torch.where(torch.isfinite(q), q, math.nan).to(torch.float8_e4m3fn)
    raw[rows, :, pos] = q.transpose(1, 2).contiguous().view(torch.uint8)
    scales.copy_(new)


def _values(codes, scales, n, block, lens):
    """The first n rows as numbers; zeros from row lens[b] on."""
    x = codes[:, :, :n].float() * scales.repeat_interleave(block, 2)[:, :, :n, None]
    return torch.where(torch.arange(n, device=x.device)[:, None] < lens[:, None, None, None], x, 0.0)


def _plain_attend(s):
    c = s["case"]
    B, H, Hk, Dh, n = c["B"], c["H"], c["Hk"], c["Dh"], c["ctx"]
    k, v = (_values(s[x + "8"], s[x + "_scale"], n, c["block"], s["lens"]) for x in "kv")
    q = s["q"].float().view(B, Hk, H // Hk, Dh) / math.sqrt(Dh)
    seen = torch.arange(n, device=q.device)[None, None, None] < s["lens"][:, None, None, None]
    sc = torch.where(seen, q @ k.transpose(2, 3), -math.inf)
    p = torch.where(seen, torch.exp(sc - sc.amax(-1, keepdim=True)), 0.0)
    return ((p @ v) / p.sum(-1, keepdim=True)).view(B, H, Dh).to(torch.bfloat16)


def _plain_sample(s):
    """In 64 bits: the filters and the draw compare running sums of up to V weights."""
    x = s["logits"].double()
    B, V = x.shape

    def per_row(name, dtype):
        p = s[name]
        return (p.to(dtype) if torch.is_tensor(p) else torch.full((B,), p, dtype=dtype, device=x.device))[:, None]

    T, top_k = per_row("temperature", torch.float64), per_row("top_k", torch.int64)
    top_p, min_p = per_row("top_p", torch.float32).double(), per_row("min_p", torch.float32).double()
    T = T.float().double()   # (the settings are 32-bit numbers)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(T > 0, T, 1.0))
    rank = torch.arange(V, device=x.device)[None]
    keep = rank < torch.where(T > 0, torch.where(top_k > 0, top_k, V), 1)
    w = torch.where(keep, w, 0.0)
    before = torch.cumsum(w, -1) - w
    keep &= (top_p >= 1.0) | (before <= top_p * w.sum(-1, keepdim=True))
    keep &= w >= min_p
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))   # back to the vocabulary's order
    cum = torch.cumsum(w, -1)
    token = (cum <= s["uniforms"].double()[:, None] * cum[:, -1:]).sum(-1).clamp_max(V - 1)
    prob = w.gather(1, token[:, None])[:, 0] / cum[:, -1]
    return [token.to(torch.int32), prob.float()]


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        return [_rotated(s[x], s["positions"], s, torch.float32).to(s[x].dtype) for x in "qk"]
    if c["op"] == "attend":
        return _plain_attend(s)
    if c["op"] == "sample":
        return _plain_sample(s)
    pos = s["lens"][:, None] + torch.arange(c["L"], device=s["lens"].device)
    # 64 bits: a rotated key next to a border of the 8-bit grid
    q, k = (_rotated(s[x], pos, s, torch.float64).float().to(torch.bfloat16) for x in "qk")
    _append(s["k8"], s["k_scale"], k, s["lens"], c["block"])
    _append(s["v8"], s["v_scale"], s["v"], s["lens"], c["block"])
    n = c["ctx"] + c["L"]
    ends = s["lens"] + c["L"]
    return [q, *(_values(s[x + "8"], s[x + "_scale"], n, c["block"], ends).to(torch.bfloat16) for x in "kv")]


def run(s):
    if not own:
        return _plain(s)
    from flashsvd_b200 import kv8, ops

    c = s["case"]
    if c["op"] == "rope":
        return list(ops.rope_qk(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=c["layout"] == "interleaved",
                                scale=s["scale"]))
    if c["op"] == "sample":
        return list(ops.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                               min_p=s["min_p"]))
    cache = kv8.KV8Cache(s["k8"], s["v8"], s["k_scale"], s["v_scale"], c["block"])
    key = (c["B"], c["H"], c["Hk"], c["Dh"], cache.max_len)
    ws = _workspaces.get(key)
    if ws is None:
        ws = _workspaces[key] = ops.make_kv8_workspace(c["B"], c["H"], c["Hk"], c["Dh"], cache.max_len, s["q"].device)
    if c["op"] == "attend":
        return ops.flash_decode_kv8(s["q"], cache, s["lens"], ws)
    rotary = kv8.Rotary(s["inv_freq"], c["layout"] == "interleaved", s["scale"])
    q = ops.kv8_append(s["k"], s["v"], cache, s["lens"], ws, q=s["q"], rotary=rotary)
    return [q, *ops.kv8_load(cache, 0, c["ctx"] + c["L"], cache_seqlens=s["lens"], seqlen_add=c["L"])]


def work(case):
    c = case
    if c["op"] == "sample":
        n = c["B"] * c["V"]
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + 24 * c["B"], "flops": 8 * n}
    row = c["Hk"] * c["Dh"]
    if c["op"] == "rope":
        es = 4 if c["dtype"] == "f32" else 2
        n = c["T"] * (c["H"] * c["Dh"] + row)
        return {"bytes": 2 * n * es + 4 * c["T"] + 4 * c["rot"], "flops": 3 * c["T"] * (c["H"] + c["Hk"]) * c["rot"]}
    if c["op"] == "attend":
        keys = sum(_lens(c))
        scales = 8 * c["Hk"] * sum(-(-n // c["block"]) for n in _lens(c))
        return {"bytes": 2 * keys * row + scales + 4 * c["B"] * c["H"] * c["Dh"] + 4 * c["B"], "flops": 4 * keys * c["H"] * c["Dh"]}
    new, held, back = c["B"] * c["L"], sum(_lens(c)) + c["B"] * c["L"], c["B"] * (c["ctx"] + c["L"])
    return {"bytes": 4 * new * c["H"] * c["Dh"] + 2 * (2 + 1) * new * row + 2 * (held + 2 * back) * row,
            "flops": 3 * new * (c["H"] + c["Hk"]) * c["rot"] + 2 * held * row}


# ---- the operators' definitions in 64 bits
def _exact_rotation(x, pos, s):
    """As complex numbers: each pair times scale * exp(i position frequency)."""
    c, r = s["case"], s["case"]["rot"]
    head = x.double()[..., :r]
    pairs = head.unflatten(-1, (2, r // 2)).transpose(-1, -2) if c["layout"] == "half" else head.unflatten(-1, (r // 2, 2))
    z = torch.view_as_complex(pairs.contiguous())
    z = z * torch.polar(torch.full_like(s["inv_freq"], s["scale"]), pos.double()[..., None] * s["inv_freq"])[..., None, :]
    y = torch.view_as_real(z)
    y = y.transpose(-1, -2).flatten(-2) if c["layout"] == "half" else y.flatten(-2)
    return torch.cat([y, x.double()[..., r:]], -1)


def _two_to(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e.round().to(torch.int32))


def _grid(y):
    """y rounded to the e4m3 numbers (3 bits behind the leading one, exponents from -6, ties to even)."""
    step = _two_to((torch.frexp(y)[1] - 1).clamp_min(-6) - 3.0)
    return torch.round(y / step) * step


def _exact_exponent(amax):
    """The smallest e >= MIN_EXP with amax <= 448 2^e."""
    e = torch.round(torch.log2(amax / E4M3_MAX)).clamp_min(MIN_EXP) - 1   # log2 may be off by an ulp
    for _ in range(2):
        e = torch.where(amax > E4M3_MAX * _two_to(e), e + 1, e)
    return e.clamp_min(MIN_EXP)


def _exact_cache(codes, scales, x, lens, n, block):
    """Values of the first n tokens after x[B, L, Hk, Dh] (bf16) went in, one sequence and block after the other."""
    out = codes[:, :, :n].double() * scales.double().repeat_interleave(block, 2)[:, :, :n, None]
    for b, first in enumerate(lens):
        end = first + x.shape[1]
        for t0 in range(first // block * block, end, block):
            lo, hi = max(first, t0), min(end, t0 + block)
            new = x[b, lo - first:hi - first].double().transpose(0, 1)
            e = _exact_exponent(new.abs().amax((1, 2)))
            if t0 < first:
                e = torch.maximum(e, torch.round(torch.log2(scales[b, :, t0 // block].double())))
            scale = _two_to(e)[:, None, None]
            out[b, :, t0:lo] = _grid(out[b, :, t0:lo] / scale) * scale
            out[b, :, lo:hi] = _grid(new / scale) * scale
        out[b, :, end:] = 0.0
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        return [_exact_rotation(s[x], s["positions"], s) for x in "qk"]
    if c["op"] == "update":
        pos = s["lens"][:, None] + torch.arange(c["L"], device=s["lens"].device)
        q, k = (_exact_rotation(s[x], pos, s) for x in "qk")
        k = k.float().to(torch.bfloat16)   # the key that the cache is given
        n = c["ctx"] + c["L"]
        return [q, *(_exact_cache(s[x + "8"], s[x + "_scale"], y, _lens(c), n, c["block"]) for x, y in (("k", k), ("v", s["v"])))]
    if c["op"] == "attend":
        G = c["H"] // c["Hk"]
        out = torch.zeros(c["B"], c["H"], c["Dh"], dtype=torch.float64, device=s["q"].device)
        for b, n in enumerate(_lens(c)):
            if n > 0:
                k, v = (s[x + "8"][b, :, :n].double() * s[x + "_scale"][b].double().repeat_interleave(c["block"], 1)[:, :n, None]
                        for x in "kv")
                q = s["q"][b].double().view(c["Hk"], G, c["Dh"])
                p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) * c["Dh"] ** -0.5, -1)
                out[b] = torch.einsum("hgn,hnd->hgd", p, v).reshape(c["H"], c["Dh"])
        return out
    tokens, probs = [], []
    setting = {k: s[k].tolist() if torch.is_tensor(s[k]) else [torch.tensor(s[k], dtype=torch.float32).item()] * c["B"]
               for k in ("temperature", "top_k", "top_p", "min_p")}
    for b in range(c["B"]):
        x = s["logits"][b].double().cpu()
        T, k, p, m = (setting[n][b] for n in ("temperature", "top_k", "top_p", "min_p"))
        if T <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            probs.append(1.0)
            continue
        w, at = torch.sort(torch.exp((x - x.max()) / T), descending=True, stable=True)
        if 0 < k < c["V"]:
            w, at = w[:int(k)], at[:int(k)]
        if p < 1.0:
            count = int((torch.cumsum(w, 0) <= p * w.sum()).sum()) + 1   # up to the one that passes p
            w, at = w[:count], at[:count]
        w, at = w[w >= m], at[w >= m]
        at, order = torch.sort(at)
        cum = torch.cumsum(w[order], 0)
        i = int(torch.searchsorted(cum, s["uniforms"][b].double().cpu() * cum[-1], right=True).clamp_max(len(at) - 1))
        tokens.append(int(at[i]))
        probs.append(float(w[order][i] / cum[-1]))
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)]
