"""The 8-bit cache: append and read-back bit for bit against the definition in 64 bits, attention within the output's
rounding.

Attention's tolerance: one bf16 rounding (half a step, 2^-8 of the value); weights are kept to 16 bits or more (2^-16
of the largest value) and scores of magnitude up to 64 to 24 bits (64 * 2^-24 * 4 = 2^-16): 2^-14 of the largest value
covers both with room."""
import math

import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _values(cache):
    from flashsvd_b200 import ops

    k, v = ops.kv8_load(cache, 0, cache.max_len)
    return k.double().cpu(), v.double().cpu()


def _same(got, want):
    return bool(((got == want) | (torch.isnan(got) & torch.isnan(want))).all())


def _rotary(R, interleaved=False, scale=1.0):
    from flashsvd_b200 import kv8

    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    return kv8.Rotary(f.to(DEV), interleaved, scale)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("Dh,R,inter", [(64, 64, False), (128, 128, False), (128, 64, True), (64, 48, False), (128, 20, False),
                                        (64, 0, False)])
def test_append_in_pieces_matches_the_definition(block, Dh, R, inter):
    """Three appends of ragged lengths over one cache, with values that grow, shrink and vanish."""
    from flashsvd_b200 import kv8, ops

    B, Hk, H, S = 3, 2, 6, 150
    gen = torch.Generator().manual_seed(block + Dh + R)
    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
    ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
    rk, rv = ref.Cache(B, Hk, S, Dh, block), ref.Cache(B, Hk, S, Dh, block)
    lens = torch.tensor([0, 5, 63], dtype=torch.int32)
    # the tokens that the sequences hold at the start
    first = torch.randn(B, 63, Hk, Dh, generator=gen).to(torch.bfloat16)
    counts = [0, 5, 63]
    ops.kv8_append(first.to(DEV), first.to(DEV), cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws,
                   new_lens=torch.tensor(counts, dtype=torch.int32, device=DEV))
    rk.append(first, [0] * B, counts), rv.append(first, [0] * B, counts)
    rot = _rotary(R, inter, 1.125) if R else None
    for L, gain in ((1, 8.0), (37, 1.0), (1, 0.0), (30, 100.0), (1, 3000.0)):
        qkv = torch.randn(B, L, H + 2 * Hk, Dh, generator=gen)
        qkv[:, :, H:] *= gain
        qkv = qkv.to(torch.bfloat16)
        q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        new = [L, max(0, L - 1), L]
        dq = qkv.to(DEV)
        out = torch.full((B, L, H, Dh), 7.0, dtype=torch.bfloat16, device=DEV)
        got = ops.kv8_append(dq[:, :, H:H + Hk], dq[:, :, H + Hk:], cache, lens.to(DEV), ws,
                             new_lens=torch.tensor(new, dtype=torch.int32, device=DEV), q=dq[:, :, :H] if R else None,
                             rotary=rot, q_out=out if R else None)
        pos = lens[:, None] + torch.arange(L)
        if R:
            f = rot.inv_freq.cpu()
            k = ref.to_bf16(ref.rotate(k, pos, f, inter, 1.125))
            want = ref.rotate(q, pos, f, inter, 1.125)
            err = (got.double().cpu() - want).abs() - want.abs() * 2.0 ** -8 - 1e-6 * q.double().abs().max()
            for b in range(B):
                assert bool((err[b, :new[b]] <= 0).all())
                assert bool((got[b, new[b]:] == 7.0).all())
        rk.append(k, lens.tolist(), new), rv.append(v, lens.tolist(), new)
        lens += torch.tensor(new, dtype=torch.int32)
        for b in range(B):
            n = int(lens[b])
            for (val, exps, scales) in zip(_values(cache), (rk, rv), (cache.k_scale, cache.v_scale)):
                assert torch.equal(val[b, :, :n], exps.val[b, :, :n])
                used = -(-n // block)
                assert torch.equal(torch.log2(scales[b, :, :used].double().cpu()), exps.exp[b, :, :used].double())
    assert ws.status() == 0


def test_append_leaves_the_rest_of_the_cache():
    from flashsvd_b200 import kv8, ops

    cache = kv8.KV8Cache.empty(2, 200, 2, 64, block=32, device=DEV)
    cache.k.view(torch.uint8).fill_(0x7b)
    cache.v.view(torch.uint8).fill_(0x13)
    cache.k_scale.fill_(3.0)
    x = torch.randn(2, 10, 2, 64, device=DEV).to(torch.bfloat16)
    ws = ops.make_kv8_workspace(2, 2, 2, 64, 200, DEV)
    ops.kv8_append(x, x, cache, torch.tensor([32, 70], dtype=torch.int32, device=DEV), ws)
    k = cache.k.view(torch.uint8)
    for b, lo in ((0, 32), (1, 70)):
        assert bool((k[b, :, lo + 10:] == 0x7b).all()) and bool((cache.v.view(torch.uint8)[b, :, :lo] == 0x13).all())
    assert bool((k[0, :, :32] == 0x7b).all())
    s = cache.k_scale.cpu()
    assert bool((s[0, :, 0] == 3.0).all() and (s[0, :, 2:] == 3.0).all() and (s[1, :, 3:] == 3.0).all())
    assert bool((s[1, :, 2] == 3.0).all())   # tokens 64..69 were there: their scale only grows


def test_append_past_the_end_drops_and_says_so():
    from flashsvd_b200 import kv8, ops

    B, S = 2, 40
    cache = kv8.KV8Cache.empty(B, S, 1, 64, block=16, device=DEV)
    ws = ops.make_kv8_workspace(B, 1, 1, 64, S, DEV)
    x = torch.randn(B, 6, 1, 64, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    guard = cache.k_scale.clone()
    ops.kv8_append(x.to(DEV), x.to(DEV), cache, torch.tensor([37, 40], dtype=torch.int32, device=DEV), ws)
    want = ref.Cache(B, 1, S, 64, 16)
    assert want.append(x, [37, 40], [6, 6])
    k, _ = _values(cache)
    assert torch.equal(k[0, :, 37:], want.val[0, :, 37:]) and bool((k[1] == 0).all())
    assert torch.equal(cache.k_scale[1], guard[1])
    assert ws.raw_status() == 4
    with pytest.raises(IndexError):
        ws.status()
    ws.clear_status()
    assert ws.status() == 0
    # queries of tokens that do not fit are rotated all the same
    rot = _rotary(64)
    q = torch.randn(B, 6, 1, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    got = ops.kv8_append(x.to(DEV), x.to(DEV), cache, torch.tensor([37, 1000], dtype=torch.int32, device=DEV), ws, q=q.to(DEV), rotary=rot)
    want = ref.rotate(q, torch.tensor([[37], [1000]]) + torch.arange(6), rot.inv_freq.cpu())
    assert bool(((got.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 1e-6 * q.double().abs().max()).all())


def test_append_borders_of_the_scale_and_values_that_are_not_finite():
    from flashsvd_b200 import kv8, ops

    Dh, block = 64, 16
    tops = [448.0, 450.0, 3.5, 3.515625, 1e-30, 0.0, 3.3e38, 2.0 ** -52, 448.0 * 2.0 ** -60]
    x = torch.zeros(1, block * len(tops), 1, Dh, dtype=torch.bfloat16)
    gen = torch.Generator().manual_seed(3)
    for i, t in enumerate(tops):
        x[0, i * block:(i + 1) * block, 0] = (torch.rand(block, Dh, generator=gen) * 2 - 1).to(torch.bfloat16) * t
        x[0, i * block + 3, 0, 5] = t
    x[0, 1, 0, 0], x[0, 2, 0, 1], x[0, 20, 0, 2] = math.inf, -math.inf, math.nan
    x[0, 2 * block:3 * block, 0, 7] = math.nan
    cache = kv8.KV8Cache.empty(1, x.shape[1], 1, Dh, block=block, device=DEV)
    ws = ops.make_kv8_workspace(1, 1, 1, Dh, x.shape[1], DEV)
    ops.kv8_append(x.to(DEV), x.to(DEV), cache, torch.zeros(1, dtype=torch.int32, device=DEV), ws)
    want = ref.Cache(1, 1, x.shape[1], Dh, block)
    want.append(x, [0], [x.shape[1]])
    for val, s in zip(_values(cache), (cache.k_scale, cache.v_scale)):
        # (read back as bf16: a code of a block near the top of bf16's range stays inside it)
        assert _same(val, want.val)
        assert torch.equal(torch.log2(s.double().cpu()), want.exp.double())


def test_load_ranges_and_rows_behind_the_end():
    from flashsvd_b200 import kv8, ops

    cache = kv8.KV8Cache.empty(2, 70, 3, 128, block=16, device=DEV)
    x = torch.randn(2, 70, 3, 128, device=DEV).to(torch.bfloat16)
    ws = ops.make_kv8_workspace(2, 3, 3, 128, 70, DEV)
    ops.kv8_append(x, -x, cache, torch.zeros(2, dtype=torch.int32, device=DEV), ws)
    k, v = ops.kv8_load(cache, 0, 70)
    assert torch.equal(k, -v)
    lens = torch.tensor([0, 33], dtype=torch.int32, device=DEV)
    for start, n in ((0, 70), (13, 40), (69, 1), (70, 0)):
        a, b = ops.kv8_load(cache, start, n)
        assert torch.equal(a, k[:, :, start:start + n]) and torch.equal(b, v[:, :, start:start + n])
        a, _ = ops.kv8_load(cache, start, n, cache_seqlens=lens, seqlen_add=2)
        for i, m in enumerate((2, 35)):
            keep = max(0, min(n, m - start))
            assert torch.equal(a[i, :, :keep], k[i, :, start:start + keep]) and not bool(a[i, :, keep:].any())


def _filled(B, Hk, S, Dh, block, gen, k_gain=1.0):
    from flashsvd_b200 import kv8, ops

    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
    ws = ops.make_kv8_workspace(B, Hk, Hk, Dh, S, DEV)
    k, v = (torch.randn(B, S, Hk, Dh, generator=gen).to(torch.bfloat16) for _ in range(2))
    ops.kv8_append((k * k_gain).to(DEV), v.to(DEV), cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws)
    return cache


@pytest.mark.parametrize("B,H,Hk,Dh,S,lens,block", [
    (1, 1, 1, 64, 1, [1], 16), (1, 4, 4, 128, 40, [33], 64), (2, 8, 4, 64, 300, [300, 0], 32), (3, 8, 4, 128, 517, [1, 516, 257], 128),
    (2, 8, 2, 64, 1030, [1030, 31], 16), (1, 16, 2, 128, 4100, [4099], 64), (8, 8, 1, 128, 129, [129, 128, 127, 65, 64, 33, 32, 1], 64),
    (8, 32, 32, 128, 260, [260] * 8, 64), (2, 48, 3, 128, 700, [699, 5], 32), (1, 3, 1, 64, 20000, [19999], 128),
    (2, 20, 4, 128, 385, [384, 385], 64), (40, 12, 12, 64, 150, [(7 * i) % 151 for i in range(40)], 16)])
def test_attention(B, H, Hk, Dh, S, lens, block):
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(B * 1000 + S)
    cache = _filled(B, Hk, S, Dh, block, gen)
    q = (2 * torch.randn(B, H, Dh, generator=gen)).to(torch.bfloat16)
    ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
    k, v = _values(cache)
    want = ref.attend(q, k, v, lens, Dh ** -0.5)
    bound = want.abs() * 2.0 ** -8 + 2.0 ** -14 * float(v.abs().max())
    n = torch.tensor(lens, dtype=torch.int32)
    for _ in range(2):   # the second call finds the arrival counters as the first one left them
        out = ops.flash_decode_kv8(q.to(DEV), cache, n.to(DEV), ws)
        assert bool(((out.double().cpu() - want).abs() <= bound).all())
    again = ops.flash_decode_kv8(q.to(DEV), cache, (n - 1).to(DEV), ws, seqlen_add=1)
    assert torch.equal(again, out)
    other = ops.flash_decode_kv8(q.to(DEV), cache, n.to(DEV), ws, scale=0.03)
    want = ref.attend(q, k, v, lens, 0.03)
    assert bool(((other.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * float(v.abs().max())).all())


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 8])
def test_attention_does_not_see_what_lies_behind_the_end(Dh, G):
    """NaN codes and scales behind the last position, in the same tile and block, change nothing."""
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(9)
    B, Hk, S = 2, 2, 300
    cache = _filled(B, Hk, S, Dh, 32, gen)
    q = torch.randn(B, Hk * G, Dh, generator=gen).to(torch.bfloat16).to(DEV)
    ws = ops.make_kv8_workspace(B, Hk * G, Hk, Dh, S, DEV)
    for n in (1, 31, 128, 200, 257):
        lens = torch.tensor([n, 0], dtype=torch.int32, device=DEV)
        want = ops.flash_decode_kv8(q, cache, lens, ws)
        assert not bool(want[1].any())
        k, v, ks, vs = (t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[0, :, n:] = 0x7f
            t.view(torch.uint8)[1] = 0xff
        for t in (cache.k_scale, cache.v_scale):
            t[0, :, -(-n // 32):] = math.nan
            t[1] = math.inf
        assert torch.equal(ops.flash_decode_kv8(q, cache, lens, ws), want)
        for t, s in ((cache.k, k), (cache.v, v)):
            t.view(torch.uint8).copy_(s.view(torch.uint8))
        cache.k_scale.copy_(ks), cache.v_scale.copy_(vs)


@pytest.mark.parametrize("Dh", [64, 128])
def test_attention_with_values_that_are_not_numbers(Dh):
    """A NaN value reaches its dimension, a NaN key or query every dimension of the heads that see it, nothing else."""
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(10)
    cache = _filled(2, 2, 200, Dh, 64, gen)
    q = torch.randn(2, 4, Dh, generator=gen).to(torch.bfloat16).to(DEV)
    ws = ops.make_kv8_workspace(2, 4, 2, Dh, 200, DEV)
    lens = torch.tensor([150, 200], dtype=torch.int32, device=DEV)
    clean = ops.flash_decode_kv8(q, cache, lens, ws)
    cache.v.view(torch.uint8)[0, 1, 77, 5] = 0x7f
    out = ops.flash_decode_kv8(q, cache, lens, ws)
    assert bool(torch.isnan(out[0, 2:, 5]).all())
    out[0, 2:, 5] = clean[0, 2:, 5]
    assert torch.equal(out, clean)
    cache.v.view(torch.uint8)[0, 1, 77, 5] = 0
    clean = ops.flash_decode_kv8(q, cache, lens, ws)
    cache.k.view(torch.uint8)[1, 0, 3, 9] = 0xff
    q[0, 0, 3] = math.inf
    out = ops.flash_decode_kv8(q, cache, lens, ws)
    assert bool(torch.isnan(out[1, :2]).all()) and bool(torch.isnan(out[0, 0]).all())
    assert torch.equal(out[1, 2:], clean[1, 2:]) and torch.equal(out[0, 1:], clean[0, 1:])


def test_attention_weights_over_wide_ranges():
    """Scores that differ by thousands, equal scores, blocks of very different scales, values of one sign."""
    from flashsvd_b200 import kv8, ops

    B, H, Hk, Dh, S, block = 1, 2, 1, 128, 640, 64
    gen = torch.Generator().manual_seed(11)
    k = torch.randn(B, S, Hk, Dh, generator=gen)
    v = torch.rand(B, S, Hk, Dh, generator=gen) + 0.5
    v *= 2.0 ** (torch.arange(S) // block * 3 - 15)[None, :, None, None]
    for gain in (0.0, 1.0, 30.0):
        cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
        ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
        ops.kv8_append((k * gain).to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), cache,
                       torch.zeros(B, dtype=torch.int32, device=DEV), ws)
        q = (3 * torch.randn(B, H, Dh, generator=gen)).to(torch.bfloat16)
        kv, vv = _values(cache)
        for n in (640, 63, 320):
            want = ref.attend(q, kv, vv, [n], Dh ** -0.5)
            got = ops.flash_decode_kv8(q.to(DEV), cache, torch.tensor([n], dtype=torch.int32, device=DEV), ws).double().cpu()
            # values of one sign: the result is a mean of positive numbers, so weights' errors are relative to it:
            # half a bf16 step, and scores to |s| 2^-20 (sums of 128 products of 24 bits; |s| up to 1500 here)
            s = float((kv[0, 0] @ q[0].double().T).abs().max()) * Dh ** -0.5
            assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -13 + s * 2.0 ** -19)).all())


def test_attention_in_a_graph_beside_a_second_workspace():
    """Two captured calls with workspaces of their own, replayed with other lengths."""
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(12)
    cache = _filled(2, 4, 900, 128, 64, gen)
    q = torch.randn(2, 8, 128, generator=gen).to(torch.bfloat16).to(DEV)
    lens = torch.tensor([900, 450], dtype=torch.int32, device=DEV)
    wss = [ops.make_kv8_workspace(2, 8, 4, 128, 900, DEV) for _ in range(2)]
    outs, graphs = [torch.empty_like(q) for _ in range(2)], []
    ops.flash_decode_kv8(q, cache, lens, wss[0])
    torch.cuda.synchronize()
    for ws, out in zip(wss, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.flash_decode_kv8(q, cache, lens, ws, out=out)
        graphs.append(graph)
    for new in ([900, 450], [1, 899], [0, 300]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        want = ops.flash_decode_kv8(q, cache, lens, ops.make_kv8_workspace(2, 8, 4, 128, 900, DEV))
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 codes: the last sequence's rows."""
    from flashsvd_b200 import kv8, ops

    B, Hk, S, Dh = 3, 8, 1 << 21, 128   # 3 * 8 * 2^21 * 128 = 6.4e9 codes each
    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=128, device=DEV)
    ws = ops.make_kv8_workspace(B, Hk, Hk, Dh, S, DEV)
    gen = torch.Generator().manual_seed(13)
    n, L = 300, 300
    k, v = (torch.randn(B, L, Hk, Dh, generator=gen).to(torch.bfloat16) for _ in range(2))
    at = S - n
    ops.kv8_append(k.to(DEV), v.to(DEV), cache, torch.full((B,), at, dtype=torch.int32, device=DEV), ws)
    kk, vv = ops.kv8_load(cache, at, n)
    want = ref.Cache(1, Hk, 2 * n, Dh, 128)
    start = at % 128   # the same place inside a block
    want.append(k[B - 1:], [start], [n])
    assert torch.equal(kk[B - 1].double().cpu(), want.val[0, :, start:start + n])
    q = torch.randn(B, Hk, Dh, generator=gen).to(torch.bfloat16)
    out = ops.flash_decode_kv8(q.to(DEV), cache, torch.full((B,), S, dtype=torch.int32, device=DEV), ws).double().cpu()
    # the positions in front hold zero keys and values: score 0, weight exp(-max)
    s = torch.einsum("hd,hnd->hn", q[B - 1].double(), kk[B - 1].double().cpu()) * Dh ** -0.5
    w = torch.exp(s - s.amax(1, keepdim=True))
    den = w.sum(1) + at * torch.exp(-s.amax(1))
    ref_out = torch.einsum("hn,hnd->hd", w, vv[B - 1].double().cpu()) / den[:, None]
    assert bool(((out[B - 1] - ref_out).abs() <= ref_out.abs() * 2.0 ** -8 + 2.0 ** -14 * float(vv.abs().max())).all())
    assert ws.status() == 0
