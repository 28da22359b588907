"""Softmax weights and queries of the attention over the 8-bit cache where few of their bits carry the result.

The weights of a tile are fp32 numbers; nothing of a weight may leave the numerator that the denominator counts."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _codes(x):
    return x.to(torch.float8_e4m3fn)


def _cache(B, Hk, S, Dh, block=128):
    from flashsvd_b200 import kv8

    return kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)


@pytest.mark.parametrize("Dh,G,pairs,n,steps", [(64, 1, 640, 2000, (20, 22.9, 24.4, 25.9, 26.1, 28, 30)),
                                                (128, 2, 320, 2000, (20, 24.4, 26.1)), (64, 4, 320, 2000, (20, 24.4, 26.1)),
                                                (128, 8, 320, 2000, (20, 24.4, 26.1)), (128, 16, 160, 2000, (20, 24.4, 26.1)),
                                                (64, 16, 160, 2000, (24.4,)), (64, 8, 320, 2000, (24.4,)),
                                                (64, 1, 300, 131071, (20, 22.9, 25.9, 26.1, 28, 30)), (128, 8, 80, 131071, (26.1,)),
                                                (64, 1, 64, 1 << 20, (22.9, 26.1, 28, 30))])
def test_a_dominant_token_in_front_of_a_long_flat_context(Dh, G, pairs, n, steps):
    """One token whose value is zero, and n - 1 equal ones at 2^-step of its weight: they alone are the result.

    Tolerance: half a bf16 step and 2^-14 of the largest value, as for attention at large.  Enough pairs that a CTA goes
    through a whole context, or most of it, with one running maximum."""
    from flashsvd_b200 import ops

    cache = _cache(pairs, 1, n, Dh)
    gen = torch.Generator(device=DEV).manual_seed(n + Dh + G)
    values = _codes(torch.rand(pairs, 1, 1, Dh, device=DEV, generator=gen) + 0.5)
    cache.v.view(torch.uint8).copy_(values.view(torch.uint8).expand(pairs, 1, n, Dh))
    at = torch.randint(0, n, (pairs,), generator=torch.Generator().manual_seed(n))
    at[0], at[1], at[2] = 0, n - 1, n // 2
    rows = torch.arange(pairs, device=DEV)
    cache.v.view(torch.uint8)[rows, 0, at.to(DEV)] = 0
    cache.k.view(torch.uint8)[rows, 0, at.to(DEV), 3] = int(_codes(torch.ones(1)).view(torch.uint8))
    q = torch.zeros(pairs, G, Dh, device=DEV, dtype=torch.bfloat16)
    q[:, :, 3] = 1.0
    lens = torch.full((pairs,), n, dtype=torch.int32, device=DEV)
    ws = ops.make_kv8_workspace(pairs, G, 1, Dh, n, DEV)
    v = values.double()[:, 0]
    for step in steps:
        scale = torch.tensor(step * math.log(2.0), dtype=torch.float32).item()
        tail = (n - 1) * math.exp(-scale)
        want = (v * tail / (1.0 + tail)).expand(pairs, G, Dh)
        got = ops.flash_decode_kv8(q, cache, lens, ws, scale=scale).double()
        assert bool(((got - want).abs() <= want * 2.0 ** -8 + 2.0 ** -14 * 1.5).all()), step
    assert ws.status() == 0


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 4, 8, 16])
def test_weights_have_their_bits(Dh, G):
    """Two tokens of values +448 and -448 and almost equal weights 1 and w: the result is 448 (1 - w) / (1 + w).

    Scores are exact (one product each; the smaller is at most 2^-6) but for a few roundings of 2^-24 of it, the
    exponential is good to 2^-22 and the sums of two terms to 2^-23: w within 2^-21, the result within 448 * 2^-22, and half
    a bf16 step.  448 * 2^-20 leaves room for what the exponential's argument adds."""
    from flashsvd_b200 import ops

    pairs = 512
    cache = _cache(pairs, 1, 2, Dh, block=16)
    one, big = (int(_codes(torch.tensor([x])).view(torch.uint8)) for x in (1.0, 448.0))
    cache.v.view(torch.uint8)[:, 0, 0], cache.v.view(torch.uint8)[:, 0, 1] = big, big | 0x80
    cache.k.view(torch.uint8)[:, 0, 1, 7] = one
    gen = torch.Generator().manual_seed(G + Dh)
    q = torch.zeros(pairs, G, Dh)
    q[:, :, 7] = -(2.0 ** (-14 + 8 * torch.rand(pairs, G, generator=gen)))
    q = q.to(torch.bfloat16)
    ws = ops.make_kv8_workspace(pairs, G, 1, Dh, 2, DEV)
    got = ops.flash_decode_kv8(q.to(DEV), cache, torch.full((pairs,), 2, dtype=torch.int32, device=DEV), ws, scale=1.0).double().cpu()
    w = torch.exp(q[:, :, 7].double())
    want = (448 * (1 - w) / (1 + w))[..., None].expand(pairs, G, Dh)
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 448 * 2.0 ** -20).all())


@pytest.mark.parametrize("Dh", [64, 128])
def test_weights_over_thirty_binades_beside_a_dominant_one(Dh):
    """Random scores over 26 units below one token of value zero, values of one sign: a mean, so errors are relative to it.

    Half a bf16 step; weights to 2^-20 of themselves (scores of up to 40 to 2^-24 each, four roundings); the weights below
    2^-33 of the largest are 2^-16 of the others together at most."""
    from flashsvd_b200 import ops

    B, Hk, G, S = 16, 40, 2, 3000
    gen = torch.Generator(device=DEV).manual_seed(Dh)
    cache = _cache(B, Hk, S, Dh, block=64)
    v = _codes(torch.rand(B, Hk, S, Dh, device=DEV, generator=gen) + 0.5)
    v[:, :, 1234].view(torch.uint8).zero_()
    cache.v.view(torch.uint8).copy_(v.view(torch.uint8))
    k = _codes(torch.randint(-15, 16, (B, Hk, S, Dh), device=DEV, generator=gen).float())
    k[..., 1:] = 0 * k[..., 1:].float().to(torch.float8_e4m3fn).float()
    k[:, :, 1234, 0] = _codes(torch.tensor([28.0], device=DEV))[0]
    cache.k.view(torch.uint8).copy_(k.view(torch.uint8))
    q = torch.zeros(B, Hk * G, Dh, device=DEV, dtype=torch.bfloat16)
    q[:, 0::2, 0], q[:, 1::2, 0] = 0.5, 0.6015625
    ws = ops.make_kv8_workspace(B, Hk * G, Hk, Dh, S, DEV)
    got = ops.flash_decode_kv8(q, cache, torch.full((B,), S, dtype=torch.int32, device=DEV), ws, scale=1.0).double()
    s = torch.einsum("bhgd,bhnd->bhgn", q.double().view(B, Hk, G, Dh), k.double())
    want = (torch.softmax(s, -1) @ v.double()).view(B, Hk * G, Dh)
    assert bool(((got - want).abs() <= want * (2.0 ** -8 + 2.0 ** -14)).all())


@pytest.mark.parametrize("Dh", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 4, 8, 16])
def test_small_query_numbers_beside_a_dominant_token(Dh, G):
    """The two opposite values again, beside a token that outweighs them 2^j times and whose value is zero: their weights
    differ by a query number far below the row's largest.

    Each number of the row has its 8 bits down to 2^-17 of the largest, below that it is off by 2^-26 of it."""
    from flashsvd_b200 import ops

    pairs = 512
    one, big = (int(_codes(torch.tensor([x])).view(torch.uint8)) for x in (1.0, 448.0))
    gen = torch.Generator().manual_seed(G + Dh)
    q = torch.zeros(pairs, G, Dh)
    q[:, :, 7] = -(2.0 ** (-14 + 8 * torch.rand(pairs, G, generator=gen)))
    q = q.to(torch.bfloat16)
    ws = ops.make_kv8_workspace(pairs, G, 1, Dh, 3, DEV)
    w = torch.exp(q[:, :, 7].double())
    cache = _cache(pairs, 1, 3, Dh, block=16)
    cache.v.view(torch.uint8)[:, 0, 0], cache.v.view(torch.uint8)[:, 0, 1] = big, big | 0x80
    cache.k.view(torch.uint8)[:, 0, 1, 7] = one
    cache.k.view(torch.uint8)[:, 0, 2, 9] = one
    three = torch.full((pairs,), 3, dtype=torch.int32, device=DEV)
    for j in (1, 5, 9, 12):
        top = torch.tensor(j * math.log(2.0)).to(torch.bfloat16)
        q[:, :, 9] = top
        got = ops.flash_decode_kv8(q.to(DEV), cache, three, ws, scale=1.0).double().cpu()
        want = (448 * (1 - w) / (1 + w + math.exp(float(top))))[..., None].expand(pairs, G, Dh)
        # (the scores below the largest one carry its roundings: 9 * 2^-23, relative to the two weights)
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 448 * math.exp(-float(top)) * 2.0 ** -19).all()), j


@pytest.mark.parametrize("Dh,G", [(64, 1), (128, 2), (64, 4), (128, 8), (64, 16), (128, 16)])
@pytest.mark.parametrize("up", [0, 8, 14, 15, 60])
def test_query_rows_with_one_large_number(Dh, G, up):
    """The row's largest number meets keys of zero: the scores come from numbers 2^up below it.

    Up to 2^15 they have all their bits, and the bound is attention's own.  At 2^60 they vanish (2^-25 of the largest is
    what a row keeps): every score is zero and the result the mean."""
    from flashsvd_b200 import kv8, ops
    from tests import kv8_reference as ref

    B, Hk, S = 3, 2, 200
    gen = torch.Generator().manual_seed(up + Dh + G)
    k, v = (torch.randn(B, S, Hk, Dh, generator=gen).to(torch.bfloat16) for _ in range(2))
    k[..., 5] = 0.0
    q = torch.randn(B, Hk * G, Dh, generator=gen)
    q = q.sign() * q.abs().clamp(0.5, 1.99)
    q[:, :, 5] = -1.5 * 2.0 ** up
    q = q.to(torch.bfloat16)
    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=32, device=DEV)
    ws = ops.make_kv8_workspace(B, Hk * G, Hk, Dh, S, DEV)
    ops.kv8_append(k.to(DEV), v.to(DEV), cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws)
    kk, vv = (x.double().cpu() for x in ops.kv8_load(cache, 0, S))
    got = ops.flash_decode_kv8(q.to(DEV), cache, torch.full((B,), S, dtype=torch.int32, device=DEV), ws).double().cpu()
    want = ref.attend(q if up < 60 else torch.zeros_like(q), kk, vv, [S] * B, Dh ** -0.5)
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * float(vv.abs().max())).all())


@pytest.mark.parametrize("Dh,G", [(64, 1), (128, 2), (64, 4), (128, 8), (64, 16)])
def test_scales_of_the_whole_range_in_one_sequence(Dh, G):
    """Blocks of tiny values, of values near bf16's largest and of zeros, wherever the likely tokens are.

    Every weight counts in the denominator, whatever its value's scale.  The results are means of numbers of one sign, so that
    errors are relative to them: half a bf16 step, and the weights' own."""
    from flashsvd_b200 import kv8, ops

    block, S = 16, 16 * 40
    gen = torch.Generator().manual_seed(Dh + G)
    size = torch.zeros(S)
    for b, x in {0: 1e-25, 3: 1e30, 7: 0.0, 8: 1.0, 9: 3e37, 17: 1e-18, 20: 1e24, 33: 0.0, 39: 1e10}.items():
        size[b * block:(b + 1) * block] = x
    v = ((torch.rand(1, S, 1, Dh, generator=gen) + 0.5) * size[None, :, None, None]).to(torch.bfloat16)
    for likely in range(0, 40, 1):
        k = torch.zeros(1, S, 1, Dh, dtype=torch.bfloat16)
        k[:, likely * block:(likely + 1) * block, :, 3] = 1.0
        cache = kv8.KV8Cache.empty(1, S, 1, Dh, block=block, device=DEV)
        ws = ops.make_kv8_workspace(1, G, 1, Dh, S, DEV)
        ops.kv8_append(k.to(DEV), v.to(DEV), cache, torch.zeros(1, dtype=torch.int32, device=DEV), ws)
        kk, vv = (x.double().cpu()[0, 0] for x in ops.kv8_load(cache, 0, S))
        q = torch.zeros(1, G, Dh)
        q[0, :, 3] = torch.linspace(2.0, 60.0, G) if G > 1 else 20.0
        q = q.to(torch.bfloat16)
        for n in (S, S - 5, 16 * 10):
            got = ops.flash_decode_kv8(q.to(DEV), cache, torch.tensor([n], dtype=torch.int32, device=DEV), ws, scale=1.0).double().cpu()[0]
            p = torch.softmax(q[0].double() @ kk[:n].T, -1)
            want = p @ vv[:n]
            # (scores of at most 60 log2(e) to 2^-22 of themselves: weights to 2^-15)
            assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -14)).all()), (likely, n)


@pytest.mark.parametrize("Dh,G", [(64, 1), (128, 2), (128, 8), (64, 16)])
@pytest.mark.parametrize("base", [-400.0, -90.0, 300.0])
def test_scores_far_from_zero(Dh, G, base):
    """All scores lie around `base`; they rise from tile to tile, or fall."""
    from flashsvd_b200 import kv8, ops
    from tests import kv8_reference as ref

    B, S = 2, 700
    gen = torch.Generator().manual_seed(Dh + G)
    for slope in (0.0, 1.0, -1.0):
        k = torch.zeros(B, S, 1, Dh)
        k[..., 0] = 1.0
        k[..., 1] = slope * (torch.arange(S) // 128 * 8)[None, :, None]   # (steps of 8: exact codes)
        k[..., 2] = torch.randint(-15, 16, (B, S, 1), generator=gen).float()
        v = torch.randn(B, S, 1, Dh, generator=gen)
        q = torch.zeros(B, G, Dh)
        q[:, :, 0], q[:, :, 1], q[:, :, 2] = base, 1.0, 0.125
        q = q.to(torch.bfloat16)
        cache = kv8.KV8Cache.empty(B, S, 1, Dh, block=32, device=DEV)
        ws = ops.make_kv8_workspace(B, G, 1, Dh, S, DEV)
        ops.kv8_append(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws)
        kk, vv = (x.double().cpu() for x in ops.kv8_load(cache, 0, S))
        lens = torch.tensor([S, 130], dtype=torch.int32)
        got = ops.flash_decode_kv8(q.to(DEV), cache, lens.to(DEV), ws, scale=1.0).double().cpu()
        want = ref.attend(q, kk, vv, lens.tolist(), 1.0)
        # (scores to 2^-22 of `base` and more: weights to 450 * 2^-22 = 2^-13)
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -12 * float(vv.abs().max())).all()), slope
