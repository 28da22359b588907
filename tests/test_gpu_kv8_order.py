"""Attention over the 8-bit cache where a CTA's first pair of (sequence, kv head) has a single tile and another pair
follows it: the factors of the second pair's queries have to be written before any warp reads them.

Every pair has queries of a magnitude of its own (its keys take the reciprocal, so that scores stay small) and every call
another scale: a factor of another pair, or of a call before, is never the right one.  Tolerance: half a bf16 step and
2^-14 of the largest value, as for attention at large (scores stay below 64, as asserted)."""
import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("G", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("Dh,lens", [(64, [100, 128, 1, 33]), (128, [128, 17, 96, 64]), (128, [257, 128, 130, 384])])
def test_query_factors_of_the_second_pair(G, Dh, lens):
    from flashsvd_b200 import kv8, ops

    B, Hk, S = 32, 32, max(lens)
    gen = torch.Generator().manual_seed(G * 1000 + Dh + S)
    e = torch.randint(-12, 13, (B, Hk), generator=gen)
    e = torch.where((torch.arange(B * Hk).view(B, Hk) & 1) == 1, e + 30, e)   # neighbours are always far apart
    gain = torch.ldexp(torch.ones(B, Hk), e)
    k = torch.randn(B, S, Hk, Dh, generator=gen) / gain[:, None, :, None]
    v = torch.randn(B, S, Hk, Dh, generator=gen)
    q = 2 * torch.randn(B, Hk, G, Dh, generator=gen) * gain[:, :, None, None]
    q = q.reshape(B, Hk * G, Dh).to(torch.bfloat16)
    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=64, device=DEV)
    ws = ops.make_kv8_workspace(B, Hk * G, Hk, Dh, S, DEV)
    ops.kv8_append(k.to(torch.bfloat16).to(DEV), v.to(torch.bfloat16).to(DEV), cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws)
    kk, vv = (x.double().cpu() for x in ops.kv8_load(cache, 0, S))
    n = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
    for scale in (Dh ** -0.5, 0.6 * Dh ** -0.5, 0.03 * Dh ** -0.5, 2 * Dh ** -0.5):
        assert float((q.double().view(B, Hk, G, Dh) @ kk.transpose(2, 3)).abs().max()) * scale < 64
        want = ref.attend(q, kk, vv, n.tolist(), scale)
        got = ops.flash_decode_kv8(q.to(DEV), cache, n.to(DEV), ws, scale=scale).double().cpu()
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * float(vv.abs().max())).all())
    assert ws.status() == 0
