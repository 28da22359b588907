"""Stretched rotary frequencies whose factor on cos and sin is no 32-bit number: rotated keys fall on the same side of every
rounding border as in exact arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("Dh,block,inter,L", [(128, 64, False, 6000), (64, 32, True, 9001), (128, 128, True, 1)])
def test_codes_of_keys_under_a_64_bit_factor(Dh, block, inter, L):
    """Bit for bit: 64-bit rotation, rounded to 32 bits and to bf16, largest magnitude of a block, e4m3 codes.  (A product
    of 64-bit numbers is off by 2^-52: of 10^7 keys one in 2^5 runs would be rounded to another 32-bit number, and one in 2^16
    of those to another bf16 number.  With a 32-bit factor several of them are.)"""
    from flashsvd_b200 import kv8, ops

    B, Hk = (1, 8) if L > 1 else (2000, 8)
    rot = kv8.rotary(Dh, scaling="yarn", factor=32.0, trained_len=4096, interleaved=inter, device=DEV)
    assert float(torch.tensor(rot.scale, dtype=torch.float32)) != rot.scale
    gen = torch.Generator(device=DEV).manual_seed(Dh + L)
    for seed in range(4):
        k = torch.randn(B, L, Hk, Dh, device=DEV, generator=gen).to(torch.bfloat16)
        starts = torch.randint(0, 20, (B,), device=DEV, generator=gen).int() * block
        S = L + 20 * block
        cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
        ws = ops.make_kv8_workspace(B, Hk, Hk, Dh, S, DEV)
        ops.kv8_append(k, k, cache, starts, ws, rotary=rot)
        pos = starts.long()[:, None] + torch.arange(L, device=DEV)
        ang = pos.double()[..., None, None] * rot.inv_freq
        c, s = rot.scale * torch.cos(ang), rot.scale * torch.sin(ang)
        x = k.double()
        a, b = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :Dh // 2], x[..., Dh // 2:])
        y = torch.stack([a * c - b * s, b * c + a * s], -1)
        y = (y.flatten(-2) if inter else y.transpose(-1, -2).flatten(-2)).float().to(torch.bfloat16).float().transpose(1, 2)
        pad = torch.zeros(B, Hk, -(-L // block) * block, Dh, device=DEV)
        pad[:, :, :L] = y
        top = pad.view(B, Hk, -1, block * Dh).abs().amax(-1)
        m, e = torch.frexp(top)   # the smallest power of two with top <= 448 times it (448 = 0.875 * 2^9)
        scale = torch.ldexp(torch.ones_like(top), torch.where(m > 0.875, e - 8, e - 9).clamp_min(-60).float())
        want = (y / scale.repeat_interleave(block, 2)[:, :, :L, None]).to(torch.float8_e4m3fn).float()
        at = pos[:, None, :, None].expand(B, Hk, L, Dh)
        got = cache.k.view(torch.uint8).gather(2, at).view(torch.float8_e4m3fn).float()
        assert torch.equal(got, want)
