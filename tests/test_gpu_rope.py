"""`rope_qk` against the rotation in 64 bits.

Tolerance: cosine and sine are rounded once (half a step, 2^-24), each product and the sum once more: 4 * 2^-24 of
|a c| + |b s| covers them; a bf16 output adds its own half step, 2^-8 of the value."""
import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _freqs(R, stretch=1.0):
    return 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R) / stretch


def _bound(x, pos, f, inter, scale, want, dtype):
    mag = ref.rotate(x.double().abs(), pos * 0, f, inter, 1.0)   # |a|, |b| at every place
    R = 2 * f.numel()
    i = torch.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if inter else (i, i + R // 2)
    both = (mag[..., a] + mag[..., b]) * abs(scale)
    bound = torch.zeros_like(mag)
    bound[..., a] = both * 4 * 2.0 ** -24
    bound[..., b] = both * 4 * 2.0 ** -24
    return bound + (want.abs() * 2.0 ** -8 if dtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,Hk,Dh,R", [(1, 32, 32, 128, 128), (1, 1, 1, 16, 2), (17, 6, 2, 64, 48), (33, 5, 5, 80, 20),
                                         (3, 40, 8, 256, 256), (50, 4, 1, 128, 96), (16, 64, 8, 128, 64), (2, 3, 1, 48, 46)])
def test_rope_qk(dtype, inter, T, H, Hk, Dh, R):
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(T * 1000 + Dh)
    q, k = torch.randn(T, H, Dh, generator=gen).to(dtype), torch.randn(T, Hk, Dh, generator=gen).to(dtype)
    pos = torch.randint(0, 200000, (T,), generator=gen, dtype=torch.int32)
    pos[0] = 0
    f, scale = _freqs(R, 1.7), 1.25
    want_q, want_k = ref.rotate(q, pos, f, inter, scale), ref.rotate(k, pos, f, inter, scale)
    packed = torch.cat([q, k, q[:, :1]], 1).to(DEV)   # strided tokens
    for qq, kk in ((q.to(DEV), k.to(DEV)), (packed[:, :H], packed[:, H:H + Hk])):
        got_q, got_k = ops.rope_qk(qq, kk, pos.to(DEV), f.to(DEV), interleaved=inter, scale=scale)
        for got, want, x in ((got_q, want_q, q), (got_k, want_k, k)):
            assert bool(((got.double().cpu() - want).abs() <= _bound(x, pos, f, inter, scale, want, dtype)).all())
            assert torch.equal(got[..., R:].cpu(), x[..., R:])
    # without k, and in place
    only, none = ops.rope_qk(q.to(DEV), None, pos.to(DEV), f.to(DEV), interleaved=inter, scale=scale)
    assert none is None and torch.equal(only, got_q)
    qi, ki = q.to(DEV), k.to(DEV)
    ops.rope_qk(qi, ki, pos.to(DEV), f.to(DEV), interleaved=inter, scale=scale, q_out=qi, k_out=ki)
    assert torch.equal(qi, got_q) and torch.equal(ki, got_k)


def test_rope_far_positions_keep_their_phase():
    from flashsvd_b200 import ops

    f = _freqs(128)
    pos = torch.tensor([131071, 1 << 20, (1 << 31) - 1, -7], dtype=torch.int32)
    q = torch.randn(4, 2, 128, generator=torch.Generator().manual_seed(1))
    got, _ = ops.rope_qk(q.to(DEV), None, pos.to(DEV), f.to(DEV))
    want = ref.rotate(q, pos, f)
    # (2^31 positions: the angle itself is good to 2^31 * 2^-53 of a radian)
    assert bool(((got.double().cpu() - want).abs() <= _bound(q, pos, f, False, 1.0, want, torch.float32) + 2.0 ** -20 * q.abs()).all())


def test_rope_no_tokens_and_infinities():
    from flashsvd_b200 import ops

    f = _freqs(64).to(DEV)
    empty = torch.empty(0, 4, 64, device=DEV)
    a, b = ops.rope_qk(empty, empty, torch.empty(0, dtype=torch.int32, device=DEV), f)
    assert a.shape == b.shape == (0, 4, 64)
    x = torch.zeros(1, 1, 96, device=DEV)
    x[..., 80] = float("inf")
    got, _ = ops.rope_qk(x, None, torch.tensor([5], dtype=torch.int32, device=DEV), f)
    assert torch.equal(got, x)   # a dimension that is not rotated


def test_rope_in_a_graph_and_on_a_side_stream():
    from flashsvd_b200 import ops

    f = _freqs(64).to(DEV)
    q = torch.randn(5, 8, 64, device=DEV).to(torch.bfloat16)
    pos = torch.arange(5, dtype=torch.int32, device=DEV)
    want, _ = ops.rope_qk(q, None, pos, f)
    out, side = torch.empty_like(q), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got, _ = ops.rope_qk(q, None, pos, f)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rope_qk(q, None, pos, f, q_out=out)
    pos.add_(3)
    graph.replay()
    assert torch.equal(out, ops.rope_qk(q, None, pos, f)[0])
