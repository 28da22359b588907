"""The cache class of the 8-bit cache: where it takes the length from, what it keeps for later calls, what it refuses."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, Hk, Dh = 4, 2, 64


def _cache(layers=1, S=24, batch=3, block=16):
    from flashsvd_b200 import runtime as R

    return R.FlashSVDV15KV8Cache(SimpleNamespace(num_hidden_layers=layers, rope_theta=10000.0), max_batch_size=batch, max_cache_len=S,
                                 device=DEV, block=block)


def _qkv(B, L, seed):
    x = torch.randn(B, L, H + 2 * Hk, Dh, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)
    return x[:, :, :H].contiguous(), x[:, :, H:H + Hk].contiguous(), x[:, :, H + Hk:].contiguous()


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_writing_in_front_of_the_end_cuts_the_sequence(device):
    """The same steps with positions that the host knows and positions that only the device knows."""
    cache = _cache()
    q, k, v = _qkv(2, 10, 1)
    cache.append(k, v, 0, query_states=q)
    assert cache.get_seq_length() == 10
    q, k, v = _qkv(2, 1, 2)
    cache.decode_step(q, k, v, 0, cache_position=torch.tensor([5], device=device))
    assert cache.get_seq_length() == 6
    # a step that does not advance is no part of the sequence
    cache.decode_step(q, k, v, 0, cache_position=torch.tensor([20], device=device), advance=False)
    assert cache.get_seq_length() == 6
    assert cache.get_mask_sizes(1) == ((7 if device == "cpu" else 24), 0)   # (no wait for the device: the cache's length)
    # the next one without a position goes behind the cut
    sl, start, _ = cache.append(k, v, 0, query_states=q)
    assert sl.tolist() == [6, 6] and start == 6 and cache.get_seq_length() == 7
    cache.decode_step(q, k, v, 0, cache_position=torch.tensor([7, 3], device=device))
    assert cache.get_seq_length() == 8
    cache.reset()
    assert cache.get_seq_length() == 0


def test_the_length_follows_a_replayed_step():
    cache = _cache()
    q, k, v = _qkv(2, 4, 3)
    cache.append(k, v, 0, query_states=q)
    q, k, v = _qkv(2, 1, 4)
    pos = torch.tensor([4], device=DEV)
    cache.decode_step(q, k, v, 0, cache_position=pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.decode_step(q, k, v, 0, cache_position=pos)
        with pytest.raises(RuntimeError, match="cache_position"):
            cache.get_seq_length()
        assert cache.get_mask_sizes(1) == (24, 0)
    for t in (5, 6, 9):
        pos.fill_(t)
        graph.replay()
        assert cache.get_seq_length() == t + 1
    pos.fill_(1000)   # dropped
    graph.replay()
    assert cache.get_seq_length() == 24
    cache.append(k, v, 0, query_states=q, cache_position=10)
    assert cache.get_seq_length() == 11


def _rotary_module():
    from flashsvd_b200 import modules as M

    return M.LlamaRotaryEmbedding(Dh, base=777.0)


def test_first_uses_cannot_be_captured():
    """A capture computes nothing, and what a replay makes it makes again every time: the call says so and keeps nothing."""
    rope, cache = _rotary_module(), _cache()
    q, k, v = _qkv(2, 1, 5)
    pos = torch.zeros(2, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: rope.rotate(q[:, 0], k[:, 0], pos), lambda: cache.rotary(Dh, torch.device(DEV)),
                     lambda: cache.append(k, v, 0, query_states=q, cache_position=pos)):
            with pytest.raises(RuntimeError, match="before the capture"):
                call()
        pos.add_(1)
    graph.replay()
    cache.append(k, v, 0, query_states=q, cache_position=pos)
    want = rope.rotate(q[:, 0], k[:, 0], pos)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        rope.rotate(q[:, 0], k[:, 0], pos)
        cache.append(k, v, 0, query_states=q, cache_position=pos)
    assert torch.equal(rope.rotate(q[:, 0], k[:, 0], pos)[0], want[0])


def test_first_uses_on_a_busy_stream_serve_other_streams():
    """What the first call makes is there when a second call on another stream asks for it."""
    q, k, v = _qkv(3, 4, 6)
    pos = torch.arange(12, device=DEV).view(3, 4)[:, 0].contiguous()
    good_rope, good = _rotary_module(), _cache()
    want = good_rope.rotate(q[:, 0], k[:, 0], pos)
    _, _, wq = good.append(k, v, 0, query_states=q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    # (memory that the allocator hands out again on that stream holds other numbers)
    with torch.cuda.stream(side):
        torch.full((1 << 20,), 3.0, dtype=torch.float64, device=DEV)
        torch.cuda.synchronize()
        rope, cache = _rotary_module(), _cache()
        torch.cuda._sleep(400_000_000)
        rope.rotate(q[:, 0], k[:, 0], pos)
        cache.append(k, v, 0, query_states=q)
    got = rope.rotate(q[:, 0], k[:, 0], pos)
    _, _, gq = cache.append(k, v, 0, query_states=q, cache_position=0)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and torch.equal(gq, wq)


def test_update_gives_zeros_behind_a_shorter_sequence():
    """What a cut or forgotten sequence left there, NaN among it, is not handed out."""
    cache = _cache()
    _, k, v = _qkv(3, 12, 7)
    k[2, 9, 0, 3] = float("nan")
    cache.append(k, v, 0, rotate=False)
    cache.reset()
    _, k, v = _qkv(3, 1, 8)
    kk, vv = cache.update(k.transpose(1, 2), v.transpose(1, 2), 0, {"cache_position": torch.tensor([10, 0, 4])})
    assert kk.shape == vv.shape == (3, Hk, 11, Dh)
    for b, n in enumerate((11, 1, 5)):
        assert bool(kk[b, :, n - 1].any()) and not bool(kk[b, :, n:].any()) and not bool(vv[b, :, n:].any())


def test_decode_step_refuses_several_tokens():
    """It attends with the first query alone: the others would be lost.  Nothing is appended."""
    cache = _cache()
    q, k, v = _qkv(2, 3, 9)
    cache.append(k, v, 0, query_states=q)
    before = cache.layers8[0].k.view(torch.uint8).clone()
    for bad in (q, q[:, 0], q[:, :0]):
        with pytest.raises(ValueError, match="one token"):
            cache.decode_step(bad, k, v, 0)
    with pytest.raises(ValueError):
        cache.decode_step(q[:, :1], k, v, 0)   # (a query for some of the tokens)
    assert cache.get_seq_length() == 3 and torch.equal(cache.layers8[0].k.view(torch.uint8), before)


def test_a_dropped_token_is_reported():
    cache = _cache(layers=2)
    q, k, v = _qkv(2, 1, 10)
    for layer in (0, 1):
        cache.decode_step(q, k, v, layer, cache_position=torch.tensor([23], device=DEV))
    assert cache.status() == 0
    before = [c.k.view(torch.uint8).clone() for c in cache.layers8]
    cache.decode_step(q, k, v, 1, cache_position=torch.tensor([24, 3], device=DEV))
    with pytest.raises(IndexError):
        cache.status()
    assert torch.equal(cache.layers8[1].k.view(torch.uint8)[0], before[1][0])
    cache.clear_status()
    assert cache.status() == 0


def test_queries_behind_the_largest_position_are_rotated():
    """A length next to 2^31: the tokens are dropped, their queries turn by the positions that they would have had.

    Half a bf16 step, and angles of 2^31 radians to 2^-20 (a 64-bit angle has 2^-21 there)."""
    from flashsvd_b200 import kv8, ops
    from tests import kv8_reference as ref

    rot = kv8.rotary(Dh, device=DEV)
    for L in (3, 40):
        cache = kv8.KV8Cache.empty(2, 24, Hk, Dh, block=16, device=DEV)
        ws = ops.make_kv8_workspace(2, H, Hk, Dh, 24, DEV)
        q, k, v = _qkv(2, L, L)
        starts = torch.tensor([2 ** 31 - 1, 2 ** 31 - 20], dtype=torch.int32, device=DEV)
        got = ops.kv8_append(k, v, cache, starts, ws, q=q, rotary=rot).double().cpu()
        pos = starts.cpu().long()[:, None] + torch.arange(L)
        want = ref.rotate(q.cpu(), pos, rot.inv_freq.cpu())
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -19 * float(q.abs().max())).all())
        assert ws.raw_status() != 0 and not bool(cache.k.view(torch.uint8).any())
