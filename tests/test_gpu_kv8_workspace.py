"""One workspace serves calls of different sizes, one after the other: what a call leaves in it means nothing to the next."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(B, H, Hk, Dh, S, seed):
    from flashsvd_b200 import kv8, ops

    gen = torch.Generator().manual_seed(seed)
    cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=32, device=DEV)
    k, v = (torch.randn(B, S, Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    ops.kv8_append(k, v, cache, lens, ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV))
    lens.fill_(S)
    q = torch.randn(B, H, Dh, generator=gen).to(torch.bfloat16).to(DEV)
    return q, cache, lens


def test_calls_of_other_sizes_in_between():
    from flashsvd_b200 import ops

    sizes = [(40, 24, 12, 64, 1500), (2, 16, 1, 64, 900), (1, 2, 2, 128, 5000), (70, 8, 8, 64, 700), (3, 32, 4, 128, 1030)]
    cases = [_case(*s, seed=i) for i, s in enumerate(sizes)]
    room = max((ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV) for B, H, Hk, Dh, S in sizes), key=lambda w: w.nbytes)
    alone = [ops.flash_decode_kv8(q, c, n, ops.make_kv8_workspace(q.shape[0], q.shape[1], c.k.shape[1], q.shape[2], c.max_len, DEV))
             for q, c, n in cases]
    for i in (0, 1, 0, 2, 3, 1, 3, 4, 0, 4, 2, 0, 1, 3):
        q, cache, lens = cases[i]
        out = torch.full_like(q, float("nan"))
        ops.flash_decode_kv8(q, cache, lens, room, out=out)
        assert torch.equal(out, alone[i]), i
    assert room.status() == 0


def test_the_counters_place_does_not_depend_on_the_sizes():
    """As many heads per kv head and the same head dimension: the same scratch, whatever batch and length."""
    from flashsvd_b200 import ops

    a, b = (ops.make_kv8_workspace(B, 2 * Hk, Hk, 64, S, DEV).nbytes for B, Hk, S in ((1, 1, 16), (500, 40, 4096)))
    assert a == b
