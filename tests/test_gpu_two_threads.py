"""Two host threads call the same operators at different sizes at once, each on a stream and with tensors of its own: no call
fails, and every result is the one of a call by itself."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _together(works):
    errors = []

    def run(work):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                work()
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # (reported by the main thread)
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=run, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


@pytest.mark.parametrize("lengths", [(64, 40), (50, 45)])
def test_appends_of_two_lengths(lengths):
    """Both want more shared memory for their tables than a kernel has by itself, one more than the other."""
    from flashsvd_b200 import kv8, ops

    H, Hk, Dh, S = 8, 4, 128, 256
    rot = kv8.rotary(Dh, device=DEV)
    outs = []

    def make(L):
        x = torch.randn(1, L, H + 2 * Hk, Dh, generator=torch.Generator().manual_seed(L)).to(torch.bfloat16).to(DEV)
        lens = torch.zeros(1, dtype=torch.int32, device=DEV)
        caches = [kv8.KV8Cache.empty(1, S, Hk, Dh, device=DEV) for _ in range(2)]
        ws = ops.make_kv8_workspace(1, H, Hk, Dh, S, DEV)

        def call(cache):
            return ops.kv8_append(x[:, :, H:H + Hk], x[:, :, H + Hk:], cache, lens, ws, q=x[:, :, :H], rotary=rot)

        want = call(caches[0])
        outs.append((want, caches, []))

        def work(mine=outs[-1][2]):
            for _ in range(1500):
                mine[:] = [call(caches[1])]

        return work

    _together([make(L) for L in lengths])
    for want, (a, b), (got,) in outs:
        assert torch.equal(got, want)
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))


def test_draws_from_two_vocabularies():
    from flashsvd_b200 import ops

    outs = []

    def make(V):
        gen = torch.Generator().manual_seed(V)
        x, u = torch.randn(148, V, generator=gen).to(DEV), torch.rand(148, generator=gen).to(DEV)
        want = ops.sample(x, u, top_p=0.9)
        mine = []
        outs.append((want, mine))

        def work():
            for _ in range(1500):
                mine[:] = [ops.sample(x, u, top_p=0.9)]

        return work

    _together([make(V) for V in (9000, 6000)])
    for want, (got,) in outs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
