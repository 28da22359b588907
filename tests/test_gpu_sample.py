"""`sample` against the definition, token for token.

Shares: weights are rounded to 2^-38 or finer and the share once to fp32: 2^-24 of the value and 2^-30."""
import math

import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(x, u, T, k, p, m, tokens, probs):
    for b in range(x.shape[0]):
        at = lambda s: float(s[b]) if torch.is_tensor(s) else float(torch.tensor(s, dtype=torch.float32))   # noqa: E731
        want, share = ref.sample_row(x[b].double(), float(u[b]), at(T), int(k[b]) if torch.is_tensor(k) else k, at(p), at(m))
        assert int(tokens[b]) == want, (b, int(tokens[b]), want)
        assert abs(float(probs[b]) - share) <= share * 2.0 ** -24 + 2.0 ** -30


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 31, 257, 1000, 4097, 32000, 70001])
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 40, 1.0, 0.0), (0.9, 0, 1.0, 0.1), (1.0, 50, 0.8, 0.05),
                                     (0.0, 0, 0.9, 0.0), (2.0, 1, 1.0, 0.0), (5.0, 3, 0.0, 0.0), (1.0, 10 ** 6, 0.999, 1.0)])
def test_sample(dtype, V, T, k, p, m):
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(V + int(100 * T) + k)
    B = 6
    x = (3 * torch.randn(B, V, generator=gen)).to(dtype)
    u = torch.rand(B, generator=gen)
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    tokens, probs = ops.sample(x.to(DEV), u.to(DEV), temperature=T, top_k=k, top_p=p, min_p=m)
    _check(x, u, T, k, p, m, tokens.cpu(), probs.cpu())
    # strided rows, settings per row, given outputs
    wide = torch.full((B, V + 24), 99.0, dtype=dtype)
    wide[:, :V] = x
    full = lambda s, dt: torch.full((B,), s, dtype=dt, device=DEV)   # noqa: E731
    out, share = torch.empty(B, dtype=torch.int32, device=DEV), torch.empty(B, device=DEV)
    ops.sample(wide.to(DEV)[:, :V], u.to(DEV), temperature=full(T, torch.float32), top_k=full(k, torch.int32),
               top_p=full(p, torch.float32), min_p=full(m, torch.float32), out=out, probs_out=share)
    assert torch.equal(out, tokens) and torch.equal(share, probs)


def test_equal_logits_go_by_index():
    from flashsvd_b200 import ops

    V = 5000
    x = torch.full((8, V), -3.0)
    x[1, 100:200], x[2, 4000:] = 1.0, 1.0
    x[3] = torch.arange(V) % 7
    x[4, ::2] = 0.0
    x[4, 1::2] = -0.0
    x[5, 17] = 2.0
    x[6, 4999] = 2.0
    u = torch.tensor([0.5, 0.25, 0.999, 0.5, 0.75, 0.9, 0.3, 0.1])
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 150, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 130, 0.5, 0.0), (0.0, 0, 1.0, 0.0),
                       (1.0, 37, 0.9, 0.99), (1e-6, 0, 0.9, 0.0), (1e6, 999, 0.3, 0.0)):
        tokens, probs = ops.sample(x.to(DEV), u.to(DEV), temperature=T, top_k=k, top_p=p, min_p=m)
        _check(x, u, T, k, p, m, tokens.cpu(), probs.cpu())


def test_infinities_and_nan():
    from flashsvd_b200 import ops

    V = 300
    x = torch.randn(7, V, generator=torch.Generator().manual_seed(2))
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 5:] = -math.inf
    x[3, 9], x[3, 200] = math.inf, math.inf
    x[4, ::3] = math.nan
    x[5] = torch.finfo(torch.float32).min
    x[6, 1:] = torch.finfo(torch.float32).min
    u = torch.tensor([0.5, 0.5, 0.9, 0.7, 0.5, 0.4, 0.99])
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.5, 20, 0.9, 0.1), (0.0, 0, 1.0, 0.0), (math.inf, 7, 1.0, 0.0)):
        tokens, probs = ops.sample(x.to(DEV), u.to(DEV), temperature=T, top_k=k, top_p=p, min_p=m)
        _check(x, u, T, k, p, m, tokens.cpu(), probs.cpu())


def test_uniforms_outside_their_range_and_no_rows():
    from flashsvd_b200 import ops

    x = torch.randn(4, 1000, generator=torch.Generator().manual_seed(3))
    bad = torch.tensor([1.0, -1.0, math.nan, math.inf])
    near = torch.tensor([1.0 - 2.0 ** -24, 0.0, 0.0, 1.0 - 2.0 ** -24])
    a, _ = ops.sample(x.to(DEV), bad.to(DEV), top_p=0.9)
    b, _ = ops.sample(x.to(DEV), near.to(DEV), top_p=0.9)
    assert torch.equal(a, b)
    t, p = ops.sample(x[:0].to(DEV), bad[:0].to(DEV))
    assert t.shape == p.shape == (0,)


def test_frequencies_follow_the_weights():
    """20000 draws over a few tokens: every count within 5 standard deviations of its share."""
    from flashsvd_b200 import ops

    x = torch.tensor([[2.0, 0.0, 1.0, -1.0, 1.5]])
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(4))
    tokens, _ = ops.sample(x.expand(n, 5).contiguous().to(DEV), u.to(DEV), temperature=0.8, top_k=4)
    w = torch.exp(x[0].double() / 0.8)
    w[3] = 0.0
    w = w / w.sum()
    count = torch.bincount(tokens.long().cpu(), minlength=5).double()
    assert bool(((count - n * w).abs() <= 5 * torch.sqrt(n * w * (1 - w))).all())


def test_sample_in_a_graph():
    from flashsvd_b200 import ops

    x = torch.randn(3, 32000, device=DEV)
    u = torch.rand(3, device=DEV)
    out = torch.empty(3, dtype=torch.int32, device=DEV)
    ops.sample(x, u, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample(x, u, top_p=0.9, top_k=100, out=out)
    for _ in range(3):
        x.copy_(torch.randn(3, 32000, device=DEV))
        u.copy_(torch.rand(3, device=DEV))
        graph.replay()
        assert torch.equal(out, ops.sample(x, u, top_p=0.9, top_k=100)[0])


@pytest.mark.parametrize("dtype,B,V", [(torch.float32, 1, 300001), (torch.float32, 2, 1 << 20), (torch.bfloat16, 1, 1 << 20),
                                       (torch.float32, 140, 50001), (torch.bfloat16, 149, 80003), (torch.float32, 75, 61007)])
def test_rows_longer_than_shared_memory_and_many_rows(dtype, B, V):
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(B + V)
    x = (4 * torch.randn(B, V, generator=gen)).to(dtype)
    u = torch.rand(B, generator=gen)
    rows = [0] if B == 1 else [0, 1] if B == 2 else [0, B // 2, B - 1]
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.8, 0, 0.9, 0.0), (1.2, 50, 0.9, 0.02), (2.5, V // 3, 0.99, 0.0), (0.0, 0, 1.0, 0.0),
                       (1.0, 0, 1.0, 0.1)):
        tokens, probs = ops.sample(x.to(DEV), u.to(DEV), temperature=T, top_k=k, top_p=p, min_p=m)
        _check(x[rows], u[rows], T, k, p, m, tokens[rows], probs[rows])


@pytest.mark.parametrize("B,V", [(140, 262144), (1, (1 << 20) - 1), (148, 160001)])
def test_masses_of_many_equal_logits(B, V):
    """More than half the row in one bin of the histogram and the rest in the next ones: its sums hold them all."""
    from flashsvd_b200 import ops

    # (32 log2(e) x = -64.49 and -64.51 sit at the two ends of the bins -64 and -65: residuals of either sign, all bits set)
    step = math.log(2.0) / 32
    for off in (64.49, 64.499, 64.02, 64.51):
        x = torch.full((V,), -off * step)
        x[V * 3 // 5:] = -(off + 2.0) * step
        x[7] = 0.0
        rows = x[None].expand(B, V).contiguous()
        u = torch.linspace(0.01, 0.99, B)
        tokens, probs = ops.sample(rows.to(DEV), u.to(DEV), top_p=0.75)
        e = torch.exp(x.double())
        order = torch.argsort(e, descending=True, stable=True)
        mass = torch.cumsum(e[order], 0)
        n = int((mass - e[order] <= 0.75 * mass[-1]).sum())   # kept: those whose preceding mass is at most the share
        kept = torch.zeros(V, dtype=torch.bool)
        kept[order[:n]] = True
        run = torch.cumsum(torch.where(kept, e, 0.0), 0)
        for b in {0, B // 2, B - 1}:
            # (equal weights by the thousand: sums of 10^5 rounded terms are good to 2^-36 of themselves, which is less than
            # half a weight, so the place is off by one at most on either side)
            want = int(torch.searchsorted(run, float(u[b]) * run[-1], right=True))
            assert abs(int(tokens[b]) - want) <= 1
            assert abs(float(probs[b]) - float(e[want] / run[-1])) <= float(e[want] / run[-1]) * 2.0 ** -16
