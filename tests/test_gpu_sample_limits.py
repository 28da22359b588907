"""`sample` at the limits of its variants: rows that just fit a CTA's shared memory and rows that just do not, the largest
vocabulary, the calls it refuses.

Shares: weights are rounded to 2^-38 or finer and the share once to fp32: 2^-24 of the value and 2^-30."""
import pytest
import torch

from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _check(x, u, T, k, p, m, tokens, probs, rows):
    for b in rows:
        want, share = ref.sample_row(x[b].double(), float(u[b]), float(torch.tensor(T)), k, float(torch.tensor(p)), float(torch.tensor(m)))
        assert int(tokens[b]) == want, (b, int(tokens[b]), want)
        assert abs(float(probs[b]) - share) <= share * 2.0 ** -24 + 2.0 ** -30


@pytest.mark.parametrize("dtype,B,V", [(torch.float32, 128, V) for V in (36092, 36093, 36094, 36500, 36861, 36862)]
                         + [(torch.bfloat16, 128, V) for V in (72183, 72190, 72500, 73000, 73721)]
                         + [(torch.float32, 37, V) for V in (144381, 144382, 145900, 147453, 147454)]
                         + [(torch.float32, 1, V) for V in (288765, 288766, 290000, 294909, 294910)]
                         + [(torch.float32, 8, 291003), (torch.bfloat16, 37, 288800), (torch.bfloat16, 1, 577600), (torch.bfloat16, 8, 585003)])
def test_rows_at_the_limit_of_shared_memory(dtype, B, V):
    from flashsvd_b200 import ops

    gen = torch.Generator().manual_seed(B + V)
    x = (4 * torch.randn(B, V, generator=gen)).to(dtype)
    u = torch.rand(B, generator=gen)
    for T, k, p, m in ((0.8, 0, 0.9, 0.0), (1.2, 50, 0.9, 0.02)):
        tokens, probs = ops.sample(x.to(DEV), u.to(DEV), temperature=T, top_k=k, top_p=p, min_p=m)
        _check(x, u, T, k, p, m, tokens, probs, {0, B - 1})
    # a row that begins off a 16-byte boundary has up to 15 bytes more
    wide = torch.zeros(B, V + 5, dtype=dtype, device=DEV)
    wide[:, 3:V + 3] = x.to(DEV)
    again, _ = ops.sample(wide[:, 3:V + 3], u.to(DEV), temperature=1.2, top_k=50, top_p=0.9, min_p=0.02)
    assert torch.equal(again, tokens)


def test_vocabularies_beyond_the_limit_are_refused():
    from flashsvd_b200 import _lib, ops

    u = torch.zeros(1, device=DEV)
    for V in ((1 << 20) + 1, 1 << 22):
        with pytest.raises((_lib.FsvdError, ValueError)):
            ops.sample(torch.zeros(1, V, device=DEV), u)
    tokens, _ = ops.sample(torch.zeros(1, 1 << 20, device=DEV), u)
    assert int(tokens) == 0


@pytest.mark.parametrize("B,V", [(1, 1 << 20), (130, 600001), (2, 90001)])
@pytest.mark.parametrize("octaves", [33.5, 36.3, 30.7])
def test_a_border_far_down_in_the_tail(B, V, octaves):
    """One likely token in front of V - 1 equal ones at 2^-octaves of its weight, and a top-p that ends among them.

    The likely token's weight is one exactly; the tail's weights, all alike, are good to 2^-39, which over V of them is far
    less than one; the sums' roundings (2^-50 of the mass) are 2^-12 of a tail weight: the number kept, and with it the place
    of a draw in the tail, is off by one at most."""
    import math

    from flashsvd_b200 import ops

    x = torch.full((V,), -octaves * math.log(2.0))
    x[5] = 0.0
    w = math.exp(float(x[0].double()))
    tail = (V - 1) * w
    p = float(torch.tensor(1.0 - 0.6 * tail / (1.0 + tail), dtype=torch.float32))
    if p * (1.0 + tail) - 1.0 < 10 * w:   # (a 32-bit p has no value between the token's share and one)
        pytest.skip("no 32-bit top-p ends in this tail")
    kept = math.floor((p * (1.0 + tail) - 1.0) / w) + 1   # of the tail: those whose preceding mass is at most p of all
    z = 1.0 + kept * w
    u = torch.tensor([1.0 - 2.0 ** -24 * (1 + b % 3) for b in range(B)])
    tokens, probs = ops.sample(x[None].expand(B, V).contiguous().to(DEV), u.to(DEV), top_p=p)
    for b in range(B):
        # (five tail tokens lie in front of the likely one)
        place = float(u[b].double()) * z
        want = 5 if place < 1.0 + 5 * w else 6 + math.floor((place - 1.0) / w) - 5
        assert abs(int(tokens[b]) - want) <= 1, (int(tokens[b]), want)
        assert abs(float(probs[b]) - (w if want != 5 else 1.0) / z) <= 2.0 ** -24 * (w if want != 5 else 1.0)


@pytest.mark.parametrize("B,n1,n2", [(1, 100000, 900000), (40, 70000, 200000), (130, 30000, 50000)])
@pytest.mark.parametrize("first", [31.02, 31.5, 31.97, 28.3])
def test_a_border_behind_the_last_counted_octave(B, n1, n2, first):
    """One likely token, n1 at 2^-first of its weight and n2 at 2^-34, among which the top-p ends: what lies in front of them
    counts in full.

    The likely token's weight is one exactly; 10^6 tail weights, each good to 2^-39 of itself and 2^-34 of itself in the
    histogram, move the number kept by less than 10^6 2^-34 2^3 (a weight of the first group is at most 2^6 of the second
    group's, and the roundings of equal weights add up): 2^-8, and sums of 64-bit numbers by 2^-50 of the mass, 2^-16 of a
    weight.  One either way."""
    import math

    from flashsvd_b200 import ops

    V = 1 + n1 + n2
    x = torch.empty(V)
    x[0], x[1:1 + n1], x[1 + n1:] = 0.0, -first * math.log(2.0), -34.0 * math.log(2.0)
    w1, w2 = math.exp(float(x[1].double())), math.exp(float(x[-1].double()))
    total = 1.0 + n1 * w1 + n2 * w2
    p = float(torch.tensor(1.0 - 0.5 * n2 * w2 / total, dtype=torch.float32))
    kept = math.floor((p * total - 1.0 - n1 * w1) / w2) + 1
    assert 100 < kept < n2 - 100
    z = 1.0 + n1 * w1 + kept * w2
    u = torch.tensor([1.0 - 2.0 ** -24 * (1 + b % 2) for b in range(B)])
    tokens, probs = ops.sample(x[None].expand(B, V).contiguous().to(DEV), u.to(DEV), top_p=p)
    for b in range(B):
        place = float(u[b].double()) * z - 1.0
        want = 0 if place < 0 else 1 + math.floor(place / w1) if place < n1 * w1 else 1 + n1 + math.floor((place - n1 * w1) / w2)
        assert abs(int(tokens[b]) - want) <= 1, (int(tokens[b]), want)
    # the share of the likely token tells what is kept: z within one tail weight, rounded once
    tokens, probs = ops.sample(x[None].expand(B, V).contiguous().to(DEV), torch.zeros(B, device=DEV), top_p=p)
    assert bool((tokens == 0).all()) and bool(((probs.double() - 1.0 / z).abs() <= 2.0 ** -24).all())


def test_temperatures_next_to_zero():
    """Positive ones below 2^-64 count as 2^-64: the largest logits share everything, zeros among them."""
    from flashsvd_b200 import ops

    V = 1000
    x = -torch.rand(4, V, generator=torch.Generator().manual_seed(1)) - 0.5
    x[0, 17], x[1, 3], x[1, 900], x[2, 5], x[3] = 0.0, -0.0, 0.0, 2.0, 0.0
    u = torch.full((4,), 0.75)
    for T in (1e-45, 1e-42, 1e-39, 1e-37, 1e-31, 1e-20):
        for T_all in (T, torch.full((4,), T, device=DEV)):
            out, share = torch.full((4,), -7, dtype=torch.int32, device=DEV), torch.full((4,), -7.0, device=DEV)
            ops.sample(x.to(DEV), u.to(DEV), temperature=T_all, out=out, probs_out=share)
            assert out.tolist() == [17, 900, 5, 750] and share.tolist()[:3] == [1.0, 0.5, 1.0]
            ops.sample(x.to(DEV), u.to(DEV), temperature=T_all, top_p=0.5, top_k=9, min_p=0.5, out=out, probs_out=share)
            assert out.tolist()[:3] == [17, 900, 5]
