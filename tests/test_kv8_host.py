"""CPU: what the operators around the 8-bit cache refuse, before anything is launched, and the rotary frequencies.

The C entries check sizes and pointers on the host; nothing here reaches a kernel."""
import ctypes as C
import math

import pytest
import torch

from tests import kv8_reference as ref

P = 1 << 20   # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    from flashsvd_b200 import _lib, build

    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.load()


def _cache(**kw):
    from flashsvd_b200._lib import FsvdKv8

    d = dict(k8=P, v8=P, k_scale=P, v_scale=P, B=2, Hk=4, S_max=100, Dh=64, block=32)
    d.update(kw)
    return C.byref(FsvdKv8(**d))


def _refused(lib, code, rc, text=""):
    assert rc == code, (rc, lib.fsvd_last_error_string())
    assert text in lib.fsvd_last_error_string().decode()


def test_rope_refusals(lib):
    def call(**kw):
        a = dict(q=P, qs=512, k=P, ks=512, pos=P, f=P, R=64, inter=0, scale=1.0, qo=P, ko=P, T=3, H=4, Hk=2, Dh=64, dt=0)
        a.update(kw)
        return lib.fsvd_rope_qk(*a.values(), None)

    for name in ("q", "pos", "f", "qo", "k", "ko"):
        _refused(lib, -1, call(**{name: None}))
    for kw, code in ((dict(R=0), -1), (dict(R=65), -1), (dict(R=66), -1), (dict(Dh=72), -2), (dict(Dh=272), -2), (dict(dt=2), -1),
                     (dict(T=-1), -1), (dict(H=0), -1), (dict(Hk=0), -1), (dict(q=P + 2), -3), (dict(qs=516), -3), (dict(ks=-512), -1),
                     (dict(dt=1, qs=514), -3)):
        _refused(lib, code, call(**kw))
    assert call(T=0) == 0


def test_append_refusals(lib):
    def call(cache=None, **kw):
        a = dict(k=P, v=P, bs=512, ts=256, lens=P, new=None, q=P, qb=512, qt=256, qo=P, f=P, R=64, inter=0, scale=1.0, H=4, L=2,
                 ws=P, n=4096)
        a.update(kw)
        return lib.fsvd_kv8_append(cache or _cache(), *a.values(), None)

    for name in ("k", "v", "lens", "q", "qo"):
        _refused(lib, -1, call(**{name: None}))
    _refused(lib, -1, call(f=None), "inv_freq")
    for kw, code in ((dict(R=66), -1), (dict(R=3), -1), (dict(L=-1), -1), (dict(H=0), -1), (dict(bs=-8), -1), (dict(ts=252), -3),
                     (dict(k=P + 8), -3), (dict(qt=4), -3), (dict(ws=None), -4), (dict(n=100), -4), (dict(ws=P + 4), -3)):
        _refused(lib, code, call(**kw))
    for kw, code in ((dict(Dh=96), -2), (dict(block=48), -2), (dict(k8=None), -1), (dict(k_scale=None), -1), (dict(B=0), -1),
                     (dict(S_max=0), -1), (dict(v8=P + 1), -3), (dict(S_max=(1 << 30) + 1), -2), (dict(B=1 << 12, Hk=1 << 12), -2)):
        _refused(lib, code, call(_cache(**kw)))
    assert call(L=0) == 0


def test_load_and_attention_refusals(lib):
    for start, n in ((-1, 2), (0, 101), (100, 1), (5, -1)):
        _refused(lib, -1, lib.fsvd_kv8_load(_cache(), start, n, None, 0, P, P, None))
    _refused(lib, -1, lib.fsvd_kv8_load(_cache(), 0, 1, None, 0, None, P, None))
    _refused(lib, -3, lib.fsvd_kv8_load(_cache(), 0, 1, None, 0, P, P + 8, None))
    assert lib.fsvd_kv8_load(_cache(), 100, 0, None, 0, P, P, None) == 0

    need = lib.fsvd_kv8_workspace_bytes(2, 8, 4, 64, 100)
    assert need > 0 and lib.fsvd_kv8_workspace_bytes(2, 8, 4, 96, 100) == 0 and lib.fsvd_kv8_workspace_bytes(0, 8, 4, 64, 100) == 0

    def attend(cache=None, q=P, lens=P, out=P, H=8, ws=P, n=need):
        return lib.fsvd_flash_decode_kv8(cache or _cache(), q, lens, 0, out, H, 0.0, ws, n, None)

    for kw, code in ((dict(q=None), -1), (dict(lens=None), -1), (dict(out=None), -1), (dict(H=6), -1), (dict(H=0), -1), (dict(H=68), -2),
                     (dict(q=P + 2), -3), (dict(ws=None), -4), (dict(n=need - 1), -4), (dict(ws=P + 8), -3)):
        _refused(lib, code, attend(**kw))


def test_sample_refusals(lib):
    def call(**kw):
        a = dict(x=P, stride=1000, dt=1, u=P, T=None, k=None, p=None, m=None, Ta=1.0, ka=0, pa=1.0, ma=0.0, out=P, probs=None, B=2, V=1000)
        a.update(kw)
        return lib.fsvd_sample(*a.values(), None)

    for kw, code in ((dict(x=None), -1), (dict(u=None), -1), (dict(out=None), -1), (dict(dt=2), -1), (dict(V=0), -1), (dict(B=-1), -1),
                     (dict(stride=-1), -1), (dict(V=(1 << 22) + 1), -2), (dict(Ta=math.nan), -1), (dict(pa=math.nan), -1),
                     (dict(ma=math.nan), -1)):
        _refused(lib, code, call(**kw))
    assert call(B=0) == 0


def test_tensor_arguments_are_checked_before_the_library_is_asked():
    from flashsvd_b200 import kv8, ops

    x = torch.zeros(3, 4, 64)
    with pytest.raises(ValueError):
        ops.rope_qk(x, None, torch.zeros(3, dtype=torch.int32), torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.rope_qk(x[0], None, torch.zeros(3, dtype=torch.int32), torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(2, 10), torch.zeros(2))
    with pytest.raises(ValueError):
        ops.sample(torch.zeros(10), torch.zeros(2))
    for kw in (dict(block=48), dict(head_dim=96), dict(max_len=0), {}):
        a = dict(batch=1, max_len=10, num_kv_heads=1, head_dim=64, block=16, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError):
            kv8.KV8Cache.empty(a.pop("batch"), a.pop("max_len"), a.pop("num_kv_heads"), a.pop("head_dim"), **a)


def test_rotary_frequencies():
    from flashsvd_b200 import kv8

    plain = kv8.rotary(64, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert plain.inv_freq.dtype == torch.float64 and plain.scale == 1.0
    assert torch.allclose(plain.inv_freq, want, rtol=1e-14, atol=0)
    assert torch.allclose(kv8.rotary(64, scaling="linear", factor=4.0, device="cpu").inv_freq, want / 4, rtol=1e-14, atol=0)
    ntk = kv8.rotary(64, scaling="ntk", factor=4.0, device="cpu").inv_freq
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(want[-1]) / 4, rel_tol=1e-12)
    yarn = kv8.rotary(64, scaling="yarn", factor=8.0, trained_len=4096, interleaved=True, device="cpu")
    turns = 4096 * want / (2 * math.pi)
    assert torch.allclose(yarn.inv_freq[turns >= 32], want[turns >= 32], rtol=1e-14, atol=0)
    assert torch.allclose(yarn.inv_freq[turns <= 1], want[turns <= 1] / 8, rtol=1e-14, atol=0)
    assert bool((yarn.inv_freq[1:] < yarn.inv_freq[:-1]).all()) and yarn.interleaved
    assert math.isclose(yarn.scale, 0.1 * math.log(8.0) + 1.0)
    for kw in (dict(rotary_dim=63), dict(rotary_dim=0), dict(scaling="other"), dict(factor=0.5), dict(scaling="yarn"), dict(theta=0.0),
               dict(factor=math.nan)):
        with pytest.raises(ValueError):
            kv8.rotary(**{"rotary_dim": 64, "device": "cpu", **kw})


def test_the_reference_forms():
    """The oracle's own pieces: rounding to e4m3 against torch's conversion, exponents at their borders."""
    x = torch.randn(20000, generator=torch.Generator().manual_seed(0)) * torch.logspace(-4, 2.1, 20000)
    x = x.clamp(-448, 448)
    assert torch.equal(ref.e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())
    assert ref.exponent(448.0) == 0 and ref.exponent(448.1) == 1 and ref.exponent(3.5) == -7 and ref.exponent(0.0) == -60


def test_sizes_that_would_not_fit_their_types(lib):
    from flashsvd_b200 import ops

    _refused(lib, -2, lib.fsvd_rope_qk(P, 1 << 24, P, 64, P, P, 64, 0, 1.0, P, P, 3, 1 << 17, 1, 64, 0, None), "heads")
    _refused(lib, -2, lib.fsvd_kv8_append(_cache(), P, P, 256, 256, P, None, P, 256, 256, P, P, 64, 0, 1.0, 1 << 17, 1, P, 1 << 20, None), "heads")
    for n in (1 << 31, -(1 << 31) - 1):
        with pytest.raises(ValueError):
            ops._add(n)
