"""The operators around the 8-bit cache in a run together, as a decoding loop uses them, and through the cache class, the
attention module, the engine and `generate_text`.

Attention's tolerance is that of its own tests: half a bf16 step and 2^-14 of the largest value."""
from types import SimpleNamespace

import pytest
import torch

from oracle import lowrank_llama as O
from tests import kv8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _values(cache, n):
    from flashsvd_b200 import ops

    k, v = ops.kv8_load(cache, 0, n)
    return k.double().cpu(), v.double().cpu()


class _Loop:
    """A one-layer model by hand: the token chooses a row of packed q, k, v; attention's output is the next logits' input."""

    def __init__(self, B, H, Hk, Dh, S, V, block, interleaved):
        from flashsvd_b200 import kv8, ops

        gen = torch.Generator().manual_seed(B + S)
        self.H, self.Hk, self.Dh, self.B = H, Hk, Dh, B
        self.table = torch.randn(V, H + 2 * Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV)
        self.head = (torch.randn(H * Dh, V, generator=gen) / 4).to(torch.bfloat16).to(DEV)
        self.cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
        self.ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
        self.rot = kv8.rotary(Dh, scaling="yarn", factor=4.0, trained_len=64, interleaved=interleaved, device=DEV)
        self.lens = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.tokens = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.u = torch.zeros(B, device=DEV)
        self.T = torch.linspace(0.5, 2.0, B, device=DEV)
        self.k = (torch.arange(B, dtype=torch.int32, device=DEV) % 3) * 7

    def prompt(self, ids, counts):
        from flashsvd_b200 import ops

        H, Hk = self.H, self.Hk
        x = self.table[ids.to(DEV)]
        new = torch.tensor(counts, dtype=torch.int32, device=DEV)
        ops.kv8_append(x[:, :, H:H + Hk], x[:, :, H + Hk:], self.cache, self.lens, self.ws, new_lens=new, q=x[:, :, :H],
                       rotary=self.rot)
        self.lens += new

    def step(self):
        from flashsvd_b200 import ops

        H, Hk = self.H, self.Hk
        x = self.table[self.tokens][:, None]
        q = ops.kv8_append(x[:, :, H:H + Hk], x[:, :, H + Hk:], self.cache, self.lens, self.ws, q=x[:, :, :H], rotary=self.rot)
        a = ops.flash_decode_kv8(q[:, 0], self.cache, self.lens, self.ws, seqlen_add=1)
        logits = a.view(self.B, -1) @ self.head
        _, share = ops.sample(logits, self.u, temperature=self.T, top_k=self.k, top_p=0.95, min_p=0.01, out=self.tokens)
        self.lens += 1
        return q, a, logits, share


@pytest.mark.parametrize("B,H,Hk,Dh,S,V,block,inter", [(3, 8, 2, 64, 100, 301, 16, False), (2, 4, 4, 128, 300, 97, 64, True),
                                                       (5, 12, 4, 128, 150, 203, 32, False)])
def test_prompt_steps_and_draws(B, H, Hk, Dh, S, V, block, inter):
    """Each stage against its definition on what the stage in front of it produced."""
    gen = torch.Generator().manual_seed(7)
    m = _Loop(B, H, Hk, Dh, S, V, block, inter)
    L = 40
    ids, counts = torch.randint(0, V, (B, L), generator=gen), [L - 9 * b for b in range(B)]
    rk, rv = ref.Cache(B, Hk, S, Dh, block), ref.Cache(B, Hk, S, Dh, block)
    f, sc = m.rot.inv_freq.cpu(), m.rot.scale

    def follow(ids, start, counts):
        x = m.table[ids.to(DEV)].cpu()
        pos = torch.tensor(start)[:, None] + torch.arange(ids.shape[1])
        rk.append(ref.to_bf16(ref.rotate(x[:, :, H:H + Hk], pos, f, inter, sc)), start, counts)
        rv.append(x[:, :, H + Hk:], start, counts)

    m.prompt(ids, counts)
    follow(ids, [0] * B, counts)
    m.tokens.copy_(torch.randint(0, V, (B,), generator=gen))
    for i in range(6):
        m.u.copy_(torch.rand(B, generator=gen))
        before, start = m.tokens.cpu().long(), m.lens.tolist()
        q, a, logits, share = m.step()
        follow(before[:, None], start, [1] * B)
        lens = m.lens.tolist()
        n = max(lens)
        kk, vv = _values(m.cache, n)
        for b in range(B):
            assert torch.equal(kk[b, :, :lens[b]], rk.val[b, :, :lens[b]]) and torch.equal(vv[b, :, :lens[b]], rv.val[b, :, :lens[b]])
        want = ref.attend(q[:, 0].double().cpu(), kk, vv, lens, Dh ** -0.5)
        top = float(rv.val.abs().max())
        assert bool(((a.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -14 * top).all())
        for b in range(B):
            token, p = ref.sample_row(logits[b].double().cpu(), float(m.u[b]), float(m.T[b]), int(m.k[b]),
                                      float(torch.tensor(0.95)), float(torch.tensor(0.01)))
            assert int(m.tokens[b]) == token and abs(float(share[b]) - p) <= p * 2.0 ** -24 + 2.0 ** -30
    assert m.ws.status() == 0


def test_captured_steps_equal_eager_ones():
    """The whole step in a graph, replayed, on a stream of its own, beside eager steps of a second model."""
    a, b = (_Loop(3, 8, 2, 128, 200, 211, 32, False) for _ in range(2))
    gen = torch.Generator().manual_seed(3)
    ids, us = torch.randint(0, 211, (3, 30), generator=gen), torch.rand(12, 3, generator=gen).to(DEV)
    for m in (a, b):
        m.prompt(ids, [30, 17, 1])
        m.u.copy_(us[0])
        m.step()
    torch.cuda.synchronize()
    keep = [t.clone() for t in (a.lens, a.tokens)]
    codes = [t.clone() for t in (a.cache.k.view(torch.uint8), a.cache.v.view(torch.uint8), a.cache.k_scale, a.cache.v_scale)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step()
    # (a capture runs nothing)
    assert torch.equal(a.lens, keep[0]) and torch.equal(a.tokens, keep[1])
    assert all(torch.equal(x, y) for x, y in zip(codes, (a.cache.k.view(torch.uint8), a.cache.v.view(torch.uint8), a.cache.k_scale,
                                                         a.cache.v_scale)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(1, 12):
        with torch.cuda.stream(side):
            a.u.copy_(us[i])
            graph.replay()
        b.u.copy_(us[i])
        want = b.step()
        torch.cuda.synchronize()
        for x, y in zip((*out, a.tokens, a.lens, a.cache.k_scale, a.cache.v_scale),
                        (*want, b.tokens, b.lens, b.cache.k_scale, b.cache.v_scale)):
            assert torch.equal(x, y)
    assert torch.equal(a.cache.k.view(torch.uint8), b.cache.k.view(torch.uint8))
    assert torch.equal(a.cache.v.view(torch.uint8), b.cache.v.view(torch.uint8))


def test_steps_on_another_stream_wait_for_their_inputs():
    """Inputs that are still being made on the calling stream when the operators are enqueued."""
    a, b = (_Loop(2, 4, 4, 64, 100, 50, 16, True) for _ in range(2))
    ids = torch.arange(40).view(2, 20)
    b.prompt(ids, [20, 11])
    want = [x.clone() for x in b.step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        table = a.table.clone()
        a.table.zero_()
        torch.cuda._sleep(2_000_000)
        a.table.copy_(table)
        a.prompt(ids, [20, 11])
        got = a.step()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_single_tokens_equal_the_tile_of_several():
    """The kernel for one token per sequence and the one for several: L = 1 against L = 2 with one of them new."""
    from flashsvd_b200 import kv8, ops

    gen = torch.Generator().manual_seed(21)
    for H, Hk, Dh, R, inter, block in ((40, 40, 128, 128, False, 64), (70, 5, 64, 64, True, 16), (6, 2, 128, 36, False, 128),
                                       (33, 33, 64, 2, True, 32)):
        B, S = 4, 2 * block + 3
        rot = kv8.rotary(R, interleaved=inter, device=DEV)
        ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
        one, two = (kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV) for _ in range(2))
        lens = torch.tensor([0, block - 1, block, S - 2], dtype=torch.int32, device=DEV)
        first = torch.randn(B, S, Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV) / 64
        for c in (one, two):
            ops.kv8_append(first, first, c, torch.zeros_like(lens), ws, new_lens=lens)
        for i, gain in enumerate((1.0, 0.01, 300.0)):   # the scale of a block that holds tokens grows, stays, grows
            x = (gain * torch.randn(B, 2, H + 2 * Hk, Dh, generator=gen)).to(torch.bfloat16).to(DEV)
            new = torch.tensor([1, 1, 1 if i else 0, 1], dtype=torch.int32, device=DEV)
            outs = []
            for c, n in ((one, 1), (two, 2)):
                out = torch.zeros(B, n, H, Dh, dtype=torch.bfloat16, device=DEV)
                ops.kv8_append(x[:, :n, H:H + Hk], x[:, :n, H + Hk:], c, lens, ws, new_lens=new, q=x[:, :n, :H], rotary=rot, q_out=out)
                outs.append(out)
            assert torch.equal(outs[0][:, 0], outs[1][:, 0])
            lens = lens + new
            for s, t in ((one.k.view(torch.uint8), two.k.view(torch.uint8)), (one.v.view(torch.uint8), two.v.view(torch.uint8)),
                         (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
                assert torch.equal(s, t)
        # the last sequence ran over the end in the third round: its token was dropped, its query was not
        assert ws.raw_status() != 0 and bool(outs[0][3].any())


def _config(shape, layers=1):
    return SimpleNamespace(hidden_size=shape.d, num_attention_heads=shape.H, num_key_value_heads=shape.Hk, head_dim=shape.Dh,
                           num_hidden_layers=layers, rope_theta=shape.theta, max_position_embeddings=64)


def _attention(shape, cfg, seed, layer_idx=0):
    from flashsvd_b200 import modules as M

    w = O.make_layer_weights(shape, torch.Generator().manual_seed(seed), torch.bfloat16)
    att = M.SVD_LlamaAttention(cfg, 0.5, layer_idx=layer_idx)
    for n in ("q_v", "q_u", "k_v", "k_u", "v_v", "v_u", "o_v", "o_u"):
        lin = getattr(att, n + "_proj")
        lin.weight = torch.nn.Parameter(w[n].clone(), requires_grad=False)
        lin.in_features, lin.out_features = w[n].shape[1], w[n].shape[0]
    return att.to(DEV), w


@pytest.mark.parametrize("B", [1, 3, 9])
def test_attention_module_over_the_8bit_cache(B):
    """Prompt, then single tokens.  What the module appends is bit for bit the reference's codes of its own projections;
    its output is the output projection of attention in 64 bits over those codes, within the roundings on the way:
    scores move by 2^-8 of sum |q k| (the query's rounding), attention by half a bf16 step more, the projection by half
    a step at its rank space and half a step at the end (2^-7 covers each with the sums' own errors)."""
    from flashsvd_b200 import ops, runtime as R

    shape = O.TINY_GQA
    cfg = _config(shape)
    att, w = _attention(shape, cfg, 31)
    H, Hk, Dh, S, Lp, block = shape.H, shape.Hk, shape.Dh, 48, 21, 16
    cache = R.FlashSVDV15KV8Cache(cfg, max_batch_size=max(B, 4), max_cache_len=S, device=DEV, block=block)
    xs = torch.randn(B, Lp + 4, shape.d, generator=torch.Generator().manual_seed(32)).to(torch.bfloat16).to(DEV)
    rk, rv = ref.Cache(B, Hk, S, Dh, block), ref.Cache(B, Hk, S, Dh, block)
    f = cache.rotary(Dh, torch.device(DEV)).inv_freq.cpu()
    ws = ops.make_workspace(ops.make_dims(dtype=torch.bfloat16, B=min(B, 8), d=shape.d, H=H, Hk=Hk, Dh=Dh, Rq=shape.Rq, Rk=shape.Rk,
                                          Rv=shape.Rv, Ro=shape.Ro), DEV)

    def project(x, name):
        v, u = getattr(att, name + "_v_proj"), getattr(att, name + "_u_proj")
        if x.shape[1] == 1 and B <= 8:
            return ops.lowrank_proj(x[:, 0].contiguous(), v.weight, u.weight, ws)[:, None]
        return u(v(x))

    with torch.inference_mode():
        t = 0
        for L in (Lp, 1, 1, 2, 1):
            x = xs[:, t:t + L] if t + L <= xs.shape[1] else xs[:, :L]
            y, _ = att(x, past_key_values=cache, cache_position=torch.arange(t, t + L) if t else None)
            q, k, v = (project(x, n).view(B, L, -1, Dh).cpu() for n in "qkv")
            pos = (t + torch.arange(L)).expand(B, L)
            rk.append(ref.to_bf16(ref.rotate(k, pos, f)), [t] * B, [L] * B)
            rv.append(v, [t] * B, [L] * B)
            kk, vv = _values(cache.layer(0, B), t + L)
            assert torch.equal(kk, rk.val[:, :, :t + L]) and torch.equal(vv, rv.val[:, :, :t + L])
            qr = ref.rotate(q, pos, f)
            Vo, Uo = w["o_v"].double(), w["o_u"].double()
            for i in range(L):
                a = ref.attend(qr[:, i], kk, vv, [t + i + 1] * B, Dh ** -0.5).reshape(B, -1)
                moved = Dh ** -0.5 * torch.einsum("bhd,bhnd->bhn", qr[:, i].abs(), kk.abs().repeat_interleave(H // Hk, 1)).max() * 2.0 ** -8
                vals = ref.attend(qr[:, i], kk, vv.abs(), [t + i + 1] * B, Dh ** -0.5).reshape(B, -1)
                ea = torch.expm1(2 * moved) * vals + a.abs() * 2.0 ** -7 + 2.0 ** -14 * float(vv.abs().max())
                p = a @ Vo.T
                ep = ea @ Vo.abs().T + p.abs() * 2.0 ** -7
                want = p @ Uo.T
                bound = ep @ Uo.abs().T + want.abs() * 2.0 ** -7 + 2.0 ** -14
                assert bool(((y[:, i].double().cpu() - want).abs() <= bound).all())
            t += L
            assert cache.get_seq_length() == t


def test_cache_class_keeps_layers_apart_and_reads_back():
    from flashsvd_b200 import ops, runtime as R

    shape = O.TINY_GQA
    cfg = _config(shape, layers=2)
    Hk, Dh = shape.Hk, shape.Dh
    cache = R.FlashSVDV15KV8Cache(cfg, max_batch_size=4, max_cache_len=20, device=DEV, block=16)
    assert cache.get_max_cache_shape() == 20 and cache.get_seq_length() == 0 and len(cache) == 2
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn(3, Hk, 9, Dh, generator=gen).to(torch.bfloat16).to(DEV) for _ in range(2))
    for layer in (0, 1):
        kk, vv = cache.update(k, v, layer)
        assert kk.shape == (3, Hk, 9, Dh) and kk.dtype == torch.bfloat16
        want = ref.Cache(3, Hk, 20, Dh, 16)
        want.append(k.transpose(1, 2).cpu(), [0] * 3, [9] * 3)
        assert torch.equal(kk.double().cpu(), want.val[:, :, :9])
    assert cache.get_seq_length(0) == cache.get_seq_length(1) == 9
    kk, _ = cache.update(k[:, :, :2], v[:, :, :2], 0, {"cache_position": torch.tensor([9, 10], device=DEV)})
    assert kk.shape[2] == 11 and cache.get_seq_length(0) == 11 and cache.get_seq_length(1) == 9
    # positions per sequence; positions that only the device knows
    x = torch.randn(3, 1, Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV)
    q = torch.randn(3, 1, shape.H, Dh, generator=gen).to(torch.bfloat16).to(DEV)
    a = cache.decode_step(q, x, x, 0, cache_position=torch.tensor([11, 4, 0]))
    b = cache.decode_step(q, x, x, 0, cache_position=torch.tensor([11, 4, 0], device=DEV))
    assert torch.equal(a, b) and a.shape == (3, shape.H, Dh)
    # a sequence of one token: attention returns its value as the codes hold it
    vv = ops.kv8_load(cache.layer(0, 3), 0, 1)[1][2, :, 0].repeat_interleave(shape.H // Hk, 0)
    assert torch.equal(a[2], vv)
    for bad in (torch.tensor([20]), torch.tensor([-1]), 20, -1):
        with pytest.raises(IndexError):
            cache.decode_step(q, x, x, 0, cache_position=bad)
    with pytest.raises(IndexError):
        cache.update(k, v, 0, {"cache_position": torch.arange(12, 21)})
    for bad in (torch.tensor([1, 3, 2, 4, 5, 6, 7, 8, 9]), torch.arange(4)):
        with pytest.raises(ValueError):
            cache.update(k, v, 0, {"cache_position": bad})
    with pytest.raises(ValueError, match="bfloat16"):
        cache.update(k.float(), v.float(), 0)
    with pytest.raises(RuntimeError, match="shape changed"):
        cache.update(k[:, :1], v[:, :1], 0)
    with pytest.raises(RuntimeError, match="exceeds max_batch_size"):
        cache.update(k[:1].expand(5, -1, -1, -1), v[:1].expand(5, -1, -1, -1), 0)
    cache.reset()
    kk, _ = cache.update(k, v, 1)
    want = ref.Cache(3, Hk, 20, Dh, 16)
    want.append(k.transpose(1, 2).cpu(), [0] * 3, [9] * 3)
    assert torch.equal(kk.double().cpu(), want.val[:, :, :9]) and cache.get_seq_length(1) == 9
    assert cache.nbytes() == sum(c.nbytes() for c in cache.layers8)


class _Tok:
    eos_token_id = None

    def __call__(self, prompt, return_tensors="pt", add_special_tokens=False):
        return {"input_ids": torch.tensor([[int(t) for t in prompt.split()]], dtype=torch.long)}

    def decode(self, ids, skip_special_tokens=False):
        return " ".join(str(int(i)) for i in ids)


def _engine(B, cls=None, **kw):
    from flashsvd_b200 import engine, packing

    shape, dtype = O.TINY, torch.float32
    w = O.make_model_weights(shape, seed=1, dtype=dtype)
    layers = [packing.pack_layer(lw, device=torch.device(DEV), dtype=dtype) for lw in w["layers"]]
    return (cls or engine.DecodeEngine)(layers=layers, embed=w["embed"].to(DEV), final_norm=w["norm"].to(DEV), lm_head=w["lm_head"].to(DEV),
                                        num_heads=shape.H, num_kv_heads=shape.Hk, head_dim=shape.Dh, batch_size=B, max_cache_len=32,
                                        rope_theta=shape.theta, eps=shape.eps, max_steps=64, **kw)


def test_engine_draws_the_next_input():
    from flashsvd_b200 import engine

    prompt = torch.randint(0, O.TINY.vocab, (3, 5), generator=torch.Generator().manual_seed(2))
    us = torch.rand(4, 3, generator=torch.Generator().manual_seed(4))
    T = torch.tensor([0.7, 1.0, 3.0], device=DEV)
    group = _engine(3, engine.EngineGroup, width=2)
    eng = _engine(3)
    for e in (eng, group):
        e.prefill(prompt)
    for u in us:
        got = eng.sample(u.to(DEV), temperature=T, top_k=50, top_p=0.9)
        assert got.data_ptr() == eng.tokens.data_ptr()
        x = eng.logits.double().cpu()
        assert got.tolist() == [ref.sample_row(x[b], float(u[b]), float(T[b]), 50, float(torch.tensor(0.9)), 0.0)[0] for b in range(3)]
        other = group.sample(u.to(DEV), temperature=T, top_k=50, top_p=0.9)
        x = torch.cat([e.logits for e in group.engines]).double().cpu()
        assert other.tolist() == [ref.sample_row(x[b], float(u[b]), float(T[b]), 50, float(torch.tensor(0.9)), 0.0)[0] for b in range(3)]
        assert torch.equal(group.tokens, other)
        for e in (eng, group):
            e.step(1)
    with pytest.raises(ValueError):
        group.sample(us[0, :2].to(DEV))
    with pytest.raises(ValueError):
        group.sample(us[0].to(DEV), temperature=T[:2])
    with pytest.raises(ValueError):
        eng.sample(us[0])
    eng.close(), group.close()


@torch.inference_mode()
def test_generate_text_draws_on_the_device():
    from flashsvd_b200 import runtime as R

    eng = _engine(1)
    prompt = torch.randint(0, O.TINY.vocab, (1, 6), generator=torch.Generator().manual_seed(2))
    text = " ".join(str(int(t)) for t in prompt[0])
    us = torch.rand(8, generator=torch.Generator().manual_seed(6))
    res = R.generate_text(eng, _Tok(), prompt=text, max_new_tokens=8, do_sample=True, temperature=1.5, top_p=0.9, top_k=40, min_p=0.01,
                          uniforms=us)
    eng.reset()
    eng.prefill(prompt)
    want = []
    for u in us:
        want.append(ref.sample_row(eng.logits[0].double().cpu(), float(u), 1.5, 40, float(torch.tensor(0.9)), float(torch.tensor(0.01)))[0])
        eng.tokens.fill_(want[-1])
        eng.step(1)
    assert res["completion_ids"] == want and res["generated_token_count"] == 8
    tok = _Tok()
    tok.eos_token_id = want[2]
    cut = R.generate_text(eng, tok, prompt=text, max_new_tokens=8, do_sample=True, temperature=1.5, top_p=0.9, top_k=40, min_p=0.01,
                          uniforms=us)
    assert cut["completion_ids"] == want[:want.index(want[2]) + 1]
    # uniforms from torch's generator: the same seed, the same text
    runs = []
    for _ in range(2):
        torch.cuda.manual_seed(9)
        runs.append(R.generate_text(eng, _Tok(), prompt=text, max_new_tokens=8, do_sample=True, top_k=100)["completion_ids"])
    assert runs[0] == runs[1]
    with pytest.raises(ValueError, match="uniforms"):
        R.generate_text(eng, _Tok(), prompt=text, max_new_tokens=8, do_sample=True, uniforms=us[:3])
    eng.close()


def test_rotary_module_rotates_without_tables():
    from flashsvd_b200 import modules as M

    rope = M.LlamaRotaryEmbedding(128, base=500000.0)
    gen = torch.Generator().manual_seed(8)
    q, k = torch.randn(7, 4, 128, generator=gen).to(torch.bfloat16), torch.randn(7, 2, 128, generator=gen).to(torch.bfloat16)
    pos = torch.tensor([0, 1, 5, 1000, 131071, 17, 2])
    got = rope.rotate(q.to(DEV), k.to(DEV), pos)
    f = 500000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    for y, x in zip(got, (q, k)):
        want = ref.rotate(x, pos, f)
        assert bool(((y.double().cpu() - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -20 * float(x.abs().max())).all())


def test_model_step_over_the_8bit_cache_eager_and_captured():
    """A transformers Llama of these modules: prompt at once or token by token fill the caches alike up to the projections'
    own roundings; a step with its position on the device, captured and replayed, equals the eager one bit for bit."""
    from flashsvd_b200 import runtime as R
    from tests.test_gpu_boundary import _hf_model

    shape, dev = O.TINY_GQA, torch.device(DEV)
    w = O.make_model_weights(shape, seed=4, dtype=torch.bfloat16)
    model = _hf_model(shape, w, torch.bfloat16, dev)
    with torch.inference_mode():
        layers = len(model.model.layers)
        ids = torch.randint(0, shape.vocab, (2, 12), generator=torch.Generator().manual_seed(8)).to(dev)
        runs = []
        for captured in (False, True):
            cache = R.FlashSVDV15KV8Cache(model.config, max_batch_size=2, max_cache_len=32, device=dev, block=16)
            logits = [R.manual_llama_decode_step(model, ids[:, :6], past_key_values=cache, cache_position=torch.arange(6)).logits.clone()]
            assert [cache.get_seq_length(i) for i in range(layers)] == [6] * layers
            if captured:
                tok, pos = ids[:, :1].clone(), torch.tensor([31], device=dev)
                R.manual_llama_decode_step(model, tok, past_key_values=cache, cache_position=pos)   # (workspaces, at a place not used)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = R.manual_llama_decode_step(model, tok, past_key_values=cache, cache_position=pos).logits
            for t in range(6, 12):
                if captured:
                    tok.copy_(ids[:, t:t + 1])
                    pos.fill_(t)
                    graph.replay()
                    logits.append(out.clone())
                else:
                    logits.append(R.manual_llama_decode_step(model, ids[:, t:t + 1], past_key_values=cache,
                                                             cache_position=torch.tensor([t])).logits.clone())
            runs.append((logits, [(c.k.view(torch.uint8)[:, :, :12].clone(), c.v.view(torch.uint8)[:, :, :12].clone()) for c in cache.layers8]))
        for x, y in zip(*(r[0] for r in runs)):
            assert bool(torch.isfinite(x).all()) and torch.equal(x, y)
        for x, y in zip(*(r[1] for r in runs)):
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
        with pytest.raises(IndexError):
            R.manual_llama_decode_step(model, ids[:, :1], past_key_values=cache, cache_position=torch.tensor([32]))


def test_calls_beside_each_other_with_workspaces_of_their_own():
    """Append, read-back, attention and sampling of two models on two streams at once, many times over."""
    models = [_Loop(4, 8, 2, 128, 400, 5003, 64, bool(i)) for i in range(2)]
    ids = torch.arange(400).view(4, 100)
    us = torch.rand(20, 4, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = []
    for m in models:
        m.prompt(ids, [100, 64, 3, 0])
        trace = []
        for u in us:
            m.u.copy_(u)
            q, a, logits, share = m.step()
            trace += [a, m.tokens.clone(), share]
        want.append(trace)
    torch.cuda.synchronize()
    again = [_Loop(4, 8, 2, 128, 400, 5003, 64, bool(i)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in again]
    got = [[], []]
    torch.cuda.synchronize()
    for m, s in zip(again, streams):
        with torch.cuda.stream(s):
            m.prompt(ids, [100, 64, 3, 0])
    for u in us:
        for i, (m, s) in enumerate(zip(again, streams)):
            with torch.cuda.stream(s):
                m.u.copy_(u)
                q, a, logits, share = m.step()
                got[i] += [a, m.tokens.clone(), share]
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_lengths_at_and_past_their_ends():
    """Negative and huge lengths: nothing is read or written outside, the flag is set where a token was dropped."""
    from flashsvd_b200 import kv8, ops

    B, H, Hk, Dh, S, block = 5, 4, 2, 64, 40, 16
    gen = torch.Generator().manual_seed(17)
    for L in (1, 3):
        cache = kv8.KV8Cache.empty(B, S, Hk, Dh, block=block, device=DEV)
        ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
        x = torch.randn(B, S, Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV)
        ops.kv8_append(x, x, cache, torch.zeros(B, dtype=torch.int32, device=DEV), ws)
        before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
        lens = torch.tensor([S, 2 ** 31 - 1, 7, 39, -5], dtype=torch.int32, device=DEV)
        new = torch.tensor([L, L, -3, 0, 0], dtype=torch.int32, device=DEV)
        y = torch.randn(B, L, Hk, Dh, generator=gen).to(torch.bfloat16).to(DEV)
        ops.kv8_append(y, y, cache, lens, ws, new_lens=new)
        after = (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)
        assert all(torch.equal(a, b) for a, b in zip(before, after))
        assert ws.raw_status() != 0
        ws.clear_status()
        ops.kv8_append(y, y, cache, lens, ws, new_lens=torch.tensor([0, 0, L + 5, 1, 0], dtype=torch.int32, device=DEV))
        assert ws.status() == 0
        k = ops.kv8_load(cache, 0, S)[0]
        old = (before[0].view(torch.float8_e4m3fn).float() * before[2].repeat_interleave(block, 2)[:, :, :S, None]).to(torch.bfloat16)
        assert torch.equal(k[0], old[0]) and torch.equal(k[1], old[1]) and torch.equal(k[4], old[4])
        q = torch.randn(B, H, Dh, generator=gen).to(torch.bfloat16).to(DEV)
        full = ops.flash_decode_kv8(q, cache, torch.tensor([S, S, 10, S, 0], dtype=torch.int32, device=DEV), ws)
        assert torch.equal(full, ops.flash_decode_kv8(q, cache, torch.tensor([2 ** 31 - 1, S, 10, S + 1, -9], dtype=torch.int32, device=DEV), ws))
        assert torch.equal(full, ops.flash_decode_kv8(q, cache, torch.tensor([2 ** 31 - 1, S - 3, 7, S, -2 ** 31], dtype=torch.int32,
                                                                             device=DEV), ws, seqlen_add=3))
        k2 = ops.kv8_load(cache, 2, 9, cache_seqlens=torch.tensor([2 ** 31 - 1, -1, 3, -2 ** 31, 11], dtype=torch.int32, device=DEV))[0]
        for b, n in enumerate((9, 0, 1, 0, 9)):
            assert torch.equal(k2[b, :, :n], k[b, :, 2:2 + n]) and not bool(k2[b, :, n:].any())


@pytest.mark.parametrize("inter,R", [(True, 64), (True, 128), (False, 128), (False, 64), (True, 36), (False, 0)])
def test_rows_on_boundaries_of_16_bytes_only(inter, R):
    """The same call with every tensor 16 bytes behind a boundary of 32."""
    from flashsvd_b200 import kv8, ops

    B, H, Hk, Dh, S = 2, 6, 2, 128, 90
    gen = torch.Generator().manual_seed(R)

    def off(t):
        return torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)[8:].view(t.shape).copy_(t)

    rot = kv8.rotary(R, interleaved=inter, device=DEV) if R else None
    ws = ops.make_kv8_workspace(B, H, Hk, Dh, S, DEV)
    caches = [kv8.KV8Cache.empty(B, S, Hk, Dh, block=32, device=DEV) for _ in range(2)]
    lens = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    for L in (70, 1):
        q, k, v = (torch.randn(B, L, n, Dh, generator=gen).to(torch.bfloat16).to(DEV) for n in (H, Hk, Hk))
        a = ops.kv8_append(k, v, caches[0], lens, ws, q=q if R else None, rotary=rot)
        b = ops.kv8_append(off(k), off(v), caches[1], lens, ws, q=off(q) if R else None, rotary=rot,
                           q_out=off(torch.zeros_like(q)) if R else None)
        assert (a is None and b is None) or torch.equal(a, b)
        lens = lens + L
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))
        assert torch.equal(caches[0].v.view(torch.uint8), caches[1].v.view(torch.uint8))
        if R:
            pos = torch.arange(L, dtype=torch.int32, device=DEV)
            a = ops.rope_qk(q[0], k[0], pos, rot.inv_freq, interleaved=inter)
            b = ops.rope_qk(off(q[0]), off(k[0]), pos, rot.inv_freq, interleaved=inter, q_out=off(q[0]), k_out=off(k[0]))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = ops.kv8_load(caches[0], 3, 60)
    b = ops.kv8_load(caches[0], 3, 60, k_out=off(torch.zeros_like(a[0])), v_out=off(torch.zeros_like(a[1])))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
