"""The decoder on a 4-bit KV cache (kv_q4), its log probabilities and scores.

The reference is LlamaModel.Forward (LlamaModel.cs:93-238) restated in numpy, 64 bits.  A level of a stored row may
legitimately fall on either side of a border that the row's fp32 rounding straddles, so the reference checks each
stored row against its own (within half a step, or beyond the end of the scale) and then attends over the stored
values.  Logits: the repository's 1e-3 of the largest."""
from __future__ import annotations

import numpy as np
import pytest

import chatnet_b200 as cn
from chatnet_b200 import configs as cf
from chatnet_b200.llama import CudaLlamaModel
from tests.parity import REL_TOL, rel_err
from tests.test_gpu_llama import small_dc

torch = pytest.importorskip("torch")
from tests import _kvq4 as ref  # noqa: E402

pytestmark = pytest.mark.gpu


def q4_dc(head_dim=64, n_heads=4, n_kv=2, max_batch=1, ctx_len=80, neox=False, wtype=cn.TYPE_Q4_0):
    dc = small_dc(wtype, max_batch=max_batch, ctx_len=ctx_len)
    m = cf.replace(dc.model, dim=head_dim * n_heads, n_heads=n_heads, n_kv_heads=n_kv, head_dim=head_dim, kv_q4=True,
                   rope_neox=neox)
    return cf.replace(dc, model=m, kv_filled=0, decode_pos=0)


class NumpyLlama:
    def __init__(self, oracle, dc, host):
        self.m, self.w = dc.model, {}
        for name, b in host.items():
            t = cf.tensor_type(dc, name)
            if t == cn.TYPE_F32:
                self.w[name] = np.asarray(b, np.float64).ravel()
            else:
                rows = b.shape[0]
                cols = self.m.hidden_dim if "ffn_down" in name else self.m.dim
                self.w[name] = oracle.dequantize(t, b, rows * cols).reshape(rows, cols).astype(np.float64)
        m = self.m
        i = np.arange(0, m.head_dim, 2, dtype=np.float32)
        th = np.arange(m.ctx_len, dtype=np.float32)[:, None] * np.exp(
            i * np.float32(1 / m.head_dim) * -np.log(np.float32(m.rope_base)))
        self.cos, self.sin = np.cos(th).astype(np.float64), np.sin(th).astype(np.float64)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.m.rms_eps) * w

    def rope(self, x, pos):  # [n, heads, hd]
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        h = x.shape[-1] // 2
        a, b = (x[..., :h], x[..., h:]) if self.m.rope_neox else (x[..., 0::2], x[..., 1::2])
        r0, r1 = a * c - b * s, a * s + b * c
        return np.concatenate([r0, r1], -1) if self.m.rope_neox else np.stack([r0, r1], -1).reshape(x.shape)

    def check_row(self, stored, x, what, tol):
        """stored values against the rows they came from (both [n, kv, hd])."""
        xb = x.reshape(*x.shape[:-1], -1, 32)
        sb = stored.reshape(xb.shape)
        lo, hi = xb.min(-1), xb.max(-1)
        d = np.abs(np.where(-lo >= hi, lo, hi))[..., None] / 8
        # half a step, the scale's fp16 rounding (2^-11 of up to 8 steps), the clipped end (7 of 8 steps), and the
        # rows' own accuracy
        err = np.abs(sb - xb)
        clipped = np.abs(xb) > 7.45 * d
        assert (err <= np.where(clipped, 1.01, 0.5 + 8 * 2.0 ** -11) * d + tol * np.abs(xb).max()).all(), what

    def forward(self, gpu, tokens, pos, seq=0, tol=REL_TOL):
        m, n = self.m, len(tokens)
        at = np.arange(pos, pos + n)
        x = self.w["token_embd.weight"][np.asarray(tokens)]
        for l in range(m.n_layers):
            W = {k: self.w[f"blk.{l}.{k}.weight"] for k in ("attn_norm", "attn_q", "attn_k", "attn_v", "attn_output",
                                                           "ffn_norm", "ffn_gate", "ffn_up", "ffn_down")}
            y = self.norm(x, W["attn_norm"])
            q = self.rope((y @ W["attn_q"].T).reshape(n, m.n_heads, m.head_dim), at)
            k = self.rope((y @ W["attn_k"].T).reshape(n, m.n_kv_heads, m.head_dim), at)
            v = (y @ W["attn_v"].T).reshape(n, m.n_kv_heads, m.head_dim)
            sk, sv = (a.astype(np.float64).reshape(-1, m.n_kv_heads, m.head_dim)
                      for a in gpu.kv_read(seq, l, 0, pos + n))
            self.check_row(sk[pos:], k, f"layer {l} k", tol)
            self.check_row(sv[pos:], v, f"layer {l} v", tol)
            o = np.empty_like(q)
            for i in range(n):
                for h in range(m.n_heads):
                    g = h // m.kv_mul
                    s = sk[:pos + i + 1, g] @ q[i, h] / np.sqrt(m.head_dim)
                    p = np.exp(s - s.max())
                    o[i, h] = p @ sv[:pos + i + 1, g] / p.sum()
            x = x + o.reshape(n, -1) @ W["attn_output"].T
            y = self.norm(x, W["ffn_norm"])
            g = y @ W["ffn_gate"].T
            x = x + (g / (1 + np.exp(-g)) * (y @ W["ffn_up"].T)) @ W["ffn_down"].T
        return self.norm(x, self.w["output_norm.weight"]) @ self.w["output.weight"].T


@pytest.fixture
def build(ctx, oracle):
    made = []

    def make(dc):
        host = cf.host_tensors(dc)
        ts = cf.device_tensors(ctx, dc, host)
        g = CudaLlamaModel(ctx, dc.model, ts)
        made.append((g, ts))
        return g, NumpyLlama(oracle, dc, host)
    yield make
    for g, ts in made:
        g.close()
        for t in ts:
            t.free()


@pytest.mark.parametrize("head_dim,n_heads,n_kv,neox", [(64, 4, 2, False), (128, 2, 1, True), (32, 8, 8, False),
                                                       (256, 2, 1, False)])
def test_decode(build, head_dim, n_heads, n_kv, neox):
    dc = q4_dc(head_dim, n_heads, n_kv, neox=neox)
    g, r = build(dc)
    g.set_prefill(0)
    for pos in range(12):
        got = g.forward([(37 * pos + 5) % dc.model.vocab], pos)
        assert rel_err(got, r.forward(g, [(37 * pos + 5) % dc.model.vocab], pos)[-1]) <= REL_TOL, pos


def test_decode_batch_ragged(build):
    dc = q4_dc(max_batch=3)
    g, r = build(dc)
    pos = [0, 20, 61]
    for b in range(3):
        g.kv_synth(b, pos[b], 11 + b, 21 + b)
    tok = np.array([3, 77, 401])
    for step in range(3):
        lg, am = g.decode(tok, pos)
        for b in range(3):
            want = r.forward(g, [int(tok[b])], pos[b], seq=b)[-1]
            assert rel_err(lg[b], want) <= REL_TOL
            assert am[b] == int(np.argmax(lg[b]))
        lp, ent, ids, tlp = g.logprobs(3, am, 5)
        x = lg.astype(np.float64)
        want = x - x.max(-1, keepdims=True)
        want = want - np.log(np.exp(want).sum(-1, keepdims=True))
        np.testing.assert_allclose(lp, want[np.arange(3), am], atol=1e-5)
        np.testing.assert_allclose(ent, -(np.exp(want) * want).sum(-1), atol=1e-5)
        order = np.argsort(-lg, axis=-1, kind="stable")[:, :5]
        np.testing.assert_array_equal(ids, order)
        np.testing.assert_allclose(tlp, np.take_along_axis(want, order, -1), atol=1e-5)
        tok, pos = am, [p + 1 for p in pos]


@pytest.mark.parametrize("head_dim,n_heads,n_kv,neox", [(64, 4, 2, False), (128, 2, 2, True), (64, 8, 1, False)])
def test_prompt(build, head_dim, n_heads, n_kv, neox):
    """A prompt in one pass, then a second piece after it, then a decode step."""
    dc = q4_dc(head_dim, n_heads, n_kv, neox=neox, ctx_len=200)
    g, r = build(dc)
    rng = np.random.default_rng(3)
    toks = rng.integers(0, dc.model.vocab, 130)
    for lo, hi in ((0, 70), (70, 129), (129, 130)):
        got = g.forward(toks[lo:hi], lo)
        assert rel_err(got, r.forward(g, toks[lo:hi], lo)[-1]) <= REL_TOL, lo


def test_cache_access(build):
    dc = q4_dc(max_batch=2, ctx_len=44)  # (the cache itself is padded to 48 positions)
    g, _ = build(dc)
    m = dc.model
    rng = np.random.default_rng(0)
    k = rng.standard_normal((20, m.kv_dim)).astype(np.float32)
    v = rng.standard_normal((20, m.kv_dim)).astype(np.float32)

    def rounded(a):
        lv, d = ref.quantize(torch.from_numpy(a).reshape(-1, m.n_kv_heads, m.head_dim))
        return ref.values(ref.pack(lv), d, torch.float32).reshape(a.shape).numpy()
    g.kv_synth(1, 44, 5, 6)
    other = g.kv_read(1, 0, 0, 44)
    g.kv_write(1, 1, 24, k, v)
    rk, rv = g.kv_read(1, 1, 24, 20)
    np.testing.assert_array_equal(rk, rounded(k))
    np.testing.assert_array_equal(rv, rounded(v))
    for a, b in zip(other, g.kv_read(1, 0, 0, 44)):
        np.testing.assert_array_equal(a, b)
    assert not g.kv_read(0, 0, 0, 44)[0].any()  # an unwritten slot holds zeros
    # the generator's rows, rounded; zeros after them
    L, C = m.n_layers, m.ctx_len
    full = [cn.synth_fill(cn.TYPE_F32, L * C, m.kv_dim, seed).reshape(L, C, -1) for seed in (5, 6)]
    g.kv_synth(0, 30, 5, 6)
    for l in range(L):
        for got, want in zip(g.kv_read(0, l, 0, C), full):
            np.testing.assert_array_equal(got[:30], rounded(want[l, :30]))
            assert not got[30:].any()


def test_score(build):
    """Scores against the logits of one forward call per token, and the prefill pass against the sequential steps."""
    for dc in (q4_dc(ctx_len=100), cf.replace(small_dc(ctx_len=100), kv_filled=0, decode_pos=0)):
        g, _ = build(dc)
        toks = np.random.default_rng(1).integers(0, dc.model.vocab, 60)
        g.set_prefill(0)
        lp, ent = g.score(toks)
        logits = np.stack([g.forward([int(t)], i) for i, t in enumerate(toks[:-1])]).astype(np.float64)
        want = logits - logits.max(-1, keepdims=True)
        want = want - np.log(np.exp(want).sum(-1, keepdims=True))
        np.testing.assert_allclose(lp, want[np.arange(59), toks[1:]], atol=1e-5)
        np.testing.assert_allclose(ent, -(np.exp(want) * want).sum(-1), atol=1e-5)
        if not dc.model.kv_q4:  # (levels of a 4-bit cache may differ between the two ways)
            g.set_prefill(16)
            lp2, ent2 = g.score(toks)
            # each logit within 1e-3 of the largest: its log probability within twice that
            tol = 2 * REL_TOL * np.abs(logits).max(-1)
            assert (np.abs(lp2 - lp) <= tol).all()


def test_refusals(build):
    dc = q4_dc()
    g, _ = build(dc)
    g.forward([1], 0)
    for bad in (dict(batch=0), dict(batch=2), dict(batch=1, top_n=65), dict(batch=1, top_n=-1)):
        with pytest.raises(ValueError):
            g.logprobs(**bad)
    with pytest.raises(ValueError):
        g.logprobs(1, [1, 2])
    for bad in (([1], 0), ([1, dc.model.vocab], 0), ([1, -1], 0), ([1, 2, 3], dc.model.ctx_len - 1), ([1, 2], -1)):
        with pytest.raises(ValueError):
            g.score(*bad)
    with pytest.raises(cn.NotSupportedError):
        bad = cf.replace(q4_dc(), model=cf.replace(q4_dc().model, dim=320, n_heads=4, n_kv_heads=4, head_dim=80))
        CudaLlamaModel(g.ctx, bad.model, cf.device_tensors(g.ctx, bad))


def test_serving_step(ctx):
    """A decode step's operators together on one stream, captured: new rows into the cache, attention, the head's
    quantized matvec, log probabilities; replayed with other inputs."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    B, kv, heads, hd, ctx_len, vocab = 4, 2, 16, 64, 256, 1000
    dim = heads * hd
    blocks = cn.synth_fill(cn.TYPE_Q4_0, vocab, dim, 9)
    W = ctx.upload(blocks, cn.TYPE_Q4_0, vocab, dim)
    Wd = torch.from_numpy(ctx.dequantize(W)).cuda().double()
    quants = {w: torch.full((B, kv, ctx_len, hd // 2), 0x88, dtype=torch.uint8, device="cuda") for w in "kv"}
    scales = {w: torch.zeros(B, kv, ctx_len, hd // 32, dtype=torch.float16, device="cuda") for w in "kv"}
    cache = cn.KvQ4Cache(quants["k"].data_ptr(), scales["k"].data_ptr(), quants["v"].data_ptr(),
                         scales["v"].data_ptr(), B, kv, hd, ctx_len)
    table = ref.rope_table(ctx_len, hd).cuda()
    q = torch.empty(B, 1, dim, device="cuda")
    k, v = (torch.empty(B, 1, kv * hd, device="cuda") for _ in range(2))
    att, logits = torch.empty(B, dim, device="cuda"), torch.empty(B, vocab, device="cuda")
    pos, tok = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    lp, ent = (torch.empty(B, device="cuda") for _ in range(2))
    ids, tlp = torch.empty(B, 3, dtype=torch.int32, device="cuda"), torch.empty(B, 3, device="cuda")
    s = torch.cuda.ExternalStream(ctx.stream)

    def step():
        ctx.kvq4_append_dev(cache, k.data_ptr(), v.data_ptr(), pos.data_ptr(), B, rope=table.data_ptr(),
                            stream=ctx.stream)
        ctx.kvq4_attend_dev(cache, q.data_ptr(), att.data_ptr(), pos.data_ptr(), B, heads, rope=table.data_ptr(),
                            stream=ctx.stream)
        cn.check(cn.N.lib().cn_matvec_dev(ctx.handle, cn.TYPE_Q4_0, W.device_ptr, vocab, dim, att.data_ptr(),
                                          logits.data_ptr(), B))
        ctx.logprobs_dev(logits.data_ptr(), B, vocab, tok.data_ptr(), lp.data_ptr(), ent.data_ptr(), 3,
                         ids.data_ptr(), tlp.data_ptr(), stream=ctx.stream)

    graph = None
    held = {w: torch.zeros(B, kv, ctx_len, hd, device="cuda", dtype=torch.float64) for w in "kv"}
    for it in range(6):
        for t in (q, k, v):
            t.normal_(generator=gen)
        pos.copy_(torch.tensor([it, it + 3, 40 + it, 200 + it], dtype=torch.int32))
        tok.random_(0, vocab, generator=gen)
        torch.cuda.synchronize()
        if it == 2:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                step()
        if graph is None:
            step()
        else:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            p = int(pos[b])
            for w, x in (("k", ref.rotate(k[b].view(1, kv, hd), table[p:p + 1], False)), ("v", v[b].view(1, kv, hd))):
                lv, d = ref.quantize(x)
                held[w][b, :, p] = ref.values(ref.pack(lv), d)[0]
            qq = ref.rotate(q[b].view(1, heads, hd), table[p:p + 1], False).double()
            want, _ = ref.attend(qq, held["k"][b], held["v"][b], p, hd ** -0.5)
            want = want.flatten()
            assert float((att[b].double() - want).abs().max()) <= 1e-5 * float(held["v"][b].abs().max())
            ref_logits = Wd @ want
            assert float((logits[b].double() - ref_logits).abs().max() / ref_logits.abs().max()) <= REL_TOL
            p64 = torch.log_softmax(logits[b].double(), -1)
            assert abs(float(lp[b]) - float(p64[int(tok[b])])) <= 1e-5
            assert torch.equal(ids[b].long(), torch.sort(logits[b], descending=True, stable=True).indices[:3])
    graph.reset()
    W.free()
