"""Log probabilities of tokens, entropies and top alternatives (cn_logprobs_dev): refusals on the CPU, values on the
GPU against torch in 64 bits.

Tolerances, u = 2^-24: x - m is rounded once (u |x - m|); the exponentials are off by at most 4 u each plus u |x - m|
from their argument, and e^d |d| <= 0.37, so S is off by at most (5 + n_terms) u relative, where n_terms <= 4096 adds in
one chain; log S adds 2 u |log S|.  So |logprob error| <= u (|x - m| + 2 |log S| + |logprob| + 5 + 4096), and the
entropy's, with T / S as well, at most three times that with |x - m| weighted by p |x - m|, below 64 u more.
"""
from __future__ import annotations

import ctypes as C

import pytest

import chatnet_b200 as cn
from chatnet_b200 import _native as N

torch = pytest.importorskip("torch")

U = 2.0 ** -24
INVALID, UNSUPPORTED = N.CN_ERR_INVALID_ARG, N.CN_ERR_UNSUPPORTED
_BUF = (C.c_uint8 * 4096)()
_P = (C.addressof(_BUF) + 255) & ~255


def _call(**kw):
    a = dict(ctx=C.cast(_BUF, C.c_void_p), type=cn.TYPE_F32, x=_P, stride=100, rows=2, vocab=100, tok=_P, top=3, lp=_P,
             ent=_P, ids=_P, tlp=_P)
    a.update(kw)
    return N.lib().cn_logprobs_dev(a["ctx"], a["type"], a["x"], a["stride"], a["rows"], a["vocab"], a["tok"], a["top"],
                                   a["lp"], a["ent"], a["ids"], a["tlp"], None)


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(x=0), dict(rows=0), dict(rows=-1), dict(vocab=0),
                                 dict(stride=99), dict(stride=1 << 41), dict(top=-1), dict(top=65),
                                 dict(top=11, vocab=10), dict(tok=0), dict(lp=0), dict(ids=0), dict(top=0),
                                 dict(top=0, ids=0), dict(tok=0, lp=0, ent=0, top=0, ids=0, tlp=0), dict(x=_P + 2),
                                 dict(type=cn.TYPE_F16, x=_P + 1)])
def test_refusals(bad):
    assert _call(**bad) == INVALID
    assert N.last_error()


def test_refuses_other_types():
    assert _call(type=cn.TYPE_Q4_0) == UNSUPPORTED


def run(ctx, x, tokens, top, vocab=None, offset=0, stream=None, entropy=True):
    """x [rows, stride] on the GPU; returns (logprob, entropy, ids, top logprobs)."""
    rows, stride = x.shape
    vocab = vocab or stride
    lp = torch.full((rows,), 7.5, device="cuda")
    ent = torch.full((rows,), 7.5, device="cuda")
    ids = torch.full((rows, max(top, 1)), -7, dtype=torch.int32, device="cuda")
    tlp = torch.full((rows, max(top, 1)), 7.5, device="cuda")
    torch.cuda.synchronize()
    ctx.logprobs_dev(x.data_ptr() + offset * x.element_size(), rows, vocab, tokens.data_ptr(), lp.data_ptr(),
                     ent.data_ptr() if entropy else 0, top, ids.data_ptr() if top else 0, tlp.data_ptr() if top else 0,
                     row_stride=stride, type_=cn.TYPE_F16 if x.dtype == torch.float16 else cn.TYPE_F32,
                     stream=(stream or torch.cuda.current_stream()).cuda_stream)
    torch.cuda.synchronize()
    return lp, ent, ids, tlp


def check(x, tokens, top, got):
    """x [rows, vocab]: every row has a distribution."""
    lp, ent, ids, tlp = got
    xd = x.double()
    p = torch.log_softmax(xd, -1)
    m = xd.amax(-1)
    ls = torch.logsumexp(xd, -1) - m

    def tol(xi, li):
        return U * ((xi - m[:, None]).abs() + 2 * ls.abs()[:, None] + li.abs() + 5 + 4096)
    t = tokens.long()[:, None]
    ok = (t[:, 0] >= 0) & (t[:, 0] < x.shape[1])
    tt = t.clamp(0, x.shape[1] - 1)
    want, xi = p.gather(1, tt), xd.gather(1, tt)
    assert lp[~ok].isnan().all()
    fin = ok & want[:, 0].isfinite()
    assert torch.equal(lp[ok & ~fin].double(), want[:, 0][ok & ~fin])
    assert ((lp.double()[:, None] - want).abs() <= tol(xi, want))[fin].all()
    h = torch.special.entr(p.exp()).sum(-1)
    assert ((ent.double() - h).abs() <= 3 * U * (5 + 4096 + 2 * ls.abs() + 64)).all()
    if top:
        order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(ids.long(), order)
        want, xi = p.gather(1, order), xd.gather(1, order)
        fin = want.isfinite()
        assert torch.equal(tlp[~fin].double(), want[~fin])
        assert ((tlp.double() - want).abs() <= tol(xi, want))[fin].all()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


SHAPES = [(1, 1, 1, 1), (1, 2, 2, 2), (3, 31, 31, 31), (2, 64, 64, 64), (5, 257, 257, 64), (1, 32000, 32000, 5),
          (32, 32000, 32000, 20), (7, 32001, 32003, 64), (3, 131071, 131077, 8), (2, 200003, 200003, 20),
          (300, 1000, 1001, 0), (2, 300000, 300000, 64), (130, 8191, 8192, 32), (1, 4099, 4099, 64), (2, 511, 511, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,vocab,stride,top", SHAPES)
def test_values(ctx, rows, vocab, stride, top, half):
    gen = _gen(vocab + rows)
    x = torch.randn(rows, stride, generator=gen, device="cuda") * 3
    x[:, vocab:] = 1e4  # past the row's end
    x[rows // 2, vocab // 2] += 30.0
    x = x.half() if half else x
    tok = torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tok[0] = vocab // 2
    if rows > 2:
        tok[1], tok[2] = -1, vocab
    check(x[:, :vocab], tok, top, run(ctx, x, tok, top, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
def test_unaligned_rows(ctx, offset, half):
    gen = _gen(offset)
    rows, vocab, stride = 4, 5003, 5011
    x = torch.randn(rows + 1, stride, generator=gen, device="cuda")
    x = x.half() if half else x
    tok = torch.tensor([0, vocab - 1, 7, 4999], dtype=torch.int32, device="cuda")
    flat = x.flatten()[offset:offset + rows * stride].reshape(rows, stride)
    got = run(ctx, x[:rows], tok, 9, vocab, offset)
    check(flat[:, :vocab], tok, 9, got)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 3000, 32000, 131071])
def test_ties_and_masks(ctx, vocab):
    x = torch.zeros(8, vocab, device="cuda")          # row 0: everything equal
    x[1] = -0.0
    x[1, vocab // 2:] = 0.0                           # row 1: -0 and +0 are one value
    x[2] = -torch.inf
    x[2, vocab - 1] = 3.0                             # row 2: one token left
    x[3, ::2] = -torch.inf                            # row 3: ties between masked ones
    x[4] = torch.arange(vocab, device="cuda") % 17    # row 4: many ties
    x[5] = torch.arange(vocab, device="cuda") * -1e-3
    x[6] = torch.arange(vocab, device="cuda") * 1e-3  # the best ones last
    x[7] = torch.finfo(torch.float32).min             # the type's lowest value as a mask
    x[7, 11] = 1.0
    tok = torch.tensor([3, vocab - 1, 0, 1, 16, 0, vocab - 1, 12], dtype=torch.int32, device="cuda")
    for top in (1, 7, 33):
        got = run(ctx, x, tok, top)
        check(x[:7], tok[:7], top, [g[:7] for g in got])
        # row 7: (lowest - 1) is the lowest again in fp32: its log probability is that value
        lp, ent, ids, tlp = (g[7] for g in got)
        assert float(lp) == torch.finfo(torch.float32).min and float(ent) == 0.0
        assert ids[0] == 11 and float(tlp[0]) == 0.0
        assert ids[1:].tolist() == [i for i in range(40) if i != 11][:top - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows", [3, 300])  # a row over several CTAs, and one CTA to a row
def test_rows_that_rise_or_hide_their_best(ctx, rows, half):
    """More candidates than a CTA keeps, and first parts of rows that hold nothing to compare with."""
    vocab = 50001
    i = torch.arange(vocab, device="cuda")
    x = torch.randn(rows, vocab, generator=_gen(11), device="cuda")
    x[0] = (i // 25).float() * 0.01                  # rising
    x[1, :45000] = -torch.inf                        # nothing at first
    x[2] = -torch.inf
    x[2, 49998] = -5.0                               # fewer values than asked for
    x[-1] = torch.where(i < 4096, -1.0, (i % 7).float())
    x = x.half() if half else x
    tok = torch.randint(45000, vocab, (rows,), generator=_gen(12), device="cuda", dtype=torch.int32)
    for top in (1, 20, 64):
        check(x, tok, top, run(ctx, x, tok, top))


@pytest.mark.gpu
def test_rows_without_a_distribution(ctx):
    for vocab in (50, 20000):
        x = torch.randn(4, vocab, generator=_gen(1), device="cuda")
        x[0, 17] = torch.nan
        x[1, 5] = torch.inf
        x[2] = -torch.inf
        tok = torch.tensor([3, 5, 0, 2], dtype=torch.int32, device="cuda")
        lp, ent, ids, tlp = run(ctx, x, tok, 6)
        assert lp[:3].isnan().all() and ent[:3].isnan().all() and tlp[:3].isnan().all()
        assert 17 not in ids[0].tolist() and ids[1, 0] == 5 and ids[2].tolist() == [0, 1, 2, 3, 4, 5]
        best = torch.sort(x[0].nan_to_num(nan=-torch.inf), descending=True, stable=True).indices[:6]
        assert torch.equal(ids[0].long(), best)
        check(x[3:], tok[3:], 6, [g[3:] for g in (lp, ent, ids, tlp)])
        few = torch.full((1, 3), torch.nan, device="cuda")
        few[0, 1] = -1.0
        assert run(ctx, few, tok[:1], 3)[2][0].tolist() == [1, 0, 2]  # NaN last, by index


@pytest.mark.gpu
def test_outputs_are_optional(ctx):
    x = torch.randn(3, 1000, generator=_gen(2), device="cuda")
    tok = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    full = run(ctx, x, tok, 4)
    ent = torch.zeros(3, device="cuda")
    ids = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    lp = torch.zeros(3, device="cuda")
    torch.cuda.synchronize()
    ctx.logprobs_dev(x.data_ptr(), 3, 1000, entropy=ent.data_ptr())
    ctx.logprobs_dev(x.data_ptr(), 3, 1000, top_n=4, top_ids=ids.data_ptr())
    ctx.logprobs_dev(x.data_ptr(), 3, 1000, tok.data_ptr(), lp.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(ent, full[1]) and torch.equal(ids, full[2]) and torch.equal(lp, full[0])


@pytest.mark.gpu
def test_streams_and_graphs(ctx):
    gen = _gen(3)
    x = torch.randn(16, 32000, generator=gen, device="cuda") * 3
    tok = torch.randint(32000, (16,), generator=gen, device="cuda", dtype=torch.int32)
    want = run(ctx, x, tok, 20)
    outs = [[torch.empty_like(w) for w in want] for _ in range(4)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(o, stream):
        ctx.logprobs_dev(x.data_ptr(), 16, 32000, tok.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), 20,
                         o[2].data_ptr(), o[3].data_ptr(), stream=stream.cuda_stream)
    for _ in range(10):
        call(outs[0], s1)
        call(outs[1], s2)
    graphs = []
    for k in (2, 3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(outs[k], torch.cuda.current_stream())
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_past_32_bits(ctx):
    """Logits of more than 2^32 bytes."""
    rows, vocab = 10000, 131071
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    x = torch.zeros(rows, vocab, device="cuda")
    x[-3:] = torch.randn(3, vocab, generator=_gen(4), device="cuda")
    tok = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    got = run(ctx, x, tok, 3)
    check(x[-3:], tok[-3:], 3, [g[-3:] for g in got])
    assert got[2][:-3].tolist() == [[0, 1, 2]] * (rows - 3)
