"""The 4-bit KV cache (cn_kvq4_*): the layout and the refusals on the CPU; append, read and attention on the GPU
against a plain restatement in 64 bits.

Tolerances of the attention.  With u = 2^-24 (half a step of fp32), a score is a sum of hd products of q, carried in
22 bits (error <= 2^-22 relative), and exact levels, in fp32: its error is at most ds = (2^-22 + (hd + 8) u) * B, B =
scale * sum |q_e k_e|; the exponential adds 4 u |argument| <= 8 u B + 4 u.  Every weight is off by a factor e^(+-D), D
= 2 ds + 8 u B + 4 u, carried in 22 bits into the sum over at most `len` positions, so
|out - exact| <= (2 D + 2^-21 + 2 (len + 64) u) * max |v|.
"""
from __future__ import annotations

import ctypes as C

import pytest

import chatnet_b200 as cn
from chatnet_b200 import _native as N
from tests import _kvq4 as ref

torch = pytest.importorskip("torch")

INVALID, UNSUPPORTED = N.CN_ERR_INVALID_ARG, N.CN_ERR_UNSUPPORTED


# ---- CPU: the restatement's layout, and refusals (which return before any device is touched) ------------------------


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256])
def test_layout_is_a_bijection(hd):
    byte, shift = ref.positions_of(hd)
    assert sorted((byte * 2 + shift // 4).tolist()) == list(range(hd))
    lv = torch.randint(0, 16, (5, hd), generator=torch.Generator().manual_seed(hd), dtype=torch.uint8)
    assert torch.equal(ref.unpack(ref.pack(lv)).to(torch.uint8), lv)
    # a chunk (2 * nb bytes) holds the dimensions e = g mod 8
    assert all(int(b) // (hd // 16) == e % 8 for e, b in enumerate(byte))


def test_quantize_rule():
    x = torch.zeros(1, 32)
    x[0, :4] = torch.tensor([-4.0, 4.0, 0.25, -0.25])  # a tie of magnitudes: the negative one sets the scale
    q, d = ref.quantize(x)
    assert float(d[0, 0]) == 0.5 and q[0, :4].tolist() == [0, 15, 9, 8]  # halves up: 8.5 + 0.5 = 9, 8.5 - 0.5 = 8


_BUF = (C.c_uint8 * 65536)()
_P = (C.addressof(_BUF) + 255) & ~255
_CTX = C.cast(_BUF, C.c_void_p)


def _cache(**kw):
    d = dict(k_quants=_P, k_scales=_P, v_quants=_P, v_scales=_P, n_seqs=4, n_kv_heads=2, head_dim=64, ctx_len=64,
             seq_rows=0)
    return N.KvQ4C(**{**d, **kw})


def _append(cache=None, **kw):
    a = dict(ctx=_CTX, k=_P, v=_P, stride=128, pos=_P, count=0, batch=1, n_new=1, rope=0, neox=0)
    a.update(kw)
    return N.lib().cn_kvq4_append_dev(a["ctx"], C.byref(cache or _cache()), a["k"], a["v"], a["stride"], a["pos"],
                                      a["count"], a["batch"], a["n_new"], a["rope"], a["neox"], None)


def _read(**kw):
    a = dict(k=_P, v=_P, stride=128, pos=_P, batch=1, n_new=1)
    a.update(kw)
    return N.lib().cn_kvq4_read_dev(_CTX, C.byref(_cache()), a["k"], a["v"], a["stride"], a["pos"], 0, a["batch"],
                                    a["n_new"], None)


def _attend(cache=None, **kw):
    a = dict(ctx=_CTX, q=_P, qs=256, out=_P, os=256, pos=_P, batch=1, n_new=1, heads=4, scale=0.125, rope=0, neox=0)
    a.update(kw)
    return N.lib().cn_kvq4_attend_dev(a["ctx"], C.byref(cache or _cache()), a["q"], a["qs"], a["out"], a["os"],
                                      a["pos"], 0, a["batch"], a["n_new"], a["heads"], a["scale"], a["rope"],
                                      a["neox"], None)


BAD_CACHES = [(dict(head_dim=80), UNSUPPORTED), (dict(head_dim=512), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
              (dict(ctx_len=60), INVALID), (dict(ctx_len=0), INVALID), (dict(n_kv_heads=0), INVALID),
              (dict(n_seqs=0), INVALID), (dict(seq_rows=64), INVALID), (dict(seq_rows=132), INVALID),
              (dict(seq_rows=-8), INVALID), (dict(seq_rows=1 << 41), INVALID), (dict(k_quants=0), INVALID),
              (dict(v_scales=0), INVALID), (dict(k_scales=_P + 8), INVALID), (dict(v_quants=_P + 4), INVALID)]


@pytest.mark.parametrize("bad,code", BAD_CACHES)
def test_bad_caches_are_refused(bad, code):
    assert _append(_cache(**bad)) == code and _attend(_cache(**bad)) == code
    assert N.last_error()


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(k=0), dict(v=0), dict(pos=0), dict(stride=127), dict(batch=0),
                                 dict(batch=5), dict(n_new=0), dict(n_new=65), dict(neox=2), dict(k=_P + 2),
                                 dict(rope=_P + 4)])
def test_bad_appends_are_refused(bad):
    assert _append(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(k=0, v=0), dict(pos=0), dict(stride=64), dict(batch=5), dict(n_new=0),
                                 dict(v=_P + 1)])
def test_bad_reads_are_refused(bad):
    assert _read(**bad) == INVALID


@pytest.mark.parametrize("bad", [dict(ctx=None), dict(q=0), dict(out=0), dict(pos=0), dict(heads=0), dict(heads=3),
                                 dict(heads=-2), dict(qs=252), dict(qs=258), dict(os=128), dict(q=_P + 4),
                                 dict(out=_P + 8), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(batch=0), dict(batch=5), dict(n_new=65),
                                 dict(neox=-1), dict(rope=_P + 4),
                                 dict(heads=1 << 26, n_new=64, qs=1 << 33, os=1 << 33)])
def test_bad_attends_are_refused(bad):
    assert _attend(**bad) == INVALID


def test_python_wrappers_raise():
    class Fake(cn.Context):
        def __init__(self):
            self.handle = _CTX

        def close(self):
            pass
    cache = cn.KvQ4Cache(_P, _P, _P, _P, 4, 2, 64, 64)
    bad = cn.KvQ4Cache(_P, _P, _P, _P, 4, 2, 80, 64)
    with pytest.raises(ValueError):
        Fake().kvq4_append_dev(cache, 0, _P, _P, 1)
    with pytest.raises(cn.NotSupportedError):
        Fake().kvq4_read_dev(bad, _P, _P, _P, 1)
    with pytest.raises(ValueError):
        Fake().kvq4_attend_dev(cache, _P, _P, _P, 1, 3)


# ---- GPU ------------------------------------------------------------------------------------------------------------


class Box:
    """A cache on the GPU whose unwritten rows hold poison: levels 15 and NaN scales."""

    def __init__(self, n_seqs, kv, hd, ctx_len, layers=1, layer=0):
        self.n_seqs, self.kv, self.hd, self.ctx_len = n_seqs, kv, hd, ctx_len
        shape = (n_seqs, layers, kv, ctx_len)
        self.full = {w: (torch.full((*shape, hd // 2), 255, dtype=torch.uint8, device="cuda"),
                         torch.full((*shape, hd // 32), torch.nan, dtype=torch.float16, device="cuda")) for w in "kv"}
        self.q = {w: tuple(t[:, layer] for t in self.full[w]) for w in "kv"}
        (kq, kd), (vq, vd) = self.q["k"], self.q["v"]
        self.cache = cn.KvQ4Cache(kq.data_ptr(), kd.data_ptr(), vq.data_ptr(), vd.data_ptr(), n_seqs, kv, hd, ctx_len,
                                  layers * kv * ctx_len)

    def fill(self, seq, n, gen):
        """Positions 0..n-1 of a sequence from random rows."""
        for w in "kv":
            x = torch.randn(self.kv, n, self.hd, generator=gen, device="cuda") * 1.5
            lv, d = ref.quantize(x)
            self.q[w][0][seq, :, :n] = ref.pack(lv)
            self.q[w][1][seq, :, :n] = d

    def values(self, w, seq):
        return ref.values(self.q[w][0][seq], self.q[w][1][seq])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


APPENDS = [  # hd, kv, batch, n_new, pos, count, rope, neox, extra stride
    (32, 1, 1, 1, [0], None, False, False, 0), (64, 4, 3, 1, [0, 511, 17], None, True, False, 0),
    (96, 3, 2, 5, [9, 100], [5, 2], True, True, 3), (128, 8, 4, 7, [-1, 505, 511, 600], [7, 7, 7, 7], True, False, 1),
    (128, 2, 2, 64, [448, 0], [0, -3], False, False, 0), (256, 2, 2, 33, [1, 490], None, True, True, 8),
    (64, 5, 2, 300, [100, 3], [300, 299], True, True, 0), (32, 2, 1, 9, [2], None, True, True, 0),
    (32, 3, 1, 9, [2], None, True, False, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kv,batch,n_new,pos,count,rope,neox,extra", APPENDS)
def test_append_and_read(ctx, hd, kv, batch, n_new, pos, count, rope, neox, extra):
    gen, ctx_len = _gen(hd + n_new), 512
    box = Box(batch, kv, hd, ctx_len, layers=2, layer=1)
    before = {w: [t.clone() for t in box.full[w]] for w in "kv"}
    stride = kv * hd + extra
    x = {w: torch.randn(batch, n_new, stride, generator=gen, device="cuda") * 3 for w in "kv"}
    # halfway values (levels' borders), a constant row and a row of zeros
    x["v"][0, 0, :32] = torch.arange(32, device="cuda") * 0.25 - 4.0
    x["v"][-1, -1, :kv * hd] = 0.0
    x["k"][-1, 0, :kv * hd] = 1.0
    table = ref.rope_table(ctx_len, hd).cuda() if rope else None
    p, c = _ints(pos), _ints(count) if count else None
    args = dict(count=c.data_ptr() if count else 0, kv_stride=stride, stream=torch.cuda.current_stream().cuda_stream)
    ctx.kvq4_append_dev(box.cache, x["k"].data_ptr(), x["v"].data_ptr(), p.data_ptr(), batch, n_new,
                        rope=table.data_ptr() if rope else 0, rope_neox=neox, **args)
    got = {w: torch.full((batch, n_new, stride), 7.5, device="cuda") for w in "kv"}
    ctx.kvq4_read_dev(box.cache, got["k"].data_ptr(), got["v"].data_ptr(), p.data_ptr(), batch, n_new, **args)
    torch.cuda.synchronize()
    for w in "kv":
        want_q, want_d = (t.clone() for t in before[w])
        want_read = torch.full((batch, n_new, stride), 7.5, device="cuda")
        for b in range(batch):
            n = min(count[b] if count else n_new, n_new, ctx_len - pos[b]) if 0 <= pos[b] < ctx_len else 0
            if n <= 0:
                continue
            rows = x[w][b, :n, :kv * hd].reshape(n, kv, hd)
            if rope and w == "k":
                rows = ref.rotate(rows, table[pos[b]:pos[b] + n], neox)
            lv, d = ref.quantize(rows)
            want_q[b, 1, :, pos[b]:pos[b] + n] = ref.pack(lv).transpose(0, 1)
            want_d[b, 1, :, pos[b]:pos[b] + n] = d.transpose(0, 1)
            want_read[b, :n, :kv * hd] = ref.values(ref.pack(lv), d, torch.float32).flatten(1)
        assert torch.equal(box.full[w][0], want_q)
        assert torch.equal(box.full[w][1].view(torch.int16), want_d.view(torch.int16))
        assert torch.equal(got[w], want_read)


@pytest.mark.gpu
def test_append_extreme_values(ctx):
    """Infinities, NaN, values whose scale over- or underflows fp16."""
    box = Box(1, 1, 64, 16)
    rows = torch.zeros(12, 64, device="cuda")
    rows[0, 3], rows[0, 5] = torch.inf, -1.0
    rows[1, 0], rows[1, 1] = -torch.inf, 3e38
    rows[2, :] = torch.nan
    rows[3, 7], rows[3, 8] = torch.nan, 2.0
    rows[4, :] = 1e-8
    rows[5, :] = 1e-40
    rows[6, 0] = 4.8e-7      # scale 2^-24, the smallest
    rows[7, :] = 6e5
    rows[8, :] = torch.linspace(-1, 1, 64, device="cuda")
    rows[9, :] = -0.0
    rows[10, 32:] = torch.linspace(-3e-5, 2e-5, 32, device="cuda")
    rows[11, :32] = torch.tensor([8.0] + [k - 7.5 for k in range(16)] + [0.5] * 15, device="cuda")  # negative scale
    p = _ints([2])
    ctx.kvq4_append_dev(box.cache, rows.data_ptr(), rows.data_ptr(), p.data_ptr(), 1, 12)
    torch.cuda.synchronize()
    lv, d = ref.quantize(rows)
    for w in "kv":
        assert torch.equal(ref.unpack(box.q[w][0][0, 0, 2:14]).to(torch.uint8), lv)
        assert torch.equal(box.q[w][1][0, 0, 2:14], d)
        assert torch.isfinite(box.values(w, 0)[0, 2:14]).all()


def _check_attend(ctx, box, batch, heads, n_new, pos, count, table, neox, gen, scale=None, q_extra=0, out_extra=0,
                  stream=None, qmul=1.0):
    hd, kv = box.hd, box.kv
    scale = hd ** -0.5 if scale is None else scale
    q = torch.randn(batch, n_new, heads * hd + q_extra, generator=gen, device="cuda") * qmul
    out = torch.full((batch, n_new, heads * hd + out_extra), 7.5, device="cuda")
    p, c = _ints(pos), _ints(count) if count else None
    torch.cuda.synchronize()
    s = (stream or torch.cuda.current_stream()).cuda_stream
    ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), batch, heads, n_new=n_new,
                        count=c.data_ptr() if count else 0, q_stride=heads * hd + q_extra,
                        out_stride=heads * hd + out_extra, scale=scale, rope=table.data_ptr() if table is not None else 0,
                        rope_neox=neox, stream=s)
    torch.cuda.synchronize()
    verify(box, q, out, heads, n_new, pos, count, table, neox, scale)
    return out


def verify(box, q, out, heads, n_new, pos, count, table, neox, scale):
    hd, u = box.hd, 2.0 ** -24
    width = heads * hd
    for b in range(len(pos)):
        n = min(count[b] if count else n_new, n_new, box.ctx_len - pos[b]) if 0 <= pos[b] < box.ctx_len else 0
        n = max(n, 0)
        assert (out[b, n:] == 7.5).all() and (out[b, :, width:] == 7.5).all()  # left as they were
        if n == 0:
            continue
        x = q[b, :n, :width].reshape(n, heads, hd)
        if table is not None:
            x = ref.rotate(x, table[pos[b]:pos[b] + n], neox)
        k, v = box.values("k", b), box.values("v", b)
        want, size = ref.attend(x.double(), k, v, pos[b], scale)
        B = float(size.max())
        ds = (2.0 ** -22 + (hd + 8) * u) * B
        D = 2 * ds + 8 * u * B + 4 * u
        seen = pos[b] + n
        tol = (2 * D + 2.0 ** -21 + 2 * (seen + 64) * u) * float(v[:, :seen].abs().max())
        err = (out[b, :n, :width].double().view(n, heads, hd) - want).abs().max()
        assert float(err) <= tol, (b, float(err), tol)


ATTENDS = [  # hd, kv, mul, ctx_len, n_new, pos, count, rope, neox
    (64, 4, 8, 64, 1, [0], None, False, False),
    (64, 4, 8, 2048, 1, [512], None, True, False),
    (128, 8, 8, 2048, 1, [2047, 0, 1, 15, 16, 17, 31, 1000], None, True, False),
    (128, 8, 8, 2048, 1, [-1, 2048, 63, 64], [1, 1, 0, 1], False, False),
    (128, 32, 1, 1024, 1, [1001, 7, 500], None, True, True),
    (96, 2, 3, 136, 1, [135, 100, 8], None, True, False),
    (32, 3, 4, 264, 1, [263, 31, 32, 33], None, True, True),
    (256, 2, 8, 520, 1, [519, 255], None, True, False),
    (256, 1, 1, 72, 3, [69, 0], None, True, True),
    (64, 1, 71, 264, 1, [200, 3], None, False, False),
    (128, 2, 12, 512, 1, [300], None, True, False),
    (128, 1, 16, 4096, 2, [4000, 4094, 4095], None, False, False),
    (128, 8, 8, 1024, 5, [1000, 0, 1021, 300], [5, 1, 5, 4], True, False),
    (64, 2, 4, 256, 16, [0, 240, 100], None, True, True),
    (64, 2, 4, 256, 17, [3, 250, 100], [17, 17, 9], True, False),
    (128, 2, 8, 512, 65, [0, 131, 440], None, True, False),
    (128, 4, 1, 512, 130, [0, 382], [130, 127], True, False),
    (96, 2, 3, 512, 67, [5, 300], None, True, True),
    (32, 1, 8, 512, 40, [0, 470], None, False, False),
    (256, 1, 4, 512, 50, [0, 123], None, True, False),
    (128, 1, 8, 16384, 1, [16001], None, False, False),
    (128, 1, 1, 8192, 33, [8000], None, False, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kv,mul,ctx_len,n_new,pos,count,rope,neox", ATTENDS)
def test_attend(ctx, hd, kv, mul, ctx_len, n_new, pos, count, rope, neox):
    gen = _gen(hd * 1000 + n_new)
    box = Box(len(pos), kv, hd, ctx_len)
    for b, p in enumerate(pos):
        if p >= 0:
            box.fill(b, min(ctx_len, p + n_new), gen)
    table = ref.rope_table(ctx_len, hd).cuda() if rope else None
    _check_attend(ctx, box, len(pos), mul * kv, n_new, pos, count, table, neox, gen)


PROMPTS = [  # sizes at which rows go 128 to a CTA: single CTAs (the first four), then clusters
    (128, 8, 8, 512, 64, [0, 1, 63, 448], None, True, False),
    (128, 4, 3, 512, 171, [0, 300, 341, -1, 511, 7, 600, 64], [171, 171, 170, 9, 171, 1, 171, 0], True, True),
    (64, 4, 8, 512, 100, [0, 412, 63, 65], None, True, False),
    (64, 1, 71, 2048, 40, [2008, 0, 1000, 24, 23, 2047], None, False, False),
    (128, 8, 8, 8192, 120, [8000], None, True, False),
    (128, 4, 8, 16384, 90, [16001, 6], [90, 77], False, False),
    (64, 4, 8, 16384, 120, [16002], None, True, True),
    (64, 8, 4, 32768, 33, [30001], None, True, True),
    (128, 1, 8, 16384, 130, [16254, 5], [130, 127], True, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,kv,mul,ctx_len,n_new,pos,count,rope,neox", PROMPTS)
def test_attend_prompts(ctx, hd, kv, mul, ctx_len, n_new, pos, count, rope, neox):
    gen = _gen(hd * 1000 + n_new + 1)
    box = Box(len(pos), kv, hd, ctx_len)
    for b, p in enumerate(pos):
        if p >= 0:
            box.fill(b, min(ctx_len, p + n_new), gen)
    table = ref.rope_table(ctx_len, hd).cuda() if rope else None
    _check_attend(ctx, box, len(pos), mul * kv, n_new, pos, count, table, neox, gen, q_extra=4, out_extra=8)


# one token, a few, a prompt of 128 rows to a CTA (8 sequences: rows enough)
FORMS = [(1, 1), (1, 24), (8, 130)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,n_new", FORMS)
def test_attend_peaked_and_flat_prompts(ctx, hd, batch, n_new):
    """As test_attend_peaked_and_flat, and with products of q and scale below fp32's normal range."""
    gen = _gen(16)
    for mul, scale in ((300.0, None), (1e4, None), (0.0, None), (1e-30, None), (1e-40, 1e-20), (1e-3, 1e-38)):
        box = Box(batch, 4, hd, 512)
        for b in range(batch):
            box.fill(b, 512, gen)
        pos = [(37 * b) % 300 for b in range(batch)]
        _check_attend(ctx, box, batch, 16, n_new, pos, None, None, False, gen, qmul=mul, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,n_new", FORMS)
@pytest.mark.parametrize("lowest", [-20, 0, 10])
def test_attend_scale_ranges(ctx, hd, batch, n_new, lowest):
    """Scales of either sign, zero, and powers of two times [1, 2) up to 2^15 for K and V, tile by tile and mixed (a
    block's values reach 8 * 60000); q small enough for the scores to differ by a few."""
    gen = _gen(17)
    box = Box(batch, 4, hd, 512)
    for b in range(batch):
        box.fill(b, 512, gen)
    for w in "kv":
        shape = box.q[w][1].shape
        e = torch.randint(lowest, 16, shape, generator=gen, device="cuda")
        e[:, :, 64:128] = lowest                             # a tile without large ones
        d = 2.0 ** e * (1 + torch.rand(shape, generator=gen, device="cuda") * 0.8)
        d = d * torch.randint(-1, 2, shape, generator=gen, device="cuda")
        box.q[w][1].copy_(d.half())
    pos = [(37 * b) % 300 for b in range(batch)]
    _check_attend(ctx, box, batch, 16, n_new, pos, None, None, False, gen, qmul=1e-5)


@pytest.mark.gpu
def test_attend_lone_nan_and_infinite_queries(ctx):
    """A row whose query is not finite leaves the rows beside it alone."""
    for batch, n_new in FORMS:
        gen = _gen(18)
        box = Box(batch, 4, 128, 512)
        for b in range(batch):
            box.fill(b, 512, gen)
        heads, hd = 16, 128
        q = torch.randn(batch, n_new, heads * hd, generator=gen, device="cuda")
        clean, out = (torch.full_like(q, 7.5) for _ in range(2))
        p = _ints([200] * batch)
        s = torch.cuda.current_stream().cuda_stream
        ctx.kvq4_attend_dev(box.cache, q.data_ptr(), clean.data_ptr(), p.data_ptr(), batch, heads, n_new=n_new, stream=s)
        q[0, 0, 3 * hd + 5], q[-1, -1, 9 * hd] = torch.nan, torch.inf
        ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), batch, heads, n_new=n_new, stream=s)
        torch.cuda.synchronize()
        x, y = (t.view(batch, n_new, heads, hd) for t in (out, clean))
        assert x[0, 0, 3].isnan().all() and x[-1, -1, 9].isnan().all()
        x[0, 0, 3], x[-1, -1, 9] = y[0, 0, 3], y[-1, -1, 9]
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_attend_strides_layers_and_scale(ctx):
    gen = _gen(5)
    for n_new in (1, 20):
        box = Box(3, 2, 128, 256, layers=3, layer=1)
        for b in range(3):
            box.fill(b, 256, gen)
        _check_attend(ctx, box, 2, 8, n_new, [100, 236], None, None, False, gen, scale=0.5, q_extra=12, out_extra=4)


@pytest.mark.gpu
def test_attend_peaked_and_flat(ctx):
    """Large queries (one position takes everything), tiny ones, and zero (the mean of the values)."""
    gen = _gen(6)
    for n_new in (1, 24):
        for mul in (300.0, 1e-30, 0.0, 1e4):
            box = Box(2, 2, 64, 128)
            for b in range(2):
                box.fill(b, 128, gen)
            _check_attend(ctx, box, 2, 8, n_new, [100, 90], None, None, False, gen, qmul=mul)


@pytest.mark.gpu
def test_attend_zero_scales_and_wide_range(ctx):
    """Rows with scale 0, scales from 2^-24 to 60000 and negative ones."""
    gen = _gen(7)
    for n_new in (1, 24):
        box = Box(1, 1, 128, 256)
        box.fill(0, 256, gen)
        d = 2.0 ** (torch.rand(1, 256, 4, generator=gen, device="cuda") * 24 - 20)
        d = d * (torch.randint(0, 3, (1, 256, 4), generator=gen, device="cuda") - 1)
        box.q["v"][1][0] = d.half()
        box.q["k"][1][0, :, ::3] = 0
        _check_attend(ctx, box, 1, 4, n_new, [200], None, None, False, gen)


@pytest.mark.gpu
def test_attend_is_deterministic_on_streams_and_in_graphs(ctx):
    gen = _gen(8)
    box = Box(4, 8, 128, 2048)
    pos = [2000, 77, 1500, 3]
    for b, p in enumerate(pos):
        box.fill(b, p + 1, gen)
    heads, hd = 64, 128
    q = torch.randn(4, 1, heads * hd, generator=gen, device="cuda")
    outs = [torch.full((4, 1, heads * hd), 7.5, device="cuda") for _ in range(5)]
    p = _ints(pos)
    torch.cuda.synchronize()

    def call(out, stream):
        ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), 4, heads, stream=stream.cuda_stream)

    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):  # two calls at once
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
    call(outs[4], torch.cuda.current_stream())
    torch.cuda.synchronize()
    verify(box, q, outs[0], heads, 1, pos, None, None, False, hd ** -0.5)
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    # new inputs and positions in place: the captured call reads them
    q.mul_(0.5)
    p.copy_(_ints([100, 10, 1400, 2]))
    for o in outs:
        o.fill_(7.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    verify(box, q, outs[2], heads, 1, [100, 10, 1400, 2], None, None, False, hd ** -0.5)


@pytest.mark.gpu
def test_prompts_on_streams_and_in_graphs(ctx):
    """Two prompt calls at once, captured ones replayed at once and with new inputs; single CTAs and clusters."""
    for kv, ctx_len, pos, n_new in ((8, 512, [0, 300, 64], 128), (1, 16384, [16000], 130)):
        gen, hd, heads, batch = _gen(19), 128, 8 * kv, len(pos)
        box = Box(batch, kv, hd, ctx_len)
        for b, x in enumerate(pos):
            box.fill(b, x + n_new, gen)
        q = torch.randn(batch, n_new, heads * hd, generator=gen, device="cuda")
        outs = [torch.full_like(q, 7.5) for _ in range(4)]
        p = _ints(pos)
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()

        def call(out, stream):
            ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), batch, heads, n_new=n_new,
                                stream=stream.cuda_stream)

        for _ in range(5):
            call(outs[0], s1)
            call(outs[1], s2)
        graphs = []
        for k in (2, 3):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call(outs[k], torch.cuda.current_stream())
            graphs.append(g)
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, (s1, s2)):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        verify(box, q, outs[0], heads, n_new, pos, None, None, False, hd ** -0.5)
        for o in outs[1:]:
            assert torch.equal(o, outs[0])
        q.mul_(0.5)
        lower = [max(x - 1, 0) for x in pos]
        p.copy_(_ints(lower))
        outs[3].fill_(7.5)
        graphs[1].replay()
        torch.cuda.synchronize()
        verify(box, q, outs[3], heads, n_new, lower, None, None, False, hd ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,n_new", FORMS)
def test_a_contexts_first_call_is_captured(batch, n_new):
    gen = _gen(20)
    box = Box(batch, 4, 64, 512)
    for b in range(batch):
        box.fill(b, 512, gen)
    q = torch.randn(batch, n_new, 16 * 64, generator=gen, device="cuda")
    out = torch.full_like(q, 7.5)
    pos = [100] * batch
    p = _ints(pos)
    torch.cuda.synchronize()
    with cn.Context(0) as fresh:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fresh.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), batch, 16, n_new=n_new,
                                  stream=torch.cuda.current_stream().cuda_stream)
        g.replay()
        torch.cuda.synchronize()
        verify(box, q, out, 16, n_new, pos, None, None, False, 0.125)
        g.reset()


@pytest.mark.gpu
def test_attend_offsets_past_32_bits(ctx):
    """A cache whose quants exceed 2^32 bytes: the last sequence's rows, and the first one's after them."""
    kv, hd, ctx_len = 8, 128, 1 << 20
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    n_seqs = 9  # 9 * 8 * 2^20 rows * 64 bytes = 4.8e9 per array
    gen = _gen(9)
    box = Box(n_seqs, kv, hd, ctx_len)
    pos = [-1] * n_seqs
    pos[0], pos[-1] = 300, ctx_len - 1
    box.fill(0, 301, gen)
    for w in "kv":  # the long one: a repeated block of rows
        lv, d = ref.quantize(torch.randn(kv, 4096, hd, generator=gen, device="cuda"))
        box.q[w][0][-1] = ref.pack(lv).repeat(1, ctx_len // 4096, 1)
        box.q[w][1][-1] = d.repeat(1, ctx_len // 4096, 1)
    # (the exact reference of 2^20 repeated rows is that of one period, each weight counted alike)
    q = torch.randn(n_seqs, 1, kv * hd, generator=gen, device="cuda")
    out = torch.full((n_seqs, 1, kv * hd), 7.5, device="cuda")
    p = _ints(pos)
    torch.cuda.synchronize()
    ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), n_seqs, kv)
    torch.cuda.synchronize()
    assert (out[1:-1] == 7.5).all()
    k = ref.values(box.q["k"][0][-1, :, :4096], box.q["k"][1][-1, :, :4096])
    v = ref.values(box.q["v"][0][-1, :, :4096], box.q["v"][1][-1, :, :4096])
    want, size = ref.attend(q[-1].double().view(1, kv, hd), k, v, 4095, hd ** -0.5)
    u, B = 2.0 ** -24, float(size.max())
    D = 2 * (2.0 ** -22 + (hd + 8) * u) * B + 8 * u * B + 4 * u
    # (2^20 positions, summed in at most 2^13 runs of at most 2^13 terms each)
    tol = (2 * D + 2.0 ** -21 + 2 * (2 ** 14 + 64) * u) * float(v.abs().max())
    assert float((out[-1].double().view(1, kv, hd) - want).abs().max()) <= tol
    k0, v0 = (ref.values(box.q[w][0][0, :, :301], box.q[w][1][0, :, :301]) for w in "kv")
    want, _ = ref.attend(q[0].double().view(1, kv, hd), k0, v0, 300, hd ** -0.5)
    assert float((out[0].double().view(1, kv, hd) - want).abs().max()) <= tol
