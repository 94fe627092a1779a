"""How exact the attention over the 4-bit KV cache is, value by value, on ordinary queries and on ones that are hard
to hold in two fp16 halves.

The bound.  With u = 2^-24 and, per position p of a row, B_p = scale * sum |q_e k_pe|: a query entry is carried to
2^-22 of itself (and to 2^-39 of the row's largest entry a, where its low half leaves fp16's range), times a scale
rounded twice (2 u); K's values are exact; hd products are added in fp32, and the exponential's argument is rounded
(hd + 8 u).  So a score is off by at most e_p = (2^-22 + (hd + 10) u) B_p + 2^-39 a * scale * sum |k_pe|, its
exponential by 8 u more, and against that of the heaviest position m the weight w_p by a factor within
exp(+-(e_p + e_m + 16 u)).  That moves an output by at most
    sum_(p != m) (exp(ln w_p + e_p + e_m + 16 u) - w_p) |v_p - o| / max(w_m, sum w_p exp(-(e_p + e_m + 16 u)));
weights times V's scales are carried to 2^-22, and sums (of weights, and of products) run over at most 64 positions
of a tile and then over the tiles: (2^-21 + 2 (136 + positions / 32) u) sum w_p |v_p| more.  That is where the halves
are normal numbers.  Below, they end at 2^-24, where the heaviest weight is 2^9 or more: each of a weight's two halves is
off by 2^-25, times |v|; and where the weight is multiplied by V's scale (in 2^-7 .. 4 here) first, so are the product's
two roundings, times levels of up to 8: positions * w_m (2^-33 max |v| + 2^-30) more.
"""
from __future__ import annotations

import pytest

import chatnet_b200 as cn  # noqa: F401
from tests import _kvq4 as ref

torch = pytest.importorskip("torch")
from tests.test_kvq4 import Box, _gen, _ints  # noqa: E402

U = 2.0 ** -24


def attend_bound(q, k, v, pos, scale):
    """q [n, heads, hd], k / v [kv, positions, hd] in 64 bits: the output and how far off it may be."""
    n, heads, hd = q.shape
    mul, seen = heads // k.shape[0], pos + n
    hidden = torch.arange(seen, device=q.device)[None] > pos + torch.arange(n, device=q.device)[:, None]
    out, tol = torch.empty_like(q), torch.empty_like(q)
    for h in range(heads):
        kk, vv, x = k[h // mul, :seen], v[h // mul, :seen], q[:, h]
        logw = torch.log_softmax((x @ kk.T * scale).masked_fill(hidden, -torch.inf), -1)
        w = logw.exp()
        out[:, h] = w @ vv
        B = x.abs() @ kk.abs().T * scale
        e = (2.0 ** -22 + (hd + 10) * U) * B
        e = e + 2.0 ** -39 * x.abs().amax(-1, keepdim=True) * scale * kk.abs().sum(-1)[None] + 8 * U
        m = logw.argmax(-1, keepdim=True)
        e = (e + e.gather(1, m)).scatter(1, m, 0.0)
        more = (torch.exp((logw + e).clamp(max=0.0)) - w).masked_fill(hidden, 0.0)  # (no weight passes 1)
        least = torch.maximum(w.gather(1, m), (w * torch.exp(-e)).sum(-1, keepdim=True))
        sums = 2.0 ** -21 + 2 * (136 + seen / 32) * U
        for i in range(n):
            off = (vv - out[i, h]).abs()
            tol[i, h] = (more[i] / least[i]) @ off + sums * (w[i] @ vv.abs())
        tol[:, h] += seen * w.gather(1, m) * (2.0 ** -33 * float(vv.abs().max()) + 2.0 ** -30)
    return out, tol


def _rows(shape, gen, ratio=0.0, border=False):
    """Queries: normal, or (border) of one magnitude that fp16 rounds by almost half a step; with a `ratio`, every row's
    entry 5 is that many times the others."""
    dev = gen.device
    x = torch.randn(*shape, generator=gen, device=dev)
    if border:
        x = torch.where(x < 0, -1.0, 1.0) * (1 + 0.95 * 2.0 ** -11)
    if ratio:
        x[..., 5] = ratio
    return x


def _cache_values(shape, gen, hole, above=False):
    """K and V rows as (levels, scales); with `hole`, K's entry 5 is 0, and with `above` no value of K is below 0."""
    made = []
    for w in "kv":
        x = torch.randn(*shape, generator=gen, device=gen.device) * 1.5
        if hole and w == "k":
            x[..., 5] = 0.0
        if above and w == "k":
            x = x.abs()
        made.append(ref.quantize(x))
    return made


# ---- CPU: restated roundings of the queries against the bound --------------------------------------------------------


def _two_halves(x):
    hi = x.half().float()
    return hi.double() + (x - hi).half().double()


def _split(x, how):
    """fp32 rows as the kernels' halves carry them, scaled by a power of two to [2^14, 2^15)."""
    sc = 2.0 ** (14 - torch.floor(torch.log2(x.abs().amax(-1, keepdim=True))))
    y = (x * sc).float()
    if how == "fp16":
        y = y.half().double()
    elif how == "row":  # a high half in steps of 16 on the row's scale
        hi = torch.round(y / 16) * 16
        y = hi.double() + (y - hi).half().double()
    else:
        y = _two_halves(y)
    return y / sc.double()


@pytest.mark.parametrize("hd", [64, 128])
def test_the_bound_tells_lost_bits(hd):
    """Halves of each entry stay within the bound; a dropped low half does not on ordinary queries, nor a high half on
    the row's scale where one entry is large."""
    gen = torch.Generator().manual_seed(hd)

    def worst(how, ratio, border):
        (lk, dk), (lv, dv) = _cache_values((2, 40, hd), gen, bool(ratio))
        k, v = ref.values(ref.pack(lk), dk), ref.values(ref.pack(lv), dv)
        q = _rows((8, 4, hd), gen, ratio, border)
        want, tol = attend_bound(q.double(), k, v, 20, hd ** -0.5)
        got, _ = attend_bound(_split(q, how), k, v, 20, hd ** -0.5)
        return float(((got - want).abs() / tol).max())

    cases = [(0.0, False)] + [(r, b) for r in (30.0, 300.0, 1e4, 1e5) for b in (False, True)]
    for ratio, border in cases:
        assert worst("halves", ratio, border) <= 1
    assert worst("fp16", 0.0, False) > 2
    assert worst("row", 1e4, True) > 2 and worst("row", 1e5, True) > 2


def _low_half_dropped(x):
    """64-bit values with 11 bits left, cut off as the high halves are."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.trunc(m * 2048) / 2048, e)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lost", ["weights", "values"])
def test_the_bound_tells_lost_bits_of_weights_and_values(hd, lost):
    """On mild queries, whose scores are off by little, it tells weights or V's values without their low halves."""
    gen = torch.Generator().manual_seed(hd + 1)
    (lk, dk), (lv, dv) = _cache_values((2, 40, hd), gen, False)
    k, v = ref.values(ref.pack(lk), dk), ref.values(ref.pack(lv), dv)
    q = _rows((8, 4, hd), gen).double() * 0.1
    want, tol = attend_bound(q, k, v, 20, hd ** -0.5)
    got = torch.empty_like(want)
    for h in range(4):
        for i in range(8):
            x = k[h // 2, :21 + i] @ q[i, h] * hd ** -0.5
            w, y = torch.exp(x - x.max()), v[h // 2, :21 + i]
            if lost == "weights":
                w, total = _low_half_dropped(w), w.sum()  # (the sum is taken before)
            else:
                y, total = y.half().double(), w.sum()
            got[i, h] = w @ y / total
    assert float(((got - want).abs() / tol).max()) > 2


# ---- GPU -------------------------------------------------------------------------------------------------------------


def check(ctx, hd, kv, mul, ctx_len, n_new, pos, gen, q, hole=False, scale=None, above=False):
    """An attention over a fresh cache against the bound; returns the worst error as a part of it."""
    scale = float(torch.tensor(hd ** -0.5 if scale is None else scale))  # (fp32)
    batch, heads = len(pos), kv * mul
    box = Box(batch, kv, hd, ctx_len)
    for b, p in enumerate(pos):
        n = p + n_new
        for w, (lv, d) in zip("kv", _cache_values((kv, n, hd), gen, hole, above)):
            box.q[w][0][b, :, :n] = ref.pack(lv)
            box.q[w][1][b, :, :n] = d
    out = torch.full((batch, n_new, heads * hd), 7.5, device="cuda")
    p = _ints(pos)
    torch.cuda.synchronize()
    ctx.kvq4_attend_dev(box.cache, q.data_ptr(), out.data_ptr(), p.data_ptr(), batch, heads, n_new=n_new, scale=scale,
                        stream=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    worst = 0.0
    for b in range(batch):
        want, tol = attend_bound(q[b].double().view(n_new, heads, hd), box.values("k", b)[:, :pos[b] + n_new],
                                 box.values("v", b)[:, :pos[b] + n_new], pos[b], scale)
        err = (out[b].double().view(n_new, heads, hd) - want).abs()
        assert not err.isnan().any()
        worst = max(worst, float((err / (tol + 1e-300)).max()))  # (0 / 0: no error)
    return worst


FORMS = [  # hd, kv, mul, ctx_len, n_new, pos: few rows (alone, split), then 128 to a CTA (single CTAs, clusters)
    (128, 2, 8, 256, 1, [60, 0, 7, 200]),
    (64, 4, 4, 256, 3, [60, 100]),
    (96, 2, 3, 136, 2, [90]),
    (32, 3, 4, 264, 1, [263, 31]),
    (256, 1, 4, 136, 5, [40, 100]),
    (128, 1, 8, 4096, 1, [1500]),
    (128, 4, 3, 512, 171, [0, 300, 41, 7, 64, 65, 63, 1]),
    (64, 4, 8, 512, 100, [0, 412, 63, 65]),
    (128, 1, 8, 16384, 20, [900]),
    (64, 4, 8, 16384, 120, [500]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("border", [False, True])
@pytest.mark.parametrize("ratio", [30.0, 300.0, 1e4, 1e5])
@pytest.mark.parametrize("form", FORMS)
def test_queries_with_one_large_entry(ctx, form, ratio, border):
    """Most of a row far below its largest entry, which meets only zeros of K."""
    hd, kv, mul, ctx_len, n_new, pos = form
    gen = _gen(31)
    q = _rows((len(pos), n_new, kv * mul, hd), gen, ratio, border).flatten(2)
    assert check(ctx, hd, kv, mul, ctx_len, n_new, pos, gen, q, hole=True) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("qmul", [0.1, 1.0])
@pytest.mark.parametrize("form", FORMS)
def test_ordinary_queries(ctx, form, qmul):
    hd, kv, mul, ctx_len, n_new, pos = form
    gen = _gen(33)
    q = _rows((len(pos), n_new, kv * mul, hd), gen).flatten(2) * qmul
    assert check(ctx, hd, kv, mul, ctx_len, n_new, pos, gen, q) <= 1


LARGE = [(30.0, None), (1e4, None), (1e6, None), (1e8, None), (3e8, None), (3e9, None), (1e20, None), (1e31, None),
         (1e36, None), (1.0, 1e35), (1e-3, 3e38), (1e20, 1e16), (1e36, 1e-38), (1e-38, 1e36)]


@pytest.mark.gpu
@pytest.mark.parametrize("signs", ["mixed", "below"])
@pytest.mark.parametrize("qmul,scale", LARGE)
@pytest.mark.parametrize("form", FORMS[::2] + FORMS[-1:])
def test_large_scores(ctx, form, qmul, scale, signs):
    """Scores up to 1e37 of either sign, and rows with none above -1e31 or so: the heaviest position's values."""
    hd, kv, mul, ctx_len, n_new, pos = form
    gen = _gen(32)
    q = _rows((len(pos), n_new, kv * mul, hd), gen).flatten(2) * qmul
    assert q.isfinite().all()
    if signs == "below":
        q = -q.abs()
    assert check(ctx, hd, kv, mul, ctx_len, n_new, pos, gen, q, scale=scale, above=signs == "below") <= 1
