"""How exact the log probabilities and entropies are, against 64 bits: ordinary rows, and rows with a favourite, where a
running reference that lags behind would cost the entropy its last digits.

The bound.  u = 2^-24; g = m - x a token's distance from the row's maximum m, p its probability, S = sum e^-g.  A thread
sums e^d and d e^d, d = x - r, with a reference r that it raises to a chunk's maximum whenever that passes r + 4, so |d|
<= max(4, g), and brings both to m at the end by D = m - r <= g + 4 (T + D S, so D meets the errors of S); h = g + 4
bounds both.  exp2 is off by 4 u at most, always the same way perhaps, and so is the fp32 log2 e, by u / 4 of d.  d and
its product with log2 e are rounded by up to 2 |d| u, each addition of a chain of N = tokens / 512 + 16 by u of its sum.
These roundings go either way: a sum of independent ones within +-c_i passes 6 sqrt(sum c_i^2) with a probability of
3e-8.  Relative to S that is
    E_S = u (sum p (4 + h / 4) + 6 sqrt(sum (p (2 h + 2))^2) + 6 sqrt(N))                       of S, and
    E_T = 2 u (sum p h (4 + h / 4) + 6 sqrt(sum (p h (2 h + 2))^2) + 6 sqrt(N) sum p h)         of T.
A token more than 4 above all others becomes its thread's reference, d = D = 0 and exp2 is exact: h = 0 for it, and
nothing of the sums over p is left.  Then |logprob - exact| <= E_S + u (g + 2 |log S| + |logprob| + 4) and |entropy -
exact| <= E_S + E_T + u (2 |log S| + 4 |T / S| + 4).
"""
from __future__ import annotations

import pytest

import chatnet_b200 as cn  # noqa: F401

torch = pytest.importorskip("torch")
from tests.test_logprobs import run  # noqa: E402

U = 2.0 ** -24


def exact(x):
    """x [rows, n] -> log probabilities, entropies, and what may be off: (for a token at distance g) and of the entropy."""
    x = x.double()
    m = x.amax(-1, keepdim=True)
    g, lp = m - x, torch.log_softmax(x, -1)
    p, log_s = lp.exp(), torch.logsumexp(x - m, -1)
    N = x.shape[-1] / 512 + 16
    gf = torch.where(g.isfinite(), g, 0.0)
    p1 = torch.where((torch.topk(x, 2, -1).values[:, 1:] < m - 4) & (g == 0), 0.0, p)
    h = gf + 4

    def sums(w):  # of p1 w (4 + h / 4) and of its independent part
        return (p1 * w * (4 + h / 4)).sum(-1) + 6 * (p1 * w * (2 * h + 2)).square().sum(-1).sqrt()
    es = U * (sums(1.0) + 6 * N ** 0.5)
    et = 2 * U * (sums(h) + 6 * N ** 0.5 * (p1 * h).sum(-1))
    t = -(p * gf).sum(-1)
    return lp, log_s - t, es[:, None] + U * (g + 2 * log_s[:, None] + lp.abs() + 4), es + et + U * (2 * log_s - 4 * t + 4)


def rows_of(kind, rows, vocab, gen):
    x = torch.randn(rows, vocab, generator=gen, device=gen.device)
    if kind == "ordinary":
        return x * 3
    if kind == "flat":
        return x * 1e-3
    i = torch.arange(rows, device=gen.device)
    if kind in ("early", "late"):  # a favourite 4.5 .. 12 above the rest, in a thread's second 16 tokens or its last
        at = min(4200, vocab // 2) + i * 37 % 3800 % max(vocab - 4200, 400) if kind == "early" else vocab - 1 - i * 37 % 900
        x[i, at] = x.amax(-1) + 4.5 + 7.5 * i / max(rows - 1, 1)
        return x
    if kind == "steps":  # every part a little higher than the one before
        return x + (torch.arange(vocab, device=gen.device) * 16 // vocab).float()
    assert kind == "two"  # two of them, the second 3.9 below
    x[i, vocab - 1 - (i * 37) % 900] = x.amax(-1) + 6
    x[i, vocab // 2] = x.amax(-1) - 3.9
    return x


KINDS = ["ordinary", "flat", "early", "late", "steps", "two"]


def lagging(x, lag):
    """The entropies by fp32 sums of 256 threads, 16 values at a time, whose references move when outgrown by `lag`."""
    rows, vocab = x.shape
    x = torch.nn.functional.pad(x, (0, -vocab % 4096), value=-torch.inf).view(rows, -1, 4, 256, 4)
    m = torch.full((rows, 256), -torch.inf)
    top = m.clone()
    S, T = torch.zeros(2, rows, 256), torch.zeros(2, rows, 256)

    def raised(to):
        nonlocal S, T, m
        d = (m - to).clamp(min=-200.0)
        f = torch.where(m == -torch.inf, 0.0, d.exp())
        T = f * (d.double() * S + T).float()
        S, m = S * f, to

    for c in range(x.shape[1]):
        cm = x[:, c].amax((1, 3))
        top = torch.maximum(top, cm)
        raised(torch.where(cm > m + lag, cm, m))
        for k in range(4):
            for j in range(4):
                d = (x[:, c, k, :, j] - m).clamp(min=-200.0)
                e = torch.exp2(d * 1.4426950408889634)
                S[j & 1] += e
                T[j & 1] = (d.double() * e + T[j & 1]).float()
    raised(top)
    big = m.amax(-1, keepdim=True).double()
    d = m.double() - big
    s, t = S.double().sum(0), T.double().sum(0)
    t, s = (d.exp() * (t + d * s)).sum(-1), (d.exp() * s).sum(-1)
    return s.log() - t / s


def test_the_bound_tells_a_lagging_reference():
    worst = {}
    for kind in KINDS:
        x = rows_of(kind, 128, 32000, torch.Generator().manual_seed(7))
        _, h, _, tol = exact(x)
        worst[kind] = [float(((lagging(x, lag) - h).abs() / tol).max()) for lag in (4.0, 16.0)]
    assert all(w[0] <= 1 for w in worst.values()), worst
    assert worst["early"][1] > 1, worst


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab,top", [(1, 32000, 5), (32, 32000, 0), (64, 151, 3), (400, 32001, 0), (300, 131071, 8)])
def test_values_and_entropies(ctx, rows, vocab, top, kind, half):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(vocab + rows)
    x = rows_of(kind, rows, max(vocab, 1000), gen)[:, -vocab:].contiguous()
    x = x.half() if half else x
    tok = torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    tok[::2] = x[::2].float().argmax(-1).int()
    lp, ent, ids, tlp = run(ctx, x, tok, top)
    for r in range(0, rows, 50):
        want, h, tol, htol = exact(x[r:r + 50])
        t = tok[r:r + 50].long()[:, None]
        assert ((lp[r:r + 50, None].double() - want.gather(1, t)).abs() <= tol.gather(1, t)).all()
        assert ((ent[r:r + 50].double() - h).abs() <= htol).all()
        if top:
            i = ids[r:r + 50].long()
            assert ((tlp[r:r + 50].double() - want.gather(1, i)).abs() <= tol.gather(1, i)).all()
