"""Cases and plain forms of the serving operators: the 4-bit KV cache (append, attend) and token log probabilities.

`run` computes an operator in elementary torch operations, or, where `own` is set, through chatnet_b200's entry
points.  Every input is made on the GPU from the seed.

The 4-bit cache of one layer holds, per (sequence, kv head, position), a row of head_dim values in blocks of 32:
value 32 b + 8 i + g of a row (block b, i < 4, g < 8) is the nibble i & 1 (low first) of byte g * 2 * nb + 2 * b +
(i >> 1), nb = head_dim / 32, and stands for scale[b] * (nibble - 8) with an fp16 scale per block.
"""
import math

import torch

own = False

_CLAMP = 524032.0  # 8 * the largest fp16 value: block maxima above it would overflow the fp16 scale
_contexts = {}


def listed():
    return [
        # one sequence's decode step, 22-layer 1.1B-shaped decoder (32/4 heads of 64): one layer at position 512
        {"name": "attend-one-512", "op": "attend", "heads": 32, "kv": 4, "hd": 64, "batch": 1, "new": 1, "top": 512,
         "ctx": 2048, "rope": True, "neox": False},
        # sixteen requests decoding together on a 70B-shaped layer (64/8 heads of 128), context 2048
        {"name": "attend-batch16-2047", "op": "attend", "heads": 64, "kv": 8, "hd": 128, "batch": 16, "new": 1,
         "top": 2047, "ctx": 2048, "rope": True, "neox": False},
        # a full batch on a layer without grouped heads (32/32 of 128), ragged odd lengths
        {"name": "attend-mha-batch32-1001", "op": "attend", "heads": 32, "kv": 32, "hd": 128, "batch": 32, "new": 1,
         "top": 1001, "ctx": 1024, "rope": True, "neox": False},
        # long documents: eight requests with up to 131 thousand positions
        {"name": "attend-batch8-131000", "op": "attend", "heads": 64, "kv": 8, "hd": 128, "batch": 8, "new": 1,
         "top": 131001, "ctx": 131072, "rope": False, "neox": False},
        # the first 512 tokens of a prompt, 7B-shaped layer
        {"name": "attend-prompt-512", "op": "attend", "heads": 32, "kv": 32, "hd": 128, "batch": 1, "new": 512,
         "top": 0, "ctx": 512, "rope": True, "neox": False},
        # a later piece of a long prompt, odd length, split-half rotation
        {"name": "attend-prompt-1111-at-6000", "op": "attend", "heads": 64, "kv": 8, "hd": 128, "batch": 1,
         "new": 1111, "top": 6000, "ctx": 8192, "rope": True, "neox": True},
        # the new rows of sixteen decoding requests go into the cache
        {"name": "append-batch16", "op": "append", "kv": 8, "hd": 128, "batch": 16, "new": 1, "top": 2047,
         "ctx": 2048, "rope": True, "neox": False},
        # a long prompt's rows go into the cache
        {"name": "append-prompt-8191", "op": "append", "kv": 32, "hd": 128, "batch": 1, "new": 8191, "top": 1,
         "ctx": 8192, "rope": True, "neox": True},
        # one request's next token with its five best alternatives
        {"name": "logprobs-one-top5", "op": "logprobs", "rows": 1, "vocab": 32000, "stride": 32000, "n": 5,
         "half": False, "masked": False},
        # a full decode batch with twenty alternatives each, part of the vocabulary banned by a grammar
        {"name": "logprobs-batch32-top20", "op": "logprobs", "rows": 32, "vocab": 32000, "stride": 32000, "n": 20,
         "half": False, "masked": True},
        # scoring a text (perplexity): the given tokens' log probabilities and the entropies alone
        {"name": "logprobs-score-4096", "op": "logprobs", "rows": 4096, "vocab": 32000, "stride": 32000, "n": 0,
         "half": False, "masked": False},
        # a large odd vocabulary in fp16 with padded rows
        {"name": "logprobs-half-131071-top8", "op": "logprobs", "rows": 300, "vocab": 131071, "stride": 131077, "n": 8,
         "half": True, "masked": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = _spread(rng, 1000, 200000)
        rows = _spread(rng, 1, max(1, min(4096, 130000000 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "stride": vocab + rng.choice([0, 0, 1, 5, 64]),
                "n": rng.choice([0, 1, 5, 8, 20, 32]), "half": rng.random() < 0.3, "masked": rng.random() < 0.4}
    hd = rng.choice([64, 128])
    kv, mul = rng.choice([(1, 8), (2, 4), (4, 8), (8, 8), (8, 4), (32, 1), (6, 3), (4, 12)])
    rope, neox = rng.random() < 0.5, rng.random() < 0.5
    if op == "append":
        new = _spread(rng, 1, 8192)
        batch = _spread(rng, 1, max(1, min(32, 8192 // new)))
        top = _spread(rng, 1, 8192)
        return {"op": op, "kv": kv, "hd": hd, "batch": batch, "new": new, "top": top,
                "ctx": -(-(top + new) // 16) * 16, "rope": rope, "neox": neox}
    if rng.random() < 0.6:  # decode, now and then a few tokens at once
        batch, new = _spread(rng, 1, 32), rng.choice([1, 1, 1, 2, 5])
        top = _spread(rng, 1, max(2, min(131000, 6000000 // (batch * kv))))
    else:
        batch = rng.choice([1, 1, 2])
        new, top = _spread(rng, 16, 1000 // batch), _spread(rng, 1, 6000 // batch)
    return {"op": op, "heads": kv * mul, "kv": kv, "hd": hd, "batch": batch, "new": new, "top": top,
            "ctx": -(-(top + new) // 16) * 16, "rope": rope, "neox": neox}


def _positions(case):
    """Each sequence's first new position: ragged between half of `top` and `top`."""
    b = case["batch"]
    return [case["top"] - (case["top"] // 2) * ((37 * i) % b) // b for i in range(b)]


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["half"] else 4) + case["rows"] * (12 + 8 * case["n"]), "flops": 6 * n}
    kv, hd, new = case["kv"], case["hd"], case["new"]
    row = hd // 2 + hd // 16
    if case["op"] == "append":
        rows = 2 * case["batch"] * new * kv  # k and v, read as fp32, written in 4 bits and read back as values
        return {"bytes": rows * (4 * hd + row) + rows * 4 * hd, "flops": rows * hd * 6}
    pos = _positions(case)
    seen = sum(new * p + new * (new + 1) // 2 for p in pos)
    cache = sum(p + new for p in pos) * kv * 2 * row
    return {"bytes": cache + 2 * 4 * case["batch"] * new * case["heads"] * hd,
            "flops": 4 * hd * case["heads"] * seen}


# ---- inputs ---------------------------------------------------------------------------------------------------


def _rotate(x, table, pos, neox):
    """Rotary embedding of x [batch, new, heads, hd] at positions pos [batch, new], table [ctx, hd / 2, 2]."""
    cs = table[pos].to(x.dtype)
    c, s = cs[..., None, :, 0], cs[..., None, :, 1]
    if neox:
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _quantize(x):
    """fp32 x [..., hd] -> (quants uint8 [..., hd / 2], scales fp16 [..., nb]): the nearest level, halves up."""
    nb = x.shape[-1] // 32
    x = torch.nan_to_num(x, nan=0.0, posinf=_CLAMP, neginf=-_CLAMP).clamp(-_CLAMP, _CLAMP).unflatten(-1, (nb, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    d = (torch.where(-lo >= hi, lo, hi) * -0.125).to(torch.float16)
    f = d.double()[..., None]  # in 64 bits: a value next to the border of two levels has to fall on its own side
    q = torch.where(f == 0, 8.0, (x.double() / f + 8.5).floor().clamp(0, 15)).to(torch.uint8)
    q = q.unflatten(-1, (2, 2, 8))                          # [..., nb, byte, nibble, g]
    q = q[..., 0, :] | (q[..., 1, :] << 4)                  # [..., nb, byte, g]
    return q.movedim(-1, -3).flatten(-3), d                 # [..., g, nb, byte]


def _values(quants, scales, dtype=torch.float32):
    """The values that a cache's rows stand for."""
    nb = scales.shape[-1]
    q = quants.unflatten(-1, (8, nb, 2)).movedim(-3, -1)    # [..., nb, byte, g]
    q = torch.stack([q & 15, q >> 4], -2)                   # [..., nb, byte, nibble, g]
    return ((q.flatten(-3).to(dtype) - 8) * scales.to(dtype)[..., None]).flatten(-2)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    st = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab, stride = case["rows"], case["vocab"], case["stride"]
        full = randn(rows, stride) * 2.5
        sure = torch.rand(rows, generator=gen, device=dev) < 0.5  # half of the rows have a clear favourite
        fav = torch.randint(vocab, (rows,), generator=gen, device=dev)
        full[torch.arange(rows, device=dev), fav] += sure * 14.0
        if case["masked"]:
            full[torch.rand(rows, stride, generator=gen, device=dev) < 0.3] = -math.inf
        tok = torch.randint(vocab, (rows,), generator=gen, device=dev)
        tok = torch.where(torch.rand(rows, generator=gen, device=dev) < 0.7, fav, tok)
        full[torch.arange(rows, device=dev), tok] = full[torch.arange(rows, device=dev), tok].clamp_min(-12.0)
        st["logits"] = full.half() if case["half"] else full
        st["tokens"] = tok.int()
        st["logprob"], st["entropy"] = (torch.empty(rows, device=dev) for _ in range(2))
        st["top_ids"] = torch.empty(rows, case["n"], dtype=torch.int32, device=dev)
        st["top_logprobs"] = torch.empty(rows, case["n"], device=dev)
        return st
    batch, new, kv, hd, ctx = case["batch"], case["new"], case["kv"], case["hd"], case["ctx"]
    st["pos"] = torch.tensor(_positions(case), dtype=torch.int32, device=dev)
    inv = 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
    ang = torch.arange(ctx, device=dev, dtype=torch.float64)[:, None] * inv
    st["table"] = torch.stack([ang.cos(), ang.sin()], -1).float() if case["rope"] else None
    st["cache"] = {}
    for which in ("k", "v"):
        quants = torch.empty(batch, kv, ctx, hd // 2, dtype=torch.uint8, device=dev)
        scales = torch.empty(batch, kv, ctx, hd // 32, dtype=torch.float16, device=dev)
        if case["op"] == "attend":
            wide = 1.0 + 3.0 * (torch.rand(kv, 1, hd, generator=gen, device=dev) < 0.05) * (which == "k")
            for b in range(batch):
                quants[b], scales[b] = _quantize(randn(kv, ctx, hd) * wide)
        else:
            quants.fill_(0x88)
            scales.zero_()
        st["cache"][which] = (quants, scales)
    if case["op"] == "attend":
        st["q"] = randn(batch, new, case["heads"] * hd)
        st["out"] = torch.empty_like(st["q"])
    else:
        st["k"], st["v"] = randn(batch, new, kv * hd) * 2.0, randn(batch, new, kv * hd)
        st["out"] = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    return st


# ---- the operators --------------------------------------------------------------------------------------------


def _attend(case, q, k, v, pos, table):
    """Plain attention in q's type: k, v [batch, kv, length, hd]."""
    batch, new, kv, hd = case["batch"], case["new"], case["kv"], case["hd"]
    at = pos.long()[:, None] + torch.arange(new, device=q.device)
    q = q.view(batch, new, case["heads"], hd)
    if table is not None:
        q = _rotate(q, table, at, case["neox"])
    q = q.view(batch, new, kv, -1, hd).permute(0, 2, 1, 3, 4)          # [batch, kv, new, mul, hd]
    s = (q.flatten(2, 3) @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).unflatten(2, (new, -1))
    hidden = torch.arange(k.shape[2], device=q.device) > at[..., None]     # [batch, new, length]
    s.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.flatten(2, 3) @ v).unflatten(2, (new, -1)) / total
    return o.permute(0, 2, 1, 3, 4).reshape(batch, new, -1)


def _logprobs(x, tokens, n):
    """Plain log probabilities in x's type: of the tokens, the entropies, the n best."""
    m = x.amax(-1, keepdim=True)
    shifted = x - m
    e = shifted.exp()
    total = e.sum(-1)
    log_total = total.log()
    entropy = log_total - torch.where(e > 0, shifted * e, torch.zeros_like(e)).sum(-1) / total
    got = {"logprob": shifted.gather(1, tokens.long()[:, None])[:, 0] - log_total, "entropy": entropy}
    if n:
        # one order on (value, lowest index first): the value's bits as an ordered whole number, then the index
        bits = (x.float() + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (order << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
        ids = 0xFFFFFFFF - (key.topk(n, -1).values & 0xFFFFFFFF)
        got["top_ids"] = ids.int()
        got["top_logprobs"] = shifted.gather(1, ids) - log_total[:, None]
    return got


def _length(case):
    return max(_positions(case)) + case["new"]


def _stored(case, st):
    """What the append puts into the cache, k and v, and at which positions."""
    batch, new, kv, hd = case["batch"], case["new"], case["kv"], case["hd"]
    at = st["pos"].long()[:, None] + torch.arange(new, device=st["pos"].device)
    k, v = (st[w].view(batch, new, kv, hd) for w in ("k", "v"))
    if st["table"] is not None:
        k = _rotate(k, st["table"], at, case["neox"])
    return [_quantize(x) for x in (k, v)], at


def _plain(st):
    case = st["case"]
    if case["op"] == "logprobs":
        return _logprobs(st["logits"][:, :case["vocab"]].float(), st["tokens"], case["n"])
    cache = st["cache"]
    if case["op"] == "append":
        got, at = _stored(case, st)
        rows = torch.arange(case["batch"], device=at.device)[:, None]
        values = []
        for which, (quants, scales) in zip(("k", "v"), got):
            cache[which][0][rows, :, at] = quants
            cache[which][1][rows, :, at] = scales
            values.append(_values(cache[which][0][rows, :, at], cache[which][1][rows, :, at]).flatten(2))
        return {"k": values[0], "v": values[1]}
    n = _length(case)
    k, v = (_values(cache[w][0][:, :, :n], cache[w][1][:, :, :n]) for w in ("k", "v"))
    return {"out": _attend(case, st["q"], k, v, st["pos"], st["table"])}


def _own(st):
    import chatnet_b200 as cn

    case, stream = st["case"], torch.cuda.current_stream().cuda_stream
    dev = st["tokens" if case["op"] == "logprobs" else "pos"].device.index
    ctx = _contexts.get(dev)
    if ctx is None:
        ctx = _contexts[dev] = cn.Context(dev)
    if case["op"] == "logprobs":
        n = case["n"]
        ctx.logprobs_dev(st["logits"].data_ptr(), case["rows"], case["vocab"], st["tokens"].data_ptr(),
                         st["logprob"].data_ptr(), st["entropy"].data_ptr(), n,
                         st["top_ids"].data_ptr() if n else 0, st["top_logprobs"].data_ptr() if n else 0,
                         row_stride=case["stride"], type_=cn.TYPE_F16 if case["half"] else cn.TYPE_F32, stream=stream)
        got = {"logprob": st["logprob"], "entropy": st["entropy"]}
        return {**got, "top_ids": st["top_ids"], "top_logprobs": st["top_logprobs"]} if n else got
    (kq, kd), (vq, vd) = st["cache"]["k"], st["cache"]["v"]
    cache = cn.KvQ4Cache(kq.data_ptr(), kd.data_ptr(), vq.data_ptr(), vd.data_ptr(), case["batch"], case["kv"],
                         case["hd"], case["ctx"])
    rope = 0 if st["table"] is None else st["table"].data_ptr()
    if case["op"] == "append":
        k, v = st["out"]
        ctx.kvq4_append_dev(cache, st["k"].data_ptr(), st["v"].data_ptr(), st["pos"].data_ptr(), case["batch"],
                            case["new"], rope=rope, rope_neox=case["neox"], stream=stream)
        ctx.kvq4_read_dev(cache, k.data_ptr(), v.data_ptr(), st["pos"].data_ptr(), case["batch"], case["new"],
                          stream=stream)
        return {"k": k, "v": v}
    ctx.kvq4_attend_dev(cache, st["q"].data_ptr(), st["out"].data_ptr(), st["pos"].data_ptr(), case["batch"],
                        case["heads"], n_new=case["new"], rope=rope, rope_neox=case["neox"], stream=stream)
    return {"out": st["out"]}


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------


def _exact_row(case, st, b, g, keys, values):
    """Attention of sequence b's queries that read kv head g, one query after another where they are few rows."""
    hd, mul, new = case["hd"], case["heads"] // case["kv"], case["new"]
    q = st["q"][b].double().view(new, case["heads"], hd)[:, g * mul:(g + 1) * mul]
    first = int(st["pos"][b])
    if st["table"] is not None:
        cs = st["table"][first:first + new].double()[:, None]
        turn = torch.complex(cs[..., 0], cs[..., 1])
        pairs = (torch.complex(q[..., :hd // 2], q[..., hd // 2:]) if case["neox"]
                 else torch.view_as_complex(q.reshape(new, mul, hd // 2, 2).contiguous())) * turn
        q = torch.cat([pairs.real, pairs.imag], -1) if case["neox"] else torch.view_as_real(pairs).flatten(-2)
    seen = first + new
    s = torch.einsum("nmd,pd->nmp", q, keys[:seen]) / math.sqrt(hd)
    late = torch.arange(seen, device=q.device)[None, :] > first + torch.arange(new, device=q.device)[:, None]
    w = torch.softmax(s.masked_fill(late[:, None], -math.inf), -1)
    return torch.einsum("nmp,pd->nmd", w, values[:seen])


def _exact_levels(case, st, which):
    """The values on the cache's grid nearest to the rows; k is rotated in fp32 first, as a decode step has it."""
    batch, new, kv, hd = case["batch"], case["new"], case["kv"], case["hd"]
    x = st[which].view(batch, new, kv, hd)
    if which == "k" and st["table"] is not None:
        cs = torch.stack([st["table"][p:p + new] for p in _positions(case)])[:, :, None]  # [batch, new, 1, hd / 2, 2]
        half = hd // 2
        a = x[..., :half] if case["neox"] else x.unflatten(-1, (half, 2))[..., 0]
        b = x[..., half:] if case["neox"] else x.unflatten(-1, (half, 2))[..., 1]
        left, right = a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]
        x = torch.cat([left, right], -1) if case["neox"] else torch.stack([left, right], -1).flatten(-2)
    x = x.double().view(batch, new, kv, hd // 32, 32)
    far = x.abs().amax(-1, keepdim=True)
    d = -torch.where(x.amin(-1, keepdim=True) == -far, -far, far) / 8
    d = d.to(torch.float16).double()
    level = torch.ceil(x / d - 0.5)
    level = torch.where(level == x / d - 0.5, level + 1, level).clamp(-8, 7)
    return torch.where(d == 0, torch.zeros_like(x), d * level).view(batch, new, kv * hd)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        x = st["logits"][:, :case["vocab"]]
        got = {"logprob": [], "entropy": [], "top_ids": None, "top_logprobs": []}
        for r in range(0, case["rows"], 256):
            p = torch.log_softmax(x[r:r + 256].double(), -1)
            got["logprob"].append(p.gather(1, st["tokens"][r:r + 256].long()[:, None])[:, 0])
            got["entropy"].append(torch.special.entr(p.exp()).sum(-1))
            if case["n"]:
                got["top_logprobs"].append(p.topk(case["n"], -1).values)
        got = {k: torch.cat(v) if v else None for k, v in got.items()}
        return got if case["n"] else {"logprob": got["logprob"], "entropy": got["entropy"]}
    if case["op"] == "append":
        return {w: _exact_levels(case, st, w) for w in ("k", "v")}
    hd, mul = case["hd"], case["heads"] // case["kv"]
    out = torch.empty(case["batch"], case["new"], case["heads"], hd, dtype=torch.float64, device=st["q"].device)
    for b in range(case["batch"]):
        for g in range(case["kv"]):
            k, v = (_values(st["cache"][w][0][b, g], st["cache"][w][1][b, g], torch.float64) for w in ("k", "v"))
            out[b, :, g * mul:(g + 1) * mul] = _exact_row(case, st, b, g, k, v)
    return {"out": out.flatten(2)}
