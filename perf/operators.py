"""Cases of the paged-cache serving operators: their inputs, their plain form, their work.

  append  the post-QKV step of a chunk of tokens over a paged cache: per-head RMSNorm of
          q and k, rotary positions with one to four axes, the new key and value rows
          written to their pages in 16 bits or quantised to int8 with one scale a row
  read    rows of sequences back from their pages, dequantised
  attn    grouped-query attention of a chunk of new tokens over the paged cache
          (one token a sequence: decoding)
  verify  verification of drafted tokens against the target's probabilities from
          given random numbers

With `own` false, `run` computes them in elementary torch operations; with `own` true it
calls the framework.  `exact` gives the same from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

D = 128      # head dimension of every decoder here
EPS = 1e-6
SECTIONS = {1: (64,), 2: (40, 24), 3: (24, 20, 20), 4: (16, 16, 16, 16)}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dial-8b-orin_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from dial_cuda import paged
    return paged


# ------------------------------------------------------------------ cases
def _append(name, seqs, q, ctx, dtype, quant, page, axes, interleaved=True, ragged=False, hq=32, hkv=8, norm=True):
    return dict(name=name, kind="append", seqs=seqs, q=q, ctx=ctx, dtype=dtype, quant=quant, page=page, axes=axes,
                interleaved=interleaved, ragged=ragged, hq=hq, hkv=hkv, norm=norm)


def _read(name, seqs, ctx, dtype, quant, page, ragged=False, hkv=8):
    return dict(name=name, kind="read", seqs=seqs, q=ctx, ctx=ctx, dtype=dtype, quant=quant, page=page, ragged=ragged, hkv=hkv)


def _attn(name, seqs, q, ctx, dtype, quant, page, ragged=False, hq=32, hkv=8):
    return dict(name=name, kind="attn", seqs=seqs, q=q, ctx=ctx, dtype=dtype, quant=quant, page=page, ragged=ragged, hq=hq, hkv=hkv)


def _verify(name, seqs, rows, vocab, dtype, probs, greedy=False, ragged=False):
    return dict(name=name, kind="verify", seqs=seqs, q=rows, vocab=vocab, dtype=dtype, probs=probs, greedy=greedy, ragged=ragged)


def listed():
    return [
        # one sequence's next token, f16 cache, text positions: the smallest call of a decode step
        _append("append_1_token_f16", 1, 1, 2049, "f16", False, 64, 1),
        # a chunk of an image prompt with (time, height, width) positions, bf16 cache
        _append("append_image_chunk_bf16", 1, 2047, 2047, "bf16", False, 64, 3),
        # ragged chunks of a batch with an int8 cache, and the rows that went in read back
        _append("append_ragged_int8", 32, 256, 2048, "f16", True, 16, 3, ragged=True),
        # a long prompt's int8 cache back to f16, as for a hand-over to another stage
        _read("read_long_int8", 1, 32768, "f16", True, 64),
        # the 16-bit caches of a batch of sequences of all lengths
        _read("read_ragged_bf16", 16, 4099, "bf16", False, 32, ragged=True),
        # decoding one sequence; a batch of 32 at 2048 tokens of context; a long ragged one
        _attn("decode_1x2049_f16", 1, 1, 2049, "f16", False, 64),
        _attn("decode_32x2049_int8", 32, 1, 2049, "bf16", True, 64),
        # verification of four drafted tokens of each of 16 sequences
        _attn("drafts_16x5_bf16", 16, 5, 8200, "bf16", False, 64, ragged=True),
        # the last chunk of a long prompt, 16-bit cache
        _attn("chunk_2048_of_16384_bf16", 1, 2048, 16384, "bf16", False, 64),
        # ragged chunks of a batch, int8 cache
        _attn("chunk_ragged_int8", 8, 777, 4100, "f16", True, 16, ragged=True),
        # three drafts of one sequence, draft tokens without probabilities
        _verify("verify_1x4_f16", 1, 4, 151936, "f16", False),
        # up to five drafts of each of 32 sequences, with the draft model's probabilities
        _verify("verify_32x6_bf16", 32, 6, 151936, "bf16", True, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attn", "attn", "attn", "verify"])
    dtype, quant, page = rng.choice(["f16", "bf16"]), rng.random() < 0.5, rng.choice([16, 32, 64, 128, 256])
    hkv = rng.choice([1, 2, 4, 8, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    ragged = rng.random() < 0.6
    if kind == "append":
        q = _log(rng, 1, 2048)
        seqs = _log(rng, 1, max(1, min(64, 8192 // q)))
        axes = rng.choice([1, 2, 3, 3, 4])
        c = _append("", seqs, q, q + _log(rng, 1, 4096) - 1, dtype, quant, page, axes, rng.random() < 0.5, ragged, hq, hkv, rng.random() < 0.7)
    elif kind == "read":
        ctx = _log(rng, 1, 32768)
        c = _read("", _log(rng, 1, max(1, min(64, 65536 // ctx))), ctx, dtype, quant, page, ragged, hkv)
    elif kind == "attn":
        q = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 2048)])
        ctx = q + _log(rng, 1, 16384) - 1
        c = _attn("", _log(rng, 1, max(1, min(64, 262144 // ctx))), q, ctx, dtype, quant, page, ragged, hq, hkv)
    else:
        vocab = rng.choice([151936, 128256, _log(rng, 1000, 151936)])
        rows = rng.randint(1, 9)
        c = _verify("", _log(rng, 1, max(1, 192 // rows)), rows, vocab, rng.choice(["f16", "bf16", "f32"]), rng.random() < 0.5,
                    rng.random() < 0.2, ragged)
    del c["name"]
    while work(c)["bytes"] > 2.3e8 or work(c)["flops"] > 5.1e11:  # no more than the largest listed ones
        if c["seqs"] > 1:
            c["seqs"] = (c["seqs"] + 1) // 2
        else:
            c["q"], c["ctx"] = (c["q"] + 1) // 2, (c["ctx"] + 1) // 2
    return c


def _lengths(c):
    """New tokens and cache rows (the new ones among them) of each sequence."""
    q, kv = [], []
    for b in range(c["seqs"]):
        f = ((b + 1) * 0.6180339887498949) % 1.0
        g = ((b + 1) * 0.7548776662466927) % 1.0
        n = c["q"] if b == 0 or not c["ragged"] else max(1, int(round(c["q"] ** f)))
        L = c.get("ctx", n)
        if c["kind"] == "read":
            L = n
        elif b and c["ragged"]:
            L = n + int(g * max(0, L - n))
        q.append(n)
        kv.append(L)
    return q, kv


def work(c):
    q, kv = _lengths(c)
    e = 4 if c["dtype"] == "f32" else 2
    T = sum(q)
    if c["kind"] == "verify":
        read = T * c["vocab"] * e + T * 8
        if c["probs"]:
            read += c["seqs"] * c["vocab"] * 4  # the draft's distribution at one row a sequence
        return {"bytes": read + T * 8 + c["seqs"] * 8, "flops": 4 * T * c["vocab"]}
    row = 2 * c["hkv"] * ((D + 4) if c["quant"] else D * 2)  # a token's keys and values as the cache holds them
    if c["kind"] == "append":
        n = c["hq"] + 2 * c["hkv"]
        moved = T * (n * D * e + c["hq"] * D * e + row + 4 * c["axes"])
        if c["quant"]:
            moved += T * (row + 2 * c["hkv"] * D * e)  # and back
        return {"bytes": moved, "flops": 8 * T * n * D}
    if c["kind"] == "read":
        return {"bytes": T * (row + 2 * c["hkv"] * D * e), "flops": 2 * T * c["hkv"] * D}
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(q, kv))
    return {"bytes": 2 * T * c["hq"] * D * e + sum(kv) * row, "flops": 4 * seen * c["hq"] * D}


# ------------------------------------------------------------------ inputs
def _quantise(x):
    """int8 codes and the scale of each row of x [..., D]: absmax / 127, halves away from zero."""
    a = x.abs().amax(-1, keepdim=True)
    s = torch.where(a > 0, (a.double() / 127.0).float(), torch.ones_like(a))
    y = x * (1.0 / s)
    r = torch.trunc(y)
    r = r + torch.sign(y) * ((y - r).abs() >= 0.5)
    return r.clamp_(-127, 127).to(torch.int8), s.squeeze(-1)


def _pages(c, g, kv, scale=1.0):
    """A pool with the sequences' pages in any order, rows of every page filled, and the block table."""
    need = [-(-L // c["page"]) for L in kv]
    n = sum(need) + 3
    order = torch.randperm(n, generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    table = torch.full((c["seqs"], max(need) + 1), -1, dtype=torch.int32)
    first, host = 0, order.cpu()
    for b, m in enumerate(need):
        table[b, :m] = host[first:first + m]
        first += m
    shape = (n, c["hkv"], c["page"], D)
    dt = DTYPES[c["dtype"]]
    s = {"table": table.cuda()}
    for name, mean in (("k", 0.0), ("v", 0.25)):
        x = torch.randn(shape, generator=g, device="cuda") * scale + mean
        if c["quant"]:
            s[name], s[name + "_scale"] = _quantise(x.to(dt).float())
        else:
            s[name] = x.to(dt)
    return s


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q, kv = _lengths(c)
    T, dt = sum(q), DTYPES[c["dtype"]]
    start = [0]
    for n in q:
        start.append(start[-1] + n)
    s = {"c": c, "max_q": max(q), "tokens": T}
    s["start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    if c["kind"] == "verify":
        V = c["vocab"]
        logits = torch.randn((T, V), generator=g, device="cuda") * 2.5
        draft = (logits + torch.randn((T, V), generator=g, device="cuda") * 0.7).softmax(-1)  # a smaller model's view
        s["logits"] = logits.to(dt)
        noise = torch.empty((T, V), device="cuda").exponential_(generator=g)
        drafted = s["logits"].float().argmax(-1) if c["greedy"] else (draft / noise).argmax(-1)
        if not c["probs"] and not c["greedy"]:
            drafted = draft.argmax(-1)  # a draft without probabilities: its best token
        wrong = torch.rand(T, generator=g, device="cuda") < 0.15
        drafted = torch.where(wrong & c["greedy"], (drafted + 1) % V, drafted)
        s["ids"] = torch.cat([drafted[:1], drafted[:-1]]).to(torch.int32)  # ids[r + 1] is the draft that row r judges
        s["temperature"] = torch.rand(c["seqs"], generator=g, device="cuda") * 0.7 + 0.5
        if c["greedy"]:
            s["temperature"].zero_()
        s["accept"] = torch.rand(T, generator=g, device="cuda")
        s["sample"] = torch.rand(c["seqs"], generator=g, device="cuda")
        s["probs"] = draft if c["probs"] else None
        return s
    s["kv"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["max_kv"] = max(kv)
    s.update(_pages(c, g, kv))
    if c["kind"] == "append":
        n = c["hq"] + 2 * c["hkv"]
        s["qkv"] = (torch.randn((T, n * D), generator=g, device="cuda") * 1.5).to(dt)
        for name in ("q_norm", "k_norm"):
            w = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
            s[name] = w.to(dt) if c["norm"] else None
        # text: the cache row; further axes: a picture's rows and columns, from a place in the prompt on
        at = torch.arange(T, device="cuda") + (s["kv"].long() - s["start"][1:].long()).repeat_interleave(torch.tensor(q, device="cuda"))
        off = int(torch.randint(0, 64, (1,), generator=g, device="cuda"))
        pos = [at, off + at // 32 % 32, off + at % 32, at // 7]
        s["positions"] = torch.stack(pos[:c["axes"]]).to(torch.int32).contiguous()
        rows = max(kv) + 128
        angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["out"] = torch.zeros((T, c["hq"], D), dtype=dt, device="cuda")
    if c["kind"] == "attn":
        s["q"] = (torch.randn((T, c["hq"], D), generator=g, device="cuda") * 1.5).to(dt)
        s["out"] = torch.zeros((T, c["hq"], D), dtype=dt, device="cuda")
    if c["kind"] == "read" or (c["kind"] == "append" and c["quant"]):
        s["k_rows"] = torch.zeros((T, c["hkv"], D), dtype=dt, device="cuda")
        s["v_rows"] = torch.zeros((T, c["hkv"], D), dtype=dt, device="cuda")
    if own:  # the handles that a serving loop keeps
        P = _framework()
        s["cache"] = P.PagedKVCache.from_tensors(s["k"], s["v"], s.get("k_scale"), s.get("v_scale"))
        s["batch"] = P.PagedBatch(s["table"], s["kv"], s["start"], max_q=s["max_q"], max_kv=s["max_kv"])
    return s


# ------------------------------------------------------------------ the plain form
def _places(s):
    """Sequence, cache row, page and row of the page of every token."""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["start"].long(), t, right=True) - 1
    row = s["kv"].long()[b] - s["start"].long()[b + 1] + t
    P = s["c"]["page"]
    return b, row, s["table"].long()[b, row // P], row % P


def _axis_of_pair(c):
    """The position axis that turns each of the D / 2 pairs."""
    n, pair = SECTIONS[c["axes"]], torch.arange(D // 2, device="cuda")
    ends = torch.tensor(n, device="cuda")
    if not c["interleaved"]:
        return torch.searchsorted(ends.cumsum(0), pair, right=True)
    axis = pair % len(n)
    return torch.where(pair < ends[axis] * len(n), axis, 0)


def _norm_rope(x, w, cos, sin):
    """x [T, heads, D] in 32 bits, the mean square in 64."""
    if w is not None:
        inv = (1.0 / (x.double().square().sum(-1, keepdim=True) / D + float(torch.tensor(EPS))).sqrt()).float()
        x = x * inv * w.float()
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_read(s):
    b, _, page, at = _places(s)
    out = []
    for name in ("k", "v"):
        x = s[name][page, :, at]
        if s["c"]["quant"]:
            x = x.float() * s[name + "_scale"][page, :, at][..., None]
        out.append(x.to(DTYPES[s["c"]["dtype"]]))
    return out


def _plain_append(s):
    c = s["c"]
    dt, hq, hkv = DTYPES[c["dtype"]], c["hq"], c["hkv"]
    x = s["qkv"].view(-1, hq + 2 * hkv, D).float()
    row = s["positions"].long()[_axis_of_pair(c)].t()  # the table row that turns each pair of each token
    pair = torch.arange(D // 2, device="cuda")
    cos, sin = s["cos"][row, pair][:, None], s["sin"][row, pair][:, None]
    q = _norm_rope(x[:, :hq], s["q_norm"], cos, sin).to(dt)
    k, v = _norm_rope(x[:, hq:hq + hkv], s["k_norm"], cos, sin), x[:, hq + hkv:]
    _, _, page, at = _places(s)
    if not c["quant"]:
        s["k"][page, :, at], s["v"][page, :, at] = k.to(dt), v.to(dt)
        return [q, s["k"], s["v"]]
    s["k"][page, :, at], s["k_scale"][page, :, at] = _quantise(k)
    s["v"][page, :, at], s["v_scale"][page, :, at] = _quantise(v)
    return [q] + _plain_read(s)


def _padded(s, dtype):
    """The sequences' keys and values as [B, kv heads, longest, D]."""
    c = s["c"]
    L = torch.arange(s["max_kv"], device="cuda")
    page = s["table"].long()[:, L // c["page"]].clamp_(min=0)  # rows behind a sequence's last are masked
    out = []
    for name in ("k", "v"):
        x = s[name][page, :, L % c["page"]].to(dtype)
        if c["quant"]:
            x *= s[name + "_scale"][page, :, L % c["page"]].to(dtype)[..., None]
        out.append(x.transpose(1, 2))
    return out


def _plain_attn(s):
    c = s["c"]
    B, Q, hkv, rep = c["seqs"], s["max_q"], c["hkv"], c["hq"] // c["hkv"]
    k, v = _padded(s, torch.float32)
    i = torch.arange(Q, device="cuda")
    n = (s["start"][1:] - s["start"][:-1]).long()
    tok = (s["start"][:-1].long()[:, None] + i).clamp_(max=s["tokens"] - 1)
    q = s["q"].float()[tok].view(B, Q, hkv, rep, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, rep * Q, D)
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(B, hkv, rep, Q, -1)
    last = s["kv"].long()[:, None] - n[:, None] + i  # the last cache row that a token sees
    x.masked_fill_((torch.arange(s["max_kv"], device="cuda") > last[..., None])[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    x.div_(x.sum(-1, keepdim=True))
    o = torch.matmul(x.view(B, hkv, rep * Q, -1), v).view(B, hkv, rep, Q, D).permute(0, 3, 1, 2, 4)
    return [o[i < n[:, None]].reshape(-1, c["hq"], D).to(DTYPES[c["dtype"]])]


def _plain_verify(s):
    c = s["c"]
    V, B, R = c["vocab"], c["seqs"], s["tokens"]
    start, t = s["start"].long(), torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(start, t, right=True) - 1
    n = start[1:] - start[:-1]
    temp = s["temperature"].double()[b][:, None]
    x = s["logits"].double()
    best = x.argmax(-1)
    logp = (x / torch.where(temp > 0, temp, 1.0)).log_softmax(-1)
    p = logp.exp()
    draft = s["ids"].long()[(t + 1).clamp_(max=R - 1)]
    q = s["probs"].double()[t, draft] if c["probs"] else torch.ones_like(s["accept"], dtype=torch.float64)
    ok = torch.where(temp[:, 0] > 0, s["accept"].double() * q < p[t, draft], draft == best)
    judged = t + 1 < start[1:][b]  # a sequence's last row judges no draft
    stop = torch.full((B,), R, device="cuda").scatter_reduce_(0, b, torch.where(ok & judged, R, t), "amin")
    w = p[stop]
    left = judged[stop][:, None]  # a rejected draft: what the target has over it
    if c["probs"]:
        rest = (w - s["probs"][stop].double()).clamp_(min=0)
    else:
        rest = w.scatter(1, draft[stop][:, None], 0.0)
    rest = torch.where(left & (rest.sum(-1, keepdim=True) > 0), rest, w)
    cum = rest.cumsum(-1)
    drawn = (cum <= s["sample"].double()[:, None] * cum[:, -1:]).sum(-1).clamp_(max=V - 1)
    drawn = torch.where(s["temperature"] > 0, drawn, best[stop])
    token = torch.where(t < stop[b], draft, torch.where(t == stop[b], drawn[b], -1))
    told = torch.where(token >= 0, logp[t, token.clamp(min=0)], 0.0).float()
    return [token.to(torch.int32), (stop - start[:-1] + 1).to(torch.int32), told]


# ------------------------------------------------------------------ a pass
def run(s):
    c = s["c"]
    if own:
        if c["kind"] == "verify":
            return list(_framework().verify_drafts(s["logits"], s["ids"], s["start"], s["temperature"], s["accept"], s["sample"],
                                                   draft_probs=s["probs"], max_q=s["max_q"]))
        if c["kind"] == "attn":
            return [s["cache"].attention(s["q"], s["batch"], out=s["out"])]
        if c["kind"] == "read":
            return list(s["cache"].read(s["batch"], out=(s["k_rows"], s["v_rows"])))
        q = s["cache"].append(s["qkv"], s["batch"], s["cos"], s["sin"], s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                              sections=SECTIONS[c["axes"]], interleaved=c["interleaved"], out=s["out"])
        if not c["quant"]:
            return [q, s["k"], s["v"]]
        return [q] + list(s["cache"].read(s["batch"], out=(s["k_rows"], s["v_rows"])))
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn, "verify": _plain_verify}[c["kind"]](s)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(s, name, b, first, last):
    """Rows first..last of sequence b's keys or values in 64 bits, [rows, kv heads, D]."""
    P = s["c"]["page"]
    parts = []
    for i in range(first // P, -(-last // P)):
        page = int(s["table"][b, i])
        lo, hi = max(first - i * P, 0), min(last - i * P, P)
        x = s[name][page, :, lo:hi].double()
        if s["c"]["quant"]:
            x = x * s[name + "_scale"][page, :, lo:hi, None].double()
        parts.append(x.transpose(0, 1))
    return torch.cat(parts)


def exact(c, seed):
    s = prepare(c, seed)
    n, kv = _lengths(c)
    start = s["start"].tolist()
    if c["kind"] == "read":
        return [torch.cat([_exact_rows(s, name, b, 0, kv[b]) for b in range(c["seqs"])]) for name in ("k", "v")]
    if c["kind"] == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        rep = c["hq"] // c["hkv"]
        for b in range(c["seqs"]):
            k, v = _exact_rows(s, "k", b, 0, kv[b]), _exact_rows(s, "v", b, 0, kv[b])
            late = torch.ones((n[b], kv[b]), dtype=torch.bool, device="cuda").triu(kv[b] - n[b] + 1)
            for h in range(c["hq"]):
                x = s["q"][start[b]:start[b + 1], h].double() @ k[:, h // rep].T / math.sqrt(D)
                out[start[b]:start[b + 1], h] = torch.softmax(x.masked_fill(late, -math.inf), -1) @ v[:, h // rep]
        return [out]
    if c["kind"] == "append":
        hq, hkv = c["hq"], c["hkv"]
        x = s["qkv"].double().view(s["tokens"], hq + 2 * hkv, D)
        axis, used = [], 0
        for a, m in enumerate(SECTIONS[c["axes"]]):
            axis += [a] * m
        if c["interleaved"]:
            axis = [0] * (D // 2)
            for a, m in enumerate(SECTIONS[c["axes"]]):
                for j in range(m if a else 0):
                    axis[a + j * c["axes"]] = a
        cos = torch.stack([s["cos"][s["positions"][a].long(), i] for i, a in enumerate(axis)], -1).double()
        sin = torch.stack([s["sin"][s["positions"][a].long(), i] for i, a in enumerate(axis)], -1).double()
        turn = torch.complex(cos, sin)[:, None]

        def turned(y, w):
            if w is not None:
                y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        def held(y):  # what int8 rows stand for
            step = y.abs().amax(-1, keepdim=True) / 127
            step = torch.where(step > 0, step, 1.0)
            return torch.floor((y / step).abs() + 0.5) * y.sign() * step

        q, k, v = turned(x[:, :hq], s["q_norm"]), turned(x[:, hq:hq + hkv], s["k_norm"]), x[:, hq + hkv:]
        if c["quant"]:
            return [q, held(k), held(v)]
        pools = [s["k"].double(), s["v"].double()]
        for b in range(c["seqs"]):
            for i in range((kv[b] - n[b]) // c["page"], -(-kv[b] // c["page"])):
                lo, hi = max(kv[b] - n[b], i * c["page"]), min(kv[b], (i + 1) * c["page"])
                t = start[b] + lo - (kv[b] - n[b])
                for pool, rows in zip(pools, (k, v)):
                    pool[int(s["table"][b, i]), :, lo - i * c["page"]:hi - i * c["page"]] = rows[t:t + hi - lo].transpose(0, 1)
        return [q] + pools
    token, count, told = [], [], []
    for b in range(c["seqs"]):
        temp = float(s["temperature"][b])
        for r in range(start[b], start[b + 1]):
            x = s["logits"][r].double()
            z = x / (temp or 1.0)
            z = z - z.max()
            w = z.exp()
            p = w / w.sum()
            judge = r + 1 < start[b + 1]
            d = int(s["ids"][r + 1]) if judge else -1
            share = (float(s["probs"][r, d]) if c["probs"] else 1.0) if judge else 1.0
            if judge and (float(s["accept"][r]) * share < float(p[d]) if temp > 0 else d == int(x.argmax())):
                pick = d
            elif temp == 0:
                pick, judge = int(x.argmax()), False
            else:
                f = p.clone()
                if judge and c["probs"]:
                    f = torch.relu(p - s["probs"][r].double())
                elif judge:
                    f[d] = 0
                if float(f.sum()) <= 0:
                    f = p
                f = f.cumsum(0)
                pick, judge = min(int(torch.searchsorted(f, (s["sample"][b].double() * f[-1]).reshape(1), right=True)), c["vocab"] - 1), False
            token.append(pick)
            told.append(float(z[pick] - w.sum().log()))
            if not judge:
                break
        count.append(r + 1 - start[b])
        token += [-1] * (start[b + 1] - r - 1)
        told += [0.0] * (start[b + 1] - r - 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    return [torch.tensor(token, **i32), torch.tensor(count, **i32), torch.tensor(told, dtype=torch.float64, device="cuda")]
