"""The cached-attention and answer operators of a decoding server, as measured.

Three operators, each in its plain form (elementary torch operations, 32 bits)
and through the framework (`own`):

  append    new keys and values into the paged 8-bit cache, keys and queries
            rotated by their positions on the way (Context.kv_append)
  attend    attention over that cache: single tokens, a few tokens, prompts
            (Context.paged_attention)
  logprobs  log probabilities of given tokens, the entropy and the top
            alternatives of each row of logits (Context.token_logprobs)

The cache holds e4m3 codes [pages, kv heads, page size, head dim] and one
power-of-two scale for each 16 tokens of a page and head.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 16  # tokens under one scale
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda:0"


# ---- cases -------------------------------------------------------------------


def listed():
    def append(name, **k):
        return dict(name=name, op="append", **k)

    def attend(name, **k):
        return dict(name=name, op="attend", **k)

    def logprobs(name, **k):
        return dict(name=name, op="logprobs", **k)

    return [
        # one user's next token, the model's sliding layers: latency
        append("append 1 token", seqs=1, new=1, past=611, hq=8, hkv=1, d=256, rot=256, page=16, dtype="f32", ragged=False),
        # 64 users decoding together, full-attention layers with a partial rotation
        append("append 64 users", seqs=64, new=1, past=2048, hq=8, hkv=1, d=512, rot=128, page=64, dtype="f32", ragged=True),
        # a few prompts at once, the model's own heads
        append("append prompts", seqs=5, new=1101, past=37, hq=8, hkv=1, d=256, rot=256, page=32, dtype="bf16", ragged=True),
        # a long prompt, grouped heads
        append("append long prompt", seqs=1, new=16384, past=0, hq=32, hkv=8, d=128, rot=128, page=64, dtype="bf16", ragged=False),
        # one user's next token at the context the reference caps its cache at
        attend("decode 1 user", seqs=1, new=1, past=2047, hq=8, hkv=1, d=256, page=16, window=0, dtype="f32", ragged=False),
        # users of all lengths, an empty one among them, full-attention layers
        attend("decode ragged", seqs=33, new=1, past=8192, hq=8, hkv=1, d=512, page=32, window=0, dtype="f32", ragged=True),
        # a very long document: few rows, a long axis
        attend("decode long", seqs=2, new=1, past=131071, hq=8, hkv=1, d=256, page=64, window=0, dtype="bf16", ragged=False),
        # a full server, grouped heads
        attend("decode server", seqs=128, new=1, past=4000, hq=32, hkv=8, d=128, page=64, window=0, dtype="bf16", ragged=True),
        # a prompt in the model's sliding layers
        attend("prompt sliding", seqs=1, new=2048, past=0, hq=8, hkv=1, d=256, page=16, window=512, dtype="bf16", ragged=False),
        # a part of a long prompt behind a long cache, grouped heads
        attend("prompt chunk", seqs=1, new=4096, past=8191, hq=32, hkv=8, d=128, page=64, window=0, dtype="bf16", ragged=False),
        # the answer of one user: the tied head's vocabulary, softcapped
        logprobs("logprobs 1 row", rows=1, vocab=262144, top=5, cap=30.0, dtype="f32"),
        # a prompt's tokens scored
        logprobs("logprobs prompt", rows=500, vocab=262144, top=20, cap=0.0, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(8, 1, 256), (8, 1, 512), (32, 8, 128), (16, 4, 64), (12, 4, 128), (6, 6, 64)]


def draw(rng):
    kind = rng.choice(["append1", "append", "decode", "decode", "prompt", "logprobs"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    if kind == "append1":
        return dict(op="append", seqs=_log(rng, 1, 256), new=rng.choice([1, 1, 2, 5]), past=_log(rng, 1, 8192), hq=hq, hkv=hkv, d=d,
                    rot=d // rng.choice([1, 2, 4]), page=page, dtype=rng.choice(list(DTYPES)), ragged=True)
    if kind == "append":
        seqs = _log(rng, 1, 16)
        # no more tokens than the listed long prompt holds, by bytes
        new = _log(rng, 16, min(16384 // seqs, 16384 * 48 * 128 // ((hq + 2 * hkv) * d * 2 * seqs)))
        return dict(op="append", seqs=seqs, new=new, past=_log(rng, 1, 4096), hq=hq, hkv=hkv, d=d, rot=d // rng.choice([1, 2, 4]), page=page,
                    dtype=rng.choice(list(DTYPES)), ragged=rng.random() < 0.7)
    if kind == "decode":
        seqs = _log(rng, 1, 192)
        most = min(131071, 900_000_000 // (2 * hkv * d * seqs))
        return dict(op="attend", seqs=seqs, new=rng.choice([1, 1, 1, 2, 4]), past=_log(rng, 16, max(most, 64)), hq=hq, hkv=hkv, d=d, page=page,
                    window=rng.choice([0, 0, 512]), dtype=rng.choice(list(DTYPES)), ragged=rng.random() < 0.7)
    if kind == "prompt":
        seqs = _log(rng, 1, 8)
        new = _log(rng, 64, 4096 // seqs)
        past = _log(rng, 1, 8192)
        while new * (new + past) * seqs * hq * d > 4096 * 8192 * 32 * 128:  # no more than the listed chunk computes
            new, past = max(64, new * 2 // 3), past * 2 // 3
        return dict(op="attend", seqs=seqs, new=new, past=past, hq=hq, hkv=hkv, d=d, page=page, window=rng.choice([0, 512]),
                    dtype=rng.choice(["f16", "bf16"]), ragged=rng.random() < 0.7)
    vocab = rng.choice([262144, 128256, 32000, 50001])
    return dict(op="logprobs", rows=_log(rng, 1, 131_000_000 // vocab), vocab=vocab, top=rng.choice([1, 5, 20]), cap=rng.choice([0.0, 30.0]),
                dtype=rng.choice(["f32", "bf16"]) if vocab * 500 < 131_000_000 else "bf16")


def _lengths(case):
    """New tokens and cache lengths (the new ones included) of each sequence: the same for every seed, so a plan of the
    sizes can be kept.  Ragged: lengths from short to the case's, and one sequence in eight that has nothing in its
    cache (for `attend` not even its own token: a row that attends to nothing)."""
    new, kv = [], []
    for b in range(case["seqs"]):
        n, past = case["new"], case["past"]
        if case["ragged"]:
            share = ((b * 7 + 3) % 16 + 1) / 16
            past = int(past * share)
            n = max(1, int(n * (((b * 5 + 2) % 8 + 1) / 8))) if n > 1 else 1
            if b % 8 == 5:
                past = 0
        new.append(n)
        kv.append(0 if case["ragged"] and b % 8 == 5 and case["op"] == "attend" and n == 1 else past + n)
    return new, kv


# ---- inputs ------------------------------------------------------------------


def _scale_of(amax):
    """2^E, E the smallest with amax <= 448 * 2^E, within [-60, 60]."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -60)).clamp(-60, 60)
    return torch.ldexp(torch.ones_like(amax), e)


def _fill(pages, hkv, page, d, g, spread):
    """Codes and scales of a cache that earlier tokens left: normal values, a few channels larger than the others."""
    codes = torch.empty(pages, hkv, page, d, dtype=torch.float8_e4m3fn, device=DEV)
    scales = torch.empty(pages, hkv, page // BLOCK, dtype=torch.float32, device=DEV)
    channel = torch.ones(hkv, 1, d, device=DEV)
    channel[:, :, :: max(1, d // 4)] = spread
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, pages, step):
        k = min(step, pages - i)
        x = torch.randn(k, hkv, page, d, device=DEV, generator=g) * channel
        x = x.view(k, hkv, page // BLOCK, BLOCK * d)
        s = _scale_of(x.abs().amax(-1))
        scales[i : i + k] = s
        codes[i : i + k] = (x / s.unsqueeze(-1)).to(torch.float8_e4m3fn).view(k, hkv, page, d)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logprobs":
        # logits of a language model: a broad bulk, a few likely tokens; the given tokens are likely ones and others
        x = torch.randn(case["rows"], case["vocab"], device=DEV, generator=g) * 2.5
        at = torch.randint(0, case["vocab"], (case["rows"], 8), device=DEV, generator=g)
        x.scatter_add_(1, at, 12 * torch.rand(case["rows"], 8, device=DEV, generator=g))
        s["logits"] = x.to(DTYPES[case["dtype"]])
        other = torch.randint(0, case["vocab"], (case["rows"],), device=DEV, generator=g)
        s["tokens"] = torch.where(torch.rand(case["rows"], device=DEV, generator=g) < 0.7, at[:, 0], other).to(torch.int32)
    else:
        new, kv = _lengths(case)
        page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
        dt = DTYPES[case["dtype"]]
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        t = start[-1]
        per = [max(1, -(-k // page)) for k in kv]
        cols, pages = max(per), sum(per)
        # pages in no order, as a server's free list leaves them
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        used = torch.arange(cols, device=DEV)[None, :] < torch.tensor(per, device=DEV)[:, None]
        s["block_table"] = torch.zeros(len(new), cols, dtype=torch.int32, device=DEV)
        s["block_table"][used] = order
        s["q_start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device=DEV)
        s["max_q"], s["max_kv"] = max(new), max(kv)
        s["q"] = torch.randn(t, hq, d, device=DEV, generator=g).to(dt)
        s["k_codes"], s["k_scale"] = _fill(pages, hkv, page, d, g, 4.0)
        s["v_codes"], s["v_scale"] = _fill(pages, hkv, page, d, g, 1.0)
        if case["op"] == "append":
            s["k"] = (torch.randn(t, hkv, d, device=DEV, generator=g) * 1.5).to(dt)
            s["v"] = torch.randn(t, hkv, d, device=DEV, generator=g).to(dt)
            pos = torch.arange(max(kv), dtype=torch.float64, device=DEV)
            freq = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
            ang = pos[:, None] * freq[None, :]
            s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float()  # [positions, rot / 2, 2]
            s["q_out"] = torch.empty_like(s["q"])
        else:
            s["out"] = torch.empty_like(s["q"])
    if own:
        # the context and the cache's handle, which a program makes once
        here = os.path.join(os.getcwd(), "gemma4-webgpu_b200")
        if here not in sys.path:
            sys.path.insert(0, here)
        import q4k

        s["ctx"] = q4k.context(0)
        if "k_codes" in s:
            s["cache"] = q4k.KVCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass ----------------------------------------------------------------


def run(s):
    c = s["case"]
    if c["op"] == "append":
        if own:
            q = s["ctx"].kv_append(s["cache"], s["k"], s["v"], s["rope"], s["block_table"], s["q_start"], s["kv_len"], q=s["q"], q_out=s["q_out"])
        else:
            q = _plain_append(s)
        return {"q": q, "k": s["k_codes"], "v": s["v_codes"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if c["op"] == "attend":
        if own:
            return s["ctx"].paged_attention(s["cache"], s["q"], s["block_table"], s["q_start"], s["kv_len"], s["max_q"], c["d"] ** -0.5,
                                            window=c["window"], out=s["out"])
        return _plain_attend(s)
    if own:
        lp, ent, tv, ti = s["ctx"].token_logprobs(s["logits"], s["tokens"], top=c["top"], cap=c["cap"])
    else:
        lp, ent, tv, ti = _plain_logprobs(s)
    return {"logprob": lp, "entropy": ent, "top_logprob": tv, "top_token": ti}


def _positions(s):
    """Each token's sequence and position."""
    t = s["q"].shape[0]
    tok = torch.arange(t, device=DEV)
    seq = (s["q_start"][None, 1:] <= tok[:, None]).sum(1)
    pos = s["kv_len"][seq] - s["q_start"][seq + 1] + tok
    return seq, pos


def _rotate(x, cos, sin):
    h = cos.shape[-1]
    a, b, rest = x[..., :h], x[..., h : 2 * h], x[..., 2 * h :]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_append(s):
    page = s["case"]["page"]
    seq, pos = _positions(s)
    cs = s["rope"][pos]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    at = s["block_table"][seq, pos // page].long() * (page // BLOCK) + pos % page // BLOCK  # 16-token block of each token
    # a block whose first token comes now is new; else it keeps what it holds, under a scale that may grow
    fresh = torch.zeros(s["k_scale"].shape[0] * (page // BLOCK), dtype=torch.bool, device=DEV)
    fresh[at[pos % BLOCK == 0]] = True
    for x, codes, scale in ((_rotate(s["k"].float(), cos, sin), s["k_codes"], s["k_scale"]), (s["v"].float(), s["v_codes"], s["v_scale"])):
        pages, hkv, _, d = codes.shape
        amax = torch.zeros(fresh.shape[0], hkv, device=DEV)
        amax.scatter_reduce_(0, at[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
        old = scale.transpose(1, 2).reshape(-1, hkv)
        need = _scale_of(amax)
        grown = torch.where(fresh[:, None], need, torch.maximum(old, need))
        touched = torch.zeros_like(fresh)
        touched[at] = True
        grown = torch.where(touched[:, None], grown, old)
        rows = touched.nonzero()[:, 0]
        by_block = codes.view(pages, hkv, page // BLOCK, BLOCK, d).transpose(1, 2)  # [pages, blocks, heads, 16, d]
        pb, bb = rows // (page // BLOCK), rows % (page // BLOCK)
        held = by_block[pb, bb].float() * (old[rows] / grown[rows])[:, :, None, None]
        by_block.view(torch.uint8)[pb, bb] = held.to(torch.float8_e4m3fn).view(torch.uint8)
        code = (x / grown[at][:, :, None]).to(torch.float8_e4m3fn)
        by_block.view(torch.uint8)[at // (page // BLOCK), at % (page // BLOCK), :, pos % BLOCK] = code.view(torch.uint8)
        scale.copy_(grown.view(pages, page // BLOCK, hkv).transpose(1, 2))
    s["q_out"].copy_(_rotate(s["q"].float(), cos, sin))
    return s["q_out"]


def _plain_attend(s):
    c = s["case"]
    page, hq, hkv, d = c["page"], c["hq"], c["hkv"], c["d"]
    nb, n = s["kv_len"].shape[0], s["max_q"]
    cols = -(-max(1, s["max_kv"]) // page)

    def values(codes, scale):
        at = s["block_table"][:, :cols].long()
        x = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scale[at].repeat_interleave(BLOCK, -1)[..., None]
        return x.transpose(1, 2).reshape(nb, hkv, cols * page, d)

    count = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(n, device=DEV)
    tok = (s["q_start"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"].float()[tok].view(nb, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(nb, hkv, -1, d)
    k, v = values(s["k_codes"], s["k_scale"]), values(s["v_codes"], s["v_scale"])
    score = torch.matmul(q, k.transpose(2, 3)).view(nb, hkv, hq // hkv, n, -1) * d**-0.5
    pos = s["kv_len"][:, None] - count[:, None] + i
    j = torch.arange(cols * page, device=DEV)
    seen = (j <= pos[..., None]) & (j < s["kv_len"][:, None, None])
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill_((j >= s["kv_len"][:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(nb, hkv, -1, cols * page), v).view(nb, hkv, hq // hkv, n, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(nb, n, hq, d)
    return o[i < count[:, None]].to(s["q"].dtype)


def _plain_logprobs(s):
    c = s["case"]
    raw = s["logits"].float()
    x = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    entropy = lse - (e * x).sum(1, keepdim=True) / total
    logprob = x.gather(1, s["tokens"].long()[:, None]) - lse
    # the largest logits, the lowest index first among equals: a whole-number key that holds both
    bits = (raw + 0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) + (c["vocab"] - torch.arange(c["vocab"], device=DEV))
    at = torch.topk(key, c["top"], dim=1).values
    at = c["vocab"] - (at & 0xFFFFFFFF)
    return logprob[:, 0], entropy[:, 0], x.gather(1, at) - lse, at.to(torch.int32)


# ---- what a pass cannot do without -----------------------------------------------


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("dtype", "f32")]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": n * (5 + (4 if case["cap"] else 0))}
    new, kv = _lengths(case)
    t, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        tables = sum(min(n, k) for n, k in zip(new, kv)) * case["rot"] * 4
        return {"bytes": t * ((2 * hq + 2 * hkv) * d * size + 2 * hkv * d) + tables + 2 * hkv * 4 * (t // BLOCK + len(new)),
                "flops": t * d * (3 * hq + 8 * hkv)}
    read = pairs = 0
    for n, k in zip(new, kv):
        w = case["window"] or k + 1
        first = max(0, k - n - w + 1) if k else 0
        read += k - first
        # positions k - n .. k - 1, each seeing min(position + 1, window) keys
        full = max(0, min(n, k - w + 1)) if w <= k else 0
        rest = n - full
        pairs += full * w + (sum(range(k - n + 1, k - n + rest + 1)) if k >= n else 0)
    return {"bytes": read * hkv * (2 * d + 8 / BLOCK) + 2 * t * hq * d * size, "flops": 4 * d * hq * pairs}


# ---- the definitions in 64 bits ------------------------------------------------


def _f64_scale(amax):
    """The power of two of a block, from the logarithm in whole numbers."""
    out = torch.full_like(amax, 2.0**-60)
    for e in range(-60, 61):
        out = torch.where(amax > 448.0 * 2.0 ** (e - 1), torch.full_like(amax, 2.0**e), out)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        lp, ent, tv, ti = [], [], [], []
        for raw, tok in zip(s["logits"].split(64), s["tokens"].split(64)):
            x = raw.double()
            order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : case["top"]]
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            logp = torch.log_softmax(x, 1)
            lp.append(logp[torch.arange(len(tok), device=DEV), tok.long()])
            ent.append(-(logp.exp() * logp).sum(1))
            tv.append(torch.gather(logp, 1, order))
            ti.append(order.int())
        return {"logprob": torch.cat(lp), "entropy": torch.cat(ent), "top_logprob": torch.cat(tv), "top_token": torch.cat(ti)}
    new, kv = _lengths(case)
    page, hq, hkv, d = case["page"], case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        t = sum(new)
        p = torch.cat([torch.arange(k - n, k, device=DEV) for n, k in zip(new, kv)])
        tab = s["rope"].double()[p]
        z = torch.complex(tab[..., 0], tab[..., 1])[:, None, :]
        half = case["rot"] // 2

        def turn(x):
            x = x.double().clone()
            y = torch.complex(x[..., :half], x[..., half : 2 * half]) * z
            x[..., :half], x[..., half : 2 * half] = y.real, y.imag
            return x

        # The scales follow from the definition; a code is whole steps of its scale, so no 64-bit value stands in its place.
        scales = {}
        for name, x in (("k_scale", turn(s["k"])), ("v_scale", s["v"].double())):
            out = s[name].double()
            amax = x.abs().amax(-1)
            t0 = 0
            for b, (n, k) in enumerate(zip(new, kv)):
                lo = (k - n) // BLOCK * BLOCK
                padded = torch.zeros(-(-(k - lo) // BLOCK) * BLOCK, hkv, dtype=torch.float64, device=DEV)
                padded[k - n - lo : k - lo] = amax[t0 : t0 + n]
                need = _f64_scale(padded.view(-1, BLOCK, hkv).amax(1))
                blk = torch.arange(lo // BLOCK, lo // BLOCK + need.shape[0], device=DEV)
                pg = s["block_table"][b, blk * BLOCK // page].long()
                sub = blk % (page // BLOCK)
                if (k - n) % BLOCK:
                    need[0] = torch.maximum(need[0], out[pg[0], :, sub[0]])
                out[pg, :, sub] = need
                t0 += n
            scales[name] = out
        return {"q": turn(s["q"]), "k": None, "v": None, **scales}
    outs = []
    t0 = 0
    for b, (n, k) in enumerate(zip(new, kv)):
        o = torch.zeros(n, hq, d, dtype=torch.float64, device=DEV)
        first = max(0, k - n - case["window"] + 1) // page * page if case["window"] else 0
        if k:
            pg = s["block_table"][b, first // page : -(-k // page)].long()
            j = torch.arange(first, k, device=DEV)
            p = torch.arange(k - n, k, device=DEV)
            ok = j[None, :] <= p[:, None]
            if case["window"]:
                ok &= p[:, None] - j[None, :] < case["window"]
            for h in range(hkv):
                kk, vv = (
                    (s[a].view(torch.uint8)[pg, h].view(torch.float8_e4m3fn).double().view(-1, BLOCK, d) * s[a[0] + "_scale"][pg, h].double().view(-1, 1, 1))
                    .reshape(-1, d)[: k - first]
                    for a in ("k_codes", "v_codes")
                )
                for r in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    a = s["q"][t0 : t0 + n, r].double() @ kk.T / math.sqrt(d)
                    o[:, r] = torch.softmax(a.masked_fill(~ok, -math.inf), 1) @ vv
        outs.append(o)
        t0 += n
    return torch.cat(outs)
