"""Measured cases of the ragged-batch attention operators: appending to a paged
key/value cache (`kv_append`), attention of new tokens over that cache
(`attention_paged`) and attention over packed whole prompts
(`attention_packed`).

`own = False` computes each operator in its plain form (elementary torch
operations in 32 bits, rounded once at the end); `own = True` makes the calls a
user of `burn_rocket_b200` makes.

A batch's lengths follow from the case alone (`lengths`), its values and its
page order from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
THETA = 1e6


def listed():
    """Head layouts 16/8 and 32/4 x 128 and 16/16 x 72 are those of the
    repository's own models; 32/4 x 64 is a generic narrow-head one."""
    return [
        # One decode step of a small serving batch: the new token of each
        # sequence is normed, rotated and stored. All latency.
        case("append_decode", "append", "f16", 16, 8, 128, 16, 32, (1, 1), (20, 2000), norms=True, mix=1),
        # Prompts of a prefill batch on their way into the cache; no q/k norm.
        case("append_prompt", "append", "bf16", 32, 4, 64, 64, 24, (150, 1601), (150, 2200), mix=2),
        # One sequence, one token: the smallest call a chat makes.
        case("decode_one", "paged", "f16", 16, 8, 128, 16, 1, (1, 1), (1437, 1437), mix=3),
        # A serving batch of very different lengths, eight query heads a KV head.
        case("decode_batch", "paged", "bf16", 32, 4, 128, 64, 64, (1, 1), (33, 8100), mix=4),
        # Few sequences with long contexts: the context has to be split to fill the GPU.
        case("decode_long", "paged", "f16", 16, 8, 128, 128, 3, (1, 1), (21001, 32700), mix=5),
        # Checking a few drafted tokens at once, over a sliding window.
        case("verify", "paged", "bf16", 32, 4, 64, 32, 16, (2, 9), (300, 5000), window=1024, mix=6),
        # Chunked prefill: the next piece of some long prompts.
        case("chunk", "paged", "bf16", 32, 4, 128, 32, 4, (512, 512), (1800, 8190), mix=7),
        # Prefill and decode in one batch: two prompt pieces among single tokens.
        case("mixed", "paged", "f16", 16, 8, 128, 16, 24, (1, 1), (40, 4050), chunks=2, chunk_len=701, mix=8),
        # A handful of short prompts.
        case("packed_small", "packed", "f16", 16, 8, 128, 0, 7, (1, 90), None, mix=9),
        # An image batch of different sizes through a tower: bidirectional, 72-wide heads.
        case("packed_images", "packed", "f16", 16, 16, 72, 0, 9, (300, 2394), None, causal=False, mix=10),
        # An embedding batch: many prompts of a few hundred tokens.
        case("packed_embed", "packed", "f16", 16, 8, 128, 0, 64, (37, 988), None, mix=11),
        # Long prompts, prefilled whole.
        case("packed_long", "packed", "bf16", 32, 4, 128, 0, 4, (901, 5003), None, mix=12),
    ]


def case(name, op, dtype, heads, kv_heads, dim, page, batch, q, kv, norms=False, window=-1, softcap=0.0, causal=True,
         chunks=0, chunk_len=0, mix=0):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch,
         "q_min": q[0], "q_max": q[1], "mix": mix}
    if name:
        c["name"] = name
    if op != "packed":
        c.update(page=page, kv_min=kv[0], kv_max=kv[1])
    if op == "append":
        c["norms"] = norms
    else:
        c.update(window=window, softcap=softcap)
    if op == "paged":
        c.update(chunks=chunks, chunk_len=chunk_len)
    if op == "packed":
        c["causal"] = causal
    return c


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(cost(c) for c in listed())
    while True:
        c = draw_any(rng)
        # the plain form holds whole padded score matrices
        q, kv = lengths(c)
        scores = 0 if c["op"] == "append" else c["batch"] * c["heads"] * max(q) * max(kv)
        held = 0 if c["op"] == "packed" else sum(kv) * c["kv_heads"] * c["dim"]
        if cost(c) <= top and scores <= 3.2e9 and held <= 4e8:
            return c


def draw_any(rng):
    op = rng.choice(["append", "paged", "paged", "packed"])
    dtype = rng.choice(["f16", "bf16"])
    heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 4, 128), (32, 4, 64), (8, 8, 64), (12, 4, 128),
                                       (14, 2, 64), (8, 1, 128)])
    mix = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        batch = log_int(rng, 1, 128)
        top = log_int(rng, 1, 1800) if rng.random() < 0.6 else 1
        q = (max(1, top // rng.randint(1, 9)), top)
        kv = (q[1], q[1] + log_int(rng, 1, 4000))
        return case(None, op, dtype, heads, kv_heads, dim, page, batch, q, kv, norms=rng.random() < 0.6, mix=mix)
    window = log_int(rng, 16, 4096) if rng.random() < 0.25 else -1
    softcap = 30.0 if rng.random() < 0.1 else 0.0
    if op == "packed":
        causal = rng.random() < 0.75
        if rng.random() < 0.2:
            heads, kv_heads, dim, causal = 16, 16, 72, False
        top = log_int(rng, 1, 6000)
        batch = log_int(rng, 1, max(1, min(96, 40000 // top)))
        return case(None, op, dtype, heads, kv_heads, dim, 0, batch, (max(1, top // rng.randint(1, 12)), top), None,
                    window=window, softcap=softcap, causal=causal, mix=mix)
    kind = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
    kv_top = log_int(rng, 10, 32768)
    kv = (max(1, kv_top // rng.randint(1, 40)), kv_top)
    batch = log_int(rng, 1, 96)
    if kind == "decode":
        return case(None, op, dtype, heads, kv_heads, dim, page, batch, (1, 1), kv, window=window, softcap=softcap,
                    mix=mix)
    if kind == "verify":
        return case(None, op, dtype, heads, kv_heads, dim, page, batch, (2, rng.randint(2, 16)), kv, window=window,
                    softcap=softcap, mix=mix)
    if kind == "chunk":
        top = log_int(rng, 17, 2048)
        batch = log_int(rng, 1, 16)
        return case(None, op, dtype, heads, kv_heads, dim, page, batch, (max(1, top // rng.randint(1, 4)), top),
                    (kv[0] + top, kv[1] + top), window=window, softcap=softcap, mix=mix)
    return case(None, op, dtype, heads, kv_heads, dim, page, max(2, batch // 2), (1, 1), kv, window=window,
                softcap=softcap, chunks=rng.randint(1, 2), chunk_len=log_int(rng, 17, 1024), mix=mix)


def lengths(c):
    """New tokens and total keys of each sequence."""
    r = random.Random(c["mix"])
    q = [r.randint(c["q_min"], c["q_max"]) for _ in range(c["batch"])]
    q[r.randrange(len(q))] = c["q_max"]
    if c["op"] == "packed":
        return q, list(q)
    kv = [r.randint(c["kv_min"], c["kv_max"]) for _ in q]
    kv[r.randrange(len(kv))] = c["kv_max"]
    for at in range(c.get("chunks", 0)):
        q[at * (len(q) // 2)] = c["chunk_len"]
    return q, [max(a, b) for a, b in zip(q, kv)]


def pairs(c):
    """(query, key) pairs that the mask lets through, and the keys that any query of its sequence sees."""
    total = seen = 0
    w = c["window"]
    for n, m in zip(*lengths(c)):
        if not c.get("causal", True):
            if w < 0:
                total += n * m
            else:
                total += sum(min(m - 1, i + w) - max(0, i - w) + 1 for i in range(n))
            seen += m
            continue
        first = m - n
        if w < 0:
            total += n * first + n * (n + 1) // 2
            seen += m
        else:
            total += sum(min(i + 1, w) for i in range(first, m))
            seen += m - max(0, first - w + 1)
    return total, seen


def work(c):
    q, kv = lengths(c)
    tokens, row = sum(q), 2 * c["dim"]
    if c["op"] == "append":
        positions = len({p for n, m in zip(q, kv) for p in range(m - n, m)})
        moved = 2 * tokens * (c["heads"] + 2 * c["kv_heads"]) * row
        table = sum(-(-m // c["page"]) - (m - n) // c["page"] for n, m in zip(q, kv))
        moved += positions * c["dim"] * 4 + 4 * table + 8 * c["batch"]
        rotated = tokens * (c["heads"] + c["kv_heads"]) * c["dim"]
        return {"bytes": moved, "flops": rotated * (7 if c["norms"] else 3)}
    total, seen = pairs(c)
    table = sum(-(-m // c["page"]) for m in kv) if c["op"] == "paged" else 0
    return {"bytes": 2 * tokens * c["heads"] * row + 2 * seen * c["kv_heads"] * row + 4 * table + 8 * c["batch"],
            "flops": 4 * total * c["heads"] * c["dim"]}


def cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def prepare(c, seed):
    dev, dt = "cuda", DTYPES[c["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    q, kv = lengths(c)
    tokens, heads, kvh, d = sum(q), c["heads"], c["kv_heads"], c["dim"]
    s = {"case": c, "q_len": q, "kv": kv, "scale": 1.0 / math.sqrt(d), "max_q": max(q), "max_kv": max(kv),
         "cu": torch.tensor([0] + q, device=dev).cumsum(0).to(torch.int32),
         "kv_len": torch.tensor(kv, device=dev, dtype=torch.int32)}
    if c["op"] == "paged":
        s["q"] = torch.randn(tokens, heads * d, device=dev, generator=g).to(dt)
    else:  # column slices of one fused q|k|v projection output
        fused = torch.randn(tokens, (heads + 2 * kvh) * d, device=dev, generator=g).to(dt)
        s["q"], s["k"], s["v"] = fused.split([heads * d, kvh * d, kvh * d], dim=1)
    if c["op"] == "packed":
        return s
    # The cache's pages lie in any order, and a few belong to others.
    used = [-(-m // c["page"]) for m in kv]
    pages = sum(used) + 5
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32).cpu().tolist()
    table = torch.full((len(kv), max(used) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s["table"] = table.to(dev)
    shape = (pages, c["page"], kvh, d)
    s["k_cache"] = torch.randn(shape, device=dev, generator=g, dtype=torch.float32).to(dt)
    s["v_cache"] = torch.randn(shape, device=dev, generator=g, dtype=torch.float32).to(dt)
    if c["op"] == "append":
        inv = THETA ** (-torch.arange(d // 2, device=dev, dtype=torch.float64) * 2 / d)
        angle = torch.arange(max(kv), device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["norms"] = [None, None]
        if c["norms"]:
            s["norms"] = [1.0 + 0.1 * torch.randn(d, device=dev, generator=g) for _ in range(2)]
        s["q_out"] = torch.zeros(tokens, heads * d, device=dev, dtype=dt)
    else:
        s["out"] = torch.zeros(tokens, heads * d, device=dev, dtype=dt)
    return s


def run(s):
    c = s["case"]
    if own:
        import burn_rocket_b200 as rb
        rb.init(0)
        heads, kvh, d = c["heads"], c["kv_heads"], c["dim"]
        if c["op"] == "append":
            rb.kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["kv_len"], heads,
                         kvh, d, s["cos"], s["sin"], q_norm=s["norms"][0], k_norm=s["norms"][1], eps=EPS,
                         q_out=s["q_out"])
            return s["q_out"], s["k_cache"], s["v_cache"]
        if c["op"] == "paged":
            return rb.attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["kv_len"], heads, kvh,
                                      d, s["scale"], max_q=s["max_q"], max_kv=s["max_kv"], softcap=c["softcap"], window=c["window"],
                                      out=s["out"])
        return rb.attention_packed(s["q"], s["k"], s["v"], s["cu"], heads, kvh, d, s["scale"],
                                   softcap=c["softcap"], is_causal=c["causal"], window=c["window"])
    return {"append": plain_append, "paged": plain_paged, "packed": plain_packed}[c["op"]](s)


# ---------------------------------------------------------------- plain forms
def token_places(s):
    """Sequence and position of each new token."""
    cu, kv = s["cu"].long(), s["kv_len"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n)
    return seq, torch.arange(s["q"].shape[0], device=n.device) - cu[seq] + (kv - n)[seq]


def normed_rotated(x, weight, cos, sin):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def plain_append(s):
    c = s["case"]
    heads, kvh, d, page, dt = c["heads"], c["kv_heads"], c["dim"], c["page"], s["q"].dtype
    seq, pos = token_places(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = normed_rotated(s["q"].reshape(-1, heads, d), s["norms"][0], cos, sin)
    k = normed_rotated(s["k"].reshape(-1, kvh, d), s["norms"][1], cos, sin)
    at = s["table"][seq, pos // page].long(), pos % page
    s["k_cache"][at] = k.to(dt)
    s["v_cache"][at] = s["v"].reshape(-1, kvh, d)
    s["q_out"].copy_(q.reshape(-1, heads * d))
    return s["q_out"], s["k_cache"], s["v_cache"]


def plain_attention(q, k, v, seen, c, scale):
    """q [B, Q, H, D], k and v [B, K, KV, D], seen [B, Q, K] -> [B, Q, H, D], all f32."""
    b, n, heads, d = q.shape
    q = q.reshape(b, n, c["kv_heads"], -1, d).permute(0, 2, 3, 1, 4)      # B KV G Q D
    s = q @ k.permute(0, 2, 3, 1)[:, :, None] * scale                     # B KV G Q K
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True).clamp_min_(-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = s @ v.permute(0, 2, 1, 3)[:, :, None] / torch.where(total > 0, total, 1)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)


def in_band(pos, key, c):
    """Whether the query at `pos` sees `key` under the case's mask."""
    w = c["window"]
    if c.get("causal", True):
        return (key <= pos) & (key > pos - w) if w >= 0 else key <= pos
    return (key - pos).abs() <= w if w >= 0 else key >= 0


def plain_paged(s):
    c = s["case"]
    heads, d, page = c["heads"], c["dim"], c["page"]
    seq, pos = token_places(s)
    n = s["cu"].diff().long()
    first = s["kv_len"].long() - n
    at = seq, pos - first[seq]
    q = torch.zeros(len(n), s["max_q"], heads, d, device=n.device)
    q[at] = s["q"].reshape(-1, heads, d).float()
    k, v = (s[x][s["table"].clamp_min(0).long()].flatten(1, 2).float() for x in ("k_cache", "v_cache"))
    key = torch.arange(k.shape[1], device=n.device)[None, None]
    place = (torch.arange(s["max_q"], device=n.device) + first[:, None])[:, :, None]
    o = plain_attention(q, k, v, in_band(place, key, c) & (key < s["kv_len"][:, None, None]), c, s["scale"])
    return o[at].reshape(-1, heads * d).to(s["q"].dtype)


def plain_packed(s):
    c = s["case"]
    heads, kvh, d = c["heads"], c["kv_heads"], c["dim"]
    cu = s["cu"].long()
    n = cu.diff()
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n)
    at = seq, torch.arange(s["q"].shape[0], device=n.device) - cu[seq]

    def padded(x, h):
        y = torch.zeros(len(n), s["max_q"], h, d, device=x.device)
        y[at] = x.reshape(-1, h, d).float()
        return y

    key = torch.arange(s["max_q"], device=n.device)
    seen = in_band(key[:, None], key, c)[None] & (key < n[:, None])[:, None]
    o = plain_attention(padded(s["q"], heads), padded(s["k"], kvh), padded(s["v"], kvh), seen, c, s["scale"])
    return o[at].reshape(-1, heads * d).to(s["q"].dtype)


# ---------------------------------------------------------------- 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    q_len, kv, heads, kvh, d = s["q_len"], s["kv"], c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "append":
        half, page = d // 2, c["page"]
        table = s["table"].cpu().tolist()
        new = [x.double() for x in (s["q"].reshape(-1, heads, d), s["k"].reshape(-1, kvh, d),
                                    s["v"].reshape(-1, kvh, d))]
        for i, w in enumerate(s["norms"]):
            if w is not None:
                new[i] = new[i] / (new[i].pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        k_cache, v_cache, at = s["k_cache"].double(), s["v_cache"].double(), 0
        q_out = torch.empty_like(new[0])
        for b, (n, m) in enumerate(zip(q_len, kv)):
            cos, sin = s["cos"][m - n:m].double()[:, None], s["sin"][m - n:m].double()[:, None]
            turned = []
            for x in (new[0][at:at + n], new[1][at:at + n]):
                y = torch.empty_like(x)
                y[..., :half] = x[..., :half] * cos - x[..., half:] * sin
                y[..., half:] = x[..., half:] * cos + x[..., :half] * sin
                turned.append(y)
            q_out[at:at + n] = turned[0]
            p = m - n
            while p < m:  # one page's slots at a time
                e = min(m, (p // page + 1) * page)
                here = slice(p - (m - n), e - (m - n))
                k_cache[table[b][p // page], p % page:p % page + e - p] = turned[1][here]
                v_cache[table[b][p // page], p % page:p % page + e - p] = new[2][at:at + n][here]
                p = e
            at += n
        return q_out.reshape(-1, heads * d), k_cache, v_cache
    out, at, group = [], 0, heads // kvh
    for b, (n, m) in enumerate(zip(q_len, kv)):
        q = s["q"][at:at + n].reshape(n, heads, d)
        if c["op"] == "paged":
            rows = s["table"][b, :-(-m // c["page"])].long()
            k, v = (s[x][rows].reshape(-1, kvh, d)[:m] for x in ("k_cache", "v_cache"))
        else:
            k, v = (s[x][at:at + m].reshape(m, kvh, d) for x in ("k", "v"))
        pos = torch.arange(m - n, m, device=q.device)[:, None]
        key = torch.arange(m, device=q.device)[None]
        w = c["window"]
        hidden = torch.zeros(n, m, dtype=torch.bool, device=q.device)
        if c.get("causal", True):
            hidden |= key > pos
        if w >= 0:
            hidden |= (pos - key >= w) if c.get("causal", True) else ((pos - key).abs() > w)
        o = torch.empty(n, heads, d, device=q.device, dtype=torch.float64)
        for h in range(heads):
            x = q[:, h].double().mm(k[:, h // group].double().t()).mul_(s["scale"])
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            o[:, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1).nan_to_num_(0.0) @ v[:, h // group].double()
        out.append(o.reshape(n, heads * d))
        at += n
    return torch.cat(out)
