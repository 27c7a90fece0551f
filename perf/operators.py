"""The operators of the 4-bit KV cache and of sliding-window attention: their cases, plain forms and 64-bit definitions.

4-bit cache.  The D elements of one (token, KV head) of K or V are held as codes c in 0..15 with one bf16 pair
(scale s, offset z) for each group of 64 elements; an element stands for s * c + z.  For a group with least element a
and largest b: s = bf16((b - a) / 15), z = bf16(a), c = round((x - z) / s) clamped to 0..15 (0 where s is 0).  A row of
codes is D / 8 little-endian 32-bit words; word 2 i + h holds elements 8 i + h D / 2 and the seven after it, element j
in bits 4 j .. 4 j + 3.

Attention.  Key n (at position kn) is visible to a query at position p iff kn <= p and, with a window W > 0,
p - kn < W or kn < sinks.  out = sum_n softmax_n(scale * <R(p - delta) q, k_n>) v_n over the visible keys, 0 where there
are none; delta is how far the key's segment lies from where its keys were rotated when they were cached.
"""
import math

import torch

own = False

GROUP = 64


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's new tokens of 8 requests (Llama-3-8B heads): latency alone
        dict(name="append-decode-8", op="append", tokens=8, q_heads=32, kv_heads=8, dim=128, page=256, norm=False),
        # a long prompt of a model with q/k norms (Qwen3-0.6B heads), an odd length
        dict(name="append-prompt-qknorm", op="append", tokens=8191, q_heads=16, kv_heads=8, dim=128, page=256,
             norm=True),
        # a short chunk, TinyLlama heads, small pages
        dict(name="append-chunk-d64", op="append", tokens=777, q_heads=32, kv_heads=4, dim=64, page=16, norm=False),
        # one request, a short context: the smallest attention call
        dict(name="int4-decode-1", op="attend", bits=4, batch=1, q_heads=16, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=600, past_hi=600, q_lo=1, q_hi=1, window=0, sinks=0),
        # the headline decode batch: 8 requests at 2048-token prompts
        dict(name="int4-decode-8", op="attend", bits=4, batch=8, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=2048, past_hi=2176, q_lo=1, q_hi=1, window=0, sinks=0),
        # a full serving batch with long ragged contexts: what the 4-bit cache is for
        dict(name="int4-decode-64-long", op="attend", bits=4, batch=64, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=4001, past_hi=16001, q_lo=1, q_hi=1, window=0, sinks=0),
        # a 64-token query over three cached 1024-token chunks placed away from where they were cached (TinyLlama)
        dict(name="int4-query-over-chunks", op="attend", bits=4, batch=1, q_heads=32, kv_heads=4, dim=64, page=256,
             chunks=3, chunk_len=1024, past_lo=0, past_hi=0, q_lo=64, q_hi=64, window=0, sinks=0),
        # a whole prompt against its own 4-bit cache
        dict(name="int4-prompt", op="attend", bits=4, batch=1, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=0, past_hi=0, q_lo=4000, q_hi=4000, window=0, sinks=0),
        # a small decode batch of a windowed model, D 64, small pages, a window that ends inside a page
        dict(name="window-decode-4-d64", op="attend", bits=16, batch=4, q_heads=32, kv_heads=4, dim=64, page=16,
             chunks=0, chunk_len=0, past_lo=700, past_hi=5000, q_lo=1, q_hi=1, window=500, sinks=4),
        # a serving batch far past its window
        dict(name="window-decode-32", op="attend", bits=16, batch=32, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=5000, past_hi=9000, q_lo=1, q_hi=1, window=4096, sinks=4),
        # two ragged prompts longer than the window
        dict(name="window-prompt", op="attend", bits=16, batch=2, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=0, past_hi=0, q_lo=3500, q_hi=4096, window=1024, sinks=4),
        # both together: long contexts in 4 bits read through a window
        dict(name="int4-window-decode-16", op="attend", bits=4, batch=16, q_heads=32, kv_heads=8, dim=128, page=256,
             chunks=0, chunk_len=0, past_lo=9000, past_hi=30000, q_lo=1, q_hi=1, window=8192, sinks=16),
    ]


HEADS = ((32, 8, 128), (16, 8, 128), (32, 4, 64), (64, 8, 128), (12, 12, 64), (20, 4, 128))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice((16, 48, 256))
    kind = rng.choice(("append", "decode", "decode", "window", "window", "query", "prompt"))
    if kind == "append":
        return dict(op="append", tokens=_log(rng, 1, 8000), q_heads=hq, kv_heads=hkv, dim=d, page=page,
                    norm=rng.random() < 0.5)
    case = dict(op="attend", bits=rng.choice((4, 16)) if kind == "window" else 4, q_heads=hq, kv_heads=hkv, dim=d,
                page=page, chunks=0, chunk_len=0, past_lo=0, past_hi=0, window=0, sinks=0)
    if kind in ("decode", "window"):
        hi = _log(rng, 64, 16000)
        case |= dict(batch=min(_log(rng, 1, 64), max(1, 400000 // hi)), past_lo=max(1, int(hi * rng.uniform(0.2, 1.0))),
                     past_hi=hi, q_lo=1, q_hi=1)
    elif kind == "query":
        case |= dict(batch=rng.choice((1, 1, 2)), chunks=rng.randint(0, 4), chunk_len=_log(rng, 100, 2000),
                     past_lo=_log(rng, 1, 500), past_hi=500, q_lo=rng.randint(1, 8), q_hi=_log(rng, 8, 300))
    else:
        hi = _log(rng, 100, 3500)
        case |= dict(batch=rng.choice((1, 2)) if hi < 2000 else 1, q_lo=max(1, hi - rng.randint(0, 99)), q_hi=hi)
    if kind == "window" or (kind in ("query", "prompt") and rng.random() < 0.4):
        case |= dict(window=_log(rng, 16, 8000), sinks=rng.choice((0, 1, 4, 64)))
        if kind != "window":
            case["bits"] = rng.choice((4, 16))
    return case


def _spread(lo, hi, n):
    """n lengths in [lo, hi], the first hi; the same for every seed."""
    return [hi - int((hi - lo) * ((0.6180339887 * b) % 1.0)) for b in range(n)]


def _lengths(c):
    return _spread(c["past_lo"], c["past_hi"], c["batch"]), _spread(c["q_lo"], c["q_hi"], c["batch"])


# ---------------------------------------------------------------- inputs
def _tables(max_pos, dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    a = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _prepare_append(case, g) if case["op"] == "append" else _prepare_attend(case, g)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _cache4(g, pages, c):
    """A 4-bit pool as a running engine holds it: codes of bell-shaped values, some channels of K with larger steps."""
    kvh, ps, d = c["kv_heads"], c["page"], c["dim"]
    lo = (_randn(g, pages, 2, kvh, ps, d // 2, dtype=torch.float16) * 2.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    hi = (_randn(g, pages, 2, kvh, ps, d // 2, dtype=torch.float16) * 2.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    codes = lo | (hi << 4)
    s = 0.35 * torch.exp(0.2 * _randn(g, pages, 2, kvh, ps, d // GROUP))
    z = -7.5 * s + 0.1 * _randn(g, pages, 2, kvh, ps, d // GROUP)
    return codes, torch.stack([s, z], -1).bfloat16()


def _prepare_append(c, g):
    n, hq, hkv, d, ps = c["tokens"], c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    cos, sin = _tables(16384, d)
    decode = n <= 64
    pages = n if decode else -(-n // ps) + 1
    order = torch.randperm(pages + 2, generator=g, device="cuda")[:pages]
    if decode:  # one new token of each request, each at its own place of its own page
        slots = order * ps + torch.randint(0, ps, (n,), generator=g, device="cuda")
        pos = torch.randint(0, 16384, (n,), generator=g, device="cuda")
    else:       # one run of tokens that starts inside a page
        at = torch.arange(n, device="cuda") + min(5, ps - 1)
        slots = order[at // ps] * ps + at % ps
        pos = torch.arange(n, device="cuda") + 100
    gain = torch.exp(0.5 * _randn(g, hkv, d))
    gains = torch.cat([torch.ones(hq, d, device="cuda"), gain, torch.ones(hkv, d, device="cuda")]).reshape(-1)
    codes, scales = _cache4(g, pages + 2, c)
    return dict(case=c, qkv=(_randn(g, n, (hq + 2 * hkv) * d) * gains).bfloat16(), positions=pos.int(),
                slots=slots.int(), codes=codes, scales=scales, cos=cos, sin=sin,
                q_norm=(1 + 0.2 * _randn(g, d)).bfloat16() if c["norm"] else None,
                k_norm=(1 + 0.5 * _randn(g, d)).bfloat16() if c["norm"] else None)


def _prepare_attend(c, g):
    hq, hkv, d, ps, b = c["q_heads"], c["kv_heads"], c["dim"], c["page"], c["batch"]
    past, nq = _lengths(c)
    ctx = c["chunks"] * c["chunk_len"]
    segs, total_pages = [], 0  # of each sequence: (first page, keys, first position, delta)
    for i in range(b):
        mine = [(c["chunk_len"], j * c["chunk_len"], (37 * (j + 1)) % (j * c["chunk_len"] + 1)) for j in range(c["chunks"])]
        mine.append((past[i] + nq[i], ctx, 0))
        for n, p0, delta in mine:
            segs.append((i, total_pages, n, p0, delta))
            total_pages += -(-n // ps)
    order = torch.randperm(total_pages + 2, generator=g, device="cuda")[:total_pages]
    order_host = order.tolist()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    per_seq = [sum(1 for s in segs if s[0] == i) for i in range(b)]
    seg_indptr = [sum(per_seq[:i]) for i in range(b + 1)]
    pages_of = [-(-s[2] // ps) for s in segs]
    qo = [sum(nq[:i]) for i in range(b + 1)]
    positions = [ctx + past[i] + t for i in range(b) for t in range(nq[i])]
    # the same plan key by key
    most = max(ctx + past[i] + nq[i] for i in range(b))
    ar = torch.arange(most, device="cuda")
    key_slot = torch.zeros(b, most, dtype=torch.int64, device="cuda")
    key_pos = torch.full((b, most), 1 << 30, dtype=torch.int64, device="cuda")
    key_delta = torch.zeros(b, most, dtype=torch.int64, device="cuda")
    at = [0] * b
    for i, first, n, p0, delta in segs:
        k = ar[:n]
        key_slot[i, at[i]:at[i] + n] = order[first + k // ps] * ps + k % ps
        key_pos[i, at[i]:at[i] + n] = p0 + k
        key_delta[i, at[i]:at[i] + n] = delta
        at[i] += n
    most_q = max(nq)
    row = torch.arange(most_q, device="cuda")[None, :]
    q_len = torch.tensor(nq, device="cuda")[:, None]
    live = row < q_len
    q_index = torch.tensor(qo[:-1], device="cuda")[:, None] + torch.minimum(row, q_len - 1)
    cos, sin = _tables(most + 16, d)
    s = dict(case=c, q=_randn(g, qo[-1], hq, d).bfloat16(), cos=cos, sin=sin, scale=d ** -0.5,
             qo_indptr=i32(qo), positions=i32(positions), seg_indptr=i32(seg_indptr),
             seg_page_indptr=i32([sum(pages_of[:j]) for j in range(len(segs) + 1)]), seg_offset=i32([0] * len(segs)),
             seg_len=i32([x[2] for x in segs]), seg_pos0=i32([x[3] for x in segs]), seg_delta=i32([x[4] for x in segs]),
             page_ids=i32(order_host), max_q=most_q, max_kv=most, key_slot=key_slot, key_pos=key_pos,
             key_delta=key_delta, q_index=q_index, live=live)
    if c["bits"] == 4:
        s["codes"], s["scales"] = _cache4(g, total_pages + 2, c)
    else:
        s["kv"] = _randn(g, total_pages + 2, 2, hkv, ps, d, dtype=torch.bfloat16)
    return s


# ----------------------------------------------------------- plain forms
def _unpack(codes, scales):
    """[..., D/2] bytes and [..., D/64, 2] pairs to the values they stand for, fp32 [..., D]."""
    d = codes.shape[-1] * 2
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], d // 16, 2, 8)
    c = c.transpose(-3, -2).reshape(*codes.shape[:-1], d // GROUP, GROUP).float()
    s = scales.float()
    return (s[..., :1] * c + s[..., 1:]).reshape(*codes.shape[:-1], d)


def _pack(x):
    """fp32 [..., D] to codes and scales."""
    d = x.shape[-1]
    g = x.reshape(*x.shape[:-1], d // GROUP, GROUP)
    a, b = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, z = ((b - a) / 15).bfloat16(), a.bfloat16()
    step = s.float()
    c = torch.where(step > 0, (g - z.float()) / torch.where(step > 0, step, 1.0), 0.0).round().clamp(0, 15)
    c = c.to(torch.uint8).reshape(*x.shape[:-1], 2, d // 16, 8).transpose(-3, -2).reshape(*x.shape[:-1], d // 2, 2)
    return c[..., 0] | (c[..., 1] << 4), torch.cat([s, z], -1)


def _rotate(x, cos, sin):
    """x [..., heads, D] fp32, cos / sin [..., 1, D/2]."""
    h = x.shape[-1] // 2
    x1, x2 = x[..., :h], x[..., h:]
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()


def run(s):
    return _run_append(s) if s["case"]["op"] == "append" else _run_attend(s)


def _run_append(s):
    c = s["case"]
    hq, hkv, d, ps = c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from braidinfer_b200 import ops

        layer = ops.KV4Layer(s["codes"], s["scales"])
        q = ops.qkv_prepare(s["qkv"], s["positions"], s["slots"], layer, hq, hkv, d, s["cos"], s["sin"], s["q_norm"],
                            s["k_norm"], 1e-6)
        return {"q": q, "kv": ops.kv4_read(layer, s["slots"])}
    x = s["qkv"].view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv].float(), x[:, hq + hkv:].float()
    if c["norm"]:
        q, k = _norm(q.float(), s["q_norm"]).bfloat16(), _norm(k, s["k_norm"])
    p = s["positions"].long()
    k = _rotate(k, s["cos"][p][:, None], s["sin"][p][:, None])
    codes, scales = _pack(torch.stack([k, v], 1))
    pg, off = s["slots"].long() // ps, s["slots"].long() % ps
    s["codes"][pg, :, :, off] = codes
    s["scales"][pg, :, :, off] = scales
    return {"q": q, "kv": _unpack(s["codes"][pg, :, :, off], s["scales"][pg, :, :, off]).bfloat16()}


def _run_attend(s):
    c = s["case"]
    hq, hkv, d, ps = c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from braidinfer_b200 import ops

        meta = ops.AttnMeta(s["qo_indptr"], s["positions"], s["seg_indptr"], s["seg_page_indptr"], s["seg_offset"],
                            s["seg_len"], s["seg_pos0"], s["seg_delta"], s["page_ids"], c["batch"], s["max_q"],
                            s["max_kv"], decode=s["max_q"] == 1)
        layer = ops.KV4Layer(s["codes"], s["scales"]) if c["bits"] == 4 else s["kv"]
        return ops.attention(s["q"], layer, meta, s["cos"], s["sin"], s["scale"], window=c["window"], sinks=c["sinks"])
    pg, off = s["key_slot"] // ps, s["key_slot"] % ps
    if c["bits"] == 4:
        kv = _unpack(s["codes"][pg, :, :, off], s["scales"][pg, :, :, off])  # [B, N, 2, Hkv, D]
    else:
        kv = s["kv"][pg, :, :, off].float()
    k, v = kv[:, :, 0], kv[:, :, 1]
    if c["chunks"]:  # keys turned from where they were cached to where they stand
        k = _rotate(k, s["cos"][s["key_delta"]][:, :, None], s["sin"][s["key_delta"]][:, :, None])
    pos = s["positions"].long()
    q = _rotate(s["q"].float(), s["cos"][pos][:, None], s["sin"][pos][:, None])
    q = q[s["q_index"]].view(c["batch"], -1, hkv, hq // hkv, d)                # [B, T, Hkv, G, D]
    qp, kp = pos[s["q_index"]][:, :, None], s["key_pos"][:, None, :]
    seen = kp <= qp
    if c["window"]:
        seen &= (qp - kp < c["window"]) | (kp < c["sinks"])
    w = torch.einsum("bthgd,bnhd->bhgtn", q, k).mul_(s["scale"]).masked_fill_(~seen[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top > float("-inf"), top, 0.0)).exp_()
    total = w.sum(-1).permute(0, 3, 1, 2)[..., None]                           # [B, T, Hkv, G, 1]
    out = torch.einsum("bhgtn,bnhd->bthgd", w, v)
    out = torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0)
    return out.reshape(c["batch"], -1, hq * d)[s["live"]].bfloat16()


# ------------------------------------------------------------------- work
def _seen_keys(c):
    """(keys that some query of its sequence sees, (query, key) pairs that see each other), over the batch."""
    past, nq = _lengths(c)
    ctx, w, sinks = c["chunks"] * c["chunk_len"], c["window"], c["sinks"]
    keys = pairs = 0
    for a, n in zip(past, nq):
        p0, end = ctx + a, ctx + a + n
        first = max(0, p0 - w + 1) if w else 0
        keys += end - first + min(first, sinks)
        for p in range(p0, end):
            lo = max(0, p - w + 1) if w else 0
            pairs += p + 1 - lo + min(lo, sinks)
    return keys, pairs


def work(case):
    c = case
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["dim"]
    row4 = d // 2 + d // GROUP * 4
    if c["op"] == "append":
        n = c["tokens"]
        moved = 2 * hkv * (2 * d + row4 + 2 * d) + (hq * 4 * d if c["norm"] else 0)
        return {"bytes": n * moved, "flops": n * (2 * hkv + (hq if c["norm"] else 0)) * d * 10}
    keys, pairs = _seen_keys(c)
    rows = sum(_lengths(c)[1])
    return {"bytes": keys * 2 * hkv * (row4 if c["bits"] == 4 else 2 * d) + rows * hq * d * 4,
            "flops": pairs * hq * d * 4}


# ------------------------------------------------------- 64-bit definition
def _values64(codes, scales, pages, offs, side):
    """fp64 [n, Hkv, D] of K (side 0) or V (side 1) at the given places."""
    words = codes[pages, side, :, offs].contiguous().view(torch.int32)          # [n, Hkv, D/8]
    sz = scales[pages, side, :, offs].double()                                  # [n, Hkv, D/64, 2]
    n, h, nw = words.shape
    out = torch.empty(n, h, nw * 8, dtype=torch.float64, device=words.device)
    for i in range(nw // 2):
        for half in range(2):
            first = 8 * i + half * nw * 4
            for j in range(8):
                pair = sz[:, :, (first + j) // GROUP]
                out[:, :, first + j] = ((words[:, :, 2 * i + half] >> (4 * j)) & 15).double() * pair[..., 0] + pair[..., 1]
    return out


def _turn64(x, cos, sin):
    h = x.shape[-1] // 2
    re, im = x[..., :h], x[..., h:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = torch.empty_like(x)
    out[..., :h] = re * c - im * s
    out[..., h:] = im * c + re * s
    return out


def _exact_append(c, s):
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = q / torch.sqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"].double()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"].double()
    at = s["positions"].long()
    k = _turn64(k, s["cos"][at], s["sin"][at])
    held = []
    for x in (k, v):
        parts = []
        for grp in x.split(GROUP, -1):
            least, largest = grp.min(-1, keepdim=True).values, grp.max(-1, keepdim=True).values
            step, zero = ((largest - least) / 15).bfloat16().double(), least.bfloat16().double()
            level = torch.where(step > 0, torch.round((grp - zero) / step.clamp(min=1e-300)), torch.zeros_like(grp))
            parts.append(level.clamp(0, 15) * step + zero)
        held.append(torch.cat(parts, -1))
    return {"q": q, "kv": torch.stack(held, 1)}


def _exact_attend(c, s):
    hq, hkv, d, ps = c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    rep = hq // hkv
    past, nq = _lengths(c)
    out = torch.zeros(sum(nq), hq, d, dtype=torch.float64, device="cuda")
    t0 = 0
    for b in range(c["batch"]):
        n = c["chunks"] * c["chunk_len"] + past[b] + nq[b]
        slots, kp, delta = s["key_slot"][b, :n], s["key_pos"][b, :n], s["key_delta"][b, :n]
        pg, off = torch.div(slots, ps, rounding_mode="floor"), slots % ps
        if c["bits"] == 4:
            k, v = (_values64(s["codes"], s["scales"], pg, off, side) for side in (0, 1))
        else:
            k, v = (s["kv"][pg, side, :, off].double() for side in (0, 1))
        qp = s["positions"][t0:t0 + nq[b]].long()
        logits = torch.empty(hq, nq[b], n, dtype=torch.float64, device="cuda")
        for dl in sorted(set(delta.tolist())):  # queries turned by their distance to where the keys were cached
            at = (qp - dl).clamp(min=0)
            q = _turn64(s["q"][t0:t0 + nq[b]].double(), s["cos"][at], s["sin"][at])
            cols = (delta == dl).nonzero()[:, 0]
            for h in range(hq):
                logits[h][:, cols] = q[:, h] @ k[cols, h // rep].T * s["scale"]
        gap = qp[:, None] - kp[None, :]
        allowed = gap >= 0
        if c["window"]:
            allowed &= (gap < c["window"]) | (kp < c["sinks"])[None, :]
        logits[:, ~allowed] = float("-inf")
        prob = torch.nan_to_num(torch.softmax(logits, -1), nan=0.0)
        for h in range(hq):
            out[t0:t0 + nq[b], h] = prob[h] @ v[:, h // rep]
        t0 += nq[b]
    return out.view(-1, hq * d)


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attend(case, s)
