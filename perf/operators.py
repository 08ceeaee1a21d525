"""Cases and measurements of the paged-KV operators around a shared, a windowed and an image-positioned cache.

Four calls of `pie_b200.ops`, with the work a serving step gives them:

  prefix   `BatchSharedPrefixDecodeWrapper.run`: one query token per request, requests of a group share the leading
           pages of their page lists (a forked context, beams, a common system prompt)
  step     `BatchDecodeWithPagedKVCacheWrapper.run` planned with `window_left` and `first_tokens`: one query token per
           request sees the last tokens of its context and the first few
  chunk    `BatchPrefillWithPagedKVCacheWrapper.run`, causal, planned with `window_left` and `first_tokens`
  axes     `rope_axes_append_paged_kv_cache`: rotary positions on several axes (time, height, width), q rotated, k rotated
           on its way into the paged cache, v copied

`run` with `own` false is the plain form in 32 bits (angles in 64); `exact` is written apart from it, in 64 bits.
"""
import math
import random

import torch

own = False

PAGE = 16
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0
WORKSPACE = 128 << 20


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # four beams that left a short prompt a moment ago: the smallest call, where latency counts
        dict(name="prefix_4_beams", op="prefix", dtype="bf16", hq=32, hkv=8, groups=1, members=4, prefix=512, suffix=40,
             mix=1),
        # beam search of a batch: 16 prompts of unequal length, four beams each
        dict(name="prefix_16x4_beams", op="prefix", dtype="bf16", hq=32, hkv=8, groups=16, members=4, prefix=2048,
             suffix=64, mix=2),
        # a batch of chats behind one system prompt, each with a conversation of its own
        dict(name="prefix_system_prompt", op="prefix", dtype="bf16", hq=32, hkv=8, groups=1, members=64, prefix=4096,
             suffix=1024, mix=3),
        # many questions about one long document, the head counts of a 70B-shaped layer
        dict(name="prefix_document", op="prefix", dtype="fp16", hq=64, hkv=8, groups=1, members=128, prefix=16384,
             suffix=512, mix=4),
        # one conversation: the smallest call
        dict(name="step_1", op="step", dtype="bf16", hq=32, hkv=8, batch=1, low=700, high=700, window=511, first=4,
             mix=5),
        # the decode batch of an 8B-shaped layer, some contexts still shorter than the window
        dict(name="step_64", op="step", dtype="bf16", hq=32, hkv=8, batch=64, low=512, high=4096, window=1023, first=4,
             mix=6),
        # a large batch with long contexts and a wide window
        dict(name="step_128_wide", op="step", dtype="fp16", hq=64, hkv=8, batch=128, low=2049, high=8191, window=4095,
             first=16, mix=7),
        # chunks of prompts that are already partly in the cache, odd lengths
        dict(name="chunk_512", op="chunk", dtype="bf16", hq=32, hkv=8, batch=8, q_low=385, q_high=512, low=600, high=6656,
             window=1023, first=4, mix=8),
        # whole prompts: the largest call
        dict(name="chunk_4096", op="chunk", dtype="bf16", hq=32, hkv=8, batch=4, q_low=4096, q_high=4096, low=4096,
             high=4096, window=1023, first=4, mix=9),
        # a decode step of a batch whose contexts hold images
        dict(name="axes_48", op="axes", dtype="bf16", hq=32, hkv=8, dim=128, batch=48, tokens=48, sections="16,24,24",
             cyclic=False, interleave=False, mix=10),
        # prompts of text and image patches
        dict(name="axes_20480", op="axes", dtype="bf16", hq=32, hkv=8, dim=128, batch=8, tokens=20480, sections="16,24,24",
             cyclic=False, interleave=False, mix=11),
        # full precision, small heads, axes dealt out in turn
        dict(name="axes_fp32_odd", op="axes", dtype="fp32", hq=12, hkv=4, dim=64, batch=3, tokens=1237,
             sections="12,10,10", cyclic=True, interleave=False, mix=12),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("prefix", "step", "chunk", "axes"))
    dtype = rng.choice(("bf16", "fp16"))
    hkv = rng.choice((1, 2, 4, 8))
    hq = hkv * rng.choice((1, 2, 4, 6, 8))
    mix = rng.randrange(1 << 20)
    if op == "prefix":
        groups = _log_int(rng, 1, 24)
        members = _log_int(rng, 1, max(1, 128 // groups))
        prefix = _log_int(rng, 16, 16384)
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, groups=groups, members=members, prefix=prefix,
                    suffix=_log_int(rng, 1, 1024 if prefix < 8192 else 512), mix=mix)
    if op == "step":
        high = _log_int(rng, 1, 8191)
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, batch=_log_int(rng, 1, 128), low=_log_int(rng, 1, high), high=high,
                    window=_log_int(rng, 1, 4096) - 1, first=_log_int(rng, 1, 64), mix=mix)
    if op == "chunk":
        q_high = _log_int(rng, 1, 2048)
        high = q_high + _log_int(rng, 1, 4096) - 1
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, batch=_log_int(rng, 1, 8), q_low=_log_int(rng, 1, q_high),
                    q_high=q_high, low=q_high, high=high, window=_log_int(rng, 1, 2048) - 1, first=_log_int(rng, 1, 64),
                    mix=mix)
    dim = rng.choice((64, 128, 256))
    sections = {64: "12,10,10", 128: rng.choice(("16,24,24", "24,20,20", "64")), 256: "32,48,48"}[dim]
    batch = _log_int(rng, 1, 64)
    return dict(op=op, dtype=rng.choice(("bf16", "fp16", "fp32")), hq=hq, hkv=hkv, dim=dim, batch=batch,
                tokens=max(batch, _log_int(rng, 1, 8192)), sections=sections, cyclic=rng.random() < 0.5,
                interleave=rng.random() < 0.3, mix=mix)


# ------------------------------------------------------------------------------------------------ lengths (host)
def _ints(rng, count, low, high):
    return [rng.randint(low, high) for _ in range(count)]


def _lengths(case):
    """What a case's `mix` says of its lengths: (query tokens, context tokens) per request, and for the shared prefix
    (tokens of the prefix, requests) per group."""
    rng = random.Random(case["mix"])
    if case["op"] == "prefix":
        shared = [PAGE * max(1, n // PAGE) for n in _ints(rng, case["groups"], (case["prefix"] + 1) // 2, case["prefix"])]
        if case["groups"] == 1:
            shared = [PAGE * max(1, case["prefix"] // PAGE)]
        members = [case["members"]] * case["groups"]
        kv = [s + n for s, m in zip(shared, members) for n in _ints(rng, m, 1, case["suffix"])]
        return [1] * len(kv), kv, shared, members
    if case["op"] == "step":
        return [1] * case["batch"], _ints(rng, case["batch"], case["low"], case["high"]), None, None
    if case["op"] == "chunk":
        q = _ints(rng, case["batch"], case["q_low"], case["q_high"])
        return q, [max(n, m) for n, m in zip(q, _ints(rng, case["batch"], case["low"], case["high"]))], None, None
    cuts = sorted(rng.sample(range(1, case["tokens"]), case["batch"] - 1)) if case["batch"] > 1 else []
    q = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return q, [n + rng.randint(0, 64) for n in q], None, None


def _visible(case, q, kv):
    """(key, query) pairs a request's query tokens see, and the distinct keys among them (step and chunk)."""
    pairs, first, w = 0, case["first"], case["window"]
    for p in range(kv - q, kv):
        low = max(0, p - w)
        pairs += p + 1 - low + min(low, first)
    low = max(0, kv - q - w)
    return pairs, kv - low + min(low, first)


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    hq, hkv = case["hq"], case["hkv"]
    q, kv, shared, members = _lengths(case)
    n = sum(q)
    if case["op"] == "axes":
        d = case["dim"]
        axes = case["sections"].count(",") + 1
        return {"bytes": n * d * es * (2 * hq + 4 * hkv) + n * 4 * (axes + 2) + 4 * sum(-(-x // PAGE) for x in kv),
                "flops": 3 * n * d * (hq + hkv)}
    d = 128
    io = 2 * n * hq * d * es
    table = 4 * (sum(-(-x // PAGE) for x in kv) + 2 * len(kv) + 1)
    if case["op"] == "prefix":
        tokens = sum(shared) + sum(kv) - sum(s * m for s, m in zip(shared, members))
        return {"bytes": tokens * 2 * hkv * d * es + io + table, "flops": 4 * d * hq * sum(kv)}
    seen = [_visible(case, a, b) for a, b in zip(q, kv)]
    return {"bytes": sum(k for _, k in seen) * 2 * hkv * d * es + io + table, "flops": 4 * d * hq * sum(p for p, _ in seen)}


# ------------------------------------------------------------------------------------------------ inputs (GPU)
def _normal(g, shape, dtype, scale):
    """N(0, scale^2) in `dtype`, made in slabs so that the 32-bit draw stays small."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        end = min(flat.numel(), at + step)
        flat[at:end] = torch.randn(end - at, generator=g, device="cuda") * scale
    return out


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _page_tables(case, kv, shared, members, seed):
    """Fragmented page lists out of one pool; the leading pages of a group's requests are the same."""
    counts = [-(-x // PAGE) for x in kv]
    free = random.Random(seed ^ 0x5A17)
    need = sum(counts) if shared is None else sum(s // PAGE for s in shared) + sum(counts) - sum(
        m * (s // PAGE) for s, m in zip(shared, members))
    pages = need + 3
    deck = list(range(pages))
    free.shuffle(deck)
    lists, at = [], 0
    if shared is None:
        for c in counts:
            lists.append(deck[at: at + c])
            at += c
    else:
        b = 0
        for s, m in zip(shared, members):
            head = deck[at: at + s // PAGE]
            at += len(head)
            for _ in range(m):
                own_pages = counts[b] - len(head)
                lists.append(head + deck[at: at + own_pages])
                at += own_pages
                b += 1
    indptr = [0]
    for c in counts:
        indptr.append(indptr[-1] + c)
    last = [x - PAGE * (c - 1) for x, c in zip(kv, counts)]
    return pages, _int32([p for x in lists for p in x]), _int32(indptr), _int32(last)


def _image_positions(rng, q, offsets):
    """Positions on three axes: runs of text (the three equal) and of image patches (time fixed, a grid of rows and
    columns), from an offset per request."""
    axes = [[], [], []]
    for n, base in zip(q, offsets):
        at, left = base, n
        while left > 0:
            if rng.random() < 0.5:
                k = min(left, rng.randint(1, 200))
                for a in axes:
                    a.extend(range(at, at + k))
                at += k
            else:
                h, w = rng.randint(2, 24), rng.randint(2, 24)
                k = min(left, h * w)
                axes[0].extend([at] * k)
                axes[1].extend(at + i // w for i in range(k))
                axes[2].extend(at + i % w for i in range(k))
                at += max(h, w)
            left -= k
    return axes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    q_lens, kv, shared, members = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case.get("dim", 128)
    pages, indices, indptr, last = _page_tables(case, kv, shared, members, seed)
    s = {"case": case, "kv": kv, "q_lens": q_lens, "indices": indices, "indptr": indptr, "last": last,
         "pool": _normal(g, (pages, 2, PAGE, hkv, d), dtype, 1.0), "q": _normal(g, (sum(q_lens), hq, d), dtype, 1.0),
         "max_kv": max(kv), "max_q": max(q_lens)}
    qo = [0]
    for n in q_lens:
        qo.append(qo[-1] + n)
    s["qo_indptr"] = _int32(qo)
    s["kv_lens"] = _int32(kv)
    if case["op"] == "prefix":
        ends = [0]
        for m in members:
            ends.append(ends[-1] + m)
        s["group_indptr"] = _int32(ends)
    if case["op"] == "axes":
        rng = random.Random(seed ^ 0x3A7)
        sections = [int(x) for x in case["sections"].split(",")]
        positions = _image_positions(rng, q_lens, [rng.randint(0, 200000) for _ in q_lens])
        s["sections"] = sections
        s["pos"] = _int32(positions[: len(sections)])
        s["k"] = _normal(g, (sum(q_lens), hkv, d), dtype, 1.0)
        s["v"] = _normal(g, (sum(q_lens), hkv, d), dtype, 1.0)
        s["batch_indices"] = _int32([b for b, n in enumerate(q_lens) for _ in range(n)])
        s["slots"] = _int32([x - n + i for n, x in zip(q_lens, kv) for i in range(n)])
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program sets up once for a step and keeps for its layers: the wrapper planned on the step's tables."""
    from pie_b200 import ops

    case = s["case"]
    dtype = TYPES[case["dtype"]]
    if case["op"] == "axes":
        s["rope"] = ops.AxisRopeConfig(sections=tuple(s["sections"]), cyclic=case["cyclic"], mode="plain", theta=THETA,
                                       scale=1.0, interleave=case["interleave"])
        return
    workspace = torch.empty(WORKSPACE, dtype=torch.uint8, device="cuda")
    if case["op"] == "prefix":
        w = ops.BatchSharedPrefixDecodeWrapper(workspace)
        w.plan(s["indptr"], s["indices"], s["last"], case["hq"], case["hkv"], 128, PAGE, group_indptr=s["group_indptr"],
               q_data_type=dtype)
    elif case["op"] == "step":
        w = ops.BatchDecodeWithPagedKVCacheWrapper(workspace)
        w.plan(s["indptr"], s["indices"], s["last"], case["hq"], case["hkv"], 128, PAGE, window_left=case["window"],
               first_tokens=case["first"], q_data_type=dtype)
    else:
        w = ops.BatchPrefillWithPagedKVCacheWrapper(workspace)
        w.plan(s["qo_indptr"], s["indptr"], s["indices"], s["last"], case["hq"], case["hkv"], 128, PAGE, causal=True,
               window_left=case["window"], first_tokens=case["first"], q_data_type=dtype)
    s["wrapper"] = w


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    if s["case"]["op"] == "axes":
        return _plain_axes(s)
    return _plain_attention(s)


def _own(s):
    if s["case"]["op"] == "axes":
        from pie_b200 import ops

        q = ops.rope_axes_append_paged_kv_cache(s["q"], s["k"], s["v"], s["pos"], s["batch_indices"], s["slots"], s["pool"],
                                                s["indices"], s["indptr"], s["last"], s["rope"])
        return q, s["pool"]
    return s["wrapper"].run(s["q"], s["pool"])


def _plain_attention(s):
    """softmax(q k^T / sqrt(d)) v over the keys each query token sees, requests padded to the longest."""
    case = s["case"]
    pool, q = s["pool"], s["q"]
    hq, hkv, d = case["hq"], case["hkv"], 128
    batch, group = len(s["kv"]), hq // hkv
    dev = q.device
    t = torch.arange(s["max_kv"], device=dev)
    kv_len = s["kv_lens"].long()[:, None]
    inside = t[None, :] < kv_len
    at = s["indptr"].long()[:-1, None] + torch.where(inside, t[None, :] // PAGE, 0)
    page = s["indices"].long()[at]
    k = pool[page, 0, (t % PAGE)[None, :]].permute(0, 2, 3, 1).float()  # [batch, hkv, d, kv]
    v = pool[page, 1, (t % PAGE)[None, :]].permute(0, 2, 1, 3).float()  # [batch, hkv, kv, d]
    # query tokens padded to [batch, most]
    q_len = (s["qo_indptr"][1:] - s["qo_indptr"][:-1]).long()[:, None]
    j = torch.arange(s["max_q"], device=dev)
    there = j[None, :] < q_len
    row = s["qo_indptr"].long()[:-1, None] + torch.where(there, j[None, :], 0)
    qp = q[row].view(batch, s["max_q"], hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * s["max_q"], d)
    scores = (qp.float() @ k) * (1.0 / math.sqrt(d))
    scores = scores.view(batch, hkv, group, s["max_q"], s["max_kv"])
    pos = (kv_len - q_len + j[None, :])[:, :, None]  # [batch, most, 1]
    sees = inside[:, None, :] & (t <= pos)
    if "window" in case:
        sees = sees & ((t >= pos - case["window"]) | (t < case["first"]))
    scores = scores.masked_fill_(~sees[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(batch, hkv, group * s["max_q"], s["max_kv"]) @ v
    o = o.view(batch, hkv, group, s["max_q"], d) / total.clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4)[there].reshape(-1, hq, d).to(q.dtype)


def _plain_axes(s):
    """Angles position x frequency with every pair's axis picked by its section, then pages written by index."""
    case = s["case"]
    d, dev = case["dim"], s["q"].device
    sections = s["sections"]
    axes, half = len(sections), sum(sections)
    i = torch.arange(half, device=dev)
    if case["cyclic"]:
        axis = i % axes
        limit = torch.tensor(sections, device=dev) * axes
        axis = torch.where(i < limit[axis], axis, 0)
    else:
        axis = (i[:, None] >= torch.cumsum(torch.tensor(sections, device=dev), 0)[None, :]).sum(1)
    freq = THETA ** (-2.0 * i.double() / (2 * half))
    angle = s["pos"].double()[axis].t() * freq[None, :]  # [n, half]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(x):
        x = x.float()
        if case["interleave"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        a, b = x[..., :half], x[..., half:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    q, k = turn(s["q"]).to(s["q"].dtype), turn(s["k"]).to(s["k"].dtype)
    slot = s["slots"].long()
    page = s["indices"].long()[s["indptr"].long()[s["batch_indices"].long()] + slot // PAGE]
    s["pool"][page, 0, slot % PAGE] = k
    s["pool"][page, 1, slot % PAGE] = s["v"]
    return q, s["pool"]


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_axes(s) if case["op"] == "axes" else _exact_attention(s)


def _exact_attention(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    indptr = s["indptr"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, kv) in enumerate(zip(s["q_lens"], s["kv"])):
        pages = s["pool"][s["indices"][indptr[b]: indptr[b + 1]].long()]
        keys = pages[:, 0].reshape(-1, hkv, 128)[:kv].double()
        values = pages[:, 1].reshape(-1, hkv, 128)[:kv].double()
        position = torch.arange(kv - n, kv, device="cuda")
        token = torch.arange(kv, device="cuda")
        hidden = token[None, :] > position[:, None]
        if "window" in case:
            hidden |= (token[None, :] + case["window"] < position[:, None]) & (token[None, :] >= case["first"])
        for h in range(hq):
            kh = h // (hq // hkv)
            logits = torch.einsum("nd,td->nt", s["q"][row: row + n, h].double(), keys[:, kh]) / 128 ** 0.5
            out[row: row + n, h] = torch.softmax(logits.masked_fill(hidden, float("-inf")), dim=-1) @ values[:, kh]
        row += n
    return out


def _exact_axes(s):
    case = s["case"]
    half = sum(s["sections"])
    axes = len(s["sections"])
    owner = []
    if case["cyclic"]:
        owner = [0] * half
        for a in range(1, axes):
            for i in range(a, axes * s["sections"][a], axes):
                owner[i] = a
    else:
        for a, count in enumerate(s["sections"]):
            owner += [a] * count
    turns = torch.empty((s["q"].shape[0], half), dtype=torch.complex128, device="cuda")
    for i, a in enumerate(owner):
        phase = s["pos"][a].double() * math.exp(-math.log(THETA) * i / half)
        turns[:, i] = torch.polar(torch.ones_like(phase), phase)

    def rotate(x):
        x = x.double()
        pairs = x.unflatten(-1, (half, 2)) if case["interleave"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turns[:, None])
        return z.flatten(-2) if case["interleave"] else z.transpose(-1, -2).flatten(-2)

    pool = s["pool"].double()
    k = rotate(s["k"])
    indptr, indices = s["indptr"].long(), s["indices"].long()
    where = indices[indptr[s["batch_indices"].long()] + s["slots"].long() // PAGE] * PAGE + s["slots"].long() % PAGE
    by_token = pool.transpose(1, 2).reshape(-1, 2, *pool.shape[3:])
    by_token[where, 0] = k
    by_token[where, 1] = s["v"].double()
    return rotate(s["q"]), by_token.view(pool.shape[0], PAGE, 2, *pool.shape[3:]).transpose(1, 2).contiguous()
