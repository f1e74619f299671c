"""Workloads of the paged serving operators: plan_pages, rope_append and paged_attention.

A case names the operator, the batch (request count and the ranges of its cached and new lengths) and the
shapes.  The lengths follow from the case alone, the values from the seed.  With ``own`` false ``run`` computes
the plain form in elementary torch operations; with ``own`` true it calls the framework.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step of a full server: every request appends one token
        dict(name="plan_decode", op="plan", requests=64, cached_lo=128, cached_hi=32768, new_lo=1, new_hi=1,
             page=16, short=False, mix=1),
        # a step that mixes chunks of prompts with decoding, many requests
        dict(name="plan_mixed", op="plan", requests=1024, cached_lo=0, cached_hi=8192, new_lo=1, new_hi=256,
             page=64, short=False, mix=2),
        # the rotation and append of one decode step, Llama-3.1-8B heads
        dict(name="rope_decode", op="rope", tokens=64, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False,
             factor=1.0, page=16, far=131072, dtype="bf16", mix=3),
        # a ragged chunk with half of each head rotated in the interleaved layout, positions scaled, Qwen2.5-7B heads
        dict(name="rope_chunk", op="rope", tokens=5001, heads=28, kv_heads=4, dim=128, rotary=64, interleaved=True,
             factor=4.0, page=32, far=131072, dtype="fp16", mix=4),
        # a whole prompt appended at once
        dict(name="rope_prompt", op="rope", tokens=32768, heads=32, kv_heads=8, dim=128, rotary=128,
             interleaved=False, factor=8.0, page=64, far=1048576, dtype="bf16", mix=5),
        # the smallest call: one user, one token
        dict(name="decode_one", op="attn", requests=1, cached_lo=4098, cached_hi=4098, new_lo=1, new_hi=1, heads=32,
             kv_heads=8, dim=128, page=16, window=0, sinks=0, dtype="bf16", mix=6),
        # a full server's decode step over ragged contexts, small pages
        dict(name="decode_batch", op="attn", requests=64, cached_lo=512, cached_hi=16384, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0, dtype="bf16", mix=7),
        # decoding behind two prompts of 128K tokens
        dict(name="decode_long", op="attn", requests=2, cached_lo=131071, cached_hi=131071, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, dim=128, page=64, window=0, sinks=0, dtype="bf16", mix=8),
        # a chunk of a long prompt over what is cached of it
        dict(name="chunk_long", op="attn", requests=1, cached_lo=32768, cached_hi=32768, new_lo=2048, new_hi=2048,
             heads=32, kv_heads=8, dim=128, page=64, window=0, sinks=0, dtype="bf16", mix=9),
        # chunks and single tokens in one batch, seven query heads to a KV head
        dict(name="chunk_mixed", op="attn", requests=16, cached_lo=0, cached_hi=16384, new_lo=1, new_hi=512, heads=28,
             kv_heads=4, dim=128, page=32, window=0, sinks=0, dtype="fp16", mix=10),
        # decode with a sliding window and four first tokens kept
        dict(name="window_decode", op="attn", requests=128, cached_lo=1024, cached_hi=32768, new_lo=1, new_hi=1,
             heads=32, kv_heads=8, dim=128, page=16, window=4096, sinks=4, dtype="bf16", mix=11),
        # chunks with a window, small heads without sharing, large pages
        dict(name="window_chunk", op="attn", requests=2, cached_lo=16384, cached_hi=16384, new_lo=2000, new_hi=2048,
             heads=16, kv_heads=16, dim=64, page=128, window=1024, sinks=128, dtype="bf16", mix=12),
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; lo may be 0."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 2)))) - 1))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "attn"])
    mix = rng.randrange(1 << 30)
    if op == "plan":
        lo, new = _log_int(rng, 0, 4096), _log_int(rng, 1, 256)
        return dict(op=op, requests=_log_int(rng, 1, 1024), cached_lo=lo, cached_hi=_log_int(rng, lo, 32768),
                    new_lo=rng.choice([0, 1, new]), new_hi=new, page=rng.choice([16, 32, 64, 128]),
                    short=rng.random() < 0.3, mix=mix)
    dtype = rng.choice(["bf16", "fp16"])
    kv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    if op == "rope":
        return dict(op=op, tokens=_log_int(rng, 1, 16384), heads=kv * min(group, 4), kv_heads=kv, dim=dim,
                    rotary=rng.choice([16, dim // 2, dim]), interleaved=rng.random() < 0.5,
                    factor=rng.choice([1.0, 4.0]), page=page, far=_log_int(rng, 32768, 1048576), dtype=dtype, mix=mix)
    window = rng.choice([0, 0, _log_int(rng, 1, 8192)])
    sinks = rng.choice([0, 4, 100]) if window else 0
    requests = _log_int(rng, 1, 64)
    new_hi = rng.choice([1, _log_int(rng, 1, 1024)])
    # the plain form's padded scores stay below those of the largest listed case
    room = int(1.5e9 / (requests * new_hi * kv * group)) - new_hi
    lo = _log_int(rng, 0, max(1, min(1024, room)))
    return dict(op=op, requests=requests, cached_lo=lo, cached_hi=max(lo, _log_int(rng, lo, max(lo, min(16384, room)))),
                new_lo=rng.choice([1, new_hi]), new_hi=new_hi, heads=kv * group, kv_heads=kv, dim=dim, page=page,
                window=window, sinks=sinks, dtype=dtype, mix=mix)


def _lengths(case):
    """(cached, new) token counts of each request, from the case alone."""
    rng = random.Random(case["mix"])
    cached = [_log_int(rng, case["cached_lo"], case["cached_hi"]) for _ in range(case["requests"])]
    new = [_log_int(rng, case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    if sum(new) == 0:
        new[0] = 1
    return cached, new


def _pages(n, page):
    return -(-n // page)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _tables(counts, width, order):
    """Rows of page numbers (-1 behind a row's last), taken in turn from ``order``."""
    table, at = torch.full((len(counts), width), -1, dtype=torch.int32), 0
    for r, n in enumerate(counts):
        table[r, :n] = order[at:at + n]
        at += n
    return table.cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    page = case["page"]
    if case["op"] == "plan":
        cached, new = _lengths(case)
        have = [_pages(c, page) for c in cached]
        need = [_pages(c + n, page) - h for c, n, h in zip(cached, new, have)]
        width = max(h + n for h, n in zip(have, need)) + 1
        order = torch.randperm(sum(have) + sum(need) + 8, generator=cpu).to(torch.int32)
        free = order[sum(have):]
        if case["short"]:  # a pool that runs out before the last request
            free = free[:max(1, sum(need) // 2)]
        return dict(case=case, cached=_ints(cached), new=_ints(new), table=_tables(have, width, order),
                    free=free.cuda(), tokens=sum(new))
    dt, D, kv, H = DTYPES[case["dtype"]], case["dim"], case["kv_heads"], case["heads"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dt)

    if case["op"] == "rope":
        T = case["tokens"]
        P = _pages(T, page) + 3
        first = int(torch.randint(0, case["far"] - T + 1, (1,), generator=cpu)) if case["far"] > T else 0
        slots = torch.randperm(P * page, generator=gen, device="cuda")[:T].to(torch.int32)
        qkv = normal(T, (H + 2 * kv) * D)
        freq = 500000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])
        return dict(case=case, q=qkv[:, :H * D].view(T, H, D), k=qkv[:, H * D:(H + kv) * D].view(T, kv, D),
                    v=qkv[:, (H + kv) * D:].view(T, kv, D), slots=slots,
                    positions=torch.arange(first, first + T, dtype=torch.int32, device="cuda"),
                    k_pages=normal(P, kv, page, D), v_pages=normal(P, kv, page, D),
                    inv_freq=(freq / case["factor"]).float().cuda(), amplitude=0.1 * math.log(case["factor"]) + 1.0)
    cached, new = _lengths(case)
    lens = [c + n for c, n in zip(cached, new)]
    counts = [_pages(n, page) for n in lens]
    P = sum(counts) + 2
    order = torch.randperm(P, generator=cpu).to(torch.int32)
    return dict(case=case, q=normal(sum(new), H, D, scale=2.0), k_pages=normal(P, kv, page, D),
                v_pages=normal(P, kv, page, D), table=_tables(counts, max(counts), order), cu_q=_ints(_starts(new)),
                kv_lens=_ints(lens), longest=max(new))


# ------------------------------------------------------------------ plain forms
def _plan_plain(s):
    page, T = s["case"]["page"], s["tokens"]
    cached, new, table, free = s["cached"].long(), s["new"].long(), s["table"], s["free"]
    R, width = table.shape
    end = new.cumsum(0)
    have, last = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = (last <= width) & (end <= T)
    need = torch.where(fits, last - have, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (upto <= free.numel()))
    taken = torch.where(served & (need > 0), upto, 0).max()
    cols = torch.arange(width, device=table.device)
    fresh = (cols >= have[:, None]) & (cols < last[:, None]) & served[:, None]
    pick = ((upto - need)[:, None] + cols - have[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[pick], table))
    kv_lens = torch.where(served, cached + new, 0)
    cu_q = torch.cat([end.new_zeros(1), end]).clamp(max=T)
    at = torch.arange(T, device=table.device)
    row = torch.searchsorted(end, at, right=True).clamp(max=R - 1)
    live = at < end[-1]
    pos = torch.where(live, cached[row] + at - (end - new)[row], 0)
    slot = table[row, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    slot = torch.where(live & served[row], slot, -1)
    info = torch.stack([taken, (~served).sum()])
    return [x.to(torch.int32) for x in (cu_q, kv_lens, pos, slot, info)] + [table]


def _rope_plain(s):
    case = s["case"]
    rd, page = case["rotary"], case["page"]
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()  # far positions: 64 bits
    cos, sin = (f(angle).mul_(s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:rd:2], y[..., 1:rd:2]
            turn = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :rd // 2], y[..., rd // 2:rd]
            turn = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turn, y[..., rd:]], -1).to(x.dtype)

    slots = s["slots"].long()
    s["k_pages"][slots // page, :, slots % page] = turned(s["k"])
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    return [turned(s["q"]), s["k_pages"], s["v_pages"]]


def _attn_plain(s):
    case, q, table = s["case"], s["q"], s["table"].long().clamp(min=0)
    T, H, D = q.shape
    kv, n = case["kv_heads"], s["longest"]
    G, R = H // kv, table.shape[0]
    cu, lens = s["cu_q"].long(), s["kv_lens"].long()
    dev = q.device

    def gathered(pages):  # [R, kv, keys, D]
        return pages[table].float().transpose(1, 2).reshape(R, kv, -1, D)

    rows = (cu[:-1, None] + torch.arange(n, device=dev)).clamp(max=T - 1)
    scores = q.float()[rows].view(R, n, kv, G, D).permute(0, 2, 3, 1, 4).reshape(R, kv, G * n, D)
    scores = (scores @ gathered(s["k_pages"]).transpose(-1, -2)).mul_(D ** -0.5)
    keys = torch.arange(scores.shape[-1], device=dev)
    pos = (lens - (cu[1:] - cu[:-1]))[:, None, None] + torch.arange(n, device=dev)[:, None]
    seen = (keys <= pos) & (keys < lens[:, None, None])
    if case["window"]:
        seen &= (keys > pos - case["window"]) | (keys < case["sinks"])
    scores.view(R, kv, G, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores @ gathered(s["v_pages"])
    out = torch.where(total > 0, out / total, 0.0).view(R, kv, G, n, D).permute(0, 3, 1, 2, 4)
    at = torch.arange(T, device=dev)
    row = torch.searchsorted(cu[1:], at, right=True)
    return out[row, at - cu[row]].reshape(T, H, D).to(q.dtype)


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan_plain, "rope": _rope_plain, "attn": _attn_plain}[op](state)
    import fftsparse_b200 as F
    s, case = state, state["case"]
    if op == "plan":
        p = F.plan_pages(s["cached"], s["new"], s["table"], s["free"], case["page"], s["tokens"])
        return [p.cu_q, p.kv_lens, p.positions, p.slot_map, p.info, s["table"]]
    if op == "rope":
        q = F.rope_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_pages"], s["v_pages"],
                          s["inv_freq"], interleaved=case["interleaved"], attn_factor=s["amplitude"])
        return [q, s["k_pages"], s["v_pages"]]
    return F.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu_q"], s["kv_lens"],
                             window=case["window"] or None, sinks=case["sinks"])


def work(case):
    page = case["page"]
    if case["op"] == "plan":
        cached, new = _lengths(case)
        R, T = len(new), sum(new)
        fresh = sum(_pages(c + n, page) - _pages(c, page) for c, n in zip(cached, new))
        # lengths in and out, positions and slots out, the page of each run of tokens in, new entries in and out
        touched = sum(_pages(c + n, page) - c // page for c, n in zip(cached, new) if n)
        return {"bytes": 4 * (2 * R + 2 * R + 1 + 2 * T + touched + fresh), "flops": 0}
    H, kv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rope":
        T = case["tokens"]
        return {"bytes": T * (2 * 2 * (H + 2 * kv) * D + 8), "flops": 3 * T * (H + kv) * case["rotary"]}
    cached, new = _lengths(case)
    W, S = case["window"], case["sinks"]
    pairs = keys = 0
    for c, n in zip(cached, new):
        if not n:
            continue
        if not W:
            pairs += n * c + n * (n + 1) // 2
            keys += c + n
        else:
            pairs += sum(min(p + 1, W) + min(S, max(0, p + 1 - W)) for p in range(c, c + n))
            first = max(0, c - W + 1)
            keys += c + n - first + min(S, first)
    T = sum(new)
    return {"bytes": 2 * (2 * T * H * D + 2 * keys * kv * D), "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "rope":
        rd, page = case["rotary"], case["page"]
        theta = torch.outer(s["positions"].double(), s["inv_freq"].double())
        turn = torch.polar(torch.full_like(theta, s["amplitude"]), theta)[:, None]

        def rotated(x):
            y = x.double()
            body = y[..., :rd].unflatten(-1, (rd // 2, 2) if case["interleaved"] else (2, rd // 2))
            dim = -1 if case["interleaved"] else -2
            z = torch.complex(*body.unbind(dim)) * turn
            return torch.cat([torch.stack([z.real, z.imag], dim).flatten(-2), y[..., rd:]], -1)

        keys, values = s["k_pages"].double().transpose(1, 2), s["v_pages"].double().transpose(1, 2)
        keys, values = keys.flatten(0, 1), values.flatten(0, 1)
        keys[s["slots"].long()] = rotated(s["k"])
        values[s["slots"].long()] = s["v"].double()
        return [rotated(s["q"])] + [x.unflatten(0, (-1, page)).transpose(1, 2) for x in (keys, values)]
    q = s["q"].double()
    T, H, D = q.shape
    G, page = H // case["kv_heads"], case["page"]
    out = torch.zeros(T, H, D, dtype=torch.float64, device="cuda")
    at = 0
    for r, (c, n) in enumerate(zip(*_lengths(case))):
        if not n:
            continue
        ids = s["table"][r, :_pages(c + n, page)].long()
        i, j = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
        hidden = j > i
        if case["window"]:
            hidden |= (j <= i - case["window"]) & (j >= case["sinks"])
        for h in range(case["kv_heads"]):
            k = s["k_pages"][ids, h].double().flatten(0, 1)[:c + n]
            v = s["v_pages"][ids, h].double().flatten(0, 1)[:c + n]
            a = torch.einsum("tgd,cd->gtc", q[at:at + n, h * G:(h + 1) * G], k) / math.sqrt(D)
            p = torch.softmax(a.masked_fill(hidden, -math.inf), -1)
            out[at:at + n, h * G:(h + 1) * G] = torch.einsum("gtc,cd->tgd", p, v)
        at += n
    return out
