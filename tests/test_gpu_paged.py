"""GPU parity of the paged serving operators against plain 64-bit evaluations.

Tolerances, with u = finfo(dtype).eps / 2 the relative size of one rounding:
  rope_append      u |y| for the result's rounding, plus (|a| + |b|) 2^-20 for the fp32 cos and sin (their
                   argument is a fraction of a turn, exact to 2^-25), products and sum, plus the dtype's smallest step
  paged_attention  u |o| for the result's rounding; u A with A = sum p |v| for the rounding of every p (the divisor
                   sums them unrounded); A e with e = 2 ((D + 2) 2^-23 S + 2^-20) for the scores' fp32
                   products (S the largest sum |q k| scale) through the exponential, both in numerator and
                   divisor, and its own approximation; keys 2^-24 max |v| for the p that fp16 flushes
"""
import math
import random

import pytest
import torch

import fftsparse_b200 as F

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16
NAN = float("nan")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ------------------------------------------------------------------ plan_pages
def plan_model(cached, new, table, free, page, T):
    table = [list(r) for r in table]
    cu, kv, pos, slot, taken, unserved, asked = [0], [], [0] * T, [-1] * T, 0, 0, 0
    end = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        first, end = end, end + n
        have, last = -(-c // page), -(-(c + n) // page)
        fits = last <= len(table[r]) and end <= T
        need = last - have if fits else 0
        served = fits and (need == 0 or asked + need <= len(free))
        for i in range(need if served else 0):
            table[r][have + i] = free[asked + i]
            taken = asked + need
        asked += need
        cu.append(min(end, T))
        kv.append(c + n if served else 0)
        unserved += not served
        for t in range(first, min(end, T)):
            pos[t] = c + t - first
            slot[t] = table[r][pos[t] // page] * page + pos[t] % page if served else -1
    return cu, kv, pos, slot, [taken, unserved], table


@pytest.mark.parametrize("R,page,spare,room,width", [
    (1, 16, 8, 0, None), (3, 16, 8, 5, None), (7, 1, 8, 0, None), (64, 16, -30, 0, None), (64, 64, -3, 3, None),
    (600, 32, 0, 40, None), (1500, 16, 8, 0, None), (1500, 128, -200, 17, None), (40, 16, 8, 0, 20), (40, 16, 8, -60, None),
    (5, 16, -10 ** 6, 0, None)])
def test_plan_pages(R, page, spare, room, width):
    rng = random.Random(R * 1000 + page)
    cached = [rng.choice([0, 1, page - 1, page, page + 1, rng.randrange(900)]) for _ in range(R)]
    new = [rng.choice([0, 1, 1, rng.randrange(90)]) for _ in range(R)]
    have = [-(-c // page) for c in cached]
    need = [-(-(c + n) // page) - h for c, n, h in zip(cached, new, have)]
    W = width or max(h + n for h, n in zip(have, need)) + 2
    order = list(range(sum(have) + sum(need) + 100))
    rng.shuffle(order)
    table, at = [], 0
    for h in have:
        table.append((order[at:at + h] + [-7] * W)[:W])
        at += h
    free = order[at:at + max(0, sum(need) + spare)]
    T = max(0, sum(new) + room)
    want = plan_model(cached, new, table, free, page, T)
    wide = torch.full((R, W + 3), -9, dtype=torch.int32, device="cuda")  # rows with a stride
    wide[:, :W] = ints(table)
    got = F.plan_pages(ints(cached), ints(new), wide[:, :W], ints(free), page, T)
    for name, a, b in zip(got._fields, got, want):
        assert a.tolist() == b, name
    assert wide[:, :W].tolist() == want[5]
    assert bool((wide[:, W:] == -9).all())


def test_plan_pages_takes_any_lengths():
    """Negative lengths count as 0, lengths near 2^31 are not served, nothing overflows."""
    big = 2 ** 31 - 1
    cached, new = [-5, big, 3, 20, big], [2, 1, -1, 4, big]
    table = [[1, 2], [3, 4], [5, 6], [7, 8], [9, 10]]
    want = plan_model(cached, new, table, [11, 12], 16, 6)
    t = ints(table)
    got = F.plan_pages(ints(cached), ints(new), t, ints([11, 12]), 16, 6)
    live = [x >= 0 for x in want[3]]
    for name, a, b in zip(got._fields, got, want):
        if name == "positions":  # of tokens that are served; the others' may pass 31 bits
            assert [x for x, s in zip(a.tolist(), live) if s] == [x for x, s in zip(b, live) if s]
        else:
            assert a.tolist() == b, name
    assert t.tolist() == want[5]


def test_plan_pages_without_requests_or_tokens():
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    p = F.plan_pages(none, none, none.view(0, 4), none, 16, 3)
    assert p.cu_q.tolist() == [0] and p.slot_map.tolist() == [-1] * 3 and p.info.tolist() == [0, 0]
    p = F.plan_pages(ints([4]), ints([0]), ints([[2]]), none, 16, 0)
    assert p.cu_q.tolist() == [0, 0] and p.kv_lens.tolist() == [4] and p.info.tolist() == [0, 0]


# ------------------------------------------------------------------ rope_append
def rotated(x, positions, inv_freq, interleaved, amp):
    """(result, |a| + |b| of each channel's pair) in 64 bits."""
    rd = 0 if inv_freq is None else 2 * inv_freq.numel()
    y = x.double()
    if rd == 0:
        return y, y.abs() * 0
    ang = (positions.double()[:, None] * inv_freq.double())[:, None]
    c, s = ang.cos() * amp, ang.sin() * amp
    ia = torch.arange(0, rd, 2) if interleaved else torch.arange(rd // 2)
    ib = ia + (1 if interleaved else rd // 2)
    a, b = y[..., ia], y[..., ib]
    out, size = y.clone(), torch.zeros_like(y)
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * amp
    return out, size


def close(got, want, size):
    f = torch.finfo(got.dtype)
    err = (got.double() - want).abs()
    tol = f.eps / 2 * want.abs() + size * 2.0 ** -20 + f.smallest_normal * f.eps
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("T,H,Hkv,D,rd,inter,dt,page,far", [
    (1, 32, 8, 128, 128, False, BF, 16, 0), (1, 1, 1, 64, 16, True, FP, 16, 5), (3, 28, 4, 128, 64, False, FP, 32, 131070),
    (17, 4, 4, 64, 64, True, BF, 64, 2 ** 20 - 9), (700, 8, 2, 128, 128, True, BF, 16, 2 ** 24), (2500, 32, 8, 128, 96, False, BF, 128, 1),
    (9, 7, 1, 128, 112, False, FP, 1, 77), (33, 2, 2, 64, 0, False, BF, 16, 3), (5000, 16, 16, 64, 32, False, BF, 16, 0)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_rope_append(T, H, Hkv, D, rd, inter, dt, page, far, layout):
    g = torch.Generator().manual_seed(T + D)
    qkv = torch.randn(T, (H + 2 * Hkv) * D + 8, generator=g).to(dt).cuda()
    q = qkv[:, :H * D].view(T, H, D)
    k = qkv[:, H * D:(H + Hkv) * D].view(T, Hkv, D)
    v = qkv[:, (H + Hkv) * D:(H + 2 * Hkv) * D].view(T, Hkv, D)
    P = -(-T // page) + 2
    shape = (P, Hkv, page, D) if layout == "heads" else (P, page, Hkv, D)
    kp = torch.randn(shape, generator=g).to(dt).cuda()
    vp = torch.randn(shape, generator=g).to(dt).cuda()
    if layout == "tokens":
        kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
    slots = torch.randperm(P * page, generator=g)[:T].to(torch.int32)
    if T > 4:  # tokens without a place
        slots[0], slots[2], slots[4] = -1, P * page, 2 ** 31 - 1
    pos = torch.arange(far, far + T, dtype=torch.int32)
    if T > 4:
        pos[3] = 0
    freq = None if rd == 0 else (10000.0 ** (-torch.arange(0, rd, 2).double() / rd)).float().cuda()
    pos, slots = pos.cuda(), slots.cuda()
    want_k, want_v = kp.double(), vp.double()
    size_k = torch.zeros_like(want_k)
    live = ((slots >= 0) & (slots < P * page)).nonzero()[:, 0]
    s = slots[live].long()
    rk, sk = rotated(k[live], pos[live], freq, inter, 1.25)
    want_k[s // page, :, s % page], size_k[s // page, :, s % page] = rk, sk
    want_v[s // page, :, s % page] = v[live].double()
    rq, sq = rotated(q, pos, freq, inter, 1.25)
    before = qkv.clone()
    got = F.rope_append(q, k, v, pos, slots, kp, vp, freq, interleaved=inter, attn_factor=1.25)
    assert got.shape == (T, H, D) and got.dtype == dt
    assert torch.equal(qkv, before)
    close(got, rq, sq)
    close(kp, want_k, size_k)
    assert torch.equal(vp.double(), want_v)
    # in place, and without q
    keep = kp.clone()
    assert F.rope_append(None, k, v, pos, slots, kp, vp, freq, interleaved=inter, attn_factor=1.25) is None
    assert torch.equal(kp, keep)
    same = F.rope_append(q, k.clone(), v, pos, slots, kp, vp, freq, interleaved=inter, attn_factor=1.25, out=q)
    assert same is q and torch.equal(q, got)


def test_rope_append_refusals():
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    pos = ints([0, 1])

    def call(q=z(2, 2, 64), k=z(2, 2, 64), kp=z(4, 2, 16, 64), f=torch.ones(32, device="cuda")):
        F.rope_append(q, k, k, pos, pos, kp, kp.clone(), f)
    call()
    for bad in (dict(f=torch.ones(4, device="cuda")), dict(f=torch.ones(40, device="cuda")),
                dict(kp=z(4, 2, 24, 64)), dict(q=z(2, 2, 32), k=z(2, 2, 32), kp=z(4, 2, 16, 32)),
                dict(q=z(2, 2, 68)[..., 2:66]), dict(q=z(2, 2, 68)[..., :64]),
                dict(f=torch.ones(32))):
        with pytest.raises(ValueError):
            call(**bad)


# ------------------------------------------------------------------ paged_attention
class Batch:
    """Ragged requests over a shuffled pool, NaN wherever nothing may be read."""

    def __init__(self, lens, H, Hkv, D, dt, page, layout="heads", seed=0, spread=2.0, window=None, sinks=0, extra=0,
                 drop=False, width=0):
        g = torch.Generator().manual_seed(seed + 7)
        self.lens, self.dt, self.page, self.window, self.sinks = lens, dt, page, window, sinks
        self.H, self.Hkv, self.D = H, Hkv, D
        T = sum(n for _, n in lens) + extra
        self.q = (torch.randn(T, H, D, generator=g) * spread).to(dt).cuda()
        counts = [-(-(c + n) // page) for c, n in lens]
        P = sum(counts) + 3
        order = torch.randperm(P, generator=g).tolist()
        shape = (P, Hkv, page, D) if layout == "heads" else (P, page, Hkv, D)
        self.kp = torch.full(shape, NAN, dtype=dt, device="cuda")
        self.vp = torch.full(shape, NAN, dtype=dt, device="cuda")
        if layout == "tokens":
            self.kp, self.vp = self.kp.transpose(1, 2), self.vp.transpose(1, 2)
        W = max(counts + [1, -(-width // page)]) + 1
        table, self.k, self.v, at = [], [], [], 0
        for (c, n), m in zip(lens, counts):
            ids = order[at:at + m]
            at += m
            k = torch.randn(Hkv, c + n, D, generator=g).to(dt).cuda()
            v = torch.randn(Hkv, c + n, D, generator=g).to(dt).cuda()
            self.k.append(k)
            self.v.append(v)
            first = max(0, c - window + 1) if window else 0  # the first key behind the sinks that is seen
            row = []
            for i, page_id in enumerate(ids):
                lo, hi = i * page, min((i + 1) * page, c + n)
                if drop and lo >= sinks and hi <= first and hi == lo + page:
                    row.append(random.Random(i).choice([-1, P, 2 ** 31 - 1, page_id]))  # gone; its memory holds NaN
                    continue
                self.kp[page_id, :, :hi - lo] = k[:, lo:hi]
                self.vp[page_id, :, :hi - lo] = v[:, lo:hi]
                row.append(page_id)
            table.append(row + [-1] * (W - m))
        self.table = ints(table).view(len(lens), W)
        self.cu = ints(starts([n for _, n in lens]))
        self.kv = ints([c + n for c, n in lens])

    def run(self, **kw):
        return F.paged_attention(self.q, self.kp, self.vp, self.table, self.cu, self.kv, window=self.window,
                                 sinks=self.sinks, **kw)

    def check(self, got, scale=None):
        G = self.H // self.Hkv
        scale = scale or self.D ** -0.5
        u = torch.finfo(self.dt).eps / 2
        at = 0
        for (c, n), k, v in zip(self.lens, self.k, self.v):
            if n:
                q = self.q[at:at + n].double().view(n, self.Hkv, G, self.D).permute(1, 2, 0, 3)
                k, v = k.double()[:, None], v.double()[:, None]
                s = q @ k.transpose(-1, -2) * scale
                S = float((q.abs() @ k.abs().transpose(-1, -2)).max()) * scale
                i, j = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
                seen = j <= i
                if self.window:
                    seen &= (j > i - self.window) | (j < self.sinks)
                p = s.masked_fill(~seen, -math.inf).softmax(-1)
                want, A = (p @ x for x in (v, v.abs()))
                e = 2 * ((self.D + 2) * 2.0 ** -23 * S + 2.0 ** -20)
                tol = u * want.abs() + (u + e) * A
                if self.dt == FP:
                    tol = tol + (c + n) * 2.0 ** -24 * float(v.abs().max())
                o = got[at:at + n].double().view(n, self.Hkv, G, self.D).permute(1, 2, 0, 3)
                err = (o - want).abs()
                assert bool((err <= tol).all()), (c, n, float(err.max()), float((err - tol).nan_to_num(9.0).max()))
            at += n


LENS = {
    "one": [(0, 1)],
    "edges": [(0, 1), (62, 1), (63, 1), (64, 1), (0, 0), (65, 3), (127, 2), (0, 64), (0, 65), (15, 1), (16, 1)],
    "decode": [(1000, 1), (1, 1), (4095, 1), (2300, 1), (0, 0), (777, 1)],
    "chunks": [(1000, 37), (0, 200), (129, 1), (0, 129), (3333, 300), (64, 64)],
    "long": [(20000, 1)],
    "longchunk": [(9001, 150)],
}


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("H,Hkv,D,dt,page,layout", [
    (32, 8, 128, BF, 16, "heads"), (28, 4, 128, FP, 32, "heads"), (4, 4, 64, BF, 64, "tokens"), (16, 1, 128, BF, 128, "heads"),
    (9, 3, 64, FP, 256, "heads"), (5, 1, 128, FP, 16, "tokens")])
def test_paged_attention(lens, H, Hkv, D, dt, page, layout):
    b = Batch(LENS[lens], H, Hkv, D, dt, page, layout)
    b.check(b.run())
    F.check_status()


@pytest.mark.parametrize("lens", ["edges", "decode", "chunks", "long", "longchunk"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 0), (100, 4), (700, 130), (5000, 64), (10 ** 9, 3)])
@pytest.mark.parametrize("H,Hkv,D,dt,page", [(8, 2, 128, BF, 16), (7, 1, 64, FP, 128)])
def test_paged_attention_window(lens, window, sinks, H, Hkv, D, dt, page):
    b = Batch(LENS[lens], H, Hkv, D, dt, page, window=window, sinks=sinks, drop=True)
    b.check(b.run())


# Long table rows and requests of 1024 rows on average: the kernel with the larger tiles.
@pytest.mark.parametrize("lens", [
    [(1000, 37), (0, 200), (129, 1), (0, 129), (3333, 300), (64, 64), (10, 1400)], [(9001, 300)], [(0, 1024)],
    [(17, 1), (40, 64), (0, 0), (0, 1000), (127, 129), (255, 600)], [(20000, 260)]])
@pytest.mark.parametrize("H,Hkv,D,dt,page,layout", [
    (32, 8, 128, BF, 16, "heads"), (28, 4, 128, FP, 32, "heads"), (16, 4, 64, BF, 64, "tokens"), (16, 1, 128, BF, 128, "heads"),
    (15, 3, 64, FP, 256, "heads"), (5, 1, 128, FP, 16, "tokens"), (100, 1, 64, BF, 16, "heads")])
def test_paged_attention_long_rows(lens, H, Hkv, D, dt, page, layout):
    assert sum(n for _, n in lens) * (H // Hkv) >= 1024 * len(lens)
    b = Batch(lens, H, Hkv, D, dt, page, layout, width=20000)
    b.check(b.run())
    F.check_status()


@pytest.mark.parametrize("D,dt,page", [(64, BF, 16), (128, FP, 128)])
def test_paged_attention_long_rows_without_sharing(D, dt, page):
    b = Batch([(50, 1100)], 3, 3, D, dt, page, width=20000)
    b.check(b.run())


@pytest.mark.parametrize("window,sinks", [(4100, 0), (5000, 4), (20000, 130), (10 ** 9, 3)])
@pytest.mark.parametrize("H,Hkv,D,dt,page", [(8, 2, 128, BF, 16), (14, 2, 64, FP, 128)])
def test_paged_attention_long_window(window, sinks, H, Hkv, D, dt, page):
    b = Batch([(20100, 600), (0, 70), (16390, 290)], H, Hkv, D, dt, page, window=window, sinks=sinks, drop=True)
    b.check(b.run())


@pytest.mark.parametrize("H,Hkv", [(128, 1), (64, 1), (66, 2), (100, 1)])
def test_paged_attention_many_heads_to_a_kv_head(H, Hkv):
    b = Batch(LENS["edges"] + [(500, 5)], H, Hkv, 64, BF, 16)
    b.check(b.run())


@pytest.mark.parametrize("lens", [[(i % 70, 1) for i in range(1300)], [(100, 9003), (7, 1)], [(40, 2)] * 1024])
@pytest.mark.parametrize("window,sinks,width", [(None, 0, 0), (90, 5, 0), (None, 0, 20000)])
def test_paged_attention_many_q_tiles(lens, window, sinks, width):
    """More q tiles than a CTA schedules by itself, and just as many as it does."""
    b = Batch(lens, 16, 1, 64, BF, 16, window=window, sinks=sinks, drop=True, width=width)
    b.check(b.run())


@pytest.mark.parametrize("width", [0, 20000])
@pytest.mark.parametrize("dt", [BF, FP])
def test_paged_attention_scores_that_grow_and_peak(dt, width):
    """Scores far apart (the running maximum moves by more than its slack) and a scale of its own."""
    b = Batch([(700, 640), (1500, 1)], 8, 2, 64, dt, 16, spread=1.0, width=width)
    ramp = torch.linspace(0.0, 1.0, 1600, device="cuda")
    for r, (c, n) in enumerate(b.lens):
        k = b.k[r].float()
        b.q[:] = b.q.abs()
        k = (k.abs() * (ramp[:c + n] * (6.0 if dt == BF else 3.0))[None, :, None]).to(dt)
        b.k[r] = k
        for i in range(-(-(c + n) // 16)):
            hi = min(16, c + n - 16 * i)
            b.kp[int(b.table[r, i]), :, :hi] = k[:, 16 * i:16 * i + hi]
    b.check(b.run(scale=0.5), scale=0.5)


@pytest.mark.parametrize("G,width,extra", [(2, 0, 4), (128, 20000, 40)])
def test_rows_of_no_request_stay_and_empty_requests_give_zeros(G, width, extra):
    b = Batch([(30, 3), (0, 5), (100, 2), (40, 0)], 2 * G, 2, 64, BF, 16, extra=extra, width=width)
    out = torch.full_like(b.q, 7.0)
    b.kv[1] = 0  # not served: its five tokens see nothing
    got = F.paged_attention(b.q, b.kp, b.vp, b.table, b.cu, b.kv, out=out)
    assert got is out
    assert bool((out[10:] == 7.0).all())
    assert bool((out[3:8] == 0.0).all())
    lens = b.lens
    b.lens = [lens[0]]
    b.check(out)
    b.lens, b.k, b.v, b.q = [lens[2]], b.k[2:3], b.v[2:3], b.q[8:]
    b.check(out[8:])


@pytest.mark.parametrize("n,G,width", [(5, 2, 0), (15, 100, 20000)])
def test_more_new_tokens_than_keys(n, G, width):
    """Two keys fewer than new tokens: the first two come before the first key and see nothing."""
    b = Batch([(0, n)], G, 1, 64, BF, 16, width=width)
    b.kv[0] = n - 2
    got = b.run()
    assert bool((got[:2] == 0.0).all())
    b.lens, b.q, b.k, b.v = [(0, n - 2)], b.q[2:], [b.k[0][:, :n - 2]], [b.v[0][:, :n - 2]]
    b.check(got[2:])


@pytest.mark.parametrize("G,width", [(2, 0), (128, 20000)])
def test_lengths_outside_their_tensors_are_kept_inside(G, width):
    """cu_q and kv_lens are device data: whatever they hold, no row outside q and no page outside the table is used."""
    b = Batch([(30, 13), (50, 14)], 2 * G, 2, 64, BF, 16, width=width)
    b.kp.nan_to_num_(0.0)
    b.vp.nan_to_num_(0.0)
    out = torch.zeros_like(b.q)
    for cu, kv in (([0, 13, 10 ** 6], [43, 64]), ([-5, 13, 27], [2 ** 31 - 1, 64]), ([27, 13, 0], [-1, 64]),
                   ([0, 27, 27], [10 ** 6, 0]), ([2 ** 31 - 1, -2 ** 31, 5], [43, 64])):
        F.paged_attention(b.q, b.kp, b.vp, b.table, ints(cu), ints(kv), out=out)
    torch.cuda.synchronize()
    F.check_status()
    b.check(b.run())


def test_strided_q_and_out():
    b = Batch(LENS["chunks"], 8, 2, 128, BF, 32)
    T = b.q.shape[0]
    wide = torch.full((T, 12, 136), NAN, dtype=BF, device="cuda")
    wide[:, 2:10, :128] = b.q
    out = torch.full((8, T, 160), 5.0, dtype=BF, device="cuda")
    got = F.paged_attention(wide[:, 2:10, :128], b.kp, b.vp, b.table, b.cu, b.kv, out=out.transpose(0, 1)[..., 16:144])
    b.check(got)
    assert bool((out[..., :16] == 5.0).all()) and bool((out[..., 144:] == 5.0).all())


def test_requests_that_share_pages():
    """Two requests with a common prefix in the same pages, and one listed twice in the batch."""
    b = Batch([(128, 5), (128, 1), (130, 70)], 8, 2, 128, BF, 16)
    b.table[1, :8] = b.table[0, :8]
    b.k[1] = torch.cat([b.k[0][:, :128], b.k[1][:, 128:]], 1)
    b.v[1] = torch.cat([b.v[0][:, :128], b.v[1][:, 128:]], 1)
    b.check(b.run())
    twice = torch.cat([b.table, b.table[2:]])
    got = F.paged_attention(torch.cat([b.q, b.q[6:]]), b.kp, b.vp, twice, ints([0, 5, 6, 76, 146]), ints([133, 129, 200, 200]))
    b.check(got)
    b.q, b.lens, b.k, b.v = b.q[6:], b.lens[2:], b.k[2:], b.v[2:]
    b.check(got[76:])


@pytest.mark.parametrize("width", [0, 20000])
def test_infinities_and_nan_stay_in_their_rows(width):
    """A request whose values are broken, and a broken row of q, leave every other row as it was."""
    lens = [(300, 40), (90, 200), (700, 600)]
    b = Batch(lens, 8, 2, 128, BF, 16, width=width)
    want = b.run().clone()
    b.vp[b.table[1, :19].long()] = math.inf
    b.kp[b.table[1, :19].long()] = NAN
    b.q[5, 3] = NAN
    b.q[250] = math.inf
    got = b.run()
    same = torch.ones(840, 8, dtype=torch.bool, device="cuda")
    same[40:240] = False
    same[5, 3] = False
    same[250] = False
    assert torch.equal(got[same], want[same])


def test_strides_of_single_rows_do_not_matter():
    b = Batch([(40, 1)], 1, 1, 64, BF, 64)
    q = torch.zeros(3, 1, 67, dtype=BF, device="cuda")
    q = q.as_strided((1, 1, 64), (67, 5, 1))
    q.copy_(b.q)
    page = int(b.table[0, 0])
    kp, vp = (x[page:page + 1].as_strided((1, 1, 64, 64), (3, 1, 64, 1), x[page].storage_offset()) for x in (b.kp, b.vp))
    b.check(F.paged_attention(q, kp, vp, ints([[0]]), b.cu, b.kv))


def test_pool_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements, its pages in use at both ends."""
    P, Hkv, page, D = 33000, 8, 64, 128
    kp = torch.empty(P, Hkv, page, D, dtype=BF, device="cuda")
    vp = torch.empty(P, Hkv, page, D, dtype=BF, device="cuda")
    assert kp.numel() > 2 ** 31
    T, n = 150, 3
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(T, Hkv, D, generator=g).to(BF).cuda() for _ in range(2))
    q = torch.randn(n, 16, D, generator=g).to(BF).cuda()
    table = ints([[P - 1, 0, P - 2]])
    pos = torch.arange(T, device="cuda")
    slots = (table[0, pos // page].long() * page + pos % page).to(torch.int32)
    F.rope_append(None, k, v, pos.to(torch.int32), slots, kp, vp, None)
    b = Batch([(T - n, n)], 16, Hkv, D, BF, page)
    b.q, b.k, b.v = q, [k.transpose(0, 1)], [v.transpose(0, 1)]
    b.check(F.paged_attention(q, kp, vp, table, ints([0, n]), ints([T])))


def test_paged_attention_refusals():
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731

    def call(q=z(2, 4, 64), kp=z(3, 2, 16, 64), scale=None):
        F.paged_attention(q, kp, kp.clone(), ints([[0]]), ints([0, 2]), ints([2]), scale=scale)
    call()
    for bad in (dict(kp=z(3, 2, 8, 64)), dict(kp=z(3, 2, 48, 64)), dict(kp=z(3, 2, 512, 64)),
                dict(q=z(2, 4, 32), kp=z(3, 2, 16, 32)), dict(q=z(2, 258, 64)), dict(q=z(2, 4, 68)[..., :64]),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=NAN)):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError):
        F.plan_pages(ints([1]), ints([1]), ints([[0]]), ints([1]), 24, 1)


@pytest.mark.parametrize("width", [0, 20000])
def test_two_streams_at_once(width):
    one = Batch(LENS["chunks"] + [(10, 1400)], 8, 2, 128, BF, 16, seed=1, width=width)
    two = Batch(LENS["decode"], 8, 2, 128, BF, 16, seed=2)
    want = one.run().clone(), two.run().clone()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, b in enumerate((one, two)):
            with torch.cuda.stream(streams[i]):
                got[i].append(b.run())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)  # the shares and the merge's order are fixed


# ------------------------------------------------------------------ together
class Server:
    """A pool, its free list and the requests' history, stepped through the three operators."""

    def __init__(self, R, H, Hkv, D, dt, page, pages, width, inv_freq, rows):
        self.H, self.Hkv, self.D, self.page, self.inv_freq = H, Hkv, D, page, inv_freq
        self.kp, self.vp = (torch.full((pages, Hkv, page, D), NAN, dtype=dt, device="cuda") for _ in range(2))
        self.table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.cached, self.new = torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")
        self.qkv = torch.zeros(rows, (H + 2 * Hkv) * D, dtype=dt, device="cuda")
        self.out = torch.full((rows, H, D), 3.0, dtype=dt, device="cuda")

    def step(self):
        H, Hkv, D, T = self.H, self.Hkv, self.D, self.qkv.shape[0]
        x = self.qkv
        self.plan = F.plan_pages(self.cached, self.new, self.table, self.free, self.page, T)
        self.q = F.rope_append(x[:, :H * D].view(T, H, D), x[:, H * D:(H + Hkv) * D].view(T, Hkv, D),
                               x[:, (H + Hkv) * D:].view(T, Hkv, D), self.plan.positions, self.plan.slot_map, self.kp, self.vp,
                               self.inv_freq)
        F.paged_attention(self.q, self.kp, self.vp, self.table, self.plan.cu_q, self.plan.kv_lens, out=self.out)


@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(graph):
    """Chunks, decoding, idle requests and a padded batch over several steps: plan, append and attention
    together against contiguous histories; the captured step is replayed with other lengths."""
    R, H, Hkv, D, dt, page, rows = 4, 8, 2, 128, BF, 16, 160
    inv_freq, _ = F.rotary_inv_freq(128, 500000.0, device="cuda")
    s = Server(R, H, Hkv, D, dt, page, 64, 24, inv_freq, rows)
    gen = torch.Generator().manual_seed(5)
    steps = [[100, 1, 0, 50], [1, 1, 33, 1], [1, 1, 1, 1], [0, 120, 1, 1], [1, 1, 1, 60]]
    if graph:
        s.step()  # loads the kernels
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            s.step()
    cached = [0] * R
    held = [(torch.empty(Hkv, 0, D, dtype=dt, device="cuda"),) * 2] * R
    for new in steps:
        s.qkv.copy_(torch.randn(rows, s.qkv.shape[1], generator=gen).to(dt))
        s.new.copy_(ints(new))
        s.cached.copy_(ints(cached))
        s.out.fill_(3.0)
        if graph:
            captured.replay()
        else:
            s.step()
        taken, unserved = s.plan.info.tolist()
        assert unserved == 0 and taken == sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        assert bool((s.out[sum(new):] == 3.0).all())
        at = 0
        for r, n in enumerate(new):
            pos = torch.arange(cached[r], cached[r] + n, device="cuda")
            x = s.qkv[at:at + n]
            want, size = rotated(x[:, H * D:(H + Hkv) * D].view(n, Hkv, D), pos, inv_freq, False, 1.0)
            ids = s.table[r, :-(-(cached[r] + n) // page)].long()
            k, v = (p[ids].transpose(0, 1).flatten(1, 2)[:, :cached[r] + n] for p in (s.kp, s.vp))
            close(k[:, cached[r]:], want.transpose(0, 1), size.transpose(0, 1))
            assert torch.equal(v[:, cached[r]:], x[:, (H + Hkv) * D:].view(n, Hkv, D).transpose(0, 1))
            for new_k, old in ((k, held[r][0]), (v, held[r][1])):  # earlier tokens are where they were
                assert torch.equal(new_k[:, :cached[r]], old)
            held[r] = (k, v)
            if n:
                b = Batch([(cached[r], n)], H, Hkv, D, dt, page)
                b.q, b.k, b.v = s.q[at:at + n], [k], [v]
                b.check(s.out[at:at + n])
            at += n
            cached[r] += n
        s.free = s.free if graph else s.free[taken:]
        if graph:
            s.free.copy_(torch.cat([s.free[taken:], s.free[:taken]]))
    F.check_status()


def test_handover_from_the_sparse_prefill():
    """A prompt attended by myattn_prefill is handed to the pages; decoding it there equals decode_attention."""
    L, H, Hkv, D, page = 1500, 8, 2, 128, 64
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(1, h, L, D, generator=g).bfloat16().cuda() for h in (H, Hkv, Hkv))
    F.myattn_prefill(q, k, v, 0)
    pages = -(-(L + 1) // page)
    kp, vp = (torch.full((pages, Hkv, page, D), NAN, dtype=BF, device="cuda") for _ in range(2))
    table = torch.full((1, pages), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")
    plan = F.plan_pages(ints([0]), ints([L]), table, free, page, L)
    F.rope_append(None, k[0].transpose(0, 1), v[0].transpose(0, 1), plan.positions, plan.slot_map, kp, vp, None)
    got = F.paged_attention(q[0, :, -1:].transpose(0, 1), kp, vp, table, ints([0, 1]), plan.kv_lens)
    want = F.decode_attention(q[:, :, -1:], k, v)
    # each is within two roundings of the exact value
    A = 2 * float(v.float().abs().max())
    assert float((got[0].float() - want[0].float()).abs().max()) <= 2 * 2.0 ** -8 * A
