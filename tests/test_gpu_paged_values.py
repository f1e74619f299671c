"""Values and lengths at which the paged operators can go wrong.

Tolerances as in test_gpu_paged.py, where a test does not derive its own.
"""
import math

import pytest
import torch

import fftsparse_b200 as F
from test_gpu_paged import BF, FP, NAN, Batch, ints

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ scores that are not finite
def poke(b, r, head, keys, channel, value):
    """Sets k[head, keys, channel] of request r, in the history and in its pages."""
    b.k[r][head, keys, channel] = value
    n = b.k[r].shape[1]
    for c in range(n)[keys]:
        b.kp[int(b.table[r, c // b.page]), head, c % b.page] = b.k[r][head, c]


def check_broken(b, got):
    """got against the definition in 64 bits: NaN where it has NaN, within the tolerance elsewhere."""
    G, u, at, broken = b.H // b.Hkv, torch.finfo(b.dt).eps / 2, 0, 0
    for (c, n), k, v in zip(b.lens, b.k, b.v):
        q = b.q[at:at + n].double().view(n, b.Hkv, G, b.D).permute(1, 2, 0, 3)
        k, v = k.double()[:, None], v.double()[:, None]
        seen = torch.arange(c + n, device="cuda") <= torch.arange(c, c + n, device="cuda")[:, None]
        s = (q @ k.transpose(-1, -2) * b.D ** -0.5).masked_fill(~seen, -math.inf)
        p = s.softmax(-1)  # NaN for a row with a NaN or +inf among the keys that it sees, or with nothing but -inf
        want, A = p @ v, p @ v.abs()
        S = (q.abs().nan_to_num(0.0, 0.0) @ k.abs().nan_to_num(0.0, 0.0).transpose(-1, -2)).max() * b.D ** -0.5
        e = 2 * ((b.D + 2) * 2.0 ** -23 * float(S) + 2.0 ** -20)
        o = got[at:at + n].double().view(n, b.Hkv, G, b.D).permute(1, 2, 0, 3)
        assert torch.equal(o.isnan(), want.isnan())
        fine = ~want.isnan()
        assert bool(((o - want).abs() <= u * want.abs() + (u + e) * A)[fine].all())
        broken += int((~fine).sum())
        at += n
    return broken


@pytest.mark.parametrize("last", [(20000, 1), (9000, 300)])  # the second: the kernel with the larger tiles
def test_broken_scores_reach_their_rows_and_no_others(last):
    b = Batch([(300, 40), (90, 200), (700, 600), last], 8, 2, 128, BF, 16)
    assert (b.q.shape[0] * 4 >= 1024 * 4) == (last[1] == 300)
    poke(b, 0, 0, slice(10, 11), 3, math.inf)         # +inf where q's channel is positive, -inf where it is negative
    b.q[5, 3] = NAN
    b.q[250] = math.inf
    poke(b, 1, 0, slice(0, 290), 7, b.k[1][0, :, 7].abs().neg() - 0.25)
    b.q[60, :4, 7] = math.inf                          # every key that the row sees scores -inf
    poke(b, 2, 1, slice(1000, 1001), slice(None), NAN)  # of no concern to the tokens before it
    # the last request's keys are spread over many shares: some of them see nothing but the broken ones
    poke(b, 3, 0, slice(6000, 6600), slice(None), NAN)
    b.q[840:, 4:, 5] = b.q[840:, 4:, 5].abs() + 0.25
    poke(b, 3, 1, slice(6000, 6600), 5, -math.inf)      # weight 0
    got = b.run()
    assert check_broken(b, got) > 0
    assert bool(got[840:, :4].isnan().all()) and bool(got[840:, 4:].isfinite().all())
    F.check_status()


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("H,Hkv,D,dt,page", [(8, 2, 128, BF, 16), (4, 4, 64, FP, 64), (14, 2, 128, FP, 32), (3, 1, 64, BF, 256)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 0), (130, 5), (5000, 100)])
@pytest.mark.parametrize("width", [0, 20000])
def test_broken_values_reach_the_tokens_that_see_them_and_no_others(H, Hkv, D, dt, page, window, sinks, width):
    """v with NaN and infinities in some channels of some keys: a channel is not finite in the rows that see such a key,
    and as it should be in all others, the tokens before it and those whose window has left it behind."""
    lens = [(0, 300), (37, 1), (700, 2200 if width else 150), (63, 70), (0, 0), (5, 4)]
    b = Batch(lens, H, Hkv, D, dt, page, window=window, sinks=sinks, width=width)
    g = torch.Generator().manual_seed(D + page)
    for r, (c, n) in enumerate(lens):
        length = c + n
        for key in [] if length < 4 else [length - 1, length - 3, c + n // 2, c + n // 3, max(0, c - 60), 0, 3]:
            h, ch = int(torch.randint(Hkv, (1,), generator=g)), torch.randperm(D, generator=g)[:5]
            b.v[r][h, key, ch] = torch.tensor([NAN, math.inf, -math.inf, -NAN, math.inf], dtype=dt, device="cuda")
            b.vp[int(b.table[r, key // page]), h, key % page] = b.v[r][h, key]
    got = b.run()
    G, u, at, broken = H // Hkv, torch.finfo(dt).eps / 2, 0, 0
    for (c, n), k, v in zip(lens, b.k, b.v):
        if not n:
            continue
        q = b.q[at:at + n].double().view(n, Hkv, G, D).permute(1, 2, 0, 3)
        k, v = k.double()[:, None], v.double()[:, None]
        i, j = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
        seen = j <= i
        if window:
            seen &= (j > i - window) | (j < sinks)
        s = q @ k.transpose(-1, -2) * D ** -0.5
        S = float((q.abs() @ k.abs().transpose(-1, -2)).max()) * D ** -0.5
        p = s.masked_fill(~seen, -math.inf).softmax(-1)
        fine = v.nan_to_num(0.0, 0.0, 0.0)
        want, A = p @ fine, p @ fine.abs()
        up, down = (seen.double() @ (x | v.isnan()).double() > 0 for x in (v == math.inf, v == -math.inf))
        e = 2 * ((D + 2) * 2.0 ** -23 * S + 2.0 ** -20)
        tol = u * want.abs() + (u + e) * A + ((c + n) * 2.0 ** -24 * float(fine.abs().max()) if dt == FP else 0.0)
        o = got[at:at + n].double().view(n, Hkv, G, D).permute(1, 2, 0, 3)
        bad = (up | down).expand_as(o)
        assert torch.equal(~o.isfinite(), bad)
        assert bool(o[(up & down).expand_as(o)].isnan().all())
        # an infinity is one, or NaN where the weight before it is 0 in the products' type
        assert bool(((o == math.inf) | o.isnan())[(up & ~down).expand_as(o)].all())
        assert bool(((o == -math.inf) | o.isnan())[(down & ~up).expand_as(o)].all())
        assert bool(((o - want).abs() <= tol)[~bad].all())
        broken += int(bad.sum())
        at += n
    assert broken > 0
    F.check_status()


# ------------------------------------------------------------------ sums of many small weights
SUM_KEYS = {FP: 16384, BF: 131072}  # keys that the tensor core sums up before the sum is taken over


def sum_error(dt):
    """Of such a sum, relative to what its terms' sizes sum to: 16 products at a time, each cut at 2^-25 of the sum,
    then the sum at its last step, 2^-23."""
    return SUM_KEYS[dt] * (2.0 ** -25 + 2.0 ** -23 / 16)


@pytest.mark.parametrize("deficit,keys", [(24.9, 131072), (25.01, 131072), (25.9, 131072), (31.9, 131072),
                                          (32.01, 131072), (25.01, 1 << 20), (25.9, 1 << 20)])
@pytest.mark.parametrize("top", [1.0, 0.0])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("dt", [FP, BF])
def test_many_keys_far_below_the_first_one(dt, chunk, top, deficit, keys):
    """The first key outweighs each of the others by 2^deficit, together they count: sum p v with v = top for the
    first key, 1 for the others.

    One rounding of the result.  P in fp16 is off by at most half of its smallest step, 2^-25; a row's maximum stands at
    2^7 or above, so each of the keys is off by at most 2^-32 of the first one's weight.  P in bf16 is off by one
    rounding.  The tensor core's sums, at most 1 of the total weight each, are off by sum_error; the ones without the
    first key in proportion to their own keys."""
    D, page = 64, 256
    k = torch.zeros(keys // page + 1, 1, page, D, dtype=dt, device="cuda")
    k[..., 0] = -16.0
    k[0, 0, 0, 0] = 0.0
    v = torch.ones_like(k)
    v[0, 0, 0] = top
    # as many (q tile, head)s as CTAs, so that a share holds a whole one
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    R, T = (1, 256 * sms) if chunk else (2 * sms, 2 * sms)
    if chunk:
        lens, cu = [keys + T], [0, T]
        more = T // page + 1
        k, v = (torch.cat([x, x[1:2].expand(more, -1, -1, -1)]) for x in (k, v))
        n = torch.arange(keys, keys + T, device="cuda").double()  # keys that a row sees besides the first one
    else:
        lens, cu = [keys] * R, list(range(R + 1))
        n = torch.full((T,), keys - 1.0, device="cuda", dtype=torch.float64)
    table = torch.arange(k.shape[0], dtype=torch.int32, device="cuda").repeat(R, 1)
    q = torch.zeros(T, 1, D, dtype=dt, device="cuda")
    q[..., 0] = 1.0
    scale = deficit * math.log(2.0) / 16.0
    got = F.paged_attention(q, k, v, table, ints(cu), ints(lens), scale=scale)[:, 0].double()
    rest = n * 2.0 ** -deficit
    want, u = (top + rest) / (1.0 + rest), torch.finfo(dt).eps / 2
    tol = u * want + sum_error(dt) + (n * 2.0 ** -32 if dt == FP else u * want)
    err = (got - want[:, None]).abs()
    assert bool((err <= tol[:, None]).all()), (float(err.max()), float(tol.min()))
    F.check_status()


@pytest.mark.parametrize("dt,keys", [(FP, 30011), (BF, 150001)])
@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (0.6, 70)])
def test_long_rows_in_one_share(chunk, dt, keys, window, sinks):
    """Rows of several sums each, whole in one share: random values against 64 bits, at the tolerance of test_gpu_paged.py
    with the sums' own error instead of one that grows with the keys."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    D, page, T = 64, 64, (256 * sms if chunk else 2 * sms)
    if chunk and dt == BF:
        keys = 90001
    window = window and int(window * keys)
    g = torch.Generator(device="cuda").manual_seed(keys)
    first = keys - T if chunk else 0  # position of the first row; a decoding row is at keys - 1
    pages = -(-keys // page)
    k, v = (torch.randn(pages, 1, page, D, generator=g, device="cuda").to(dt) for _ in range(2))
    q = (torch.randn(T, 1, D, generator=g, device="cuda") * 2).to(dt)
    R = 1 if chunk else T
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(R, 1)
    got = F.paged_attention(q, k, v, table, ints([0, T] if chunk else list(range(T + 1))), ints([keys] * R), window=window,
                            sinks=sinks if window else 0)
    u = torch.finfo(dt).eps / 2
    k, v = k.double().flatten(0, 2)[:keys], v.double().flatten(0, 2)[:keys]
    rows = torch.randperm(T, generator=torch.Generator().manual_seed(1))[:300].cuda()
    s = q[rows, 0].double() @ k.T * D ** -0.5
    S = float((q[rows, 0].double().abs() @ k.abs().T).max()) * D ** -0.5
    i, j = (rows + first if chunk else torch.full_like(rows, keys - 1))[:, None], torch.arange(keys, device="cuda")
    seen = j <= i
    if window:
        seen &= (j > i - window) | (j < sinks)
    p = s.masked_fill(~seen, -math.inf).softmax(-1)
    p = torch.where(seen.any(-1, keepdim=True), p, 0.0)  # a row before the first key: zeros
    want, A = p @ v, p @ v.abs()
    e = 2 * ((D + 2) * 2.0 ** -23 * S + 2.0 ** -20)
    tol = u * want.abs() + (u + e + sum_error(dt)) * A + (keys * 2.0 ** -32 * float(v.abs().max()) if dt == FP else 0.0)
    assert bool(((got[rows, 0].double() - want).abs() <= tol).all())
    F.check_status()


# ------------------------------------------------------------------ tensors whose rows overlap
def test_outputs_whose_rows_overlap_are_refused():
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    T, H, Hkv, D, P, page = 3, 4, 2, 64, 2, 16
    q, k, pool = z(T, H, D), z(T, Hkv, D), z(P, Hkv, page, D)

    def attend(out):
        F.paged_attention(q, pool, pool.clone(), ints([[0]]), ints([0, T]), ints([T]), out=out)

    def append(out=None, kp=pool, vp=pool.clone()):
        F.rope_append(q, k, k.clone(), ints([0, 1, 2]), ints([0, 1, 2]), kp, vp, None, out=out)

    wide = z(H, T + 1, D + 8)
    for out in (q, z(T, H, D), wide[:, :T, :D].transpose(0, 1), wide[:, 1:, 8:].transpose(0, 1)):
        attend(out)
        append(out)
    for out in (z(1, H, D).expand(T, H, D), z(T, 1, D).expand(T, H, D), z(1000).as_strided((T, H, D), (D, D, 1)),
                z(1000).as_strided((T, H, D), (H * D - 8, D, 1)), z(1000).as_strided((T, H, D), (H * D, D - 8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            attend(out)
        with pytest.raises(ValueError, match="overlap"):
            append(out)
    append(kp=z(P, page, Hkv, D).transpose(1, 2))
    for bad in (z(1, Hkv, page, D).expand(P, -1, -1, -1), z(P, 1, page, D).expand(-1, Hkv, -1, -1),
                z(P, Hkv, 1, D).expand(-1, -1, page, -1), z(9000).as_strided((P, Hkv, page, D), (page * D, page * D, D, 1))):
        with pytest.raises(ValueError, match="overlap"):
            append(kp=bad)
        with pytest.raises(ValueError, match="overlap"):
            append(vp=bad)
    # inputs may be broadcast
    F.rope_append(z(1, H, D).expand(T, H, D), z(T, 1, D).expand(T, Hkv, D), k, ints([0, 1, 2]), ints([0, 1, 2]), pool,
                  pool.clone(), None)


# ------------------------------------------------------------------ page numbers of no pool
@pytest.mark.parametrize("page", [1, 16, 4096])
def test_page_numbers_outside_every_pool_give_no_slot(page):
    """A slot is an int32: a page number whose slots do not fit, or a negative one, gives -1 and never another page's slot."""
    most = 2 ** 31 // page
    pages = [x for x in (-1, -most, -2 ** 31, most, most + 5, 2 ** 31 - 1, 0, most - 1) if x < 2 ** 31]
    R, have = len(pages), -(-(page - 1) // page)
    new = page + 2  # ends in the third page; the first one is in the table unless a page is a token
    free = ints([x for p in pages for x in (p, p, 3)[have:]])
    p = F.plan_pages(ints([page - 1] * R), ints([new] * R), ints([[x, -9, -9] for x in pages]), free, page, new * R)
    assert p.info.tolist() == [(3 - have) * R, 0]
    want = []
    for x in pages:
        for pos in range(page - 1, 2 * page + 1):
            at = (x, x, 3)[pos // page]
            want.append(at * page + pos % page if 0 <= at < most else -1)
    assert p.slot_map.tolist() == want


# ------------------------------------------------------------------ schedules
def schedule_bound(lens, G):
    """The q tiles that a call makes room for; up to 1024 of them every CTA builds the schedule itself."""
    T = sum(n for _, n in lens)
    return T // (128 // G) + min(len(lens), T)


@pytest.mark.parametrize("R,G,bound", [(193, 8, 205), (400, 4, 412), (964, 8, 1024), (965, 8, 1025), (512, 128, 1024)])
def test_schedules_of_many_requests(R, G, bound):
    """More requests than a CTA scans at a time (192), up to the last size whose schedule it builds itself and the next."""
    lens = [(i * 37 % 131, 1) for i in range(R)]
    assert schedule_bound(lens, G) == bound
    b = Batch(lens, G, 1, 64, BF, 16)
    b.check(b.run())
    F.check_status()


@pytest.mark.parametrize("lens,G,bound", [
    ([(7, 460)], 64, 231), ([(7, 1900), (0, 1), (300, 90)], 64, 998),
    ([(i * 11 % 90, i % 3) for i in range(450)], 64, 675)])
def test_schedules_of_many_q_tiles(lens, G, bound):
    """More q tiles than the threads that scan them, and idle requests among them."""
    assert schedule_bound(lens, G) == bound
    b = Batch(lens, G, 1, 64, BF, 16)
    b.check(b.run())


@pytest.mark.parametrize("lens,G,bound", [
    ([(7, 1700)], 64, 851), ([(7, 1700), (90, 30), (0, 64)], 64, 900), ([(0, 2046)], 64, 1024), ([(5, 2048)], 64, 1025),
    ([(i % 90, 8) for i in range(113)], 128, 1017)])
def test_schedules_of_the_larger_tiles(lens, G, bound):
    """Tiles of 256 rows: more of them than the 384 that a CTA scans at a time."""
    T = sum(n for _, n in lens)
    assert schedule_bound(lens, G) == bound and T * G >= 1024 * len(lens)
    b = Batch(lens, G, 1, 64, BF, 16, width=20000)
    b.check(b.run())
    F.check_status()
