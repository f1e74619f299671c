"""Host side of the paged operators without a GPU: refusals, rotary frequencies and
the share arithmetic of the paged attention's schedule."""
import ctypes
import math
import random

import pytest
import torch

import fftsparse_b200 as F


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------ refusals
def plan_args(**kw):
    a = dict(cached_lens=ints(3, 4), new_lens=ints(1, 1), block_table=torch.zeros(2, 4, dtype=torch.int32),
             free_pages=ints(5, 6), page_size=16, num_tokens=2)
    return dict(a, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(cached_lens=torch.zeros(2)), TypeError),
    (dict(cached_lens=torch.zeros(2, 1, dtype=torch.int32)), ValueError),
    (dict(new_lens=ints(1)), ValueError),
    (dict(new_lens=torch.ones(2, dtype=torch.int64)), TypeError),
    (dict(new_lens=ints(1, 2, 3, 4)[::2]), ValueError),
    (dict(block_table=torch.zeros(3, 4, dtype=torch.int32)), ValueError),
    (dict(block_table=torch.zeros(4, 2, dtype=torch.int32).t()), ValueError),
    (dict(block_table=torch.zeros(2, 4)), TypeError),
    (dict(free_pages=torch.zeros(2, 2, dtype=torch.int32)), ValueError),
    (dict(num_tokens=-1), ValueError),
    (dict(), ValueError),  # a good call, on CPU tensors
])
def test_plan_refusals(kw, err):
    with pytest.raises(err):
        F.plan_pages(**plan_args(**kw))


def rope_args(**kw):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(3, 4, 64, dtype=bf), k=torch.zeros(3, 2, 64, dtype=bf), v=torch.zeros(3, 2, 64, dtype=bf),
             positions=ints(0, 1, 2), slot_map=ints(0, 1, 2), k_pages=torch.zeros(2, 2, 16, 64, dtype=bf),
             v_pages=torch.zeros(2, 2, 16, 64, dtype=bf), inv_freq=torch.ones(32))
    return dict(a, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(k=torch.zeros(3, 2, 64)), TypeError),
    (dict(v=torch.zeros(3, 1, 64, dtype=torch.bfloat16)), ValueError),
    (dict(v=torch.zeros(3, 2, 64, dtype=torch.float16)), TypeError),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), ValueError),
    (dict(positions=ints(0, 1)), ValueError),
    (dict(slot_map=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(k_pages=torch.zeros(2, 3, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k_pages=torch.zeros(2, 3, 16, 64, dtype=torch.bfloat16),
          v_pages=torch.zeros(2, 3, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(inv_freq=torch.ones(32, dtype=torch.float64)), ValueError),
    (dict(q=None, out=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(), ValueError),
])
def test_rope_append_refusals(kw, err):
    with pytest.raises(err):
        F.rope_append(**rope_args(**kw))


def attn_args(**kw):
    bf = torch.bfloat16
    a = dict(q=torch.zeros(3, 4, 64, dtype=bf), k_pages=torch.zeros(2, 2, 16, 64, dtype=bf),
             v_pages=torch.zeros(2, 2, 16, 64, dtype=bf), block_table=torch.zeros(2, 1, dtype=torch.int32),
             cu_q=ints(0, 1, 3), kv_lens=ints(4, 4))
    return dict(a, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(q=torch.zeros(3, 4, 64)), TypeError),
    (dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(cu_q=ints(0, 1)), ValueError),
    (dict(cu_q=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(kv_lens=ints(4, 4, 4)), ValueError),
    (dict(block_table=torch.zeros(1, 1, dtype=torch.int32)), ValueError),
    (dict(window=0), ValueError),
    (dict(sinks=4), ValueError),
    (dict(window=8, sinks=-1), ValueError),
    (dict(out=torch.zeros(3, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(k_pages=torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16),
          v_pages=torch.zeros(0, 2, 16, 64, dtype=torch.bfloat16)), ValueError),
    (dict(), ValueError),
])
def test_paged_attention_refusals(kw, err):
    with pytest.raises(err):
        F.paged_attention(**attn_args(**kw))


# ------------------------------------------------------------------ rotary frequencies
def test_rotary_frequencies_of_each_scaling():
    d, base, L0 = 64, 10000.0, 4096
    f = [base ** (-2 * i / d) for i in range(d // 2)]

    def got(scaling, **kw):
        return F.rotary_inv_freq(d, base, scaling, **kw)

    def near(t, want):  # fp32: half a step
        w = torch.tensor(want, dtype=torch.float64)
        return bool(((t.double() - w).abs() <= torch.finfo(torch.float32).eps / 2 * w * 1.001).all())

    t, a = got(None)
    assert t.dtype == torch.float32 and a == 1.0 and near(t, f)
    t, a = got({"rope_type": "linear", "factor": 4.0})
    assert a == 1.0 and near(t, [x / 4 for x in f])
    dyn = {"type": "dynamic", "factor": 2.0, "original_max_position_embeddings": L0}
    assert near(got(dyn, seq_len=100)[0], f)
    grown = base * (2.0 * 16384 / L0 - 1.0) ** (d / (d - 2))
    assert near(got(dyn, seq_len=16384)[0], [grown ** (-2 * i / d) for i in range(d // 2)])

    t, _ = got({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                "original_max_position_embeddings": L0})
    want = []
    for x in f:
        wl = 2 * math.pi / x
        if wl > L0 / 1.0:
            want.append(x / 8)
        elif wl < L0 / 4.0:
            want.append(x)
        else:
            s = (L0 / wl - 1.0) / 3.0
            want.append((1 - s) * x / 8 + s * x)
    assert near(t, want)

    t, a = got({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": L0})
    lo = math.floor(d * math.log(L0 / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(d * math.log(L0 / (1 * 2 * math.pi)) / (2 * math.log(base)))
    want = []
    for i, x in enumerate(f):
        ramp = min(1.0, max(0.0, (i - lo) / (hi - lo)))
        want.append(x / 4 * ramp + x * (1 - ramp))
    assert near(t, want) and abs(a - (0.1 * math.log(4.0) + 1.0)) < 1e-12
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": L0}
    assert got(dict(yarn, attention_factor=1.5))[1] == 1.5
    m = [0.1 * x * math.log(4.0) + 1.0 for x in (0.7, 0.4)]
    assert abs(got(dict(yarn, mscale=0.7, mscale_all_dim=0.4))[1] - m[0] / m[1]) < 1e-12


@pytest.mark.parametrize("args", [(0, 1e4, None), (15, 1e4, None), (64, 1e4, {"rope_type": "bogus"}),
                                  (64, 1e4, {"rope_type": "linear"}), (2, 1e4, {"rope_type": "dynamic"})])
def test_rotary_frequency_refusals(args):
    with pytest.raises(ValueError):
        F.rotary_inv_freq(*args)


# ------------------------------------------------------------------ schedule
BM, BN, MIN_SHARE, OVERHEAD = 128, 64, 4, 3


def keys_of(pos0, ntok, window, sinks):
    hi = max(0, pos0 + ntok)
    lo = max(0, pos0 - window + 1) if window else 0
    nt, wt0 = -(-hi // BN), lo // BN
    st = min(-(-min(sinks, hi) // BN), wt0)
    return hi, lo, st, wt0, max(1, st + nt - wt0)


@pytest.mark.parametrize("seed", range(40))
def test_shares_cover_every_key_tile_once_and_the_join_finds_its_partials(seed):
    """The line of (q tile, head)s is cut into shares as the kernel cuts it; every key that a row sees lies
    in exactly one visited tile, every slot is written once, and the join of each cut (q tile, head)
    waits for the shares that hold parts of it and reads just the slots they wrote."""
    rng = random.Random(seed)
    G = rng.choice([1, 2, 4, 7, 8, 16, 128])
    Hkv, ctas = rng.choice([1, 2, 8]), rng.choice([1, 3, 8, 296])
    window = rng.choice([0, 0, 1, 50, 700])
    sinks = rng.choice([0, 4, 130]) if window else 0
    tpt = BM // G
    line, at = [], 0  # (begin, x, head, key tiles)
    x = 0
    for _ in range(rng.randrange(1, 12)):
        n = rng.choice([0, 1, 1, rng.randrange(1, 300)])
        kv = rng.choice([0, n, n + rng.randrange(0, 3000), rng.randrange(0, n + 1)])
        for i in range(0, n, tpt):
            t = (kv - n + i, min(tpt, n - i))
            g = keys_of(*t, window, sinks)
            visited = [j if j < g[2] else j - g[2] + g[3] for j in range(g[4])]
            assert len(set(visited)) == len(visited)
            for pos in range(max(0, t[0]), t[0] + t[1]):
                seen = [c for c in range(pos + 1) if not window or c > pos - window or c < sinks]
                assert {c // BN for c in seen} <= set(visited)
                assert all(c < g[0] and (c >= g[1] or c < sinks) for c in seen)
            for h in range(Hkv):
                line.append((at, x, h, g[4]))
                at += g[4] + OVERHEAD
            x += 1
    length = at
    per = max(MIN_SHARE, -(-length // ctas))
    assert per * ctas >= length
    covered, wrote, arrived, whole = set(), {}, {}, set()
    for c in range(ctas):
        u, u1, first = per * c, min(length, per * (c + 1)), True
        while u < u1:
            begin, x, h, n = max(s for s in line if s[0] <= u)
            a, b = u - begin, min(n + OVERHEAD, u1 - begin)
            u = begin + b
            o0, o1 = max(0, a - OVERHEAD), max(0, b - OVERHEAD)
            if o0 == o1:
                continue
            j0, j1 = n - o1, n - o0  # a share that opens a (q tile, head) takes the last keys
            for j in range(j0, j1):
                assert (x, h, j) not in covered
                covered.add((x, h, j))
            if j1 - j0 == n:
                whole.add((x, h))
            else:
                slot = 2 * c + (0 if first else 1)
                assert slot not in wrote
                wrote[slot] = (x, h)
                s0, s1 = (begin + OVERHEAD) // per, (begin + OVERHEAD + n - 1) // per
                arrived.setdefault(s0, []).append((x, h, begin, s1))
            first = False
    assert len(covered) == sum(n for *_, n in line)
    cut = set()
    for s0, parts in arrived.items():
        assert len(set(parts)) == 1  # a counter belongs to one (q tile, head)
        x, h, begin, s1 = parts[0]
        assert len(parts) == s1 - s0 + 1 > 1
        slots = [2 * s + (0 if per * s >= begin else 1) for s in range(s0, s1 + 1)]
        assert slots == sorted(s for s, at in wrote.items() if at == (x, h))
        cut.add((x, h))
    assert whole | cut == {(x, h) for _, x, h, _ in line} and not whole & cut


def test_codes_stored_into_the_host_word_are_raised_once():
    from fftsparse_b200 import status as S
    w = S.StatusWord("cpu")
    for look in (w.poll_direct, w.poll, w.check):
        look()  # zero: nothing to report
        ctypes.c_int32.from_address(w.direct_ptr).value = 11
        with pytest.raises(S.WaitTimeout, match="paged attention") as exc:
            look()
        assert exc.value.code == 11
        look()  # cleared by the raise


@pytest.mark.parametrize("name", ["page_plan", "rope_append", "paged_attn"])
def test_foreign_argument_blocks_are_refused(name):
    """The blocks that the package packs have the header's sizes; another size is refused before anything else."""
    from fftsparse_b200 import _lib, paged
    lib = _lib.load()
    call = getattr(lib, f"ffts_{name}")
    size = {"page_plan": paged._PLAN, "rope_append": paged._ROPE, "paged_attn": paged._ATTN}[name].size
    for wrong in (0, size - 8, size + 8):
        assert call(wrong.to_bytes(8, "little") + bytes(size), None) == _lib.FFTS_E_INVALID
        assert b"foreign" in lib.ffts_last_error_string()
    assert call(None, None) == _lib.FFTS_E_INVALID
    if not torch.cuda.is_available():  # the right size passes on to the look for a device
        assert call(size.to_bytes(8, "little") + bytes(size), None) == _lib.FFTS_E_CUDA


def test_workspace_query_needs_no_gpu():
    from fftsparse_b200 import _lib
    lib = _lib.load()
    small, large = (lib.ffts_paged_workspace_bytes(t, 4, 32, 8, 128) for t in (4, 100000))
    assert 0 < small < large
    assert lib.ffts_paged_workspace_bytes(0, 4, 32, 8, 128) == 0
    assert lib.ffts_paged_workspace_bytes(4, 4, 30, 8, 128) == 0
