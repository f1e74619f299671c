"""Values and lengths at which the paged operators can go wrong.

Tolerances as in test_gpu_paged.py, where a test does not derive its own.
"""
import math

import pytest
import torch

import fftsparse_b200 as F
from test_gpu_paged import BF, NAN, Batch

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
