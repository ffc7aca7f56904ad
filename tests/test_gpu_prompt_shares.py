"""Packed prompts whose keys are cut into shares: several sequences in a call, sequences too short for a share each, values that
are not finite at the ends of shares.  The number of shares follows from the call's sizes; each case says what it is meant to
reach on a GPU of 148 SMs."""
import math

import pytest

from test_gpu_paged_ops import DT, kept, tctx  # noqa: F401
from test_gpu_prompt_attention import attend64, check, run, starts

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CASES = [  # rows of each sequence, keys before them, H, KV, D
    ([513, 513], [3500, 3100], 20, 5, 128),                            # three shares, 270 units: a list
    ([513], [3500], 40, 10, 64),                                       # three shares of one sequence, 270 units
    ([200, 1, 0, 33, 5], [6000, 300, 50, 0, 2000], 8, 2, 64),          # three shares of one unit each; sequences of one tile
    ([300, 300, 7, 7, 7, 7], [5000, 5000, 0, 0, 0, 0], 10, 5, 96),     # three, a list, most entries with one tile
    ([1, 1, 1, 1, 1, 2], [9000, 20, 4000, 0, 100, 7000], 40, 10, 128), # seven, a list, 128 queries a unit
    ([70, 300, 3], [0, 4000, 9000], 15, 5, 80),                        # seven, a list
    ([130, 1, 64], [2900, 6000, 10], 10, 5, 64),                       # four, without a list
    ([90, 20, 90], [3900, 0, 4000], 64, 8, 128)]                       # two, without a list


def case(rows, before, H, KV, D, kind):
    g = torch.Generator(device="cuda").manual_seed(sum(rows) + D)
    qs, ks = starts(rows), starts([r + b for r, b in zip(rows, before)])
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(DT[kind]) for n, h in ((qs[-1], H), (ks[-1], KV), (ks[-1], KV)))
    return qs, ks, (q * 1.5).to(DT[kind]), k, v


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,before,H,KV,D", CASES)
def test_shares_of_several_sequences(tctx, kind, rows, before, H, KV, D):
    qs, ks, q, k, v = case(rows, before, H, KV, D, kind)
    got, lse = run(tctx, kind, q, k, v, qs, ks, 1 / math.sqrt(D))
    check(kind, got, lse, *attend64(q, k, v, qs, ks, 1 / math.sqrt(D)))
    for _ in range(3):  # whichever CTA takes which unit: the same bits
        again, l2 = run(tctx, kind, q, k, v, qs, ks, 1 / math.sqrt(D))
        assert torch.equal(again, got) and torch.equal(l2, lse)


@pytest.mark.parametrize("D,H,KV", [(64, 10, 5), (80, 8, 2), (128, 20, 5)])
def test_rows_that_see_nothing_beside_shares(tctx, D, H, KV):
    """More rows than keys, no keys at all, and a long sequence in one call."""
    g = torch.Generator(device="cuda").manual_seed(D)
    qs, ks = starts([300, 40, 90, 5]), starts([3, 5000, 0, 70])
    q = torch.randn(qs[-1] + 2, H, D, device="cuda", generator=g).half()
    k, v = (torch.randn(ks[-1], KV, D, device="cuda", generator=g).half() for _ in range(2))
    got, lse = run(tctx, "f16", q, k, v, qs, ks, 0.1)
    check("f16", got, lse, *attend64(q, k, v, qs, ks, 0.1), last=qs[-1])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,before,H,KV,D", [CASES[0], CASES[3], CASES[4], CASES[6]])
def test_what_is_not_seen_stays_out_of_every_share(tctx, kind, rows, before, H, KV, D):
    """NaN behind the last key, and an infinity and a NaN of V on the diagonal of the longest sequence: they reach the rows from
    theirs on, whichever share holds them."""
    qs, ks, q, k, v = case(rows, before, H, KV, D, kind)
    k, v = (torch.cat([t, torch.zeros(70, KV, D, dtype=t.dtype, device="cuda")]) for t in (k, v))
    want, want_lse = run(tctx, kind, q, k, v, qs, ks, 0.1)
    k2, v2 = k.clone(), v.clone()
    k2[ks[-1]:], v2[ks[-1]:] = math.nan, math.nan
    got, lse = run(tctx, kind, q, k2, v2, qs, ks, 0.1)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    s = max(range(len(rows)), key=lambda i: rows[i] + before[i])
    G, n = H // KV, rows[s]
    first = n // 2  # row of the sequence that is the first to see the key
    key = ks[s] + before[s] + first
    v2[key, 0, 5], v2[key, 1, 60] = math.inf, math.nan
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[qs[s] + first:qs[s + 1], :G, 5] = True
    bad[qs[s] + first:qs[s + 1], G:2 * G, 60] = True
    got, lse = run(tctx, kind, q, k2, v2, qs, ks, 0.1)
    assert not torch.isfinite(got[bad]).any()
    assert torch.equal(got[~bad], want[~bad]) and torch.equal(lse, want_lse)
