"""Attention over the quantised cache at the ends of its ranges: rows of q with one element far above the others, weights in two
parts for fp16 outputs, every call the same bits.  Tolerances are stated where they are used, from the roundings the operator
makes."""
import math

import numpy as np
import pytest

from test_gpu_paged_ops import DT, UNIT, kept, tctx  # noqa: F401
from test_gpu_quant_ops import attend64, decode, pools_of, run_attention, values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def score_sizes(fmt, kp, table, page, D, s, n, q, G):
    """Of each row of sequence s (all see its n keys), the largest sum over a key of |q| times what a group's codes and scales may
    add up to on the way: codes 0 .. 255 and 128 times the scale, or 0 .. 15 and the minimum; and of those factors alone."""
    at = np.arange(n)
    rows = kp[table[s, at // page], :, at % page]
    _, d, m = decode(fmt, rows, D)
    f = np.repeat((383 * d.astype(np.float64) if fmt == "q8" else 15 * d.astype(np.float64) + np.abs(m.astype(np.float64))), 32, -1)
    H = q.shape[1]
    both = np.array([[np.abs(f[:, h // G] * np.abs(q[r, h])).sum(-1).max() for h in range(H)] for r in range(q.shape[0])])
    alone = np.array([f[:, h // G].sum(-1).max() for h in range(H)])
    return both, alone


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D,H,KV,rows,n", [(64, 4, 1, 1, 40), (128, 8, 2, 1, 70), (128, 16, 1, 1, 33), (64, 8, 1, 3, 90), (128, 4, 1, 8, 64),
                                          (256, 4, 2, 2, 50)])
def test_rows_with_one_element_far_above_the_others(tctx, fmt, kind, D, H, KV, rows, n):
    """The largest element of a row is 2^21 times the others and meets groups of zeros: the scores are the small elements'."""
    rng = np.random.default_rng(D + rows)
    page, G = 32, H // KV
    kp, vp, table, n_pages, most = pools_of(rng, fmt, [n], KV, page, D)
    at, w = (D, 2) if fmt == "q8" else (D // 2, 4)
    out_at = int(rng.integers(0, D))
    kp[..., at + w * (out_at // 32):at + w * (out_at // 32) + w] = 0  # its group: scale (and minimum) zero
    q = rng.standard_normal((rows, H, D)) * 2.0 ** -6
    q[..., out_at] = np.where(rng.random((rows, H)) < 0.8, 2.0 ** 15, 0.0)  # some rows have none
    q = torch.as_tensor(q).to(DT[kind]).cuda()
    bits = np.zeros((rows, 1), bool)  # every row sees the prefix, all n keys
    scale = 64 / math.sqrt(D)
    got, lse = run_attention(tctx, fmt, kind, q, kp, vp, table, n_pages, most, page, D, KV, [0, rows], [n], [n], bits, scale)
    q64 = q.double().cpu().numpy()
    want, want_lse, mag, _ = attend64(fmt, q64, kp, vp, table, page, D, [0, rows], [n], [n], bits, scale)
    both, alone = score_sizes(fmt, kp, table, page, D, 0, n, np.where(np.arange(D) == out_at, 0, q64), G)
    # a score is off by 2^-18 of what its sums pass through (as elsewhere), and by what the elements of q lose: 2^-36 of the row's
    # power of two each, 2^-34 a group's sum, which is less than 2^-35 an element
    ex = np.floor(np.log2(np.abs(q64).max(-1)))
    err = scale * (both * 2.0 ** -18 + alone * 2.0 ** (ex - 35))
    assert err.max() < 0.01
    part = (2.0 ** -11 + 2.0 ** -17 + 2 * err)[..., None]
    g, ll = got.double().cpu().numpy(), lse.double().cpu().numpy()
    assert (np.abs(ll - want_lse) <= 2.0 ** -17 * np.maximum(1, np.abs(want_lse)) + err).all(), np.abs(ll - want_lse).max()
    assert (np.abs(g - want) <= UNIT[kind] * np.abs(want) + part * mag + 1e-6).all()
