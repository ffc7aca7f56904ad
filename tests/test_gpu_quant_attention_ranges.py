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


def one_part(fmt, q, kp, vp, table, page, D, n, scale):
    """What weights rounded once to fp16 would give: the mistake that the test below has to see."""
    KV = kp.shape[1]
    G = q.shape[1] // KV
    at = np.arange(n)
    pg = table[0, at // page]
    k = values(fmt, kp, D)[pg, :, at % page]
    code, d, m = (x[pg, :, at % page].astype(np.float64) for x in decode(fmt, vp, D))
    if fmt == "q4":
        code, m = code - 8, m + 8 * d
    out = np.zeros(q.shape)
    for h in range(q.shape[1]):
        s = scale * (k[:, h // G] @ q[0, h]) / math.log(2)
        dd, mm, c = d[:, h // G], m[:, h // G], code[:, h // G].reshape(n, -1, 32)
        p = 2.0 ** (s - (s + np.log2(dd.max(-1))).max() + 12)
        w = (p[:, None] * dd).astype(np.float16).astype(np.float64)
        out[0, h] = (((w[..., None] * c).sum(0) + (p[:, None] * mm).sum(0)[:, None]) / p.sum()).reshape(D)
    return out.astype(np.float16).astype(np.float64)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 5, 33])
def test_fp16_outputs_take_weights_in_two_parts(tctx, fmt, D, n):
    rng = np.random.default_rng(D + n)
    H = KV = 8
    page = 16
    kp, vp, table, n_pages, most = pools_of(rng, fmt, [n], KV, page, D)
    q = torch.as_tensor(rng.standard_normal((1, H, D))).half().cuda()
    q64 = q.double().cpu().numpy()
    both, _ = score_sizes(fmt, kp, table, page, D, 0, n, q64, 1)
    scale = float(np.float32(0.25 / both.max()))  # scores whose own error is below 2^-20
    got, _ = run_attention(tctx, fmt, "f16", q, kp, vp, table, n_pages, most, page, D, KV, [0, 1], [0], [n], None, scale)
    want, _, mag, _ = attend64(fmt, q64, kp, vp, table, page, D, [0, 1], None, [n], None, scale)
    # weights to 2^-22 in two parts, exponentials and fp32 sums to 2^-18, a score's error twice (it is in the sum, too), one store
    tol = UNIT["f16"] * np.abs(want) + (2.0 ** -18 + 2.0 ** -22 + 2 * 2.0 ** -20) * mag + 2.0 ** -24
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    assert (np.abs(one_part(fmt, q64, kp, vp, table, page, D, n, scale) - want) > tol).any()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_every_call_gives_the_same_bits(tctx, fmt, kind):
    """Sequences cut over many blocks and whole ones: the pieces are joined in the order of their keys."""
    rng = np.random.default_rng(8)
    lens, H, KV, D, page = [9000, 40, 2500], 16, 4, 128, 64
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D)
    q = torch.as_tensor(rng.standard_normal((9, H, D))).to(DT[kind]).cuda()
    args = (tctx, fmt, kind, q, kp, vp, table, n_pages, most, page, D, KV, [0, 1, 4, 9], [0] * 3, lens, None, 0.1)
    want, want_lse = run_attention(*args)
    for _ in range(10):
        got, lse = run_attention(*args)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
