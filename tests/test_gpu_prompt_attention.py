"""Attention of packed prompts on the GPU against a plain computation in 64 bits.  The tolerance is stated where it is
used, from the roundings the operator makes."""
import math

import numpy as np
import pytest

from test_gpu_paged_ops import DT, KEEP, UNIT, dev, kept, ptr, tctx  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def attend64(q, k, v, q_start, k_start, scale, max_q=None, max_k=None):
    """Outputs, logarithms, sums of weighted sizes of v, and the largest sum of a score's sizes; on the GPU in 64 bits."""
    R, H, D = q.shape
    G = H // k.shape[1]
    out, mag = (torch.zeros(R, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
    lse, reach = torch.full((R, H), -math.inf, dtype=torch.float64, device="cuda"), torch.zeros(R, H, dtype=torch.float64, device="cuda")
    for s in range(len(q_start) - 1):
        r0, r1, k0, k1 = q_start[s], q_start[s + 1], k_start[s], k_start[s + 1]
        n, m = r1 - r0, k1 - k0
        if n == 0 or m == 0:
            continue
        hide = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(H):
            kk, vv, qq = k[k0:k1, h // G].double(), v[k0:k1, h // G].double(), q[r0:r1, h].double()
            sc = (scale * (qq @ kk.T)).masked_fill(hide, -math.inf)
            some = ~hide.all(1)
            p = torch.softmax(sc[some], -1)
            rows = torch.arange(r0, r1, device="cuda")[some]
            out[rows, h], mag[rows, h], lse[rows, h] = p @ vv, p @ vv.abs(), torch.logsumexp(sc[some], -1)
            reach[rows, h] = (scale * (qq[some].abs() @ kk.abs().T)).amax(-1)
    return out, lse, mag, reach


def run(tctx, kind, q, k, v, q_start, k_start, scale, max_q=None, max_k=None, **strides):
    import ulb_capi as U
    H, D, KV = q.shape[1], q.shape[2], k.shape[1]
    R = q.shape[0]
    out = torch.full((R + 2, H, D), 5.0, dtype=DT[kind], device="cuda")
    lse = torch.full((R + 2, H), 5.0, device="cuda")
    n = max(b - a for a, b in zip(q_start, q_start[1:])) if max_q is None else max_q
    m = max(b - a for a, b in zip(k_start, k_start[1:])) if max_k is None else max_k
    tctx.prompt_attention(U.dtype_id(kind), H, KV, D, len(q_start) - 1, R, k.shape[0], n, m, scale, ptr(q), ptr(k), ptr(v), ptr(dev(q_start)),
                          ptr(dev(k_start)), ptr(out), ptr(lse), **strides)
    tctx.sync()
    last = q_start[-1]
    assert (out[last:] == 5).all() and (lse[last:] == 5).all()  # rows behind the last sequence
    return out[:R], lse[:R]


def check(kind, got, lse, want, want_lse, mag, reach, last=None):
    # weights are rounded once to the rows' type, exponentials and fp32 sums are good to 2^-18; a score is off by at most
    # 2^-18 of the sum of its products' sizes; the output is rounded once
    part = UNIT[kind] + 2.0 ** -17 + 2 * reach * 2.0 ** -18
    tol = UNIT[kind] * want.abs() + part[..., None] * mag + 1e-6
    g = got.double()[:last]
    assert torch.isfinite(g).all()
    worst = ((g - want[:last]).abs() / tol[:last])
    assert worst.numel() == 0 or worst.max() <= 1, (worst.max(), (worst > 1).nonzero()[:8].tolist())
    empty = (want_lse == -math.inf)[:last]
    ll = lse.double()[:last]
    assert (ll[empty] == -math.inf).all() and (g[empty] == 0).all()
    full = want_lse[:last][~empty]
    assert ((ll[~empty] - full).abs() <= 2.0 ** -17 * full.abs().clamp(min=1) + reach[:last][~empty] * 2.0 ** -18).all()


def starts(sizes):
    return np.concatenate([[0], np.cumsum(sizes)]).tolist()


CASES = [  # rows of each sequence, keys before them, H, KV, D
    ([1], [0], 1, 1, 64), ([500], [0], 32, 4, 64), ([3, 0, 130, 1], [0, 5, 7, 400], 8, 2, 128), ([64, 65, 63], [0, 0, 0], 4, 4, 80),
    ([257, 129, 128], [0, 1, 64], 6, 2, 96), ([300], [1000], 8, 1, 128), ([70, 200], [3, 0], 4, 2, 256), ([1] * 40, [0] * 20 + [333] * 20, 8, 2, 64),
    ([1], [5000], 32, 8, 128), ([2], [9000], 5, 5, 64), ([1500, 700], [0, 0], 16, 4, 128), ([1030], [0], 64, 1, 128), ([513], [3000], 12, 4, 128)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,before,H,KV,D", CASES)
def test_prompt_attention(tctx, kind, rows, before, H, KV, D):
    g = torch.Generator(device="cuda").manual_seed(sum(rows) + D)
    qs, ks = starts(rows), starts([r + b for r, b in zip(rows, before)])
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(DT[kind]) for n, h in ((qs[-1], H), (ks[-1], KV), (ks[-1], KV)))
    q = (q * 1.5).to(DT[kind])
    got, lse = run(tctx, kind, q, k, v, qs, ks, 1 / math.sqrt(D))
    check(kind, got, lse, *attend64(q, k, v, qs, ks, 1 / math.sqrt(D)))


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_rows_that_see_nothing_and_rows_behind_the_last(tctx, D):
    """More rows than keys: the first see nothing; sequences without keys; rows of q behind the last sequence."""
    g = torch.Generator(device="cuda").manual_seed(D)
    qs, ks = [0, 70, 200, 205, 400], [0, 3, 3, 80, 230]
    q = torch.randn(407, 8, D, device="cuda", generator=g).half()
    k, v = (torch.randn(250, 2, D, device="cuda", generator=g).half() for _ in range(2))
    got, lse = run(tctx, "f16", q, k, v, qs, ks, 0.1)
    check("f16", got, lse, *attend64(q, k, v, qs, ks, 0.1), last=400)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_what_is_not_seen_never_touches_a_result(tctx, kind, D):
    g = torch.Generator(device="cuda").manual_seed(D)
    H, KV = 8, 2
    qs, ks = starts([200, 90, 150]), starts([200, 300, 150])
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).to(DT[kind]) for n, h in ((qs[-1], H), (ks[-1] + 70, KV), (ks[-1] + 70, KV)))
    want, want_lse = run(tctx, kind, q, k, v, qs, ks, 0.1)
    v2, k2 = v.clone(), k.clone()
    v2[ks[-1]:], k2[ks[-1]:] = math.nan, math.nan  # behind the last sequence
    got, lse = run(tctx, kind, q, k2, v2, qs, ks, 0.1)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # an infinity in V and a NaN in K of single keys reach the rows from theirs on, of their sequence and kv head
    v2[100, 0, 5], v2[150, 1, 60], k2[ks[1] + 280, 1, 3] = math.inf, math.nan, math.nan
    got, lse = run(tctx, kind, q, k2, v2, qs, ks, 0.1)
    G = H // KV
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[100:200, :G, 5] = True
    bad[150:200, G:, 60] = True
    odd = got[bad]
    assert (torch.isnan(odd) | torch.isinf(odd)).all()
    bad[qs[1] + 70:qs[2], G:] = True
    assert torch.isnan(got[qs[1] + 70:qs[2], G:]).all()
    assert torch.equal(got[~bad], want[~bad])


def test_many_values_that_are_not_finite(tctx):
    """An infinity in every key of the diagonal's tiles, in one column: finite elsewhere, as without them."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n, H, KV, D = 300, 4, 2, 128
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).half() for h in (H, KV, KV))
    want, _ = run(tctx, "f16", q, k, v, [0, n], [0, n], 0.1)
    v[:, :, 77] = math.inf
    got, _ = run(tctx, "f16", q, k, v, [0, n], [0, n], 0.1)
    keep = [i for i in range(D) if i != 77]
    assert torch.equal(got[:, :, keep], want[:, :, keep]) and (got[:, :, 77] == math.inf).all()


@pytest.mark.parametrize("D,H,KV", [(64, 4, 2), (128, 6, 1)])
def test_many_prompts_of_every_length(tctx, D, H, KV):
    """More sequences than the ordering block has warps, many without rows or keys, some long: a list of units and CTAs that
    take several."""
    rng = np.random.default_rng(D)
    n = 700
    rows = [int(x) for x in rng.integers(0, 40, n) * (rng.random(n) < 0.5)]
    rows[333], rows[5] = 1200, 700
    keys = [r + int(x) if rng.random() < 0.9 else int(x) for r, x in zip(rows, rng.integers(0, 30, n))]
    qs, ks = starts(rows), starts(keys)
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v = (torch.randn(m, h, D, device="cuda", generator=g).half() for m, h in ((qs[-1], H), (ks[-1], KV), (ks[-1], KV)))
    got, lse = run(tctx, "f16", q, k, v, qs, ks, 0.1)
    check("f16", got, lse, *attend64(q, k, v, qs, ks, 0.1))


def test_packed_projections_bounds_and_clamps(tctx):
    """q, k and v as slices of one projection's rows; max_q and max_k below the sequences' own."""
    g = torch.Generator(device="cuda").manual_seed(8)
    H, KV, D, n = 12, 4, 64, 333
    qkv = torch.randn(n, (H + 2 * KV) * D + 8, device="cuda", generator=g).bfloat16()
    q, k, v = (t.reshape(n, -1, D) for t in (qkv[:, :H * D], qkv[:, H * D:(H + KV) * D], qkv[:, (H + KV) * D:(H + 2 * KV) * D]))
    qs = [0, 200, 333]
    want, want_lse = run(tctx, "bf16", q.contiguous(), k.contiguous(), v.contiguous(), qs, qs, 0.125)
    row = qkv.shape[1]
    import ulb_capi as U
    out, lse = torch.empty_like(want), torch.empty_like(want_lse)
    tctx.prompt_attention(U.T_BF16, H, KV, D, 2, n, n, 200, 200, 0.125, ptr(qkv), ptr(qkv) + H * D * 2, ptr(qkv) + (H + KV) * D * 2, ptr(dev(qs)),
                          ptr(dev(qs)), ptr(out), ptr(lse), q_row=row, k_row=row, v_row=row)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    # contents out of range: nothing outside is touched, other sequences keep their results
    a, b, c = q.contiguous(), k.contiguous(), v.contiguous()
    got = torch.full_like(want, 5.0)
    tctx.prompt_attention(U.T_BF16, H, KV, D, 3, n, n, 200, 200, 0.125, ptr(a), ptr(b), ptr(c), ptr(dev([0, 200, 100, 1 << 30])),
                          ptr(dev([0, 200, -5, 1 << 30])), ptr(got))
    assert torch.equal(got[:100], want[:100])
    got = torch.full_like(want, 5.0)
    tctx.prompt_attention(U.T_BF16, H, KV, D, 2, n, n, 90, 100, 0.125, ptr(a), ptr(b), ptr(c), ptr(dev(qs)), ptr(dev(qs)), ptr(got))
    ref = attend64(a, b, c, [0, 90], [0, 100], 0.125)
    assert ((got[:90].double() - ref[0][:90]).abs() <= 2.0 ** -6 * ref[2][:90] + 1e-6).all()
    assert (got[90:200] == 5).all()


def test_prompt_attention_captured_on_another_stream(tctx):
    import ulb_capi as U
    g = torch.Generator(device="cuda").manual_seed(2)
    H, KV, D, n = 8, 2, 128, 700
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).half() for h in (H, KV, KV))
    want, _ = run(tctx, "f16", q, k, v, [0, 300, n], [0, 300, n], 0.1)
    at = dev([0, 300, n])
    outs = [torch.zeros_like(want) for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    tctx.use_stream(side.cuda_stream)
    graphs = [tctx.capture(lambda o=o: tctx.prompt_attention(U.T_F16, H, KV, D, 2, n, n, 400, 400, 0.1, ptr(q), ptr(k), ptr(v), ptr(at), ptr(at), ptr(o)))
              for o in outs]
    for x in graphs + graphs:
        U.check(U.lib().ulb_graph_launch(tctx.h, x))
    tctx.sync()
    assert all(torch.equal(o, want) for o in outs)
    for x in graphs:
        U.lib().ulb_graph_free(x)
    tctx.use_stream(torch.cuda.current_stream().cuda_stream)


def test_equals_the_tree_attention_of_the_same_rows(tctx):
    """A prompt over its own pages, causal, by the paged operator: both within their tolerances of the same outputs."""
    import ulb_capi as U
    g = torch.Generator(device="cuda").manual_seed(5)
    H, KV, D, n, page = 8, 2, 128, 256, 64
    q, k, v = (torch.randn(n, h, D, device="cuda", generator=g).half() for h in (H, KV, KV))
    got, lse = run(tctx, "f16", q, k, v, [0, n], [0, n], 0.1)
    kp, vp = (t.reshape(n // page, page, KV, D).transpose(1, 2).contiguous() for t in (k, v))
    c = U.CacheDesc(dtype=U.T_F16, n_layer=1, n_head_kv=KV, head_dim=D, page=page, n_pages=4, n_seq=1, max_pages=4)
    out, l2 = torch.empty_like(got), torch.empty_like(lse)
    tctx.tree_attention(c, H, n, n, n, 0.1, ptr(q), ptr(kp), ptr(vp), ptr(dev([[0, 1, 2, 3]])), ptr(dev([0, n])), ptr(dev([0])), ptr(dev([n])), None, 0,
                        ptr(out), ptr(l2))
    _, _, mag, _ = attend64(q, k, v, [0, n], [0, n], 0.1)
    assert ((out.double() - got.double()).abs() <= 2.0 ** -8 * mag + 1e-6).all() and (l2 - lse).abs().max() < 1e-4
