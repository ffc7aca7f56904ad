"""Head norms with rotation and their gradient at the ends of their ranges: heads of any size, small eps, handles that scale,
values that are not finite.  Tolerances are stated where they are used, from the roundings each operator makes."""
import math

import numpy as np
import pytest

from test_gpu_paged_ops import DT, KEEP, UNIT, dev, frequencies, kept, ptr, rotate, tctx  # noqa: F401
from test_gpu_quant_ops import normed, pair_sizes

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SIZES = [0.0, 1e-18, 1e-16, 1e-14, 1e-6, 1.0, 1e6, 1e13, 1e15, 1e16, 1e17]


def gradient64(x, w, dy, pos, f, m, rot, half, eps):
    """g, n, s, dx in 64 bits."""
    s = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    g = rotate(dy, pos, f, m, rot, half, sign=-1.0)
    n = x * s
    return g, n, s, s * (w * g - n * (w * g * n).mean(-1, keepdims=True))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [1.2e-38, 1e-30, 1e-6])
@pytest.mark.parametrize("H,KV,D", [(3, 1, 64), (4, 2, 128), (2, 1, 256), (2, 0, 80)])
def test_heads_of_any_size(tctx, kind, layout, eps, H, KV, D):
    """Heads of zeros and of rms 1e-18 to 1e17 side by side: outputs and gradients, each to its own size."""
    import ulb_capi as U
    rng = np.random.default_rng(D + H)
    eps = float(np.float32(eps))
    M = len(SIZES)
    size = np.stack([np.roll(SIZES, h) for h in range(H + KV)], 1)[..., None]
    x = torch.as_tensor(rng.standard_normal((M, H + KV, D)) * size).to(DT[kind]).cuda()
    dy = torch.as_tensor(rng.standard_normal((M, H + KV, D))).to(DT[kind]).cuda()
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    pos = rng.integers(0, 131072, M)
    r = U.Rope(tctx, D, layout=layout)
    f, m = frequencies(D, 10000.0)
    q, k, gq, gk = (t.contiguous() for t in (x[:, :H], x[:, H:], dy[:, :H], dy[:, H:]))
    y, dx = ([torch.empty_like(q), torch.empty_like(k)] for _ in range(2))
    dw = [torch.empty(D, device="cuda") for _ in range(2)]
    p = ptr(dev(pos))
    r.norm_apply(U.dtype_id(kind), ptr(q), ptr(k), M, H, KV, ptr(w[0]), ptr(w[1]), eps, p, ptr(y[0]), ptr(y[1]))
    r.norm_grad(U.dtype_id(kind), ptr(q), ptr(k), ptr(gq), ptr(gk), M, H, KV, ptr(w[0]), ptr(w[1]), eps, p, ptr(dx[0]), ptr(dx[1]), ptr(dw[0]),
                ptr(dw[1]))
    half = layout == "half"
    for i, (a, b) in enumerate(((q, gq), (k, gk))):
        if a.shape[1] == 0:
            continue
        x64, y64, w64 = (t.double().cpu().numpy() for t in (a, b, w[i]))
        g, n, s, want = gradient64(x64, w64, y64, pos, f, m, D, half, eps)
        # a head at a time: the sum of squares to 2^-20, the factor, products and sums to 2^-20, sines to 2^-21 of a pair, one store
        out = rotate(n * w64, pos, f, m, D, half)
        big = np.abs(n * w64).max(-1, keepdims=True) * 1.5
        assert (np.abs(y[i].double().cpu().numpy() - out) <= (UNIT[kind] + 2.0 ** -19) * big).all()
        big = s * (np.abs(w64 * g).max(-1, keepdims=True) * (1 + np.abs(n).max(-1, keepdims=True) ** 2)) * 1.5
        got = dx[i].double().cpu().numpy()
        # float32's smallest steps (2^-149, and 2^-133 of a bf16 store) where a gradient is as small as that
        assert (np.abs(got - want) <= UNIT[kind] * np.abs(want) + 2.0 ** -18 * big + (2.0 ** -133 if kind == "bf16" else 2.0 ** -148)).all()
        terms = (pair_sizes(y64, D, half) * np.abs(n)).sum((0, 1))
        chain = max(1.0, M * a.shape[1] / 64)
        assert (np.abs(dw[i].double().cpu().numpy() - (g * n).sum((0, 1))) <= (2.0 ** -18 + chain * 2.0 ** -24) * terms + 1e-30).all()
    r.close()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KV,D", [(5, 3, 64), (3, 3, 128), (3, 1, 80), (1, 2, 8)])
def test_what_is_not_finite_stays_with_its_kind(tctx, kind, layout, H, KV, D):
    """An infinity in the last q head, or in the first k head: the other kind's rows and weight keep their gradients to the bit,
    although one warp works on both (heads are no whole steps of 4 or 2)."""
    import ulb_capi as U
    rng = np.random.default_rng(D)
    M = 9
    x, dy = (torch.as_tensor(rng.standard_normal((M, H + KV, D))).to(DT[kind]).cuda() for _ in range(2))
    w = dev(rng.uniform(0.5, 1.5, D), torch.float32)
    pos = dev(rng.integers(0, 999, M))
    r = U.Rope(tctx, D, layout=layout)

    def gradients(x, dy):
        q, k, gq, gk = (t.contiguous() for t in (x[:, :H], x[:, H:], dy[:, :H], dy[:, H:]))
        KEEP.extend([q, k, gq, gk])
        out = [torch.empty_like(q), torch.empty_like(k), *(torch.empty(D, device="cuda") for _ in range(2))]
        r.norm_grad(U.dtype_id(kind), ptr(q), ptr(k), ptr(gq), ptr(gk), M, H, KV, ptr(w), ptr(w), 1e-6, ptr(pos), *map(ptr, out))
        return out

    want = gradients(x, dy)
    assert all(torch.isfinite(t).all() for t in want)
    for which in (0, 1):
        for value in (math.inf, math.nan):
            bad = dy.clone()
            bad[4, H - 1 + which, 5] = value
            got = gradients(x, bad)
            assert torch.equal(got[1 - which], want[1 - which]) and torch.equal(got[3 - which], want[3 - which])
            assert not torch.isfinite(got[2 + which]).all()
            head = H - 1 if which == 0 else 0
            assert not torch.isfinite(got[which][4, head]).any()
            got[which][4, head] = want[which][4, head]
            assert torch.equal(got[which], want[which])
    r.close()


HANDLES = [(dict(scaling="yarn", factor=4.0, orig_len=4096), None), (dict(attn_scale=0.3), 0.3),
           (dict(scaling="yarn", factor=40.0, orig_len=2048, attn_scale=2.5), 2.5), (dict(scaling="linear", factor=8.0), None)]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("more,factor", HANDLES)
@pytest.mark.parametrize("M,H,KV,D,rot", [(7, 5, 3, 64, 64), (33, 4, 2, 128, 64), (5, 3, 1, 80, 48), (4, 2, 0, 256, 256)])
def test_handles_that_scale(tctx, kind, layout, more, factor, M, H, KV, D, rot):
    """m multiplies what turns, and nothing past rot_dim, in the outputs, in their gradients and in those of the weights."""
    import ulb_capi as U
    rng = np.random.default_rng(M + rot)
    eps, half = 1e-5, layout == "half"
    f, m = frequencies(rot, 10000.0, scaling=more.get("scaling", "none"), factor=more.get("factor", 1.0), orig=more.get("orig_len", 4096))
    m = m if factor is None else factor

    def turn(x, pos, sign=1.0):
        y = rotate(x, pos, f, m, rot, half, sign)
        y[..., rot:] = x[..., rot:]
        return y

    x, dy = (torch.as_tensor(rng.standard_normal((M, H + KV, D))).to(DT[kind]).cuda() for _ in range(2))
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    pos = rng.integers(0, 131072, M)
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout, **more)
    q, k, gq, gk = (t.contiguous() for t in (x[:, :H], x[:, H:], dy[:, :H], dy[:, H:]))
    y, dx = ([torch.empty_like(q), torch.empty_like(k)] for _ in range(2))
    dw = [torch.empty(D, device="cuda") for _ in range(2)]
    p = ptr(dev(pos))
    r.norm_apply(U.dtype_id(kind), ptr(q), ptr(k), M, H, KV, ptr(w[0]), ptr(w[1]), eps, p, ptr(y[0]), ptr(y[1]))
    r.norm_grad(U.dtype_id(kind), ptr(q), ptr(k), ptr(gq), ptr(gk), M, H, KV, ptr(w[0]), ptr(w[1]), eps, p, ptr(dx[0]), ptr(dx[1]), ptr(dw[0]),
                ptr(dw[1]))
    top = max(m, 1.0)
    for i, (a, b) in enumerate(((q, gq), (k, gk))):
        if a.shape[1] == 0:
            continue
        x64, y64, w64 = (t.double().cpu().numpy() for t in (a, b, w[i]))
        s = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps)
        n, g = x64 * s, turn(y64, pos, -1.0)
        out = turn(n * w64, pos)
        # the roundings of the plain handle, times the factor
        big = np.abs(n * w64).max(-1, keepdims=True) * 1.5 * top
        assert (np.abs(y[i].double().cpu().numpy() - out) <= (UNIT[kind] + 2.0 ** -19) * big).all()
        want = s * (w64 * g - n * (w64 * g * n).mean(-1, keepdims=True))
        size = pair_sizes(y64, rot, half) * top  # what an element of g is made of: its error is below 2^-20 of this
        big = s * ((np.abs(w64) * size).max(-1, keepdims=True) * (1 + np.abs(n).max(-1, keepdims=True) ** 2))
        assert (np.abs(dx[i].double().cpu().numpy() - want) <= UNIT[kind] * np.abs(want) + 2.0 ** -18 * big).all()
        assert (np.abs(dw[i].double().cpu().numpy() - (g * n).sum((0, 1))) <= 2.0 ** -17 * (size * np.abs(n)).sum((0, 1)) + 1e-30).all()
        # differences of the 64-bit function along a random direction: the formula itself
        u, v, h = rng.standard_normal(x64.shape), rng.standard_normal(D), 1e-5
        loss = lambda z: (turn(normed(x64 + z * u, w64 + z * v, eps), pos) * y64).sum()  # noqa: E731
        slope, along = (loss(h) - loss(-h)) / (2 * h), (want * u).sum() + ((g * n).sum((0, 1)) * v).sum()
        assert abs(slope - along) <= 1e-5 * (np.abs(want * u).sum() + np.abs((g * n).sum((0, 1)) * v).sum())
    r.close()
