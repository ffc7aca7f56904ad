"""Paged cache operators on the GPU against plain computations in 64 bits: rotary positions,
attention of drafted trees over pages, page moves and the page book, logits under penalties and
grammars.  Tolerances are stated where they are used, from the roundings each operator makes."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # relative rounding of one store


@pytest.fixture(scope="module")
def tctx():
    import ulb_capi as U
    c = U.Context(0)
    c.use_stream(torch.cuda.current_stream().cuda_stream)
    yield c
    c.sync()
    c.close()


KEEP = []  # device arrays of the running test: calls take bare addresses


@pytest.fixture(autouse=True)
def kept():
    yield
    torch.cuda.synchronize()
    KEEP.clear()


def dev(x, dtype=torch.int32):
    KEEP.append(torch.as_tensor(np.asarray(x), dtype=dtype).cuda())
    return KEEP[-1]


def ptr(t):
    return None if t is None else t.data_ptr()


def refused(fn, *a, code=None, **k):
    import ulb_capi as U
    with pytest.raises(U.UlbError) as e:
        fn(*a, **k)
    assert e.value.code in ((U.EINVAL, U.EUNSUPPORTED) if code is None else (code,)), e.value


# ---------------------------------------------------------------------------------------------- rotary
def frequencies(rot, base, scaling="none", factor=1.0, orig=4096, fast=32.0, slow=1.0, low=1.0, high=4.0, ff=None):
    w, m = [], 1.0
    for i in range(rot // 2):
        b = base * factor ** (rot / (rot - 2)) if scaling == "ntk" else base
        f = b ** (-2.0 * i / rot)
        if ff is not None:
            f /= float(ff[i])
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            e = lambda n: rot * math.log(orig / (2 * math.pi * n)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(math.floor(e(fast)), 0), min(math.ceil(e(slow)), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f * (1 - r) + f / factor * r
            m = 0.1 * math.log(factor) + 1
        elif scaling == "wavelength":
            wave = 2 * math.pi / f
            if wave > orig / low:
                f /= factor
            elif wave >= orig / high:
                x = (orig / wave - low) / (high - low)
                f = (1 - x) * f / factor + x * f
        w.append(f)
    return np.array(w), m


def rotate(x, pos, w, m, rot, half, sign=1.0):
    """x [M][H][D] as float64."""
    a = np.asarray(pos, np.float64)[:, None] * w[None]
    c, s = (m * np.cos(a))[:, None], (m * sign * np.sin(a))[:, None]
    y = x.copy()
    i0, i1 = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def rope_tol(kind, x, m):
    # two products and a sum of the pair in fp32, sines to 2^-22 (angle rounded to 2^-25 of pi), one store
    big = np.abs(x).max() * max(m, 1.0) * 1.5
    return UNIT[kind] * big + 2.0 ** -21 * big


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,H,D,rot", [(1, 1, 64, 64), (3, 5, 80, 40), (7, 32, 128, 128), (300, 9, 96, 96),
                                       (2, 3, 256, 64), (5, 2, 10, 6), (4, 3, 66, 2), (4097, 40, 128, 64)])
def test_rope_matches_formula(tctx, kind, layout, M, H, D, rot):
    import ulb_capi as U
    rng = np.random.default_rng(M * D + rot)
    x = torch.as_tensor(rng.standard_normal((M, H, D))).to(DT[kind]).cuda()
    pos = rng.integers(0, 131072, M)
    pos[0] = 0
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout, base=10000.0)
    out = torch.empty_like(x)
    r.apply(U.dtype_id(kind), ptr(x), M, H, ptr(dev(pos)), ptr(out))
    w, m = frequencies(rot, 10000.0)
    x64 = x.double().cpu().numpy()
    want = rotate(x64, pos, w, m, rot, layout == "half")
    assert np.abs(out.double().cpu().numpy() - want).max() <= rope_tol(kind, x64, m)
    # in place gives the same bits
    r.apply(U.dtype_id(kind), ptr(x), M, H, ptr(dev(pos)), ptr(x))
    assert torch.equal(x, out)
    r.close()


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0), ("yarn", 1.0), ("wavelength", 8.0)])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_rope_scalings_far_and_negative_positions(tctx, scaling, factor, base):
    import ulb_capi as U
    rng = np.random.default_rng(3)
    D, H = 128, 4
    pos = np.array([0, 1, -1, 4095, 4096, 131071, 1 << 20, (1 << 31) - 1, -(1 << 31)])
    x = torch.as_tensor(rng.standard_normal((len(pos), H, D)), dtype=torch.float32).cuda()
    ff = rng.uniform(1, 8, D // 2).astype(np.float32)
    for f in (None, ff):
        r = U.Rope(tctx, D, base=base, scaling=scaling, factor=factor, orig_len=4096, freq_factors=f)
        out = torch.empty_like(x)
        r.apply(U.T_F32, ptr(x), len(pos), H, ptr(dev(pos)), ptr(out))
        w, m = frequencies(D, base, scaling, factor, ff=f)
        x64 = x.double().cpu().numpy()
        want = rotate(x64, pos, w, m, D, False)
        # the reference's own angle: a frequency good to 2^-52 times 2^31 positions is good to 2^-21
        assert np.abs(out.double().cpu().numpy() - want).max() <= rope_tol("f32", x64, m) + 2.0 ** -20 * np.abs(x64).max()
        r.close()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_gradient(tctx, layout):
    """The inverse call is the transpose of the forward one: <R x, g> = <x, R^T g>, and its values are
    the differences of <R x, g> in x (the map is linear, so a difference quotient is exact but for
    rounding)."""
    import ulb_capi as U
    rng = np.random.default_rng(5)
    M, H, D, rot = 6, 3, 96, 64
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout, base=1e4, scaling="yarn", factor=4.0, orig_len=2048)
    pos = dev(rng.integers(0, 9000, M))
    x, g = (torch.as_tensor(rng.standard_normal((M, H, D)), dtype=torch.float32).cuda() for _ in range(2))
    fwd = lambda v: (lambda o: (r.apply(U.T_F32, ptr(v), M, H, ptr(pos), ptr(o)), o)[1])(torch.empty_like(v))  # noqa: E731
    gx = torch.empty_like(g)
    r.apply(U.T_F32, ptr(g), M, H, ptr(pos), ptr(gx), inverse=True)
    w, m = frequencies(rot, 1e4, "yarn", 4.0, orig=2048)
    want = rotate(g.double().cpu().numpy(), pos.cpu().numpy(), w, m, rot, layout == "half", -1.0)
    assert np.abs(gx.double().cpu().numpy() - want).max() <= rope_tol("f32", want, m)
    for _ in range(12):
        i = tuple(int(rng.integers(0, n)) for n in (M, H, D))
        a, b = x.clone(), x.clone()
        a[i] += 0.5
        b[i] -= 0.5
        quotient = ((fwd(a).double() - fwd(b).double()) * g.double()).sum().item()
        assert abs(quotient - gx[i].item()) <= 64 * 2.0 ** -22 * 8
    r.close()


def test_rope_strides_and_unaligned_rows(tctx):
    """Heads and rows apart, and a first element on an odd address, take the narrow path."""
    import ulb_capi as U
    rng = np.random.default_rng(6)
    M, H, D = 5, 3, 64
    r = U.Rope(tctx, D)
    w, m = frequencies(D, 1e4)
    pos = dev(rng.integers(0, 5000, M))
    for off, row, head in ((1, 1000, 67), (8, 800, 72), (4, 404, 68)):
        buf = torch.as_tensor(rng.standard_normal(off + M * row), dtype=torch.float16).cuda()
        out = torch.full((off + M * row,), 7.0, dtype=torch.float16, device="cuda")
        view = lambda t: torch.as_strided(t, (M, H, D), (row, head, 1), off)  # noqa: E731
        r.apply(U.T_F16, buf.data_ptr() + 2 * off, M, H, ptr(pos), out.data_ptr() + 2 * off, row, head, row, head)
        x = view(buf).double().cpu().numpy()
        want = rotate(x, pos.cpu().numpy(), w, m, D, False)
        assert np.abs(view(out).double().cpu().numpy() - want).max() <= rope_tol("f16", x, m)
        rest = out.clone()
        view(rest).fill_(7.0)
        assert bool((rest == 7.0).all())  # nothing between the heads is written
    r.close()


@pytest.mark.parametrize("kin,kout", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16")])
@pytest.mark.parametrize("H,Hkv,D,page,nhd", [(4, 4, 64, 16, False), (8, 2, 128, 256, False), (6, 3, 80, 32, True), (5, 1, 96, 64, True)])
def test_rope_append(tctx, kin, kout, H, Hkv, D, page, nhd):
    import ulb_capi as U
    rng = np.random.default_rng(D + page)
    S, most, n_pages, M = 3, 3, 11, 37
    table = np.full((S, most), -1)
    ids = rng.permutation(n_pages)
    table[0, :3], table[1, :2], table[2, 0] = ids[:3], ids[3:5], ids[5]
    table[2, 1] = n_pages + 4  # outside the pool: unmapped
    qkv = torch.as_tensor(rng.standard_normal((M, (H + 2 * Hkv) * D)), dtype=DT[kin]).cuda()
    seq = rng.integers(0, S, M)
    seq[3], seq[4] = -1, S  # no such sequence
    slot = rng.permutation(3 * page + 5)[:M] if 3 * page + 5 >= M else np.arange(M)
    slot[5] = -2
    pos = rng.integers(0, 60000, M)
    shape = (n_pages, page, Hkv, D) if nhd else (n_pages, Hkv, page, D)
    k, v = (torch.full(shape, 3.0, dtype=DT[kout], device="cuda") for _ in range(2))
    cache = U.CacheDesc(dtype=U.dtype_id(kout), n_head_kv=Hkv, head_dim=D, page=page, n_pages=n_pages, n_seq=S, max_pages=most,
                        head_stride=D if nhd else 0, pos_stride=Hkv * D if nhd else 0, page_stride=page * Hkv * D if nhd else 0)
    qo = torch.zeros(M, H, D, dtype=DT[kout], device="cuda")
    r = U.Rope(tctx, D, layout="half")
    es, base, row = qkv.element_size(), qkv.data_ptr(), (H + 2 * Hkv) * D
    r.append(cache, U.dtype_id(kin), base, base + H * D * es, base + (H + Hkv) * D * es, H, ptr(dev(pos)), ptr(dev(seq)),
             ptr(dev(slot)), ptr(dev(table)), M, ptr(qo), ptr(k), ptr(v), row, row, row)
    x = qkv.double().cpu().numpy().reshape(M, H + 2 * Hkv, D)
    w, m = frequencies(D, 1e4)
    y = rotate(x, pos, w, m, D, True)
    tol = rope_tol(kout, x, m)
    assert np.abs(qo.double().cpu().numpy() - y[:, :H]).max() <= tol
    wk, wv = np.full(shape, 3.0), np.full(shape, 3.0)
    for i in range(M):
        if not (0 <= seq[i] < S and 0 <= slot[i] < most * page):
            continue
        p, o = table[seq[i], slot[i] // page], slot[i] % page
        if 0 <= p < n_pages:
            at = (p, o) if nhd else (p, slice(None), o)
            wk[at], wv[at] = y[i, H:H + Hkv], x[i, H + Hkv:]
    assert np.abs(k.double().cpu().numpy() - wk).max() <= tol
    assert np.abs(v.double().cpu().numpy() - wv).max() <= UNIT[kout] * np.abs(x).max()
    r.close()


def test_rope_arrays_at_odd_addresses(tctx):
    import ulb_capi as U
    r = U.Rope(tctx, 64)
    x = torch.zeros(4096, device="cuda")
    p = dev([0] * 8)
    c = U.CacheDesc(dtype=U.T_F16, n_head_kv=1, head_dim=64, page=16, n_pages=1, n_seq=1, max_pages=1)
    refused(r.apply, U.T_F32, ptr(x), 4, 1, ptr(p) + 2, ptr(x), code=U.EINVAL)
    for i in range(4):
        a = [ptr(p) + (2 if j == i else 0) for j in range(4)]
        refused(r.append, c, U.T_F32, ptr(x), ptr(x), ptr(x), 1, *a, 4, ptr(x), ptr(x), ptr(x), code=U.EINVAL)
    r.close()


def test_rope_refusals(tctx):
    import ulb_capi as U
    for kw in (dict(head_dim=64, rot_dim=63), dict(head_dim=64, rot_dim=66), dict(head_dim=0), dict(head_dim=64, base=1.0),
               dict(head_dim=64, base=float("nan")), dict(head_dim=64, scaling="linear", factor=0.0),
               dict(head_dim=64, scaling="yarn", factor=2.0, orig_len=0),
               dict(head_dim=64, scaling="wavelength", factor=2.0, orig_len=100, low_freq=4.0, high_freq=4.0),
               dict(head_dim=64, rot_dim=2, scaling="ntk", factor=2.0), dict(head_dim=64, freq_factors=[0.0] * 32),
               dict(head_dim=64, attn_scale=-1.0)):
        refused(U.Rope, tctx, **kw)
    r = U.Rope(tctx, 64)
    x = torch.zeros(4, 64, device="cuda")
    p = dev([0] * 4)
    refused(r.apply, U.T_Q4_0, ptr(x), 4, 1, ptr(p), ptr(x))
    refused(r.apply, U.T_F32, ptr(x), -1, 1, ptr(p), ptr(x))
    refused(r.apply, U.T_F32, ptr(x), 4, 0, ptr(p), ptr(x))
    refused(r.apply, U.T_F32, None, 4, 1, ptr(p), ptr(x))
    refused(r.apply, U.T_F32, ptr(x) + 2, 4, 1, ptr(p), ptr(x))
    refused(r.apply, U.T_F32, ptr(x), 2, 1, ptr(p), ptr(x), out_row=128)
    r.apply(U.T_F32, None, 0, 1, None, None)  # no rows: nothing to do
    c = U.CacheDesc(dtype=U.T_F16, n_head_kv=1, head_dim=128, page=16, n_pages=1, n_seq=1, max_pages=1)
    refused(r.append, c, U.T_F32, ptr(x), ptr(x), ptr(x), 1, ptr(p), ptr(p), ptr(p), ptr(p), 4, ptr(x), ptr(x), ptr(x))
    for bad in (dict(dtype=U.T_F32), dict(page=48), dict(head_dim=60), dict(n_pages=0), dict(pos_stride=65), dict(pos_stride=56)):
        c = U.CacheDesc(**{**dict(dtype=U.T_F16, n_head_kv=1, head_dim=64, page=16, n_pages=1, n_seq=1, max_pages=1), **bad})
        refused(r.append, c, U.T_F32, ptr(x), ptr(x), ptr(x), 1, ptr(p), ptr(p), ptr(p), ptr(p), 4, ptr(x), ptr(x), ptr(x))
    r.close()


# ---------------------------------------------------------------------------------------------- attention
def pack_bits(bits, words):
    rows, n = bits.shape
    wide = np.zeros((rows, words * 32), np.uint64)
    wide[:, :min(n, words * 32)] = bits[:, :words * 32]
    return (wide.reshape(rows, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


class Attention:
    """A random call and its 64-bit answer."""

    def __init__(self, kind, H, Hkv, D, page, seqs, seed=0, nhd=False, causal=False, unmapped=(), empty_rows=False,
                 stale=None, sharp=1.0, spare_pages=2, slots=None):
        """seqs: (prefix, rows) of each sequence; slots: cached tree slots when not one a row;
        stale: value in every cache place that no row may see."""
        rng = np.random.default_rng(seed)
        self.kind, self.H, self.Hkv, self.D, self.page, self.causal = kind, H, Hkv, D, page, causal
        self.prefix = [p for p, _ in seqs]
        self.n = [r for _, r in seqs]
        self.slots = list(self.n) if slots is None else list(slots)
        self.len = [p + s for p, s in zip(self.prefix, self.slots)]
        self.start = np.concatenate([[0], np.cumsum(self.n)])
        self.rows = int(self.start[-1])
        need = [(x + page - 1) // page for x in self.len]
        self.most = max(need + [1])
        self.n_pages = sum(need) + spare_pages
        ids = rng.permutation(self.n_pages)
        self.table = np.full((len(seqs), self.most), -1)
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = ids[at:at + m]
            at += m
        for s, j, value in unmapped:
            self.table[s, j] = value if value < 0 else self.n_pages + value
        W = self.words = max(1, (max(self.slots + [1]) + 31) // 32)
        self.see = []
        for s in range(len(seqs)):
            b = rng.random((self.n[s], self.slots[s])) < 0.5
            if not empty_rows:
                for i in range(self.n[s]):
                    if self.slots[s]:
                        b[i, min(i, self.slots[s] - 1)] = True
            else:
                b[::2] = False
            self.see.append(b)
        f = lambda *sh: torch.as_tensor(rng.standard_normal(sh)).to(DT[kind]).cuda()  # noqa: E731
        shape = (self.n_pages, page, Hkv, D) if nhd else (self.n_pages, Hkv, page, D)
        self.nhd = nhd
        self.q, self.k, self.v = f(max(self.rows, 1), H, D) * sharp, f(*shape), f(*shape)
        if stale is not None:
            seen = np.zeros((self.n_pages, page), bool)
            for s in range(len(seqs)):
                for t in range(self.len[s]):
                    p = self.table[s, t // page]
                    if 0 <= p < self.n_pages and self.n[s] and any(self.visible(s, i)[t] for i in range(self.n[s])):
                        seen[p, t % page] = True
            hide = torch.as_tensor(~seen).cuda()
            hide = hide[:, :, None, None] if nhd else hide[:, None, :, None]
            self.k.masked_fill_(hide, stale)
            self.v.masked_fill_(hide, stale)
        self.mask = None if causal else torch.as_tensor(
            np.concatenate([pack_bits(b, W) for b in self.see] + [np.zeros((0, W), np.int32)])).cuda()

    def visible(self, s, i):
        n, page = self.len[s], self.page
        t = np.arange(n)
        mapped = np.array([0 <= self.table[s, x // page] < self.n_pages for x in t], bool)
        if self.causal:
            return mapped & (t <= n - self.n[s] + i)
        out = np.ones(n, bool)
        out[self.prefix[s]:] = self.see[s][i]
        return mapped & out

    def run(self, ctx, lse=True):
        import ulb_capi as U
        H, Hkv, D, page = self.H, self.Hkv, self.D, self.page
        c = U.CacheDesc(dtype=U.dtype_id(self.kind), n_head_kv=Hkv, head_dim=D, page=page, n_pages=self.n_pages,
                        n_seq=len(self.n), max_pages=self.most)
        if self.nhd:
            c.head_stride, c.pos_stride, c.page_stride = D, Hkv * D, page * Hkv * D
        out = torch.full((max(self.rows, 1), H, D), 9.0, dtype=DT[self.kind], device="cuda")
        ls = torch.full((max(self.rows, 1), H), 9.0, device="cuda") if lse else None
        self.keep = [dev(self.table), dev(self.start), dev(self.prefix), dev(self.len)]
        self.again = lambda: ctx.tree_attention(  # the bare call, which allocates nothing
            c, H, self.rows, max(self.n + [0]), max(self.len + [0]), 1 / math.sqrt(D), ptr(self.q), ptr(self.k), ptr(self.v),
            *[ptr(t) for t in self.keep], ptr(self.mask), 0 if self.causal else self.words, ptr(out), ptr(ls))
        torch.cuda.current_stream().synchronize()
        self.again()
        return out, ls

    def check(self, ctx):
        out, ls = self.run(ctx)
        out, ls = out.double().cpu().numpy(), ls.double().cpu().numpy()
        q, k, v = (x.double().cpu() for x in (self.q, self.k, self.v))
        u, G = UNIT[self.kind], self.H // self.Hkv
        for s in range(len(self.n)):
            if not self.n[s]:
                continue
            pages = torch.as_tensor(np.clip(self.table[s, :(self.len[s] + self.page - 1) // self.page], 0, self.n_pages - 1))
            see = torch.as_tensor(np.stack([self.visible(s, i) for i in range(self.n[s])]))
            for h in range(self.H):
                kk, vv = (x[pages, :, h // G] if self.nhd else x[pages, h // G] for x in (k, v))
                kk, vv = (x.reshape(-1, self.D)[:self.len[s]] for x in (kk, vv))
                rows = slice(int(self.start[s]), int(self.start[s + 1]))
                kz, vz = (torch.where(see.any(0)[:, None], x, torch.zeros_like(x)) for x in (kk, vv))
                sc = torch.where(see, q[rows, h] @ kz.T / math.sqrt(self.D), torch.tensor(-math.inf, dtype=torch.float64))
                none = ~see.any(1)
                l = torch.logsumexp(sc, 1) if sc.shape[1] else torch.full((self.n[s],), -math.inf, dtype=torch.float64)
                p = torch.exp(sc - torch.where(none, torch.zeros_like(l), l)[:, None])
                want, size = p @ vz, p @ vz.abs()
                got = torch.as_tensor(out[rows, h])
                # weights and the output each rounded once; scores to fp32 (hd products, |s| <= 2^6:
                # 2^-24 * 2^6 * a few); f16 weights below 2^-14 keep 2^-25 (times the tallest v)
                tol = (u + 2.0 ** -15) * size + u * want.abs() + 1e-6
                if self.kind == "f16":
                    top = torch.exp(sc.max(1).values - l).nan_to_num(0.0) if sc.shape[1] else l * 0
                    tol = tol + (2.0 ** -25 * see.sum(1) * top * float(vz.abs().max()) if sc.shape[1] else 0 * l)[:, None]
                assert bool(((got - want).abs() <= tol).all()), (s, h, float(((got - want).abs() - tol).max()))
                gl = torch.as_tensor(ls[rows, h])
                assert bool((gl[none] == -math.inf).all()) and bool((got[none] == 0).all())
                assert bool(((gl - l)[~none].abs() <= 2e-5 * (1 + l[~none].abs())).all())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 80, 96, 128, 256])
@pytest.mark.parametrize("H,Hkv,rows", [(4, 4, 1), (8, 2, 3), (8, 1, 4), (6, 2, 21), (4, 1, 70), (16, 1, 40)])
def test_tree_attention_shapes(tctx, kind, D, H, Hkv, rows):
    Attention(kind, H, Hkv, D, 64, [(300, rows), (17, max(1, rows // 2)), (0, rows)], seed=D + rows).check(tctx)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
def test_tree_attention_lengths(tctx, page, prefix):
    """Around every tile, split and page edge; a single row and a tree."""
    Attention("f16", 4, 2, 64, page, [(prefix, 1)], seed=prefix).check(tctx)
    Attention("bf16", 4, 1, 128, page, [(prefix, 33), (max(0, prefix - 3), 2)], seed=prefix + 1, nhd=True).check(tctx)


@pytest.mark.parametrize("H,Hkv,rows", [(4, 4, 1), (8, 1, 9), (8, 1, 40)])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_long_split(tctx, D, H, Hkv, rows):
    """Thousands of positions over many splits, with sequences far shorter than the longest."""
    Attention("f16", H, Hkv, D, 256, [(9001, rows)], seed=1).check(tctx)
    Attention("bf16", H, Hkv, D, 16, [(8191, rows), (0, 1), (130, rows), (5000, max(1, rows // 2))], seed=2).check(tctx)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 64), (8, 1, 128)])
def test_tree_attention_causal(tctx, kind, H, Hkv, D):
    """No masks: chains, prompt chunks longer than any mask, and a chunk that begins its sequence."""
    Attention(kind, H, Hkv, D, 32, [(100, 7), (0, 150), (900, 260), (3, 1)], causal=True, seed=4).check(tctx)


@pytest.mark.parametrize("stale", [math.nan, math.inf, -math.inf, None])
@pytest.mark.parametrize("D,H,rows", [(64, 2, 3), (128, 2, 5), (128, 4, 70), (64, 8, 40)])
def test_tree_attention_rows_that_see_nothing_and_stale_places(tctx, stale, D, H, rows):
    """Empty rows give zeros and -inf, and what no row sees (stale slots, unmapped pages' places,
    positions past the end) may hold anything."""
    for kind in ("f16", "bf16"):
        Attention(kind, H, 1, D, 16, [(0, rows), (40, rows), (0, 1)], empty_rows=True, stale=stale, seed=6).check(tctx)


@pytest.mark.parametrize("D,H,rows", [(64, 2, 3), (128, 1, 40), (128, 4, 40), (128, 8, 10), (64, 16, 12), (96, 4, 40)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_tree_attention_value_that_some_rows_see(tctx, D, H, rows, value):
    """An infinite or NaN V in a slot reaches the rows that see the slot and no other."""
    a = Attention("f16", H, 1, D, 64, [(70, rows)], seed=8)
    slot, d = rows // 2, 5
    a.see[0][:, slot] = np.arange(rows) % 3 == 0
    a.mask = torch.as_tensor(pack_bits(a.see[0], a.words)).cuda()
    clean, _ = a.run(tctx)
    t = 70 + slot
    a.v[int(a.table[0, t // 64]), 0, t % 64, d] = value
    out, _ = a.run(tctx)
    hit = torch.as_tensor(np.arange(rows) % 3 == 0).cuda()
    assert bool((out[hit][:, :, d].float() == value).all()) if value == math.inf else bool(out[hit][:, :, d].isnan().all())
    out[:, :, d] = clean[:, :, d].where(hit[:, None], out[:, :, d])
    # the other rows and columns: the element left out of the product changes no other bit
    assert torch.equal(out, clean) or bool(((out - clean).abs() <= 2e-3).all())
    assert bool(out.isfinite().all())


def test_tree_attention_unmapped_pages(tctx):
    Attention("f16", 4, 2, 64, 16, [(100, 4), (333, 9)], unmapped=[(0, 2, -1), (1, 0, -7), (1, 5, 3), (1, 21, -1)], seed=9).check(tctx)
    Attention("bf16", 8, 1, 128, 64, [(1000, 17)], unmapped=[(0, 3, 0), (0, 15, -1)], seed=10).check(tctx)
    Attention("bf16", 2, 1, 128, 64, [(64, 2)], unmapped=[(0, 0, -1), (0, 1, -1)], seed=10).check(tctx)  # no keys at all


def test_tree_attention_more_slots_than_rows(tctx):
    """A draft step's newest level: few rows over the slots of the whole tree."""
    Attention("f16", 8, 2, 64, 32, [(50, 3), (7, 4), (90, 0)], slots=[40, 4, 64], seed=11).check(tctx)
    Attention("f16", 8, 1, 128, 32, [(50, 30), (7, 4), (90, 0)], slots=[140, 4, 64], seed=11).check(tctx)


@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_large_scores(tctx, D):
    """Scores of hundreds: the running maximum moves between tiles, weights underflow."""
    a = Attention("f16", 4, 1, D, 64, [(700, 5), (200, 40)], seed=12, sharp=40.0)
    out, ls = a.run(tctx)
    assert bool(out.isfinite().all()) and bool(ls.isfinite().all())
    q, k, v = (x.double().cpu() for x in (a.q, a.k, a.v))
    for s, h in ((0, 0), (1, 3)):
        pages = torch.as_tensor(a.table[s, :(a.len[s] + 63) // 64])
        kk, vv = (x[pages, 0].reshape(-1, D)[:a.len[s]] for x in (k, v))
        see = torch.as_tensor(np.stack([a.visible(s, i) for i in range(a.n[s])]))
        sc = (q[int(a.start[s]):int(a.start[s + 1]), h] @ kk.T / math.sqrt(D)).masked_fill(~see, -math.inf)
        want = torch.softmax(sc, 1) @ vv
        # a score of 2^9 rounded to fp32 moves a weight by 2^9 2^-24 a few times over; products of hd terms
        err = (out[int(a.start[s]):int(a.start[s + 1]), h].double().cpu() - want).abs().max()
        assert err <= 4 * UNIT["f16"] * float(vv.abs().max())


def test_tree_attention_past_32_bit_offsets(tctx):
    """Pages more than 2^31 elements into the pools."""
    import ulb_capi as U
    D, page, Hkv, H = 128, 256, 8, 8
    per = Hkv * page * D
    n_pages = (1 << 31) // per + 8
    k = torch.zeros(n_pages * per, dtype=torch.float16, device="cuda")
    v = torch.zeros(n_pages * per, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(13)
    last = [n_pages - 1, n_pages - 3]
    f = lambda *sh: torch.as_tensor(rng.standard_normal(sh), dtype=torch.float16).cuda()  # noqa: E731
    kv = [(f(Hkv, page, D), f(Hkv, page, D)) for _ in last]
    for p, (a, b) in zip(last, kv):
        k[p * per:(p + 1) * per], v[p * per:(p + 1) * per] = a.reshape(-1), b.reshape(-1)
    rows, n = 17, 500
    for rows in (2, 17, 130):
        q = f(rows, H, D)
        c = U.CacheDesc(dtype=U.T_F16, n_head_kv=Hkv, head_dim=D, page=page, n_pages=n_pages, n_seq=1, max_pages=2)
        out = torch.zeros(rows, H, D, dtype=torch.float16, device="cuda")
        keep = [dev(last), dev([0, rows]), dev([n - rows]), dev([n])]
        tctx.tree_attention(c, H, rows, rows, n, 1 / math.sqrt(D), ptr(q), ptr(k), ptr(v), *[ptr(t) for t in keep], None, 0, ptr(out))
        kk, vv = (torch.cat([x[i] for x in kv], 1)[:, :n].double() for i in (0, 1))
        sc = torch.einsum("rhd,htd->hrt", q.double(), kk) / math.sqrt(D)
        sc = sc.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(rows, device="cuda")[:, None] + n - rows, -math.inf)
        want = torch.einsum("hrt,htd->rhd", torch.softmax(sc, -1), vv)
        # |v| < 6, weights and output rounded once each
        assert float((out.double() - want).abs().max()) <= 2 * UNIT["f16"] * 6


def test_tree_attention_repeats_bits_and_captures(tctx):
    """The same call gives the same bits, alone and replayed from a graph, and on a stream of its own."""
    import ulb_capi as U
    a = Attention("bf16", 8, 2, 128, 64, [(3000, 20), (100, 3)], seed=14)
    one, l1 = a.run(tctx)
    two, l2 = a.run(tctx)
    assert torch.equal(one, two) and torch.equal(l1, l2)
    torch.cuda.synchronize()
    with U.Context(0) as c:
        first, lf = a.run(c)
        c.sync()
        assert torch.equal(one, first) and torch.equal(l1, lf)
        g = c.capture(a.again)
        first.zero_()
        torch.cuda.synchronize()
        U.check(U.lib().ulb_graph_launch(c.h, g))
        c.sync()
        assert torch.equal(one, first)
        U.lib().ulb_graph_free(g)


def test_tree_attention_follows_the_stream(tctx):
    """Inputs still being written by the caller's stream are waited for, on every stream in turn."""
    a = Attention("f16", 4, 4, 64, 64, [(2000, 8)], seed=15)
    want, _ = a.run(tctx)
    q = a.q.clone()
    try:
        for st in (torch.cuda.Stream(), torch.cuda.Stream()):
            torch.cuda.synchronize()
            with torch.cuda.stream(st):
                tctx.use_stream(st.cuda_stream)
                a.q.zero_()
                out, _ = a.run(tctx)
                torch.cuda._sleep(20_000_000)
                a.q.copy_(q)
                a.again()
                got = out.clone()
            st.synchronize()
            assert torch.equal(got, want)
    finally:
        tctx.use_stream(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("rows", [299, 592, 600, 620])
def test_tree_attention_row_tiles_for_every_sm_and_more(tctx, rows):
    """64 heads a kv head: so many row tiles that one group of blocks walks all keys (299 rows: 75 tiles of
    256 queries), exactly one an SM (592), and more than one pass over the rows."""
    Attention("bf16", 128, 2, 64, 64, [(200, rows), (130, 3), (70, 0), (0, rows // 2)], causal=True, seed=rows).check(tctx)
    Attention("f16", 64, 1, 128, 64, [(900, rows)], seed=rows + 1).check(tctx)
    tctx.sync()


def test_use_stream_and_another_programs_capture():
    """A stream under capture is refused and the capture goes on; a context switched to it before takes part."""
    import ulb_capi as U
    a = Attention("f16", 8, 2, 64, 64, [(300, 8)], seed=16)
    st, x = torch.cuda.Stream(), torch.zeros(4, device="cuda")
    with U.Context(0) as c:
        want, _ = a.run(c)
        c.sync()
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            x.add_(1)
            st.synchronize()
            g.capture_begin()
            try:
                refused(c.use_stream, st.cuda_stream, code=U.EINVAL)
                x.add_(1)
            finally:
                g.capture_end()
            g.replay()
            st.synchronize()
            assert x.tolist() == [2.0] * 4
            c.use_stream(st.cuda_stream)
            out, _ = a.run(c)
            out.zero_()
            st.synchronize()
            h = torch.cuda.CUDAGraph()
            h.capture_begin()
            try:
                a.again()
                refused(c.use_stream, None, code=U.EINVAL)
            finally:
                h.capture_end()
            assert not bool(out.any())
            h.replay()
            st.synchronize()
            assert torch.equal(out, want)
        c.use_stream(None)


@pytest.mark.parametrize("D", [64, 80, 96, 128])
@pytest.mark.parametrize("H,Hkv,rows", [(8, 1, 9), (16, 2, 16), (6, 2, 40), (8, 1, 33)])
def test_tree_attention_tensor_core_form(tctx, D, H, Hkv, rows):
    """65 queries a kv head and more, which run on the tensor cores whatever the length: one tile of
    rows and two, tile and page edges, ragged batches, empty rows, unmapped pages, other layouts."""
    for prefix in (0, 1, 63, 64, 65, 190, 700):
        Attention("bf16", H, Hkv, D, 16, [(prefix, rows)], seed=prefix + D).check(tctx)
    Attention("f16", H, Hkv, D, 64, [(500, rows), (3, 1), (0, 0), (129, rows // 2), (0, rows)], seed=D, nhd=True).check(tctx)
    Attention("f16", H, Hkv, D, 32, [(0, rows), (100, rows), (0, 1)], empty_rows=True, stale=math.nan, seed=D + 1).check(tctx)
    Attention("bf16", H, Hkv, D, 128, [(0, rows), (300, rows)], empty_rows=True, stale=-math.inf, seed=D + 2).check(tctx)
    Attention("f16", H, Hkv, D, 16, [(333, rows), (90, rows)], unmapped=[(0, 0, -1), (0, 5, 3), (0, 20, -9), (1, 5, -1)], seed=D + 3).check(tctx)
    Attention("f16", H, Hkv, D, 256, [(900, rows), (0, rows)], causal=True, seed=D + 4).check(tctx)
    Attention("bf16", H, Hkv, D, 64, [(77, rows), (5, rows)], slots=[rows + 90, rows], seed=D + 5).check(tctx)


@pytest.mark.parametrize("D", [64, 80, 96, 128])
@pytest.mark.parametrize("H,Hkv,rows", [(2, 2, 1), (8, 2, 3), (8, 4, 16)])
def test_tree_attention_tensor_core_form_by_bytes(tctx, D, H, Hkv, rows):
    """Few queries over much K and V (by the longest sequence) run there too."""
    import ulb_capi as U
    need = max(2048, (64 << 20) // (4 * Hkv * D * 3))
    a = Attention("f16", H, Hkv, D, 64, [(700, rows), (2500, rows), (0, rows)], seed=D + rows)
    assert max(a.len) < need
    out, ls = a.run(tctx)
    # the same call with a bound on the lengths that makes it large: the other form
    c = U.CacheDesc(dtype=U.T_F16, n_head_kv=Hkv, head_dim=D, page=64, n_pages=a.n_pages, n_seq=3, max_pages=a.most + need // 64 + 1)
    table = np.full((3, c.max_pages), -1)
    table[:, :a.most] = a.table
    o2, l2 = torch.empty_like(out), torch.empty_like(ls)
    tctx.tree_attention(c, H, a.rows, rows, need + 64, 1 / math.sqrt(D), ptr(a.q), ptr(a.k), ptr(a.v), ptr(dev(table)),
                        *[ptr(t) for t in a.keep[1:]], ptr(a.mask), a.words, ptr(o2), ptr(l2))
    # either form is within the weights' and the output's rounding of the exact result (values within 5)
    assert float((out.double() - o2.double()).abs().max()) <= 4 * UNIT["f16"] * 5
    assert float((ls.double() - l2.double()).abs().max()) <= 4e-5 * (1 + float(ls.abs().max()))


@pytest.mark.parametrize("D", [64, 128])
def test_tree_attention_row_tiles_half_empty_over_long_pieces(tctx, D):
    """Two streams of 128 queries of which the second has none, over more K and V tiles than both rings
    hold: a last row tile of 64 queries, and sequences on either side of 128 queries in one call."""
    Attention("bf16", 32, 4, D, 64, [(32000, 40)], seed=D).check(tctx)
    tctx.sync()
    a = [(6000 + 97 * i, 17 + (5 * i) % 17) for i in range(16)]
    Attention("f16", 8, 2, D, 128, a, seed=D + 1).check(tctx)
    tctx.sync()


@pytest.mark.parametrize("where", ["past the end", "a slot"])
@pytest.mark.parametrize("H,Hkv,rows", [(32, 8, 40), (16, 8, 40)])
def test_tree_attention_values_that_nobody_sees_cost_nothing(tctx, where, H, Hkv, rows):
    """NaN in V past the ends, or in a slot that no row sees, leaves the answer and the time as they are."""
    a = Attention("bf16", H, Hkv, 128, 64, [(1000, rows)] * 24, seed=41)
    for b in a.see:
        b[:, 7] = False
    a.mask = torch.as_tensor(np.concatenate([pack_bits(b, a.words) for b in a.see])).cuda()

    def time():
        out, _ = a.run(tctx)
        ms = []
        for _ in range(12):
            t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            t0.record()
            a.again()
            t1.record()
            t1.synchronize()
            ms.append(t0.elapsed_time(t1))
        return out, sorted(ms)[3]

    want, clean = time()
    for s in range(24):
        for t in (range(a.len[s], 64 * len(a.table[s])) if where == "past the end" else [1007]):
            a.v[int(a.table[s, t // 64]), :, t % 64] = math.nan
    got, stale = time()
    assert torch.equal(got, want)
    # the same work; the bound is for the clock of a call of some 50 us
    assert stale <= 1.5 * clean, (stale, clean)


@pytest.mark.parametrize("kind,causal", [("f16", True), ("bf16", False)])
def test_tree_attention_many_rows_over_many_small_pages(tctx, kind, causal):
    """Head dim 256, a thousand rows over 1537 pages of 16 positions, which one block walks: page ids
    come and go under way, some of them unmapped."""
    import ulb_capi as U
    rng = np.random.default_rng(31)
    H, D, page, rows, n = 32, 256, 16, 1024, 24580
    pages = (n + page - 1) // page
    table = rng.permutation(pages)
    for j, value in ((3, -1), (511, -5), (512, pages), (700, -1), (1023, -1), (1400, pages + 9), (1530, -1)):
        table[j] = value
    g = torch.Generator(device="cuda").manual_seed(31)
    q, k, v = (torch.randn(*sh, device="cuda", generator=g).to(DT[kind]) for sh in ((rows, H, D), (pages, 1, page, D), (pages, 1, page, D)))
    see = np.ones((rows, n), bool)
    see[:, n - 40:] = rng.random((rows, 40)) < 0.5
    if causal:
        see = np.arange(n)[None] <= np.arange(rows)[:, None] + n - rows
    see &= ((table >= 0) & (table < pages))[np.arange(n) // page]
    mask = None if causal else torch.as_tensor(pack_bits(see[:, n - 40:], 2)).cuda()
    # unmapped or past the end: nothing that a row may see
    k[:, 0].view(-1, D)[int(table[-1]) * page + n % page:(int(table[-1]) + 1) * page] = math.nan
    v[:, 0].view(-1, D)[int(table[-1]) * page + n % page:(int(table[-1]) + 1) * page] = math.inf
    c = U.CacheDesc(dtype=U.dtype_id(kind), n_head_kv=1, head_dim=D, page=page, n_pages=pages, n_seq=1, max_pages=pages)
    out, lse = torch.zeros_like(q), torch.zeros(rows, H, device="cuda")
    tctx.tree_attention(c, H, rows, rows, n, 1 / 16, ptr(q), ptr(k), ptr(v), ptr(dev(table)), ptr(dev([0, rows])), ptr(dev([n - 40])),
                        ptr(dev([n])), ptr(mask), 0 if causal else 2, ptr(out), ptr(lse))
    tctx.sync()
    at = torch.as_tensor(np.clip(table, 0, pages - 1)).cuda()
    kk, vv = (x[at, 0].reshape(-1, D)[:n].double() for x in (k, v))
    u = UNIT[kind]
    for r in (0, 1, 63, 500, 777, 1023):
        s = torch.as_tensor(see[r]).cuda()
        sc = (q[r].double() @ kk.T / 16).masked_fill(~s[None], -math.inf)
        l = torch.logsumexp(sc, 1)
        p, vz = torch.exp(sc - l[:, None]), torch.where(s[:, None], vv, torch.zeros_like(vv))
        want, size = p @ vz, p @ vz.abs()
        assert bool(((out[r].double() - want).abs() <= (u + 2.0 ** -15) * size + u * want.abs() + 1e-6).all())
        assert bool(((lse[r].double() - l).abs() <= 2e-5 * (1 + l.abs())).all())


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [17.0, 17.3, 25.5])
@pytest.mark.parametrize("at", [0, 4000])
@pytest.mark.parametrize("D,H,rows,seqs,n", [(256, 2, 1, 600, 8191), (64, 4, 1, 160, 30001), (128, 8, 10, 160, 30001), (64, 8, 40, 80, 30001)])
def test_tree_attention_one_key_that_outweighs_thousands(tctx, D, H, rows, seqs, n, at, bits, kind):
    """A key of score s whose V is zero, all others of score zero with V = 1: they answer, however
    little each of them weighs.  Every sequence reads the same pages."""
    import ulb_capi as U
    page = 256
    pages = (n + page - 1) // page
    scale = float(np.float32(bits * math.log(2) / 16))
    q, k, v = (torch.zeros(*sh, dtype=DT[kind], device="cuda") for sh in ((seqs * rows, H, D), (pages, 1, page, D), (pages, 1, page, D)))
    q[:, :, 0], v[:] = 4.0, 1.0
    k[at // page, 0, at % page, 0], v[at // page, 0, at % page] = 4.0, 0.0
    c = U.CacheDesc(dtype=U.dtype_id(kind), n_head_kv=1, head_dim=D, page=page, n_pages=pages, n_seq=seqs, max_pages=pages)
    out, lse = torch.zeros_like(q), torch.zeros(seqs * rows, H, device="cuda")
    mask = torch.full((seqs * rows, 1), -1, dtype=torch.int32, device="cuda")
    tctx.tree_attention(c, H, seqs * rows, rows, n, scale, ptr(q), ptr(k), ptr(v), ptr(dev(np.tile(np.arange(pages), (seqs, 1)))),
                        ptr(dev(np.arange(seqs + 1) * rows)), ptr(dev([n - 32] * seqs)), ptr(dev([n] * seqs)), ptr(mask), 1, ptr(out), ptr(lse))
    tctx.sync()
    top = math.exp(16 * scale)
    want, l = (n - 1) / (n - 1 + top), math.log(n - 1 + top)
    # a weight and the output rounded once each; the score (|s| < 2^5) and its exponential in fp32
    assert float((out.double() - want).abs().max()) <= (2 * UNIT[kind] + 2.0 ** -15) * want
    assert float((lse.double() - l).abs().max()) <= 2e-5 * (1 + l)


@pytest.mark.parametrize("D,H,Hkv", [(64, 4, 4), (128, 8, 1), (256, 4, 1)])
def test_tree_attention_row_ranges_out_of_order(tctx, D, H, Hkv):
    """Row ranges that end before they begin or lie outside the call's rows touch no row of others."""
    import ulb_capi as U
    low, high = -2 ** 31, 2 ** 31 - 1
    a = Attention("f16", H, Hkv, D, 64, [(200, 40)] * 4, seed=D)
    want, _ = a.run(tctx)
    c = U.CacheDesc(dtype=U.T_F16, n_head_kv=Hkv, head_dim=D, page=64, n_pages=a.n_pages, n_seq=4, max_pages=a.most)
    for start, rows in (([high, high, 160, 120, 160], [(120, 160)]), ([0, 150, low, -1, -1], [(0, 40)]),
                        ([high, low, low, low, low], []), ([500, 40, 80, low, 0], [(40, 80)])):
        out = torch.full((a.rows + 40, H, D), 9.0, dtype=torch.float16, device="cuda")
        q = torch.cat([a.q, a.q[:40] + 1])  # rows past the call's, which it must not read or write
        tctx.tree_attention(c, H, a.rows, 40, max(a.len), 1 / math.sqrt(D), ptr(q), ptr(a.k), ptr(a.v), ptr(a.keep[0]), ptr(dev(start)),
                            ptr(a.keep[2]), ptr(a.keep[3]), ptr(a.mask), a.words, ptr(out), None)
        tctx.sync()
        for b, e in rows:
            assert torch.equal(out[b:e], want[b:e])
            out[b:e] = 9.0
        assert bool((out == 9.0).all())


def test_tree_attention_refusals(tctx):
    import ulb_capi as U
    x = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    i = dev([0, 1, 1, 1])
    good = dict(dtype=U.T_F16, n_head_kv=2, head_dim=64, page=16, n_pages=4, n_seq=1, max_pages=4)

    def call(cache=None, n_head=4, rows=1, max_rows=1, max_len=1, scale=0.1, q=x.data_ptr(), mask=ptr(i), words=1, **k):
        tctx.tree_attention(U.CacheDesc(**{**good, **(cache or {})}), n_head, rows, max_rows, max_len, scale, q, ptr(x), ptr(x),
                            ptr(i), ptr(i), ptr(i), ptr(i), mask, words, ptr(x))

    for kw in (dict(cache=dict(head_dim=72)), dict(cache=dict(page=24)), dict(cache=dict(dtype=U.T_F32)), dict(n_head=5),
               dict(n_head=0), dict(n_head=2 * 65), dict(scale=0.0), dict(scale=float("nan")), dict(rows=-1), dict(words=-1),
               dict(mask=None), dict(words=0), dict(q=x.data_ptr() + 2), dict(q=None), dict(cache=dict(page_stride=4)),
               dict(cache=dict(n_seq=70000))):
        refused(call, **kw)
    call(rows=0)
    call()


# ---------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("L,Hkv,page,D,nhd", [(1, 1, 16, 64, False), (3, 2, 64, 80, False), (2, 3, 256, 128, True), (2, 8, 256, 256, False)])
def test_pages_copy_and_compact(tctx, kind, L, Hkv, page, D, nhd):
    import ulb_capi as U
    rng = np.random.default_rng(page + D)
    n_pages, S, most = 13, 4, 3
    shape = (L, n_pages, page, Hkv, D) if nhd else (L, n_pages, Hkv, page, D)
    k, v = (torch.as_tensor(rng.standard_normal(shape)).to(DT[kind]).cuda() for _ in range(2))
    cache = U.CacheDesc(dtype=U.dtype_id(kind), n_layer=L, n_head_kv=Hkv, head_dim=D, page=page, n_pages=n_pages, n_seq=S, max_pages=most)
    if nhd:
        cache.head_stride, cache.pos_stride, cache.page_stride = D, Hkv * D, page * Hkv * D
        cache.layer_stride = n_pages * page * Hkv * D
    wk, wv = k.clone(), v.clone()
    cut = lambda t, p, n: t[:, p, :n] if nhd else t[:, p, :, :n]  # noqa: E731
    moves = [(0, 5, page), (1, 6, 1), (2, 7, page - 1), (3, 8, 0), (0, 9, page + 100), (4, n_pages, 5), (-1, 10, 5), (1, 11, -3)]
    for a, b, n in moves:
        if 0 <= a < n_pages and 0 <= b < n_pages:
            n = min(max(n, 0), page)
            for w in (wk, wv):
                cut(w, b, n).copy_(cut(w, a, n).clone())
    tctx.pages_copy(cache, ptr(k), ptr(v), ptr(dev(moves)), len(moves))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    # paths across page edges; one empty, one longer than a block's tile, one on an unmapped page
    table = rng.permutation(n_pages)[:S * most].reshape(S, most)
    table[3, 1] = -1
    max_src = min(100, 2 * page - 2)
    base = np.array([page - 3, 2, 0, page - 2])
    count = np.array([min(7, max_src), max_src, 0, min(6, max_src)])
    src = np.stack([np.sort(rng.permutation(3 * page - page)[:max_src]) for _ in range(S)])
    src[3, :count[3]] = np.arange(1, count[3] + 1)
    tctx.pages_compact(cache, ptr(k), ptr(v), ptr(dev(table)), ptr(dev(base)), ptr(dev(count)), ptr(dev(src)), max_src)
    for s in range(S):
        for w in (wk, wv):
            old = w.clone()
            for i in range(count[s]):
                f, t = base[s] + src[s, i], base[s] + i
                pf, pt = (table[s, x // page] if x // page < most else -1 for x in (f, t))
                if pf >= 0 and pt >= 0:
                    if nhd:
                        w[:, pt, t % page] = old[:, pf, f % page]
                    else:
                        w[:, pt, :, t % page] = old[:, pf, :, f % page]
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_pages_past_32_bit_offsets(tctx):
    import ulb_capi as U
    Hkv, page, D = 8, 256, 128
    per = Hkv * page * D
    n = (1 << 31) // per + 4
    k = torch.empty(n * per, dtype=torch.float16, device="cuda")
    v = torch.empty(n * per, dtype=torch.float16, device="cuda")
    k[:per], v[:per] = 1.5, 2.5
    k[(n - 1) * per:], v[(n - 1) * per:] = 0.0, 0.0
    cache = U.CacheDesc(dtype=U.T_F16, n_layer=1, n_head_kv=Hkv, head_dim=D, page=page, n_pages=n, n_seq=1, max_pages=1)
    tctx.pages_copy(cache, ptr(k), ptr(v), ptr(dev([[0, n - 1, page]])), 1)
    assert bool((k[(n - 1) * per:] == 1.5).all()) and bool((v[(n - 1) * per:] == 2.5).all())


def test_page_book_keeps_every_sequence(tctx):
    """Random reserves, forks, roll-backs and defragmentations: every sequence reads back what was
    written to it, whoever it shared pages with."""
    import ulb_capi as U
    rng = np.random.default_rng(21)
    L, Hkv, page, D, n_pages, S, most = 2, 2, 16, 64, 40, 6, 12
    k = torch.zeros(L, n_pages, Hkv, page, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    cache = U.CacheDesc(dtype=U.T_F16, n_layer=L, n_head_kv=Hkv, head_dim=D, page=page, n_pages=n_pages, n_seq=S, max_pages=most)
    book = U.Pages(tctx, cache, ptr(k), ptr(v))
    words = [[] for _ in range(S)]  # what each position holds
    import ctypes as C

    def table():
        t = np.empty((S, most), np.int32)
        tctx.sync()
        U.check(U.lib().ulb_memcpy_d2h(tctx.h, t.ctypes.data_as(C.c_void_p), book.table, t.nbytes))
        return t

    for step in range(300):
        what = rng.integers(0, 5)
        s = int(rng.integers(0, S))
        if what <= 1:  # append, or write again from some earlier position
            n0 = len(words[s]) if what == 0 else int(rng.integers(0, len(words[s]) + 1))
            n1 = min(n0 + int(rng.integers(0, 40)), most * page)
            try:
                book.reserve(s, n0, n1)
            except U.UlbError as e:
                assert e.code == U.ENOMEM
                continue
            t = table()
            new = [float(rng.integers(1, 2000)) for _ in range(n1 - n0)]
            if n1 > n0:
                at = np.arange(n0, n1)
                pg, of = torch.as_tensor(t[s, at // page]).long().cuda(), torch.as_tensor(at % page).cuda()
                val = torch.as_tensor(new, dtype=torch.float16, device="cuda")
                for pool, add in ((k, 0.0), (v, 1.0)):
                    pool[:, pg, :, of] = (val + add)[:, None, None, None].expand(-1, L, Hkv, D)
                words[s] = words[s][:n0] + new
        elif what == 2:
            d = int(rng.integers(0, S))
            if d != s and not words[d] and book.mapped(d) == 0:
                n = int(rng.integers(0, len(words[s]) + 1))
                book.fork(s, d, n)
                words[d] = words[s][:n]
        elif what == 3:
            n = int(rng.integers(0, len(words[s]) + 1)) * int(rng.integers(0, 2))
            book.truncate(s, n)
            words[s] = words[s][:n]
        elif step % 7 == 0:
            used = book.defrag()
            t = table()
            assert t.max() < max(used, 1) and used == n_pages - book.free
        if step % 5 == 0:
            t = table()
            for q in range(S):
                at = np.arange(len(words[q]))
                pg, of = torch.as_tensor(t[q, at // page]).long().cuda(), torch.as_tensor(at % page).cuda()
                val = torch.as_tensor(words[q], dtype=torch.float16, device="cuda")
                assert torch.equal(k[:, pg, :, of], val[:, None, None, None].expand(-1, L, Hkv, D))
                assert torch.equal(v[:, pg, :, of], (val + 1)[:, None, None, None].expand(-1, L, Hkv, D))
                assert bool((t[q, book.mapped(q):] == -1).all())
    book.close()


def test_pages_refusals(tctx):
    import ulb_capi as U
    x = torch.zeros(1 << 12, dtype=torch.float16, device="cuda")
    c = U.CacheDesc(dtype=U.T_F16, n_layer=1, n_head_kv=1, head_dim=64, page=16, n_pages=4, n_seq=2, max_pages=3)
    bad = U.CacheDesc(dtype=U.T_F16, n_layer=1, n_head_kv=1, head_dim=64, page=17, n_pages=4, n_seq=2, max_pages=3)
    refused(tctx.pages_copy, bad, ptr(x), ptr(x), ptr(x), 1)
    refused(tctx.pages_copy, c, ptr(x), None, ptr(x), 1)
    refused(tctx.pages_copy, c, ptr(x) + 2, ptr(x), ptr(x), 1)
    refused(tctx.pages_copy, c, ptr(x), ptr(x), ptr(x), -1)
    refused(tctx.pages_compact, c, ptr(x), ptr(x), ptr(x), ptr(x), ptr(x), None, 1)
    refused(tctx.pages_compact, c, ptr(x), ptr(x), ptr(x), ptr(x), ptr(x), ptr(x), -1)
    tctx.pages_copy(c, None, None, None, 0)
    b = U.Pages(tctx, c, ptr(x), ptr(x))
    b.reserve(0, 0, 40)
    refused(b.reserve, 0, 0, 49)          # past max_pages
    refused(b.reserve, 2, 0, 1)
    refused(b.reserve, 0, 5, 4)
    refused(b.reserve, 1, 0, 17, code=U.ENOMEM)  # one page left
    assert b.free == 1 and b.mapped(1) == 0
    refused(b.fork, 0, 0, 1)
    refused(b.fork, 0, 1, 49)
    b.fork(0, 1, 17)
    refused(b.fork, 0, 1, 1)              # holds pages
    refused(b.truncate, 0, -1)
    b.close()


# ---------------------------------------------------------------------------------------------- logits
class Logits:
    def __init__(self, kind, V, sizes, seed=0, history=50, biases=5, nodes=True, grammar="rows", params=True, pad=0, far=False):
        rng = np.random.default_rng(seed)
        self.kind, self.V, self.ld = kind, V, V + pad
        self.start = np.concatenate([[0], np.cumsum(sizes)])
        self.rows, S = int(self.start[-1]), len(sizes)
        self.S, self.sizes = S, sizes
        x = rng.standard_normal((self.rows, self.ld)) * 4
        x[:, :V][rng.random((self.rows, V)) < 0.002] = -np.inf
        self.x = torch.as_tensor(x).to(DT[kind]).cuda()
        few = max(1, V // 7)
        tok = lambda n: rng.integers(0, few, n) * 7 % V  # noqa: E731
        hl = [history] + [int(rng.integers(0, history + 1)) for _ in range(S - 1)]
        self.hs = np.concatenate([[0], np.cumsum(hl)])
        self.hist = np.concatenate([tok(n) for n in hl] + [np.zeros(0, int)]) if history else None
        if history and self.hist.size > 4:
            self.hist[1], self.hist[2] = -1, V + 3  # ignored
        self.prompt = np.array([n // 3 for n in hl])
        self.tok = tok(self.rows) if nodes else None
        self.words = (max(sizes) + 31) // 32
        bits = np.zeros((self.rows, max(sizes)), bool)
        for s, n in enumerate(sizes):
            b = rng.random((n, n)) < 0.4
            b[np.arange(n), np.arange(n)] = True
            bits[self.start[s]:self.start[s + 1], :n] = b
        self.bits = bits
        self.params = np.stack([rng.uniform(0.8, 1.6, S), rng.uniform(-0.5, 1, S), rng.uniform(-0.2, 0.5, S)], 1).astype(np.float32) if params else None
        nb = [int(rng.integers(0, biases + 1)) for _ in range(S)] if biases else None
        if biases:
            self.bs = np.concatenate([[0], np.cumsum(nb)])
            self.bt = np.concatenate([np.sort(rng.integers(0, max(1, V // 3), n)) for n in nb] + [np.zeros(0, int)])
            self.bv = (rng.standard_normal(self.bt.size) * 3).astype(np.float32)
        self.biases = biases
        self.allow = self.row_allow = None
        if grammar:
            n = self.rows if grammar == "rows" else 3
            self.allow_bits = rng.random((n, (V + 31) // 32 * 32)) < 0.5
            self.allow_bits[0] = False  # allows nothing
            self.allow = pack_bits(self.allow_bits, (V + 31) // 32)
            if grammar == "index":
                self.row_allow = rng.integers(-1, 4, self.rows)

    def run(self, ctx, in_place=False):
        import ulb_capi as U
        out = self.x.clone() if in_place else torch.full((self.rows, self.ld), 5.0, device="cuda")
        self.keep = dict(row_start=dev(self.start))
        if self.params is not None:
            self.keep["params"] = dev(self.params, torch.float32)
        if self.hist is not None:
            self.keep.update(history=dev(self.hist), history_start=dev(self.hs), prompt=dev(self.prompt))
        if self.tok is not None:
            self.keep.update(node_tokens=dev(self.tok), words=torch.as_tensor(pack_bits(self.bits, self.words)).cuda())
        if self.biases:
            self.keep.update(bias_start=dev(self.bs), bias_tokens=dev(np.append(self.bt, 0)), bias_values=dev(np.append(self.bv, 0), torch.float32))
        if self.allow is not None:
            self.keep["allow"] = torch.as_tensor(self.allow).cuda()
            if self.row_allow is not None:
                self.keep["row_allow"] = dev(self.row_allow)
        k = {n: ptr(t) for n, t in self.keep.items()}
        ctx.logits_process(U.dtype_id(self.kind), ptr(out) if in_place else ptr(self.x), ptr(out), self.V, self.S, self.rows,
                           k.pop("row_start"), max_rows=max(self.sizes), ld_in=self.ld, ld_out=self.ld,
                           n_words=self.words if self.tok is not None else 0,
                           n_allow=0 if self.allow is None else len(self.allow), **k)
        return out

    def check(self, ctx, in_place=False):
        out = self.run(ctx, in_place)
        rest = out[:, self.V:].cpu()
        assert torch.equal(rest, self.x[:, self.V:].cpu() if in_place else torch.full_like(rest, 5.0))
        got = out[:, :self.V].double().cpu().numpy()
        x = self.x[:, :self.V].double().cpu().numpy()
        for s in range(self.S):
            seen, made = np.zeros(self.V, bool), np.zeros(self.V)
            if self.hist is not None:
                h = self.hist[self.hs[s]:self.hs[s + 1]]
                ok = (h >= 0) & (h < self.V)
                seen[h[ok]] = True
                np.add.at(made, h[self.prompt[s]:][ok[self.prompt[s]:]], 1)
            bias = np.zeros(self.V)
            if self.biases:
                b = slice(self.bs[s], self.bs[s + 1])
                np.add.at(bias, self.bt[b], self.bv[b].astype(np.float64))
            rep, pres, freq = self.params[s].astype(np.float64) if self.params is not None else (1.0, 0.0, 0.0)
            for r in range(self.start[s], self.start[s + 1]):
                n = made.copy()
                if self.tok is not None:
                    for j in np.nonzero(self.bits[r])[0]:
                        n[self.tok[self.start[s] + j]] += 1
                was = seen | (n > 0)
                y = np.where(was, np.where(x[r] > 0, x[r] / rep, x[r] * rep), x[r])
                y = y - freq * n - pres * (n > 0) + bias
                size = np.abs(np.where(np.isfinite(x[r]), x[r], 0)) * 2 + np.abs(freq * n) + abs(pres) + np.abs(bias) + 10
                if self.allow is not None:
                    a = r if self.row_allow is None else self.row_allow[r]
                    if 0 <= a < len(self.allow):
                        y = np.where(self.allow_bits[a, :self.V], y, -np.inf)
                assert np.array_equal(np.isinf(y), np.isinf(got[r])), (s, r)
                f = np.isfinite(y)
                # a handful of fp32 operations on values of that size
                assert (np.abs(got[r] - y)[f] <= 8 * 2.0 ** -24 * size[f]).all(), (s, r, np.abs(got[r] - y)[f].max())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,pad", [(1, 0), (31, 1), (1000, 0), (32003, 0), (32000, 0), (5001, 3), (40003, 5)])
def test_logits_shapes(tctx, kind, V, pad):
    Logits(kind, V, [3, 1, 5], seed=V, pad=pad).check(tctx)
    Logits(kind, V, [1], seed=V + 1, pad=pad, nodes=False, grammar="index").check(tctx)


@pytest.mark.parametrize("kw", [dict(history=0), dict(biases=0), dict(nodes=False), dict(grammar=None), dict(params=False),
                                dict(history=0, biases=0, nodes=False, grammar=None, params=False), dict(history=9000),
                                dict(biases=400), dict(grammar="index")])
def test_logits_parts(tctx, kw):
    Logits("f32", 4099, [2, 7], seed=3, **kw).check(tctx)
    Logits("f32", 4096, [9], seed=4, **kw).check(tctx, in_place=True)


def test_logits_large_trees_and_batches(tctx):
    Logits("f32", 2048, [200, 1, 63], seed=5).check(tctx)
    Logits("f16", 20000, [1] * 130, seed=6, nodes=False).check(tctx)
    Logits("bf16", 50, [1000], seed=7).check(tctx)  # many nodes of one token in one chunk


def test_logits_then_sampler(tctx):
    """A grammar that allows one token makes the sampler draw it, greedily and not."""
    import ctypes as C

    import ulb_capi as U
    V, rows = 3001, 6
    x = torch.randn(rows, V, device="cuda")
    want = np.array([0, 31, 32, 1500, 2999, 3000])
    bits = np.zeros((rows, (V + 31) // 32 * 32), bool)
    bits[np.arange(rows), want] = True
    allow = torch.as_tensor(pack_bits(bits, (V + 31) // 32)).cuda()
    st = dev(np.arange(rows + 1))
    tctx.logits_process(U.T_F32, ptr(x), ptr(x), V, rows, rows, ptr(st), max_rows=1, allow=ptr(allow), n_allow=rows)
    for t in (0.0, 0.8):
        out = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        w = U.Warp(t, 0, 1.0)
        U.check(U.lib().ulb_sample(tctx.h, ptr(x), rows, V, V, C.byref(w), 1, 0, 0, U.RNG_DRAFT, ptr(out)))
        assert out.cpu().tolist() == want.tolist()


def test_logits_refusals(tctx):
    import ulb_capi as U
    x = torch.zeros(4, 64, device="cuda")
    i = dev([0, 1, 2, 3, 4])
    ok = dict(dtype=U.T_F32, logits=ptr(x), out=ptr(x), V=64, n_seq=4, rows=4, row_start=ptr(i))
    call = lambda **k: tctx.logits_process(**{**ok, **k})  # noqa: E731
    for kw in (dict(dtype=U.T_Q4_0), dict(V=0), dict(ld_in=63), dict(ld_out=32), dict(row_start=None), dict(logits=None), dict(rows=-1),
               dict(history=ptr(i)), dict(node_tokens=ptr(i)), dict(node_tokens=ptr(i), words=ptr(i), n_words=33),
               dict(bias_start=ptr(i)), dict(dtype=U.T_F16), dict(ld_out=128), dict(logits=ptr(x) + 1)):
        refused(call, **kw)
    call()
    call(rows=0, row_start=None)
