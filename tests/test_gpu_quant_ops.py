"""Head norms with rotation, the quantised cache and its attention on the GPU against plain computations in 64 bits and
against GGUF's own quantisers.  Tolerances are stated where they are used, from the roundings each operator makes."""
import math

import numpy as np
import pytest

from test_gpu_paged_ops import DT, KEEP, UNIT, dev, frequencies, kept, ptr, refused, rotate, tctx  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FORMATS = {"q8": 8, "q4": 3}


# ---------------------------------------------------------------------------------------------- norms with rotation
def normed(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def norm_case(rng, kind, M, H, KV, D, wide):
    """Rows of q, k and v heads side by side (a pad of `wide` elements behind each row), weights, positions."""
    row = (H + 2 * KV) * D + wide
    qkv = torch.as_tensor(rng.standard_normal((M, row)) * 2).to(DT[kind]).cuda()
    KEEP.append(qkv)
    q = qkv[:, :H * D].reshape(M, H, D)
    k = qkv[:, H * D:(H + KV) * D].reshape(M, KV, D)
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    pos = rng.integers(0, 131072, M)
    return qkv, row, q, k, w, pos


SHAPES = [(1, 1, 1, 64, 64), (3, 5, 5, 80, 48), (7, 32, 8, 128, 128), (300, 9, 3, 96, 96), (2, 3, 1, 256, 64), (5, 2, 0, 8, 8), (6, 3, 1, 80, 24), (9, 5, 3, 64, 56),
          (4, 3, 2, 72, 32), (1030, 40, 8, 128, 64), (17, 64, 8, 64, 64)]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,H,KV,D,rot", SHAPES)
def test_norm_rope_matches_formula(tctx, kind, layout, M, H, KV, D, rot):
    import ulb_capi as U
    rng = np.random.default_rng(M * D + rot)
    wide = 8 if M % 2 else 3  # rows that are, and are not, whole 16-byte steps apart
    qkv, row, q, k, (wq, wk), pos = norm_case(rng, kind, M, H, KV, D, wide)
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout)
    oq, ok = torch.empty(M, H, D, dtype=DT[kind], device="cuda"), torch.empty(M, max(KV, 1), D, dtype=DT[kind], device="cuda")
    e = qkv.element_size()
    r.norm_apply(U.dtype_id(kind), ptr(qkv), ptr(qkv) + H * D * e, M, H, KV, ptr(wq), ptr(wk), 1e-5, ptr(dev(pos)), ptr(oq), ptr(ok),
                 q_row=row, k_row=row)
    f, m = frequencies(rot, 10000.0)
    for got, x, w in ((oq, q, wq), (ok, k, wk)):
        if x.shape[1] == 0:
            continue
        n = normed(x.double().cpu().numpy(), w.double().cpu().numpy(), 1e-5)
        want = rotate(n, pos, f, m, rot, layout == "half")
        # the sum of squares goes through at most 8 + 5 roundings, the factor and the products four, the sines are good to
        # 2^-21 of a pair whose length is at most sqrt 2 of its larger element, and one store
        big = np.abs(n).max() * 1.5
        assert np.abs(got.double().cpu().numpy() - want).max() <= UNIT[kind] * big + 2.0 ** -19 * big
    r.close()


def test_norm_rope_in_place_on_other_streams_and_captured(tctx):
    import ulb_capi as U
    rng = np.random.default_rng(5)
    M, H, KV, D = 33, 6, 2, 128
    r = U.Rope(tctx, D, layout="half")
    q, k = (torch.as_tensor(rng.standard_normal((M, n, D))).half().cuda() for n in (H, KV))
    w = dev(rng.uniform(0.5, 1.5, D), torch.float32)
    pos = dev(rng.integers(0, 999, M))
    oq, ok = torch.empty_like(q), torch.empty_like(k)
    args = (U.T_F16, ptr(q), ptr(k), M, H, KV, ptr(w), ptr(w), 1e-6, ptr(pos))
    r.norm_apply(*args, ptr(oq), ptr(ok))
    want = oq.clone(), ok.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    tctx.use_stream(side.cuda_stream)
    oq.zero_(), ok.zero_()
    torch.cuda.synchronize()
    g = tctx.capture(lambda: r.norm_apply(*args, ptr(oq), ptr(ok)))
    for _ in range(2):
        U.check(U.lib().ulb_graph_launch(tctx.h, g))
    tctx.sync()
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])
    U.lib().ulb_graph_free(g)
    r.norm_apply(*args, ptr(q), ptr(k))  # in place
    tctx.sync()
    tctx.use_stream(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    r.close()


def pair_sizes(x, rot, half):
    """|a| + |b| at both elements of each pair, |x| at the others."""
    y = np.abs(x)
    i0, i1 = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., i0] = y[..., i1] = y[..., i0] + y[..., i1]
    return y


def norm_loss(x, w, pos, f, m, rot, half, dy, eps):
    return (rotate(normed(x, w, eps), pos, f, m, rot, half) * dy).sum()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,H,KV,D,rot", [(1, 1, 1, 64, 64), (3, 5, 5, 80, 48), (70, 32, 8, 128, 128), (31, 9, 3, 96, 32), (2, 3, 1, 256, 64),
                                          (5, 2, 0, 16, 16), (2049, 12, 4, 64, 64)])
def test_norm_rope_gradient(tctx, kind, layout, M, H, KV, D, rot):
    import ulb_capi as U
    rng = np.random.default_rng(M + D)
    eps = 1e-5
    qkv, row, q, k, (wq, wk), pos = norm_case(rng, kind, M, H, KV, D, 8 if M % 2 else 5)
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout)
    e, f, m = qkv.element_size(), *frequencies(rot, 10000.0)
    dy = [torch.as_tensor(rng.standard_normal((M, n, D))).to(DT[kind]).cuda() for n in (H, KV)]
    dx = [torch.empty_like(t) for t in dy]
    dw = [torch.full((D,), math.nan, device="cuda") for _ in range(2)]
    call = lambda: r.norm_grad(U.dtype_id(kind), ptr(qkv), ptr(qkv) + H * D * e, ptr(dy[0]), ptr(dy[1]), M, H, KV, ptr(wq), ptr(wk), eps,  # noqa: E731
                               ptr(dev(pos)), ptr(dx[0]), ptr(dx[1]), ptr(dw[0]), ptr(dw[1]), q_row=row, k_row=row)
    call()
    first = [t.clone() for t in dw]
    for i, (x, w) in enumerate(((q, wq), (k, wk))):
        if x.shape[1] == 0:
            assert torch.isnan(dw[i]).all()  # no heads: not touched
            continue
        x64, w64, y64 = (t.double().cpu().numpy() for t in (x, w, dy[i]))
        s = 1 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps)
        g = rotate(y64, pos, f, m, rot, layout == "half", sign=-1.0)
        n = x64 * s
        want = s * (w64 * g - n * (w64 * g * n).mean(-1, keepdims=True))
        # as the forward pass: two sums of a head, products, sines to 2^-21, one store; the two terms are at most this large
        big = (s * (np.abs(w64 * g).max(-1, keepdims=True) * (1 + np.abs(n) * np.abs(n).max(-1, keepdims=True)))).max() * 1.5
        got = dx[i].double().cpu().numpy()
        assert np.abs(got - want).max() <= UNIT[kind] * np.abs(want).max() + 2.0 ** -18 * big
        # a term g n of a weight's gradient: g = a cos + b sin is off by 2^-21 (the sines) plus 2^-23 (its own roundings) of
        # |a| + |b|, however small g itself, and n by 2^-20 of itself: together below 2^-18 of (|a| + |b|) |n|.  A lane adds
        # at most M H / 64 of them one by one
        terms = (pair_sizes(y64, rot, layout == "half") * np.abs(n)).sum((0, 1))
        chain = max(1.0, M * x.shape[1] / 64)
        assert (np.abs(dw[i].double().cpu().numpy() - (g * n).sum((0, 1))) <= (2.0 ** -18 + chain * 2.0 ** -24) * terms + 1e-30).all()
        # differences of the 64-bit function along a random direction: the quotient is off by its third derivative (h^2)
        u, v = rng.standard_normal(x64.shape), rng.standard_normal(D)
        h = 1e-5
        loss = lambda z: norm_loss(x64 + z * u, w64 + z * v, pos, f, m, rot, layout == "half", y64, eps)  # noqa: E731
        slope = (loss(h) - loss(-h)) / (2 * h)
        along = (want * u).sum() + ((g * n).sum((0, 1)) * v).sum()
        size = np.abs(want * u).sum() + np.abs((g * n).sum((0, 1)) * v).sum()
        assert abs(slope - along) <= 1e-5 * size
    call()
    for a, b in zip(first, dw):
        assert torch.equal(a, b) or torch.isnan(a).all()  # the same bits
    r.close()


def test_norm_rope_gradient_of_no_rows_and_captured(tctx):
    import ulb_capi as U
    r = U.Rope(tctx, 64)
    w = dev(np.ones(64), torch.float32)
    dw = [torch.full((64,), 3.0, device="cuda") for _ in range(2)]
    r.norm_grad(U.T_F32, None, None, None, None, 0, 4, 2, ptr(w), ptr(w), 1e-6, None, None, None, ptr(dw[0]), ptr(dw[1]))
    assert not dw[0].any() and not dw[1].any()
    rng = np.random.default_rng(0)
    x, dy = (torch.as_tensor(rng.standard_normal((40, 6, 64)), dtype=torch.float32).cuda() for _ in range(2))
    q, k, dq, dk = x[:, :4].contiguous(), x[:, 4:].contiguous(), dy[:, :4].contiguous(), dy[:, 4:].contiguous()
    pos = dev(np.arange(40))
    outs = [[torch.empty_like(q), torch.empty_like(k), *(torch.empty(64, device="cuda") for _ in range(2))] for _ in range(2)]
    call = lambda o: r.norm_grad(U.T_F32, ptr(q), ptr(k), ptr(dq), ptr(dk), 40, 4, 2, ptr(w), ptr(w), 1e-6, ptr(pos), *map(ptr, o))  # noqa: E731
    call(outs[0])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    tctx.use_stream(side.cuda_stream)
    graphs = [tctx.capture(lambda: call(outs[1])) for _ in range(2)]  # two graphs, one workspace, one after the other
    for g in graphs:
        U.check(U.lib().ulb_graph_launch(tctx.h, g))
    tctx.sync()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for g in graphs:
        U.lib().ulb_graph_free(g)
    tctx.use_stream(torch.cuda.current_stream().cuda_stream)
    # the gradients of the outputs may be overwritten by those of the rows
    want = [t.clone() for t in outs[0]]
    r.norm_grad(U.T_F32, ptr(q), ptr(k), ptr(dq), ptr(dk), 40, 4, 2, ptr(w), ptr(w), 1e-6, ptr(pos), ptr(dq), ptr(dk), ptr(outs[0][2]),
                ptr(outs[0][3]))
    assert torch.equal(dq, want[0]) and torch.equal(dk, want[1]) and torch.equal(outs[0][2], want[2])
    r.close()


def test_norm_rope_refusals(tctx):
    import ulb_capi as U
    x = torch.zeros(4096, device="cuda")
    r = U.Rope(tctx, 64, layout="half", rot_dim=64)
    p = ptr(x)
    good = dict(dtype=U.T_F32, q=p, k=p, M=2, n_head=2, n_head_kv=1, q_weight=p, k_weight=p, eps=1e-6, pos=p, q_out=p + 4096, k_out=p + 8192)
    r.norm_apply(**good)
    for bad in (dict(dtype=2), dict(M=-1), dict(n_head=0), dict(n_head_kv=-1), dict(eps=0.0), dict(eps=math.nan), dict(q_row=-1), dict(q=None),
                dict(k=None), dict(q_weight=None), dict(pos=None), dict(k_out=None), dict(q=p + 2), dict(pos=p + 2), dict(k_weight=p + 1),
                dict(q_out=p, q_row=256)):
        refused(r.norm_apply, **{**good, **bad})
    g = dict(dtype=U.T_F32, q=p, k=p, dq_out=p, dk_out=p, M=2, n_head=2, n_head_kv=1, q_weight=p, k_weight=p, eps=1e-6, pos=p, dq=p + 4096,
             dk=p + 8192, dq_weight=p + 12000, dk_weight=p + 12800)
    for bad in (dict(dq_weight=None), dict(dk_weight=None), dict(dq_out=None), dict(dk=None), dict(dq_weight=p + 2), dict(dq=p + 2), dict(eps=-1.0)):
        refused(r.norm_grad, **{**g, **bad})
    for bad in (dict(head_dim=66), dict(head_dim=264), dict(head_dim=64, rot_dim=36, layout="half")):
        h = U.Rope(tctx, **bad)
        refused(h.norm_apply, **good, code=U.EUNSUPPORTED)
        h.close()
    r.close()


# ---------------------------------------------------------------------------------------------- the quantised cache
def row_bytes(fmt, D):
    used = D + D // 16 if fmt == "q8" else D // 2 + D // 8
    return (used + 15) // 16 * 16


def decode(fmt, rows, D):
    """Codes and scales of rows of bytes [..., row_bytes], as the header describes them: codes [..., D], d, m [..., D / 32]."""
    if fmt == "q8":
        d = np.ascontiguousarray(rows[..., D:D + D // 16]).view(np.float16)
        return np.ascontiguousarray(rows[..., :D]).view(np.int8).astype(np.int64), d, np.zeros_like(d)
    w = np.ascontiguousarray(rows[..., :D // 2]).view(np.uint32)
    code = np.empty(rows.shape[:-1] + (D,), np.int64)
    at = (0, 16, 4, 20)
    for c in range(D // 64):
        for i in range(8):
            for e in range(4):
                for h in range(2):
                    code[..., c * 64 + h * 32 + 4 * i + e] = (w[..., c * 8 + i] >> (at[e] + 8 * h)) & 15
    s = np.ascontiguousarray(rows[..., D // 2:D // 2 + D // 8]).view(np.float16)
    return code, s[..., 0::2], s[..., 1::2]


def values(fmt, rows, D, dtype=np.float64):
    code, d, m = decode(fmt, rows, D)
    with np.errstate(invalid="ignore"):
        return code.astype(dtype) * np.repeat(d.astype(dtype), 32, -1) + np.repeat(m.astype(dtype), 32, -1)


def gguf_blocks(fmt, x):
    """What GGUF's quantiser makes of fp32 rows [..., D]: codes, d, m."""
    import gguf
    t = gguf.GGMLQuantizationType.Q8_0 if fmt == "q8" else gguf.GGMLQuantizationType.Q4_1
    raw = gguf.quants.quantize(np.ascontiguousarray(x, np.float32), t)
    if fmt == "q8":
        b = raw.reshape(x.shape[:-1] + (-1, 34))
        d = np.ascontiguousarray(b[..., :2]).view(np.float16)[..., 0]
        return np.ascontiguousarray(b[..., 2:]).view(np.int8).reshape(x.shape).astype(np.int64), d, np.zeros_like(d)
    b = raw.reshape(x.shape[:-1] + (-1, 20))
    dm = np.ascontiguousarray(b[..., :4]).view(np.float16)
    code = np.concatenate([b[..., 4:] & 15, b[..., 4:] >> 4], -1).reshape(x.shape).astype(np.int64)
    return code, dm[..., 0], dm[..., 1]


def append_case(rng, M, H, KV, D, page, n_seq, max_pages, kind):
    qkv = torch.as_tensor(rng.standard_normal((M, (H + 2 * KV) * D)) * 2).to(DT[kind]).cuda()
    n_pages = n_seq * max_pages + 2
    table = rng.permutation(n_pages)[:n_seq * max_pages].reshape(n_seq, max_pages).astype(np.int32)
    places = rng.permutation(n_seq * max_pages * page)[:M]
    return qkv, table, n_pages, places // (max_pages * page), places % (max_pages * page)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("M,H,KV,D,page,in_kind,kind,norm", [
    (1, 1, 1, 64, 16, "f32", "f16", False), (5, 5, 5, 128, 32, "f16", "f16", True), (70, 32, 8, 128, 64, "bf16", "bf16", True),
    (33, 3, 1, 256, 256, "f32", "bf16", True), (300, 4, 2, 64, 16, "f32", "f16", False), (64, 12, 4, 128, 128, "f16", "bf16", False)])
def test_append_writes_ggufs_blocks_and_read_gives_their_values(tctx, fmt, M, H, KV, D, page, in_kind, kind, norm):
    import ulb_capi as U
    rng = np.random.default_rng(M + D)
    n_seq, max_pages = 3, max(2, (M + page - 1) // page)
    qkv, table, n_pages, seq, slot = append_case(rng, M, H, KV, D, page, n_seq, max_pages, in_kind)
    RB = row_bytes(fmt, D)
    k, v = (torch.full((n_pages, KV, page, RB), 0xA5, dtype=torch.uint8, device="cuda") for _ in range(2))
    d = U.QuantDesc(FORMATS[fmt], U.dtype_id(kind), KV, D, page, n_pages, n_seq, max_pages)
    assert d.row_bytes == RB
    r = U.Rope(tctx, D, layout="half")
    pos = rng.integers(0, 131072, M)
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    q_out = torch.empty(M, H, D, dtype=DT[kind], device="cuda")
    t_seq, t_slot, t_table = dev(seq), dev(slot), dev(table)
    e = qkv.element_size()
    more = dict(q_weight=ptr(w[0]), k_weight=ptr(w[1]), eps=1e-5) if norm else {}
    r.quant_append(d, U.dtype_id(in_kind), ptr(qkv), ptr(qkv) + H * D * e, ptr(qkv) + (H + KV) * D * e, H, ptr(dev(pos)), ptr(t_seq),
                   ptr(t_slot), ptr(t_table), M, ptr(q_out), ptr(k), ptr(v), q_row=(H + 2 * KV) * D, k_row=(H + 2 * KV) * D,
                   v_row=(H + 2 * KV) * D, **more)
    x = qkv.double().cpu().numpy().reshape(M, H + 2 * KV, D)
    f, m = frequencies(D, 10000.0)
    q64, k64 = x[:, :H], x[:, H:H + KV]
    if norm:
        q64, k64 = (normed(y, t.double().cpu().numpy(), 1e-5) for y, t in ((q64, w[0]), (k64, w[1])))
    big = max(np.abs(q64).max(), np.abs(k64).max()) * 1.5
    q64, k64 = (rotate(y, pos, f, m, D, True) for y in (q64, k64))
    assert np.abs(q_out.double().cpu().numpy() - q64).max() <= UNIT[kind] * big + 2.0 ** -19 * big
    page_of = table[seq, slot // page]
    kr, vr = (p.cpu().numpy()[page_of, :, slot % page] for p in (k, v))
    # V is quantised as it is: GGUF's blocks to the bit
    for got, want in zip(decode(fmt, vr, D), gguf_blocks(fmt, x[:, H + KV:].astype(np.float32))):
        assert (got == want).all()
    # K to within half a step of its scale (full range / 127 or / 15, kept to 2^-11 of it) and the arithmetic before
    got = values(fmt, kr, D)
    g = k64.reshape(M, KV, D // 32, 32)
    step = np.abs(g).max(-1) / 127 if fmt == "q8" else (g.max(-1) - g.min(-1)) / 15
    most = 127 if fmt == "q8" else 15
    slack = step * (0.5 + most * 2.0 ** -11 + 0.001) + (np.abs(g.min(-1)) * 2.0 ** -11 if fmt == "q4" else 0) + 2.0 ** -18 * big
    assert (np.abs(got.reshape(g.shape) - g) <= slack[..., None]).all()
    # nothing else was written, but what a row does not use
    untouched = np.ones((n_pages, page), bool)
    untouched[page_of, slot % page] = False
    for p in (k, v):
        assert (p.cpu().numpy().transpose(0, 2, 1, 3)[untouched] == 0xA5).all()
    # read back: the values, rounded once
    for to in ("f32", kind):
        ko, vo = (torch.empty(M, KV, D, dtype=DT[to], device="cuda") for _ in range(2))
        tctx.quant_read(d, U.dtype_id(to), ptr(k), ptr(v), ptr(t_table), ptr(t_seq), ptr(t_slot), M, ptr(ko), ptr(vo))
        for o, rows in ((ko, kr), (vo, vr)):
            assert torch.equal(o.cpu(), torch.as_tensor(values(fmt, rows, D, np.float32)).to(DT[to]))
    r.close()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("layout,rot,D", [("interleaved", 64, 64), ("interleaved", 40, 128), ("half", 64, 64), ("half", 256, 256)])
def test_append_layouts_and_rows_at_any_address(tctx, fmt, layout, rot, D):
    """The same rows 16-byte aligned and one element further on give the same bytes, and K their rotation."""
    import ulb_capi as U
    rng = np.random.default_rng(D + rot)
    M, H, KV, page = 19, 3, 2, 32
    x = torch.as_tensor(rng.standard_normal((M, H + 2 * KV, D)), dtype=torch.float32).cuda()
    d = U.QuantDesc(FORMATS[fmt], U.T_F16, KV, D, page, 1, 1, 1)
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout)
    pos, seq, slot, table = dev(rng.integers(0, 9999, M)), dev([0] * M), dev(rng.permutation(page)[:M]), dev([[0]])
    w = dev(rng.uniform(0.5, 1.5, D), torch.float32)
    row, got = (H + 2 * KV) * D, []
    for shift in (0, 1):
        flat = torch.zeros(M * (row + 1) + 8, device="cuda")
        rows = flat[shift:shift + M * (row + shift)].view(M, row + shift)
        rows[:, :row] = x.reshape(M, row)
        k, v = (torch.zeros(1, KV, page, d.row_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
        q_out = torch.zeros(M * H * D + 1, dtype=torch.float16, device="cuda")
        at, n = ptr(rows), (row + shift)
        r.quant_append(d, U.T_F32, at, at + H * D * 4, at + (H + KV) * D * 4, H, ptr(pos), ptr(seq), ptr(slot), ptr(table), M,
                       ptr(q_out) + 2 * shift, ptr(k), ptr(v), q_row=n, k_row=n, v_row=n, k_weight=ptr(w), eps=1e-6)
        got.append((k, v, q_out[shift:shift + M * H * D]))
        KEEP.extend([flat, rows])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    f, m = frequencies(rot, 10000.0)
    x64, half = x.double().cpu().numpy(), layout == "half"
    k64 = rotate(normed(x64[:, H:H + KV], w.double().cpu().numpy(), 1e-6), pos.cpu().numpy(), f, m, rot, half)
    q64 = rotate(x64[:, :H], pos.cpu().numpy(), f, m, rot, half)
    assert np.abs(got[0][2].double().cpu().numpy().reshape(q64.shape) - q64).max() <= (2.0 ** -11 + 2.0 ** -19) * np.abs(q64).max() * 1.5
    val = values(fmt, got[0][0].cpu().numpy()[0].transpose(1, 0, 2)[slot.cpu().numpy()], D).reshape(M, KV, -1, 32)
    g = k64.reshape(val.shape)
    step = np.abs(g).max(-1) / 127 if fmt == "q8" else (g.max(-1) - g.min(-1)) / 15
    most = 127 if fmt == "q8" else 15  # as in the test above
    slack = step * (0.5 + most * 2.0 ** -11 + 0.001) + (np.abs(g.min(-1)) * 2.0 ** -11 if fmt == "q4" else 0) + 2.0 ** -18 * np.abs(k64).max() * 1.5
    assert (np.abs(val - g) <= slack[..., None]).all()
    r.close()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_groups_of_odd_values(tctx, fmt):
    """Zeros, one value throughout, tiny, huge and not finite values, each in a group of its own."""
    import ulb_capi as U
    D, page = 256, 16
    x = np.random.default_rng(1).standard_normal((1, 1, D)).astype(np.float32)
    x[0, 0, 0:32] = 0
    x[0, 0, 32:64] = -2.5
    x[0, 0, 64:96] *= 1e-42
    x[0, 0, 96:128] *= 1e9
    x[0, 0, 130] = np.inf
    x[0, 0, 170] = np.nan
    x[0, 0, 192:224] *= 1e-6
    d = U.QuantDesc(FORMATS[fmt], U.T_F16, 1, D, page, 1, 1, 1)
    k, v = (torch.zeros(1, 1, page, row_bytes(fmt, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    t = torch.as_tensor(x).cuda()
    z, q_out = dev([0]), torch.empty(1, 1, D, dtype=torch.float16, device="cuda")
    r = U.Rope(tctx, D)
    r.quant_append(d, U.T_F32, ptr(t), ptr(t), ptr(t), 1, ptr(z), ptr(z), ptr(z), ptr(z), 1, ptr(q_out), ptr(k), ptr(v))
    got = values(fmt, v.cpu().numpy()[0, :, 0], D)[0]
    assert (got[0:32] == 0).all()
    step = 127 if fmt == "q8" else 1
    assert np.abs(got[32:64] + 2.5).max() <= 2.5 * 2.0 ** -11 * (1 if step == 1 else 1.01)
    assert np.abs(got[64:96]).max() <= 6e-8
    assert np.isfinite(got[96:128]).all() and np.abs(got[96:128]).max() <= 127 * 65504
    assert np.isnan(got[128:160]).all() and np.isnan(got[160:192]).all()
    # scales below 2^-14 are multiples of 2^-24 in 16 bits, so one is off by up to 2^-25 and a code of 127 (15) by as many
    # times that (8 bits: a scale of 2.2e-8 is stored as zero); then the minimum's own 2^-25 and half a step of the codes
    tiny = x[0, 0, 192:224]
    most, half = (127, np.abs(tiny).max() / 254) if fmt == "q8" else (15, (tiny.max() - tiny.min()) / 30)
    assert np.abs(got[192:224] - tiny).max() <= (most + 1) * 2.0 ** -25 + 1.001 * half and np.isfinite(got[224:]).all()
    assert (k == v).all()  # position 0 turns nothing
    r.close()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_rows_without_a_place(tctx, fmt):
    import ulb_capi as U
    D, page, H, KV = 64, 16, 4, 2
    rng = np.random.default_rng(2)
    n_pages, n_seq, max_pages = 4, 2, 2
    table = dev([[3, -1], [9, 0]])
    seq, slot = dev([0, 0, 0, 1, 1, 2, -1, 0, 1]), dev([0, 16, -1, 0, 16, 0, 0, 32, 31])  # 0 0, 1 16 and 1 31 have one
    M = seq.numel()
    qkv = torch.as_tensor(rng.standard_normal((M, (H + 2 * KV) * D)), dtype=torch.float32).cuda()
    d = U.QuantDesc(FORMATS[fmt], U.T_BF16, KV, D, page, n_pages, n_seq, max_pages)
    k, v = (torch.full((n_pages, KV, page, row_bytes(fmt, D)), 0x5A, dtype=torch.uint8, device="cuda") for _ in range(2))
    q_out = torch.zeros(M, H, D, dtype=torch.bfloat16, device="cuda")
    r = U.Rope(tctx, D)
    row = (H + 2 * KV) * D
    args = (d, U.T_F32, ptr(qkv), ptr(qkv) + H * D * 4, ptr(qkv) + (H + KV) * D * 4, H, ptr(dev(np.arange(M))), ptr(seq), ptr(slot), ptr(table))
    r.quant_append(*args, M, ptr(q_out), ptr(k), ptr(v), q_row=row, k_row=row, v_row=row)
    assert (q_out.abs().amax((1, 2)) > 0).all()
    written = np.zeros((n_pages, page), bool)
    for p, at in ((3, 0), (0, 0), (0, 15)):
        written[p, at] = True
    for t in (k, v):
        changed = (t.cpu().numpy().transpose(0, 2, 1, 3) != 0x5A).any((2, 3))
        assert (changed == written).all()
    ko, vo = (torch.full((M, KV, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    tctx.quant_read(d, U.T_BF16, ptr(k), ptr(v), ptr(table), ptr(seq), ptr(slot), M, ptr(ko), ptr(vo))
    has = torch.tensor([True, False, False, False, True, False, False, False, True])
    for o in (ko, vo):
        assert not o.cpu()[~has].any() and (o.cpu()[has].abs().amax((1, 2)) > 0).all()
    # refusals
    good = dict(cache=d, in_dtype=U.T_F32, q=ptr(qkv), k=ptr(qkv), v=ptr(qkv), n_head=H, pos=ptr(seq), row_seq=ptr(seq), slot=ptr(slot),
                block_table=ptr(table), M=M, q_out=ptr(q_out), k_pool=ptr(k), v_pool=ptr(v))
    for bad in (dict(in_dtype=8), dict(n_head=0), dict(M=-1), dict(q=None), dict(q_out=None), dict(slot=None), dict(k_pool=ptr(k) + 8),
                dict(q=ptr(qkv) + 2), dict(row_seq=ptr(seq) + 2), dict(q_row=-8), dict(q_weight=ptr(qkv), eps=0.0), dict(k_weight=ptr(qkv) + 2)):
        refused(r.quant_append, **{**good, **bad})
    for other in (dict(head_dim=128), dict(head_dim=64, rot_dim=32, layout="half")):
        h = U.Rope(tctx, **other)
        refused(h.quant_append, **good)
        h.close()
    r.quant_append(**{**good, "M": 0, "q": None})
    r.close()


# ---------------------------------------------------------------------------------------------- attention over it
def random_pool(rng, fmt, n, KV, page, D):
    """Rows of random codes with ordinary scales."""
    RB = row_bytes(fmt, D)
    rows = rng.integers(0, 256, (n, KV, page, RB), dtype=np.uint8)
    groups = D // 32
    d = (rng.uniform(0.5, 2.0, (n, KV, page, groups)) * (2 / 127 if fmt == "q8" else 0.27)).astype(np.float16)
    if fmt == "q8":
        rows[..., D:D + 2 * groups] = d.view(np.uint8)
    else:
        s = np.stack([d, (-2 * rng.uniform(0.8, 1.2, d.shape)).astype(np.float16)], -1).reshape(n, KV, page, 2 * groups)
        rows[..., D // 2:D // 2 + 4 * groups] = np.ascontiguousarray(s).view(np.uint8)
    return rows


def pools_of(rng, fmt, lens, KV, page, D, unmapped=0.0):
    need = [(x + page - 1) // page for x in lens]
    most = max(1, max(need) + 1)
    n_pages = sum(need) + 1
    order = list(rng.permutation(n_pages))
    table = np.full((len(lens), most), -1, np.int32)
    for s, x in enumerate(need):
        for j in range(x):
            p = order.pop()
            if rng.random() >= unmapped:
                table[s, j] = p
    return random_pool(rng, fmt, n_pages, KV, page, D), random_pool(rng, fmt, n_pages, KV, page, D), table, n_pages, most


def attend64(fmt, q, kp, vp, table, page, D, starts, prefix, lens, bits, scale):
    """Outputs, logarithms, and the sum of the sizes of each output's terms: p d |c|, in 4 bits p (d |c - 8| + |m + 8 d|), over l."""
    R, H, _ = q.shape
    KV = kp.shape[1]
    G = H // KV
    out, lse, mag = np.zeros((R, H, D)), np.full((R, H), -np.inf), np.zeros((R, H, D))
    reach = np.zeros((R, H))
    kv_, vv_ = values(fmt, kp, D), values(fmt, vp, D)
    code, d, m = decode(fmt, vp, D)
    d, m = (np.repeat(x.astype(np.float64), 32, -1) for x in (d, m))
    sizes = np.abs(vv_) if fmt == "q8" else np.abs(d * (code - 8)) + np.abs(m + 8 * d)
    for s, n in enumerate(lens):
        rows = range(starts[s], starts[s + 1])
        at = np.arange(n)
        pg = table[s, at // page] if n else np.zeros(0, np.int32)
        mapped = (pg >= 0) & (pg < kp.shape[0])
        k, v, size = (x[np.where(mapped, pg, 0), :, at % page] for x in (kv_, vv_, sizes))
        for i, r in enumerate(rows):
            if bits is None:
                see = at <= n - len(rows) + i
            else:
                j = at - prefix[s]
                see = (j < 0) | ((j >= 0) & (j < bits.shape[1]) & bits[r][np.clip(j, 0, bits.shape[1] - 1)])
            see = see & mapped
            if not see.any():
                continue
            for h in range(H):
                kk, vv = k[see, h // G], v[see, h // G]
                sc = scale * (kk @ q[r, h])
                mx = sc.max()
                p = np.exp(sc - mx)
                out[r, h] = p @ vv / p.sum()
                mag[r, h] = p @ size[see, h // G] / p.sum()
                lse[r, h] = mx + np.log(p.sum())
                reach[r, h] = scale * (np.abs(kk) @ np.abs(q[r, h])).max()
    return out, lse, mag, reach


def pack_bits(bits):
    w = (bits.shape[1] + 31) // 32
    wide = np.zeros((bits.shape[0], w * 32), np.uint8)
    wide[:, :bits.shape[1]] = bits
    return np.packbits(wide, axis=1, bitorder="little").view(np.int32), w


def run_attention(tctx, fmt, kind, q, kp, vp, table, n_pages, most, page, D, KV, starts, prefix, lens, bits, scale, max_len=None, max_rows=None):
    import ulb_capi as U
    R, H, _ = q.shape
    d = U.QuantDesc(FORMATS[fmt], U.dtype_id(kind), KV, D, page, n_pages, len(lens), most)
    t = [torch.as_tensor(x).cuda() for x in (kp, vp)]
    KEEP.extend(t)
    out = torch.full((R + 1, H, D), 5.0, dtype=DT[kind], device="cuda")
    lse = torch.full((R + 1, H), 5.0, device="cuda")
    words, nw = (None, 0) if bits is None else pack_bits(bits)
    rows = [b - a for a, b in zip(starts, starts[1:])]
    tctx.quant_attention(d, H, R, max(rows) if max_rows is None else max_rows, max(max(lens), 1) if max_len is None else max_len, scale, ptr(q), ptr(t[0]),
                         ptr(t[1]), ptr(dev(table)), ptr(dev(starts)), ptr(dev(prefix)), ptr(dev(lens)), None if words is None else ptr(dev(words)), nw,
                         ptr(out), ptr(lse))
    tctx.sync()
    assert (out[R] == 5).all() and (lse[R] == 5).all()  # the row behind the last sequence
    return out[:R], lse[:R]


def check_attention(kind, got, lse, want, want_lse, mag, reach):
    # weights are rounded once to 2^-11 (a bound for two parts, too), exponentials and fp32 sums are good to 2^-18; a score's products are exact and
    # its sum is off by at most 2^-18 of the sum of their sizes (`reach`); the output is rounded once
    part = 2.0 ** -11 + 2.0 ** -17 + 2 * reach * 2.0 ** -18
    tol = UNIT[kind] * np.abs(want) + part[..., None] * mag + 1e-6
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    assert (np.abs(g - want) <= tol).all(), np.max(np.abs(g - want) / tol)
    ll = lse.double().cpu().numpy()
    empty = want_lse == -np.inf
    assert (ll[empty] == -np.inf).all() and (g[empty] == 0).all()
    assert (np.abs(ll[~empty] - want_lse[~empty]) <= 2.0 ** -17 * np.maximum(1, np.abs(want_lse[~empty])) + reach[~empty] * 2.0 ** -18).all()


CASES = [  # sequences' lengths, rows each, H, KV, D, page
    ([1], [1], 1, 1, 64, 16), ([500], [1], 32, 4, 64, 256), ([33, 1, 0, 700], [1, 1, 1, 1], 8, 2, 128, 32),
    ([5000], [5], 64, 8, 128, 256), ([40, 17, 300], [3, 0, 9], 12, 4, 128, 16), ([2049] * 5, [1] * 5, 5, 5, 128, 128),
    ([1000, 129], [7, 12], 4, 4, 256, 64), ([64], [64], 8, 2, 64, 64), ([3, 2], [8, 4], 4, 1, 128, 16), ([12000], [1], 8, 1, 256, 256),
    ([260] * 70, [1] * 70, 8, 2, 64, 16), ([257, 31], [33, 20], 6, 2, 128, 32), ([130, 40], [3, 1], 64, 1, 64, 32)]


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens,rows,H,KV,D,page", CASES)
def test_quant_attention_causal(tctx, fmt, kind, lens, rows, H, KV, D, page):
    rng = np.random.default_rng(sum(lens) + D)
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D)
    starts = np.concatenate([[0], np.cumsum(rows)]).tolist()
    q = torch.as_tensor(rng.standard_normal((starts[-1], H, D)) * 1.5).to(DT[kind]).cuda()
    scale = 1 / math.sqrt(D)
    got, lse = run_attention(tctx, fmt, kind, q, kp, vp, table, n_pages, most, page, D, KV, starts, [0] * len(lens), lens, None, scale)
    check_attention(kind, got, lse, *attend64(fmt, q.double().cpu().numpy(), kp, vp, table, page, D, starts, None, lens, None, scale))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("nodes,prefix,H,KV,D,page", [(7, 0, 4, 2, 64, 16), (40, 333, 8, 2, 128, 64), (3, 1000, 8, 8, 256, 16), (16, 31, 16, 2, 128, 32),
                                                      (70, 5000, 2, 2, 64, 256)])
def test_quant_attention_of_trees_with_unmapped_pages(tctx, fmt, nodes, prefix, H, KV, D, page):
    rng = np.random.default_rng(nodes)
    lens, starts, pre = [prefix + nodes, prefix // 2 + nodes], [0, nodes, 2 * nodes], [prefix, prefix // 2]
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D, unmapped=0.2)
    bits = rng.random((2 * nodes, nodes)) < 0.3
    bits[0] = False  # sees the prefix only, or nothing
    q = torch.as_tensor(rng.standard_normal((2 * nodes, H, D))).half().cuda()
    got, lse = run_attention(tctx, fmt, "f16", q, kp, vp, table, n_pages, most, page, D, KV, starts, pre, lens, bits, 0.1)
    check_attention("f16", got, lse, *attend64(fmt, q.double().cpu().numpy(), kp, vp, table, page, D, starts, pre, lens, bits, 0.1))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_what_is_not_seen_never_touches_a_result(tctx, fmt):
    """NaN and infinite scales past the end, in slots that a row does not see, and on the page behind the last position."""
    rng = np.random.default_rng(9)
    D, KV, H, page, n = 128, 2, 8, 64, 300
    kp, vp, table, n_pages, most = pools_of(rng, fmt, [n], KV, page, D)
    bits = np.tril(np.ones((6, 6), bool))
    bits[:, 2] = False  # nobody sees slot 2; slot 4 is row 4's and 5's alone
    q = torch.as_tensor(rng.standard_normal((6, H, D))).half().cuda()
    args = (table, n_pages, most, page, D, KV, [0, 6], [n - 6], [n], bits, 0.1)
    want, want_lse = run_attention(tctx, fmt, "f16", q, kp, vp, *args)
    bk, bv = kp.copy(), vp.copy()
    at = D if fmt == "q8" else D // 2
    for pool, odd in ((bk, 0x7E00), (bv, 0x7C00)):
        for pos in (n - 4, n, n + 1, page * (n // page) + page - 1):
            pool[table[0, pos // page], :, pos % page, at:at + 16 if fmt == "q4" else at + 8] = np.frombuffer(np.uint16(odd).tobytes() * (8 if fmt == "q4" else 4), np.uint8)
    got, lse = run_attention(tctx, fmt, "f16", q, bk, bv, *args)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # what some rows see reaches those rows only
    bv[table[0, (n - 2) // page], 0, (n - 2) % page, at:at + 2] = np.frombuffer(np.uint16(0x7E00).tobytes(), np.uint8)
    got, _ = run_attention(tctx, fmt, "f16", q, bk, bv, *args)
    bad = torch.zeros(6, H, D, dtype=torch.bool, device="cuda")
    bad[4:, :H // KV, :32] = True
    assert torch.isnan(got[bad]).all()
    # the other elements of the rows that see the key: its weights are taken against the largest scale that it has left, so the
    # weights of both calls may round differently, each by 2^-11 of a term, and their outputs by half a step
    rest = ~bad
    rest[4:, :H // KV, 32:] = False
    assert torch.equal(got[rest], want[rest])
    mag = attend64(fmt, q.double().cpu().numpy(), kp, vp, table, page, D, [0, 6], [n - 6], [n], bits, 0.1)[2][4:, :H // KV, 32:]
    a, b = (x[4:, :H // KV, 32:].double().cpu().numpy() for x in (got, want))
    assert (np.abs(a - b) <= 2 * 2.0 ** -11 * (mag + np.abs(b))).all()


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("kind,size", [("bf16", 2.0 ** 100), ("bf16", 2.0 ** -100), ("f16", 2.0 ** -14), ("f16", 2.0 ** 12)])
def test_rows_of_any_size_and_scales_of_any_size(tctx, fmt, kind, size):
    """q from 2^-100 to 2^100 with a scale that undoes it; V's scales from 2^-20 to 2^12 among the keys of one row."""
    rng = np.random.default_rng(4)
    D, KV, H, page, n = 64, 1, 4, 16, 200
    kp, vp, table, n_pages, most = pools_of(rng, fmt, [n], KV, page, D)
    groups, at = 2, D if fmt == "q8" else D // 2
    d = (2.0 ** rng.integers(-20, 13, (n_pages, KV, page, groups))).astype(np.float16)
    if fmt == "q8":
        vp[..., at:at + 4] = d.view(np.uint8)
    else:
        vp[..., at:at + 8] = np.stack([d, -d], -1).reshape(n_pages, KV, page, 4).view(np.uint8)
    vp[table[0, 3], :, 5] = 0  # a row of zeros
    q = (torch.as_tensor(rng.standard_normal((1, H, D))) * size).to(DT[kind]).cuda()
    scale = 0.125 / size
    got, lse = run_attention(tctx, fmt, kind, q, kp, vp, table, n_pages, most, page, D, KV, [0, 1], [n], [n], None, scale)
    check_attention(kind, got, lse, *attend64(fmt, q.double().cpu().numpy(), kp, vp, table, page, D, [0, 1], None, [n], None, scale))


def test_quant_attention_bad_contents_of_arrays(tctx):
    """Row ranges, lengths and page ids out of range cost results, never an access: the other sequences keep theirs."""
    rng = np.random.default_rng(11)
    fmt, D, KV, H, page = "q8", 64, 2, 4, 16
    lens = [50, 60, 70]
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D)
    q = torch.as_tensor(rng.standard_normal((3, H, D))).half().cuda()
    base = (n_pages, most, page, D, KV)
    want, want_lse = run_attention(tctx, fmt, "f16", q, kp, vp, table, *base, [0, 1, 2, 3], [0] * 3, lens, None, 0.1)
    t2 = table.copy()
    t2[1] = [n_pages, -5, 1 << 30, -1, 7][:most] + [9999] * max(0, most - 5)
    got, lse = run_attention(tctx, fmt, "f16", q, kp, vp, t2, *base, [0, 1, 2, 3], [-7, 1 << 30, 0], [50, 1 << 30, 70], None, 0.1, max_len=70)
    for i in (0, 2):
        assert torch.equal(got[i], want[i]) and torch.equal(lse[i], want_lse[i])
    got, lse = run_attention(tctx, fmt, "f16", q, kp, vp, table, *base, [-9, 1, 2, 1 << 30], [0] * 3, [50, -4, 70], None, 0.1, max_rows=1)
    assert torch.equal(got[0], want[0]) and not got[1].any() and torch.equal(got[2], want[2])


def test_quant_attention_of_many_sequences(tctx):
    """More sequences than a block has threads, most without rows or keys: those that have some keep their own."""
    rng = np.random.default_rng(13)
    fmt, D, KV, H, page, n_seq = "q4", 64, 2, 4, 16, 1500
    lens = [int(x) if i % 7 == 0 else 0 for i, x in enumerate(rng.integers(0, 90, n_seq))]
    rows = [int(x) for x in rng.integers(0, 3, n_seq) * (rng.random(n_seq) < 0.3)]
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D)
    starts = np.concatenate([[0], np.cumsum(rows)]).tolist()
    q = torch.as_tensor(rng.standard_normal((starts[-1], H, D))).half().cuda()
    got, lse = run_attention(tctx, fmt, "f16", q, kp, vp, table, n_pages, most, page, D, KV, starts, [0] * n_seq, lens, None, 0.1)
    check_attention("f16", got, lse, *attend64(fmt, q.double().cpu().numpy(), kp, vp, table, page, D, starts, None, lens, None, 0.1))


@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_pools_past_two_gigabytes(tctx, fmt):
    """Rows written, read and attended on pages whose bytes begin past 2^31."""
    import ulb_capi as U
    rng = np.random.default_rng(14)
    D, KV, H, page, n = 128, 8, 16, 256, 300
    d = U.QuantDesc(FORMATS[fmt], U.T_F16, KV, D, page, 1, 1, 2)
    d.n_pages = n_pages = 2 ** 31 // (KV * page * d.row_bytes) + 3
    table = dev([[n_pages - 1, n_pages - 2]])
    k, v = (torch.empty(n_pages, KV, page, d.row_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    row = (H + 2 * KV) * D
    x = torch.as_tensor(rng.standard_normal((n, row))).half().cuda()
    seq, slot, z = dev([0] * n), dev(np.arange(n)), dev([0])
    q = torch.empty(n, H, D, dtype=torch.float16, device="cuda")
    r = U.Rope(tctx, D)
    r.quant_append(d, U.T_F16, ptr(x), ptr(x) + H * D * 2, ptr(x) + (H + KV) * D * 2, H, ptr(slot), ptr(seq), ptr(slot), ptr(table), n, ptr(q), ptr(k),
                   ptr(v), q_row=row, k_row=row, v_row=row)
    tail = [t[-2:].cpu().numpy() for t in (k, v)]
    o = [torch.empty(n, KV, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    tctx.quant_read(d, U.T_F16, ptr(k), ptr(v), ptr(table), ptr(seq), ptr(slot), n, ptr(o[0]), ptr(o[1]))
    at = np.arange(n)
    for got, t in zip(o, tail):
        assert torch.equal(got.cpu(), torch.as_tensor(values(fmt, t[1 - at // page, :, at % page], D, np.float32)).half())
    out, lse = torch.empty(1, H, D, dtype=torch.float16, device="cuda"), torch.empty(1, H, device="cuda")
    tctx.quant_attention(d, H, 1, 1, n, 0.1, ptr(q) + (n - 1) * H * D * 2, ptr(k), ptr(v), ptr(table), ptr(dev([0, 1])), ptr(z), ptr(dev([n])), None, 0,
                         ptr(out), ptr(lse))
    check_attention("f16", out, lse, *attend64(fmt, q[n - 1:].double().cpu().numpy(), *tail, np.array([[1, 0]]), page, D, [0, 1], None, [n], None, 0.1))
    r.close()


def test_quant_attention_captured_in_two_graphs_on_another_stream(tctx):
    import ulb_capi as U
    rng = np.random.default_rng(12)
    fmt, D, KV, H, page, lens = "q4", 128, 8, 32, 64, [9000, 40]
    kp, vp, table, n_pages, most = pools_of(rng, fmt, lens, KV, page, D)
    q = torch.as_tensor(rng.standard_normal((2, H, D))).bfloat16().cuda()
    want, want_lse = run_attention(tctx, fmt, "bf16", q, kp, vp, table, n_pages, most, page, D, KV, [0, 1, 2], [0, 0], lens, None, 0.1)
    d = U.QuantDesc(FORMATS[fmt], U.T_BF16, KV, D, page, n_pages, 2, most)
    t = [torch.as_tensor(x).cuda() for x in (kp, vp)]
    a = [dev(table), dev([0, 1, 2]), dev([0, 0]), dev(lens)]
    outs = [torch.zeros_like(want) for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    tctx.use_stream(side.cuda_stream)
    graphs = [tctx.capture(lambda o=o: tctx.quant_attention(d, H, 2, 1, 9000, 0.1, ptr(q), ptr(t[0]), ptr(t[1]), *map(ptr, a), None, 0, ptr(o))) for o in outs]
    for _ in range(3):
        for g in graphs:
            U.check(U.lib().ulb_graph_launch(tctx.h, g))
    tctx.sync()
    for o in outs:
        assert torch.equal(o, want)
    for g in graphs:
        U.lib().ulb_graph_free(g)
    tctx.use_stream(torch.cuda.current_stream().cuda_stream)


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("fmt", ["q8", "q4"])
def test_a_sequence_step_by_step_with_the_page_book(tctx, fmt):
    """A prompt appended and attended as a prompt, forked, extended by chains of drafts, compacted and rolled back on a
    quantised cache: every step's attention equals the 64-bit one over what the cache holds."""
    import ulb_capi as U
    rng = np.random.default_rng(21)
    H, KV, D, page, kind = 8, 2, 128, 16, "bf16"
    n_pages, n_seq, max_pages = 40, 3, 12
    d = U.QuantDesc(FORMATS[fmt], U.dtype_id(kind), KV, D, page, n_pages, n_seq, max_pages)
    k, v = (torch.zeros(n_pages, KV, page, d.row_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    view = d.pages_view()
    book = U.Pages(tctx, view, ptr(k), ptr(v))
    r = U.Rope(tctx, D, layout="half")
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    row = (H + 2 * KV) * D

    def append(seq, slot, pos):
        M = len(seq)
        x = torch.as_tensor(rng.standard_normal((M, row))).to(DT[kind]).cuda()
        q = torch.empty(M, H, D, dtype=DT[kind], device="cuda")
        r.quant_append(d, U.dtype_id(kind), ptr(x), ptr(x) + H * D * 2, ptr(x) + (H + KV) * D * 2, H, ptr(dev(pos)), ptr(dev(seq)),
                       ptr(dev(slot)), book.table, M, ptr(q), ptr(k), ptr(v), q_row=row, k_row=row, v_row=row, q_weight=ptr(w[0]),
                       k_weight=ptr(w[1]), eps=1e-6)
        KEEP.append(x)
        return q, x

    def host_table():
        t = np.empty((n_seq, max_pages), np.int32)
        torch.cuda.synchronize()
        U.check(U.lib().ulb_memcpy_d2h(tctx.h, U._ptr(t), book.table, t.nbytes))
        return t

    def attend(q, starts, lens):
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        n = [b - a for a, b in zip(starts, starts[1:])]
        tctx.quant_attention(d, H, q.shape[0], max(n), max(lens), 0.09, ptr(q), ptr(k), ptr(v), book.table, ptr(dev(starts)),
                             ptr(dev([0] * n_seq)), ptr(dev(lens)), None, 0, ptr(out), ptr(lse))
        check_attention(kind, out, lse, *attend64(fmt, q.double().cpu().numpy(), k.cpu().numpy(), v.cpu().numpy(), host_table(), page, D,
                                                  starts, None, lens, None, 0.09))

    book.reserve(0, 0, 37)
    q, x = append([0] * 37, range(37), range(37))
    # the prompt itself is attended as it is, before it is quantised
    ko = torch.empty(37, KV, D, dtype=DT[kind], device="cuda")
    vo = torch.empty_like(ko)
    tctx.quant_read(d, U.dtype_id(kind), ptr(k), ptr(v), book.table, ptr(dev([0] * 37)), ptr(dev(range(37))), 37, ptr(ko), ptr(vo))
    out = torch.empty_like(q)
    tctx.prompt_attention(U.dtype_id(kind), H, KV, D, 1, 37, 37, 37, 37, 0.09, ptr(q), ptr(ko), ptr(vo), ptr(dev([0, 37])), ptr(dev([0, 37])), ptr(out))
    attend(q, [0, 37, 37, 37], [37, 0, 0])
    book.fork(0, 1, 37)
    book.fork(0, 2, 20)
    for s, n in ((0, 37), (1, 37), (2, 20)):
        book.reserve(s, n, n + 4)
    seq = np.repeat([0, 1, 2], 4)
    slot = np.concatenate([np.arange(37, 41), np.arange(37, 41), np.arange(20, 24)])
    q, _ = append(seq, slot, slot)
    attend(q, [0, 4, 8, 12], [41, 41, 24])
    before = k.cpu().numpy(), v.cpu().numpy(), host_table()
    # drafts 0 and 3 of sequence 0, 2 of sequence 1 accepted
    tctx.pages_compact(view, ptr(k), ptr(v), book.table, ptr(dev([37, 37, 20])), ptr(dev([2, 1, 0])), ptr(dev([[0, 3, 0], [2, 0, 0], [0, 0, 0]])), 3)
    now, t = k.cpu().numpy(), host_table()
    for s, to, fro in ((0, 37, 37), (0, 38, 40), (1, 37, 39)):
        assert (now[t[s, to // page], :, to % page] == before[0][t[s, fro // page], :, fro % page]).all()
    for s, n in ((0, 39), (1, 38), (2, 20)):
        book.truncate(s, n)
        book.reserve(s, n, n + 1)
    book.defrag()
    q, _ = append([0, 1, 2], [39, 38, 20], [39, 38, 20])
    attend(q, [0, 1, 2, 3], [40, 39, 21])
    book.close()
    r.close()
