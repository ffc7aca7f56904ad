"""A prompt written to the quantised cache in chunks: what is cached is read back and attended as a prompt, with the outputs
checked, and by the cache's own attention; handles that scale.  Tolerances are stated where they are used."""
import math

import numpy as np
import pytest

from test_gpu_paged_ops import DT, KEEP, UNIT, dev, frequencies, kept, ptr, rotate, tctx  # noqa: F401
from test_gpu_prompt_attention import attend64 as prompt64, check as check_prompt
from test_gpu_quant_ops import FORMATS, attend64, check_attention, normed, values

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HANDLES = [({}, 1.0), (dict(scaling="yarn", factor=4.0, orig_len=4096), None), (dict(attn_scale=0.3), 0.3)]


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("layout,rot", [("half", 128), ("interleaved", 128), ("interleaved", 48)])
@pytest.mark.parametrize("more,factor", HANDLES)
def test_a_chunk_over_what_is_cached(tctx, fmt, layout, rot, more, factor):
    import ulb_capi as U
    rng = np.random.default_rng(rot + len(more))
    H, KV, D, page, kind, n, last = 8, 2, 128, 32, "bf16", 300, 41
    half, scale = layout == "half", 0.09
    f, m = frequencies(rot, 10000.0, scaling=more.get("scaling", "none"), factor=more.get("factor", 1.0))
    m = m if factor is None else factor
    max_pages = n_pages = (n + page - 1) // page + 1
    d = U.QuantDesc(FORMATS[fmt], U.dtype_id(kind), KV, D, page, n_pages, 1, max_pages)
    table = dev([rng.permutation(n_pages)])
    kp, vp = (torch.zeros(n_pages, KV, page, d.row_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    r = U.Rope(tctx, D, rot_dim=rot, layout=layout, **more)
    w = [dev(rng.uniform(0.5, 1.5, D), torch.float32) for _ in range(2)]
    row = (H + 2 * KV) * D
    x = torch.as_tensor(rng.standard_normal((n, row))).to(DT[kind]).cuda()
    q = torch.empty(n, H, D, dtype=DT[kind], device="cuda")
    seq, slot = dev([0] * n), dev(np.arange(n))
    pos = np.arange(n) + 1000
    at = dev(pos)
    for a, b in ((0, 100), (100, n - last), (n - last, n)):  # chunk by chunk
        p = ptr(x) + a * row * 2
        r.quant_append(d, U.dtype_id(kind), p, p + H * D * 2, p + (H + KV) * D * 2, H, ptr(at) + a * 4, ptr(seq) + a * 4, ptr(slot) + a * 4,
                       ptr(table), b - a, ptr(q) + a * H * D * 2, ptr(kp), ptr(vp), q_row=row, k_row=row, v_row=row, q_weight=ptr(w[0]),
                       k_weight=ptr(w[1]), eps=1e-6)
    # q and K: normed, turned, the factor on what turns
    x64 = x.double().cpu().numpy().reshape(n, H + 2 * KV, D)

    def turned(y, weight):
        y = normed(y, weight.double().cpu().numpy(), 1e-6)
        z = rotate(y, pos, f, m, rot, half)
        z[..., rot:] = y[..., rot:]
        return z

    q64, k64 = turned(x64[:, :H], w[0]), turned(x64[:, H:H + KV], w[1])
    big = 1.5 * max(np.abs(q64).max(), np.abs(k64).max()) * max(1.0, 1 / m)
    assert np.abs(q.double().cpu().numpy() - q64).max() <= (UNIT[kind] + 2.0 ** -19) * big
    pages = table.cpu().numpy()[0, np.arange(n) // page]
    cached = [values(fmt, t.cpu().numpy()[pages, :, np.arange(n) % page], D) for t in (kp, vp)]
    # K to within half a step of its group's scale (kept to 2^-11 of it, a code is at most 127 or 15 of them), the minimum's
    # 2^-11, and the arithmetic before
    g = k64.reshape(n, KV, D // 32, 32)
    most = 127 if fmt == "q8" else 15
    step = np.abs(g).max(-1) / 127 if fmt == "q8" else (g.max(-1) - g.min(-1)) / 15
    slack = step * (0.5 + most * 2.0 ** -11 + 0.001) + (np.abs(g.min(-1)) * 2.0 ** -11 if fmt == "q4" else 0) + 2.0 ** -18 * big
    assert (np.abs(cached[0].reshape(g.shape) - g) <= slack[..., None]).all()
    # all of it read back, the last chunk attended as a prompt
    ko, vo = (torch.empty(n, KV, D, dtype=DT[kind], device="cuda") for _ in range(2))
    tctx.quant_read(d, U.dtype_id(kind), ptr(kp), ptr(vp), ptr(table), ptr(seq), ptr(slot), n, ptr(ko), ptr(vo))
    for o, c in zip((ko, vo), cached):
        assert torch.equal(o.cpu(), torch.as_tensor(c.astype(np.float32)).to(DT[kind]))
    rows = q[n - last:]
    out, lse = torch.empty_like(rows), torch.empty(last, H, device="cuda")
    tctx.prompt_attention(U.dtype_id(kind), H, KV, D, 1, last, n, last, n, scale, ptr(rows), ptr(ko), ptr(vo), ptr(dev([0, last])), ptr(dev([0, n])),
                          ptr(out), ptr(lse))
    check_prompt(kind, out, lse, *prompt64(rows, ko, vo, [0, last], [0, n], scale))
    # and by the cache's attention, as a chain of the same rows
    out2, lse2 = torch.empty_like(rows), torch.empty_like(lse)
    tctx.quant_attention(d, H, last, last, n, scale, ptr(rows), ptr(kp), ptr(vp), ptr(table), ptr(dev([0, last])), ptr(dev([0])), ptr(dev([n])), None, 0,
                         ptr(out2), ptr(lse2))
    check_attention(kind, out2, lse2, *attend64(fmt, rows.double().cpu().numpy(), kp.cpu().numpy(), vp.cpu().numpy(), table.cpu().numpy(), page, D,
                                                [0, last], None, [n], None, scale))
    r.close()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_whole_prompt_from_the_cache(tctx, D):
    """The rows of a prompt attended over what the cache gives back of all of them: the first row sees itself only."""
    import ulb_capi as U
    rng = np.random.default_rng(D)
    H, KV, page, kind, n = 4, 2, 16, "f16", 37
    d = U.QuantDesc(FORMATS["q8"], U.T_F16, KV, D, page, 3, 1, 3)
    kp, vp = (torch.zeros(3, KV, page, d.row_bytes, dtype=torch.uint8, device="cuda") for _ in range(2))
    r = U.Rope(tctx, D, layout="half")
    row = (H + 2 * KV) * D
    x = torch.as_tensor(rng.standard_normal((n, row))).half().cuda()
    q = torch.empty(n, H, D, dtype=torch.float16, device="cuda")
    seq, slot, table = dev([0] * n), dev(np.arange(n)), dev([[2, 0, 1]])
    r.quant_append(d, U.T_F16, ptr(x), ptr(x) + H * D * 2, ptr(x) + (H + KV) * D * 2, H, ptr(slot), ptr(seq), ptr(slot), ptr(table), n, ptr(q), ptr(kp),
                   ptr(vp), q_row=row, k_row=row, v_row=row)
    ko, vo = (torch.empty(n, KV, D, dtype=torch.float16, device="cuda") for _ in range(2))
    tctx.quant_read(d, U.T_F16, ptr(kp), ptr(vp), ptr(table), ptr(seq), ptr(slot), n, ptr(ko), ptr(vo))
    out, lse = torch.empty_like(q), torch.empty(n, H, device="cuda")
    scale = 1 / math.sqrt(D)
    tctx.prompt_attention(U.T_F16, H, KV, D, 1, n, n, n, n, scale, ptr(q), ptr(ko), ptr(vo), ptr(dev([0, n])), ptr(dev([0, n])), ptr(out), ptr(lse))
    check_prompt(kind, out, lse, *prompt64(q, ko, vo, [0, n], [0, n], scale))
    assert torch.equal(out[0], vo[0].repeat_interleave(H // KV, 0))
    r.close()
