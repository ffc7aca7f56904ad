"""Timed cases of the operators around an attention whose cache is held in 8 or 4 bits.

A layer of such a model normalises its q and k heads and turns them to their positions ("norm", its
backward pass "norm_grad"), writes K and V to the pages of a cache as Q8_0 or Q4_1 blocks and reads
them back for a later chunk of the prompt ("store"), attends the new tokens of every sequence over those
pages ("decode"), and attends whole prompts, packed one behind the other, causally ("prompt").

`own` picks the side that run() takes: False, elementary torch operations in 32 bits rounded once at
the end; True, the framework's entry points.  exact() is the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- cases
def _norm(name, op, rows, heads, kv, dim, rot, layout, kind, far=16384):
    return dict(name=name, op=op, rows=rows, heads=heads, kv=kv, dim=dim, rot=rot, layout=layout, kind=kind, far=far)


def _store(name, seqs, rows, heads, kv, dim, layout, bits, kind, page, normed):
    return dict(name=name, op="store", seqs=seqs, rows=rows, heads=heads, kv=kv, dim=dim, rot=dim, layout=layout, bits=bits,
                kind=kind, page=page, normed=normed, far=32768)


def _decode(name, seqs, rows, low, high, heads, kv, dim, bits, kind, page):
    return dict(name=name, op="decode", seqs=seqs, rows=rows, low=low, high=high, heads=heads, kv=kv, dim=dim, bits=bits,
                kind=kind, page=page)


def _prompt(name, seqs, low, high, before, heads, kv, dim, kind):
    return dict(name=name, op="prompt", seqs=seqs, low=low, high=high, before=before, heads=heads, kv=kv, dim=dim, kind=kind)


def listed():
    return [
        # q and k of one step of eight sequences: only latency counts
        _norm("norm 8 rows", "norm", 8, 32, 4, 64, 64, "half", "f16"),
        # q and k of a fine-tuning batch, forward; an odd number of rows
        _norm("norm 16381 rows", "norm", 16381, 32, 8, 128, 128, "half", "bf16"),
        # their gradients and those of the two weights, half of a head turned, a small batch in 32 bits
        _norm("gradient 1000 rows", "norm_grad", 1000, 32, 8, 128, 64, "interleaved", "f32"),
        # the gradients of the batch above
        _norm("gradient 16381 rows", "norm_grad", 16381, 32, 8, 128, 128, "half", "bf16"),
        # one new token of each of 64 sequences written to the cache and looked at again: latency
        _store("store 64 rows q8", 64, 64, 32, 8, 128, "half", 8, "bf16", 64, True),
        # three prompts written in 4 bits and read back for their next chunk
        _store("store 8190 rows q4", 3, 8190, 32, 8, 128, "interleaved", 4, "f16", 256, False),
        # one token of one sequence in a short context: latency
        _decode("decode 1 token q8", 1, 1, 500, 500, 32, 4, 64, 8, "f16", 256),
        # a serving batch of 64 sequences of ragged lengths, 4 bits
        _decode("decode 64 sequences q4", 64, 1, 256, 8192, 32, 8, 128, 4, "bf16", 64),
        # one long context and a chain of five drafts, 8 bits
        _decode("decode 100001 keys q8", 1, 5, 100001, 100001, 64, 8, 128, 8, "bf16", 256),
        # a short prompt: latency
        _prompt("prompt 500 tokens", 1, 500, 500, 0, 32, 4, 64, "f16"),
        # the next 513 tokens of a long prompt whose first 30000 are in the cache
        _prompt("prompt 513 after 30000", 1, 513, 513, 30000, 32, 8, 128, "bf16"),
        # the largest: four prompts of different lengths packed into one call
        _prompt("prompt 4 packed", 4, 1500, 6001, 0, 32, 8, 128, "bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "store", "decode", "decode", "prompt", "prompt"])
    kind = rng.choice(["f16", "bf16"])
    heads, kv = rng.choice([(32, 32), (32, 8), (32, 4), (64, 8), (8, 2), (5, 5), (12, 4)])
    dim = rng.choice([64, 64, 128, 128, 256])
    layout = rng.choice(["interleaved", "half"])
    if op in ("norm", "norm_grad"):
        dim = rng.choice([dim, dim, 80, 96])
        c = _norm("", op, _log(rng, 1, 16000), heads, kv, dim, rng.choice([dim, dim, 32]), layout, rng.choice(["f32", kind]),
                  rng.choice([4096, 131072]))
        c["rows"] = max(1, min(c["rows"], int(6e7 / ((heads + kv) * dim))))
    elif op == "store":
        c = _store("", _log(rng, 1, 64), _log(rng, 1, 8000), heads, kv, dim, layout, rng.choice([4, 8]), kind,
                   rng.choice([16, 32, 64, 128, 256]), rng.random() < 0.5)
        c["rows"] = max(1, min(c["rows"], int(3e7 / ((heads + 2 * kv) * dim))))
        c["seqs"] = min(c["seqs"], c["rows"])
    elif op == "decode":
        seqs, rows, high = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 9]), _log(rng, 8, 100000)
        c = _decode("", seqs, rows, max(1, high // rng.choice([1, 2, 16])), high, heads, kv, dim, rng.choice([4, 8]), kind,
                    rng.choice([16, 32, 64, 128, 256]))
        while c["seqs"] * (c["high"] + 300) * kv * dim > 2.5e8 or c["seqs"] * c["rows"] * c["high"] * heads > 2e8:
            big = "seqs" if c["seqs"] > 1 and c["seqs"] * 500 > c["high"] else "high"
            c[big] = max(1, c[big] // 2)
            c["low"] = min(c["low"], c["high"])
    else:
        dim = rng.choice([64, 128, dim, 80, 96])
        high = _log(rng, 1, 6000)
        c = _prompt("", _log(rng, 1, 16), max(1, high // rng.choice([1, 2, 8])), high, rng.choice([0, 0, _log(rng, 1, 20000)]), heads,
                    kv, dim, kind)
        while c["seqs"] * heads * c["high"] * (c["high"] + c["before"]) * dim > 3e11:
            big = "seqs" if c["seqs"] > 2 else "before" if c["before"] > 2 * c["high"] else "high"
            c[big] = max(1, c[big] // 2)
            c["low"] = min(c["low"], c["high"])
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------- inputs
def _row_bytes(c):
    """Bytes of a position's head in the pool: codes, then the scales of its groups of 32, in 16-byte steps."""
    used = c["dim"] + c["dim"] // 16 if c["bits"] == 8 else c["dim"] // 2 + c["dim"] // 8
    return (used + 15) // 16 * 16


def _table(r, pages_of, most):
    """Pages of each sequence in random order: int32 [seqs][most], -1 where none is mapped."""
    total = sum(pages_of)
    order = torch.randperm(total, generator=r).to(torch.int32)
    t = torch.full((len(pages_of), most), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(pages_of):
        t[s, :n] = order[at:at + n]
        at += n
    return t, total


def _lengths(c):
    """Rows of each prompt of a case: the longest first, the others spread between both bounds."""
    return [c["high"] - int((c["high"] - c["low"] + 1) * (i * 0.618 % 1.0)) for i in range(c["seqs"])]


def _starts(sizes):
    at = [0]
    for n in sizes:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    c, dev = case, "cuda"
    r = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=dev).manual_seed(seed)
    h, kv, d = c["heads"], c["kv"], c["dim"]

    def normal(*shape, kind="f32", scale=1.0):
        return (torch.randn(shape, device=dev, generator=g) * scale).to(TYPES[kind])

    def ints(v):
        return torch.as_tensor(v).to(torch.int32).to(dev)

    def weight():  # around one, as trained norms are
        return torch.rand(d, device=dev, generator=g) + 0.5

    def sizes(low, high):
        return [high] + [int(torch.randint(low, high + 1, (1,), generator=r)) for _ in range(c["seqs"] - 1)]

    s = {"case": c}
    if c["op"] in ("norm", "norm_grad"):
        m, kind = c["rows"], c["kind"]
        # rows as the projection leaves them: q, k and v heads side by side
        s.update(qkv=normal(m, h + 2 * kv, d, kind=kind, scale=2.0), wq=weight(), wk=weight(),
                 pos=ints(torch.randint(0, c["far"], (m,), generator=r)),
                 q_out=torch.empty(m, h, d, dtype=TYPES[kind], device=dev), k_out=torch.empty(m, kv, d, dtype=TYPES[kind], device=dev))
        if c["op"] == "norm_grad":
            s.update(dq=normal(m, h, d, kind=kind), dk=normal(m, kv, d, kind=kind), dwq=torch.empty(d, device=dev),
                     dwk=torch.empty(d, device=dev))
    elif c["op"] == "store":
        m, seqs = c["rows"], c["seqs"]
        deep = (m + seqs - 1) // seqs
        base = torch.randint(0, 3 * c["page"], (seqs,), generator=r)
        most = (3 * c["page"] + deep + c["page"] - 1) // c["page"]
        table, n = _table(r, [most] * seqs, most)
        seq = torch.arange(m) % seqs
        s.update(qkv=normal(m, h + 2 * kv, d, kind=c["kind"], scale=2.0), wq=weight(), wk=weight(),
                 pos=ints(torch.randint(0, c["far"], (m,), generator=r)), row_seq=ints(seq),
                 slot=ints(base[seq] + torch.arange(m) // seqs), table=ints(table),
                 k=torch.zeros(n, kv, c["page"], _row_bytes(c), dtype=torch.uint8, device=dev),
                 v=torch.zeros(n, kv, c["page"], _row_bytes(c), dtype=torch.uint8, device=dev),
                 q_out=torch.empty(m, h, d, dtype=TYPES[c["kind"]], device=dev),
                 k_out=torch.empty(m, kv, d, dtype=TYPES[c["kind"]], device=dev),
                 v_out=torch.empty(m, kv, d, dtype=TYPES[c["kind"]], device=dev))
    elif c["op"] == "decode":
        n_row, page = c["rows"], c["page"]
        length = [x + n_row for x in sizes(c["low"], c["high"])]
        most = (max(length) + page - 1) // page
        table, n = _table(r, [(x + page - 1) // page for x in length], most)
        start = [i * n_row for i in range(c["seqs"] + 1)]
        k, v = (torch.empty(n, kv, page, _row_bytes(c), dtype=torch.uint8, device=dev) for _ in range(2))
        for pool in (k, v):  # written in parts: the unpacked values are larger than the pool
            for p in range(0, n, 512):
                part = pool[p:p + 512]
                part.copy_(_pack(c, *_quantise(c, normal(part.shape[0], kv, page, d))))
        s.update(k=k, v=v, table=ints(table), start=ints(start), length=ints(length), max_len=max(length),
                 prefix=ints([x - n_row for x in length]),
                 q=normal(c["seqs"] * n_row, h, d, kind=c["kind"], scale=1.5),
                 out=torch.empty(c["seqs"] * n_row, h, d, dtype=TYPES[c["kind"]], device=dev),
                 lse=torch.empty(c["seqs"] * n_row, h, device=dev))
    else:
        rows = _lengths(c)
        keys = [n + c["before"] for n in rows]
        s.update(rows=sum(rows), keys=sum(keys), max_rows=max(rows), max_keys=max(keys), q_start=ints(_starts(rows)),
                 k_start=ints(_starts(keys)), q=normal(sum(rows), h, d, kind=c["kind"], scale=1.5),
                 k=normal(sum(keys), kv, d, kind=c["kind"]), v=normal(sum(keys), kv, d, kind=c["kind"]),
                 out=torch.empty(sum(rows), h, d, dtype=TYPES[c["kind"]], device=dev), lse=torch.empty(sum(rows), h, device=dev))
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _turns(c, pos):
    """Cosines and sines of each row's pairs; the angles alone need 64 bits."""
    base = 1e4 if c["dim"] == 64 else 5e5
    w = base ** (-2.0 * torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda") / c["rot"])
    angle = pos.double()[:, None, None] * w
    return angle.cos().float(), angle.sin().float()


def _halves(c, x):
    rot = c["rot"]
    return (x[..., :rot:2], x[..., 1:rot:2]) if c["layout"] == "interleaved" else (x[..., :rot // 2], x[..., rot // 2:rot])


def _turn(c, x, co, si):
    out = x.clone()
    a, b = _halves(c, x)
    first, second = _halves(c, out)
    first.copy_(a * co - b * si)
    second.copy_(a * si + b * co)
    return out


def _scaled(x):
    """x and the factor that norms each head: 1 / sqrt(mean x^2 + eps)."""
    x = x.float()
    return x, torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_norm(c, x, w, co, si):
    x, f = _scaled(x)
    return _turn(c, x * f * w, co, si)


def _plain_norm_grad(c, x, w, co, si, dy):
    x, f = _scaled(x)
    g, n = _turn(c, dy.float(), co, -si), x * f
    gw = g * w
    dx = f * (gw - n * (gw * n).mean(-1, keepdim=True))
    return dx.to(dy.dtype), (g * n).sum((0, 1), dtype=torch.float64).float()


def _quantise(c, x):
    """Q8_0 or Q4_1 blocks of 32 values: codes, scales and minima (None in 8 bits), the last two in 16 bits.  Codes next to
    a border go by these very operations, which are the formats' own (a quotient, not a product with 1 / 127)."""
    x = x.float().unflatten(-1, (-1, 32))
    if c["bits"] == 8:
        d = x.abs().amax(-1, keepdim=True)
        d = d / torch.full_like(d, 127.0)
        y = x * torch.where(d == 0, 0.0, 1.0 / d)
        return torch.copysign((y.abs() + 0.5).floor(), y).clamp(-127, 127).to(torch.int8), d.half(), None
    low = x.amin(-1, keepdim=True)
    d = (x.amax(-1, keepdim=True) - low) / torch.full_like(low, 15.0)
    y = (x - low) * torch.where(d == 0, 0.0, 1.0 / d)
    return (y + 0.5).floor().clamp(0, 15).to(torch.uint8), d.half(), low.half()


def _pack(c, code, d, low):
    """Rows of the pool.  8 bits: the codes in order.  4 bits: word i of each 32 bytes holds elements 4 i .. 4 i + 3 of two
    neighbouring groups, the first's at bits 0, 16, 4, 20, the second's at 8, 24, 12, 28.  Then the groups' scales (4 bits:
    scale and minimum in turn) in 16 bits, then zeros."""
    if c["bits"] == 8:
        parts = [code.flatten(-2).view(torch.uint8), d.flatten(-2).view(torch.uint8)]
    else:
        x = code.unflatten(-2, (-1, 2)).unflatten(-1, (8, 4)).movedim(-3, -2)  # [..., two groups' pairs, word, group, element]
        low_bits, high_bits = x[..., (0, 1), :][..., (0, 1)], x[..., (2, 3)]  # bytes 0, 2 hold elements 0 | 2 and 1 | 3
        both = low_bits | (high_bits << 4)  # [..., word, group, 2]: the bytes of group g at places g and g + 2
        parts = [both.transpose(-1, -2).flatten(-4), torch.cat([d, low], -1).flatten(-2).contiguous().view(torch.uint8)]
    row = torch.cat(parts, -1)
    return torch.nn.functional.pad(row, (0, _row_bytes(c) - row.shape[-1]))


def _unpack(c, row):
    """The values that rows of the pool stand for, in 32 bits."""
    d = c["dim"]
    if c["bits"] == 8:
        code = row[..., :d].contiguous().view(torch.int8).unflatten(-1, (-1, 32))
        return (code.float() * row[..., d:d + d // 16].contiguous().view(torch.float16).float()[..., None]).flatten(-2)
    both = row[..., :d // 2].unflatten(-1, (-1, 8, 2, 2)).transpose(-1, -2)  # [..., pair, word, group, 2]
    code = torch.cat([both & 15, both >> 4], -1).movedim(-2, -3).flatten(-2).flatten(-3, -2)
    scale = row[..., d // 2:d // 2 + d // 8].contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))
    return (code.float() * scale[..., :1] + scale[..., 1:]).flatten(-2)


def _heads_of(s):
    """The q, k and v heads of the rows."""
    c = s["case"]
    return s["qkv"].split([c["heads"], c["kv"], c["kv"]], 1)


def _plain_store(s):
    c, kind = s["case"], TYPES[s["case"]["kind"]]
    q, k, v = _heads_of(s)
    co, si = _turns(c, s["pos"])
    q, k = (_plain_norm(c, x, w, co, si) if c["normed"] else _turn(c, x.float(), co, si) for x, w in ((q, s["wq"]), (k, s["wk"])))
    slot = s["slot"].long()
    page, at = s["table"][s["row_seq"].long(), slot // c["page"]].long(), slot % c["page"]
    s["k"][page, :, at] = _pack(c, *_quantise(c, k))
    s["v"][page, :, at] = _pack(c, *_quantise(c, v))
    return q.to(kind), _unpack(c, s["k"][page, :, at]).to(kind), _unpack(c, s["v"][page, :, at]).to(kind)


def _softmax(scores, vals):
    """Weighted sums and logarithms of the weights' sums; scores are -inf where nothing is seen."""
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    return (scores @ vals) / total.clamp(min=1e-38), (top + total.log()).squeeze(-1)


def _of_row(start, rows):
    """The sequence of each row, and its place in it."""
    n = (start[1:] - start[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(n.numel(), device=start.device), n, output_size=rows)
    return seq, torch.arange(rows, device=start.device) - start[seq]


def _plain_attend(s, q, keys, vals, q_len, k_len, seq, row):
    """q [b][rows][h][d] over keys, vals [b][kv][wide][d]: row i of n sees the keys up to its own, the last of them for the last row."""
    c = s["case"]
    b, h, kv, d = q.shape[0], c["heads"], c["kv"], c["dim"]
    group, n, wide = h // kv, q.shape[1], keys.shape[2]
    q = q.view(b, n, kv, group, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    scores = (q @ keys.transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    last = (k_len - q_len)[:, None] + torch.arange(n, device="cuda")
    hide = torch.arange(wide, device="cuda") > last[:, :, None]
    scores.view(b, kv, group, n, wide).masked_fill_(hide[:, None, None], -math.inf)
    out, lse = _softmax(scores, vals)
    out = out.view(b, kv, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d)[seq, row].to(TYPES[c["kind"]])
    return out, lse.view(b, kv, group, n).permute(0, 3, 1, 2).reshape(b, n, h)[seq, row]


def _plain_decode(s):
    c = s["case"]
    table = s["table"].clamp(min=0).long()
    keys, vals = (_unpack(c, p[table]).permute(0, 2, 1, 3, 4).flatten(2, 3) for p in (s["k"], s["v"]))
    seq, row = _of_row(s["start"], s["q"].shape[0])
    q = s["q"].float().view(c["seqs"], c["rows"], c["heads"], c["dim"])
    return _plain_attend(s, q, keys, vals, torch.full_like(s["length"], c["rows"]), s["length"], seq, row)


def _padded(x, start, wide, of, at):
    out = torch.zeros(start.numel() - 1, wide, *x.shape[1:], device="cuda")
    out[of, at] = x.float()
    return out


def _plain_prompt(s):
    of, at = _of_row(s["k_start"], s["keys"])
    seq, row = _of_row(s["q_start"], s["rows"])
    keys, vals = (_padded(s[x], s["k_start"], s["max_keys"], of, at).transpose(1, 2) for x in ("k", "v"))
    q = _padded(s["q"], s["q_start"], s["max_rows"], seq, row)
    return _plain_attend(s, q, keys, vals, s["q_start"].diff(), s["k_start"].diff(), seq, row)


def _plain(s):
    c = s["case"]
    if c["op"] == "decode":
        return _plain_decode(s)
    if c["op"] == "prompt":
        return _plain_prompt(s)
    if c["op"] == "store":
        return _plain_store(s)
    q, k, _ = _heads_of(s)
    co, si = _turns(c, s["pos"])
    if c["op"] == "norm":
        return _plain_norm(c, q, s["wq"], co, si).to(q.dtype), _plain_norm(c, k, s["wk"], co, si).to(k.dtype)
    return _plain_norm_grad(c, q, s["wq"], co, si, s["dq"]) + _plain_norm_grad(c, k, s["wk"], co, si, s["dk"])


# ---------------------------------------------------------------------------------------------- the framework's
_program = {}


def _context():
    """The context and the rotary handles that a program keeps, on torch's stream."""
    if not _program:
        sys.path.insert(0, os.path.join(ROOT, "universal-loader_b200"))
        import ulb_capi

        _program.update(u=ulb_capi, ctx=ulb_capi.Context(torch.cuda.current_device()), ropes={})
    _program["ctx"].use_stream(torch.cuda.current_stream().cuda_stream)
    return _program["u"], _program["ctx"]


def _rotary(u, ctx, c):
    key = (c["dim"], c["rot"], c["layout"])
    if key not in _program["ropes"]:
        _program["ropes"][key] = u.Rope(ctx, c["dim"], rot_dim=c["rot"], layout=c["layout"], base=1e4 if c["dim"] == 64 else 5e5)
    return _program["ropes"][key]


def _cache(u, s):
    """The description of the state's cache, which a program keeps beside it."""
    if "cache" not in s:
        c = s["case"]
        s["cache"] = u.QuantDesc(format=u.T_Q8_0 if c["bits"] == 8 else u.T_Q4_1, dtype=u.dtype_id(c["kind"]), n_head_kv=c["kv"],
                                 head_dim=c["dim"], page=c["page"], n_pages=s["k"].shape[0], n_seq=s["table"].shape[0],
                                 max_pages=s["table"].shape[1])
    return s["cache"]


def _framework(s):
    c = s["case"]
    u, ctx = _context()
    h, kv, d = c["heads"], c["kv"], c["dim"]
    kind, scale = u.dtype_id(c["kind"]), 1.0 / math.sqrt(d)
    if c["op"] == "decode":
        ctx.quant_attention(_cache(u, s), h, s["q"].shape[0], c["rows"], s["max_len"], scale, s["q"].data_ptr(), s["k"].data_ptr(),
                            s["v"].data_ptr(), s["table"].data_ptr(), s["start"].data_ptr(), s["prefix"].data_ptr(),
                            s["length"].data_ptr(), None, 0, s["out"].data_ptr(), s["lse"].data_ptr())
        return s["out"], s["lse"]
    if c["op"] == "prompt":
        ctx.prompt_attention(kind, h, kv, d, c["seqs"], s["rows"], s["keys"], s["max_rows"], s["max_keys"], scale,
                             s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["q_start"].data_ptr(),
                             s["k_start"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr())
        return s["out"], s["lse"]
    rope, m, row, q = _rotary(u, ctx, c), s["qkv"].shape[0], (h + 2 * kv) * d, s["qkv"].data_ptr()
    k = q + h * d * BYTES[c["kind"]]
    if c["op"] == "store":
        normed = dict(q_weight=s["wq"].data_ptr(), k_weight=s["wk"].data_ptr(), eps=EPS) if c["normed"] else {}
        rope.quant_append(_cache(u, s), kind, q, k, k + kv * d * BYTES[c["kind"]], h, s["pos"].data_ptr(), s["row_seq"].data_ptr(),
                          s["slot"].data_ptr(), s["table"].data_ptr(), m, s["q_out"].data_ptr(), s["k"].data_ptr(),
                          s["v"].data_ptr(), q_row=row, k_row=row, v_row=row, **normed)
        ctx.quant_read(_cache(u, s), kind, s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["row_seq"].data_ptr(),
                       s["slot"].data_ptr(), m, s["k_out"].data_ptr(), s["v_out"].data_ptr())
        return s["q_out"], s["k_out"], s["v_out"]
    if c["op"] == "norm":
        rope.norm_apply(kind, q, k, m, h, kv, s["wq"].data_ptr(), s["wk"].data_ptr(), EPS, s["pos"].data_ptr(),
                        s["q_out"].data_ptr(), s["k_out"].data_ptr(), q_row=row, k_row=row)
        return s["q_out"], s["k_out"]
    rope.norm_grad(kind, q, k, s["dq"].data_ptr(), s["dk"].data_ptr(), m, h, kv, s["wq"].data_ptr(), s["wk"].data_ptr(), EPS,
                   s["pos"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(), s["dwq"].data_ptr(), s["dwk"].data_ptr(),
                   q_row=row, k_row=row)
    return s["q_out"], s["dwq"], s["k_out"], s["dwk"]


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    h, kv, d = c["heads"], c["kv"], c["dim"]
    if c["op"] in ("norm", "norm_grad"):
        n, e = c["rows"] * (h + kv) * d, BYTES[c["kind"]]
        if c["op"] == "norm":
            return {"bytes": 2 * n * e + 4 * c["rows"] + 8 * d, "flops": 8 * n}
        return {"bytes": 3 * n * e + 4 * c["rows"] + 16 * d, "flops": 16 * n}
    if c["op"] == "store":
        m = c["rows"]
        return {"bytes": m * (2 * h + 2 * kv + 2 * kv) * d * 2 + 2 * 2 * m * kv * _row_bytes(c) + 12 * m,
                "flops": 8 * m * (h + 2 * kv) * d}
    if c["op"] == "decode":
        keys = c["high"] + (c["seqs"] - 1) * (c["low"] + c["high"]) / 2 + c["seqs"] * c["rows"]
        rows = c["seqs"] * c["rows"]
        return {"bytes": 2 * keys * kv * _row_bytes(c) + rows * h * (d * 4 + 4), "flops": 4 * keys * c["rows"] * h * d}
    rows = sum(_lengths(c))
    pairs = sum(n * (n + 1) / 2 for n in _lengths(c)) + rows * c["before"]
    keys = rows + c["seqs"] * c["before"]
    return {"bytes": 2 * keys * kv * d * 2 + rows * h * (d * 4 + 4), "flops": 4 * pairs * h * d}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_turn(c, x, pos, sign):
    """Pairs as complex numbers times exp(i pos w)."""
    rot = c["rot"]
    base = 1e4 if c["dim"] == 64 else 5e5
    w = torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(pos.numel(), rot // 2, dtype=torch.float64, device="cuda"), sign * pos.double()[:, None] * w[None])
    part = x[..., :rot]
    if c["layout"] == "interleaved":
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * turn[:, None]
        y = torch.view_as_real(z).reshape(part.shape)
    else:
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn[:, None]
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _exact_norm(c, x, w, pos):
    x = x.double()
    return _exact_turn(c, x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double(), pos, 1.0)


def _exact_norm_grad(c, x, w, pos, dy):
    """The gradient by the quotient rule: y = w x / s, s = sqrt(mean x^2 + eps), ds/dx = x / (n s)."""
    x, g = x.double(), _exact_turn(c, dy.double(), pos, -1.0)
    s = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    ds = -(g * w.double() * x).sum(-1, keepdim=True) / s ** 2
    return g * w.double() / s + ds * x / (c["dim"] * s), (g * x / s).sum(0).sum(0)


def _exact_blocks(c, x):
    """What the blocks of x stand for."""
    x = x.double().reshape(*x.shape[:-1], -1, 32)
    if c["bits"] == 8:
        d = x.abs().max(-1, keepdim=True).values / 127
        code = torch.where(d > 0, torch.trunc(x / d + 0.5 * x.sign()), torch.zeros_like(x))
        return (code * d.half().double()).flatten(-2)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    d = (high - low) / 15
    code = torch.where(d > 0, torch.trunc((x - low) / d + 0.5), torch.zeros_like(x))
    return (code * d.half().double() + low.half().double()).flatten(-2)


def _exact_values(c, rows):
    """The values of rows of the pool, taken apart byte by byte."""
    d, at = c["dim"], torch.arange(c["dim"], device="cuda")
    if c["bits"] == 8:
        code = rows[..., :d].view(torch.int8).double()
        scale = rows[..., d:d + d // 16].contiguous().view(torch.float16).double()
        return code * scale[..., at // 32]
    scale = rows[..., d // 2:d // 2 + d // 8].contiguous().view(torch.float16).double()
    byte = at // 64 * 32 + at % 32 // 4 * 4 + at // 32 % 2 + at % 2 * 2
    code = torch.div(rows[..., byte].long(), torch.where(at % 4 >= 2, 16, 1), rounding_mode="floor") % 16
    return code.double() * scale[..., at // 32 * 2] + scale[..., at // 32 * 2 + 1]


def _exact_rows(c, q, keys, vals):
    """Rows q [n][h][d] that end with the keys [m][kv][d]: head by head."""
    n, m = q.shape[0], keys.shape[0]
    out, lse = torch.empty_like(q, dtype=torch.float64), torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    hide = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
    for h in range(c["heads"]):
        j = h // (c["heads"] // c["kv"])
        score = (q[:, h].double() @ keys[:, j].double().T / math.sqrt(c["dim"])).masked_fill_(hide, -math.inf)
        lse[:, h] = torch.logsumexp(score, 1)
        out[:, h] = torch.exp(score - lse[:, h, None]) @ vals[:, j].double()
    return out, lse


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("decode", "prompt"):
        outs, lses = [], []
        for b in range(c["seqs"]):
            if c["op"] == "decode":
                n, page = int(s["length"][b]), c["page"]
                pages = s["table"][b, :(n + page - 1) // page].long()
                keys, vals = (_exact_values(c, p[pages].transpose(1, 2).reshape(-1, c["kv"], p.shape[-1])[:n]) for p in (s["k"], s["v"]))
                rows = slice(b * c["rows"], (b + 1) * c["rows"])
            else:
                rows, of = (slice(int(s[x][b]), int(s[x][b + 1])) for x in ("q_start", "k_start"))
                keys, vals = s["k"][of], s["v"][of]
            out, lse = _exact_rows(c, s["q"][rows], keys, vals)
            outs.append(out)
            lses.append(lse)
        return torch.cat(outs), torch.cat(lses)
    q, k, v = s["qkv"][:, :c["heads"]], s["qkv"][:, c["heads"]:c["heads"] + c["kv"]], s["qkv"][:, c["heads"] + c["kv"]:]
    if c["op"] == "store":
        q, k = (_exact_norm(c, x, w, s["pos"]) if c["normed"] else _exact_turn(c, x.double(), s["pos"], 1.0)
                for x, w in ((q, s["wq"]), (k, s["wk"])))
        return q, _exact_blocks(c, k), _exact_blocks(c, v)
    if c["op"] == "norm":
        return _exact_norm(c, q, s["wq"], s["pos"]), _exact_norm(c, k, s["wk"], s["pos"])
    return _exact_norm_grad(c, q, s["wq"], s["pos"], s["dq"]) + _exact_norm_grad(c, k, s["wk"], s["pos"], s["dk"])
