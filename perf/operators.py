"""Timed cases of the cache-side operators of a speculative step kept outside the built-in loop.

A step of such a program rotates its q and k rows and appends K and V to the pages of a cache
("rope_append", its gradient form "rope_grad"), attends a tree of drafted tokens over those pages
("tree_attention"), changes the logits by penalties, biases and grammar masks ("logits"), and moves what
the tree left in the cache ("pages_copy": copies on write of forked sequences, "pages_compact": the
accepted path of each tree).

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


# ---------------------------------------------------------------------------------------------- cases
def _rope(name, op, rows, heads, kv, dim, rot, layout, scaling, factor, base, kind, page=256, far=4096):
    return dict(name=name, op=op, rows=rows, heads=heads, kv=kv, dim=dim, rot=rot, layout=layout, scaling=scaling,
                factor=factor, base=base, kind=kind, page=page, far=far)


def _attn(name, seqs, nodes, low, high, heads, kv, dim, kind, page):
    return dict(name=name, op="tree_attention", seqs=seqs, nodes=nodes, low=low, high=high, heads=heads, kv=kv, dim=dim,
                kind=kind, page=page)


def _pages(name, op, layers, kv, dim, page, kind, moves):
    return dict(name=name, op=op, layers=layers, kv=kv, dim=dim, page=page, kind=kind, moves=moves)


def _logits(name, seqs, nodes, vocab, history, biases, grammar, kind):
    return dict(name=name, op="logits", seqs=seqs, nodes=nodes, vocab=vocab, history=history, biases=biases,
                grammar=grammar, kind=kind)


def listed():
    return [
        # the draft model's decode step of eight sequences: one row each, only latency counts
        _rope("append decode 8 rows", "rope_append", 8, 32, 4, 64, 64, "interleaved", "none", 1.0, 1e4, "f16"),
        # verify rows of 64 sequences with trees of 16 nodes under a context scaled eight times
        _rope("append verify 1024 rows", "rope_append", 1024, 64, 8, 128, 128, "half", "yarn", 8.0, 5e5, "bf16", far=32768),
        # gradient of the q and k rows of a fine-tuning batch, half of each head rotated, odd row count
        _rope("gradient 16381 rows", "rope_grad", 16381, 40, 0, 128, 64, "half", "wavelength", 8.0, 5e5, "f32", far=16384),
        # one token of one sequence in a short context: latency
        _attn("attend 1 token", 1, 1, 500, 500, 32, 4, 64, "f16", 256),
        # one tree of 63 nodes, every head with keys of its own
        _attn("attend 63 nodes mha", 1, 63, 8191, 8191, 32, 32, 128, "f16", 256),
        # 64 sequences of ragged lengths with trees of up to 16 nodes, grouped heads, small pages
        _attn("attend 64 sequences", 64, 16, 256, 4096, 32, 8, 128, "bf16", 64),
        # the largest: one tree of 64 nodes over a long context, grouped heads
        _attn("attend 131072 keys", 1, 64, 131001, 131001, 64, 8, 128, "bf16", 256),
        # sixteen forked sequences' tail pages copied on write, in all layers
        _pages("fork 16 pages", "pages_copy", 32, 8, 128, 256, "f16", 16),
        # the accepted paths of 64 trees moved to their positions
        _pages("compact 64 paths", "pages_compact", 16, 8, 64, 256, "f16", 64),
        # one row in a short conversation: latency
        _logits("logits 1 row", 1, 1, 32000, 200, 4, False, "f32"),
        # a decode batch with penalties, biases and a grammar
        _logits("logits 64 rows", 64, 1, 128256, 2000, 16, True, "f32"),
        # eight trees of 63 nodes: each node with its own path and its own grammar state
        _logits("logits 504 nodes", 8, 63, 128256, 6000, 16, True, "f16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope_append", "rope_grad", "tree_attention", "tree_attention", "pages_copy", "pages_compact",
                     "logits", "logits"])
    kind = rng.choice(["f16", "bf16"])
    heads, kv = rng.choice([(32, 32), (32, 8), (32, 4), (64, 8), (8, 2), (5, 5), (12, 4)])
    if op in ("rope_append", "rope_grad"):
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 2, 32])
        c = _rope("", op, _log(rng, 1, 12000), heads, kv if op == "rope_append" else 0, dim, rot,
                  rng.choice(["interleaved", "half"]), rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
                  rng.choice([2.0, 4.0, 8.0]), rng.choice([1e4, 5e5]), kind if op == "rope_append" else
                  rng.choice(["f32", kind]), rng.choice([16, 64, 256]), rng.choice([4096, 32768, 131072]))
        c["rows"] = min(c["rows"], int(6e8 / (heads * dim * 8)))
    elif op == "tree_attention":
        dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
        seqs, nodes, high = _log(rng, 1, 64), _log(rng, 1, 160), _log(rng, 8, 100000)
        c = _attn("", seqs, nodes, max(0, high // rng.choice([1, 2, 16])), high, heads, kv, dim, kind,
                  rng.choice([16, 32, 64, 128, 256]))
        while 4.0 * c["seqs"] * c["nodes"] * (c["high"] + c["nodes"]) * heads * dim > 1.5e11 or \
                c["seqs"] * (c["high"] + c["nodes"] + 256) * kv * dim * 4 > 4e8:
            big = max(("seqs", 1.0), ("nodes", 0.8), ("high", 0.01), key=lambda p: c[p[0]] * p[1])[0]
            c[big] = max(1, c[big] // 2)
            c["low"] = min(c["low"], c["high"])
    elif op == "pages_copy":
        c = _pages("", op, rng.choice([1, 2, 16, 22, 32]), rng.choice([2, 4, 8]), rng.choice([64, 80, 128]),
                   rng.choice([16, 64, 128, 256]), kind, _log(rng, 1, 16))
    elif op == "pages_compact":
        c = _pages("", op, rng.choice([1, 2, 16]), rng.choice([2, 4, 8]), rng.choice([64, 80, 128]),
                   rng.choice([16, 64, 128]), kind, _log(rng, 1, 64))
    else:
        c = _logits("", _log(rng, 1, 64), _log(rng, 1, 80), rng.choice([32000, 128256, _log(rng, 1000, 140000)]),
                    _log(rng, 1, 12000), _log(rng, 1, 300), rng.random() < 0.7, rng.choice(["f32", "f16", "bf16"]))
        while c["seqs"] * c["nodes"] * c["vocab"] > 6e7:
            big = "seqs" if c["seqs"] > c["nodes"] else "nodes"
            c[big] = max(1, c[big] // 2)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------- inputs
def _tree(r, n):
    """A random tree of n nodes in the order they were drafted: the path of each as rows of bits."""
    bits = torch.zeros(n, n, dtype=torch.bool)
    for j in range(n):
        up = -1 if j < 2 else int(torch.randint(max(-1, j - 12), j, (1,), generator=r))
        if up >= 0:
            bits[j] = bits[up]
        bits[j, j] = True
    return bits


def _words(bits):
    """Rows of bits packed into 32-bit words, bit j of word w for column 32 w + j."""
    rows, n = bits.shape
    w = (n + 31) // 32
    wide = torch.zeros(rows, w * 32, dtype=torch.int64)
    wide[:, :n] = bits
    v = (wide.view(rows, w, 32) << torch.arange(32)).sum(-1)
    return torch.where(v >= 2 ** 31, v - 2 ** 32, v).to(torch.int32)


def _sizes(seqs, nodes):
    """Nodes of each sequence's tree: `nodes` down to half of that."""
    return [nodes - 5 * i % (nodes - max(1, nodes // 2) + 1) for i in range(seqs)]


def _trees(r, seqs, nodes):
    """Random trees of those sizes, one a sequence: where their rows start, and the rows' words."""
    sizes = _sizes(seqs, nodes)
    words = torch.zeros(sum(sizes), (nodes + 31) // 32, dtype=torch.int32)
    start = [0]
    for n in sizes:
        words[start[-1]:start[-1] + n, :(n + 31) // 32] = _words(_tree(r, n))
        start.append(start[-1] + n)
    return start, words


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


def prepare(case, seed):
    c, dev = case, "cuda"
    r = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, kind="f32", scale=1.0):
        return (torch.randn(shape, device=dev, generator=g) * scale).to(TYPES[kind])

    s = {"case": c}
    if c["op"] in ("rope_append", "rope_grad"):
        m, h, kv, d = c["rows"], c["heads"], c["kv"], c["dim"]
        s["pos"] = torch.randint(0, c["far"], (m,), generator=r).to(torch.int32).to(dev)
        if c["op"] == "rope_grad":
            s["x"] = normal(m, h, d, kind=c["kind"])
            s["out"] = torch.empty_like(s["x"])
            return s
        s["qkv"] = normal(m, h + 2 * kv, d)  # as the projection leaves them, in 32 bits
        seqs = max(1, m // 16)
        most = (64 + c["page"] - 1) // c["page"] + 1
        table, n = _table(r, [most] * seqs, most)
        seq = torch.arange(m) % seqs
        slot = 3 + torch.arange(m) // seqs  # a sequence's rows in slots that follow one another
        s.update(table=table.to(dev), row_seq=seq.to(torch.int32).to(dev), slot=slot.to(torch.int32).to(dev),
                 q_out=torch.zeros(m, h, d, dtype=TYPES[c["kind"]], device=dev),
                 k=normal(n, kv, c["page"], d, kind=c["kind"]), v=normal(n, kv, c["page"], d, kind=c["kind"]))
    elif c["op"] == "tree_attention":
        start, words = _trees(r, c["seqs"], c["nodes"])
        prefix = [c["high"]] + [int(torch.randint(c["low"], c["high"] + 1, (1,), generator=r)) for _ in range(c["seqs"] - 1)]
        length = [p + start[i + 1] - start[i] for i, p in enumerate(prefix)]
        most = (max(length) + c["page"] - 1) // c["page"]
        table, n = _table(r, [(x + c["page"] - 1) // c["page"] for x in length], most)
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        s.update(rows=start[-1], max_rows=c["nodes"], max_len=max(length), start=ints(start), prefix=ints(prefix),
                 length=ints(length), words=words.to(dev), table=table.to(dev),
                 q=normal(start[-1], c["heads"], c["dim"], kind=c["kind"], scale=1.5),
                 k=normal(n, c["kv"], c["page"], c["dim"], kind=c["kind"]),
                 v=normal(n, c["kv"], c["page"], c["dim"], kind=c["kind"]),
                 out=torch.empty(start[-1], c["heads"], c["dim"], dtype=TYPES[c["kind"]], device=dev),
                 lse=torch.empty(start[-1], c["heads"], device=dev))
    elif c["op"] == "pages_copy":
        n = 2 * c["moves"] + 3
        order = torch.randperm(n, generator=r)
        count = torch.randint(1, c["page"] + 1, (c["moves"],), generator=r)
        count[0] = c["page"]
        moves = torch.stack([order[:c["moves"]], order[c["moves"]:2 * c["moves"]], count], 1)
        s.update(moves=moves.to(torch.int32).to(dev),
                 k=normal(c["layers"], n, c["kv"], c["page"], c["dim"], kind=c["kind"]),
                 v=normal(c["layers"], n, c["kv"], c["page"], c["dim"], kind=c["kind"]))
    elif c["op"] == "pages_compact":
        nodes, most_src = 16, 6
        most = (nodes + c["page"] - 1) // c["page"] + 1
        table, n = _table(r, [most] * c["moves"], most)
        base = torch.randint(0, most * c["page"] - nodes + 1, (c["moves"],), generator=r)
        count = torch.randint(0, most_src + 1, (c["moves"],), generator=r)
        src = torch.stack([torch.randperm(nodes, generator=r)[:most_src].sort().values for _ in range(c["moves"])])
        ints = lambda v: v.to(torch.int32).to(dev)  # noqa: E731
        s.update(table=ints(table), base=ints(base), count=ints(count), src=ints(src),
                 k=normal(c["layers"], n, c["kv"], c["page"], c["dim"], kind=c["kind"]),
                 v=normal(c["layers"], n, c["kv"], c["page"], c["dim"], kind=c["kind"]))
    else:
        v = c["vocab"]
        start, words = _trees(r, c["seqs"], c["nodes"])
        rows = start[-1]
        sizes = [c["history"]] + [int(torch.randint(1, c["history"] + 1, (1,), generator=r)) for _ in range(c["seqs"] - 1)]
        at = [0]
        for x in sizes:
            at.append(at[-1] + x)
        few = max(2, v // 16)  # words come back within a conversation
        # a sequence's history: its prompt, then what it generated
        hist = torch.randint(0, few, (at[-1],), generator=r) * 16 % v
        prompt = [x // 2 for x in sizes]
        # biases: a few tokens of each sequence, in the order of their ids
        nb = min(c["biases"], v)
        bias_tok = torch.stack([torch.randint(0, v, (nb,), generator=r).sort().values for _ in range(c["seqs"])])
        ints = lambda x: torch.as_tensor(x).to(torch.int32).to(dev)  # noqa: E731
        s.update(rows=rows, start=ints(start), words=words.to(dev), history=ints(hist), history_start=ints(at),
                 prompt=ints(prompt), node_tokens=ints(torch.randint(0, few, (rows,), generator=r) * 16 % v),
                 params=torch.stack([torch.empty(c["seqs"]).uniform_(1.0, 1.5, generator=r),
                                     torch.empty(c["seqs"]).uniform_(0.0, 1.0, generator=r),
                                     torch.empty(c["seqs"]).uniform_(0.0, 0.5, generator=r)], 1).to(dev),
                 bias_start=ints(torch.arange(c["seqs"] + 1) * nb), bias_tok=ints(bias_tok.reshape(-1)),
                 bias_val=normal(c["seqs"] * nb, scale=5.0),
                 logits=normal(rows, v, kind=c["kind"], scale=3.0), out=torch.empty(rows, v, device=dev))
        if c["grammar"]:
            # three words of four are cut; one row in eight is free of the grammar
            allow = torch.randint(-2 ** 31, 2 ** 31, (rows, (v + 31) // 32), device=dev, generator=g)
            more = torch.randint(-2 ** 31, 2 ** 31, (rows, (v + 31) // 32), device=dev, generator=g)
            s["allow"] = (allow & more).to(torch.int32)
            s["row_allow"] = ints(torch.where(torch.rand(rows, generator=r) < 0.125, -1, torch.arange(rows)))
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _frequencies(c):
    """Radians a position for each pair, and the factor on the rotated part, in 64 bits."""
    rot, base, f = c["rot"], c["base"], c["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "ntk":
        base = base * f ** (rot / (rot - 2))
    w = base ** (-2.0 * i / rot)
    if c["scaling"] == "linear":
        return w / f, 1.0
    if c["scaling"] == "yarn":  # original context 4096, ramp between 32 rotations and one
        low = max(math.floor(rot * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
        high = min(math.ceil(rot * math.log(4096 / (1 * 2 * math.pi)) / (2 * math.log(base))), rot - 1)
        ramp = ((i - low) / (max(high - low, 0.001))).clamp(0, 1)
        return w / f * ramp + w * (1 - ramp), 0.1 * math.log(f) + 1.0
    if c["scaling"] == "wavelength":  # original context 4096, low and high frequency factors 1 and 4
        turns = 4096 * w / (2 * math.pi)
        mix = ((turns - 1) / 3).clamp(0, 1)
        return (1 - mix) * w / f + mix * w, 1.0
    return w, 1.0


def _turn(c, x, pos, sign):
    """x [rows][heads][dim] rotated to its positions, in 32 bits; the angles alone need 64."""
    w, m = _frequencies(c)
    angle = pos.double()[:, None] * w
    co, si = (angle.cos() * m).float()[:, None], (sign * angle.sin() * m).float()[:, None]
    x, rot = x.float(), c["rot"]
    out = x.clone()
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if c["layout"] == "interleaved" else (x[..., :rot // 2], x[..., rot // 2:rot])
    first, second = a * co - b * si, a * si + b * co
    if c["layout"] == "interleaved":
        out[..., :rot:2], out[..., 1:rot:2] = first, second
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = first, second
    return out


def _places(table, seq, pos, page):
    return table[seq, pos // page].long(), pos % page


def _seen(words, n):
    at = torch.arange(n, device=words.device)
    return (words[:, at // 32] >> (at % 32)) & 1 != 0


def _of_row(start, rows):
    n = (start[1:] - start[:-1]).long()
    return torch.repeat_interleave(torch.arange(n.numel(), device=start.device), n, output_size=rows)


def _plain_attention(s):
    c = s["case"]
    b, h, kv, d, page = c["seqs"], c["heads"], c["kv"], c["dim"], c["page"]
    group, wide = h // kv, s["table"].shape[1] * page
    keys = s["k"][s["table"].clamp(min=0).long()].float().permute(0, 2, 1, 3, 4).reshape(b, kv, wide, d)
    vals = s["v"][s["table"].clamp(min=0).long()].float().permute(0, 2, 1, 3, 4).reshape(b, kv, wide, d)
    seq = _of_row(s["start"], s["rows"])
    row = torch.arange(s["rows"], device="cuda") - s["start"][seq]
    q = torch.zeros(b, s["max_rows"], h, d, device="cuda")
    q[seq, row] = s["q"].float()
    q = q.view(b, -1, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d)
    at = torch.arange(wide, device="cuda")
    # slot j of the tree is position prefix + j
    node = at[None] - s["prefix"][:, None]
    bits = torch.zeros(b, s["max_rows"], s["words"].shape[1] * 32, dtype=torch.bool, device="cuda")
    bits[seq, row] = _seen(s["words"], s["words"].shape[1] * 32)
    inside = (node >= 0) & (at[None] < s["length"][:, None])
    see = torch.gather(bits, 2, node.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, s["max_rows"], -1))
    see = (node < 0)[:, None] | (see & inside[:, None])
    scores = (q @ keys.transpose(2, 3)) * (1.0 / math.sqrt(d))
    scores = scores.view(b, kv, -1, group, wide).masked_fill_(~see[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.view(b, kv, -1, wide) @ vals).view(b, kv, -1, group, d) / total.clamp(min=1e-38)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, -1, h, d)[seq, row].to(TYPES[c["kind"]])
    return out, lse.permute(0, 2, 1, 3).reshape(b, -1, h)[seq, row]


def _plain_logits(s):
    c = s["case"]
    v, b = c["vocab"], c["seqs"]
    x = s["logits"].float()
    seq = _of_row(s["start"], s["rows"])
    total = s["history"].numel()
    of = _of_row(s["history_start"], total)
    made = torch.arange(total, device="cuda") - s["history_start"][of] >= s["prompt"][of]
    place = of * v + s["history"]
    count = torch.zeros(b * v, device="cuda").scatter_add_(0, place, made.float()).view(b, v)[seq]
    seen = torch.zeros(b * v, dtype=torch.bool, device="cuda").index_fill_(0, place, True).view(b, v)[seq]
    # the tokens of a row's path, its own among them, count as generated
    path = _seen(s["words"], c["nodes"])
    node = (s["start"][seq].long()[:, None] + torch.arange(c["nodes"], device="cuda")).clamp(max=s["rows"] - 1)
    count.scatter_add_(1, s["node_tokens"][node].long(), path.float())
    rep, presence, frequency = s["params"][seq].split(1, 1)
    x = torch.where(seen | (count > 0), torch.where(x > 0, x / rep, x * rep), x)
    x = x - frequency * count - presence * (count > 0)
    of = _of_row(s["bias_start"], s["bias_tok"].numel())
    x = x + torch.zeros(b * v, device="cuda").index_put_((of * v + s["bias_tok"],), s["bias_val"], accumulate=True).view(b, v)[seq]
    if c["grammar"]:
        ok = _seen(s["allow"], v)[s["row_allow"].clamp(min=0).long()] | (s["row_allow"] < 0)[:, None]
        x = x.masked_fill(~ok, -math.inf)
    return x


def _plain(s):
    c = s["case"]
    if c["op"] == "rope_grad":
        return _turn(c, s["x"], s["pos"], -1.0).to(TYPES[c["kind"]])
    if c["op"] == "rope_append":
        h, kv = c["heads"], c["kv"]
        page, at = _places(s["table"], s["row_seq"], s["slot"], c["page"])
        turned = _turn(c, s["qkv"][:, :h + kv], s["pos"], 1.0).to(TYPES[c["kind"]])
        s["k"][page, :, at] = turned[:, h:]
        s["v"][page, :, at] = s["qkv"][:, h + kv:].to(TYPES[c["kind"]])
        return turned[:, :h], s["k"], s["v"]
    if c["op"] == "tree_attention":
        return _plain_attention(s)
    if c["op"] == "pages_copy":
        src, dst, n = s["moves"].long().unbind(1)
        part = (torch.arange(c["page"], device="cuda") < n[:, None])[None, :, None, :, None]
        s["k"][:, dst] = torch.where(part, s["k"][:, src], s["k"][:, dst])
        s["v"][:, dst] = torch.where(part, s["v"][:, src], s["v"][:, dst])
        return s["k"], s["v"]
    if c["op"] == "pages_compact":
        i = torch.arange(s["src"].shape[1], device="cuda")
        seq = torch.arange(c["moves"], device="cuda")[:, None].expand(-1, i.numel())
        to = s["base"][:, None] + i
        fro = torch.where(i < s["count"][:, None], s["base"][:, None] + s["src"], to)  # or onto itself
        (pf, of), (pt, ot) = _places(s["table"], seq, fro, c["page"]), _places(s["table"], seq, to, c["page"])
        s["k"][:, pt, :, ot] = s["k"][:, pf, :, of]
        s["v"][:, pt, :, ot] = s["v"][:, pf, :, of]
        return s["k"], s["v"]
    return _plain_logits(s)


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
    key = (c["dim"], c["rot"], c["layout"], c["scaling"], c["factor"], c["base"])
    if key not in _program["ropes"]:
        _program["ropes"][key] = u.Rope(ctx, c["dim"], rot_dim=c["rot"], layout=c["layout"], base=c["base"],
                                        scaling=c["scaling"], factor=c["factor"], orig_len=4096, beta_fast=32.0,
                                        beta_slow=1.0, low_freq=1.0, high_freq=4.0)
    return _program["ropes"][key]


def _cache(u, s):
    """The description of the state's cache, which a program keeps beside it."""
    if "cache" not in s:
        c, k = s["case"], s["k"]
        layers = c.get("layers", 1)
        seqs, most = s["table"].shape if "table" in s else (1, 1)
        s["cache"] = u.CacheDesc(dtype=u.dtype_id(c["kind"]), n_layer=layers, n_head_kv=c["kv"], head_dim=c["dim"],
                                 page=c["page"], n_pages=k.shape[-4], n_seq=seqs, max_pages=most)
    return s["cache"]


def _framework(s):
    c = s["case"]
    u, ctx = _context()
    if c["op"] == "rope_grad":
        _rotary(u, ctx, c).apply(u.dtype_id(c["kind"]), s["x"].data_ptr(), s["x"].shape[0], c["heads"], s["pos"].data_ptr(),
                                 s["out"].data_ptr(), inverse=True)
        return s["out"]
    if c["op"] == "rope_append":
        h, kv, d, m = c["heads"], c["kv"], c["dim"], c["rows"]
        q, row = s["qkv"].data_ptr(), (h + 2 * kv) * d
        _rotary(u, ctx, c).append(_cache(u, s), u.dtype_id("f32"), q, q + h * d * 4, q + (h + kv) * d * 4, h,
                                  s["pos"].data_ptr(), s["row_seq"].data_ptr(), s["slot"].data_ptr(),
                                  s["table"].data_ptr(), m, s["q_out"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                                  q_row=row, k_row=row, v_row=row)
        return s["q_out"], s["k"], s["v"]
    if c["op"] == "tree_attention":
        ctx.tree_attention(_cache(u, s), c["heads"], s["rows"], s["max_rows"], s["max_len"], 1.0 / math.sqrt(c["dim"]),
                           s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(),
                           s["start"].data_ptr(), s["prefix"].data_ptr(), s["length"].data_ptr(), s["words"].data_ptr(),
                           s["words"].shape[1], s["out"].data_ptr(), s["lse"].data_ptr())
        return s["out"], s["lse"]
    if c["op"] == "pages_copy":
        ctx.pages_copy(_cache(u, s), s["k"].data_ptr(), s["v"].data_ptr(), s["moves"].data_ptr(), c["moves"])
        return s["k"], s["v"]
    if c["op"] == "pages_compact":
        ctx.pages_compact(_cache(u, s), s["k"].data_ptr(), s["v"].data_ptr(), s["table"].data_ptr(), s["base"].data_ptr(),
                          s["count"].data_ptr(), s["src"].data_ptr(), s["src"].shape[1])
        return s["k"], s["v"]
    ctx.logits_process(u.dtype_id(c["kind"]), s["logits"].data_ptr(), s["out"].data_ptr(), c["vocab"], c["seqs"], s["rows"],
                       s["start"].data_ptr(), max_rows=c["nodes"], params=s["params"].data_ptr(),
                       history=s["history"].data_ptr(), history_start=s["history_start"].data_ptr(),
                       prompt=s["prompt"].data_ptr(), node_tokens=s["node_tokens"].data_ptr(), words=s["words"].data_ptr(),
                       n_words=s["words"].shape[1], bias_start=s["bias_start"].data_ptr(), bias_tokens=s["bias_tok"].data_ptr(),
                       bias_values=s["bias_val"].data_ptr(), allow=s["allow"].data_ptr() if c["grammar"] else None,
                       row_allow=s["row_allow"].data_ptr() if c["grammar"] else None,
                       n_allow=s["rows"] if c["grammar"] else 0)
    return s["out"]


def run(state):
    return _framework(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "rope_grad":
        n = c["rows"] * c["heads"] * c["dim"]
        return {"bytes": 2 * n * BYTES[c["kind"]] + 4 * c["rows"], "flops": 3 * n}
    if c["op"] == "rope_append":
        n = c["rows"] * (c["heads"] + 2 * c["kv"]) * c["dim"]
        return {"bytes": n * (4 + BYTES[c["kind"]]) + 12 * c["rows"], "flops": 3 * n}
    if c["op"] == "tree_attention":
        keys = c["high"] + (c["seqs"] - 1) * (c["low"] + c["high"]) / 2
        rows = sum(_sizes(c["seqs"], c["nodes"]))
        keys += rows
        pairs = keys * rows / c["seqs"]
        return {"bytes": 2 * keys * c["kv"] * c["dim"] * 2 + rows * c["heads"] * (c["dim"] * 4 + 4),
                "flops": 4 * pairs * c["heads"] * c["dim"]}
    if c["op"] == "pages_copy":
        positions = c["page"] + (c["moves"] - 1) * (c["page"] + 1) / 2
        return {"bytes": 2 * 2 * c["layers"] * c["kv"] * positions * c["dim"] * 2, "flops": 0}
    if c["op"] == "pages_compact":
        return {"bytes": 2 * 2 * c["layers"] * c["kv"] * c["moves"] * 3 * c["dim"] * 2 + 32 * c["moves"], "flops": 0}
    rows = sum(_sizes(c["seqs"], c["nodes"]))
    history = c["history"] * (1 + c["seqs"]) / 2
    return {"bytes": rows * c["vocab"] * (BYTES[c["kind"]] + 4 + (0.125 if c["grammar"] else 0)) + 4 * history
            + 8 * c["seqs"] * c["biases"], "flops": 4 * rows * c["vocab"]}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_turn(c, x, pos, sign):
    """Pairs as complex numbers times m exp(i pos w)."""
    rot, base, f, m = c["rot"], c["base"], c["factor"], 1.0
    w = []
    for i in range(rot // 2):
        b = base * f ** (rot / (rot - 2.0)) if c["scaling"] == "ntk" else base
        e = b ** (-2.0 * i / rot)
        if c["scaling"] == "linear":
            e /= f
        elif c["scaling"] == "yarn":
            edge = lambda n: rot * math.log(4096 / (n * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            low, high = max(math.floor(edge(32)), 0), min(math.ceil(edge(1)), rot - 1)
            part = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            e = e * (1 - part) + e / f * part
            m = 0.1 * math.log(f) + 1.0
        elif c["scaling"] == "wavelength":
            wave = 2 * math.pi / e
            if wave > 4096 / 1.0:
                e /= f
            elif wave > 4096 / 4.0:
                mix = (4096 / wave - 1.0) / (4.0 - 1.0)
                e = (1 - mix) * e / f + mix * e
        w.append(e)
    turn = torch.polar(torch.full((pos.numel(), rot // 2), m, dtype=torch.float64, device="cuda"),
                       sign * pos.double()[:, None] * torch.tensor(w, dtype=torch.float64, device="cuda")[None])
    x = x.double()
    part = x[..., :rot]
    if c["layout"] == "interleaved":
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * turn[:, None]
        y = torch.view_as_real(z).reshape(part.shape)
    else:
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn[:, None]
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., rot:]], -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope_grad":
        return _exact_turn(c, s["x"], s["pos"], -1.0)
    if c["op"] == "rope_append":
        h, kv = c["heads"], c["kv"]
        x = _exact_turn(c, s["qkv"][:, :h + kv], s["pos"], 1.0)
        k, v = s["k"].double(), s["v"].double()
        slot = s["slot"].long()
        page = s["table"][s["row_seq"].long(), torch.div(slot, c["page"], rounding_mode="floor")].long()
        k.transpose(1, 2)[page, slot % c["page"]] = x[:, h:]
        v.transpose(1, 2)[page, slot % c["page"]] = s["qkv"][:, h + kv:].double()
        return x[:, :h], k, v
    if c["op"] == "tree_attention":
        out = torch.zeros(s["rows"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
        lse = torch.full((s["rows"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
        start, prefix, length = s["start"].tolist(), s["prefix"].tolist(), s["length"].tolist()
        group = c["heads"] // c["kv"]
        for b in range(c["seqs"]):
            r0, r1, n = start[b], start[b + 1], length[b]
            pages = s["table"][b, :(n + c["page"] - 1) // c["page"]].long()
            bit = torch.arange(r1 - r0, device="cuda")
            tree = (s["words"][r0:r1].long()[:, bit // 32] // (2 ** (bit % 32))) % 2 == 1
            hide = torch.cat([torch.zeros(r1 - r0, prefix[b], dtype=torch.bool, device="cuda"), ~tree], 1)
            for j in range(c["kv"]):
                keys = s["k"][pages, j].reshape(-1, c["dim"])[:n].double()
                vals = s["v"][pages, j].reshape(-1, c["dim"])[:n].double()
                for h in range(j * group, (j + 1) * group):
                    score = s["q"][r0:r1, h].double() @ keys.T / math.sqrt(c["dim"])
                    score[hide] = -math.inf
                    lse[r0:r1, h] = torch.logsumexp(score, 1)
                    out[r0:r1, h] = torch.exp(score - lse[r0:r1, h, None]) @ vals
        return out, lse
    if c["op"] == "pages_copy":
        k, v = s["k"].double(), s["v"].double()
        for src, dst, n in s["moves"].tolist():
            k[:, dst, :, :n] = k[:, src, :, :n]
            v[:, dst, :, :n] = v[:, src, :, :n]
        return k, v
    if c["op"] == "pages_compact":
        k, v = s["k"].double(), s["v"].double()
        table, page = s["table"].tolist(), c["page"]
        for q, (base, count, src) in enumerate(zip(s["base"].tolist(), s["count"].tolist(), s["src"].tolist())):
            for i in range(count):
                a, b = base + src[i], base + i
                for pool in (k, v):
                    pool[:, table[q][b // page], :, b % page] = pool[:, table[q][a // page], :, a % page]
        return k, v
    x = s["logits"].double()
    start, at, prompt = s["start"].tolist(), s["history_start"].tolist(), s["prompt"].tolist()
    bias_at, params = s["bias_start"].tolist(), s["params"].double().tolist()
    for b in range(c["seqs"]):
        old = s["history"][at[b]:at[b + 1]].long()
        before = torch.bincount(old, minlength=c["vocab"]) > 0
        made = torch.bincount(old[prompt[b]:], minlength=c["vocab"])
        shift = torch.zeros(c["vocab"], dtype=torch.float64, device="cuda")
        shift.index_add_(0, s["bias_tok"][bias_at[b]:bias_at[b + 1]].long(), s["bias_val"][bias_at[b]:bias_at[b + 1]].double())
        rep, presence, frequency = params[b]
        tokens, n = s["node_tokens"][start[b]:start[b + 1]].long(), start[b + 1] - start[b]
        bit = torch.arange(n, device="cuda")
        for r in range(start[b], start[b + 1]):
            path = tokens[(s["words"][r].long()[bit // 32] // (2 ** (bit % 32))) % 2 == 1]
            times = made + torch.bincount(path, minlength=c["vocab"])
            old_or_path = before | (times > 0)
            y = x[r]
            y = torch.where(old_or_path & (y > 0), y / rep, torch.where(old_or_path, y * rep, y))
            x[r] = y - frequency * times - presence * (times > 0).double() + shift
            if c["grammar"] and (a := int(s["row_allow"][r])) >= 0:
                bits = torch.arange(32, device="cuda")
                ok = ((s["allow"][a].long()[:, None] >> bits) & 1).reshape(-1)[:c["vocab"]] == 1
                x[r] = torch.where(ok, x[r], torch.full_like(x[r], -math.inf))
    return x
