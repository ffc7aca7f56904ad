"""A speculative step kept by the caller, from the paged cache operators of include/ulb.h.

A one-layer toy model (random weights, projections by torch) decodes several continuations of one prompt:

  ulb_pages_*        the prompt's pages are shared by every continuation (fork) and copied when one of
                     them writes; pages past the accepted positions go back
  ulb_rope_append    q and k of the rows turned to their positions, K and V into the pages
  ulb_tree_attention the rows of each continuation's drafted tree over its pages
  ulb_logits_process penalties, biases and a grammar on the logits of every node
  ulb_sample         greedy tokens
  ulb_pages_compact  K and V of the accepted path to their positions

and prints whether the trees gave the tokens that decoding one row at a time gives.

  python examples/paged_step.py [continuations] [tokens]
"""
import ctypes as C
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "universal-loader_b200"))
import ulb_capi as U  # noqa: E402

VOCAB, WIDTH, HEADS, KV, DIM, PAGE = 2048, 512, 8, 2, 64, 16
TREE = [-1, -1, 0, 0, 1, 2]  # parent of each node: two children of the root, two and one below, one deeper


def ints(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


class Program:
    def __init__(self, seqs, most, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        f = lambda *s: torch.randn(*s, device="cuda", generator=g) / math.sqrt(s[0])  # noqa: E731
        self.embed = torch.randn(VOCAB, WIDTH, device="cuda", generator=g)
        self.wqkv, self.wo = f(WIDTH, (HEADS + 2 * KV) * DIM) * 2, f(HEADS * DIM, WIDTH) * 4
        self.ctx = U.Context(torch.cuda.current_device())
        self.ctx.use_stream(torch.cuda.current_stream().cuda_stream)
        self.rope = U.Rope(self.ctx, DIM, layout="half", base=10000.0)
        self.per_seq = (most + PAGE - 1) // PAGE + 1
        pages = seqs * self.per_seq
        self.cache = U.CacheDesc(dtype=U.T_BF16, n_layer=1, n_head_kv=KV, head_dim=DIM, page=PAGE, n_pages=pages, n_seq=seqs,
                                 max_pages=self.per_seq)
        self.k = torch.zeros(pages, KV, PAGE, DIM, dtype=torch.bfloat16, device="cuda")
        self.v = torch.zeros_like(self.k)
        self.book = U.Pages(self.ctx, self.cache, self.k.data_ptr(), self.v.data_ptr())
        # one token in sixteen is outside the grammar, one token is asked for, one discouraged
        bits = torch.arange(VOCAB, device="cuda") % 16 != 5
        words = (bits.view(-1, 32).long() << torch.arange(32, device="cuda")).sum(1)
        self.allow = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)

    def rows(self, tokens, pos, seq, slot, start, prefix, length, mask, words):
        """Logits of rows: appended to the cache, attended, projected."""
        m = tokens.numel()
        x = self.embed[tokens.long()]
        qkv = x @ self.wqkv
        q = torch.empty(m, HEADS, DIM, dtype=torch.bfloat16, device="cuda")
        o = torch.empty_like(q)
        table = self.book.table
        base, row = qkv.data_ptr(), (HEADS + 2 * KV) * DIM
        self.rope.append(self.cache, U.T_F32, base, base + HEADS * DIM * 4, base + (HEADS + KV) * DIM * 4, HEADS, pos.data_ptr(),
                         seq.data_ptr(), slot.data_ptr(), table, m, q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), row, row, row)
        counts = start[1:] - start[:-1]
        self.ctx.tree_attention(self.cache, HEADS, m, int(counts.max()), int(length.max()), 1 / math.sqrt(DIM), q.data_ptr(),
                                self.k.data_ptr(), self.v.data_ptr(), table, start.data_ptr(), prefix.data_ptr(),
                                length.data_ptr(), None if mask is None else mask.data_ptr(), words, o.data_ptr())
        y = x + o.float().view(m, -1) @ self.wo
        return (y @ self.embed.T / math.sqrt(WIDTH)).contiguous()

    def choose(self, logits, start, histories, prompt, node_tokens=None, mask=None):
        """Greedy tokens of rows under the penalties of their contexts and the grammar."""
        n, rows = len(histories), logits.shape[0]
        at = [0]
        for h in histories:
            at.append(at[-1] + len(h))
        keep = [ints(sum(histories, [])), ints(at), ints([prompt] * n), torch.tensor([[1.3, 0.4, 0.2]] * n, device="cuda"),
                ints([2 * i for i in range(n + 1)]), ints([7, 1000] * n), torch.tensor([2.0, -3.0] * n, device="cuda"),
                ints([0] * rows)]
        hist, at, pr, params, bs, bt, bv, allowed = keep
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.ctx.logits_process(U.T_F32, p(logits), p(logits), VOCAB, n, rows, p(start), params=p(params), history=p(hist),
                                history_start=p(at), prompt=p(pr), node_tokens=p(node_tokens), words=p(mask),
                                n_words=0 if mask is None else 1, bias_start=p(bs), bias_tokens=p(bt), bias_values=p(bv),
                                allow=p(self.allow), row_allow=p(allowed), n_allow=1)
        out = torch.empty(rows, dtype=torch.int32, device="cuda")
        warp = U.Warp(0.0, 0, 1.0)
        U.check(U.lib().ulb_sample(self.ctx.h, p(logits), rows, VOCAB, VOCAB, C.byref(warp), 0, 0, 0, U.RNG_DRAFT, p(out)))
        return out.tolist()

    def close(self):
        self.ctx.sync()
        self.book.close()
        self.rope.close()
        self.ctx.close()


def start(p, prompt, first):
    """The prompt into sequence 0, shared by the others; `first`: the token each continuation begins with."""
    n = len(prompt)
    p.book.reserve(0, 0, n)
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    p.rows(ints(prompt), at, torch.zeros_like(at), at, ints([0, n]), ints([0]), ints([n]), None, 0)
    for s in range(1, len(first)):
        p.book.fork(0, s, n)
    return [prompt + [t] for t in first]


def decode_rows(p, prompt, first, tokens):
    """One row a step: the last token's K and V go in, its logits choose the next."""
    seqs = start(p, prompt, first)
    n = len(first)
    while min(len(s) for s in seqs) < len(prompt) + tokens:
        pos = [len(s) - 1 for s in seqs]
        for s in range(n):
            p.book.reserve(s, pos[s], pos[s] + 1)
        st = ints(range(n + 1))
        logits = p.rows(ints([s[-1] for s in seqs]), ints(pos), ints(range(n)), ints(pos), st, ints(pos), ints([x + 1 for x in pos]), None, 0)
        for s, t in zip(seqs, p.choose(logits, st, [list(s) for s in seqs], len(prompt))):
            s.append(t)
    return seqs


def decode_trees(p, prompt, first, tokens, draft):
    """A tree a step: row 0 the last token, the rest drafted below it; the longest path that the rows' own
    choices agree with is kept."""
    seqs = start(p, prompt, first)
    n, size, steps = len(first), 1 + len(TREE), 0
    depth, bits = [0], [1]
    for i, up in enumerate(TREE):  # row 1 + i; its parent's row is 1 + up (0: the root row)
        depth.append(depth[1 + up] + 1)
        bits.append(bits[1 + up] | 1 << (1 + i))
    mask = ints(bits * n)
    while min(len(s) for s in seqs) < len(prompt) + tokens:
        base = [len(s) - 1 for s in seqs]
        nodes = [[s[-1]] + draft(s, TREE) for s in seqs]
        for s in range(n):
            p.book.reserve(s, base[s], base[s] + size)
        st = ints([size * i for i in range(n + 1)])
        flat = ints(sum(nodes, []))
        logits = p.rows(flat, ints([b + d for b in base for d in depth]), ints([s for s in range(n) for _ in depth]),
                        ints([b + j for b in base for j in range(size)]), st, ints(base), ints([b + size for b in base]), mask, 1)
        # a row's context is the history before the root row, then its path; the root row's own token is on every path
        took = p.choose(logits, st, [s[:-1] for s in seqs], len(prompt), flat, mask)
        paths = []
        for s in range(n):
            row, path = 0, [0]
            while True:
                want = took[size * s + row]
                seqs[s].append(want)
                child = [1 + i for i, up in enumerate(TREE) if 1 + up == row and nodes[s][1 + i] == want]
                if not child:
                    break
                row = child[0]
                path.append(row)
            paths.append(path)
        at, count, src = ints(base), ints([len(x) for x in paths]), ints([x + [size] * (size - len(x)) for x in paths])
        p.ctx.pages_compact(p.cache, p.k.data_ptr(), p.v.data_ptr(), p.book.table, at.data_ptr(), count.data_ptr(), src.data_ptr(), size)
        for s in range(n):
            p.book.truncate(s, base[s] + len(paths[s]))
        steps += 1
    return seqs, steps


def main(continuations=4, tokens=48, seed=3):
    r = torch.Generator().manual_seed(seed)
    prompt = torch.randint(0, VOCAB, (37,), generator=r).tolist()
    first = torch.randint(0, VOCAB, (continuations,), generator=r).tolist()
    most = len(prompt) + tokens + 2 * (1 + len(TREE))
    a = Program(continuations, most)
    rows = [s[:len(prompt) + tokens] for s in decode_rows(a, prompt, first, tokens)]
    a.close()

    def draft(s, tree):
        """A draft that is right about half of the time: the known continuation, or a token by chance."""
        i = next(j for j, f in enumerate(first) if rows[j][len(prompt)] == s[len(prompt)])
        known = rows[i][len(s):] + [0] * 8
        level, out = {-1: 0}, []
        for j, up in enumerate(tree):
            level[j] = level[up] + 1
            guess = known[level[j] - 1] if int(torch.randint(0, 2, (1,), generator=r)) else int(torch.randint(0, VOCAB, (1,), generator=r))
            out.append(guess)
        return out

    b = Program(continuations, most)
    trees, steps = decode_trees(b, prompt, first, tokens, draft)
    free = b.book.free
    b.close()
    trees = [s[:len(prompt) + tokens] for s in trees]
    same = sum(x == y for x, y in zip(rows, trees))
    print("%d of %d continuations of %d tokens are the same from trees; %d tree steps where rows took %d; %d pages free at the end"
          % (same, continuations, tokens, steps, tokens - 1, free))
    return same, steps


if __name__ == "__main__":
    main(*[int(x) for x in sys.argv[1:3]])
