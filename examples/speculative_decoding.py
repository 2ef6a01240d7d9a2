"""Speculative decoding of a small random decoder: the operators between a layer's projections at work together.

Several continuations of one prompt run at once. The prompt is taken in as one chain on row 0 of the cache and the other
rows are forked from it, sharing its full pages. Each step drafts a tree of likely next tokens for every continuation,
norms and turns the heads and appends the whole draft to the cache's pages, lets each drafted token see its ancestors
(the prompt's pages being read once for all rows), and keeps the path that the model's own choice of tokens, or its
probabilities and random numbers, take: what was kept moves up behind the committed tokens. At the end the rows are freed.

    python examples/speculative_decoding.py [--continuations 4] [--tokens 96] [--width 256] [--layers 2] [--temperature 40]

The weights are random (there is nothing to download), so the text means nothing; the greedy tokens are those that
decoding one token at a time gives, in fewer steps, and drawn ones have the same distribution.
"""
import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ingot_amd import Heads, KvCache, KvTable, Session  # noqa: E402
from ingot_amd import _lib as L  # noqa: E402


class Decoder:
    """Layers of attention and a SiLU feed-forward part over a paged bf16 cache, f32 between the projections."""

    def __init__(self, sess, rng, vocab=97, width=256, layers=2, heads=8, kv_heads=2, page_size=16, pages=96, rows=4,
                 max_tokens=512, norms=False):
        self.sess, self.vocab, self.width, self.heads, self.kv, self.rows = sess, vocab, width, heads, kv_heads, rows
        self.dim = width // heads
        self.max_tokens, self.page = max_tokens, page_size
        self.embed = rng.normal(0, 1, (vocab, width)).astype(np.float32)

        def weight(n, k, gain):
            w = rng.normal(0, gain / np.sqrt(k), (n, k)).astype(np.float32)
            return sess.upload_weight(w, trans=True, pack_dtype=L.DT_BF16)

        self.layers = [dict(qkv=weight((heads + 2 * kv_heads) * self.dim, width, 1.0), out=weight(width, width, 0.7),
                            up=weight(4 * width, width, 1.0), down=weight(width, 4 * width, 0.7)) for _ in range(layers)]
        # the head leans towards the next token in a cycle of six, so that a text repeats itself and drafts have a chance
        after = np.arange(vocab) // 6 * 6 + (np.arange(vocab) + 1) % 6
        head = self.embed[np.argsort(np.minimum(after, vocab - 1), kind="stable")] + rng.normal(0, 2, self.embed.shape)
        self.head = sess.upload_weight(head.astype(np.float32), trans=True, pack_dtype=L.DT_BF16)
        self.cos, self.sin = sess.rotary_table(max_tokens, self.dim)
        if norms:  # of the query and key heads of each layer
            for w in self.layers:
                w["norms"] = [sess.to_device(rng.normal(1, 0.2, self.dim).astype(np.float32)) for _ in range(2)]
        max_pages = -(-max_tokens // page_size)
        shape = (layers, pages, kv_heads, page_size, self.dim)
        self.cache = KvCache(sess.empty(L.DT_BF16, shape), sess.empty(L.DT_BF16, shape))
        table = [np.full((rows, max_pages), -1), np.zeros(rows), np.zeros(pages), np.zeros(1)]
        dev = [sess.to_device(a.astype(np.int32)) for a in table]
        # lengths before and after a step: the two tables differ in which they call the length
        self.lengths = [dev[1], sess.to_device(np.zeros(rows, np.int32))]
        self.tables = [KvTable(dev[0], n, dev[2], dev[3]) for n in self.lengths]

    @property
    def table(self):
        return self.tables[0]

    def _ints(self, *arrays):
        return [self.sess.to_device(np.asarray(a, np.int32)) for a in arrays]

    def fork(self, src, dst):
        """Rows dst[i] become copies of rows src[i]."""
        a, b = self._ints(src, dst)
        self.sess.kv_fork(self.cache, self.table, a, b)
        self._served()
        free(a, b)

    def drop(self, rows):
        a, = self._ints(rows)
        self.sess.kv_free(self.cache, self.table, a)
        free(a)

    def _served(self):
        if self.table.missing.numpy()[0]:
            raise MemoryError("the cache has too few pages")

    def step(self, rows, drafts, shared=0):
        """Logits of every drafted token, on the host (see forward)."""
        logits, starts = self.forward(rows, drafts, shared)
        got = logits.numpy()
        self._served()
        free(logits)
        return [got[starts[b]:starts[b + 1]] for b in range(len(rows))]

    def forward(self, rows, drafts, shared=0):
        """Logits of every drafted token, and where each sequence's begin. drafts[b]: (token, parent, depth) of each node of
        the sequence on rows[b], parents before their children and -1 for the root; the nodes' keys and values are then in
        the cache, behind the committed ones. shared: committed tokens that all rows have in common."""
        s, counts = self.sess, [len(d) for d in drafts]
        starts = np.concatenate([[0], np.cumsum(counts)])
        n, most = int(starts[-1]), max(counts)
        base = self.table.lengths.numpy()
        mask = np.zeros((n, -(-most // 32)), np.uint32)
        tokens, positions = np.zeros(n, np.int64), np.zeros(n, np.int64)
        for b, draft in enumerate(drafts):
            for i, (token, parent, depth) in enumerate(draft):
                t = starts[b] + i
                if parent >= 0:
                    mask[t] = mask[starts[b] + parent]
                mask[t, i // 32] |= np.uint32(1 << (i % 32))
                tokens[t], positions[t] = token, base[rows[b]] + depth
        d_rows, d_starts, d_counts, d_pos = self._ints(rows, starts, counts, positions)
        d_mask = s.to_device(mask.view(np.int32))
        s.kv_reserve(self.cache, self.table, d_rows, d_counts)
        wide = (self.heads + 2 * self.kv) * self.dim
        x = s.to_device(self.embed[tokens])
        new = lambda cols: s.empty(L.DT_F32, (n, cols))  # noqa: E731
        qkv, att, mid, y, logits = new(wide), new(self.width), new(4 * self.width), new(self.width), new(self.vocab)
        q, k, v = (Heads(qkv, n, heads, self.dim, first * self.dim, wide, self.dim)
                   for heads, first in ((self.heads, 0), (self.kv, self.heads), (self.kv, self.heads + self.kv)))
        out = Heads(att, n, self.heads, self.dim, 0, self.width, self.dim)
        d_group = self._ints([0, len(rows)], [shared])
        for i, w in enumerate(self.layers):
            s.gemm(x, w["qkv"], qkv, n)
            where = dict(rows=d_rows, layer=i)
            turn = (d_pos, self.cos, self.sin, q, self.cache, self.table, d_starts)
            if "norms" in w:
                s.norm_rotary_append(q, k, v, *w["norms"], *turn, **where)
            else:
                s.rotary_append(q, k, v, *turn, **where)
            see = dict(max_nodes=most, max_tokens=int(base.max()) + most, mask=d_mask, **where)
            if shared:
                s.prefix_attention(q, self.cache, self.table, d_starts, out, *d_group, max_shared=shared, **see)
            else:
                s.tree_attention(q, self.cache, self.table, d_starts, out, **see)
            s.gemm(att, w["out"], y, n, beta=1.0, c=x, c_mode=L.C_FULL)
            s.gemm(y, w["up"], mid, n, act=L.ACT_SILU)
            s.gemm(mid, w["down"], x, n, beta=1.0, c=y, c_mode=L.C_FULL)
        s.gemm(x, self.head, logits, n)
        free(d_rows, d_starts, d_counts, d_pos, d_mask, *d_group, x, qkv, att, mid, y)
        return logits, starts

    def verify(self, rows, drafts, temperature, rng, shared=0):
        """One step whose drafts are verified on the device: the path kept of each, and the token that follows it, drawn at
        `temperature` (0: the likeliest)."""
        s, n = self.sess, len(rows)
        logits, starts = self.forward(rows, drafts, shared)
        flat = [node for draft in drafts for node in draft]
        most = max(len(d) for d in drafts)
        d_starts, d_tokens, d_parents = self._ints(starts, [t for t, _, _ in flat], [p for _, p, _ in flat])
        out = [s.empty(L.DT_I32, shape) for shape in ((n, most), (n,), (n,))]
        numbers = [s.to_device(a.astype(np.float32)) for a in (np.full(n, temperature), rng.random(len(flat)), rng.random(n))]
        s.verify_drafts(logits, d_starts, d_tokens, *out, parents=d_parents, temperature=numbers[0], accept_u=numbers[1],
                        sample_u=numbers[2])
        nodes, counts, tokens = (t.numpy() for t in out)
        self._served()
        free(logits, d_starts, d_tokens, d_parents, *out, *numbers)
        return [(nodes[b, :counts[b]].tolist(), int(tokens[b])) for b in range(n)]


    def accept(self, rows, paths):
        """Commits nodes paths[b] of the last step's draft on row rows[b]; its other nodes are forgotten."""
        most = max(len(p) for p in paths)
        nodes = np.full((len(paths), most), -1)
        for b, p in enumerate(paths):
            nodes[b, :len(p)] = p
        d_rows, d_nodes, d_counts = self._ints(rows, nodes, [len(p) for p in paths])
        self.sess.copy_d2d(self.lengths[1], self.lengths[0])  # rows that are not listed keep their length
        self.sess.kv_compact(self.cache, self.table, d_rows, d_nodes, d_counts, self.lengths[1])
        self.lengths.reverse()
        self.tables.reverse()
        free(d_rows, d_nodes, d_counts)


def free(*tensors):
    for t in tensors:
        t.free()


def chain(tokens):
    return [(t, i - 1, i) for i, t in enumerate(tokens)]


def draft_tree(text, depth, breadth, nodes):
    """Guesses after the last token of `text`: what followed each token before, newest first, `breadth` of them, down to
    `depth` tokens and at most `nodes` nodes. The root is the last token itself."""
    after = {}
    for a, b in zip(text, text[1:]):
        after.setdefault(a, [])
        after[a] = [b] + [t for t in after[a] if t != b]
    tree, level = [(text[-1], -1, 0)], [0]
    for d in range(1, depth + 1):
        below = []
        for parent in level:
            for token in after.get(tree[parent][0], [])[:breadth]:
                if len(tree) < nodes:
                    below.append(len(tree))
                    tree.append((token, parent, d))
        level = below
    return tree


def longest_path(tree, logits):
    """The nodes on the path the model takes itself, and the token it gives after the last of them."""
    node, path = 0, [0]
    while True:
        token = int(np.argmax(logits[node]))
        node = next((i for i, (t, parent, _) in enumerate(tree) if parent == node and t == token), None)
        if node is None:
            return path, token
        path.append(node)


def generate(model, prompt, continuations, tokens, depth=5, breadth=3, nodes=24, temperature=None, rng=None):
    """`continuations` texts of `tokens` tokens after `prompt`, each begun with another of the likeliest next tokens; and
    the steps it took. depth 0 decodes one token at a time. With a temperature the drafts are verified on the device, by
    numbers of `rng`; without one the text is the likeliest, and the host looks for its path."""
    rows = list(range(continuations))
    logits = model.step([0], [chain(prompt)])[0]
    model.accept([0], [list(range(len(prompt)))])
    if continuations > 1:
        model.fork([0] * (continuations - 1), rows[1:])
    begin = np.argsort(-logits[-1], kind="stable")[:continuations]
    texts = [list(prompt) + [int(t)] for t in begin]
    goal, steps = len(prompt) + tokens, 0
    active = [r for r in rows if len(texts[r]) < goal]
    while active:
        trees = [draft_tree(texts[r], depth, breadth, nodes) for r in active]
        if temperature is None:
            found = [longest_path(t, l) for t, l in zip(trees, model.step(active, trees))]
        else:
            found = model.verify(active, trees, temperature, rng, shared=len(prompt))
        model.accept(active, [path for path, _ in found])
        for r, tree, (path, token) in zip(active, trees, found):
            texts[r] += [tree[i][0] for i in path[1:]] + [token]
        steps += 1
        active = [r for r in active if len(texts[r]) < goal]
    model.drop(rows)
    return [t[:goal] for t in texts], steps


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--continuations", type=int, default=4)
    p.add_argument("--tokens", type=int, default=96)
    p.add_argument("--width", type=int, default=256)
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--temperature", type=float, default=40.0, help="of the drawn texts: the logits of random weights are large")
    a = p.parse_args()
    rng = np.random.default_rng(1)
    with Session(0) as sess:
        model = Decoder(sess, rng, width=a.width, layers=a.layers, rows=a.continuations, max_tokens=64 + a.tokens,
                        pages=a.continuations * (-(-(64 + a.tokens) // 16) + 1), norms=True)
        prompt = rng.integers(0, model.vocab, 33).tolist()
        for name, depth, heat in (("one token at a time", 0, None), ("drafted trees", 5, None),
                                  ("drafted trees, verified on the device", 5, 0.0), ("drawn", 5, a.temperature)):
            generate(model, prompt, a.continuations, a.tokens, depth=depth, temperature=heat, rng=rng)
            t = time.perf_counter()
            texts, steps = generate(model, prompt, a.continuations, a.tokens, depth=depth, temperature=heat, rng=rng)
            print(f"{name}: {steps} steps, {(time.perf_counter() - t) * 1e3:.1f} ms", flush=True)
        print("pages still held:", int(model.table.references.numpy().sum()))
        for t in texts:
            print(" ".join(map(str, t[33:57])), "...")


if __name__ == "__main__":
    main()
