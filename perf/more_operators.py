"""Performance cases of more decoder-step operators: norms of queries and keys with their rotation, attention of a batch
that shares a long prefix, and the verification of drafted tokens.

They stand next to the rotation, the attention and the page operations of the decoder step: every head of the queries
and keys is normed before it is turned and appended to the cache's pages; sequences that were forked from one prompt hold
its pages in common, so their attention reads that prefix once for all of them; and the target's logits of the drafted
tokens decide, by given random numbers, which of them are kept and which token follows. One token without a draft is
ordinary sampling.

Inputs are torch tensors on the GPU made from the seed. With `own` the framework's entry points read and write them in
place; without it the same results come from elementary torch operations in 32 bits (the verification in 64: a random
number next to the border of two of 10^5 tokens must fall on the same side).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def listed():
    return [
        # One new token of one sequence, the decode workload's 16 heads of 128: norm, rotate, append (latency).
        dict(name="norm_append_token", kind="append", batch=1, nodes=1, ctx=517, heads=16, kv_heads=16, dim=128, rot=128,
             interleaved=False, x="f32", cache="bf16", page=16, per_head=False),
        # Drafts of 32 sequences, shared key heads of 80, half the head rotated in neighbour pairs, a weight for each head.
        dict(name="norm_append_drafts", kind="append", batch=32, nodes=16, ctx=900, heads=32, kv_heads=8, dim=80, rot=40,
             interleaved=True, x="bf16", cache="bf16", page=32, per_head=True),
        # The queries of a long prompt.
        dict(name="norm_prompt", kind="norm", tokens=8191, heads=32, dim=128, rot=128, interleaved=False, x="bf16",
             per_head=False),
        # Ordinary sampling: one token of one sequence, no draft (latency).
        dict(name="sample_token", kind="verify", batch=1, nodes=1, vocab=32000, x="f32", draft="tree"),
        # Eight drafted trees over a vocabulary whose rows start at odd addresses.
        dict(name="verify_trees", kind="verify", batch=8, nodes=24, vocab=50001, x="bf16", draft="tree"),
        # Chains drawn from a draft model, whose own logits count in the acceptance.
        dict(name="verify_chains", kind="verify", batch=32, nodes=6, vocab=131072, x="f32", draft="chain"),
        # Many sequences with trees, a large vocabulary.
        dict(name="verify_many", kind="verify", batch=64, nodes=16, vocab=128000, x="bf16", draft="tree"),
        # Four answers to one short prompt, one token each: f32 activations, 16 heads with their own keys (latency).
        dict(name="prefix_few", kind="prefix", batch=4, groups=1, nodes=1, shared=512, ctx=60, heads=16, kv_heads=16,
             dim=128, x="f32", cache="bf16", page=16, mask="chain"),
        # 32 answers to one prompt, ordinary batched decoding.
        dict(name="prefix_batch", kind="prefix", batch=32, groups=1, nodes=1, shared=4096, ctx=300, heads=32, kv_heads=8,
             dim=128, x="bf16", cache="bf16", page=32, mask="chain"),
        # Drafted trees of several groups, f32 queries over a bf16 cache, prefixes that end inside a page among them.
        dict(name="prefix_trees", kind="prefix", batch=24, groups=5, nodes=16, shared=3000, ctx=500, heads=32, kv_heads=8,
             dim=128, x="f32", cache="bf16", page=64, mask="tree"),
        # An f32 cache, heads of 80, pages that are no power of two.
        dict(name="prefix_f32", kind="prefix", batch=9, groups=3, nodes=3, shared=1500, ctx=200, heads=12, kv_heads=12,
             dim=80, x="f32", cache="f32", page=24, mask="tree"),
        # Many answers to two very long prompts.
        dict(name="prefix_long", kind="prefix", batch=128, groups=2, nodes=1, shared=32768, ctx=600, heads=32, kv_heads=8,
             dim=128, x="bf16", cache="bf16", page=64, mask="chain"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "append", "append", "verify", "verify", "verify", "prefix", "prefix", "prefix", "prefix"))
    kv_heads = rng.choice((1, 2, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 5, 8))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
    x, cache = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f32")))
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 100, 128))
    turn = dict(rot=dim // rng.choice((1, 1, 2, 4)), interleaved=rng.random() < 0.5, per_head=rng.random() < 0.3)
    held = dict(heads=heads, kv_heads=kv_heads, dim=dim, x=x, cache=cache, page=page)
    if kind == "norm":
        case = dict(tokens=_size(rng, 1, 8191), heads=heads, dim=dim, x=x, **turn)
    elif kind == "append":
        case = dict(batch=_size(rng, 1, 64), nodes=_size(rng, 1, 48), ctx=_size(rng, 1, 3000), **held, **turn)
    elif kind == "verify":
        case = dict(batch=_size(rng, 1, 64), nodes=rng.choice((1, _size(rng, 2, 10), _size(rng, 2, 64))),
                    vocab=_size(rng, 50, 200000), x=x, draft=rng.choice(("tree", "tree", "chain")))
    else:
        batch = _size(rng, 2, 128)
        case = dict(batch=batch, groups=min(batch, _size(rng, 1, 8)), nodes=rng.choice((1, 1, _size(rng, 2, 24))),
                    shared=_size(rng, 1, 32768), ctx=_size(rng, 1, 2000), mask=rng.choice(("tree", "chain")), **held)
    case = dict(kind=kind, **case)
    while _too_large(case):  # nothing above the largest listed case of its kind
        side = next(k for k in ("tokens", "batch", "nodes", "vocab", "shared", "ctx") if case.get(k, 1) > 2)
        case[side] = max(1, case[side] * 3 // 4)
    if kind == "prefix":
        case["groups"] = min(case["groups"], case["batch"])
    return case


def _too_large(case):
    most = [work(c) for c in listed() if c["kind"] == case["kind"]]
    need = work(case)
    pool = case.get("batch", 0) * (case.get("ctx", 0) + case.get("nodes", 1) + case.get("page", 0))
    pool = (pool + case.get("groups", 0) * case.get("shared", 0)) * case.get("kv_heads", 0) * case.get("dim", 0)
    return pool > 3e8 or any(need[k] > max(w[k] for w in most) for k in need)


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _pages_of(tokens, page):
    return -(-tokens // page)


def _ints(*shape, lo, hi, g):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _drafts(case, g):
    """Node counts of each sequence's draft and the parents of its nodes (-1: follows the committed tokens), [batch, nodes]."""
    b, n = case["batch"], case["nodes"]
    spread = n - torch.arange(b, device="cuda") * 5 % (n // 2 + 1)  # half the draft's room up to all of it
    count = spread[torch.randperm(b, generator=g, device="cuda")].clamp(min=1)
    i = torch.arange(n, device="cuda")
    back = (torch.rand((b, n), generator=g, device="cuda") * torch.clamp(i, max=6)).long()
    return count, i - 1 - back  # one of the six nodes before


def _starts(count):
    start = torch.zeros(count.numel() + 1, dtype=torch.int64, device="cuda")
    start[1:] = torch.cumsum(count, 0)
    return start


def _ancestors(parent):
    """[batch, nodes, nodes] truth values: node j is node i itself or an ancestor of it."""
    b, n = parent.shape
    link = torch.zeros((b, n, n + 1), device="cuda")
    link.scatter_(2, torch.where(parent < 0, torch.full_like(parent, n), parent)[:, :, None], 1.0)
    reach = ((link[:, :, :n] + torch.eye(n, device="cuda")) > 0).float()
    for _ in range(max(1, math.ceil(math.log2(max(2, n))))):
        reach = (torch.bmm(reach, reach) > 0).float()
    return reach > 0


def _bits(seen):
    """Truth values [rows, nodes] as 32-bit words."""
    rows, n = seen.shape
    words = -(-n // 32)
    padded = torch.zeros((rows, 32 * words), dtype=torch.int64, device="cuda")
    padded[:, :n] = seen.long()
    value = (padded.view(rows, words, 32) << torch.arange(32, device="cuda")).sum(2)
    return torch.where(value >= 1 << 31, value - (1 << 32), value).to(torch.int32).contiguous()


def _pool(case, num_pages, g):
    """Keys and values, [layer, page, head, slot, dim]: a cache in use, so unused slots hold old values."""
    shape = (1, num_pages, case["kv_heads"], case["page"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["cache"]])
    return k, torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["cache"]])


def _angles(case, rows):
    """cos and sin of every position, made once by a program when it loads a model."""
    r = case["rot"]
    f = 10000.0 ** (-torch.arange(0, r // 2, device="cuda", dtype=torch.float64) * 2.0 / r)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _group_of(first, batch):
    return torch.searchsorted(first[1:].long().contiguous(), torch.arange(batch, device="cuda"), right=True)


def prepare(case, seed):
    g = _generator(seed)
    t = {}
    kind, page = case["kind"], case.get("page", 1)

    def normal(*shape, dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[dtype])

    def weight(heads):  # trained weights lie around 1
        shape = (heads, case["dim"]) if case["per_head"] else (case["dim"],)
        return 1.0 + 0.2 * torch.randn(shape, generator=g, device="cuda")

    if kind == "norm":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        t["x"] = normal(n, h, d, dtype=case["x"])
        t["y"] = torch.empty_like(t["x"])
        t["q_weight"] = weight(h)
        start = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        t["positions"] = torch.arange(start, start + n, device="cuda", dtype=torch.int32)
        t["cos"], t["sin"] = _angles(case, start + n)
    elif kind == "append":
        b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        t["lengths"] = _ints(b, lo=case["ctx"] // 2, hi=case["ctx"] + 1, g=g)
        count, parent = _drafts(case, g)
        start = _starts(count)
        total = int(start[-1])
        t["starts"] = start.to(torch.int32)
        most = _pages_of(case["ctx"] + case["nodes"], page)
        num_pages = b * most + 3
        need = (t["lengths"].long() + count + page - 1) // page
        at = torch.arange(most, device="cuda")
        order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)[:b * most].view(b, most)
        t["pages"] = torch.where(at[None, :] < need[:, None], order, torch.full_like(order, -1)).contiguous()
        t["k_pool"], t["v_pool"] = _pool(case, num_pages, g)
        t["q"] = normal(total, h, d, dtype=case["x"])
        t["k"], t["v"] = normal(total, kv, d, dtype=case["x"]), normal(total, kv, d, dtype=case["x"])
        t["y"] = torch.empty_like(t["q"])
        t["q_weight"], t["k_weight"] = weight(h), weight(kv)
        used = torch.arange(case["nodes"], device="cuda")[None, :] < count[:, None]
        t["positions"] = (t["lengths"][:, None] + _ancestors(parent).sum(2) - 1)[used].to(torch.int32)
        t["cos"], t["sin"] = _angles(case, case["ctx"] + case["nodes"])
    elif kind == "verify":
        b, n, vocab = case["batch"], case["nodes"], case["vocab"]
        count, parent = _drafts(case, g)
        if case["draft"] == "chain":
            parent = torch.arange(n, device="cuda").expand(b, n) - 1
        else:
            parent = torch.where(torch.arange(n, device="cuda") > 0, parent.clamp(min=0), parent)
        start = _starts(count)
        total = int(start[-1])
        t["starts"] = start.to(torch.int32)
        used = torch.arange(n, device="cuda")[None, :] < count[:, None]
        # one sequence of four is greedy, the others have temperatures from 0.4 to 1.2
        greedy = torch.arange(b, device="cuda") % 4 == 3
        t["temperature"] = torch.where(greedy, 0.0, 0.4 + 0.8 * torch.rand(b, generator=g, device="cuda"))
        t["accept_u"] = torch.rand(total, generator=g, device="cuda")
        t["sample_u"] = torch.rand(b, generator=g, device="cuda")
        # logits: a wide floor and eight likely tokens in each row
        logits = 2.5 * torch.randn((total, vocab), generator=g, device="cuda")
        part = vocab // 8  # one of them in each eighth of the vocabulary, from a random place on
        likely = torch.randint(0, vocab, (total, 1), generator=g, device="cuda") + part * torch.arange(8, device="cuda")
        likely = (likely + torch.randint(0, part, (total, 8), generator=g, device="cuda")) % vocab
        height = 17.0 - 0.9 * torch.arange(8, device="cuda") + 0.7 * torch.randn((total, 8), generator=g, device="cuda")
        logits.scatter_(1, likely, height)
        t["logits"] = logits.to(DTYPES[case["x"]])
        above = (start[:-1, None] + parent.clamp(min=0))[used]  # row of each token's parent
        if case["draft"] == "chain":
            # the draft model is a noisy copy of the target, and the tokens are drawn from it
            drafted = logits.add_(torch.randn((total, vocab), generator=g, device="cuda"), alpha=0.5)
            t["draft"] = drafted.to(DTYPES[case["x"]])
            seq = _owner(start, total)[0]
            heat = t["temperature"][seq][:, None]
            noise = -torch.log(-torch.log(torch.rand((total, vocab), generator=g, device="cuda").clamp(1e-20, 1 - 1e-7)))
            drawn = (t["draft"].float() + heat * noise).argmax(dim=1)
            t["tokens"] = drawn[above].to(torch.int32)
        else:
            # children are the likely tokens of their parent, in turn
            earlier = torch.tril(parent[:, :, None] == parent[:, None, :], -1).sum(2)[used]
            t["tokens"] = likely[above, earlier % 8].to(torch.int32)
            t["parents"] = parent[used].to(torch.int32)
        t["accepted"] = torch.empty((b, n), dtype=torch.int32, device="cuda")
        t["counts"] = torch.empty(b, dtype=torch.int32, device="cuda")
        t["next"] = torch.empty(b, dtype=torch.int32, device="cuda")
    else:
        b, h, n, d, groups = case["batch"], case["heads"], case["nodes"], case["dim"], case["groups"]
        # groups of uneven size, at least one sequence each; two prefixes of three end with a page
        cut = (torch.arange(groups + 1, device="cuda") * b + groups // 2) // groups
        cut[0], cut[-1] = 0, b
        t["first"] = cut.to(torch.int32)
        owner = _group_of(t["first"], b)
        shared = _ints(groups, lo=case["shared"] // 2, hi=case["shared"] + 1, g=g).long()
        whole = torch.arange(groups, device="cuda") % 3 != 2
        shared = torch.where(whole, shared // page * page, shared)
        t["shared"] = shared.to(torch.int32)
        t["lengths"] = (shared[owner] + _ints(b, lo=case["ctx"] // 2, hi=case["ctx"] + 1, g=g)).to(torch.int32)
        count, parent = _drafts(case, g)
        start = _starts(count)
        total = int(start[-1])
        t["starts"] = start.to(torch.int32)
        own_most, all_most = _pages_of(case["ctx"] + n, page) + 1, _pages_of(case["shared"] + case["ctx"] + n, page)
        shared_most = _pages_of(case["shared"], page)
        num_pages = groups * shared_most + b * own_most + 3
        order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
        full = (shared // page)[owner][:, None]
        at = torch.arange(all_most, device="cuda")[None, :]
        common = owner[:, None] * shared_most + at
        private = groups * shared_most + torch.arange(b, device="cuda")[:, None] * own_most + at - full
        need = ((t["lengths"].long() + count + page - 1) // page)[:, None]
        index = torch.where(at < full, common, private).clamp(0, num_pages - 1)
        t["pages"] = torch.where(at < need, order[index], torch.full_like(order[index], -1)).contiguous()
        t["k_pool"], t["v_pool"] = _pool(case, num_pages, g)
        # a prefix that ends inside a page: each sequence has its own copy of that page's first slots
        part = full[:, 0].clamp(max=all_most - 1)
        mine, theirs = (t["pages"][r, part].long().clamp(min=0) for r in (torch.arange(b, device="cuda"), cut[owner]))
        keep = (torch.arange(page, device="cuda")[None, :] < (shared % page)[owner][:, None])[:, None, :, None]
        for pool in (t["k_pool"], t["v_pool"]):
            pool[0, mine] = torch.where(keep, pool[0, theirs], pool[0, mine])
        t["q"] = normal(total, h, d, dtype=case["x"])
        t["y"] = torch.empty_like(t["q"])
        if case["mask"] == "tree":
            # one node in sixteen is a place in the draft that was not filled: it sees committed tokens only
            seen = _ancestors(parent) & (torch.rand((b, n, 1), generator=g, device="cuda") > 1 / 16)
            t["mask"] = _bits(seen[torch.arange(n, device="cuda")[None, :] < count[:, None]])
    torch.cuda.synchronize()  # a library session works on its own stream
    return dict(case=dict(case), tensors=t)


# ---- one pass ----

def run(state):
    if own:
        if "calls" not in state:
            state["calls"], state["out"] = _own_calls(state["case"], state["tensors"])
        for call in state["calls"]:
            call()
        return state["out"]
    case, t = state["case"], state["tensors"]
    return PLAIN[case["kind"]](case, t)


# ---- the framework's entry points ----

_session = None


def _own_calls(case, t):
    """The prepared calls of one pass (argument blocks, as a serving program keeps them) and the buffers they write."""
    global _session
    from ingot_amd import DeviceTensor, KvCache, KvTable, Session
    from ingot_amd import _lib as L

    if _session is None:
        _session = Session(0)
    s, kind = _session, case["kind"]
    codes = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.int32: L.DT_I32}
    d = {n: DeviceTensor(s, codes[v.dtype], v.shape, v.data_ptr(), False) for n, v in t.items()}
    if kind == "norm":
        return [s.prepare_norm_rotary(d["x"], d["q_weight"], d["positions"], d["cos"], d["sin"], d["y"], eps=EPS,
                                      interleaved=case["interleaved"])], [t["y"]]
    if kind == "verify":
        return [s.prepare_verify_drafts(d["logits"], d["starts"], d["tokens"], d["accepted"], d["counts"], d["next"],
                                        parents=d.get("parents"), draft=d.get("draft"), temperature=d["temperature"],
                                        accept_u=d["accept_u"], sample_u=d["sample_u"])], [
            t[n] for n in ("accepted", "counts", "next")]
    cache, table = KvCache(d["k_pool"], d["v_pool"]), KvTable(d["pages"], d["lengths"])
    if kind == "append":
        return [s.prepare_norm_rotary_append(d["q"], d["k"], d["v"], d["q_weight"], d["k_weight"], d["positions"], d["cos"],
                                             d["sin"], d["y"], cache, table, d["starts"], eps=EPS,
                                             interleaved=case["interleaved"])], [t["y"], t["k_pool"], t["v_pool"]]
    return [s.prepare_prefix_attention(d["q"], cache, table, d["starts"], d["y"], d["first"], d["shared"],
                                       max_shared=case["shared"], max_nodes=case["nodes"],
                                       max_tokens=case["shared"] + case["ctx"] + case["nodes"], mask=d.get("mask"),
                                       scale=1.0 / math.sqrt(case["dim"]))], [t["y"]]


# ---- the plain forms ----

def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight


def _rotated(x, positions, cos, sin, interleaved):
    """x [tokens, heads, dim] in 32 bits, its first 2 · cos.shape[1] dimensions rotated."""
    half = cos.shape[1]
    c, s = cos[positions.long()][:, None, :], sin[positions.long()][:, None, :]
    part = x[..., :2 * half]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_norm(case, t):
    t["y"].copy_(_rotated(_normed(t["x"], t["q_weight"]), t["positions"], t["cos"], t["sin"], case["interleaved"]))
    return [t["y"]]


def _owner(starts, total):
    """Sequence of each token and its number within it."""
    token = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts[1:].long().contiguous(), token, right=True)
    return seq, token - starts.long()[seq]


def _plain_append(case, t):
    seq, node = _owner(t["starts"], t["q"].shape[0])
    at = t["lengths"].long()[seq] + node
    page = t["pages"][seq, at // case["page"]].long()
    slot = at % case["page"]
    turn = (t["positions"], t["cos"], t["sin"], case["interleaved"])
    t["y"].copy_(_rotated(_normed(t["q"], t["q_weight"]), *turn))
    t["k_pool"][0, page, :, slot] = _rotated(_normed(t["k"], t["k_weight"]), *turn).to(t["k_pool"].dtype)
    t["v_pool"][0, page, :, slot] = t["v"].to(t["v_pool"].dtype)
    return [t["y"], t["k_pool"], t["v_pool"]]


def _plain_verify(case, t):
    b, n, vocab = case["batch"], case["nodes"], case["vocab"]
    starts, total = t["starts"].long(), t["logits"].shape[0]
    count = starts[1:] - starts[:-1]
    heat = t["temperature"].double()
    hot = heat > 0
    seq, _ = _owner(t["starts"], total)
    cold = torch.where(hot, heat, torch.ones_like(heat))[seq][:, None]

    def weights(logits):
        x = logits.double()
        top, best = x.max(dim=1, keepdim=True)
        return torch.exp((x - top) / cold), best[:, 0]

    e, best = weights(t["logits"])
    mass = e.sum(dim=1)
    i = torch.arange(n, device="cuda")
    there = i[None, :] < count[:, None]
    row = (starts[:-1, None] + i).clamp(max=total - 1)  # [batch, nodes]
    token = t["tokens"].long()[row]
    parent = t["parents"].long()[row] if "parents" in t else (i - 1).expand(b, n)
    above = (starts[:-1, None] + parent.clamp(min=0)).clamp(max=total - 1)
    p = e[above, token] / mass[above]
    u = t["accept_u"].double()[row]
    # siblings come in turn: a token is kept if u falls below its share of what the rejected ones before it left
    before = torch.tril(parent[:, :, None] == parent[:, None, :], -1) & there[:, None, :] & (i > 0)
    again = (before & (token[:, :, None] == token[:, None, :])).any(dim=2)
    p = torch.where(again, torch.zeros_like(p), p)
    left = 1.0 - (before * p[:, None, :]).sum(dim=2)
    if "draft" in t:
        d, _ = weights(t["draft"])
        drawn = d.sum(dim=1)
        kept = u * (d[above, token] / drawn[above]) < p
    else:
        kept = u * left < p
    kept = torch.where(hot[:, None], kept, token == best[above]) & there & (i > 0)
    kept = (kept & ~(before & kept[:, None, :]).any(dim=2)) | (i == 0)  # the first of the siblings
    jump = parent.clamp(min=0)
    for _ in range(max(1, math.ceil(math.log2(max(2, n))))):  # kept up to the root
        kept = kept & torch.gather(kept, 1, jump)
        jump = torch.gather(jump, 1, jump)
    size = kept.sum(dim=1)
    t["counts"].copy_(size)
    order = torch.sort(torch.where(kept, i, n + i), dim=1).values
    t["accepted"].copy_(torch.where(order < n, order, torch.full_like(order, -1)))
    last = torch.where(kept, i, torch.full_like(i, -1)).amax(dim=1)
    at = starts[:-1] + last
    w = e[at]
    failed = there & (parent == last[:, None]) & (i > 0)  # children of the last node: none was kept
    if "draft" in t:
        rest = (w / mass[at][:, None] - d[at] / drawn[at][:, None]).clamp(min=0)
        w = torch.where(failed.any(dim=1)[:, None], rest, w)
    else:
        gone = torch.zeros((b, vocab + 1), dtype=torch.bool, device="cuda")
        gone.scatter_(1, torch.where(failed, token, torch.full_like(token, vocab)), True)
        w = torch.where(gone[:, :vocab], torch.zeros_like(w), w)
    run = torch.cumsum(w, dim=1)
    drawn_at = (run <= t["sample_u"].double()[:, None] * run[:, -1:]).sum(dim=1).clamp(max=vocab - 1)
    t["next"].copy_(torch.where(hot, drawn_at, best[at]))
    return [t["accepted"], t["counts"], t["next"]]


def _plain_prefix(case, t):
    b, n, h, kv, d, page = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim", "page"))
    total, r, groups, most = t["q"].shape[0], h // kv, case["groups"], case["shared"]
    starts, lengths, shared = t["starts"].long(), t["lengths"].long(), t["shared"].long()
    count = starts[1:] - starts[:-1]
    first = t["first"].long()
    owner = _group_of(t["first"], b)
    scale = 1.0 / math.sqrt(d)

    def scores(q, pages, pos):
        """Scores [seqs, kv, rows, keys] of q [seqs, rows, heads, dim], and the values, at positions pos [seqs, keys]."""
        m = q.shape[1]
        where = torch.gather(pages, 1, (pos // page).clamp(0, pages.shape[1] - 1)).clamp(min=0)
        k = t["k_pool"][0][where, :, pos % page].float().permute(0, 2, 3, 1).contiguous()
        v = t["v_pool"][0][where, :, pos % page].float().permute(0, 2, 1, 3).contiguous()
        q = q.float().view(-1, m, kv, r, d).permute(0, 2, 1, 3, 4).reshape(-1, kv, m * r, d)
        return torch.matmul(q, k) * scale, v

    def parts(score, v):
        """Maximum, sum and weighted values of the scores."""
        top = score.amax(dim=-1, keepdim=True)
        e = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        return top, e.sum(dim=-1, keepdim=True), torch.matmul(e, v)

    # the prefix, once for all tokens of a group
    lo, hi = starts[first[:-1]], starts[first[1:]]
    in_group = torch.arange(-(-b // groups) * n, device="cuda")
    token = (lo[:, None] + in_group).clamp(max=total - 1)
    pos = torch.arange(most, device="cuda").expand(groups, most)
    s, v = scores(t["q"][token], t["pages"].long()[first[:-1]], pos)
    s = torch.where((pos < shared[:, None])[:, None, None, :], s, float("-inf"))
    seq, at = _owner(t["starts"], total)
    group = owner[seq]
    place = torch.arange(total, device="cuda") - lo[group]
    m1, l1, o1 = (z.view(groups, kv, -1, r, z.shape[-1]).permute(0, 2, 1, 3, 4)[group, place] for z in parts(s, v))
    # the rest of each sequence
    keys = case["ctx"] + n
    i = torch.arange(n, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=total - 1)
    pos = shared[owner][:, None] + torch.arange(keys, device="cuda")
    s, v = scores(t["q"][token], t["pages"].long(), pos)
    node = pos - lengths[:, None]
    if "mask" in t:
        word = torch.gather(t["mask"][token], 2, (node.clamp(0, n - 1) // 32)[:, None, :].expand(b, n, keys))
        drafted = ((word >> (node.clamp(min=0) % 32)[:, None, :]) & 1) > 0
    else:
        drafted = node[:, None, :] <= i[None, :, None]
    visible = (node < 0)[:, None, :] | (drafted & ((node >= 0) & (node < count[:, None]))[:, None, :])
    s = torch.where(visible[:, None, :, None, :], s.view(b, kv, n, r, keys), float("-inf")).view(b, kv, n * r, keys)
    m2, l2, o2 = (z.view(b, kv, n, r, z.shape[-1]).permute(0, 2, 1, 3, 4)[seq, at] for z in parts(s, v))
    top = torch.maximum(m1, m2)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    w1, w2 = torch.exp(m1 - top), torch.exp(m2 - top)
    mass = w1 * l1 + w2 * l2
    mixed = (w1 * o1 + w2 * o2) / torch.where(mass == 0, torch.ones_like(mass), mass)
    t["y"].copy_(mixed.reshape(total, h, d))
    return [t["y"]]


PLAIN = {"norm": _plain_norm, "append": _plain_append, "verify": _plain_verify, "prefix": _plain_prefix}


# ---- what a pass cannot do without ----

def _bytes(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    """Counted at three quarters of the case's context, prefix and draft, the mean of what prepare makes."""
    kind = case["kind"]
    n = max(1, 0.75 * case.get("nodes", 1))
    rows = case.get("batch", 1) * n
    if kind == "verify":
        model = (2 if case["draft"] == "chain" and case["nodes"] > 1 else 1) * rows * case["vocab"]
        return {"bytes": model * _bytes(case["x"]) + 16 * rows + 20 * case["batch"], "flops": 4 * model}
    h, d, xb = case["heads"], case["dim"], _bytes(case["x"])
    if kind == "norm":
        rows = case["tokens"]
        return {"bytes": 2 * rows * h * d * xb + rows * (4 * case["rot"] + 4) + 4 * d, "flops": rows * h * (4 * d + 3 * case["rot"])}
    kv, cb = case["kv_heads"], _bytes(case["cache"])
    if kind == "append":
        return {"bytes": rows * (2 * h * d + 2 * kv * d) * xb + rows * 2 * kv * d * cb + rows * (4 * case["rot"] + 8) + 8 * d
                + 8 * case["batch"], "flops": rows * (h + kv) * (4 * d + 3 * case["rot"])}
    prefix, ctx = 0.75 * case["shared"], 0.75 * case["ctx"]
    keys = case["groups"] * prefix + case["batch"] * (ctx + n)
    table = 4 * (keys / case["page"] + 3 * case["batch"])
    return {"bytes": keys * 2 * kv * d * cb + 2 * rows * h * d * xb + table,
            "flops": 4.0 * rows * h * d * (prefix + ctx + (n + 1) / 2)}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    t = prepare(case, seed)["tensors"]
    kind, page = case["kind"], case.get("page", 1)

    def turned(x, weight):
        half = case["rot"] // 2
        p = t["positions"].long()
        unit = torch.complex(t["cos"].double(), t["sin"].double())[p].unsqueeze(1)
        x = x.double()
        x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:2], half, 2).contiguous()) * unit
            x[..., :2 * half] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    if kind == "norm":
        return [turned(t["x"], t["q_weight"])]
    starts = t["starts"].tolist()
    if kind == "append":
        kp, vp, k, v = t["k_pool"].double(), t["v_pool"].double(), turned(t["k"], t["k_weight"]), t["v"].double()
        lengths, pages = t["lengths"].tolist(), t["pages"].cpu()
        token, where, slots = [], [], []
        for b in range(case["batch"]):
            for i in range(starts[b + 1] - starts[b]):
                token.append(starts[b] + i)
                where.append(int(pages[b, (lengths[b] + i) // page]))
                slots.append((lengths[b] + i) % page)
        token, where, slots = (torch.tensor(z, device="cuda") for z in (token, where, slots))
        kp[0, where, :, slots], vp[0, where, :, slots] = k[token], v[token]
        return [turned(t["q"], t["q_weight"]), kp, vp]
    if kind == "verify":
        accepted = torch.full(t["accepted"].shape, -1, dtype=torch.int32)
        counts, after = [], []
        tokens, u, v = t["tokens"].tolist(), t["accept_u"].tolist(), t["sample_u"].tolist()
        for b, heat in enumerate(t["temperature"].tolist()):
            lo, n = starts[b], starts[b + 1] - starts[b]
            parents = t["parents"][lo:lo + n].tolist() if "parents" in t else list(range(-1, n - 1))
            path = [0]
            while True:
                row = lo + path[-1]
                children = [i for i in range(1, n) if parents[i] == path[-1]]
                if heat == 0:
                    best = int(t["logits"][row].float().cpu().argmax())
                    kept = next((i for i in children if tokens[lo + i] == best), None)
                    if kept is None:
                        after.append(best)
                        break
                    path.append(kept)
                    continue
                p = torch.softmax(t["logits"][row].double() / heat, dim=0)
                kept = None
                for i in children:
                    token = tokens[lo + i]
                    if "draft" in t:
                        q = torch.softmax(t["draft"][row].double() / heat, dim=0)
                        taken = u[lo + i] * float(q[token]) < float(p[token])
                        rest = (p - q).clamp(min=0)
                    else:
                        taken = u[lo + i] * float(p.sum()) < float(p[token])
                        rest = p.clone()
                        rest[token] = 0
                    if taken:
                        kept = i
                        break
                    p = rest
                if kept is None:
                    c = torch.cumsum(p, 0)
                    after.append(int(torch.searchsorted(c, v[b] * c[-1:], right=True)[0]))
                    break
                path.append(kept)
            counts.append(len(path))
            accepted[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
        return [accepted, torch.tensor(counts, dtype=torch.int32), torch.tensor(after, dtype=torch.int32)]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if work(case)["flops"] > 4e11:
        return None
    out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
    for b, held in enumerate(t["lengths"].tolist()):
        lo, hi = starts[b], starts[b + 1]
        n = hi - lo
        rows = t["pages"][b, :_pages_of(held + n, page)].long()
        seen = torch.ones((n, held + n), dtype=torch.bool, device="cuda")
        if "mask" in t:
            words = t["mask"][lo:hi].long() & 0xFFFFFFFF
            shift = torch.arange(n, device="cuda")
            seen[:, held:] = (words[:, shift // 32] >> (shift % 32)) & 1 == 1
        else:
            seen[:, held:] = torch.arange(n, device="cuda")[None, :] <= torch.arange(n, device="cuda")[:, None]
        for a in range(kv):
            k = t["k_pool"][0, rows, a].reshape(-1, d)[:held + n].double()
            v = t["v_pool"][0, rows, a].reshape(-1, d)[:held + n].double()
            heads = slice(a * (h // kv), (a + 1) * (h // kv))
            q = t["q"][lo:hi, heads].double()
            s = (q.reshape(-1, d) @ k.t().contiguous()).view(n, h // kv, -1) / math.sqrt(d)
            p = torch.nan_to_num(torch.softmax(s.masked_fill(~seen[:, None, :], float("-inf")), dim=-1), nan=0.0)
            out[lo:hi, heads] = (p.reshape(-1, held + n) @ v).view(n, h // kv, d)
    return [out]
