"""Performance cases of the decoder-step operators: rotary positions, attention of drafted tokens over a paged cache,
and the page operations of that cache.

Together they are one step of a serving program that decodes with drafted tokens: the queries and keys of the new
tokens are rotated and the keys and values written into the cache's pages; every drafted token attends to the
committed tokens of its sequence and to its own ancestors in the draft; the accepted path is then moved to the front,
sequences are forked, leave and come in. One drafted token without a tree is ordinary decoding, a chain of tokens a
prompt taken in pieces.

Inputs are torch tensors on the GPU made from the seed. With `own` the framework's entry points read and write them in
place; without it the same results come from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One new token of one sequence, the decode workload's 16 heads of 128: rotate, append (latency).
        dict(name="append_token", kind="append", batch=1, nodes=1, ctx=517, heads=16, kv_heads=16, dim=128, rot=128,
             interleaved=False, x="f32", cache="bf16", page=16),
        # 32 sequences with drafts of up to 16 tokens, shared key heads, a quarter of the head rotated in neighbour pairs.
        dict(name="append_drafts", kind="append", batch=32, nodes=16, ctx=900, heads=32, kv_heads=8, dim=128, rot=32,
             interleaved=True, x="bf16", cache="bf16", page=32),
        # The queries of a long prompt, f32.
        dict(name="rotary_prompt", kind="rotary", tokens=8191, heads=32, dim=128, rot=128, interleaved=False, x="f32"),
        # One token of one sequence: 16 heads of 128 with their own keys, f32 activations over a bf16 cache (latency).
        dict(name="attend_token", kind="attend", batch=1, nodes=1, ctx=517, heads=16, kv_heads=16, dim=128, x="f32",
             cache="bf16", page=16, mask="chain"),
        # Eight sequences, drafted trees of up to 16 nodes, bf16 throughout.
        dict(name="attend_tree", kind="attend", batch=8, nodes=16, ctx=2048, heads=32, kv_heads=8, dim=128, x="bf16",
             cache="bf16", page=64, mask="tree"),
        # Many sequences, one token each (ordinary batched decoding).
        dict(name="attend_batch", kind="attend", batch=64, nodes=1, ctx=2000, heads=32, kv_heads=8, dim=128, x="f32",
             cache="bf16", page=32, mask="chain"),
        # Large trees over long contexts.
        dict(name="attend_long", kind="attend", batch=4, nodes=64, ctx=32768, heads=32, kv_heads=8, dim=128, x="bf16",
             cache="bf16", page=64, mask="tree"),
        # An f32 cache, heads of 80, pages that are no power of two and end inside a tile.
        dict(name="attend_f32", kind="attend", batch=3, nodes=7, ctx=1100, heads=12, kv_heads=12, dim=80, x="f32",
             cache="f32", page=24, mask="tree"),
        # A piece of a prompt after earlier pieces: a chain of tokens.
        dict(name="attend_chunk", kind="attend", batch=2, nodes=500, ctx=3500, heads=16, kv_heads=4, dim=128, x="bf16",
             cache="bf16", page=64, mask="chain"),
        # Pages of a whole model copied, as when a shared prefix is made private.
        dict(name="pages_copy", kind="copy", layers=16, pages=512, page=32, kv_heads=8, dim=128, cache="bf16", count=200),
        # Every sequence forks into new ones (several answers to one prompt), part-filled pages copied.
        dict(name="pages_fork", kind="fork", layers=16, batch=16, copies=3, ctx=1000, page=32, kv_heads=8, dim=128,
             cache="bf16"),
        # The accepted path of each draft moved to the front of it, all layers.
        dict(name="pages_compact", kind="compact", layers=16, batch=16, nodes=24, depth=6, ctx=700, page=16, kv_heads=8,
             dim=128, cache="bf16"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append", "rotary", "attend", "attend", "attend", "attend", "copy", "fork", "compact", "admit"))
    kv_heads = rng.choice((1, 2, 4, 8, 12))
    heads = kv_heads * rng.choice((1, 1, 2, 4, 5, 8))
    dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
    x, cache = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f32")))
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 100, 128))
    rot = dim // rng.choice((1, 1, 2, 4))
    interleaved = rng.random() < 0.5
    layers = rng.choice((1, 2, 8, 16))
    held = dict(kv_heads=kv_heads, dim=dim, cache=cache, page=page)
    if kind == "rotary":
        case = dict(tokens=_size(rng, 1, 8191), heads=heads, dim=dim, rot=rot, interleaved=interleaved, x=x)
    elif kind == "append":
        case = dict(batch=_size(rng, 1, 64), nodes=_size(rng, 1, 48), ctx=_size(rng, 1, 3000), heads=heads, rot=rot,
                    interleaved=interleaved, x=x, **held)
    elif kind == "attend":
        case = dict(batch=_size(rng, 1, 64), nodes=rng.choice((1, _size(rng, 2, 64), _size(rng, 2, 500))),
                    ctx=_size(rng, 1, 30000), heads=heads, x=x, mask=rng.choice(("tree", "chain")), **held)
    elif kind == "copy":
        case = dict(layers=layers, pages=0, count=_size(rng, 1, 200), **held)
    elif kind == "fork":
        case = dict(layers=layers, batch=_size(rng, 1, 16), copies=rng.randint(1, 4), ctx=_size(rng, 1, 1000), **held)
    elif kind == "compact":
        nodes = _size(rng, 2, 64)
        case = dict(layers=layers, batch=_size(rng, 1, 32), nodes=nodes, depth=rng.randint(1, min(nodes, 12)),
                    ctx=_size(rng, 1, 1000), **held)
    else:
        case = dict(layers=1, batch=_size(rng, 1, 128), ctx=_size(rng, 1, 4000), kv_heads=1, dim=64, cache=cache, page=page)
    case = dict(kind=kind, **case)
    while _too_large(case):  # nothing above the largest listed case of its kind
        side = next(k for k in ("tokens", "count", "batch", "nodes", "ctx", "layers") if case.get(k, 1) > 1)
        case[side] = max(1, case[side] * 3 // 4)
    if kind == "copy":
        case["pages"] = 2 * case["count"] + rng.randint(1, 60)
    if kind == "compact":
        case["depth"] = min(case["depth"], case["nodes"])
    return case


def _too_large(case):
    most = [work(c) for c in listed() if c["kind"] == case["kind"]]
    need = work(case)
    tokens = case.get("batch", 1) * (case.get("ctx", 0) + case.get("nodes", 1) + case.get("page", 0))
    pool = tokens * case.get("layers", 1) * case.get("kv_heads", 1) * case["dim"] if "batch" in case else 0
    return pool > 3e8 or any(need[k] > max(w[k] for w in most) for k in need if most)


# ---- inputs ----

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))


def _pages_of(tokens, page):
    return -(-tokens // page)


def _lengths(case, g, count):
    """Committed tokens of each sequence: from half the case's context up to all of it."""
    ctx = case["ctx"]
    return torch.randint(max(0, ctx // 2), ctx + 1, (count,), generator=g, device="cuda", dtype=torch.int32)


def _tables(held, page, num_pages, max_pages, g):
    """Page tables [seqs, max_pages] of sequences that hold `held` tokens, on pages in no order; -1 past the end."""
    need = (held.long() + page - 1) // page
    at = torch.arange(max_pages, device="cuda")
    used = at[None, :] < need[:, None]
    order = torch.randperm(num_pages, generator=g, device="cuda").to(torch.int32)
    index = torch.cumsum(used.flatten(), 0).view(used.shape) - 1
    return torch.where(used, order[index.clamp(min=0)], torch.full_like(index, -1, dtype=torch.int32)).contiguous()


def _pool(case, layers, num_pages, g):
    """Keys and values, [layer, page, head, slot, dim]: a cache in use, so unused slots hold old values."""
    shape = (layers, num_pages, case["kv_heads"], case["page"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["cache"]])
    return k, torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["cache"]])


def _references(pages, num_pages):
    flat = pages.flatten().long()
    return torch.zeros(num_pages + 1, dtype=torch.int32, device="cuda").index_add_(
        0, torch.where(flat < 0, torch.full_like(flat, num_pages), flat),
        torch.ones(flat.numel(), dtype=torch.int32, device="cuda"))[:num_pages].contiguous()


def _angles(case, rows):
    """cos and sin of every position, made once by a program when it loads a model (long contexts: frequencies / 2)."""
    r = case["rot"]
    f = 10000.0 ** (-torch.arange(0, r // 2, device="cuda", dtype=torch.float64) * 2.0 / r) / 2.0
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cos(a).float(), torch.sin(a).float()


def _drafts(case, g):
    """Node counts of each sequence's draft, parents (-1: follows the committed tokens) and depths, [batch, nodes]."""
    b, n = case["batch"], case["nodes"]
    spread = n - torch.arange(b, device="cuda") * 5 % (n // 2 + 1)  # half the draft's room up to all of it
    count = spread[torch.randperm(b, generator=g, device="cuda")].clamp(min=1)
    i = torch.arange(n, device="cuda")
    back = (torch.rand((b, n), generator=g, device="cuda") * torch.clamp(i, max=6)).long()
    parent = i - 1 - back  # one of the six nodes before
    return count, parent


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


def prepare(case, seed):
    g = _generator(seed)
    t = {}
    kind, page = case["kind"], case.get("page", 1)

    def normal(*shape, dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[dtype])

    if kind == "rotary":
        n, h, d = case["tokens"], case["heads"], case["dim"]
        t["x"] = normal(n, h, d, dtype=case["x"])
        t["y"] = torch.empty_like(t["x"])
        start = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        t["positions"] = torch.arange(start, start + n, device="cuda", dtype=torch.int32)
        t["cos"], t["sin"] = _angles(case, start + n)
    elif kind in ("append", "attend"):
        b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        t["lengths"] = _lengths(case, g, b)
        count, parent = _drafts(case, g)
        start = torch.zeros(b + 1, dtype=torch.int64, device="cuda")
        start[1:] = torch.cumsum(count, 0)
        total = int(start[-1])
        t["starts"] = start.to(torch.int32)
        max_pages = _pages_of(case["ctx"] + case["nodes"], page)
        num_pages = b * max_pages + 3
        t["pages"] = _tables(t["lengths"] + count.to(torch.int32), page, num_pages, max_pages, g)
        t["k_pool"], t["v_pool"] = _pool(case, 1, num_pages, g)
        used = torch.arange(case["nodes"], device="cuda")[None, :] < count[:, None]
        t["q"] = normal(total, h, d, dtype=case["x"])
        t["y"] = torch.empty_like(t["q"])
        seen = _ancestors(parent)
        if kind == "append":
            t["k"], t["v"] = normal(total, kv, d, dtype=case["x"]), normal(total, kv, d, dtype=case["x"])
            t["positions"] = (t["lengths"][:, None] + seen.sum(2) - 1)[used].to(torch.int32)
            t["cos"], t["sin"] = _angles(case, case["ctx"] + case["nodes"])
        elif case["mask"] == "tree":
            # one node in sixteen is a place in the draft that was not filled: it sees committed tokens only
            seen &= (torch.rand((b, case["nodes"], 1), generator=g, device="cuda") > 1 / 16)
            t["mask"] = _bits(seen[used])
    elif kind == "copy":
        t["k_pool"], t["v_pool"] = _pool(case, case["layers"], case["pages"], g)
        order = torch.randperm(case["pages"], generator=g, device="cuda").to(torch.int32)
        t["source"], t["target"] = order[:case["count"]].clone(), order[case["count"]:2 * case["count"]].clone()
    elif kind == "fork":
        b, n = case["batch"], case["batch"] * case["copies"]
        most = _pages_of(case["ctx"], page)
        num_pages = b * most + n + 5
        lengths = _lengths(case, g, b)
        t["lengths"] = torch.cat((lengths, torch.zeros(n, dtype=torch.int32, device="cuda")))
        t["pages"] = torch.full((b + n, most + 2), -1, dtype=torch.int32, device="cuda")
        t["pages"][:b, :most] = _tables(lengths, page, num_pages, most, g)
        t["references"] = _references(t["pages"], num_pages)
        t["k_pool"], t["v_pool"] = _pool(case, case["layers"], num_pages, g)
        t["source"] = torch.arange(n, device="cuda", dtype=torch.int32) % b
        t["target"] = b + torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        t["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    elif kind == "compact":
        b, n = case["batch"], case["nodes"]
        t["lengths"] = _lengths(case, g, b)
        max_pages = _pages_of(case["ctx"] + n, page)
        t["pages"] = _tables(t["lengths"] + n, page, b * max_pages + 1, max_pages, g)
        t["k_pool"], t["v_pool"] = _pool(case, case["layers"], b * max_pages + 1, g)
        t["sequences"] = torch.arange(b, device="cuda", dtype=torch.int32)
        pick = torch.argsort(torch.rand((b, n), generator=g, device="cuda"), dim=1)[:, :case["depth"]]
        t["accepted"] = torch.sort(pick, dim=1).values.to(torch.int32).contiguous()
        t["counts"] = torch.randint(0, case["depth"] + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        t["new_lengths"] = torch.empty_like(t["lengths"])
    else:  # admit: half of the sequences are done; their pages are freed and as many new prompts are given pages
        b = case["batch"]
        stay = (b + 1) // 2
        most = _pages_of(case["ctx"], page)
        num_pages = (b + 1) * most + 7
        t["lengths"] = _lengths(case, g, b)
        t["pages"] = _tables(t["lengths"], page, num_pages, most, g)
        t["references"] = _references(t["pages"], num_pages)
        t["k_pool"], t["v_pool"] = _pool(case, 1, num_pages, g)
        t["sequences"] = torch.randperm(b, generator=g, device="cuda").to(torch.int32)[:stay].contiguous()
        t["needs"] = torch.randint(1, case["ctx"] + 1, (stay,), generator=g, device="cuda", dtype=torch.int32)
        t["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
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
    if kind == "rotary":
        return [s.prepare_rotary(d["x"], d["positions"], d["cos"], d["sin"], d["y"], interleaved=case["interleaved"])], [t["y"]]
    cache = KvCache(d["k_pool"], d["v_pool"])
    if kind == "copy":
        return [s.prepare_kv_copy(cache, d["source"], d["target"])], [t["k_pool"], t["v_pool"]]
    table = KvTable(d["pages"], d["lengths"], d.get("references"), d.get("missing"))
    if kind == "append":
        return [s.prepare_rotary_append(d["q"], d["k"], d["v"], d["positions"], d["cos"], d["sin"], d["y"], cache, table,
                                        d["starts"], interleaved=case["interleaved"])], [t["y"], t["k_pool"], t["v_pool"]]
    if kind == "attend":
        return [s.prepare_tree_attention(d["q"], cache, table, d["starts"], d["y"], max_nodes=case["nodes"],
                                         max_tokens=case["ctx"] + case["nodes"], mask=d.get("mask"),
                                         scale=1.0 / math.sqrt(case["dim"]))], [t["y"]]
    if kind == "fork":
        return [s.prepare_kv_fork(cache, table, d["source"], d["target"])], [
            t[n] for n in ("pages", "lengths", "references", "missing", "k_pool", "v_pool")]
    if kind == "compact":
        return [s.prepare_kv_compact(cache, table, d["sequences"], d["accepted"], d["counts"], d["new_lengths"])], [
            t[n] for n in ("new_lengths", "k_pool", "v_pool")]
    return [s.prepare_kv_free(cache, table, d["sequences"]), s.prepare_kv_reserve(cache, table, d["sequences"], d["needs"])], [
        t[n] for n in ("pages", "lengths", "references", "missing")]


# ---- the plain forms ----

def _rotated(x, positions, cos, sin, interleaved):
    """x [tokens, heads, dim] in 32 bits, its first 2 · cos.shape[1] dimensions rotated."""
    half = cos.shape[1]
    c, s = cos[positions.long()][:, None, :], sin[positions.long()][:, None, :]
    x = x.float()
    part = x[..., :2 * half]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_rotary(case, t):
    t["y"].copy_(_rotated(t["x"], t["positions"], t["cos"], t["sin"], case["interleaved"]))
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
    t["y"].copy_(_rotated(t["q"], *turn))
    t["k_pool"][0, page, :, slot] = _rotated(t["k"], *turn).to(t["k_pool"].dtype)
    t["v_pool"][0, page, :, slot] = t["v"].to(t["v_pool"].dtype)
    return [t["y"], t["k_pool"], t["v_pool"]]


def _plain_attend(case, t):
    b, n, h, kv, d, page = (case[k] for k in ("batch", "nodes", "heads", "kv_heads", "dim", "page"))
    total, g, keys = t["q"].shape[0], h // kv, case["ctx"] + n
    starts, lengths = t["starts"].long(), t["lengths"].long()
    count = starts[1:] - starts[:-1]
    pos = torch.arange(keys, device="cuda")
    where = t["pages"].long()[:, pos // page].clamp(min=0)  # [batch, keys]
    k = t["k_pool"][0][where, :, pos % page].float().permute(0, 2, 3, 1).contiguous()  # [batch, kv, dim, keys]
    v = t["v_pool"][0][where, :, pos % page].float().permute(0, 2, 1, 3).contiguous()  # [batch, kv, keys, dim]
    i = torch.arange(n, device="cuda")
    token = (starts[:-1, None] + i).clamp(max=total - 1)  # [batch, nodes]
    q = t["q"][token].float().view(b, n, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * g, d)
    node = pos[None, :] - lengths[:, None]  # [batch, keys]: number in the draft, negative where committed
    if "mask" in t:
        word = torch.gather(t["mask"][token], 2, (node.clamp(0, n - 1) // 32)[:, None, :].expand(b, n, keys))
        drafted = ((word >> (node.clamp(min=0) % 32)[:, None, :]) & 1) > 0
    else:
        drafted = node[:, None, :] <= i[None, :, None]
    visible = (node < 0)[:, None, :] | (drafted & ((node >= 0) & (node < count[:, None]))[:, None, :])
    score = torch.matmul(q, k) * (1.0 / math.sqrt(d))
    score = torch.where(visible[:, None, :, None, :], score.view(b, kv, n, g, keys), float("-inf"))
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    mass = weight.sum(dim=-1, keepdim=True)
    mixed = torch.matmul(weight.view(b, kv, n * g, keys), v).view(b, kv, n, g, d)
    mixed = mixed / torch.where(mass == 0, torch.ones_like(mass), mass)
    seq, at = _owner(t["starts"], total)
    t["y"].copy_(mixed.permute(0, 2, 1, 3, 4).reshape(b, n, h, d)[seq, at])
    return [t["y"]]


def _plain_copy(case, t):
    s, d = t["source"].long(), t["target"].long()
    for pool in (t["k_pool"], t["v_pool"]):
        pool[:, d] = pool[:, s]
    return [t["k_pool"], t["v_pool"]]


def _add_references(t, pages, step):
    """references[p] += step for every page p >= 0 of `pages`."""
    spare = t["references"].shape[0]
    r = torch.cat((t["references"], torch.zeros(1, dtype=torch.int32, device="cuda")))
    flat = pages.flatten().long()
    r.index_add_(0, torch.where(flat < 0, torch.full_like(flat, spare), flat), torch.full_like(flat, step, dtype=torch.int32))
    t["references"].copy_(r[:spare])


def _free_pages(t, most):
    """The lowest `most` pages that nothing refers to."""
    pages = t["references"].shape[0]
    number = torch.arange(pages, device="cuda")
    return torch.sort(torch.where(t["references"] <= 0, number, torch.full_like(number, pages))).values[:most]


def _plain_fork(case, t):
    src, dst, page = t["source"].long(), t["target"].long(), case["page"]
    _add_references(t, t["pages"][dst], -1)
    lengths = t["lengths"][src]
    full, rest = lengths // page, lengths % page
    at = torch.arange(t["pages"].shape[1], device="cuda")
    rows = torch.where(at[None, :] < full[:, None], t["pages"][src], torch.full_like(t["pages"][src], -1))
    _add_references(t, rows, 1)
    rank = torch.cumsum((rest > 0).long(), 0) - 1
    fresh = _free_pages(t, src.numel())[rank.clamp(min=0)].to(torch.int32)
    fresh = torch.where(rest > 0, fresh, torch.full_like(fresh, -1))
    rows = torch.where((at[None, :] == full[:, None]) & (rest > 0)[:, None], fresh[:, None], rows)
    _add_references(t, fresh, 1)
    old = t["pages"][src, full.long().clamp(max=t["pages"].shape[1] - 1)].long().clamp(min=0)
    slot = torch.arange(page, device="cuda")
    keep = (slot[None, :] < rest[:, None])[None, :, None, :, None]
    to = torch.where(rest > 0, fresh, old.to(torch.int32)).long()
    for pool in (t["k_pool"], t["v_pool"]):
        pool[:, to] = torch.where(keep, pool[:, old], pool[:, to])
    t["pages"][dst] = rows
    t["lengths"][dst] = lengths
    t["missing"].zero_()
    return [t[n] for n in ("pages", "lengths", "references", "missing", "k_pool", "v_pool")]


def _plain_compact(case, t):
    page, depth = case["page"], case["depth"]
    i = torch.arange(depth, device="cuda")
    lengths = t["lengths"].long()
    to = lengths[:, None] + i
    taken = i[None, :] < t["counts"][:, None]
    at = torch.where(taken, lengths[:, None] + t["accepted"].long(), to)
    b = t["sequences"].long()[:, None]
    from_page, to_page = t["pages"][b, at // page].long(), t["pages"][b, to // page].long()
    for pool in (t["k_pool"], t["v_pool"]):
        pool[:, to_page, :, to % page] = pool[:, from_page, :, at % page]
    t["new_lengths"].copy_(t["lengths"] + t["counts"])
    return [t[n] for n in ("new_lengths", "k_pool", "v_pool")]


def _plain_admit(case, t):
    rows, page = t["sequences"].long(), case["page"]
    _add_references(t, t["pages"][rows], -1)
    need = (t["needs"].long() + page - 1) // page
    first = torch.cumsum(need, 0) - need
    at = torch.arange(t["pages"].shape[1], device="cuda")
    index = first[:, None] + at
    free = _free_pages(t, t["references"].shape[0])
    taken = at[None, :] < need[:, None]
    given = torch.where(taken, free[index.clamp(max=free.numel() - 1)], torch.full_like(index, -1)).to(torch.int32)
    _add_references(t, given, 1)
    t["pages"][rows] = given
    t["lengths"][rows] = 0
    t["missing"].zero_()
    return [t[n] for n in ("pages", "lengths", "references", "missing")]


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend, "copy": _plain_copy,
         "fork": _plain_fork, "compact": _plain_compact, "admit": _plain_admit}


# ---- what a pass cannot do without ----

def _bytes(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    """Counted at three quarters of the case's context and draft, the mean of what prepare makes."""
    kind = case["kind"]
    if kind == "rotary":
        n, h, d, r = case["tokens"], case["heads"], case["dim"], case["rot"]
        return {"bytes": 2 * n * h * d * _bytes(case["x"]) + n * (4 * r + 4), "flops": 3 * n * h * r}
    if kind in ("append", "attend"):
        b, n, ctx = case["batch"], max(1, 0.75 * case["nodes"]), 0.75 * case["ctx"]
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        rows = b * n
        table = 4 * b * ((ctx + n) / case["page"] + 2)
    if kind == "append":
        r = case["rot"]
        return {"bytes": rows * (2 * h * d + 2 * kv * d) * _bytes(case["x"]) + rows * 2 * kv * d * _bytes(case["cache"])
                + rows * (4 * r + 8) + 8 * b, "flops": 3 * rows * (h + kv) * r}
    if kind == "attend":
        return {"bytes": b * (ctx + n) * 2 * kv * d * _bytes(case["cache"]) + 2 * rows * h * d * _bytes(case["x"]) + table,
                "flops": 4.0 * rows * h * d * (ctx + (n + 1) / 2)}
    slot = 2 * case["layers"] * case["kv_heads"] * case["dim"] * _bytes(case["cache"])  # one token's keys and values
    if kind == "copy":
        return {"bytes": case["count"] * (2 * case["page"] * slot + 8), "flops": 0}
    if kind == "fork":
        n = case["batch"] * case["copies"]
        pages = 0.75 * case["ctx"] / case["page"]
        return {"bytes": n * (case["page"] / 2 * 2 * slot + 8 * pages + 16) + 8 * (case["batch"] * pages + n), "flops": 0}
    if kind == "compact":
        return {"bytes": case["batch"] * (case["depth"] / 2 * (2 * slot + 4) + 16), "flops": 0}
    pages = 0.5 * case["ctx"] / case["page"]
    return {"bytes": 4 * case["batch"] * (2 * pages + 4) + 8 * (case["batch"] + 1) * _pages_of(case["ctx"], case["page"]), "flops": 0}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    t = prepare(case, seed)["tensors"]
    kind, page = case["kind"], case.get("page", 1)

    def turned(x):
        half = case["rot"] // 2
        p = t["positions"].long()
        unit = torch.complex(t["cos"].double(), t["sin"].double())[p].unsqueeze(1)
        x = x.double().clone()
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:2], half, 2).contiguous()) * unit
            x[..., :2 * half] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * unit
            x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    if kind == "rotary":
        return [turned(t["x"])]
    if kind == "append":
        kp, vp, k, v = t["k_pool"].double(), t["v_pool"].double(), turned(t["k"]), t["v"].double()
        starts, lengths, pages = t["starts"].tolist(), t["lengths"].tolist(), t["pages"].cpu()
        token, where, slots = [], [], []
        for b in range(case["batch"]):
            for i in range(starts[b + 1] - starts[b]):
                token.append(starts[b] + i)
                where.append(int(pages[b, (lengths[b] + i) // page]))
                slots.append((lengths[b] + i) % page)
        token, where, slots = (torch.tensor(z, device="cuda") for z in (token, where, slots))
        kp[0, where, :, slots], vp[0, where, :, slots] = k[token], v[token]
        return [turned(t["q"]), kp, vp]
    if kind == "attend":
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        if work(case)["flops"] > 2e12:
            return None
        out = torch.zeros(t["q"].shape, dtype=torch.float64, device="cuda")
        starts, lengths = t["starts"].tolist(), t["lengths"].tolist()
        for b in range(case["batch"]):
            lo, hi, held = starts[b], starts[b + 1], lengths[b]
            n = hi - lo
            rows = t["pages"][b, :_pages_of(held + n, page)].long()
            seen = torch.ones((n, held + n), dtype=torch.bool, device="cuda")
            for i in range(n):
                if "mask" not in t:
                    seen[i, held + i + 1:] = False
            if "mask" in t:
                words = t["mask"][lo:hi].long() & 0xFFFFFFFF
                shift = torch.arange(n, device="cuda")
                seen[:, held:] = (words[:, shift // 32] >> (shift % 32)) & 1 == 1
            for a in range(kv):
                k = t["k_pool"][0, rows, a].reshape(-1, d)[:held + n].double()
                v = t["v_pool"][0, rows, a].reshape(-1, d)[:held + n].double()
                heads = slice(a * (h // kv), (a + 1) * (h // kv))
                q = t["q"][lo:hi, heads].double()
                s = (q.reshape(-1, d) @ k.t().contiguous()).view(n, h // kv, -1) / math.sqrt(d)
                s = s.masked_fill(~seen[:, None, :], float("-inf"))
                p = torch.nan_to_num(torch.softmax(s, dim=-1), nan=0.0)
                out[lo:hi, heads] = (p.reshape(-1, held + n) @ v).view(n, h // kv, d)
        return [out]
    if kind == "copy":
        kp, vp = t["k_pool"].double(), t["v_pool"].double()
        for a, b in zip(t["source"].tolist(), t["target"].tolist()):
            kp[:, b], vp[:, b] = kp[:, a].clone(), vp[:, a].clone()
        return [kp, vp]
    if kind == "compact":
        kp, vp = t["k_pool"].double(), t["v_pool"].double()
        pages, lengths, counts = t["pages"].tolist(), t["lengths"].tolist(), t["counts"].tolist()
        for b, path in enumerate(t["accepted"].tolist()):
            for i, node in enumerate(path[:counts[b]]):
                f, g = lengths[b] + node, lengths[b] + i
                for pool in (kp, vp):
                    pool[:, pages[b][g // page], :, g % page] = pool[:, pages[b][f // page], :, f % page].clone()
        return [None, kp, vp]
    if kind == "fork":
        kp, vp = t["k_pool"].double(), t["v_pool"].double()
        unused = [p for p, r in enumerate(t["references"].tolist()) if r <= 0]
        pages, lengths = t["pages"].tolist(), t["lengths"].tolist()
        for row in t["source"].tolist():
            full, rest = lengths[row] // page, lengths[row] % page
            if rest:
                fresh, old = unused.pop(0), pages[row][full]
                for pool in (kp, vp):
                    pool[:, fresh, :, :rest] = pool[:, old, :, :rest]
        return [None, None, None, None, kp, vp]
    return None  # whole numbers, and values that are moved and not computed
