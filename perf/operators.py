"""The operators of decoding with drafted tokens, and the sizes at which their speed counts.

A step of the engine may bring a tree of drafted tokens for each request: row 0 of a request is its last decided token, the
other rows are guesses, and every row names the row before it (its parent).  One pass of the model over all rows tells
which guesses it would have made itself.  Four operators stand around that pass:

  tables   lengths and page lists (on the GPU) become block tables, cache slots, positions and visibility bits of the rows;
  attend   every row attends to its request's cached text and to its own ancestors in the tree;
  accept   the model's choice at every row from its logits, and the longest path of the tree that agrees with it;
  keep     the cache rows of that path move next to the request's text, in every layer.

Lengths and tree sizes follow from a case alone (spread over the range it names); page numbers, trees and values follow
from the seed.
"""
import math

import torch

own = False

SPARE_PAGES = 7


# ---------------------------------------------------------------------------------------------------------- the cases
def listed():
    bf, f32 = "bfloat16", "float32"
    return [
        # one user's request in front of a short tree: nothing but latency
        dict(name="tables-1", kind="tables", requests=1, lo=510, hi=510, nodes_lo=8, nodes=8, page=16, chain=False),
        # a full serving batch, long contexts, trees of 64 rows: the block table is what there is to write
        dict(name="tables-512", kind="tables", requests=512, lo=100, hi=32000, nodes_lo=1, nodes=64, page=16, chain=False),
        # one request with heads as in GPT-2 small, a tree of eight rows
        dict(name="attend-1", kind="attend", dtype=bf, requests=1, lo=510, hi=510, nodes_lo=8, nodes=8, page=16, heads=12,
             kv_heads=12, dim=64, strided=False),
        # a small serving batch of the same model, contexts up to its last position
        dict(name="attend-8", kind="attend", dtype=bf, requests=8, lo=200, hi=990, nodes_lo=32, nodes=32, page=16, heads=12,
             kv_heads=12, dim=64, strided=False),
        # many requests with small trees, three query heads to a key head, queries read from the fused projection
        dict(name="attend-64", kind="attend", dtype=bf, requests=64, lo=500, hi=4000, nodes_lo=4, nodes=16, page=16, heads=12,
             kv_heads=4, dim=64, strided=True),
        # the largest: long documents, wide trees, grouped heads of 128
        dict(name="attend-long", kind="attend", dtype=bf, requests=4, lo=8000, hi=32000, nodes_lo=64, nodes=64, page=64,
             heads=32, kv_heads=8, dim=128, strided=False),
        # the 32-bit path: a small batch
        dict(name="attend-f32-8", kind="attend", dtype=f32, requests=8, lo=100, hi=1000, nodes_lo=16, nodes=16, page=16,
             heads=12, kv_heads=12, dim=64, strided=False),
        # the 32-bit path: odd sizes throughout, heads as in GPT-2 XL
        dict(name="attend-f32-odd", kind="attend", dtype=f32, requests=5, lo=333, hi=7001, nodes_lo=1, nodes=37, page=24,
             heads=25, kv_heads=25, dim=64, strided=True),
        # one user's tree, GPT-2's vocabulary
        dict(name="accept-1", kind="accept", requests=1, lo=510, hi=510, nodes_lo=8, nodes=8, vocab=50257, depth=8),
        # a serving batch of wide trees: the logits are what there is to read
        dict(name="accept-64", kind="accept", requests=64, lo=100, hi=1000, nodes_lo=32, nodes=32, vocab=50257, depth=8),
        # one user's tree, the layers of GPT-2 small
        dict(name="keep-1", kind="keep", dtype=bf, requests=1, lo=510, hi=510, nodes_lo=8, nodes=8, page=16, kv_heads=12,
             dim=64, layers=12, depth=8),
        # a serving batch on the layers of GPT-2 large (short contexts: what lies before the tree is not touched)
        dict(name="keep-32", kind="keep", dtype=bf, requests=32, lo=3, hi=40, nodes_lo=8, nodes=32, page=16, kv_heads=20,
             dim=64, layers=36, depth=8),
    ]


_HEADS = [(12, 12, 64), (25, 25, 64), (20, 20, 64), (12, 4, 64), (32, 8, 128), (16, 2, 128), (6, 3, 32), (8, 8, 16), (10, 2, 80),
          (4, 1, 256), (6, 2, 48)]
_PAGES = [1, 8, 16, 16, 16, 24, 32, 64, 100, 128]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "attend", "attend", "attend", "attend", "accept", "keep"])
    requests = _log(rng, 1, 64)
    nodes = _log(rng, 1, 64)
    nodes_lo = rng.choice([0, 1, nodes]) if requests > 1 else nodes
    if kind == "tables":
        chain = rng.random() < 0.3
        requests = _log(rng, 1, 512)
        return dict(kind=kind, requests=requests, lo=rng.choice([0, 1, 50]), hi=_log(rng, 64, 32000), nodes_lo=nodes_lo,
                    nodes=_log(rng, 64, 512) if chain and requests <= 64 else nodes, page=rng.choice(_PAGES[1:]), chain=chain)
    if kind == "attend":
        heads, kv_heads, dim = rng.choice(_HEADS)
        case = dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), requests=requests, lo=rng.choice([0, 1, 37]),
                    hi=_log(rng, 40, 32000), nodes_lo=nodes_lo, nodes=nodes, page=rng.choice(_PAGES), heads=heads,
                    kv_heads=kv_heads, dim=dim, strided=rng.random() < 0.5)
        top = {c["name"]: work(c) for c in listed()}["attend-long"]
        while work(case)["bytes"] > top["bytes"] or work(case)["flops"] > top["flops"] / (8 if case["dtype"] == "float32" else 1):
            case["hi"] = max(case["lo"] + 1, case["hi"] // 2)
        return case
    if kind == "accept":
        vocab = rng.choice([257, 1000, 32000, 50257, 50257, 131072])
        rows = max(1, 64 * 32 * 50257 // vocab)
        requests = min(requests, rows)
        nodes = max(1, min(nodes, rows // requests))
        return dict(kind=kind, requests=requests, lo=5, hi=_log(rng, 10, 1000), nodes_lo=rng.choice([min(1, nodes), nodes]), nodes=nodes,
                    vocab=vocab, depth=rng.choice([4, 8, 16]))
    heads, kv_heads, dim = rng.choice(_HEADS)
    return dict(kind=kind, dtype=rng.choice(["bfloat16", "float32"]), requests=min(requests, 32), lo=1, hi=rng.randint(2, 40),
                nodes_lo=min(nodes, 32, rng.choice([1, 64])), nodes=min(nodes, 32), page=rng.choice(_PAGES), kv_heads=kv_heads,
                dim=min(dim, 64), layers=_log(rng, 1, 20), depth=rng.choice([4, 8, 16]))


def _spread(lo, hi, n, turn):
    """``n`` whole numbers that fill lo..hi evenly, in a mixed order; the first is hi."""
    if n == 1:
        return [hi]
    return [hi - int((hi - lo) * ((i * turn) % 1.0)) for i in range(n)]


def _lengths(case):
    return _spread(case["lo"], case["hi"], case["requests"], 0.6180339887498949)


def _nodes(case):
    return _spread(case["nodes_lo"], case["nodes"], case["requests"], 0.41421356237309503)


def _words(case):
    return -(-case["nodes"] // 32)


def _pages(case):
    """Pages a request holds, and the width of the block table."""
    held = [-(-(a + n) // case["page"]) for a, n in zip(_lengths(case), _nodes(case))]
    return held, max(16, 1 << (max(max(held), 1) - 1).bit_length())


def _element(case):
    return 2 if case.get("dtype") == "bfloat16" else 4


def work(case):
    lengths, nodes = _lengths(case), _nodes(case)
    S, T = case["requests"], sum(nodes)
    if case["kind"] == "tables":
        held, width = _pages(case)
        words = 0 if case["chain"] else _words(case)
        return {"bytes": 4 * (S + 2 * (S + 1) + (0 if case["chain"] else T) + sum(held) + S * width + 3 * T + S + T * words),
                "flops": T * (1 + words)}
    if case["kind"] == "attend":
        keys = sum(a + n for a, n in zip(lengths, nodes) if n)
        seen = sum(n * (a + 1) for a, n in zip(lengths, nodes))
        held, _ = _pages(case)
        return {"bytes": _element(case) * (2 * keys * case["kv_heads"] * case["dim"] + 2 * T * case["heads"] * case["dim"])
                + 4 * (sum(held) + T * _words(case) + 2 * S),
                "flops": 4 * case["heads"] * case["dim"] * seen}
    if case["kind"] == "accept":
        return {"bytes": 4 * (T * case["vocab"] + 3 * T + S * (case["depth"] + 5)), "flops": T * case["vocab"]}
    moved = sum(min(n, (case["depth"] + 1) // 2) - 1 for n in nodes if n)      # half of the paths' greatest length, row 0 stays
    row = _element(case) * case["kv_heads"] * case["dim"]
    return {"bytes": 2 * max(1, moved) * row * 2 * case["layers"] + 4 * S * (case["depth"] + 4), "flops": 0}


# ---------------------------------------------------------------------------------------------------------- the inputs
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return _ints(out)


def _rows(cu, total):
    """Request and place within the request of each of ``total`` rows."""
    seq = torch.repeat_interleave(torch.arange(cu.numel() - 1, device=cu.device), (cu[1:] - cu[:-1]).long(), output_size=total)
    return seq, torch.arange(total, device=cu.device) - cu.long()[seq]


def _trees(local, gen):
    """Random trees: a row hangs on the one before it or on any earlier row; row 0 of a request is its root."""
    u, w = torch.rand((2, local.numel()), generator=gen, device="cuda")
    any_before = torch.minimum((w * local).long(), (local - 1).clamp(min=0))
    return torch.where(local == 0, -1, torch.where(u < 0.5, local - 1, any_before)).int()


def _reach(parents, cu, most):
    """[S, most, most] of 0 and 1: row j lies on the way from row i to the root (i itself among them)."""
    S = cu.numel() - 1
    seq, local = _rows(cu, parents.numel())
    r = torch.eye(most, device=cu.device).repeat(S, 1, 1)
    has = parents >= 0
    r[seq, local, parents.long().clamp(min=0)] = torch.where(has, 1.0, r[seq, local, parents.long().clamp(min=0)])
    steps = max(1, (most - 1).bit_length())
    for _ in range(steps):                      # twice as many steps up each time
        r = (r @ r > 0).float()
    return r


def _pack_bits(seen, words):
    """[rows, n] of truth values as [rows, words] 32-bit words, bit b of word w for column 32 w + b."""
    rows, n = seen.shape
    full = torch.zeros((rows, 32 * words), dtype=torch.int64, device=seen.device)
    full[:, :n] = seen
    v = (full.view(rows, words, 32) << torch.arange(32, device=seen.device)).sum(-1)
    return torch.where(v >= 1 << 31, v - (1 << 32), v).int()


def _tables(case, gen):
    """Page lists (a random order of a pool's pages) and the block table they make."""
    held, width = _pages(case)
    cu_pages = _starts(held)
    total = sum(held)
    ids = torch.randperm(total + SPARE_PAGES, generator=gen, device="cuda")[:total].int()
    seq, local = _rows(cu_pages, total)
    table = torch.zeros((case["requests"], width), dtype=torch.int32, device="cuda")
    table[seq, local] = ids
    return ids, cu_pages, table, total + SPARE_PAGES


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)
    S, nodes = case["requests"], _nodes(case)
    T, words = sum(nodes), _words(case)
    st = dict(case=case, lengths=_ints(_lengths(case)), cu_nodes=_starts(nodes), total=T)
    seq, local = _rows(st["cu_nodes"], T)
    st["parents"] = None if case.get("chain") else _trees(local, gen)

    def ints(*shape):
        return torch.empty(shape, dtype=torch.int32, device="cuda")

    if case["kind"] == "tables":
        st["pages"], st["cu_pages"], table, _ = _tables(case, gen)
        st.update(block_table=torch.empty_like(table), slots=ints(T), positions=ints(T), token_seq=ints(T), ctx_len=ints(S),
                  ancestors=None if case["chain"] else ints(T, words))
        return st
    if case["kind"] == "accept":
        V = case["vocab"]
        st["logits"] = torch.randn((T, V), generator=gen, device="cuda")
        st["tokens"] = torch.randint(0, V, (T,), generator=gen, device="cuda").int()
        # most drafts are what the model would have said after their parent
        up = (st["cu_nodes"].long()[seq] + st["parents"].long()).clamp(min=0)
        agrees = (torch.rand(T, generator=gen, device="cuda") < 0.7) & (local > 0)
        if T:
            st["tokens"] = torch.where(agrees, st["logits"].argmax(1)[up].int(), st["tokens"])
        st.update(chosen=ints(T), path=ints(S, case["depth"]), accepted=ints(S), next_token=ints(S), new_lengths=ints(S))
        return st
    _, _, st["block_table"], pages = _tables(case, gen)
    dt, Hkv, D, ps = _dtype(case), case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "keep":
        st["planes"] = torch.randn((2 * case["layers"], pages, Hkv, ps, D), generator=gen, device="cuda").to(dt)
        # paths of half the greatest length, rows of the tree in rising order, row 0 first
        keep = torch.clamp(st["cu_nodes"][1:] - st["cu_nodes"][:-1], max=(case["depth"] + 1) // 2)
        most = max(case["nodes"], case["depth"])
        col = torch.arange(most, device="cuda")
        rank = torch.rand((S, most), generator=gen, device="cuda") + 10.0 * (col >= (st["cu_nodes"][1:] - st["cu_nodes"][:-1])[:, None])
        rank[:, 0] = -1.0
        order = rank.argsort(1)[:, :case["depth"]]
        kept = torch.arange(case["depth"], device="cuda") < keep[:, None]
        order = torch.where(kept, order, most).sort(1).values
        st["path"] = torch.where(kept, order, -1).int()
        st["accepted"] = keep.int()
        return st
    # keys, values and queries as a projection leaves them: unit variance, some heads with sharper scores than others
    H = case["heads"]
    pool = torch.randn((2, pages, Hkv, ps, D), generator=gen, device="cuda", dtype=dt)
    wide = (H + 2 * Hkv) * D if case["strided"] else H * D
    q = torch.randn((T, wide), generator=gen, device="cuda")
    q[:, :H * D] *= torch.linspace(0.5, 3.0, H, device="cuda").repeat_interleave(D)
    st.update(q=q.to(dt)[:, :H * D], k_pages=pool[0], v_pages=pool[1], out=torch.empty((T, H * D), dtype=dt, device="cuda"),
              scale=D ** -0.5)
    reach = _reach(st["parents"], st["cu_nodes"], case["nodes"])
    st["ancestors"] = _pack_bits(reach[seq, local] > 0, words)
    return st


# ---------------------------------------------------------------------------------------------------------- plain forms
def _plain_tables(st):
    case, S, T = st["case"], st["case"]["requests"], st["total"]
    ps, (_, width) = case["page"], _pages(case)
    cu, lengths, cu_pages = st["cu_nodes"].long(), st["lengths"].long(), st["cu_pages"].long()
    seq, local = _rows(st["cu_nodes"], T)
    held = cu_pages[1:] - cu_pages[:-1]
    col = torch.arange(width, device="cuda")
    at = (cu_pages[:-1, None] + col).clamp(max=max(0, st["pages"].numel() - 1))
    table = torch.where(col < held[:, None], st["pages"][at], 0)
    place = lengths[seq] + local
    slots = torch.where(place // ps < held[seq], table[seq, (place // ps).clamp(max=width - 1)] * ps + place % ps, -1)
    if st["parents"] is None:
        depth, out = local, {}
    else:
        reach = _reach(st["parents"], st["cu_nodes"], case["nodes"])[seq, local]
        depth = reach.sum(1).long() - 1
        out = {"ancestors": _pack_bits(reach > 0, _words(case))}
    return dict(out, block_table=table.int(), slots=slots.int(), positions=(lengths[seq] + depth).int(), token_seq=seq.int(),
                ctx_len=(lengths + cu[1:] - cu[:-1]).int())


def _plain_attend(st):
    case = st["case"]
    S, N, H, Hkv, D, ps = (case[k] for k in ("requests", "nodes", "heads", "kv_heads", "dim", "page"))
    T, G = st["total"], H // Hkv
    seq, local = _rows(st["cu_nodes"], T)
    lengths = st["lengths"].long()
    q = torch.zeros((S, N, Hkv, G, D), device="cuda")
    q[seq, local] = st["q"].float().reshape(T, Hkv, G, D)
    pos = torch.arange(case["hi"] + N, device="cuda")
    page = st["block_table"].long()[:, pos // ps]
    held = pos < (lengths + (st["cu_nodes"][1:] - st["cu_nodes"][:-1]))[:, None]
    k = st["k_pages"][page, :, pos % ps].float().permute(0, 2, 3, 1)                       # [S, Hkv, D, keys]
    v = torch.where(held[:, :, None, None], st["v_pages"][page, :, pos % ps].float(), 0.0).permute(0, 2, 1, 3)
    bits = ((st["ancestors"][:, :, None] >> torch.arange(32, device="cuda")) & 1).reshape(T, -1)
    seen = torch.zeros((S, N, bits.shape[1]), dtype=torch.bool, device="cuda")
    seen[seq, local] = bits.bool()
    j = pos[None, :] - lengths[:, None]
    in_tree = torch.gather(seen, 2, j.clamp(0, seen.shape[2] - 1)[:, None, :].expand(S, N, -1)) & (j >= 0)[:, None] & held[:, None]
    visible = ((j < 0)[:, None] | in_tree)[:, None, :, None, :]                            # [S, 1, N, 1, keys]
    s = (q.permute(0, 2, 1, 3, 4).reshape(S, Hkv, N * G, D) @ k).view(S, Hkv, N, G, -1) * st["scale"]
    s = torch.where(visible, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.view(S, Hkv, N * G, -1) @ v).view(S, Hkv, N, G, D) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 2, 1, 3, 4).reshape(S, N, H * D)[seq, local].to(st["out"].dtype)


def _plain_accept(st):
    case, S, T = st["case"], st["case"]["requests"], st["total"]
    N, depth, V = case["nodes"], case["depth"], case["vocab"]
    cu, parents, tokens = st["cu_nodes"].long(), st["parents"].long(), st["tokens"].long()
    seq, local = _rows(st["cu_nodes"], T)
    logits = st["logits"]
    top = logits.amax(1, keepdim=True)
    chosen = torch.where(logits == top, torch.arange(V, device="cuda"), V).amin(1)
    said = chosen[(cu[seq] + parents).clamp(min=0)]
    hit = (parents < 0) & (local == 0) | (parents >= 0) & (tokens == said)
    # of several children with the right token only the lowest counts
    grid = torch.full((S, N, 2), -2, device="cuda")
    grid[seq, local] = torch.stack((parents, tokens), 1)
    same = (grid[:, :, None] == grid[:, None]).all(-1)
    first = same.float().argmax(-1) == torch.arange(N, device="cuda")
    ok = torch.zeros((S, N), dtype=torch.bool, device="cuda")
    ok[seq, local] = hit & first[seq, local]
    reach = _reach(st["parents"], st["cu_nodes"], N)
    on = ok & ((reach * ~ok[:, None, :]).sum(-1) == 0)                                     # a row and all rows above it agree
    rows = torch.where(on, torch.arange(N, device="cuda"), N).sort(1).values
    rows = torch.nn.functional.pad(rows, (0, max(0, depth - N)), value=N)[:, :depth]
    path = torch.where(rows < N, rows, -1)
    accepted = (path >= 0).sum(1)
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])[:, 0]
    nxt = torch.where(accepted > 0, chosen[(cu[:-1] + last).clamp(0, max(0, T - 1))], -1)
    return dict(chosen=chosen.int(), path=path.int(), accepted=accepted.int(), next_token=nxt.int(),
                new_lengths=(st["lengths"] + accepted).int())


def _plain_keep(st):
    ps, depth = st["case"]["page"], st["case"]["depth"]
    k = torch.arange(depth, device="cuda")
    live = k < st["accepted"][:, None]
    src = st["lengths"].long()[:, None] + torch.where(live, st["path"].long(), 0)
    dst = st["lengths"].long()[:, None] + torch.where(live, k, 0)
    src, dst = src.reshape(-1), dst.reshape(-1)
    req = torch.arange(st["case"]["requests"], device="cuda").repeat_interleave(depth)
    table = st["block_table"].long()
    rows = st["planes"][:, table[req, src // ps], :, src % ps]
    st["planes"][:, table[req, dst // ps], :, dst % ps] = rows
    return st["planes"]


def run(st):
    case = st["case"]
    if not own:
        return {"tables": _plain_tables, "attend": _plain_attend, "accept": _plain_accept, "keep": _plain_keep}[case["kind"]](st)
    from mini_llm_b200 import ops
    if case["kind"] == "tables":
        ops.draft_tables(st["lengths"], st["cu_nodes"], st["parents"], st["pages"], st["cu_pages"], case["page"],
                         block_table=st["block_table"], slot_mapping=st["slots"], positions=st["positions"],
                         token_seq=st["token_seq"], ctx_len=st["ctx_len"], ancestors=st["ancestors"])
        out = dict(block_table=st["block_table"], slots=st["slots"], positions=st["positions"], token_seq=st["token_seq"],
                   ctx_len=st["ctx_len"])
        return out if st["ancestors"] is None else dict(out, ancestors=st["ancestors"])
    if case["kind"] == "attend":
        ops.tree_attention(st["q"], st["k_pages"], st["v_pages"], st["block_table"], st["lengths"], st["cu_nodes"], st["ancestors"],
                           st["out"], num_heads=case["heads"], num_kv_heads=case["kv_heads"], head_dim=case["dim"],
                           scale=st["scale"], max_nodes=case["nodes"], max_length=case["hi"])
        return st["out"]
    if case["kind"] == "accept":
        ops.accept_drafts(st["tokens"], st["parents"], st["cu_nodes"], st["lengths"], logits=st["logits"], chosen=st["chosen"],
                          path=st["path"], accepted=st["accepted"], next_token=st["next_token"], new_lengths=st["new_lengths"])
        return {k: st[k] for k in ("chosen", "path", "accepted", "next_token", "new_lengths")}
    ops.keep_accepted(st["planes"], st["block_table"], st["lengths"], st["path"], st["accepted"])
    return st["planes"]


# ---------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definition, request by request; the integer outputs of ``tables`` and ``accept`` have no such value."""
    if case["kind"] in ("tables", "accept"):
        return None
    st = prepare(case, seed)
    lengths, table, ps = _lengths(case), st["block_table"].tolist(), case["page"]
    if case["kind"] == "keep":
        planes = st["planes"].double()
        path, accepted = st["path"].tolist(), st["accepted"].tolist()
        before = planes.clone()
        for s, L in enumerate(lengths):
            for k in range(accepted[s]):
                a, b = L + path[s][k], L + k
                planes[:, table[s][b // ps], :, b % ps] = before[:, table[s][a // ps], :, a % ps]
        return planes
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    parents, cu = st["parents"].tolist(), st["cu_nodes"].tolist()
    out = torch.zeros((st["total"], H * D), dtype=torch.float64, device="cuda")
    for s, L in enumerate(lengths):
        n = cu[s + 1] - cu[s]
        if n == 0:
            continue
        keys = L + n
        ids = torch.tensor(table[s][:-(-keys // ps)], device="cuda")
        blocked = torch.ones((n, keys), dtype=torch.bool)
        blocked[:, :L] = False
        for i in range(n):
            j = i
            while j >= 0:
                blocked[i, L + j] = False
                j = parents[cu[s] + j]
        blocked = blocked.cuda()
        for g in range(Hkv):
            K = st["k_pages"][ids, g].double().reshape(-1, D)[:keys]
            V = st["v_pages"][ids, g].double().reshape(-1, D)[:keys]
            for h in range(g * (H // Hkv), (g + 1) * (H // Hkv)):
                x = (st["q"][cu[s]:cu[s + 1], h * D:(h + 1) * D].double() @ K.T) * (1.0 / math.sqrt(D))
                out[cu[s]:cu[s + 1], h * D:(h + 1) * D] = torch.softmax(x.masked_fill(blocked, -math.inf), 1) @ V
    return out
