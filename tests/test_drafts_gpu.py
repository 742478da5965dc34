"""The kernels of decoding with drafted tokens, each against its plain statement in 64 bits (tests/plain_drafts.py), at the sizes
and masks where they can go wrong."""
import math
import random

import pytest
import torch

import plain_drafts as P

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def ops():
    from mini_llm_b200 import ops as o
    o.library()
    return o


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def tree(n, rng, chain=0.5):
    return [-1 if i == 0 else i - 1 if rng.random() < chain else rng.randrange(i) for i in range(n)]


def page_lists(places, ps, rng):
    """A page list for each number of places, from a shuffled pool, and the pool's size."""
    need = [-(-p // ps) for p in places]
    ids = list(range(sum(need) + 3))
    rng.shuffle(ids)
    out = []
    for n in need:
        out.append(ids[:n])
        ids = ids[n:]
    return out, sum(need) + 3


# ------------------------------------------------------------------------------------------------ tables
def run_tables(ops, lengths, trees, pages, ps, width, words, ancestors=True):
    chain = isinstance(trees[0], int)
    counts = [t if chain else len(t) for t in trees]
    T, S = sum(counts), len(trees)
    def full(*shape):
        return torch.full(shape, -77, dtype=torch.int32, device=DEV)
    got = dict(block_table=full(S, width), slots=full(T), positions=full(T), token_seq=full(T), ctx_len=full(S),
               ancestors=full(T, words) if ancestors else None)
    ops.draft_tables(ints(lengths), ints(starts(counts)), None if chain else ints([p for t in trees for p in t]),
                     ints([p for l in pages for p in l]), ints(starts([len(l) for l in pages])), ps,
                     block_table=got["block_table"], slot_mapping=got["slots"], positions=got["positions"],
                     token_seq=got["token_seq"], ctx_len=got["ctx_len"], ancestors=got["ancestors"])
    return got


def same_tables(got, want):
    for k, v in got.items():
        if v is not None:
            assert v.tolist() == want[k], k


@pytest.mark.parametrize("words", [1, 2, 8])
@pytest.mark.parametrize("ps", [1, 3, 16, 100])
def test_tables_of_trees(ops, words, ps):
    rng = random.Random(words * 1000 + ps)
    most = 32 * words
    counts = [1, most, 0, most - 1, 2, 33 if words > 1 else 31, 17]
    lengths = [0, 1, 40, 1023, ps, 5 * ps - 1, 700]
    trees = [tree(n, rng, c) for n, c in zip(counts, (0.5, 1.0, 0.5, 0.0, 0.5, 0.9, 0.5))]
    pages, _ = page_lists([a + n for a, n in zip(lengths, counts)], ps, rng)
    width = max(map(len, pages)) + 2
    same_tables(run_tables(ops, lengths, trees, pages, ps, width, words), P.tables(lengths, trees, pages, ps, width, words))


def test_tables_where_pages_are_missing_given_back_or_more_than_the_table_holds(ops):
    """Rows without a page are stored nowhere; a page that was given back is none; the table is cut at its width."""
    lengths, trees = [30, 5, 12], [[-1, 0, 0, 1], [-1, 0], [-1, 0, 1]]
    pages = [[4, -1, 9, 2, 8], [7], [3, 5, -1, -1]]
    same_tables(run_tables(ops, lengths, trees, pages, 6, 4, 1), P.tables(lengths, trees, pages, 6, 4, 1))


def test_tables_of_parents_that_are_no_earlier_row(ops):
    """A row that names itself, a later row or nonsense hangs on the text."""
    trees = [[-1, 1, 5, -9, 2, 4], [3, 0, 0, 2]]
    pages = [[1, 2], [3, 4]]
    same_tables(run_tables(ops, [3, 9], trees, pages, 8, 3, 1), P.tables([3, 9], trees, pages, 8, 3, 1))


def test_rows_past_the_bits_take_no_part(ops):
    rng = random.Random(3)
    trees = [tree(40, rng), tree(300, rng), tree(5, rng)]
    pages, _ = page_lists([50, 310, 20], 16, rng)
    for words in (1, 8):
        same_tables(run_tables(ops, [10, 10, 15], trees, pages, 16, 32, words),
                    P.tables([10, 10, 15], trees, pages, 16, 32, words))


@pytest.mark.parametrize("bits", [0, 2])
def test_tables_of_rows_that_follow_one_another(ops, bits):
    """Prompt portions of any length; with bits, every row sees those before it as far as the words reach."""
    rng = random.Random(5)
    lengths, counts = [0, 700, 31, 0, 64], [1, 600, 33, 0, 64]
    pages, _ = page_lists([a + n for a, n in zip(lengths, counts)], 16, rng)
    got = run_tables(ops, lengths, counts, pages, 16, 2000, max(bits, 1), ancestors=bits > 0)
    want = P.tables(lengths, counts, pages, 16, 2000, max(bits, 1))
    same_tables(got, want)


def test_tables_of_many_requests(ops):
    rng = random.Random(8)
    S = 700
    lengths = [rng.randrange(0, 3000) for _ in range(S)]
    trees = [tree(rng.randrange(0, 20), rng) for _ in range(S)]
    pages, _ = page_lists([a + len(t) for a, t in zip(lengths, trees)], 16, rng)
    same_tables(run_tables(ops, lengths, trees, pages, 16, 256, 1), P.tables(lengths, trees, pages, 16, 256, 1))


# ------------------------------------------------------------------------------------------------ attention
def bits_of(seen, words):
    out = []
    for row in seen:
        v = [sum(1 << b for b in range(32) if 32 * w + b < len(row) and row[32 * w + b]) for w in range(words)]
        out.append([x - (1 << 32) if x >= 1 << 31 else x for x in v])
    return ints(out).view(-1, words)


def ways(trees):
    """What every row sees of its own tree: itself and the rows on its way to the root."""
    out = []
    for parents in trees:
        for i in range(len(parents)):
            row, j = [False] * len(parents), i
            while j >= 0:
                row[j] = True
                j = parents[j]
            out.append(row)
    return out


class Case:
    def __init__(self, dtype, lengths, counts, H, Hkv, d, ps, seed=0, strided=False, spare=None):
        rng = random.Random(seed)
        self.lengths, self.counts, self.H, self.Hkv, self.d, self.ps = lengths, counts, H, Hkv, d, ps
        self.trees = [tree(n, rng) for n in counts]
        self.pages, P_ = page_lists([a + n for a, n in zip(lengths, counts)], ps, rng)
        self.width = max([len(p) for p in self.pages] + [1]) + 1
        self.table = [p + [0] * (self.width - len(p)) for p in self.pages]
        g = torch.Generator().manual_seed(seed)
        T = sum(counts)
        wide = (H + 2 * Hkv) * d if strided else H * d
        self.q = (2 * torch.randn(T, wide, generator=g)).to(dtype).to(DEV)[:, :H * d]
        self.k = torch.randn(P_, Hkv, ps, d, generator=g).to(dtype).to(DEV)
        self.v = torch.randn(P_, Hkv, ps, d, generator=g).to(dtype).to(DEV)
        self.scale = d ** -0.5
        self.seen = ways(self.trees)
        self.words = max(1, -(-max(counts) // 32))
        self.dtype = dtype
        out = torch.full((T, wide), 7.0, dtype=dtype, device=DEV)
        self.out_base, self.out = out, out[:, :H * d]

    def place(self, s, pos):
        return self.pages[s][pos // self.ps], pos % self.ps

    def run(self, ops, **hints):
        ops.tree_attention(self.q, self.k, self.v, ints(self.table), ints(self.lengths), ints(starts(self.counts)),
                           bits_of(self.seen, self.words), self.out, num_heads=self.H, num_kv_heads=self.Hkv, head_dim=self.d,
                           scale=self.scale, **hints)
        return self.out

    def check(self, ops, **hints):
        got = self.run(ops, **hints).cpu().double()
        want = P.attend(self.q, self.k, self.v, self.table, self.lengths, self.counts, self.seen, self.H, self.scale, self.ps)
        rel, absolute = P.tolerance(self.dtype, self.q, self.k, self.v, self.scale, max(a + n for a, n in zip(self.lengths, self.counts)))
        same = (got == want) | (got.isnan() & want.isnan())
        off = torch.where(same, 0.0, (got - want).abs() - rel * want.abs())
        assert not off.isnan().any() and float(off.amax()) <= absolute, (float(off.amax()), absolute)
        if self.out_base.shape[1] > self.out.shape[1]:
            assert bool((self.out_base[:, self.out.shape[1]:] == 7.0).all())


BOTH = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("H,Hkv,d", [(2, 2, 16), (4, 2, 32), (3, 1, 48), (4, 4, 64), (6, 2, 64), (4, 1, 80), (8, 1, 128), (2, 1, 256)])
def test_attention_over_head_layouts(ops, dtype, H, Hkv, d):
    Case(dtype, [0, 1, 63, 64, 130, 517], [1, 3, 8, 16, 17, 40], H, Hkv, d, 16, seed=d + H, strided=True).check(ops)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("ps", [1, 5, 8, 24, 32, 64, 100, 128, 300])
def test_attention_over_page_sizes(ops, dtype, ps):
    Case(dtype, [ps, 2 * ps - 1, 333, 0], [7, 9, 33, 2], 4, 2, 64, ps, seed=ps).check(ops)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n", [1, 4, 5, 8, 16, 17, 32, 33, 64, 65, 128, 200, 256])
def test_attention_over_tree_sizes(ops, dtype, n):
    """Every tile of rows, whole and one row over, with a tree that crosses tiles of keys."""
    Case(dtype, [100, 37], [n, max(1, n // 3)], 2, 2, 64, 16, seed=n).check(ops)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("S,length", [(1, 9000), (3, 4097), (40, 300)])
def test_attention_over_spans(ops, dtype, S, length):
    """One long request in many spans, some, and more requests than the GPU has places for."""
    Case(dtype, [length - 7 * s for s in range(S)], [8] * S, 4, 2, 64, 16, seed=S).check(ops)


@pytest.mark.parametrize("dtype,lengths,n,H,Hkv,d,ps", [
    (torch.bfloat16, [6001, 3000, 9], 40, 8, 2, 128, 64), (torch.bfloat16, [2500, 6001], 20, 8, 2, 128, 16),
    (torch.bfloat16, [5000, 64], 48, 3, 1, 64, 16), (torch.bfloat16, [4000, 700], 100, 6, 2, 64, 8), (torch.bfloat16, [7000], 70, 8, 1, 80, 32),
    (torch.float32, [3000, 1, 900], 20, 4, 2, 128, 16), (torch.bfloat16, [3000, 1, 900], 70, 4, 2, 64, 5)])
def test_long_texts_and_wide_trees(ops, dtype, lengths, n, H, Hkv, d, ps):
    """Keys shared out among blocks, in every kernel that takes many rows: several segments a block, values that come late."""
    counts = [n, max(1, n // 2), 3][:len(lengths)]
    c = Case(dtype, lengths, counts, H, Hkv, d, ps, seed=n + d)
    filler = torch.randn(1 << 27, device=DEV)             # more than L2: keys and values come from memory
    for _ in range(3):
        filler.mul_(1.0)
        c.out.fill_(7.0)
        c.check(ops)


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("n,H,Hkv,d,page", [(4, 2, 2, 48, 16), (30, 2, 1, 64, 16), (12, 8, 1, 128, 16), (50, 8, 2, 128, 8), (9, 4, 2, 64, 5)])
def test_many_short_texts_between_long_ones(ops, dtype, n, H, Hkv, d, page):
    """Keys shared out where most pairs are shorter than what comes before each of them: pieces that end and begin anywhere, blocks of
    more segments than fit one list, requests without rows."""
    rng = random.Random(n + d)
    lengths = [rng.choice((0, 1, 5, 63, 64, 65, 200)) for _ in range(70)] + [3000, 0, 1500]
    counts = [rng.choice((0, 1, n // 2, n)) for _ in lengths]
    counts[70] = n
    for hints in (dict(max_nodes=n, max_length=100000), dict(max_nodes=n, max_length=3000)):
        Case(dtype, lengths, counts, H, Hkv, d, page, seed=n + d).check(ops, **hints)


@pytest.mark.parametrize("dtype", BOTH)
def test_hints_only_change_how_the_work_is_cut(ops, dtype):
    for hints in (dict(), dict(max_nodes=20, max_length=700), dict(max_nodes=1, max_length=1), dict(max_nodes=256, max_length=100000)):
        Case(dtype, [700, 3, 128], [20, 5, 1], 4, 2, 32, 16, seed=2).check(ops, **hints)


@pytest.mark.parametrize("dtype", BOTH)
def test_masks_that_leave_rows_empty_or_are_no_tree(ops, dtype):
    """A row without a visible key gives zeros; the bits decide, whatever the tree."""
    c = Case(dtype, [0, 0, 90], [5, 40, 40], 4, 2, 64, 16, seed=4)
    rng = random.Random(1)
    c.seen = [[rng.random() < 0.3 for _ in row] for row in c.seen]
    c.seen[0] = [False] * 5
    c.seen[7] = [False] * 40
    c.seen[8] = [False] * 39 + [True]
    c.check(ops)
    assert bool((c.out[0] == 0).all()) and bool((c.out[7] == 0).all())


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("counts", [[6, 20], [40, 64]])
def test_infinities_and_nan_in_masked_places_have_no_effect(ops, dtype, counts):
    """Keys and values of rows that others do not see, what lies behind a request's last row, pages nobody holds."""
    c = Case(dtype, [61, 130], counts, 4, 2, 64, 16, seed=6)
    held = {c.place(s, p) for s in range(2) for p in range(c.lengths[s] + c.counts[s])}
    for page in range(c.k.shape[0]):
        for off in range(c.ps):
            if (page, off) not in held:
                c.k[page, :, off], c.v[page, :, off] = NAN, INF
    c.seen = [list(r) for r in c.seen]
    for s, bad in ((0, 3), (1, counts[1] - 1), (1, 0)):
        page, off = c.place(s, c.lengths[s] + bad)
        c.k[page, :, off], c.v[page, :, off] = (NAN, NAN) if bad else (INF, -INF)
        base = sum(c.counts[:s])
        for i in range(c.counts[s]):
            c.seen[base + i][bad] = False
    c.check(ops)
    assert bool(c.out.float().isfinite().all())


@pytest.mark.parametrize("dtype", BOTH)
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it_and_no_other(ops, dtype):
    c = Case(dtype, [70, 5], [20, 10], 4, 2, 64, 16, seed=9)
    c.trees = [[-1] + [0] * 19, [-1] + [0] * 9]
    c.seen = ways(c.trees)
    for s, row, head, col, value in ((0, 4, 0, 3, INF), (0, 9, 1, 63, NAN), (1, 2, 0, 0, -INF)):
        page, off = c.place(s, c.lengths[s] + row)
        c.v[page, head, off, col] = value
    c.check(ops)
    bad = ~c.out.float().isfinite()
    assert sorted(set(bad.any(1).nonzero().flatten().tolist())) == [4, 9, 22]
    assert int(bad.sum()) == 6                       # two query heads to each key/value head


@pytest.mark.parametrize("dtype", BOTH)
def test_scores_far_apart(ops, dtype):
    """A maximum that moves by hundreds within a walk, and keys at the type's ends of range."""
    c = Case(dtype, [400], [8], 2, 2, 64, 16, seed=11)
    c.k[c.pages[0][3]] *= 60.0
    c.k[c.pages[0][20]] *= -90.0
    c.check(ops)
    c.k[c.pages[0][5]] = torch.finfo(dtype).min / 2 ** 70
    c.k[c.pages[0][6]] = 0.0
    got = c.run(ops).double().cpu()
    want = P.attend(c.q, c.k, c.v, c.table, c.lengths, c.counts, c.seen, 2, c.scale, 16)
    assert float((got - want).abs().amax()) <= (0.03 if dtype == torch.bfloat16 else 1e-4)


@pytest.mark.parametrize("dtype", BOTH)
def test_rows_at_any_address(ops, dtype):
    """Queries and results that do not start at 16 bytes, rows an odd stride apart, a table that is a slice."""
    c = Case(dtype, [90, 17], [9, 30], 3, 3, 32, 16, seed=12)
    T, w = c.q.shape
    q = torch.zeros(T * (w + 5) + 1, dtype=dtype, device=DEV)[1:].view(T, w + 5)[:, :w]
    q.copy_(c.q)
    out = torch.full((T * (w + 3) + 1,), 7.0, dtype=dtype, device=DEV)
    view = out[1:].view(T, w + 3)[:, :w]
    wide = torch.full((2, c.width + 9), -5, dtype=torch.int32, device=DEV)
    wide[:, 4:4 + c.width] = ints(c.table)
    c.run(ops)
    ops.tree_attention(q, c.k, c.v, wide[:, 4:4 + c.width], ints(c.lengths), ints(starts(c.counts)), bits_of(c.seen, c.words), view,
                       num_heads=3, num_kv_heads=3, head_dim=32, scale=c.scale)
    assert torch.equal(view, c.out)
    assert bool((out[1:].view(T, w + 3)[:, w:] == 7.0).all()) and float(out[0]) == 7.0


@pytest.mark.parametrize("dtype", BOTH)
def test_a_chain_is_causal_attention(ops, dtype):
    """Rows that follow one another see what the engine's own attention of a prompt portion sees."""
    class Ctx:
        pass
    c = Case(dtype, [130, 0], [40, 7], 4, 2, 64, 16, seed=13)
    c.trees = [list(range(-1, n - 1)) for n in c.counts]
    c.seen = ways(c.trees)
    got = c.run(ops).clone()
    ctx = Ctx()
    ctx.token_seq = ints([0] * 40 + [1] * 7)
    ctx.positions = ints(list(range(130, 170)) + list(range(7)))
    ops.paged_attention(c.q, c.k, c.v, ints(c.table), ctx, c.out, num_heads=4, num_kv_heads=2, head_dim=64, scale=c.scale, impl="simt")
    rel, absolute = P.tolerance(dtype, c.q, c.k, c.v, c.scale, 170)
    assert bool(((got.double() - c.out.double()).abs() <= 2 * absolute + 2 * rel * c.out.double().abs()).all())


@pytest.mark.parametrize("dtype", BOTH)
def test_a_pool_past_32_bits_of_elements(ops, dtype):
    """Rows of keys whose offset in elements does not fit 32 bits."""
    ps, Hkv, d = 64, 8, 128
    pages = (1 << 32) // (ps * Hkv * d) + 40 if dtype == torch.bfloat16 else (1 << 31) // (ps * Hkv * d) + 40
    k = torch.empty((pages, Hkv, ps, d), dtype=dtype, device=DEV)
    c = Case(dtype, [250], [12], 8, 8, d, ps, seed=14)
    ids = [pages - 1 - 3 * i for i in range(len(c.pages[0]))]
    for new, old in zip(ids, c.pages[0]):
        k[new] = c.k[old]
    want = c.run(ops).clone()
    v = torch.empty_like(k)
    for new, old in zip(ids, c.pages[0]):
        v[new] = c.v[old]
    c.k, c.v, c.table = k, v, [ids + [0] * (c.width - len(ids))]
    assert torch.equal(c.run(ops), want)
    del k, v, c
    torch.cuda.empty_cache()


def test_attention_on_another_stream_and_in_a_graph(ops):
    c = Case(torch.bfloat16, [500, 90], [8, 30], 4, 2, 64, 16, seed=15)
    want = c.run(ops).clone()
    table, lengths, cu, bits = ints(c.table), ints(c.lengths), ints(starts(c.counts)), bits_of(c.seen, c.words)
    torch.cuda.synchronize()
    def go():
        ops.tree_attention(c.q, c.k, c.v, table, lengths, cu, bits, c.out, num_heads=4, num_kv_heads=2, head_dim=64, scale=c.scale)
    side = torch.cuda.Stream()
    c.out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        go()
    side.synchronize()
    assert torch.equal(c.out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        c.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, want)


def test_the_same_call_has_the_same_bits(ops):
    for dtype in BOTH:
        c = Case(dtype, [3000, 10, 700], [40, 3, 17], 8, 2, 64, 16, seed=16)
        first = c.run(ops).clone()
        for _ in range(5):
            assert torch.equal(c.run(ops), first)


# ------------------------------------------------------------------------------------------------ acceptance
def run_accept(ops, trees, tokens, lengths, depth, logits=None, chosen=None):
    S, T = len(trees), sum(map(len, trees))
    got = dict(chosen=ints(chosen) if chosen is not None else torch.full((T,), -77, dtype=torch.int32, device=DEV),
               path=torch.full((S, depth), -77, dtype=torch.int32, device=DEV), accepted=ints([-77] * S), next_token=ints([-77] * S),
               new_lengths=ints([-77] * S))
    ops.accept_drafts(ints(tokens), ints([p for t in trees for p in t]), ints(starts([len(t) for t in trees])), ints(lengths),
                      logits=logits, **got)
    return {k: v.tolist() for k, v in got.items()}


def agreeing(trees, chosen, V, rng, share=0.7):
    tokens = []
    for parents in trees:
        base = len(tokens)
        tokens += [chosen[base + p] if p >= 0 and rng.random() < share else rng.randrange(V) for p in parents]
    return tokens


@pytest.mark.parametrize("V", [1, 2, 3, 5, 97, 1000, 32000, 50257])
@pytest.mark.parametrize("depth", [1, 4, 40])
def test_acceptance(ops, V, depth):
    rng = random.Random(V + depth)
    counts = [1, 0, 33, 8, 64, 2, 17]
    trees = [tree(n, rng) for n in counts]
    logits = torch.randn(sum(counts), V, generator=torch.Generator().manual_seed(V)).to(DEV)
    chosen = logits.cpu().argmax(1).tolist()
    tokens = agreeing(trees, chosen, V, rng)
    lengths = [5, 6, 0, 100, 7, 1, 1000]
    path, accepted, nexts, new = P.accept(chosen, tokens, trees, lengths, depth)
    got = run_accept(ops, trees, tokens, lengths, depth, logits)
    assert got == dict(chosen=chosen, path=path, accepted=accepted, next_token=nexts, new_lengths=new)
    # the same choices, given
    assert run_accept(ops, trees, tokens, lengths, depth, chosen=chosen) == got


def test_acceptance_of_the_largest_trees(ops):
    rng = random.Random(2)
    trees = [tree(256, rng, 0.9), list(range(-1, 255)), [-1] + [0] * 255]
    chosen = [rng.randrange(3) for _ in range(768)]
    tokens = agreeing(trees, chosen, 3, rng, 0.95)
    path, accepted, nexts, new = P.accept(chosen, tokens, trees, [1, 2, 3], 256)
    assert run_accept(ops, trees, tokens, [1, 2, 3], 256, chosen=chosen) == dict(chosen=chosen, path=path, accepted=accepted,
                                                                                   next_token=nexts, new_lengths=new)


def test_ties_nan_and_infinities_in_the_logits(ops):
    """The lowest of equal logits; NaN is never chosen; a row of nothing but NaN or -inf takes token 0."""
    V = 5003
    x = torch.randn(6, V, generator=torch.Generator().manual_seed(1))
    x[0, [4000, 17, 18, 2500]] = 50.0
    x[1, 3000] = INF
    x[1, 3001] = INF
    x[2] = NAN
    x[2, 4999] = -3.0
    x[3] = NAN
    x[4] = -INF
    x[5] = -INF
    x[5, 77] = -1e38
    got = run_accept(ops, [[-1, 0, 0, 0, 0, 0]], [0] * 6, [3], 4, x.to(DEV))
    assert got["chosen"] == [17, 3000, 4999, 0, 0, 77]


def test_of_several_children_with_the_token_the_lowest_counts(ops):
    trees, tokens = [[-1, 0, 0, 0, 2, 3]], [9, 4, 5, 5, 6, 6]
    got = run_accept(ops, trees, tokens, [10], 4, chosen=[5, 0, 6, 6, 8, 7])
    assert got["path"] == [[0, 2, 4, -1]] and got["next_token"] == [8] and got["new_lengths"] == [13]


def test_logits_at_any_address(ops):
    """Rows that start at every distance from a 16-byte boundary, and that end at every one."""
    for V in (5, 2049, 50257):
        for skew in range(4):
            T = 5
            base = torch.full((T * (V + 7) + 8,), 99.0, device=DEV)
            rows = base[skew:skew + T * (V + 7)].view(T, V + 7)[:, :V]
            rows.copy_(torch.randn(T, V, generator=torch.Generator().manual_seed(skew)))
            rows[0, V - 1], rows[1, 0], rows[2, V // 2], rows[3, min(3, V - 1)] = 30.0, 30.0, 30.0, 30.0
            got = run_accept(ops, [[-1, 0, 1, 2, 3]], [0] * 5, [0], 2, rows)
            assert got["chosen"] == rows.cpu().argmax(1).tolist()


def test_lengths_in_place(ops):
    lengths = ints([4, 9])
    path, acc, nxt = torch.empty((2, 3), dtype=torch.int32, device=DEV), ints([0, 0]), ints([0, 0])
    ops.accept_drafts(ints([1, 2, 3]), ints([-1, 0, -1]), ints([0, 2, 3]), lengths, chosen=ints([2, 5, 6]), path=path, accepted=acc,
                      next_token=nxt, new_lengths=lengths)
    assert lengths.tolist() == [6, 10] and nxt.tolist() == [5, 6]


# ------------------------------------------------------------------------------------------------ kept rows
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.float32, 64), (torch.bfloat16, 16), (torch.float32, 3),
                                     (torch.bfloat16, 5), (torch.float32, 256)])
@pytest.mark.parametrize("ps", [1, 4, 16])
def test_kept_rows(ops, dtype, d, ps):
    rng = random.Random(d + ps)
    lengths, counts, depth = [0, 5, 16, 33, 7, 2], [64, 30, 1, 20, 25, 3], 24
    paths = []
    for s, n in enumerate(counts):
        paths.append([0] + sorted(rng.sample(range(1, n), min(n - 1, (23, 9, 0, 1, 16, 0)[s]))))
    paths[4] = list(range(0, 17)) + [19, 24]             # stays where it is, then two moves
    paths[5] = []                                        # a request that kept nothing
    pages, P_ = page_lists([a + n for a, n in zip(lengths, counts)], ps, rng)
    width = max(map(len, pages)) + 1
    table = [p + [0] * (width - len(p)) for p in pages]
    planes = torch.randn(6, P_, 3, ps, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    accepted = [len(p) for p in paths]
    want = P.keep(planes, table, lengths, paths, accepted, ps)
    got = planes.to(DEV).view(3, 2, P_, 3, ps, d)
    ops.keep_accepted(got, ints(table), ints(lengths), ints([p + [-1] * (depth - len(p)) for p in paths]), ints(accepted))
    assert torch.equal(got.view(6, P_, 3, ps, d).cpu(), want)


def test_rows_without_a_page_stay(ops):
    """Rows past the block table are neither read nor written."""
    planes = torch.arange(2 * 4 * 4 * 4, dtype=torch.float32, device=DEV).view(2, 4, 1, 4, 4)
    before = planes.clone()
    ops.keep_accepted(planes, ints([[1, 3]]), ints([6]), ints([[0, 3, 5, -1]]), ints([3]))
    assert torch.equal(planes, before)
    ops.keep_accepted(planes, ints([[1, 3]]), ints([3]), ints([[0, 4, 5, -1]]), ints([2]))
    before[:, 3, :, 0] = before[:, 3, :, 3]
    assert torch.equal(planes, before)


# ------------------------------------------------------------------------------------------------ together
def test_a_round_of_all_four(ops):
    """Tables, attention, acceptance and kept rows behind one another on the stream, and the next round from what they left: the
    second round's attention sees the accepted path's keys and values where a chain would have put them."""
    rng = random.Random(21)
    ps, H, d, depth = 16, 4, 64, 6
    lengths, counts = [40, 7, 0], [12, 1, 30]
    trees = [tree(n, rng) for n in counts]
    pages, P_ = page_lists([a + n + 40 for a, n in zip(lengths, counts)], ps, rng)
    width = max(map(len, pages))
    pool = torch.randn(2, P_, H, ps, d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(DEV)
    T = sum(counts)
    chosen = [rng.randrange(50) for _ in range(T)]
    tokens = agreeing(trees, chosen, 50, rng, 0.9)
    got = run_tables(ops, lengths, trees, pages, ps, width, 1)
    L, cu = ints(lengths), ints(starts(counts))
    path, acc, nxt = torch.empty((3, depth), dtype=torch.int32, device=DEV), ints([0] * 3), ints([0] * 3)
    new = ints([0] * 3)
    ops.accept_drafts(ints(tokens), ints([p for t in trees for p in t]), cu, L, chosen=ints(chosen), path=path, accepted=acc,
                      next_token=nxt, new_lengths=new)
    before = pool.clone()
    ops.keep_accepted(pool, got["block_table"], L, path, acc)
    want_path, want_acc, _, want_new = P.accept(chosen, tokens, trees, lengths, depth)
    assert acc.tolist() == want_acc and new.tolist() == want_new and max(want_acc) > 2
    q = torch.randn(3, H * d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    out = torch.empty_like(q)
    ops.tree_attention(q, pool[0], pool[1], got["block_table"], new, ints([0, 1, 2, 3]), ints([[1], [1], [1]]), out, num_heads=H,
                       num_kv_heads=H, head_dim=d, scale=d ** -0.5)
    moved = P.keep(before.cpu(), [p + [0] * (width - len(p)) for p in pages], lengths, want_path, want_acc, ps)
    want = P.attend(q, moved[0], moved[1], [p + [0] * (width - len(p)) for p in pages], want_new, [1, 1, 1], [[True]] * 3, H, d ** -0.5, ps)
    rel, absolute = P.tolerance(torch.bfloat16, q, pool[0], pool[1], d ** -0.5, 60)
    assert bool(((out.cpu().double() - want).abs() <= absolute + rel * want.abs()).all())


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(ops):
    c = Case(torch.float32, [9], [3], 2, 2, 32, 16)
    table, L, cu, bits = ints(c.table), ints(c.lengths), ints(starts(c.counts)), bits_of(c.seen, c.words)
    def attention(**kw):
        a = dict(q=c.q, k=c.k, v=c.v, table=table, L=L, cu=cu, bits=bits, out=c.out, H=2, Hkv=2, d=32, scale=0.1)
        a.update(kw)
        ops.tree_attention(a["q"], a["k"], a["v"], a["table"], a["L"], a["cu"], a["bits"], a["out"], num_heads=a["H"],
                           num_kv_heads=a["Hkv"], head_dim=a["d"], scale=a["scale"])
    attention()
    for kw, words in ((dict(q=c.q.cpu()), "CUDA"), (dict(q=c.q.half()), "k_pages"), (dict(out=c.out.bfloat16()), "out"), (dict(H=3), "head counts"),
                      (dict(d=16), "head counts"), (dict(cu=cu[:1]), "starts"), (dict(bits=bits[:2]), "ancestors"),
                      (dict(bits=torch.zeros(3, 9, dtype=torch.int32, device=DEV)), "ancestors"), (dict(L=L.long()), "int32"),
                      (dict(table=torch.cat([table, table])), "block_table"), (dict(scale=0.0), "scale"), (dict(scale=NAN), "scale"),
                      (dict(k=c.k[:, :, :8]), "contiguous"), (dict(v=c.v[1:]), "pages")):
        with pytest.raises(ops.KernelError, match=words):
            attention(**kw)
    k = torch.zeros(4, 2, 16, 24, device=DEV)
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        attention(k=k, v=k, q=torch.zeros(3, 48, device=DEV), out=torch.zeros(3, 48, device=DEV), d=24)
    flat = torch.zeros(4 * 2 * 16 * 32 + 1, device=DEV)[1:].view(4, 2, 16, 32)
    with pytest.raises(ops.KernelError, match="aligned"):
        attention(k=flat, v=flat)

    def tabled(**kw):
        T = 3
        a = dict(lengths=L, cu=cu, parents=ints([-1, 0, 0]), pages=ints([0]), cu_pages=ints([0, 1]), ps=16, block_table=table.clone(),
                 slot_mapping=ints([0] * T), positions=ints([0] * T), token_seq=ints([0] * T), ctx_len=ints([0]), ancestors=bits.clone())
        a.update(kw)
        ops.draft_tables(*[a.pop(k) for k in ("lengths", "cu", "parents", "pages", "cu_pages", "ps")], **a)
    tabled()
    for kw, words in ((dict(ps=0), "pages of 0"), (dict(ancestors=None), "ancestors"), (dict(parents=ints([-1])), "parent"),
                      (dict(positions=ints([0])), "fit"), (dict(cu_pages=ints([0])), "fit"), (dict(cu=ints([0])), "starts"),
                      (dict(ancestors=torch.zeros(3, 9, dtype=torch.int32, device=DEV)), "ancestors"), (dict(pages=ints([0]).float()), "int32")):
        with pytest.raises(ops.KernelError, match=words):
            tabled(**kw)

    def accepts(**kw):
        a = dict(tokens=ints([1, 2, 3]), parents=ints([-1, 0, 0]), cu=cu, lengths=L, chosen=ints([0] * 3), path=ints([[0, 0]]), accepted=ints([0]),
                 next_token=ints([0]), new_lengths=ints([0]), logits=None)
        a.update(kw)
        ops.accept_drafts(*[a.pop(k) for k in ("tokens", "parents", "cu", "lengths")], **a)
    accepts()
    for kw, words in ((dict(logits=torch.zeros(2, 5, device=DEV)), "logits"), (dict(logits=torch.zeros(3, 5, device=DEV).bfloat16()), "float32"),
                      (dict(path=ints([0])), "fit"), (dict(path=torch.zeros(1, 0, dtype=torch.int32, device=DEV)), "fit"), (dict(chosen=ints([0])), "fit"), (dict(accepted=ints([0, 0])), "fit"),
                      (dict(logits=torch.zeros(3, 10, device=DEV)[:, ::2]), "rows")):
        with pytest.raises(ops.KernelError, match=words):
            accepts(**kw)

    def keeps(**kw):
        a = dict(planes=c.k, table=table, lengths=L, path=ints([[0, 1]]), accepted=ints([1]))
        a.update(kw)
        ops.keep_accepted(*[a[k] for k in ("planes", "table", "lengths", "path", "accepted")])
    keeps()
    for kw, words in ((dict(planes=c.k[:, :, :8]), "contiguous"), (dict(path=ints([0])), "path"), (dict(accepted=ints([1, 2])), "accepted"),
                      (dict(table=torch.cat([table, table])), "block_table"), (dict(planes=c.k[0, 0]), "planes")):
        with pytest.raises(ops.KernelError, match=words):
            keeps(**kw)


def test_nothing_to_do(ops):
    """No rows at all, or requests that bring none."""
    c = Case(torch.float32, [9, 4], [0, 1], 2, 2, 32, 16)
    c.check(ops)
    e = torch.zeros(0, dtype=torch.int32, device=DEV)
    ops.tree_attention(c.q[:0], c.k, c.v, ints(c.table), ints([9, 4]), ints([0, 0, 0]), e.view(0, 1), c.out[:0], num_heads=2, num_kv_heads=2,
                       head_dim=32, scale=0.1)
    got = run_tables(ops, [4, 5], [[], []], [[1], [2]], 16, 2, 1)
    assert got["ctx_len"].tolist() == [4, 5] and got["block_table"].tolist() == [[1, 0], [2, 0]]
    assert run_accept(ops, [[], []], [], [4, 5], 2, torch.zeros(0, 7, device=DEV))["accepted"] == [0, 0]
