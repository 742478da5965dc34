"""Decoding with drafted tokens, stated request by request in plain Python and 64 bits: tables, attention over a tree, the accepted
path, the kept cache rows."""
import math

import torch

F64 = torch.float64


def tables(lengths, trees, pages, page_size, width, words):
    """``trees``: a parent list per request, or a number of rows that follow one another; ``pages``: a page list per request."""
    out = dict(block_table=[], slots=[], positions=[], token_seq=[], ctx_len=[], ancestors=[])
    for s, (L, tree, held) in enumerate(zip(lengths, trees, pages)):
        chain = isinstance(tree, int)
        parents = list(range(-1, tree - 1)) if chain else tree
        out["block_table"].append([max(p, 0) for p in held[:width]] + [0] * (width - len(held)))
        out["ctx_len"].append(L + len(parents))
        for i in range(len(parents)):
            part = chain or i < 32 * words
            way = {i}
            j = parents[i] if 0 <= parents[i] < i else -1
            while j >= 0:
                way.add(j)
                j = parents[j] if 0 <= parents[j] < j else -1
            place = L + i
            page = held[place // page_size] if part and place // page_size < len(held) else -1
            out["slots"].append(page * page_size + place % page_size if page >= 0 else -1)
            out["positions"].append(L + len(way) - 1 if part else L)
            out["token_seq"].append(s)
            bits = [sum(1 << b for b in range(32) if part and 32 * w + b in way) for w in range(words)]
            out["ancestors"].append([b - (1 << 32) if b >= 1 << 31 else b for b in bits])
    return out


def attend(q, k_pages, v_pages, table, lengths, counts, seen, heads, scale, page_size):
    """[T, heads * d] in 64 bits; ``seen[row][j]``: whether the row sees row j of its request.  Masked places are never touched."""
    Hkv, d = k_pages.shape[1], k_pages.shape[3]
    q, k_pages, v_pages = q.cpu().to(F64), k_pages.cpu(), v_pages.cpu()
    out = torch.zeros(q.shape, dtype=F64)
    row = 0
    for s, (L, n) in enumerate(zip(lengths, counts)):
        at = torch.arange(L + n)
        page = torch.tensor(table[s])[at // page_size].long()
        K = k_pages[page, :, at % page_size].to(F64)              # [keys, Hkv, d]
        V = v_pages[page, :, at % page_size].to(F64)
        for i in range(n):
            vis = list(range(L)) + [L + j for j in range(n) if seen[row][j]]
            if vis:
                for h in range(heads):
                    g = h // (heads // Hkv)
                    x = scale * (K[vis, g] @ q[row, h * d:(h + 1) * d])
                    out[row, h * d:(h + 1) * d] = torch.softmax(x, 0) @ V[vis, g]
            row += 1
    return out


def accept(chosen, tokens, trees, lengths, depth):
    """(path, accepted, next_token, new_lengths) as lists."""
    paths, accepted, nexts, new = [], [], [], []
    first = 0
    for parents, L in zip(trees, lengths):
        n, path = len(parents), []
        at = 0 if n else None
        while at is not None and len(path) < depth:
            path.append(at)
            at = next((j for j in range(at + 1, n) if parents[j] == at and tokens[first + j] == chosen[first + at]), None)
        paths.append(path + [-1] * (depth - len(path)))
        accepted.append(len(path))
        nexts.append(chosen[first + path[-1]] if path else -1)
        new.append(L + len(path))
        first += n
    return paths, accepted, nexts, new


def keep(planes, table, lengths, path, accepted, page_size):
    """A copy of ``planes`` [planes, pages, heads, page_size, d] with the rows moved."""
    out = planes.clone()
    for s, L in enumerate(lengths):
        for k in range(accepted[s]):
            a, b = L + path[s][k], L + k
            out[:, table[s][b // page_size], :, b % page_size] = planes[:, table[s][a // page_size], :, a % page_size]
    return out


def tolerance(dtype, q, k_pages, v_pages, scale, keys):
    """(relative, absolute) bounds of an attention's error.  Rounding errors of 2^-24 in the d products of a score and in the sums
    over keys add up like their square root (four times that is allowed for); a score's error is a weight's relative one, counted
    twice since it also stands in the sum below the bar.  bfloat16: one rounding of the result (2^-9, twice that allowed for) and
    weights in two terms (2^-17 of each, and as much of their sum)."""
    d = q.shape[1] // max(1, q.shape[1] // k_pages.shape[3])
    fine = torch.where(torch.isfinite(k_pages.float()), k_pages.float(), 0.0)
    top = scale * float(q.float().abs().amax() * fine.abs().amax()) * math.sqrt(d)
    v = torch.where(torch.isfinite(v_pages.float()), v_pages.float(), 0.0)
    vmax, eps = float(v.abs().amax()), 2.0 ** -24
    absolute = (2 * (4 * math.sqrt(d) + 4) * top + 4 * math.sqrt(keys + 8)) * eps * vmax
    return (0.0, absolute) if dtype == torch.float32 else (2.0 ** -8, absolute + 2.0 ** -15 * vmax)
