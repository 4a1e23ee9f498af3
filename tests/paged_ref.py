"""Plain restatements in 64 bits of the paged-cache and draft-tree operators,
request by request (test infrastructure only), and builders of their inputs."""
import math

import numpy as np
import torch

TDT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# unit roundoff of a type: half the spacing of its numbers at 1
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def random_tree(n, rng, shape="mixed"):
    """Parents of n nodes: "chain", "star", "forest" (several roots) or "mixed"."""
    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "star":
        return [-1] + [0] * (n - 1) if n else []
    if shape == "forest":
        return [-1 if rng.random() < 0.3 else int(rng.integers(0, i)) if i else -1 for i in range(n)]
    return [int(rng.integers(max(0, i - 5), i)) if i else -1 for i in range(n)]


def chain_of(parents, i):
    """Node i and its ancestors."""
    found = []
    while i >= 0:
        found.append(i)
        i = parents[i]
    return found


def deal_pages(rows, page, rng, spare=2, pad=1):
    """A block table for requests of `rows` rows over shuffled pages: (table
    int32, pages of the pool).  Unused entries hold -1."""
    counts = [-(-r // page) for r in rows]
    perm = rng.permutation(sum(counts) + spare).astype(np.int32)
    table = np.full((len(rows), max(counts + [1]) + pad), -1, np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = perm[at:at + c]
        at += c
    return table, sum(counts) + spare


def attention(q, k, v, lens, cu, parents, scale):
    """q (n, H, D); k, v: per request (rows, KV, D) arrays of its cache rows
    (len + nodes); everything in float64.  Returns out, lse and w = sum p |v|
    (what a rounding of the weights scales with)."""
    n_tok, H, D = q.shape
    out = np.zeros((n_tok, H, D))
    w = np.zeros((n_tok, H, D))
    lse = np.full((n_tok, H), -np.inf)
    for b, ln in enumerate(lens):
        n = cu[b + 1] - cu[b]
        par = parents[cu[b]:cu[b + 1]] if parents is not None else [i - 1 for i in range(n)]
        KV = k[b].shape[1]
        for i in range(n):
            rows = list(range(ln)) + [ln + j for j in chain_of(par, i)]
            for h in range(H):
                g = h // (H // KV)
                s = k[b][rows, g] @ q[cu[b] + i, h] * scale
                m = s.max()
                p = np.exp(s - m)
                z = p.sum()
                out[cu[b] + i, h] = p @ v[b][rows, g] / z
                w[cu[b] + i, h] = p @ np.abs(v[b][rows, g]) / z
                lse[cu[b] + i, h] = m + math.log(z)
    return out, lse, w


def rotate(x, cos, sin, n_rot, style):
    """x (n, heads, D) rotated by cos / sin (n, n_rot / 2), float64."""
    y = x.copy()
    c, s = cos[:, None], sin[:, None]
    if style == "norm":
        a, b = x[..., 0:n_rot:2], x[..., 1:n_rot:2]
        y[..., 0:n_rot:2], y[..., 1:n_rot:2] = a * c - b * s, a * s + b * c
    else:
        h = n_rot // 2
        a, b = x[..., :h], x[..., h:n_rot]
        y[..., :h], y[..., h:n_rot] = a * c - b * s, a * s + b * c
    return y


def plan(lens, add, held, table, ring, state, page, max_tokens, parents):
    """Request by request; returns a dict of the arrays after the step."""
    table, ring = table.copy(), ring.copy()
    head, count = state
    size, wide = len(ring), table.shape[1]
    taken = back = wanted = 0
    old_count = count
    cu, seq, pos, slot, held_out = [0], [], [], [], []
    for b in range(len(lens)):
        n = max(add[b], 0)
        ok, h = False, held[b]
        if add[b] < 0:
            for j in range(h):
                ring[(head + old_count + back + j) % size] = table[b, j]
            back += h
            h = 0
        else:
            want = -(-(lens[b] + n) // page)
            need = max(0, want - h) if want <= wide else 0
            wanted += need
            ok = want <= wide and (need == 0 or wanted <= old_count)
            if ok and need:
                for j in range(need):
                    table[b, h + j] = ring[(head + wanted - need + j) % size]
                taken = wanted
                h += need
        held_out.append(h)
        base = cu[-1]
        par = [i - 1 for i in range(n)] if parents is None else [int(x) for x in parents[base:base + n]]
        for i in range(n):
            row = lens[b] + i
            seq.append(b)
            pos.append(lens[b] + len(chain_of(par, i)) - 1)
            slot.append(int(table[b, row // page]) * page + row % page if ok else -1)
        cu.append(base + n)
    pad = max_tokens - len(seq)
    return dict(table=table, ring=ring, held=held_out, cu=cu, seq=seq + [-1] * pad,
                pos=pos + [0] * pad, slot=slot + [-1] * pad,
                state=[(head + taken) % size, old_count - taken + back])


def constrain(x, cu, parents, tokens, hist, start, prompt, rep, pres, freq, bias, mask):
    """x (n, V); bias: per request a list of (id, value); mask (n, V) bool or
    None.  Each operation rounded to float32 where the inputs are float32."""
    x = x.copy()
    V = x.shape[1]
    for b in range(len(cu) - 1):
        par = parents[cu[b]:cu[b + 1]]
        h = hist[start[b]:start[b + 1]]
        told = set(int(t) for t in h[:prompt[b]] if 0 <= t < V)
        for r in range(cu[b], cu[b + 1]):
            said = {}
            path = [tokens[cu[b] + i] for i in chain_of(par, r - cu[b])] if tokens is not None else []
            for t in list(h[prompt[b]:]) + path:
                if 0 <= t < V:
                    said[int(t)] = said.get(int(t), 0) + 1
            for i, val in dict(bias[b]).items():
                if 0 <= i < V:
                    x[r, i] = x[r, i] + val
            for t in told | set(said):
                x[r, t] = x[r, t] / rep[b] if x[r, t] > 0 else x[r, t] * rep[b]
            for t, c in said.items():
                x[r, t] = x[r, t] - freq[b] * x.dtype.type(c)
                x[r, t] = x[r, t] - pres[b]
        if mask is not None:
            x[cu[b]:cu[b + 1]][~mask[cu[b]:cu[b + 1]]] = -np.inf
    return x


def accept(picks, tokens, parents, cu):
    """Per request: (path, the last node's pick or -1)."""
    found = []
    for b in range(len(cu) - 1):
        n, base = cu[b + 1] - cu[b], cu[b]
        at, path = (0 if n else None), []
        while at is not None:
            path.append(at)
            at = next((i for i in range(at + 1, n) if parents[base + i] == at
                       and tokens[base + i] == picks[base + at]), None)
        found.append((path, int(picks[base + path[-1]]) if path else -1))
    return found
