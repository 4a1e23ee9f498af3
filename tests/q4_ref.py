"""Plain restatements of normed heads, the 4-bit cache and sampled verification
(test infrastructure only), and builders of their inputs."""
import numpy as np

from tests.paged_ref import rotate

MAX_D = 8160.0  # largest magnitude of a block's scale


def bf16_round(x):
    """float32 values rounded to 8 significant bits, to nearest even."""
    u = np.asarray(x, np.float32).view(np.uint32)
    r = u + 0x7fff + ((u >> 16) & 1)
    return np.where((u & 0x7f800000) == 0x7f800000, u, r & 0xffff0000).astype(np.uint32).view(np.float32)


def quantize(x):
    """Rows (..., D) f32 -> codes (..., D) int, scales (..., D / 32) float16, by the
    definition in b2attn.h, one f32 operation at a time."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        hi, lo = b.max(-1), b.min(-1)
        m = np.where(hi > -lo, hi, lo)
        d = np.clip(bf16_round(m * np.float32(-0.125)), -MAX_D, MAX_D).astype(np.float16)
        d = np.where(d == 0, np.float16(0), d)
        nan = np.isnan(b).any(-1)
        t = np.floor(b / d.astype(np.float32)[..., None] + np.float32(8.5))
        code = np.where(np.isnan(t), 0, np.clip(t, 0, 15)).astype(np.int64)
    code = np.where(d[..., None] == 0, 8, code)
    return code.reshape(x.shape), np.where(nan, np.float16(np.nan), d)


def values(code, d):
    """What codes and scales stand for, float64."""
    c = code.reshape(*code.shape[:-1], -1, 32).astype(np.float64) - 8
    return (c * d.astype(np.float64)[..., None]).reshape(code.shape)


def granule_places(D):
    """Byte and bit offsets of a granule's codes, bytes of its scales: (K codes [16, D],
    V codes [16, D], K scales [16, D / 32], V scales), from the layout's description,
    value by value."""
    nb = min(4, D // 32)
    k, v = np.zeros((16, D, 2), int), np.zeros((16, D, 2), int)
    ks, vs = np.zeros((16, D // 32), int), np.zeros((16, D // 32), int)
    for r in range(16):
        for dim in range(D):
            bit = 4 * (dim % 8 // 2) + 16 * (dim % 2)
            block, word = dim // 32, dim % 32 // 8
            plane, at = dim // 128, block % 4
            kw = ((plane * 16 + r) * 4 + word) * nb + at
            vw = 2 * D + (dim // 8) * 16 + r
            k[r, dim] = 4 * kw + bit // 8, bit % 8
            v[r, dim] = 4 * vw + bit // 8, bit % 8
        for b in range(D // 32):
            ks[r, b] = 16 * D + 2 * (r * (D // 32) + b)
            vs[r, b] = 17 * D + 2 * (r * (D // 32) + b)
    return k, v, ks, vs


def pack(kc, kd, vc, vd):
    """A pool (pages, KV, page_rows / 16, 18 D) uint8 from codes (pages, rows, KV, D) and
    scales (pages, rows, KV, D / 32)."""
    P, R, KV, D = kc.shape
    pool = np.zeros((P, KV, R // 16, 18 * D), np.uint8)
    places = granule_places(D)
    for which, (c, d) in enumerate(((kc, kd), (vc, vd))):
        g = c.reshape(P, R // 16, 16, KV, D).transpose(0, 3, 1, 2, 4)
        at, bit = places[which][..., 0], places[which][..., 1]
        for shift in (0, 4):
            pick = bit == shift
            pool[..., at[pick]] |= (g[..., pick] << shift).astype(np.uint8)
        s = np.ascontiguousarray(d.reshape(P, R // 16, 16, KV, D // 32).transpose(0, 3, 1, 2, 4)).view(np.uint8)
        s = s.reshape(P, KV, R // 16, 16, D // 32, 2)
        for e in (0, 1):
            pool[..., places[2 + which] + e] = s[..., e]
    return pool


def unpack(pool):
    """(K values, V values) (pages, rows, KV, D) float64 of a pool, and the scales."""
    P, KV, G, width = pool.shape
    D = width // 18
    places = granule_places(D)
    out = []
    for which in (0, 1):
        at, bit = places[which][..., 0], places[which][..., 1]
        code = (pool[..., at] >> bit) & 15
        raw = np.stack([pool[..., places[2 + which] + e] for e in (0, 1)], -1)
        d = np.ascontiguousarray(raw).view(np.float16)[..., 0]
        code = code.transpose(0, 2, 3, 1, 4).reshape(P, G * 16, KV, D)
        d = d.transpose(0, 2, 3, 1, 4).reshape(P, G * 16, KV, D // 32)
        out += [values(code.astype(np.int64), d), d]
    return out


def normed(x, w, eps):
    """Heads (n, heads, D) normed, one rounded f32 operation after the sum (64 bits)."""
    x = np.asarray(x, np.float32)
    if w is None:
        return x
    mean = ((x.astype(np.float64) ** 2).sum(-1, keepdims=True) / x.shape[-1] + float(np.float32(eps))).astype(np.float32)
    return x * (np.float32(1) / np.sqrt(mean)) * np.asarray(w, np.float32)


def heads32(x, w, eps, cos, sin, n_rot, style):
    """Normed and rotated heads in f32, an operation at a time: what the kernels compute
    bit for bit."""
    y = normed(x, w, eps)
    return rotate(y, cos.astype(np.float32), sin.astype(np.float32), n_rot, style)


def heads64(x, w, eps, cos, sin, n_rot, style):
    """The same in 64 bits."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    return rotate(x, cos.astype(np.float64), sin.astype(np.float64), n_rot, style)


def verify(logits, cu, parents, tokens, uniforms, draws, temperature, draft):
    """picks (n,), -1 off the path; all in float64, node by node.  Also the least relative
    distances that a child's decision and a draw had to their borders."""
    n, V = logits.shape
    picks = np.full(n, -1, np.int64)
    margin = drawn = np.inf
    for b in range(len(cu) - 1):
        base, end = cu[b], cu[b + 1]
        cur = base
        while base < end:
            x = logits[cur].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, x)
            top = x.max()
            if top == -np.inf:
                break
            best = int(np.argmax(x))
            T = 1.0 if temperature is None else float(temperature[b])
            if not T > 0 or top == np.inf:
                r = (np.arange(V) == best).astype(np.float64)
            else:
                with np.errstate(invalid="ignore"):
                    r = np.where(x > -np.inf, np.exp((x - top) / T), 0.0)
            total = r.sum()
            out, nxt = [], None
            for c in range(cur + 1, end):
                p = parents[c] if parents is not None else c - base - 1
                t = int(tokens[c])
                if base + p != cur or not 0 <= t < V:
                    continue
                q = 1.0 if draft is None else float(draft[cur, t])
                left, right = float(uniforms[c]) * q * total, r[t]
                margin = min(margin, abs(left - right) / max(left, right, 1e-300))
                if left < right:
                    nxt = c
                    break
                if draft is None:
                    r[t] = 0.0
                else:
                    r = np.maximum(r / total - draft[cur].astype(np.float64), 0.0)
                    out.append(t)
                    r[out] = 0.0
                total = r.sum()
            if nxt is not None:
                picks[cur] = tokens[nxt]
                cur = nxt
                continue
            if not total > 0:
                picks[cur] = best
                left = [c for c in range(cur + 1, end) if tokens[c] == best and
                        base + (parents[c] if parents is not None else c - base - 1) == cur]
                if left:
                    cur = left[0]
                    continue
            else:
                cum = np.cumsum(r)
                goal = float(draws[b]) * cum[-1]
                picks[cur] = min(int(np.searchsorted(cum, goal, side="right")), int(np.nonzero(r)[0][-1]))
                drawn = min(drawn, np.abs(cum - goal).min() / cum[-1])
            break
    return picks, margin, drawn
