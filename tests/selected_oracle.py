"""Plain statements in 64 bits of decode attention that reads less of the paged cache, and inputs
for it (numpy; caches as fp32 arrays of bf16 values)."""
import numpy as np

from oracle import decode_oracle as O

D = 128
SCALE = D ** -0.5


def bf16(a):
    """The nearest bf16 values, as fp32."""
    return O.bf16_round(np.asarray(a, np.float32))


def pool(rng, pages, page, hkv, layout):
    shape = (pages, page, hkv, D) if layout == "NHD" else (pages, hkv, page, D)
    return bf16(rng.standard_normal(shape, dtype=np.float32) * 0.5)


def tables(rng, lens, page, pages, extra=1):
    """Distinct pages for sequences of these lengths, -1 behind the last."""
    need = [-(-n // page) for n in lens]
    assert sum(need) <= pages
    order = rng.permutation(pages).astype(np.int32)
    t = np.full((len(lens), max(need + [0]) + extra), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t


def rows(cache, table, positions, head, page, layout):
    """Cached rows of one head at positions, [n, D] in 64 bits."""
    positions = np.asarray(positions, np.int64)
    p, o = table[positions // page], positions % page
    got = cache[p, o, head] if layout == "NHD" else cache[p, head, o]
    return got.astype(np.float64)


def attention(q, k, v, scale=SCALE):
    """(softmax(scale q k^T) v, sum of weights times |v|): of zeros where there are no keys."""
    if len(k) == 0:
        return np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    z = scale * (q.astype(np.float64) @ k.T)
    e = np.exp(z - z.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True)
    return p @ v, p @ np.abs(v)


def over_positions(q, kc, vc, lens, table, page, layout, hkv, positions):
    """Attention of every query row over positions(row, head); (out, weights times |v|)."""
    t, hq, _ = q.shape
    g = hq // hkv
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(t):
        for h in range(hkv):
            pos = positions(i, h)
            k = rows(kc, table[i], pos, h, page, layout)
            v = rows(vc, table[i], pos, h, page, layout)
            s = slice(h * g, (h + 1) * g)
            out[i, s], mass[i, s] = attention(q[i, s], k, v)
    return out, mass


def tolerance(out, mass):
    """The result is rounded to bf16 (half a step: 2^-8 of the value), and so is each weight on its
    way into the product with the values (2^-8 of the sum of weights times |v|).  A score is off by at
    most 2^-17 of the sum of |q k| (128 products added in fp32), here below 2^-14, a weight by
    twice that."""
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -8 + 2.0 ** -12) * mass + 1e-30


def bounds_of(kc, page, block, layout):
    """[pages, hkv, page // block, 2, D] of whole blocks."""
    k = kc if layout == "HND" else kc.swapaxes(1, 2)
    k = k.reshape(k.shape[0], k.shape[1], page // block, block, D)
    return np.stack([k.min(3), k.max(3)], 3)


def select(q, bounds, lens, table, block, count, keep_first, keep_last):
    """[tokens, hkv, count]; q [tokens, hq, D], table [tokens, pages]."""
    t, hq, _ = q.shape
    hkv, per = bounds.shape[1], bounds.shape[2]
    g = hq // hkv
    got = np.full((t, hkv, count), -1, np.int32)
    for i in range(t):
        n = -(-int(lens[i]) // block)
        b = np.arange(n)
        page = table[i, b // per]
        for h in range(hkv):
            of = bounds[np.where(page < 0, 0, page), h, b % per].astype(np.float64)  # [n, 2, D]
            a = q[i, h * g:(h + 1) * g, None].astype(np.float64)
            with np.errstate(invalid="ignore"):
                score = np.maximum(a * of[:, 0], a * of[:, 1]).sum(-1).max(0)
            # no-number scores first, blocks without a page last
            kind = np.where(page < 0, 2, np.where(np.isnan(score), 0, 1))
            kept = (b < keep_first) | (b >= n - keep_last)
            order = sorted(range(n), key=lambda x: (not kept[x], kind[x],
                                                    -score[x] if kind[x] == 1 else 0, x))
            best = sorted(order[:count])
            got[i, h, :len(best)] = best
    return got
