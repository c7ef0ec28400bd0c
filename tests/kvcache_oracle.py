"""KV caches that take less memory, plainly and in 64 bits: rows in 4 bits, attention over them with sums
of weights, eviction by those sums.

bf16 values travel as float32 arrays that hold them exactly."""
import numpy as np

from oracle import decode_oracle as O

D = 128


def bf16(x):
    """Nearest bf16 of a float32 array, as float32."""
    return O.bf16_round(np.asarray(x, np.float32))


def randn(rng, *shape, scale=0.5):
    off = rng.standard_normal(shape[-2:]).astype(np.float32) * 0.5
    return bf16(rng.standard_normal(shape).astype(np.float32) * np.float32(scale) + off)


# ------------------------------------------------------------------------------- 4 bits
def quantise(x, group):
    """(lowest [..., groups], scale, codes [..., 128]) of bf16 rows."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], D // group, group)
    bad = ~np.isfinite(g).all(-1)
    lo, hi = np.where(bad, 0, g.min(-1)), np.where(bad, 0, g.max(-1))
    s = bf16(np.float32(hi / 2 - lo / 2) / np.float32(7.5)).astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        y = np.where(s[..., None] > 0, (np.where(bad[..., None], 0, g) - lo[..., None]) /
                     s[..., None], 0)
    code = np.clip(np.rint(y), 0, 15).astype(np.uint8)
    return np.where(bad, np.nan, lo), np.where(bad, np.nan, s), code.reshape(x.shape)


def values(x, group):
    """What 4 bits keep of bf16 rows, in 64 bits."""
    lo, s, code = quantise(x, group)
    c = code.reshape(*x.shape[:-1], D // group, group).astype(np.float64)
    return (lo[..., None] + s[..., None] * c).reshape(x.shape)


def _bits(x):
    return O.bf16_round_bits(np.asarray(x, np.float32))


def pack(k, v, group):
    """Units [n / 16, bytes] of the rows of n tokens of one head."""
    ng, units = D // group, []
    for t in range(0, len(k), 16):
        parts, pairs = [], []
        for kv, x in enumerate((k[t:t + 16], v[t:t + 16])):
            lo, s, code = quantise(x, group)
            words = np.zeros((16, 16), np.uint32)
            for w in range(16):
                place = w % 4 * 4 + w // 4 if kv == 0 else w % 8 * 2 + w // 8
                for j in range(8):
                    words[:, place] |= code[:, 8 * w + j].astype(np.uint32) << np.uint32(4 * j)
            parts.append(words.view(np.uint8).reshape(-1))
            pair = np.stack([_bits(s), _bits(lo)], -1).astype(np.uint16)
            pair[np.isnan(lo)] = 0x7fc0
            pairs.append(np.ascontiguousarray(pair.reshape(16, ng, 2)).view(np.uint8).reshape(-1))
        units.append(np.concatenate(parts + pairs))
    return np.stack(units)


def pool_q4(pages, page, hkv, group, fill=0xFF):
    """Without tokens: by default every pair is no number."""
    return np.full((pages, hkv, page // 16, 2048 + 128 * (D // group)), fill, np.uint8)


def put(pool, k, v, slots, group):
    """Rows [n, hkv, 128] into the pool's slots."""
    ng, page = D // group, pool.shape[2] * 16
    for h in range(k.shape[1]):
        rows = []                                  # token by token: unit of its own, row 0 of it
        for t in range(0, len(k)):
            pad_k, pad_v = np.zeros((16, D), np.float32), np.zeros((16, D), np.float32)
            pad_k[0], pad_v[0] = k[t, h], v[t, h]
            rows.append(pack(pad_k, pad_v, group)[0])
        for unit, slot in zip(rows, slots):
            if slot < 0:
                continue
            u, i = pool[slot // page, h, slot % page // 16], slot % 16
            u[i * 64:i * 64 + 64] = unit[:64]
            u[1024 + i * 64:1024 + i * 64 + 64] = unit[1024:1088]
            n = 4 * ng
            u[2048 + i * n:2048 + i * n + n] = unit[2048:2048 + n]
            a = 2048 + 16 * n
            u[a + i * n:a + i * n + n] = unit[a:a + n]


def tables(rng, lens, page, pages, cols=None):
    """Page tables in random order, -1 behind the last page."""
    need = [-(-n // page) for n in lens]
    order = rng.permutation(pages)[:sum(need)]
    t = np.full((len(lens), max(max(need, default=1), cols or 1)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t


def slots_of(table, n, page):
    p = np.arange(n)
    return table[p // page].astype(np.int64) * page + p % page


# --------------------------------------------------------------------------- attention
def attention(q, k, v, lens, seq_of, scale):
    """q [tokens, hq, D]; k, v per sequence [n, hkv, D], in 64 bits.  (out, mass: sum p |v| with v
    counted from its group's lowest where `v` says so, reach: largest sum of |q k| scale a token
    and head has, weights per sequence [hkv, n])."""
    hkv = k[0].shape[1]
    g = q.shape[1] // hkv
    out = np.zeros(q.shape)
    mass, reach = np.zeros(q.shape), np.zeros(q.shape[:2])
    sums = [np.zeros((hkv, len(x))) for x in k]
    for t in range(len(q)):
        s, n = seq_of[t], lens[t]
        if s < 0 or n <= 0:
            continue
        for h in range(q.shape[1]):
            kk, vv, qq = k[s][:n, h // g], v[s][:n, h // g], q[t, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                z = kk @ qq * scale
                reach[t, h] = np.max(np.abs(kk) @ np.abs(qq)) * abs(scale)
                e = np.exp(z - z.max())
                e /= e.sum()
                out[t, h], mass[t, h] = e @ vv, e @ np.abs(vv)
            sums[s][h // g, :n] += e
    return out, mass, reach, sums


def evict(n, w, budget, first, last):
    """[(from, to)] of the rows that move, for one sequence and head with sums w [n]."""
    if n <= budget:
        return []
    w = np.where(np.isnan(w), -np.inf, w)
    middle = budget - last
    rank = sorted(range(first, n - last), key=lambda i: (-w[i], i))
    stay = set(range(first)) | set(rank[:middle - first])
    free = [i for i in range(middle) if i not in stay]
    movers = sorted(i for i in stay if i >= middle)
    assert len(free) == len(movers)
    return list(zip(movers, free)) + [(n - last + i, middle + i) for i in range(last)]
