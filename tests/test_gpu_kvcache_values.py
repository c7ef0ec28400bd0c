"""4-bit caches on the GPU: values that are no numbers, scales far apart, bad pages of long evictions."""
import numpy as np
import pytest
import torch

import kvcache_oracle as S
from gpu_util import dev, host_f32
from test_gpu_kvcache_small import Batch, check_sums, ints, raw, weight_error

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def ops():
    from fastkernels_b200 import ops as _ops
    return _ops


def near(got, b):
    """Against 64 bits, element by element, where neither is no number; which are has to agree.  Relative
    to what the weights give, not to the largest scale of all: bf16 of the result; per key the
    weight's error (weight_error) and, of the codes' part, fp16's (2^-11) or, below fp16's numbers,
    2^-25 where the largest weight times scale is 2^4 at least (of scales so small that this takes
    more than 2^118: 2^-25 of 2^-118); sums of products in fp32, 2^-22 of the whole each; half of
    bf16's smallest step, 2^-134."""
    kv = [[S.values(x, b.group) for x in side] for side in (b.k, b.v)]
    out, _, reach, sums = S.attention(b.q, *kv, b.q_lens, b.seq_of, b.scale)

    def given(rows):
        with np.errstate(invalid="ignore"):
            return S.attention(b.q, kv[0], [np.repeat(x, b.group, -1) for x in rows], b.q_lens, b.seq_of,
                               b.scale)[0]
    low = given([np.abs(S.quantise(x, b.group)[0]) for x in b.v])
    step = 15 * given([S.quantise(x, b.group)[1] for x in b.v])
    keys = max(b.lens)
    rel = weight_error(reach)[..., None] + (keys / 16 + 8) * 2.0 ** -22
    tol = np.abs(out) * 2.0 ** -8 + low * rel + step * (2.0 ** -11 + rel + keys * 2.0 ** -29) + \
        keys * 15 * 2.0 ** -143 + 2.0 ** -134
    got = host_f32(got).astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(out))
    d = np.where(np.isnan(out), 0, np.abs(got - out) - tol)
    assert (d <= 0).all(), (d.max(), np.unravel_index(d.argmax(), d.shape))
    return out, reach, sums


# ------------------------------------------------------------------------ values that are no numbers
@pytest.mark.parametrize("hq,hkv,page,group", [(4, 4, 64, 64), (8, 2, 16, 64), (8, 2, 64, 128),
                                               (8, 1, 256, 64), (6, 2, 32, 128), (32, 2, 64, 64)])
@pytest.mark.parametrize("lens,counts", [([70, 40], [5, 3]), ([64, 33], [2, 8]), ([5, 2500], [5, 4])])
@pytest.mark.parametrize("sums", [False, True])
def test_tokens_see_no_value_of_later_ones(ops, hq, hkv, page, group, lens, counts, sums):
    """A drafted token whose value or key is no number: only it and those behind it see it, in that group
    of channels (of a key: in all)."""
    rng = np.random.default_rng(hq + page + sum(lens))
    for back, what in ((1, np.nan), (2, np.inf), (2, "key"), (counts[0], -np.inf)):
        b = Batch(rng, lens, hq, hkv, group, page, counts)
        if what == "key":
            b.k[0][lens[0] - back, 0, 3] = np.nan
        else:
            b.v[0][lens[0] - back, 0, 100] = what
            b.v[1][lens[1] - 1, hkv - 1, 5] = what
        w = ops.new_attn_weights(b.tables.max() + 4, page, hkv)
        got = ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale,
                                       cu_seqlens_q=ints(b.cu), weights=w if sums else None)
        out, reach, want = near(got, b)
        seen = counts[0] - back                      # tokens before it
        assert not np.isnan(out[:seen]).any() and np.isnan(out[seen:counts[0]]).any()
        if sums and what != "key":
            check_sums(b, w, reach, want, None)


# -------------------------------------------------------------------------------- scales far apart
def steered(rng, lens, hkv, group, levels, v, slopes, counts=None):
    """A batch whose logits are slopes[head] * levels[token], in units of e: the keys' first channel says
    the level, the queries' first channel the slope."""
    hq = len(slopes)
    k = []
    for n in lens:
        x = S.randn(rng, n, hkv, D, scale=0.01) * np.float32(0.02)
        x[:, :, 0] = levels(n)[:, None]
        k.append(S.bf16(x))
    b = Batch(rng, lens, hq, hkv, group, 64, counts, k=k, v=v)
    b.q[...] = S.bf16(rng.standard_normal(b.q.shape).astype(np.float32) * np.float32(0.01))
    b.q[:, :, 0] = np.asarray(slopes, np.float32) * np.float32(8.0)
    b.scale = 0.125
    return b


@pytest.mark.parametrize("hq,hkv,group,counts", [(4, 4, 64, None), (8, 2, 64, None), (8, 2, 128, None),
                                                 (8, 1, 64, None), (16, 1, 128, None),
                                                 (16, 1, 64, None), (8, 2, 64, [3, 4]),
                                                 (5, 1, 128, [1, 6])])
@pytest.mark.parametrize("far", [22, 28, 60, 100])
def test_a_large_scale_counts_by_its_weight(ops, hq, hkv, group, counts, far):
    """One token's values are 2^far times the others' and its weight is less than 2^-far: what the others
    give is as exact as without it, wherever it stands, and for the heads that look at nothing else
    it is exact too."""
    rng = np.random.default_rng(far + hq)
    deep = far * 0.6931 + 14.0
    lens = [300, 2500]
    for place in (0, 20, 150, 290):
        v = [S.randn(rng, n, hkv, D) for n in lens]
        for x in v:
            x[place] = S.bf16(x[place] * np.float32(2.0 ** far))

        def levels(n):
            at = rng.uniform(-2, 0, n).astype(np.float32)
            at[place] = -deep
            return at
        # of every KV head's, the last query head looks the other way
        slopes = np.ones(hq)
        g = hq // hkv
        if g > 1:
            slopes[g - 1::g] = -1.0
        b = steered(rng, lens, hkv, group, levels, v, slopes, counts)
        got = ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale,
                                       cu_seqlens_q=ints(b.cu) if counts else None)
        near(got, b)


@pytest.mark.parametrize("hq,hkv,group", [(4, 4, 64), (8, 2, 128), (8, 1, 64), (16, 1, 64), (16, 1, 128)])
def test_scales_that_fall_while_logits_rise(ops, hq, hkv, group):
    """The largest weight times scale so far shrinks from step to step, and one group of channels is far
    below the other."""
    rng = np.random.default_rng(hq)
    lens = [400, 90]
    v = []
    for n in lens:
        x = S.randn(rng, n, hkv, D) * np.exp2(-np.arange(n) / 8.0 + 30)[:, None, None]
        x[:, :, 64:] *= 2.0 ** -40
        v.append(S.bf16(x.astype(np.float32)))

    def levels(n):
        return (np.arange(n) / 6.0).astype(np.float32) - 30
    near(*both(ops, steered(rng, lens, hkv, group, levels, v, np.ones(hq))))
    near(*both(ops, steered(rng, lens, hkv, group, levels, v, -np.ones(hq))))


@pytest.mark.parametrize("hq,hkv,group", [(4, 4, 64), (8, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("size", [-126, -100, 100])
def test_values_near_the_ends_of_the_type(ops, hq, hkv, group, size):
    rng = np.random.default_rng(hq)
    lens = [200, 33]
    v = [S.bf16((S.randn(rng, n, hkv, D).astype(np.float64) * 2.0 ** size).astype(np.float32))
         for n in lens]
    b = Batch(rng, lens, hq, hkv, group, 64, v=v)
    near(*both(ops, b))


def both(ops, b):
    return ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale), b


# ---------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("n,budget,first,last,cols", [(10000, 6000, 4, 100, 0), (10000, 9000, 0, 0, 0),
                                                      (40000, 24000, 16, 300, 30)])
@pytest.mark.parametrize("many", [False, True])
def test_bad_pages_of_evictions_with_many_moves(ops, n, budget, first, last, cols, many):
    """More moves than a list holds, and places among the first that take nothing: the i-th token that
    stays still goes to the i-th place that became free, or nowhere.  many: so many bad pages that
    tokens of them stay."""
    rng = np.random.default_rng(n + budget)
    pages = -(-n // 64) + 2
    table = np.full(-(-n // 64) + cols, -1, np.int32)
    table[:-(-n // 64)] = rng.permutation(pages)[:-(-n // 64)]
    live = -(-(n - last) // 64) - 1
    bad = np.sort(rng.permutation(np.arange(first // 64 + 1, live))[:(n - budget) // 64 + 8 if many else 5])
    if not many:
        bad[:2] = first // 64 + 1, first // 64 + 3                # places that the first round fills
    table[bad] = np.where(np.arange(len(bad)) % 2, -1, pages)
    at = np.arange(n)
    there = ~np.isin(at // 64, bad)
    slot = np.where(there, table[at // 64].astype(np.int64) * 64 + at % 64, 0)
    # most of what stays stands behind the budget
    key = rng.random(n).astype(np.float32) + (at > 0.45 * n)
    w = np.full(pages * 64, -5.0, np.float32)
    w[slot[there]] = key[there]
    rows = rng.integers(0, 2 ** 15, (pages * 64, 2, D), dtype=np.int16)
    middle = budget - last
    order = sorted(range(first, n - last), key=lambda i: (-(key[i] if there[i] else -np.inf), i))
    stay = np.zeros(n, bool)
    stay[:first] = True
    stay[order[:middle - first]] = True
    movers = np.flatnonzero(stay & (at >= middle) & (at < n - last))
    free = np.flatnonzero(~stay[:middle])
    assert len(movers) == len(free) and len(movers) > (8192 if cols else min(1500, n - budget - 300))
    moves = list(zip(movers, free)) + [(n - last + i, middle + i) for i in range(last)]
    want_w, want = w.copy(), rows.copy()
    for a, b in moves:
        if there[a] and there[b]:
            want_w[slot[b]], want[slot[b]] = w[slot[a]], rows[slot[a]]
    pools = [raw(rows[:, i].reshape(pages, 64, 1, D)).view(torch.bfloat16) for i in range(2)]
    dw, st = raw(w.reshape(pages, 1, 64)), ops.new_status("cuda")
    new = ops.evict_kvcache(tuple(pools), dw, ints([n]), ints([table]), budget, first, last, status=st)
    assert new.tolist() == [budget] and int(st.item()) == 2
    np.testing.assert_array_equal(dw.cpu().numpy().reshape(-1), want_w)
    for i, x in enumerate(pools):
        np.testing.assert_array_equal(x.view(torch.int16).cpu().numpy().reshape(-1, D), want[:, i])


def test_budgets_beyond_32_bits_are_refused(ops):
    from fastkernels_b200._lib import FkError
    w, cache = ops.new_attn_weights(4, 16, 1), ops.new_kvcache_q4(4, 16, 1)
    lens, t = ints([60]), ints([[0, 1, 2, 3]])
    for args in ((2 ** 32 + 20,), (2 ** 31,), (40, 2 ** 32 + 1), (40, 0, 2 ** 32 + 1), (-2 ** 32 + 20,)):
        with pytest.raises(FkError, match="32 bits"):
            ops.evict_kvcache(cache, w, lens, t, *args)
    assert ops.evict_kvcache(cache, w, lens, t, 2 ** 31 - 1).tolist() == [60]
