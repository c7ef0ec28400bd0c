"""KV caches that take less memory on the GPU: 4 bits a value, sums of softmax weights, eviction."""
import numpy as np
import pytest
import torch

import kvcache_oracle as S
from gpu_util import dev, host_f32

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(scope="module")
def ops():
    from fastkernels_b200 import ops as _ops
    return _ops


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def raw(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---------------------------------------------------------------------------- store and load
def special_rows(rng, n, hkv):
    """Rows whose groups are hard to cut: ties, one value, the type's ends, no numbers."""
    x = S.randn(rng, n, hkv, D)
    x[0] = S.bf16(rng.integers(-8, 9, (hkv, D)))              # many quotients are halves
    x[1] = 0.0
    x[2] = S.bf16(np.float32(1.0078125))                       # all equal
    x[3] = S.bf16(rng.uniform(-3.3e38, 3.3e38, (hkv, D)).astype(np.float32))
    x[4] = S.bf16(rng.integers(-200, 200, (hkv, D)) * np.float32(2.0 ** -133))
    x[5, :, 3] = np.inf
    x[6, :, 77] = np.nan
    x[7, 0, 5] = -np.inf
    x[8] = S.bf16(np.exp2(rng.uniform(-30, 3, (hkv, D))).astype(np.float32))
    x[9] = S.bf16(np.arange(D, dtype=np.float32) * 0.5)        # (x - lo) / s close to halves
    x[10, :, :64] = 0.0
    x[11] = S.bf16(rng.integers(0, 31, (hkv, D)) * np.float32(0.5))
    return x


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("page,hkv,wide", [(16, 1, True), (64, 5, False), (192, 2, True),
                                           (256, 8, False)])
def test_store_is_exact_and_loads_back(ops, group, page, hkv, wide):
    rng = np.random.default_rng(page + hkv + group)
    n, pages = 61, 2 + 200 // page
    k, v = special_rows(rng, n, hkv), special_rows(rng, n, hkv)[::-1].copy()
    slots = rng.permutation(pages * page)[:n]
    slots[20], slots[33] = -1, -7
    want = S.pool_q4(pages, page, hkv, group, fill=0x5A)
    cache = raw(want)
    S.put(want, k, v, slots, group)
    # rows of a packed projection: heads dense, tokens further apart
    both = torch.zeros((n, 2 * hkv + 1, D), dtype=torch.bfloat16, device="cuda")
    both[:, :hkv], both[:, hkv:2 * hkv] = dev(k), dev(v)
    st = ops.new_status("cuda")
    idx = torch.tensor(slots, dtype=torch.int64 if wide else torch.int32, device="cuda")
    ops.store_kvcache_q4(both[:, :hkv], both[:, hkv:2 * hkv], cache, idx, status=st)
    np.testing.assert_array_equal(cache.cpu().numpy(), want)
    got = ops.load_kvcache_q4(cache, idx, status=st)
    for x, y in zip((k, v), got):
        back = S.bf16(S.values(x, group).astype(np.float32))
        back[slots < 0] = 0.0
        np.testing.assert_array_equal(host_f32(y), back)
        assert np.isnan(back).any()
    assert int(st.item()) == 0


def test_slots_behind_the_pool_are_flagged(ops):
    cache = ops.new_kvcache_q4(2, 16, 2, group=128)
    x = torch.ones((3, 2, D), dtype=torch.bfloat16, device="cuda")
    for wide in (torch.int32, torch.int64):
        cache.zero_()
        st = ops.new_status("cuda")
        slots = torch.tensor([32, 5, 2 ** 31 - 1 if wide is torch.int32 else 2 ** 40], dtype=wide,
                             device="cuda")
        ops.store_kvcache_q4(x, x, cache, slots, status=st)
        assert int(st.item()) == 1
        st.zero_()
        k, v = ops.load_kvcache_q4(cache, slots, status=st)
        assert int(st.item()) == 1
        assert k[1].eq(1).all() and k[0].eq(0).all() and v[2].eq(0).all()


def test_nothing_to_store_or_load(ops):
    cache = ops.new_kvcache_q4(2, 64, 2)
    x = torch.ones((0, 2, D), dtype=torch.bfloat16, device="cuda")
    ops.store_kvcache_q4(x, x, cache, ints([]))
    assert ops.load_kvcache_q4(cache, ints([]))[0].shape == (0, 2, D)
    assert not cache.any()


# -------------------------------------------------------------------------------- attention
class Batch:
    """Sequences of `lens` tokens in a pool that holds nothing else but no numbers."""

    def __init__(self, rng, lens, hq, hkv, group, page, q_counts=None, q_scale=1.0, k=None, v=None,
                 spare=3):
        self.page, self.group, self.hkv = page, group, hkv
        self.lens = list(lens)
        pages = sum(-(-n // page) for n in lens) + spare
        self.tables = S.tables(rng, lens, page, pages, cols=max(1, -(-max(lens) // page)) + 1)
        self.k = k or [S.randn(rng, n, hkv, D) for n in lens]
        self.v = v or [S.randn(rng, n, hkv, D) for n in lens]
        self.counts = q_counts or [1] * len(lens)
        tokens = sum(self.counts)
        self.q = S.bf16(rng.standard_normal((tokens, hq, D)).astype(np.float32) * q_scale)
        self.seq_of = [s for s, c in enumerate(self.counts) for _ in range(c)]
        self.q_lens = [max(0, n - c + 1 + j) for n, c in zip(lens, self.counts) for j in range(c)]
        self.cu = np.concatenate([[0], np.cumsum(self.counts)])
        self.scale = D ** -0.5

    def cache(self, ops):
        """Through the store (tested above)."""
        c = raw(S.pool_q4(self.tables.max() + 4, self.page, self.hkv, self.group))
        for i, n in enumerate(self.lens):
            if n:
                ops.store_kvcache_q4(dev(self.k[i]), dev(self.v[i]), c,
                                     torch.tensor(S.slots_of(self.tables[i], n, self.page)).cuda())
        return c

    def expect(self):
        kv = [[S.values(x, self.group) for x in side] for side in (self.k, self.v)]
        return S.attention(self.q, *kv, self.q_lens, self.seq_of, self.scale)

    def spread(self):
        """Largest step of the values' scales."""
        return max([float(np.nanmax(S.quantise(x, self.group)[1])) for x in self.v if len(x)],
                   default=0.0)


def weight_error(reach):
    """Relative error of a softmax weight: logits are sums of products with |sum| <= reach, in fp32 with
    16 accumulations, each off by 2^-23 of the partial sum at most, twice (the codes' part and the
    lowest's: |s c| + |lo| <= 3 max |x| counts as 4), and 2^-20 for the exponential; the same for the
    sum that divides."""
    return 2 * (4 * 16 * 2.0 ** -23 * reach * 1.45 + 2.0 ** -20)


def close_out(got, out, mass, reach, keys, spread):
    """bf16 of the result; weights to fp16 (2^-11 each, on the part counted from the lowest: at most
    twice the mass and the spread); what is below fp16's numbers: 2^-25 of 1/64 of the largest
    scale's power of two, 15 steps, per key."""
    rel = weight_error(reach)[..., None]
    tol = np.abs(out) * 2.0 ** -8 + (2 * mass + 15 * spread) * (2.0 ** -11 + rel) + \
        keys * 15 * spread * 2.0 ** -29
    d = np.abs(host_f32(got).astype(np.float64) - out)
    assert (d <= tol).all(), ((d - tol).max(), np.unravel_index((d - tol).argmax(), d.shape))


def check(ops, b, use_cu, **kw):
    st = ops.new_status("cuda")
    got = ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale,
                                   cu_seqlens_q=ints(b.cu) if use_cu else None, status=st, **kw)
    out, mass, reach, _ = b.expect()
    close_out(got, out, mass, reach, max(b.lens), b.spread())
    assert int(st.item()) == 0
    return got


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 500]


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("hq,hkv,page", [(8, 8, 16), (8, 4, 64), (6, 2, 32), (32, 8, 256),
                                         (10, 2, 16), (7, 1, 64), (16, 2, 192), (12, 1, 32),
                                         (64, 4, 16), (11, 1, 128)])
def test_attention_of_any_ratio_and_page(ops, hq, hkv, page, group):
    rng = np.random.default_rng(hq * page + group)
    check(ops, Batch(rng, EDGES, hq, hkv, group, page), False)


@pytest.mark.parametrize("lens", [[1], [5000], [40000], [1] * 700, [0, 0, 3, 0], [2048] * 3,
                                  list(range(1, 300, 7))])
def test_attention_split_and_whole(ops, lens):
    rng = np.random.default_rng(len(lens))
    check(ops, Batch(rng, lens, 8, 2, 64, 64), False)


@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 1), (16, 1), (2, 2)])
@pytest.mark.parametrize("lens", [[100], [128], [129], [33, 0], [257], [1025], [5, 4000]])
def test_few_pairs_under_wide_tables(ops, hq, hkv, lens):
    """Runs of the fewest steps: pairs that one warp has whole, a CTA has alone, or several have."""
    rng = np.random.default_rng(sum(lens) + hq)
    b = Batch(rng, lens, hq, hkv, 64, 64)
    wide = np.full((len(lens), 40), -1, np.int32)
    wide[:, :min(40, b.tables.shape[1])] = b.tables[:, :40]
    if max(lens) <= 2048:
        b.tables = wide
    check(ops, b, False)
    w = ops.new_attn_weights(b.tables.max() + 4, 64, hkv)
    ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale, weights=w)
    _, _, reach, sums = b.expect()
    check_sums(b, w, reach, sums, None)


@pytest.mark.parametrize("hq,hkv,group,page", [(8, 2, 64, 64), (5, 5, 128, 16), (16, 1, 64, 32),
                                               (9, 3, 128, 256), (12, 2, 64, 16)])
@pytest.mark.parametrize("counts", [[1, 4, 1, 7], [0, 40, 0, 3], [2, 2, 2, 2], [1, 1, 1, 1],
                                    [17, 16, 15, 5]])
def test_attention_of_several_tokens_of_a_sequence(ops, hq, hkv, group, page, counts):
    rng = np.random.default_rng(sum(counts) + hq)
    check(ops, Batch(rng, [130, 77, 33, 12], hq, hkv, group, page, counts), True)


def test_rows_of_no_sequence_stay_as_they_are(ops):
    rng = np.random.default_rng(1)
    b = Batch(rng, [90, 40, 7], 8, 2, 64, 64, [2, 3, 1])
    pad = 5
    q = np.concatenate([b.q[:2] * 0, b.q, np.full((pad, 8, D), np.nan, np.float32)])
    lens = [9, 9] + b.q_lens + [100000] * pad          # of padded rows: any number
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device="cuda")
    w = ops.new_attn_weights(b.tables.max() + 4, 64, 2)
    st = ops.new_status("cuda")
    cache = b.cache(ops)
    for weights in (None, w):
        out.fill_(3.0)
        ops.paged_decode_attn_q4(dev(q), cache, ints(lens), ints(b.tables), b.scale,
                                 cu_seqlens_q=ints(b.cu + 2), weights=weights, out=out, status=st)
        assert out[:2].eq(3).all() and out[-pad:].eq(3).all() and int(st.item()) == 0
        o, mass, reach, _ = b.expect()
        close_out(out[2:-pad], o, mass, reach, 90, b.spread())


def test_strided_rows_and_tables(ops):
    rng = np.random.default_rng(2)
    b = Batch(rng, [300, 65, 2], 8, 2, 128, 64)
    wide = torch.zeros((3, 20, D), dtype=torch.bfloat16, device="cuda")
    wide[:, 4:12] = dev(b.q)
    t = torch.full((3, 11), -1, dtype=torch.int32, device="cuda")
    t[:, :b.tables.shape[1]] = ints(b.tables)
    out = torch.full((3, 24, D), 9.0, dtype=torch.bfloat16, device="cuda")
    got = ops.paged_decode_attn_q4(wide[:, 4:12], b.cache(ops), ints(b.q_lens),
                                   t[:, :b.tables.shape[1]], b.scale, out=out[:, 8:16])
    o, mass, reach, _ = b.expect()
    close_out(got, o, mass, reach, 300, b.spread())
    assert out[:, :8].eq(9).all() and out[:, 16:].eq(9).all()


@pytest.mark.parametrize("case", ["sharp", "far scales", "offset keys", "growing", "flat", "tiny q"])
def test_values_of_every_size(ops, case):
    """Logits far apart, scales from 2^-20 to 2^10 in one context, keys around a large value, logits that
    grow from step to step, values without any spread, queries near the type's end."""
    rng = np.random.default_rng(5)
    lens, hkv = [257, 40, 1000], 2
    k = [S.randn(rng, n, hkv, D) for n in lens]
    v = [S.randn(rng, n, hkv, D) for n in lens]
    q_scale = 1.0
    if case == "sharp":
        q_scale = 8.0
    elif case == "far scales":
        v = [S.bf16(x * np.exp2(rng.integers(-20, 11, (len(x), hkv, 1)))) for x in v]
    elif case == "offset keys":
        k = [S.bf16(x + 6.0) for x in k]
    elif case == "growing":
        k = [S.bf16(x * (0.1 + np.arange(len(x)) / 100)[:, None, None].astype(np.float32)) for x in k]
    elif case == "flat":
        v = [np.full_like(x, 0.75) for x in v]
    else:
        q_scale = 2.0 ** -100
    b = Batch(rng, lens, 8, hkv, 64, 64, q_scale=q_scale, k=k, v=v)
    got = ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables), b.scale)
    out, mass, reach, _ = b.expect()
    close_out(got, out, mass, reach, max(lens), b.spread())
    if case == "flat":
        assert got.eq(0.75).all()


def test_no_numbers_stay_in_their_sequence(ops):
    rng = np.random.default_rng(6)
    b = Batch(rng, [100, 100, 100], 4, 2, 64, 64)
    b.k[0][50, 0, 3] = np.nan                       # KV head 0 of sequence 0
    b.v[1][7, 1, 100] = np.inf                      # the second group of head 1 of sequence 1
    got = host_f32(ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables),
                                            b.scale))
    nan = np.isnan(got)
    assert nan[0, :2].all() and not nan[0, 2:].any()
    assert nan[1, 2:, 64:].all() and not nan[1, 2:, :64].any() and not nan[1, :2].any()
    assert not nan[2].any()
    b.q[2, 3, 5] = np.inf
    got = host_f32(ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints(b.q_lens), ints(b.tables),
                                            b.scale))
    assert np.isnan(got[2, 3]).all() and not np.isnan(got[2, :3]).any()


def test_bad_pages_are_left_out_and_flagged(ops):
    rng = np.random.default_rng(7)
    for page in (16, 64):
        b = Batch(rng, [200, 200, 64], 8, 2, 64, page)
        cache = b.cache(ops)
        t = b.tables.copy()
        t[0, 1], t[1, 0] = -1, cache.shape[0]
        gone = {0: np.arange(page, 2 * page), 1: np.arange(page)}
        st = ops.new_status("cuda")
        w = ops.new_attn_weights(cache.shape[0], page, 2)
        for weights in (None, w):
            st.zero_()
            got = ops.paged_decode_attn_q4(dev(b.q), cache, ints(b.q_lens), ints(t), b.scale,
                                           status=st, weights=weights)
            assert int(st.item()) == 2
            kv = [[S.values(np.delete(x, gone.get(i, []), 0), 64) for i, x in enumerate(side)]
                  for side in (b.k, b.v)]
            out, mass, reach, _ = S.attention(b.q, *kv, [len(x) for x in kv[0]], b.seq_of, b.scale)
            close_out(got, out, mass, reach, 200, b.spread())
        # every weight is in the pool
        assert abs(float(w.sum()) - 3 * 8) < 1e-3


def test_contexts_beyond_the_table_are_cut_and_flagged(ops):
    rng = np.random.default_rng(8)
    b = Batch(rng, [128, 50], 8, 2, 64, 64)
    t = ints(b.tables[:, :2])
    st = ops.new_status("cuda")
    got = ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints([2 ** 31 - 1, 50]), t, b.scale, status=st)
    assert int(st.item()) == 2
    out, mass, reach, _ = b.expect()
    close_out(got, out, mass, reach, 128, b.spread())
    assert ops.paged_decode_attn_q4(dev(b.q), b.cache(ops), ints([-5, 0]), t, b.scale).eq(0).all()


def test_far_pages(ops):
    """A pool beyond 2^32 bytes: the pages at its end."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [500, 70], 8, 8, 64, 256)
    pages = 15500
    cache = torch.zeros((pages, 8, 16, 2304), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 2 ** 32
    far = np.where(b.tables >= 0, b.tables + pages - 10, -1)
    for i, n in enumerate(b.lens):
        slots = torch.tensor(S.slots_of(far[i], n, 256)).cuda()
        ops.store_kvcache_q4(dev(b.k[i]), dev(b.v[i]), cache, slots)
        k, _ = ops.load_kvcache_q4(cache, slots)
        np.testing.assert_array_equal(host_f32(k), S.bf16(S.values(b.k[i], 64).astype(np.float32)))
    got = ops.paged_decode_attn_q4(dev(b.q), cache, ints(b.q_lens), ints(far), b.scale)
    out, mass, reach, _ = b.expect()
    close_out(got, out, mass, reach, 500, b.spread())


def test_calls_share_a_workspace_and_repeat_their_bits(ops):
    rng = np.random.default_rng(10)
    a, b = Batch(rng, [900, 33], 8, 2, 64, 64), Batch(rng, [5, 700, 1300], 16, 2, 64, 64)
    size = max(ops.paged_decode_attn_q4_workspace_bytes(2, 2, 8, 2, D),
               ops.paged_decode_attn_q4_workspace_bytes(3, 3, 16, 2, D))
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    ca, cb = a.cache(ops), b.cache(ops)

    def both():
        return [ops.paged_decode_attn_q4(dev(x.q), c, ints(x.q_lens), ints(x.tables), x.scale,
                                         workspace=ws) for x, c in ((a, ca), (b, cb))]
    first = both()
    for x, got in zip((a, b), first):
        out, mass, reach, _ = x.expect()
        close_out(got, out, mass, reach, 1300, x.spread())
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, both()))


def test_captured_calls_follow_their_inputs(ops):
    """Two graphs with workspaces of their own, replayed with other lengths and tables, on a side
    stream."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [400, 90, 1], 8, 2, 64, 64)
    cache = b.cache(ops)
    q, lens, t = dev(b.q), ints([3, 3, 1]), ints(b.tables)
    w = ops.new_attn_weights(cache.shape[0], 64, 2)
    size = ops.paged_decode_attn_q4_workspace_bytes(3, 3, 8, 2, D, True, t.shape[1] * 64)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(q) for _ in range(2)]
    ops.paged_decode_attn_q4(q, cache, lens, t, b.scale, workspace=ws, out=outs[0], weights=w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_decode_attn_q4(q, cache, lens, t, b.scale, workspace=ws, out=outs[0], weights=w)
        ops.paged_decode_attn_q4(q, cache, lens, t, b.scale, out=outs[1])
    lens.copy_(ints(b.q_lens))
    w.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    side.synchronize()
    out, mass, reach, sums = b.expect()
    for got in outs:
        close_out(got, out, mass, reach, 400, b.spread())
    check_sums(b, w, reach, sums, None)


# ---------------------------------------------------------------------------- sums of weights
def gather_sums(b, w):
    """Entries per sequence [hkv, n]."""
    w = w.cpu().numpy().astype(np.float64)
    out = []
    for i, n in enumerate(b.lens):
        p = np.arange(n)
        out.append(w[b.tables[i, p // b.page], :, p % b.page].T if n else np.zeros((b.hkv, 0)))
    return out


def check_sums(b, w, reach, sums, old):
    rel = weight_error(reach.max()) if reach.size else 0
    for i, (got, want) in enumerate(zip(gather_sums(b, w), sums)):
        base = 0.0 if old is None else old[i]
        total = base + want
        tol = want * rel + 2.0 ** -22 * np.abs(total) + 2.0 ** -126
        assert (np.abs(got - total) <= tol).all(), (np.abs(got - total) - tol).max()


@pytest.mark.parametrize("start", ["own", "zero", "part"])
@pytest.mark.parametrize("hq,hkv,group,page,counts", [
    (8, 2, 64, 64, None), (12, 4, 128, 16, None), (32, 2, 64, 256, None),
    (8, 2, 64, 64, [3, 1, 20, 0, 2]), (5, 1, 128, 32, [1, 6, 33, 2, 1])])
def test_sums_of_weights(ops, hq, hkv, group, page, counts, start):
    rng = np.random.default_rng(hq + page)
    b = Batch(rng, [70, 33, 700, 5, 300], hq, hkv, group, page, counts)
    cache = b.cache(ops)
    pages = cache.shape[0]
    before = rng.uniform(0, 3, (pages, hkv, page)).astype(np.float32)
    w = raw(before)
    frm = {"own": None, "zero": [0] * 5, "part": [10, 40, 650, 0, 299]}[start]
    st = ops.new_status("cuda")
    got = ops.paged_decode_attn_q4(
        dev(b.q), cache, ints(b.q_lens), ints(b.tables), b.scale,
        cu_seqlens_q=ints(b.cu) if counts else None, weights=w,
        weights_from=None if frm is None else ints(frm), status=st)
    out, mass, reach, sums = b.expect()
    close_out(got, out, mass, reach, 700, b.spread())
    assert int(st.item()) == 0
    old = gather_sums(b, torch.from_numpy(before))
    touched = np.zeros(before.shape, bool)
    for i, n in enumerate(b.lens):
        if b.counts[i] == 0:
            continue                                # no query: as it was
        f = frm[i] if frm else max(0, n - b.counts[i] + 1) - 1
        old[i][:, max(0, f):] = 0
        p = np.arange(n)
        touched[b.tables[i, p // page], :, p % page] = True
    check_sums(b, w, reach, sums, old)
    np.testing.assert_array_equal(w.cpu().numpy()[~touched], before[~touched])
    again = raw(before)
    ops.paged_decode_attn_q4(dev(b.q), cache, ints(b.q_lens), ints(b.tables), b.scale,
                             cu_seqlens_q=ints(b.cu) if counts else None, weights=again,
                             weights_from=None if frm is None else ints(frm))
    assert torch.equal(w, again)


@pytest.mark.parametrize("hq,hkv,page,layout,counts", [
    (8, 2, 64, "NHD", None), (8, 1, 16, "HND", None), (16, 1, 256, "NHD", None),
    (3, 3, 32, "NHD", [3, 1, 20, 0, 2]), (16, 4, 64, "HND", [1, 6, 33, 2, 1])])
@pytest.mark.parametrize("start", ["own", "zero"])
def test_sums_of_weights_over_bf16(ops, hq, hkv, page, layout, counts, start):
    rng = np.random.default_rng(hq + page)
    b = Batch(rng, [70, 33, 2500, 5, 300], hq, hkv, 64, page, counts)
    pages = b.tables.max() + 2
    kc, vc = (np.full((pages, page, hkv, D), np.nan, np.float32) for _ in range(2))
    for i, n in enumerate(b.lens):
        p = np.arange(n)
        kc[b.tables[i, p // page], p % page] = b.k[i]
        vc[b.tables[i, p // page], p % page] = b.v[i]
    if layout == "HND":
        kc, vc = kc.transpose(0, 2, 1, 3), vc.transpose(0, 2, 1, 3)
    before = rng.uniform(0, 3, (pages, hkv, page)).astype(np.float32)
    w = raw(before)
    frm = None if start == "own" else [0] * 5
    st = ops.new_status("cuda")
    tokens = len(b.q)
    q = np.concatenate([b.q, np.zeros((2, hq, D), np.float32)]) if counts else b.q
    lens = b.q_lens + [10 ** 6] * (len(q) - tokens)
    res = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_decode_attn_weights(
        dev(q), dev(kc), dev(vc), ints(lens), ints(b.tables), b.scale, w,
        cu_seqlens_q=ints(b.cu) if counts else None, out=res,
        weights_from=None if frm is None else ints(frm), kv_layout=layout, status=st)
    assert res[tokens:].eq(3).all() and int(st.item()) == 0
    out, mass, reach, sums = S.attention(b.q, [x.astype(np.float64) for x in b.k],
                                         [x.astype(np.float64) for x in b.v], b.q_lens, b.seq_of,
                                         b.scale)
    d = np.abs(host_f32(res[:tokens]) - out)
    # bf16 of the result and of each weight
    assert (d <= np.abs(out) * 2.0 ** -8 + mass * (2.0 ** -8 + weight_error(reach)[..., None])).all()
    old = gather_sums(b, torch.from_numpy(before))
    touched = np.zeros(before.shape, bool)
    for i, n in enumerate(b.lens):
        if b.counts[i] == 0:
            continue
        f = 0 if frm else max(0, n - b.counts[i] + 1) - 1
        old[i][:, max(0, f):] = 0
        p = np.arange(n)
        touched[b.tables[i, p // page], :, p % page] = True
    check_sums(b, w, reach, sums, old)
    np.testing.assert_array_equal(w.cpu().numpy()[~touched], before[~touched])


def test_contexts_beyond_max_context_len_are_cut_and_flagged(ops):
    rng = np.random.default_rng(12)
    b = Batch(rng, [128, 50], 8, 2, 64, 64)
    cache = b.cache(ops)
    w = ops.new_attn_weights(cache.shape[0], 64, 2)
    st = ops.new_status("cuda")
    ops.paged_decode_attn_q4(dev(b.q), cache, ints(b.q_lens), ints(b.tables), b.scale, weights=w,
                             max_context_len=100, status=st)
    assert int(st.item()) == 2
    got = gather_sums(b, w)
    assert got[0][:, 100:].sum() == 0 and abs(got[0].sum() - 8) < 1e-4
    kc = torch.randn((cache.shape[0], 64, 2, D), device="cuda").bfloat16()
    st.zero_()
    w.zero_()
    ops.paged_decode_attn_weights(dev(b.q), kc, kc, ints(b.q_lens), ints(b.tables), b.scale, w,
                                  max_context_len=100, status=st)
    assert int(st.item()) == 2
    got = gather_sums(b, w)
    assert got[0][:, 100:].sum() == 0 and abs(got[0].sum() - 8) < 1e-4


# -------------------------------------------------------------------------------- eviction
def run_evict(ops, rng, lens, budget, first, last, weights, page, hkv, kind, group=64, cols=None):
    pages = sum(-(-n // page) for n in lens) + 2
    t = S.tables(rng, lens, page, pages, cols)
    w = np.full((pages, hkv, page), -3.0, np.float32)
    for i, n in enumerate(lens):
        p = np.arange(n)
        w[t[i, p // page], :, p % page] = weights(n).T
    if kind == "q4":
        pools = [rng.integers(0, 256, (pages, hkv, page // 16, 2048 + 128 * (D // group)),
                              dtype=np.uint8)]
    else:
        shape = (pages, page, hkv, D) if kind == "NHD" else (pages, hkv, page, D)
        pools = [rng.integers(0, 2 ** 15, shape, dtype=np.int16) for _ in range(2)]
    want, want_w = [x.copy() for x in pools], w.copy()

    def row(x, i, h, pos):
        a, o = t[i, pos // page], pos % page
        if kind == "NHD":
            return [x[a, o, h]]
        if kind == "HND":
            return [x[a, h, o]]
        u, j, n = x[a, h, o // 16], o % 16, 4 * (D // group)
        return [u[j * 64:j * 64 + 64], u[1024 + j * 64:1088 + j * 64],
                u[2048 + j * n:2048 + j * n + n], u[2048 + 16 * n + j * n:2048 + 16 * n + j * n + n]]
    moved = 0
    for i, n in enumerate(lens):
        p = np.arange(n)
        for h in range(hkv):
            for src, dst in S.evict(n, w[t[i, p // page], h, p % page], budget, first, last):
                moved += 1
                for x, y in zip(pools, want):
                    for a, b in zip(row(x, i, h, src), row(y, i, h, dst)):
                        b[...] = a
                want_w[t[i, dst // page], h, dst % page] = w[t[i, src // page], h, src % page]
    dev_w = raw(w)
    caches = [raw(x) for x in pools]
    if kind != "q4":
        caches = [x.view(torch.bfloat16) for x in caches]
    st = ops.new_status("cuda")
    new = ops.evict_kvcache(caches[0] if kind == "q4" else tuple(caches), dev_w, ints(lens), ints(t),
                            budget, keep_first=first, keep_last=last,
                            kv_layout="NHD" if kind == "q4" else kind, status=st)
    assert new.tolist() == [min(n, budget) for n in lens]
    np.testing.assert_array_equal(dev_w.cpu().numpy(), want_w)
    for x, y in zip(caches, want):
        x = x if kind == "q4" else x.view(torch.int16)
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    assert int(st.item()) == 0
    return moved


def spread_weights(rng, hkv):
    return lambda n: (rng.random((hkv, n)) ** 6 * 3).astype(np.float32)


@pytest.mark.parametrize("kind,group", [("NHD", 0), ("HND", 0), ("q4", 64), ("q4", 128)])
@pytest.mark.parametrize("budget,first,last,page,hkv", [
    (64, 4, 10, 16, 2), (100, 0, 0, 64, 3), (1, 0, 0, 16, 1), (1, 0, 1, 32, 2), (1, 1, 0, 64, 1),
    (130, 1, 129, 64, 2), (200, 200, 0, 32, 1), (77, 3, 40, 192, 5)])
def test_eviction(ops, kind, group, budget, first, last, page, hkv):
    rng = np.random.default_rng(budget + page)
    lens = [0, 1, budget - 1, budget, budget + 1, budget + 17, 2 * budget + 300, 3]
    moved = run_evict(ops, rng, lens, budget, first, last, spread_weights(rng, hkv), page, hkv, kind,
                      group)
    assert (moved == 0) == (first == budget)       # only the first stay: none has to move


@pytest.mark.parametrize("name", ["equal", "few values", "no numbers", "infinite", "signs",
                                  "one octave", "neighbours"])
def test_eviction_of_any_weights(ops, name):
    """Ties go to the lower place, whatever the entries are."""
    rng = np.random.default_rng(13)
    hkv = 2

    def weights(n):
        x = rng.random((hkv, n)).astype(np.float32)
        if name == "equal":
            x[:] = 0.0
        elif name == "few values":
            x = np.floor(x * 3).astype(np.float32)
        elif name == "no numbers":
            x[x < 0.7] = np.nan
        elif name == "infinite":
            x[x < 0.3], x[x > 0.8] = -np.inf, np.inf
        elif name == "signs":
            x = (x - 0.5).astype(np.float32)
            x[rng.random(x.shape) < 0.3] = -0.0
            x[rng.random(x.shape) < 0.3] = 0.0
        elif name == "one octave":
            x = 1 + x
        else:
            x = np.float32(1) + rng.integers(0, 40, x.shape) * np.float32(2.0 ** -23)
        return x.astype(np.float32)
    for kind in ("NHD", "q4"):
        for lens, budget, first, last in (([700, 300, 90], 200, 4, 20), ([1000], 150, 0, 0)):
            run_evict(ops, rng, lens, budget, first, last, weights, 64, hkv, kind)


@pytest.mark.parametrize("kind", ["NHD", "q4"])
@pytest.mark.parametrize("n,budget,first,last", [(30000, 9000, 16, 300), (20000, 19990, 0, 5000),
                                                 (13000, 500, 4, 0)])
def test_eviction_of_long_contexts(ops, kind, n, budget, first, last):
    """More keys than are kept, more moves than fit a list."""
    rng = np.random.default_rng(14)
    run_evict(ops, rng, [n, budget + 40], budget, first, last, spread_weights(rng, 1), 256, 1, kind,
              cols=-(-n // 256) + 30)


@pytest.mark.parametrize("name", ["spread", "equal", "few values"])
@pytest.mark.parametrize("kind,lens,hkv,budget,first,last", [
    ("NHD", [13000, 10241, 100, 10240], 2, 700, 4, 20),
    ("q4", [10500, 12000, 10240, 11000], 5, 2500, 0, 300),
    ("HND", [10500, 11200, 3000, 10241, 14000], 8, 300, 5, 64), ("q4", [10400] * 7, 8, 1024, 0, 0),
    ("NHD", [70000], 1, 40000, 16, 100), ("q4", [400000], 1, 900, 0, 1),
    ("q4", [11000, 10800, 10801], 2, 10800, 4, 1000), ("HND", [20000], 1, 1, 0, 0)])
def test_eviction_of_few_long_contexts(ops, kind, lens, hkv, budget, first, last, name):
    """A sequence and head is cut by several CTAs: 8, 6, 3, 2 of them, with ties in all."""
    rng = np.random.default_rng(len(lens) + budget)

    def weights(n):
        if name == "spread":
            return spread_weights(rng, hkv)(n)
        return np.floor(rng.random((hkv, n)) * (3 if name == "few values" else 1)).astype(np.float32)
    run_evict(ops, rng, lens, budget, first, last, weights, 64, hkv, kind)


def test_evictions_side_by_side_and_captured(ops):
    """Few long sequences on two streams at once, and in a graph whose lengths change: the same bits as
    one after another."""
    rng = np.random.default_rng(17)
    pages, hkv, budget, lens = 200, 2, 700, [12000, 300, 6144, 6145, 700, 701, 0, 12800]
    start = [torch.from_numpy(rng.integers(0, 256, (pages, hkv, 4, 2304), dtype=np.uint8)).cuda(),
             raw(rng.random((pages, hkv, 64)).astype(np.float32))]
    t = ints([rng.permutation(pages)])

    def cut(state, n, out=None):
        return ops.evict_kvcache(state[0], state[1], n, t, budget, 4, 100, out=out)
    want = []
    for n in lens:
        state = [x.clone() for x in start]
        want.append((state, cut(state, ints([n])).tolist()))
    torch.cuda.synchronize()
    states, news = [[x.clone() for x in start] for _ in lens], [ints([-1]) for _ in lens]
    sizes = [ints([n]) for n in lens]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, n in enumerate(sizes):
        with torch.cuda.stream(streams[i % 2]):
            cut(states[i], n, news[i])
    torch.cuda.synchronize()
    state, n, new = [x.clone() for x in start], ints([lens[0]]), ints([-1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cut(state, n, new)
    for i, (ref, length) in enumerate(want):
        for x, y in zip(states[i], ref):
            assert torch.equal(x, y)
        for x, y in zip(state, start):
            x.copy_(y)
        n.fill_(lens[i])
        graph.replay()
        for x, y in zip(state, ref):
            assert torch.equal(x, y)
        assert news[i].tolist() == new.tolist() == length == [min(lens[i], budget)]


def test_bad_pages_of_few_long_contexts(ops):
    """Their tokens count as the smallest and do not move; others' do, whichever CTA has them."""
    pages, n, budget = 210, 13000, 1000
    table = np.arange(204, dtype=np.int32)
    table[[3, 150]] = -1, pages
    w = ops.new_attn_weights(pages, 64, 1)
    w[100:110] = 1.0                            # 640 tokens that stay, behind the budget
    cache = ops.new_kvcache_q4(pages, 64, 1)
    cache[100:110] = 7
    st = ops.new_status("cuda")
    assert ops.evict_kvcache(cache, w, ints([n]), ints([table]), budget, status=st).tolist() == [budget]
    assert int(st.item()) == 2
    # the first 360 of good pages stay, below place 424; the places of the fourth page take nothing
    want = torch.zeros(pages * 64)
    want[424:1000] = want[6400:7040] = 1
    assert torch.equal(w.cpu().flatten(), want)


def test_eviction_flags_bad_pages_and_long_contexts(ops):
    w = ops.new_attn_weights(6, 16, 1)
    cache = ops.new_kvcache_q4(6, 16, 1)
    for lens, t in (([60], [[0, 1, -1, 2]]), ([60], [[0, 1, 6, 2]]), ([1000], [[0, 1, 2, 3]])):
        st = ops.new_status("cuda")
        new = ops.evict_kvcache(cache, w, ints(lens), ints(t), 20, keep_last=4, status=st)
        assert int(st.item()) == 2 and new.tolist() == [20]
    assert not cache.any() and not w.any()


def test_eviction_of_pools_with_strided_pages(ops):
    """K and V as halves of one pool, as an engine may lay them out."""
    rng = np.random.default_rng(15)
    both = torch.randint(0, 2 ** 15, (8, 2, 64, 2, D), dtype=torch.int16, device="cuda")
    both = both.view(torch.bfloat16)
    dense = [both[:, i].clone() for i in range(2)]
    w = raw(rng.random((8, 2, 64)).astype(np.float32))
    w2 = w.clone()
    lens, t = ints([200, 130]), ints([[3, 1, 7, 0], [2, 5, 4, -1]])
    out = ints([0, 0])
    assert ops.evict_kvcache((both[:, 0], both[:, 1]), w, lens, t, 100, 2, 9, out=out) is out
    ops.evict_kvcache(tuple(dense), w2, lens, t, 100, 2, 9)
    assert torch.equal(w, w2) and out.tolist() == [100, 100]
    for i in range(2):
        assert torch.equal(both[:, i].view(torch.int16), dense[i].view(torch.int16))


# ------------------------------------------------------------------- the calls one after another
@pytest.mark.parametrize("packed", [True, False])
def test_a_cache_with_a_budget(ops, packed):
    """Prompts are stored, attended over as the cache has them, weighed by their last tokens, cut, and
    decoded from with a cut every few tokens: against the same steps in 64 bits.  The cut of each step
    is checked by itself (a weight next to the border may fall on either side of it in 64 bits)."""
    rng = np.random.default_rng(16)
    hq, hkv, page, group, budget, first, last, window = 8, 2, 64, 64, 96, 4, 16, 8
    prompts, steps = [300, 150, 60], 40
    cols, pages = 6, 20
    t = np.stack([rng.permutation(pages)[:18].reshape(3, 6)])[0].astype(np.int32)
    dt = ints(t)
    cache = ops.new_kvcache_q4(pages, page, hkv, group=group)
    kc, vc = (torch.zeros((pages, page, hkv, D), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    caches = cache if packed else (kc, vc)
    w = ops.new_attn_weights(pages, page, hkv)
    scale = D ** -0.5
    keep = (lambda x: S.values(x, group)) if packed else (lambda x: x.astype(np.float64))
    spread = 0.0
    # 64-bit state per sequence: rows and sums per head
    k64, v64, w64 = [], [], []
    st = ops.new_status("cuda")

    def store(k, v, slots):
        slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
        if packed:
            ops.store_kvcache_q4(dev(k), dev(v), cache, slots, status=st)
        else:
            ops.store_kvcache(dev(k), dev(v), kc, vc, slots, status=st)

    def attend(q, lens, cu, frm, tables=dt):
        kw = dict(cu_seqlens_q=cu, weights_from=frm, status=st)
        if packed:
            return ops.paged_decode_attn_q4(dev(q), cache, ints(lens), tables, scale, weights=w, **kw)
        return ops.paged_decode_attn_weights(dev(q), kc, vc, ints(lens), tables, scale, w, **kw)

    def compare(got, q, lens, seq_of, frm):
        """All heads hold rows of their own: one attention per KV head."""
        g = hq // hkv
        for h in range(hkv):
            kk = [x[h][:, None] for x in k64]
            vv = [x[h][:, None] for x in v64]
            out, mass, reach, sums = S.attention(q[:, h * g:(h + 1) * g], kk, vv, lens, seq_of, scale)
            part = got[:, h * g:(h + 1) * g]
            if packed:
                close_out(part, out, mass, reach, max(lens), spread)
            else:
                d = np.abs(host_f32(part) - out)
                assert (d <= np.abs(out) * 2.0 ** -8 +
                        mass * (2.0 ** -8 + weight_error(reach)[..., None])).all()
            for s in set(seq_of):
                w64[s][h][frm[s]:] = 0
                w64[s][h] += sums[s][0]
                n = len(w64[s][h])
                p = np.arange(n)
                dev_w = w.cpu().numpy()[t[s, p // page], h, p % page]
                np.testing.assert_allclose(dev_w, w64[s][h], rtol=weight_error(reach.max()) * steps,
                                           atol=1e-6)
                w64[s][h][:] = dev_w                  # and on from what the device has

    def cut(lens):
        new = ops.evict_kvcache(caches, w, ints(lens), dt, budget, first, last, status=st).tolist()
        for s, n in enumerate(lens):
            for h in range(hkv):
                moves = S.evict(n, w64[s][h], budget, first, last)
                for x in (k64, v64, w64):
                    old = x[s][h].copy()
                    for a, b in moves:
                        x[s][h][b] = old[a]
                    x[s][h] = x[s][h][:new[s]].copy()
        return new

    for s, n in enumerate(prompts):
        k, v = S.randn(rng, n, hkv, D), S.randn(rng, n, hkv, D)
        spread = max(spread, float(S.quantise(v, group)[1].max()))
        slots = S.slots_of(t[s], n, page)
        store(k, v, slots)
        k64.append([keep(k)[:, h].copy() for h in range(hkv)])
        v64.append([keep(v)[:, h].copy() for h in range(hkv)])
        w64.append([np.zeros(n) for _ in range(hkv)])
        if packed:
            # the prompt's own attention, over what the cache has of it
            rows = ops.load_kvcache_q4(cache, torch.tensor(slots, dtype=torch.int32, device="cuda"))
            cu = ints([0, n])
            q = S.randn(rng, n, hq, D)
            got = ops.prefill_attn(dev(q), *rows, cu, cu, n, scale)
            out, mass, _, _ = S.attention(q, [S.bf16(keep(k).astype(np.float32)).astype(np.float64)],
                                          [S.bf16(keep(v).astype(np.float32)).astype(np.float64)],
                                          np.arange(1, n + 1), [0] * n, scale)
            assert np.abs(host_f32(got) - out).max() < 2e-2
    q = S.randn(rng, 3 * window, hq, D)
    lens = [n - window + 1 + j for n in prompts for j in range(window)]
    got = attend(q, lens, ints(np.arange(4) * window), ints([0, 0, 0]))
    compare(got, q, lens, [s for s in range(3) for _ in range(window)], [0, 0, 0])
    lens = cut(prompts)
    assert lens == [96, 96, 60]
    for step in range(steps):
        k, v, q = S.randn(rng, 3, hkv, D), S.randn(rng, 3, hkv, D), S.randn(rng, 3, hq, D)
        spread = max(spread, float(S.quantise(v, group)[1].max()))
        store(k, v, [S.slots_of(t[s], lens[s] + 1, page)[-1] for s in range(3)])
        lens = [n + 1 for n in lens]
        for s in range(3):
            for h in range(hkv):
                k64[s][h] = np.concatenate([k64[s][h], keep(k)[s, h][None]])
                v64[s][h] = np.concatenate([v64[s][h], keep(v)[s, h][None]])
                w64[s][h] = np.concatenate([w64[s][h], [0.0]])
        compare(attend(q, lens, None, None), q, lens, [0, 1, 2], [n - 1 for n in lens])
        if step % 8 == 7:
            lens = cut(lens)
    assert max(lens) == budget and int(st.item()) == 0
