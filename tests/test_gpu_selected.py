"""Decode attention over selected blocks on the GPU: bounds of the keys of every block, the choice
of blocks, attention over them, and the three together."""
import numpy as np
import pytest
import torch

import selected_oracle as S
from gpu_util import dev, host_f32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from fastkernels_b200 import ops as _ops
    return _ops


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def close(got, out, mass):
    d = np.abs(host_f32(got).astype(np.float64) - out)
    over = d - S.tolerance(out, mass)
    assert (over <= 0).all(), (over.max(), np.unravel_index(over.argmax(), over.shape))


# ------------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("page,block,layout,hkv", [(16, 16, "HND", 8), (64, 64, "NHD", 3),
                                                   (256, 64, "NHD", 8), (64, 16, "HND", 1),
                                                   (256, 128, "HND", 2), (32, 32, "NHD", 5)])
def test_bounds_of_new_tokens(ops, page, block, layout, hkv):
    rng = np.random.default_rng(page + block + hkv)
    lens = [1, page, page + 1, 3 * page + block // 2 + 1, 0, 2 * page, block]
    new = [1, page, 1, 2 * page + 3, 0, 0, block]
    pages = 24
    kc = S.pool(rng, pages, page, hkv, layout)
    t = S.tables(rng, lens, page, pages)
    bounds = np.full((pages, hkv, page // block, 2, S.D), 7.0, np.float32)
    want = bounds.copy()
    for i, (n, f) in enumerate(zip(lens, new)):
        for b in range((n - f) // block, -(-n // block) if f else 0):
            pos = np.arange(b * block, min(n, (b + 1) * block))
            at = (t[i, b * block // page], slice(None), b * block % page // block)
            k = np.stack([S.rows(kc, t[i], pos, h, page, layout) for h in range(hkv)])
            want[at] = np.stack([k.min(1), k.max(1)], 1)
    st = ops.new_status("cuda")
    got = dev(bounds)
    cu = np.concatenate([[0], np.cumsum(new)])
    r = ops.key_bounds(dev(kc), got, ints(lens), ints(t), cu_new=ints(cu), max_new=max(new),
                       kv_layout=layout, status=st)
    assert r is got
    np.testing.assert_array_equal(host_f32(got), want)
    assert int(st.item()) == 0
    # one token each: the last block only
    one = dev(bounds)
    ops.key_bounds(dev(kc), one, ints(lens), ints(t), kv_layout=layout)
    for i, n in enumerate(lens):
        if n:
            b = (n - 1) // block
            page_of, sub = t[i, b * block // page], b * block % page // block
            k = np.stack([S.rows(kc, t[i], np.arange(b * block, n), h, page, layout)
                          for h in range(hkv)])
            np.testing.assert_array_equal(host_f32(one)[page_of, :, sub],
                                          np.stack([k.min(1), k.max(1)], 1))
    assert (host_f32(one) == 7.0).sum() > 0


def test_bounds_carry_infinities_and_no_numbers(ops):
    rng = np.random.default_rng(3)
    kc = S.pool(rng, 4, 64, 2, "NHD")
    kc[1, 5, 0, 7] = np.inf
    kc[1, 9, 1, 3] = np.nan
    kc[1, 40, 1, 2] = -np.inf
    kc[1, 50:, :, :] = np.nan                       # behind the last token: not read
    got = torch.zeros((4, 2, 1, 2, 128), dtype=torch.bfloat16, device="cuda")
    ops.key_bounds(dev(kc), got, ints([50]), ints([[1]]), cu_new=ints([0, 50]), max_new=50)
    want = np.stack([kc[1, :50].min(0), kc[1, :50].max(0)], 1)     # numpy carries NaN on
    np.testing.assert_array_equal(host_f32(got)[1, :, 0], want)
    assert np.isnan(want).sum() == 2


def test_bounds_bad_pages_and_lengths_are_flagged(ops):
    kc = dev(np.ones((4, 64, 2, 128), np.float32))
    b = torch.zeros((4, 2, 1, 2, 128), dtype=torch.bfloat16, device="cuda")
    for lens, t in (([10], [[4]]), ([10], [[-1]]), ([65], [[0]])):
        st = ops.new_status("cuda")
        ops.key_bounds(kc, b, ints(lens), ints(t), status=st)
        assert int(st.item()) == 2
    assert float(b[1:].abs().sum()) == 0            # the cut context's page 0 alone was written


@pytest.mark.parametrize("max_new", [1, 16, 17, 100])
def test_bounds_of_more_new_tokens_than_said(ops, max_new):
    """The newest max_new of a sequence that has more are taken, and that is flagged; the others of
    the batch have what they had."""
    rng = np.random.default_rng(4)
    lens, new, page, block = [300, 64, 130, 7], [300, 1, 101, 1], 64, 16
    kc = S.pool(rng, 12, page, 2, "NHD")
    t = S.tables(rng, lens, page, 12)
    want = np.full((12, 2, page // block, 2, S.D), 7.0, np.float32)
    for i, n in enumerate(lens):
        for b in range((n - min(new[i], max_new)) // block, -(-n // block)):
            pos = np.arange(b * block, min(n, (b + 1) * block))
            k = np.stack([S.rows(kc, t[i], pos, h, page, "NHD") for h in range(2)])
            want[t[i, b * block // page], :, b * block % page // block] = np.stack([k.min(1), k.max(1)], 1)
    got = torch.full(want.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    st = ops.new_status("cuda")
    ops.key_bounds(dev(kc), got, ints(lens), ints(t), cu_new=ints(np.cumsum([0, *new])), max_new=max_new,
                   status=st)
    np.testing.assert_array_equal(host_f32(got), want)
    assert int(st.item()) == 8
    st = ops.new_status("cuda")                     # as many as said: no flag
    ops.key_bounds(dev(kc), got, ints(lens), ints(t), cu_new=ints(np.cumsum([0, *new])), max_new=300,
                   status=st)
    assert int(st.item()) == 0


# ------------------------------------------------------------------------------- select
def select_case(seed, t, hq, hkv, page, block, longest, rows=None):
    rng = np.random.default_rng(seed)
    n_tables = t if rows is None else max(rows) + 1
    full = [longest] * n_tables
    pages = n_tables * -(-longest // page) + 1
    table = S.tables(rng, full, page, pages)
    off = rng.standard_normal((hkv, 1, 1, S.D)) * 0.5
    lo = off - np.abs(rng.standard_normal((pages, hkv, page // block, 1, S.D)))
    hi = off + np.abs(rng.standard_normal((pages, hkv, page // block, 1, S.D)))
    bounds = S.bf16(np.concatenate([np.minimum(lo, hi), np.maximum(lo, hi)], 3))
    q = S.bf16(rng.standard_normal((t, hq, S.D)))
    return rng, q, bounds, table


def check_select(ops, q, bounds, lens, table, block, count, first, last, rows=None, status=0):
    st = ops.new_status("cuda")
    got = ops.select_blocks(dev(q), dev(bounds), ints(lens), ints(table), block, count,
                            keep_first=first, keep_last=last,
                            table_rows=None if rows is None else ints(rows), status=st)
    of = table if rows is None else table[np.asarray(rows)]
    want = S.select(q, bounds, lens, of, block, count, first, last)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    assert int(st.item()) == status
    return want


@pytest.mark.parametrize("t,hq,hkv,page,block,longest,count,first,last", [
    (5, 8, 2, 64, 64, 3000, 8, 1, 1), (3, 32, 8, 256, 64, 6000, 16, 1, 2),
    (2, 16, 1, 16, 16, 4000, 64, 0, 1), (2, 5, 5, 32, 32, 2000, 7, 3, 4),
    (1, 10, 2, 256, 128, 9000, 9, 0, 9), (1, 12, 4, 16, 16, 70000, 128, 1, 1),
    (7, 7, 1, 64, 16, 900, 1, 0, 1), (2, 6, 2, 64, 32, 333, 11, 11, 0)])
def test_select_is_that_of_64_bits(ops, t, hq, hkv, page, block, longest, count, first, last):
    if last == 0:
        first, last = count - 1, 1
    rng, q, bounds, table = select_case(t * 100 + hq, t, hq, hkv, page, block, longest)
    lens = rng.integers(1, longest + 1, t)
    lens[0] = longest
    check_select(ops, q, bounds, lens, table, block, count, first, last)


@pytest.mark.parametrize("lens", [[0, 1, 64, 65, 128, 129, 192, 193]])
def test_select_short_contexts(ops, lens):
    """Contexts of no token, one, and around the number of blocks that are taken."""
    _, q, bounds, table = select_case(9, len(lens), 8, 2, 64, 64, 256)
    want = check_select(ops, q, bounds, lens, table, 64, 2, 0, 1)
    assert (want[0] == -1).all() and want[1, 0].tolist() == [0, -1]


def test_select_rows_of_a_portion(ops):
    """Tokens of two prompts that select with their prompt's table, out of order too."""
    rows = [1, 1, 1, 0, 0, 1, 0]
    rng, q, bounds, table = select_case(11, len(rows), 12, 4, 64, 32, 2000, rows)
    lens = [1990, 1991, 1992, 700, 701, 33, 2000]
    check_select(ops, q, bounds, lens, table, 32, 6, 1, 1, rows)


@pytest.mark.parametrize("hq,hkv,n", [(8, 8, 301), (32, 4, 640), (10, 10, 250), (16, 8, 300),
                                      (48, 3, 90), (35, 5, 70), (9, 1, 130), (12, 4, 64)])
def test_select_many_tokens(ops, hq, hkv, n):
    """As many tokens as let a warp choose for each; groups of tokens that end with a table."""
    rows = [0] * 37 + [1] * (n - 38) + [2]
    rng, q, bounds, table = select_case(hq + n, n, hq, hkv, 64, 16, 1500, rows)
    lens = rng.integers(1, 1501, n)
    q[5:9] = 0                                     # padded tokens
    check_select(ops, q, bounds, lens, table, 16, 9, 1, 2, rows)


@pytest.mark.parametrize("hq,hkv,n", [(8, 8, 301), (4, 2, 90), (10, 2, 130), (16, 1, 70)])
def test_select_scores_every_token_of_a_run(ops, hq, hkv, n):
    """The scores that the choice starts from, [tokens, KV heads, blocks up to a multiple of four] at
    the workspace's start as fp32 in the order of whole numbers: off by 2^-18 sum |q| max |bound| at
    most, whatever the number of query heads of a KV head."""
    rows = [0] * 37 + [1] * (n - 38) + [2]
    rng, q, bounds, table = select_case(hq + n, n, hq, hkv, 64, 16, 1500, rows)
    cols, per, g = table.shape[1], 4, hq // hkv
    ws = torch.zeros(ops.select_blocks_workspace_bytes(n, hq, hkv, 64, 16, cols), dtype=torch.uint8,
                     device="cuda")
    ops.select_blocks(dev(q), dev(bounds), ints([1500] * n), ints(table), 16, 9, keep_first=1,
                      keep_last=2, table_rows=ints(rows), workspace=ws)
    keys = ws.view(torch.int32)[:n * hkv * cols * per].view(n, hkv, cols * per).cpu().numpy()
    keys = keys.view(np.uint32)[:, :, :-(-1500 // 16) - 3]            # blocks 1 .. 91 of 94
    got = np.where(keys >> 31, keys & 0x7fffffff, ~keys).astype(np.uint32).view(np.float32)
    b = np.arange(1, 1 + got.shape[2])
    for i in range(n):
        of = bounds[table[rows[i], b // per], :, b % per].astype(np.float64)       # [blocks, hkv, 2, D]
        a = q[i].reshape(hkv, g, 1, S.D).astype(np.float64)
        want = np.maximum(a * of[:, :, 0].swapaxes(0, 1)[:, None],
                          a * of[:, :, 1].swapaxes(0, 1)[:, None]).sum(-1).max(1)
        reach = np.abs(a).sum(-1).max() * np.abs(of).max()
        assert (np.abs(got[i] - want) <= 2.0 ** -18 * reach).all(), i


@pytest.mark.parametrize("what", ["few values", "one block", "zero query", "equal blocks"])
def test_select_takes_the_first_of_equals(ops, what):
    rng, q, bounds, table = select_case(13, 4, 8, 2, 64, 64, 64 * 700)
    if what == "few values":                       # sums of small whole numbers: many equal scores
        bounds = np.sort(rng.integers(-1, 2, bounds.shape).astype(np.float32), 3)
        q = rng.integers(-1, 2, q.shape).astype(np.float32)
    elif what == "one block":
        bounds[:] = bounds[:1, :, :1]
    elif what == "zero query":
        q[:] = 0
        q[1, 3, 5] = -0.0
    else:                                          # every block twice
        bounds[table[:, 1:700:2]] = bounds[table[:, 0:699:2]]
    check_select(ops, q, bounds, [64 * 700, 64 * 699 + 1, 64 * 40, 64 * 333 + 5], table, 64, 33, 1,
                 2)


def test_select_by_differences_that_fp32_loses(ops):
    """Blocks whose scores differ behind the 24th bit."""
    rng, q, bounds, table = select_case(17, 2, 4, 2, 64, 64, 64 * 300)
    q[:] = 1.0
    bounds[:] = 0
    bounds[..., 1, 0] = 2.0 ** 20                  # a large part that all share
    bounds[..., 1, 1:8] = S.bf16(rng.standard_normal((*bounds.shape[:3], 7)) * 2.0 ** -10)
    bounds[..., 0, :] = np.minimum(bounds[..., 1, :], 0)
    check_select(ops, q, bounds, [64 * 300, 64 * 211], table, 64, 20, 0, 1)


def test_select_with_infinities_and_no_numbers(ops):
    rng, q, bounds, table = select_case(19, 3, 4, 2, 64, 64, 64 * 200)
    bounds[table[0, 10], 0, 0, 1, 3] = np.inf
    bounds[table[0, 20], 0, 0, 0, 4] = -np.inf
    bounds[table[1, 30], 1, 0, :, 5] = np.nan
    bounds[table[1, 31], 1, 0, 1, 6] = 3e38
    q[1, 2:, 6] = 100.0                            # the product is past fp32's range
    q[2, 0, 9] = 0.0
    bounds[table[2, 40], 0, 0, 1, 9] = np.inf      # zero times infinity is no number
    check_select(ops, q, bounds, [64 * 200] * 3, table, 64, 12, 1, 1)


def test_select_bad_pages_and_rows(ops):
    rng, q, bounds, table = select_case(23, 2, 4, 2, 64, 64, 64 * 100)
    table[0, 50] = -1
    check_select(ops, q, bounds, [6400, 6400], table, 64, 10, 1, 1, status=2)
    # with no other blocks left it is taken after all
    check_select(ops, q, bounds, [64 * 60, 64 * 60], table, 64, 59, 1, 1, status=2)
    st = ops.new_status("cuda")
    got = ops.select_blocks(dev(q), dev(bounds), ints([6400, 99999]), ints(table), 64, 4,
                            table_rows=ints([2, 1]), status=st)
    assert int(st.item()) == 2
    assert (got[0] == -1).all() and int(got[1, 0, -1]) == table.shape[1] - 1


# ------------------------------------------------------------------------------- attend
def attend_case(seed, lens, hq, hkv, page, block, layout, count, rows=None, wild=False):
    rng = np.random.default_rng(seed)
    t = len(lens)
    n_tables = t if rows is None else max(rows) + 1
    seq = [max([n for i, n in enumerate(lens) if (i if rows is None else rows[i]) == s] + [0])
           for s in range(n_tables)]
    pages = sum(-(-n // page) for n in seq) + 2
    table = S.tables(rng, seq, page, pages)
    kc, vc = (S.pool(rng, pages, page, hkv, layout) for _ in range(2))
    # what is behind a sequence's last token, and in nobody's pages, must not matter
    live = np.zeros((pages, page), bool)
    for s, n in enumerate(seq):
        for pos in range(n):
            live[table[s, pos // page], pos % page] = True
    for c in (kc, vc):
        (c if layout == "NHD" else c.swapaxes(1, 2))[~live] = np.nan
    sel = np.full((t, hkv, count), -1, np.int32)
    for i, n in enumerate(lens):
        blocks = -(-n // block)
        for h in range(hkv):
            if wild:       # any order, gaps, twice, past the end
                sel[i, h] = rng.integers(-2, blocks + 2, count)
            elif blocks:
                k = min(count, blocks)
                some = np.sort(rng.choice(blocks - 1, k - 1, replace=False)) if k > 1 else []
                sel[i, h, :k] = [*some, blocks - 1]
    q = S.bf16(rng.standard_normal((t, hq, S.D)))
    return q, kc, vc, table, sel


def attend_oracle(q, kc, vc, lens, table, sel, page, block, layout, hkv, rows):
    of = table if rows is None else table[np.asarray(rows)]

    def positions(i, h):
        return [x for b in sel[i, h] if b >= 0
                for x in range(b * block, min(lens[i], (b + 1) * block))]
    return S.over_positions(q, kc, vc, lens, of, page, layout, hkv, positions)


@pytest.mark.parametrize("page,block,layout,hq,hkv,lens,count", [
    (64, 64, "NHD", 8, 2, [1, 64, 65, 700, 1500], 5), (16, 16, "HND", 10, 2, [5, 300, 1200], 40),
    (256, 64, "NHD", 16, 1, [2000, 3, 257], 9), (256, 16, "NHD", 6, 6, [400, 17], 11),
    (64, 32, "HND", 14, 2, [900, 31, 33], 13), (32, 32, "NHD", 4, 4, [1, 2, 999], 16),
    (256, 256, "HND", 8, 1, [3000, 255], 4), (16, 16, "NHD", 16, 1, [2100], 128),
    (64, 64, "HND", 9, 3, [0, 40, 128, 0], 3), (256, 128, "NHD", 2, 2, [1100, 130, 127], 7),
    (192, 64, "NHD", 4, 2, [600, 193], 6), (16, 16, "NHD", 4, 2, [1, 16, 17, 900], 1),
    (512, 192 + 64, "NHD", 4, 1, [1500, 512], 3), (384, 192, "HND", 4, 2, [1500, 384, 191], 5)])
@pytest.mark.parametrize("wild", [False, True])
def test_attention_over_selected_blocks(ops, page, block, layout, hq, hkv, lens, count, wild):
    q, kc, vc, table, sel = attend_case(page + hq + count, lens, hq, hkv, page, block, layout,
                                        count, wild=wild)
    st = ops.new_status("cuda")
    got = ops.selected_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(sel), block,
                            S.SCALE, kv_layout=layout, status=st)
    close(got, *attend_oracle(q, kc, vc, lens, table, sel, page, block, layout, hkv, None))
    assert int(st.item()) == 0


def test_selected_many_tokens_of_prompts(ops):
    rows = [i % 3 for i in range(60)]
    lens = [500 + 13 * i for i in range(60)]
    q, kc, vc, table, sel = attend_case(5, lens, 8, 4, 64, 16, "NHD", 24, rows)
    got = ops.selected_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(sel), 16,
                            S.SCALE, table_rows=ints(rows))
    close(got, *attend_oracle(q, kc, vc, lens, table, sel, 64, 16, "NHD", 4, rows))


def test_selected_one_expanded_table_and_strided_rows(ops):
    """Tokens of one prompt on one row of a table that is expanded, q inside packed rows, results
    inside wider rows that stay as they are around them."""
    lens = [200, 201, 202, 203]
    rows = [0, 0, 0, 0]
    q, kc, vc, table, sel = attend_case(6, lens, 8, 2, 64, 64, "NHD", 3, rows)
    packed = torch.zeros((4, 12 * 128), dtype=torch.bfloat16, device="cuda")
    packed[:, :1024] = dev(q).view(4, 1024)
    out = torch.full((6, 10, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.selected_attn(packed[:, :1024].view(4, 8, 128), dev(kc), dev(vc), ints(lens),
                      ints(table).expand(4, -1), ints(sel), 64, S.SCALE, out=out[:4, :8])
    close(out[:4, :8], *attend_oracle(q, kc, vc, lens, table, sel, 64, 64, "NHD", 2, rows))
    assert (out[4:] == 3.0).all() and (out[:, 8:] == 3.0).all()


def test_selected_bad_pages_are_left_out(ops):
    lens = [640, 640]
    q, kc, vc, table, sel = attend_case(7, lens, 4, 2, 64, 64, "NHD", 10)
    broken = table.copy()
    broken[0, 4], broken[1, 0] = 10 ** 6, -5
    st = ops.new_status("cuda")
    got = ops.selected_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(broken), ints(sel), 64,
                            S.SCALE, status=st)
    assert int(st.item()) == 2
    sel[0][sel[0] == 4] = -1
    sel[1][sel[1] == 0] = -1
    close(got, *attend_oracle(q, kc, vc, lens, table, sel, 64, 64, "NHD", 2, None))


def test_selected_keys_that_are_no_numbers_are_seen(ops):
    lens = [2000, 640]
    q, kc, vc, table, sel = attend_case(17, lens, 4, 2, 64, 64, "NHD", 20)
    good = host_f32(ops.selected_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(sel), 64,
                                      S.SCALE))
    b = int(sel[0, 1, 5])
    kc[table[0, b], 9, 1] = np.nan
    got = host_f32(ops.selected_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(sel), 64,
                                     S.SCALE))
    assert np.isnan(got[0, 2:]).all() and (got[0, :2] == good[0, :2]).all()
    assert (got[1] == good[1]).all()


def test_selected_large_scores(ops):
    """Scores of some hundreds: the largest key of a row alone counts, whichever block holds it."""
    q, kc, vc, table, sel = attend_case(8, [1000, 777], 8, 2, 64, 64, "NHD", 8)
    q = S.bf16(q * 60)
    got = ops.selected_attn(dev(q), dev(kc), dev(vc), ints([1000, 777]), ints(table), ints(sel), 64,
                            S.SCALE)
    out, mass = attend_oracle(q, kc, vc, [1000, 777], table, sel, 64, 64, "NHD", 2, None)
    # scores up to 2^9, each off by at most 2^-17 of the sum of |q k| (below 2^12 * 2^-3): 2^-8
    d = np.abs(host_f32(got) - out)
    assert (d <= S.tolerance(out, mass) + 2 * 2.0 ** -8 * mass).all()


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("page,block,layout,hq,hkv", [(64, 64, "NHD", 8, 2), (16, 16, "HND", 10, 2),
                                                      (256, 32, "NHD", 4, 4)])
def test_steps_with_sparse_attention(ops, page, block, layout, hq, hkv):
    """A prompt is stored, then single tokens: store, bounds, choice and attention of each step."""
    rng = np.random.default_rng(page)
    lens, steps, count = [block * 9 + 3, block * 4, 1], block + 3, 5
    pages = sum(-(-(n + steps) // page) for n in lens) + 1
    table = S.tables(rng, [n + steps for n in lens], page, pages)
    kc, vc = (S.pool(rng, pages, page, hkv, layout) for _ in range(2))
    gk, gv = dev(kc), dev(vc)
    bounds = ops.new_key_bounds(gk, block, layout)
    cu = np.concatenate([[0], np.cumsum(lens)])
    ops.key_bounds(gk, bounds, ints(lens), ints(table), cu_new=ints(cu), max_new=max(lens),
                   kv_layout=layout)
    store = ops.store_kvcache if layout == "NHD" else ops.store_kvcache_hnd
    st = ops.new_status("cuda")
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        new_k, new_v = (S.bf16(rng.standard_normal((3, hkv, S.D)) * 0.7) for _ in range(2))
        slots = []
        for i, n in enumerate(lens):
            p, o = table[i, (n - 1) // page], (n - 1) % page
            slots.append(p * page + o)
            for c, x in ((kc, new_k), (vc, new_v)):
                (c[p, o] if layout == "NHD" else c[p, :, o])[...] = x[i]
        q = S.bf16(rng.standard_normal((3, hq, S.D)))
        store(dev(new_k), dev(new_v), gk, gv, ints(slots), status=st)
        ops.key_bounds(gk, bounds, ints(lens), ints(table), kv_layout=layout, status=st)
        sel = ops.select_blocks(dev(q), bounds, ints(lens), ints(table), block, count, status=st)
        got = ops.selected_attn(dev(q), gk, gv, ints(lens), ints(table), sel, block, S.SCALE,
                                kv_layout=layout, status=st)
        want = S.select(q, S.bounds_of(kc, page, block, layout), lens, table, block, count, 1, 1)
        np.testing.assert_array_equal(sel.cpu().numpy(), want)
        close(got, *attend_oracle(q, kc, vc, lens, table, want, page, block, layout, hkv, None))
    assert int(st.item()) == 0


def test_all_blocks_selected_is_ordinary_attention(ops):
    rng = np.random.default_rng(4)
    lens = [700, 64, 1, 333]
    table = S.tables(rng, lens, 64, 40)
    kc, vc = (dev(S.pool(rng, 40, 64, 2, "NHD")) for _ in range(2))
    q = dev(S.bf16(rng.standard_normal((4, 8, S.D))))
    bounds = ops.new_key_bounds(kc, 64)
    sel = ops.select_blocks(q, bounds, ints(lens), ints(table), 64, 11)
    got = ops.selected_attn(q, kc, vc, ints(lens), ints(table), sel, 64, S.SCALE)
    ws = torch.empty(ops.attn_workspace_bytes(4, 8, 128, 16), dtype=torch.uint8, device="cuda")
    want = ops.paged_decode_attn(q, kc, vc, ints(lens), ints(table), S.SCALE, ws, 16)
    # both within their tolerance of the same values, |v| below 3
    assert (got.float() - want.float()).abs().max() <= 2 * (2.0 ** -8 * 3 + 2.0 ** -8 * 3)


def test_chain_in_a_graph_and_on_another_stream(ops):
    """Captured once with a workspace of its own, replayed with other inputs in the same buffers, and
    run eagerly on a side stream meanwhile."""
    rng = np.random.default_rng(21)
    lens = np.array([900, 2000, 40], np.int32)
    table = S.tables(rng, [2100] * 3, 64, 120)
    kc, vc = (S.pool(rng, 120, 64, 2, "NHD") for _ in range(2))
    gk, gv, gt, gl = dev(kc), dev(vc), ints(table), ints(lens)
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device="cuda")
    bounds = dev(S.bounds_of(kc, 64, 64, "NHD"))
    n = ops.selected_attn_workspace_bytes(3, 8, 2, 128, 6, 64)

    def chain(ws):
        sel = ops.select_blocks(q, bounds, gl, gt, 64, 6)
        return sel, ops.selected_attn(q, gk, gv, gl, gt, sel, 64, S.SCALE, workspace=ws)
    spaces = [torch.empty(max(n, 1), dtype=torch.uint8, device="cuda") for _ in range(2)]
    chain(spaces[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sel, out = chain(spaces[0])
    side = torch.cuda.Stream()
    for _ in range(3):
        a = S.bf16(rng.standard_normal((3, 8, S.D)))
        lens = rng.integers(1, 2100, 3).astype(np.int32)
        q.copy_(dev(a))
        gl.copy_(ints(lens))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sel2, out2 = chain(spaces[1])
        g.replay()
        torch.cuda.synchronize()
        want = S.select(a, S.bounds_of(kc, 64, 64, "NHD"), lens, table, 64, 6, 1, 1)
        np.testing.assert_array_equal(sel.cpu().numpy(), want)
        np.testing.assert_array_equal(sel2.cpu().numpy(), want)
        assert torch.equal(out, out2)
        close(out, *attend_oracle(a, kc, vc, lens, table, want, 64, 64, "NHD", 2, None))


def test_launches_are_counted(ops):
    """Two kernels choose blocks; attention over them is one, and a join where tokens are few."""
    from fastkernels_b200 import _lib
    rng, q, bounds, table = select_case(17, 3, 8, 2, 64, 64, 3000)
    lens, kc = ints([3000, 700, 1]), dev(S.pool(rng, len(bounds), 64, 2, "NHD"))

    def launches(f):
        before = _lib.lib.fk_launch_count()
        return f(), _lib.lib.fk_launch_count() - before
    sel, n = launches(lambda: ops.select_blocks(dev(q), dev(bounds), lens, ints(table), 64, 16))
    assert n == 2
    _, n = launches(lambda: ops.select_blocks(dev(q), dev(bounds), lens, ints(table), 64, 16,
                                              table_rows=ints([0, 1, 2])))
    assert n == 2
    for count, joined in ((16, True), (2, False)):      # 8 tiles of 128 keys a token and head; one
        part = sel[:, :, :count].contiguous()
        assert (ops.selected_attn_workspace_bytes(3, 8, 2, S.D, count, 64) > 0) is joined
        _, n = launches(lambda: ops.selected_attn(dev(q), kc, kc, lens, ints(table), part, 64, S.SCALE))
        assert n == 1 + joined
    _, n = launches(lambda: ops.key_bounds(kc, dev(bounds), lens, ints(table)))
    assert n == 1


def test_nothing_to_do(ops):
    kc = dev(np.ones((2, 64, 2, 128), np.float32))
    q = torch.empty((0, 4, 128), dtype=torch.bfloat16, device="cuda")
    none, t = ints([]), ints(np.zeros((0, 3)))
    b = ops.new_key_bounds(kc, 64)
    ops.key_bounds(kc, b, none, t)
    sel = ops.select_blocks(q, b, none, t, 64, 3)
    assert sel.shape == (0, 2, 3)
    assert ops.selected_attn(q, kc, kc, none, t, sel, 64, 0.1).shape == (0, 4, 128)
