"""Decode attention of batches whose sequences begin with the same pages, on the GPU."""
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


def widened(table, page):
    """With room for more than 2048 tokens, whose calls are not one launch without a schedule."""
    extra = max(0, 2048 // page + 1 - table.shape[1])
    return np.concatenate([table, np.full((len(table), extra), -1, np.int32)], 1)


def build(seed, groups, page, layout, hq, hkv, extra_rows=(), wide=True):
    """groups: (prefix tokens, [tokens behind it of each row]).  Rows of a group share the whole
    pages of its prefix.  extra_rows: lengths of rows behind the last group.  What is behind
    a row's last token, and in nobody's pages, is no number."""
    rng = np.random.default_rng(seed)
    lens, starts, prefix = [], [0], []
    plan = []                                     # (shared pages, own pages) of each row
    for p, own in groups:
        prefix.append(p)
        starts.append(starts[-1] + len(own))
        whole = p // page
        for s in own:
            n = max(0, p + s)
            lens.append(n)
            plan.append((whole, max(0, -(-n // page) - whole)))
    for n in extra_rows:
        lens.append(n)
        plan.append((0, -(-n // page)))
    total = sum(p // page for p, _ in groups) + sum(o for _, o in plan) + 2
    order = rng.permutation(total).astype(np.int32)
    cols = max(s + o for s, o in plan) + 1
    table = np.full((len(lens), cols), -1, np.int32)
    at, row = 0, 0
    live = np.zeros((total, page), bool)
    for p, own in groups:
        common = order[at:at + p // page]
        at += len(common)
        live[common] = True
        for _ in own:
            table[row, :len(common)] = common
            row += 1
    for i, (shared, own) in enumerate(plan):
        table[i, shared:shared + own] = order[at:at + own]
        at += own
        for pos in range(shared * page, lens[i]):
            live[table[i, pos // page], pos % page] = True
    kc, vc = (S.pool(rng, total, page, hkv, layout) for _ in range(2))
    for c in (kc, vc):
        (c if layout == "NHD" else c.swapaxes(1, 2))[~live] = np.nan
    q = S.bf16(rng.standard_normal((len(lens), hq, S.D)))
    if wide:
        table = widened(table, page)
    return q, kc, vc, np.array(lens, np.int32), table, starts, prefix


def run(ops, case, layout, status=None, **kw):
    q, kc, vc, lens, table, starts, prefix = case
    return ops.shared_prefix_attn(dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(starts),
                                  ints(prefix), S.SCALE, kv_layout=layout, status=status, **kw)


def check(ops, case, page, layout, hkv, **kw):
    q, kc, vc, lens, table, _, _ = case
    st = ops.new_status("cuda")
    got = run(ops, case, layout, st, **kw)
    out, mass = S.over_positions(q, kc, vc, lens, table, page, layout, hkv,
                                 lambda i, h: range(lens[i]))
    d = np.abs(host_f32(got).astype(np.float64) - out)
    over = d - S.tolerance(out, mass)
    assert (over <= 0).all(), (over.max(), np.unravel_index(over.argmax(), over.shape))
    assert int(st.item()) == 0
    return got


@pytest.mark.parametrize("page,layout,hq,hkv", [(64, "NHD", 8, 2), (16, "HND", 16, 2),
                                                (256, "NHD", 4, 4), (32, "NHD", 10, 2),
                                                (64, "HND", 16, 1), (16, "NHD", 7, 1),
                                                (192, "NHD", 6, 2)])
def test_groups_of_all_kinds(ops, page, layout, hq, hkv):
    groups = [(4 * page, [1, 5, page, page + 1]),        # ordinary
              (page, [3]),                               # alone
              (0, [7, 300]),                             # nothing in common
              (9 * page, [0, 1, 2 * page + 3]),          # a row that ends with the common part
              (5 * page, [-page - 3, 2, -5 * page, 1]),  # rows that end inside it, one empty
              (2 * page + 5, [20, 30]),                  # ends inside a page
              (page - 1, [page, 9])]                     # not one whole page
    for wide in (True, False):
        check(ops, build(page + hq, groups, page, layout, hq, hkv, extra_rows=[70, 0, 1], wide=wide),
              page, layout, hkv)


@pytest.mark.parametrize("g", [1, 3, 4, 16])
def test_small_calls_are_one_launch(ops, g):
    from fastkernels_b200 import _lib
    case = build(40 + g, [(512, [1, 200, 64]), (256, [9, -1, -256])], 64, "HND", 2 * g, 2,
                 extra_rows=[5], wide=False)
    before = _lib.lib.fk_launch_count()
    check(ops, case, 64, "HND", 2)
    assert _lib.lib.fk_launch_count() == before + 1


@pytest.mark.parametrize("rows,hq,hkv", [(2, 2, 2), (33, 4, 1), (32, 8, 2), (40, 16, 1),
                                         (130, 2, 2), (65, 12, 3), (26, 10, 2), (129, 2, 1),
                                         (17, 32, 2)])
def test_rows_of_a_group_over_tiles(ops, rows, hq, hkv):
    """Numbers of rows times query heads around and past the tiles of a product."""
    case = build(rows + hq, [(320, [i % 70 for i in range(rows)])], 64, "NHD", hq, hkv)
    check(ops, case, 64, "NHD", hkv)


@pytest.mark.parametrize("prefix", [16, 112, 128, 144, 2048, 12304])
def test_lengths_of_the_common_part(ops, prefix):
    case = build(prefix, [(prefix, [5, 300, 1]), (prefix + 160, [1, 2])], 16, "HND", 4, 2)
    check(ops, case, 16, "HND", 2)


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("short,bad", [(100, np.nan), (700, np.inf), (1023, np.nan)])
def test_what_a_short_row_does_not_see(ops, short, bad, wide):
    """A row that ends inside the common part, with keys or values behind its end that are no numbers or
    infinite: they are the others' results alone."""
    case = build(31, [(1024, [50, 60, short - 1024, 700, -1024])], 64, "NHD", 16, 4, wide=wide)
    q, kc, vc, lens, table, starts, prefix = case
    kc, vc = np.nan_to_num(kc), np.nan_to_num(vc)
    p, o = table[0, short // 64], short % 64              # the first position behind its end
    vc[p, o, 1] = bad
    kc[p, o, 2] = bad
    case = (q, kc, vc, lens, table, starts, prefix)
    got = host_f32(run(ops, case, "NHD", max_splits=4))
    assert lens.tolist() == [1074, 1084, short, 1724, 0]
    want, mass = S.over_positions(q[2:3], kc, vc, lens[2:3], table[2:3], 64, "NHD", 4,
                                  lambda i, h: range(short))
    assert (np.abs(got[2:3] - want) <= S.tolerance(want, mass)).all()
    assert (got[4] == 0).all()
    assert not np.isfinite(got[:2, 4:8]).any()            # the heads of the value's KV head
    assert np.isfinite(got[:, :4]).all() and np.isfinite(got[:, 12:]).all()
    if np.isnan(bad):                                     # a key's: every score of its KV head's rows
        assert np.isnan(got[:2, 8:12]).all()


@pytest.mark.parametrize("wide", [True, False])
def test_what_is_no_number_is_seen(ops, wide):
    """Keys, values and queries that are no numbers, in the common part and in a row's own: the rows that see
    them have no numbers, the others what they had."""
    case = build(35, [(640, [50, 600, 0]), (64, [700, 3])], 64, "NHD", 8, 4, wide=wide)
    q, kc, vc, lens, table, starts, prefix = case
    good = host_f32(run(ops, case, "NHD"))

    def changed(**kw):
        a, b, c = (x.copy() for x in (q, kc, vc))
        if "key" in kw:
            row, pos, head = kw["key"]
            b[table[row, pos // 64], pos % 64, head] = np.nan
        if "value" in kw:
            row, pos, head = kw["value"]
            c[table[row, pos // 64], pos % 64, head, 7] = np.nan
        if "query" in kw:
            a[kw["query"]] = np.nan
        got = host_f32(run(ops, (a, b, c, lens, table, starts, prefix), "NHD"))
        return got, got != good
    got, other = changed(key=(0, 300, 1))
    assert np.isnan(got[:3, 2:4]).all() and not other[:, :2].any() and not other[3:].any()
    got, other = changed(key=(1, 700, 2))
    assert np.isnan(got[1, 4:6]).all() and other.sum() == 2 * 128
    got, other = changed(value=(2, 10, 3))
    assert np.isnan(got[:3, 6:, 7]).all() and other.sum() == 3 * 2
    got, other = changed(query=2)                         # a row that the common part alone answers
    assert np.isnan(got[2]).all() and not other[[0, 1, 3, 4]].any()


def test_pages_far_behind(ops):
    """Pages more than 2^32 bytes into a pool."""
    pages = 34000
    pool = torch.zeros((pages, 64, 8, 128), dtype=torch.bfloat16, device="cuda")
    assert pool.numel() * 2 > 2 ** 32
    rng = np.random.default_rng(3)
    small = S.pool(rng, 40, 64, 8, "NHD")
    pool[-40:] = dev(small)
    case = build(33, [(1024, [70, 300, 5])], 64, "NHD", 16, 8)
    q, _, _, lens, table, starts, prefix = case
    far = np.where(table >= 0, table + pages - 40, -1).astype(np.int32)
    assert table.max() < 40
    args = [ints(lens), ints(starts), ints(prefix)]
    near = ops.shared_prefix_attn(dev(q), dev(small), dev(small), args[0], ints(table), *args[1:],
                                  S.SCALE)
    got = ops.shared_prefix_attn(dev(q), pool, pool, args[0], ints(far), *args[1:], S.SCALE)
    assert torch.equal(got, near)
    for block in (16, 64):
        sel = ops.select_blocks(dev(q), dev(S.bounds_of(small, 64, block, "NHD")), args[0], ints(table),
                                block, 9)
        b = ops.new_key_bounds(pool, block)
        ops.key_bounds(pool, b, args[0], ints(far), cu_new=ints(np.cumsum([0, *lens])),
                       max_new=int(max(lens)))
        assert torch.equal(ops.select_blocks(dev(q), b, args[0], ints(far), block, 9), sel)
        near, got = (ops.selected_attn(dev(q), c, c, args[0], ints(t), sel, block, S.SCALE)
                     for c, t in ((dev(small), table), (pool, far)))
        assert torch.equal(got, near)


def test_contexts_near_two_to_31(ops):
    """Contexts whose ends leave 32 bits no room are cut at 2^30 tokens, and that is flagged.  A table
    lists one page again and again, so every whole number of them has one result."""
    page, cols, splits = 1 << 16, 1 << 15, 64
    rng = np.random.default_rng(6)
    kc = S.bf16(rng.standard_normal((1, page, 1, S.D), dtype=np.float32) * 0.25)
    vc = S.bf16(np.linspace(-2, 2, S.D) + 0.25 * rng.standard_normal((1, page, 1, S.D)))
    q = S.bf16(rng.standard_normal((4, 2, S.D)))
    lens = [2 ** 31 - 1, 2 ** 31 - 700, 2 ** 31 - 1, 300]
    table = torch.zeros((1, cols), dtype=torch.int32, device="cuda").expand(4, cols)
    st = ops.new_status("cuda")
    got = ops.shared_prefix_attn(dev(q), dev(kc), dev(vc), ints(lens), table, ints([0, 2]),
                                 ints([2 ** 31 - 1]), S.SCALE, max_splits=splits, status=st)
    assert int(st.item()) == 2
    out, mass = S.over_positions(q, kc, vc, lens, np.zeros((4, 1), np.int32), page, "NHD", 1,
                                 lambda i, h: range(min(lens[i], page)))
    d = np.abs(host_f32(got) - out)
    # a CTA adds up 2^30 / 128 / 148 steps of 8 products into one sum, a split 2^23 / 64 of one a warp
    steps = max(2 ** 23 / 148 * 8, 2 ** 23 / 64)
    assert (d <= S.tolerance(out, mass) + 2 * steps * 2.0 ** -23 * mass).all(), d.max()
    assert (d[3] <= S.tolerance(out, mass)[3]).all()


def test_many_groups(ops):
    rng = np.random.default_rng(2)
    groups = [(int(rng.integers(0, 9)) * 16, [int(x) for x in rng.integers(1, 60, rng.integers(1, 5))])
              for _ in range(90)]
    check(ops, build(1, groups, 16, "NHD", 4, 2), 16, "NHD", 2)


def test_no_groups_and_one_row(ops):
    for wide in (True, False):
        check(ops, build(1, [], 64, "NHD", 8, 2, extra_rows=[1, 700, 64, 0], wide=wide), 64, "NHD", 2)
        check(ops, build(2, [(640, [11])], 64, "NHD", 8, 2, wide=wide), 64, "NHD", 2)
        check(ops, build(3, [(1280, [1, 1])], 64, "NHD", 8, 2, wide=wide), 64, "NHD", 2, max_splits=1)


def test_large_scores(ops):
    """Scores of some hundreds, the largest in either part."""
    case = build(8, [(1024, [200, 300, 1]), (64, [700, 3])], 64, "NHD", 8, 2)
    q, kc, vc, lens, table = case[:5]
    q[:] = S.bf16(q * 60)
    got = run(ops, case, "NHD")
    out, mass = S.over_positions(q, kc, vc, lens, table, 64, "NHD", 2, lambda i, h: range(lens[i]))
    # scores off by at most 2^-17 of the sum of |q k| (below 2^9): 2^-8
    d = np.abs(host_f32(got) - out)
    assert (d <= S.tolerance(out, mass) + 2 * 2.0 ** -8 * mass).all()


@pytest.mark.parametrize("own", [0, 1, 300])
@pytest.mark.parametrize("rise", [0, 1, 16])
def test_scores_of_many_thousands(ops, own, rise):
    """Logits of 10^4 to 10^5, of either sign, that differ by some units from key to key, and with
    `rise` by tens or hundreds more from one run of 100 keys to the next.  Queries and keys are
    whole numbers, so that scores are exact in fp32."""
    rng = np.random.default_rng(50 + own)
    case = build(13, [(1024, [own] * 20), (2048, [own, own + 60])], 64, "NHD", 8, 2)
    q, kc, vc, lens, table, starts, prefix = case
    q[:] = rng.integers(-3, 4, q.shape)
    q[..., :64] = rng.integers(7, 70, (*q.shape[:2], 1)) * rng.choice([-1, 1], (*q.shape[:2], 1))
    kc[:] = np.where(np.isnan(kc), kc, rng.integers(-3, 4, kc.shape))
    kc[..., :63] = np.where(np.isnan(kc[..., :63]), np.nan, 255.0)
    kc[..., 63] = 0.0
    for i, n in enumerate(lens):
        pos = np.arange(n)
        kc[table[i, pos // 64], pos % 64, :, 63] = (pos // 100 * rise % 256)[:, None]
    assert np.array_equal(S.bf16(q), q) and np.array_equal(S.bf16(kc), kc, equal_nan=True)
    case = (q, kc, vc, lens, table, starts, prefix)
    st = ops.new_status("cuda")
    got = run(ops, case, "NHD", st)
    out, mass = S.over_positions(q, kc, vc, lens, table, 64, "NHD", 2, lambda i, h: range(lens[i]))
    # an exponent s log2(e) below 2^18 is off by half a step, 2^-7, where it is rounded before the
    # maximum is taken off: a weight by a factor 2^(2^-7) < 1 + 2^-7 / ln(4), the result by twice that
    d = np.abs(host_f32(got).astype(np.float64) - out)
    over = d - S.tolerance(out, mass) - 2.0 ** -6 * mass
    assert (over <= 0).all(), ((over > 0).any(-1).mean(), over.max())
    assert int(st.item()) == 0


def test_strided_rows_and_neighbours_of_the_result(ops):
    case = build(5, [(256, [5, 9, 70])], 64, "NHD", 8, 2)
    packed = torch.zeros((3, 12 * 128), dtype=torch.bfloat16, device="cuda")
    packed[:, :1024] = dev(case[0]).view(3, 1024)
    out = torch.full((5, 10, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    q, kc, vc, lens, table, starts, prefix = case
    ops.shared_prefix_attn(packed[:, :1024].view(3, 8, 128), dev(kc), dev(vc), ints(lens),
                           ints(table), ints(starts), ints(prefix), S.SCALE, out=out[:3, :8])
    assert torch.equal(out[:3, :8], run(ops, case, "NHD"))
    assert (out[3:] == 3.0).all() and (out[:, 8:] == 3.0).all()


def test_bad_pages_are_flagged_and_left_out(ops):
    case = build(6, [(256, [5, 9, 70]), (128, [3, 4])], 64, "NHD", 8, 2)
    q, kc, vc, lens, table, starts, prefix = case
    good = host_f32(run(ops, case, "NHD"))
    broken = table.copy()
    broken[2, 1], broken[4, 2] = 10 ** 6, -7       # the longest row's is read for its group
    st = ops.new_status("cuda")
    got = host_f32(run(ops, (q, kc, vc, lens, broken, starts, prefix), "NHD", st))
    assert int(st.item()) == 2
    assert np.isfinite(got).all() and (got[3] == good[3]).all()
    narrow = broken[:, :7]
    st = ops.new_status("cuda")
    got = host_f32(run(ops, (q, kc, vc, lens, narrow, starts, prefix), "NHD", st))
    assert int(st.item()) == 2 and np.isfinite(got).all()


@pytest.mark.parametrize("wide", [True, False])
def test_groups_that_do_not_fit_the_batch(ops, wide):
    """Starts past the batch or below the one before are flagged; nobody has anything in common
    then, and all rows have their results."""
    case = build(7, [(128, [5, 9, 70]), (64, [3, 4])], 64, "NHD", 4, 2, wide=wide)
    q, kc, vc, lens, table, _, prefix = case
    good = host_f32(run(ops, case, "NHD"))
    for starts in ([0, 3, 99], [-4, 3, 5], [0, 3, 1]):
        st = ops.new_status("cuda")
        got = host_f32(run(ops, (q, kc, vc, lens, table, starts, prefix), "NHD", st))
        assert int(st.item()) == 8
        assert np.abs(got - good).max() <= 2.0 ** -6


def test_in_a_graph_with_other_lengths(ops):
    """Captured once; replayed with other lengths, groups and queries in the same buffers."""
    rng = np.random.default_rng(9)
    case = build(9, [(640, [400, 500, 600]), (320, [100, 900])], 64, "NHD", 8, 2)
    q, kc, vc, lens, table, starts, prefix = case
    kc, vc = np.nan_to_num(kc), np.nan_to_num(vc)
    a = [dev(q), dev(kc), dev(vc), ints(lens), ints(table), ints(starts), ints(prefix)]
    ws = torch.empty(ops.shared_prefix_workspace_bytes(5, 2, 8, 2, 128, 16), dtype=torch.uint8,
                     device="cuda")
    ops.shared_prefix_attn(*a, S.SCALE, workspace=ws, max_splits=16)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.shared_prefix_attn(*a, S.SCALE, workspace=ws, max_splits=16)
    for step in range(3):
        q = S.bf16(rng.standard_normal(q.shape))
        lens = (lens - rng.integers(0, 90, 5)).astype(np.int32)
        shorter = [640 - 64 * step, 320 - 128 * step]
        a[0].copy_(dev(q))
        a[3].copy_(ints(lens))
        a[6].copy_(ints(shorter))
        g.replay()
        want, mass = S.over_positions(q, kc, vc, lens, table, 64, "NHD", 2,
                                      lambda i, h: range(lens[i]))
        d = np.abs(host_f32(out) - want)
        assert (d <= S.tolerance(want, mass)).all()


@pytest.mark.parametrize("rows", [2, 30])
def test_planned_layers(ops, rows):
    """One schedule, several layers with other queries and caches by it, in a graph too."""
    case = build(11, [(640, [40 + i for i in range(rows)]), (320, [100, 900])], 64, "NHD", 16, 8)
    q, kc, vc, lens, table, starts, prefix = case
    b = len(lens)
    n = ops.shared_prefix_workspace_bytes(b, 2, 16, 8, 128, 16)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    args = [ints(lens), ints(table)]
    groups = [ints(starts), ints(prefix)]
    layers = [(dev(S.bf16(q * f)), dev(kc), dev(S.bf16(vc * f))) for f in (1.0, 0.5, 2.0)]

    def run_all():
        ops.shared_prefix_plan(*args, 64, 16, 8, 128, *groups, ws, 16)
        return [ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, workspace=ws, max_splits=16,
                                       planned=True) for x in layers]
    want = [ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, max_splits=16) for x in layers]
    for a, b_ in zip(run_all(), want):
        assert torch.equal(a, b_)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run_all()
    for _ in range(2):
        g.replay()
        for a, b_ in zip(got, want):
            assert torch.equal(a, b_)


def test_planned_without_its_schedule(ops):
    """A workspace without a schedule, or with that of a step of other sizes: zeros and a flag."""
    case = build(12, [(640, [40 + i for i in range(20)]), (320, [100, 900])], 64, "NHD", 16, 8)
    q, kc, vc, lens, table, starts, prefix = case
    n = ops.shared_prefix_workspace_bytes(len(lens), 2, 16, 8, 128, 16)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    args, groups = [ints(lens), ints(table)], [ints(starts), ints(prefix)]
    x = [dev(q), dev(kc), dev(vc)]

    def planned():
        status = ops.new_status("cuda")
        out = torch.full_like(x[0], 7.0)
        ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, workspace=ws, out=out, status=status,
                               planned=True, max_splits=16)
        return out, int(status.item())
    want = ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, max_splits=16)
    out, status = planned()
    assert status == 8 and not out.any()
    # the schedule of fewer rows, of longer tables, of other splits
    ops.shared_prefix_plan(args[0][:20], args[1][:20], 64, 16, 8, 128, ints([0, 20]), ints([640]),
                           ws, 16)
    assert planned()[1] == 8
    wide = torch.cat([args[1], torch.full_like(args[1], -1)], dim=1)
    ops.shared_prefix_plan(args[0], wide, 64, 16, 8, 128, *groups, ws, 16)
    assert planned()[1] == 8
    ops.shared_prefix_plan(*args, 64, 16, 8, 128, *groups, ws, 8)
    assert planned()[1] == 8
    ops.shared_prefix_plan(*args, 64, 16, 8, 128, *groups, ws, 16)
    out, status = planned()
    assert status == 0 and torch.equal(out, want)


@pytest.mark.parametrize("word", [-1, -2 ** 31, 2 ** 31 - 1, 3, "normal", "-0.5", "-0.01", "-1.5", "-3.0"])
def test_planned_on_any_words(ops, word):
    """Whatever a workspace holds instead of a schedule of these sizes, and behind the schedule of others:
    zeros and a flag, and nothing but the counter is written."""
    case = build(12, [(640, [40 + i for i in range(20)]), (320, [100, 900])], 64, "NHD", 16, 8)
    q, kc, vc, lens, table, starts, prefix = case
    n = ops.shared_prefix_workspace_bytes(len(lens), 2, 16, 8, 128, 16)
    args, groups = [ints(lens), ints(table)], [ints(starts), ints(prefix)]
    x = [dev(q), dev(kc), dev(vc)]
    words = torch.empty(n // 4, dtype=torch.int32, device="cuda")
    if isinstance(word, int):
        words.fill_(word)
    elif word == "normal":
        torch.manual_seed(5)
        words.copy_(torch.randn(n // 4, device="cuda").view(torch.int32))
    else:
        words.copy_(torch.full((n // 4,), float(word), device="cuda").view(torch.int32))
    ws = words.view(torch.uint8)

    def planned():
        status = ops.new_status("cuda")
        out = torch.full_like(x[0], 7.0)
        before = words.clone()
        ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, workspace=ws, out=out, status=status,
                               planned=True, max_splits=16)
        assert int(status.item()) == 8 and not out.any()
        changed = (words != before).nonzero().flatten().tolist()
        assert changed in ([], [2])
    planned()
    wide = torch.cat([args[1], torch.full_like(args[1], -1)], dim=1)
    for other in ((args[0][:20], args[1][:20], 64, 16, 8, 128, ints([0, 20]), ints([640]), ws, 16),
                  (args[0], wide, 64, 16, 8, 128, *groups, ws, 16),
                  (*args, 64, 16, 8, 128, *groups, ws, 8)):
        ops.shared_prefix_plan(*other)
        planned()


def test_planned_after_another_schedule_in_its_place(ops):
    """paged_decode_attn in the workspace of a schedule leaves one of its own there: the planned call
    behind it gives zeros and a flag, and after a new schedule its result."""
    case = build(12, [(640, [40 + i for i in range(20)]), (320, [100, 900])], 64, "NHD", 16, 8)
    q, kc, vc, lens, table, starts, prefix = case
    args, groups = [ints(lens), ints(table)], [ints(starts), ints(prefix)]
    x = [dev(q), dev(kc), dev(vc)]
    ws = torch.empty(max(ops.shared_prefix_workspace_bytes(len(lens), 2, 16, 8, 128, 16),
                         ops.attn_workspace_bytes(len(lens), 16, 128, 16)), dtype=torch.uint8, device="cuda")

    def planned():
        status = ops.new_status("cuda")
        out = torch.full_like(x[0], 7.0)
        ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, workspace=ws, out=out, status=status,
                               planned=True, max_splits=16)
        return out, int(status.item())
    want = ops.shared_prefix_attn(*x, *args, *groups, S.SCALE, max_splits=16)
    for whole in (True, False):
        ops.shared_prefix_plan(*args, 64, 16, 8, 128, *groups, ws, 16)
        if whole:
            ops.paged_decode_attn(*x, *args, S.SCALE, ws, 16)
        else:
            ops.paged_decode_attn_plan(*args, 64, 16, 8, 128, ws, 16)
        out, status = planned()
        assert status == 8 and not out.any()
    ops.shared_prefix_plan(*args, 64, 16, 8, 128, *groups, ws, 16)
    out, status = planned()
    assert status == 0 and torch.equal(out, want)


def test_calls_on_two_streams(ops):
    """Two calls at once, each with a workspace of its own."""
    cases = [build(20 + i, [(2048, [70 + 5 * i] * 12), (640, [300, 9])], 64, "NHD", 16, 4)
             for i in range(2)]
    want = [run(ops, c, "NHD") for c in cases]
    side = [torch.cuda.Stream() for _ in cases]
    tensors = [[dev(c[0]), dev(c[1]), dev(c[2])] + [ints(x) for x in c[3:]] for c in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, a in zip(side, tensors):
            with torch.cuda.stream(s):
                got.append(ops.shared_prefix_attn(*a, S.SCALE))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_same_bits_every_time(ops):
    case = build(10, [(4096, [40, 50, 60, 1000] * 4), (320, [100, 900])], 64, "NHD", 8, 2)
    first = run(ops, case, "NHD")
    for _ in range(3):
        assert torch.equal(run(ops, case, "NHD"), first)
