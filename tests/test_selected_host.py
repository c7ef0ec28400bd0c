"""What the calls of decode attention that reads less of the cache refuse, without a GPU, and their
plain statements against slower ones."""
import ctypes

import numpy as np
import pytest

import selected_oracle as S
from fastkernels_b200 import _lib

L = _lib.lib
INVALID, UNSUPPORTED, WORKSPACE, ALIGNMENT = -1, -2, -3, -4
P = 0x10000          # a non-null, 16-byte aligned stand-in; never dereferenced


def err():
    return L.fk_last_error().decode()


def call(fn, names, defaults, kw):
    assert set(kw) <= set(names), kw
    a = dict(defaults)
    a.update(kw)
    return fn(*[a[n] for n in names])


CACHE = dict(num_pages=8, page=64, kv_stride=64 * 2 * 128, layout=0, lens=P, tables=P, ts=4, cols=4,
             status=None, stream=None)


def bounds(**kw):
    names = "k num_pages page kv_stride layout hkv d bounds block lens tables ts cols cu n max_new " \
            "status stream".split()
    return call(L.fk_key_bounds, names,
                dict(CACHE, k=P, hkv=2, d=128, bounds=P, block=64, cu=None, n=3, max_new=1), kw)


def select(**kw):
    names = "q qs bounds num_pages page block lens rows tables ts cols num_tables n hq hkv d count " \
            "first last sel ws wsb status stream".split()
    return call(L.fk_select_blocks, names,
                dict(CACHE, q=P, qs=1024, bounds=P, block=64, rows=None, num_tables=3, n=3, hq=8,
                     hkv=2, d=128, count=4, first=1, last=1, sel=P, ws=P, wsb=1 << 30), kw)


def attend(**kw):
    names = "q qs out os k v num_pages page kv_stride layout lens rows tables ts cols num_tables sel " \
            "count block n hq hkv d scale ws wsb status stream".split()
    return call(L.fk_selected_attn, names,
                dict(CACHE, q=P, qs=1024, out=P, os=1024, k=P, v=P, rows=None, num_tables=3, sel=P,
                     count=4, block=64, n=3, hq=8, hkv=2, d=128, scale=0.1, ws=P, wsb=1 << 30), kw)


def shared(**kw):
    names = "planned q qs out os k v num_pages page kv_stride layout lens tables ts cols starts prefix groups " \
            "n hq hkv d scale splits ws wsb status stream".split()
    return call(L.fk_shared_prefix_attn, names,
                dict(CACHE, planned=0, q=P, qs=1024, out=P, os=1024, k=P, v=P, starts=P, prefix=P, groups=1,
                     n=3, hq=8, hkv=2, d=128, scale=0.1, splits=4, ws=P, wsb=1 << 30), kw)


def test_empty_calls_launch_nothing():
    before = L.fk_launch_count()
    assert bounds(n=0) == 0 and bounds(max_new=0, cu=P) == 0
    assert select(n=0, q=None) == 0 and attend(n=0, q=None) == 0 and shared(n=0, q=None) == 0
    assert L.fk_launch_count() == before


@pytest.mark.parametrize("fn", [bounds, select, attend, shared])
def test_common_refusals(fn):
    assert fn(n=-1) == INVALID and "negative" in err()
    assert fn(d=64) == UNSUPPORTED and "head_dim" in err()
    assert fn(lens=None) == INVALID and "null" in err()
    assert fn(tables=None) == INVALID
    assert fn(num_pages=0) == INVALID and "sizes" in err()
    assert fn(num_pages=1 << 31) == INVALID
    assert fn(cols=0) == INVALID
    assert fn(ts=-1) == INVALID and "stride" in err()
    if fn is not select:
        assert fn(kv_stride=64 * 2 * 128 - 8) == INVALID and "stride" in err()
        assert fn(layout=2) == INVALID and "kv_layout" in err()
        assert fn(kv_stride=64 * 2 * 128 + 4) == ALIGNMENT
    if fn is not bounds:
        assert fn(hq=5) == INVALID and "multiple" in err()
        assert fn(hq=34, qs=34 * 128, **({} if fn is select else {"os": 34 * 128})) == UNSUPPORTED
        assert fn(q=None) == INVALID and fn(q=P + 8) == ALIGNMENT
        assert fn(qs=1016) == INVALID and fn(qs=1028) == ALIGNMENT
    if fn is not shared:
        for block in (0, -16, 8, 24, 48, 80, 96):
            assert fn(block=block) == UNSUPPORTED and "block" in err()
        assert fn(block=128) == INVALID and "whole number" in err()


def test_bounds_refusals():
    assert bounds(k=P + 2) == ALIGNMENT and bounds(bounds=P + 8) == ALIGNMENT
    assert bounds(k=None) == INVALID and bounds(bounds=None) == INVALID
    assert bounds(max_new=2) == INVALID and "cu_new" in err()
    assert bounds(max_new=-1, cu=P) == INVALID
    assert bounds(n=65536) == UNSUPPORTED
    assert bounds(hkv=0) == INVALID


def test_select_refusals():
    assert select(count=0, first=0) == INVALID
    assert select(last=0) == INVALID and "at least the last" in err()
    assert select(first=4) == INVALID and select(first=-1) == INVALID
    assert select(last=2 ** 31 - 1, first=1) == INVALID
    assert select(num_tables=2) == INVALID and "tables" in err()
    assert select(cols=16385) == UNSUPPORTED and "16384" in err()
    assert select(sel=None) == INVALID and select(bounds=None) == INVALID
    need = L.fk_select_blocks_workspace_bytes(3, 8, 2, 64, 64, 4)
    assert need >= 3 * 2 * 4 * 4
    assert select(wsb=16) == WORKSPACE and select(ws=None) == WORKSPACE
    assert select(ws=P + 16) == WORKSPACE and "aligned" in err()
    assert L.fk_select_blocks_workspace_bytes(3, 8, 2, 64, 128, 4) == 0


def test_attend_refusals():
    assert attend(count=-1) == INVALID and attend(count=0) == INVALID
    assert attend(sel=None) == INVALID and attend(num_tables=2) == INVALID
    assert attend(page=48, kv_stride=48 * 2 * 128, block=16) == UNSUPPORTED
    need = L.fk_selected_attn_workspace_bytes(3, 8, 2, 128, 4, 64)
    assert attend(wsb=need - 1) == (WORKSPACE if need else 0) or need == 0
    if need:
        assert attend(ws=None) == WORKSPACE and attend(ws=P + 16) == WORKSPACE
    assert attend(out=P + 2) == ALIGNMENT and attend(os=512) == INVALID
    assert L.fk_selected_attn_workspace_bytes(0, 8, 2, 128, 4, 64) == 0


def test_shared_refusals():
    assert shared(groups=-1) == INVALID and shared(starts=None) == INVALID
    assert shared(prefix=None) == INVALID and shared(splits=0) == INVALID
    for scale in (0.0, -0.1, float("nan")):
        assert shared(scale=scale) == INVALID and "scale" in err()
    assert shared(splits=1 << 14) == INVALID
    assert shared(n=1 << 20, cols=1 << 20) == UNSUPPORTED
    assert shared(page=48, kv_stride=48 * 2 * 128) == UNSUPPORTED and "block_size" in err()
    need = L.fk_shared_prefix_workspace_bytes(3, 1, 8, 2, 128, 4)
    assert need > 0
    assert shared(wsb=need - 1) == WORKSPACE and shared(ws=None) == WORKSPACE
    assert shared(ws=P + 16) == WORKSPACE and "aligned" in err()
    assert L.fk_shared_prefix_workspace_bytes(3, 1, 8, 2, 128, 0) == 0


def test_plan_refusals():
    def plan(**kw):
        names = "lens page cols starts prefix groups n hq hkv d splits ws wsb status stream".split()
        return call(L.fk_shared_prefix_plan, names,
                    dict(CACHE, starts=P, prefix=P, groups=1, n=300, hq=8, hkv=2, d=128, splits=4, ws=P,
                         wsb=1 << 30), kw)
    need = L.fk_shared_prefix_workspace_bytes(300, 1, 8, 2, 128, 4)
    assert plan(n=0) == 0 and plan(n=-1) == INVALID
    assert plan(lens=None) == INVALID and plan(starts=None) == INVALID
    assert plan(wsb=need - 1) == WORKSPACE and plan(ws=P + 16) == WORKSPACE
    assert plan(d=64) == UNSUPPORTED and plan(hq=5) == INVALID and plan(splits=0) == INVALID
    assert plan(page=48) == UNSUPPORTED and plan(cols=0) == INVALID
    assert plan(n=16385, wsb=1 << 40) == UNSUPPORTED and "16384" in err()
    before = L.fk_launch_count()
    assert plan(n=3) == 0 and L.fk_launch_count() == before      # a small call needs no schedule


def test_wrappers_refuse_cpu_tensors_and_odd_layouts():
    import torch
    from fastkernels_b200 import ops
    q = torch.zeros((2, 4, 128), dtype=torch.bfloat16)
    cache = torch.zeros((3, 64, 2, 128), dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.shared_prefix_attn(q, cache, cache, i, i[:, None], i, i, 0.1),
              lambda: ops.key_bounds(cache, cache, i, i[:, None]),
              lambda: ops.select_blocks(q, cache, i, i[:, None], 64, 2),
              lambda: ops.selected_attn(q, cache, cache, i, i[:, None], i, 64, 0.1),
              lambda: ops.new_key_bounds(cache, 64)):
        with pytest.raises(_lib.FkError, match="CUDA tensor"):
            f()


def test_workspace_sizes_follow_the_device(monkeypatch):
    """The bytes depend on the SMs of the current device: a size asked for on one is not another's."""
    from types import SimpleNamespace
    from fastkernels_b200 import ops
    sms = [148]
    monkeypatch.setattr(ops, "lib", SimpleNamespace(
        **{f"fk_{n}_workspace_bytes": lambda *a: 1000 * sum(a) + sms[0]
           for n in ("shared_prefix", "select_blocks", "selected_attn")}))
    sizes = (1000, 1, 8, 2, 128, 4)
    for f in (ops.shared_prefix_workspace_bytes, ops.select_blocks_workspace_bytes,
              ops.selected_attn_workspace_bytes):
        name = "fk_" + f.__name__
        assert hasattr(L, name)
        for dev, n in ((0, 148), (1, 132), (0, 148)):
            sms[0] = n
            assert f(*sizes) == 1000 * sum(sizes) + n
            assert ops._bytes_on(dev, name, *sizes) == 1000 * sum(sizes) + n
    ops._bytes_on.cache_clear()


def test_the_bound_of_a_block_is_above_its_logits():
    rng = np.random.default_rng(1)
    kc = S.pool(rng, 6, 64, 2, "NHD")
    b = S.bounds_of(kc, 64, 16, "NHD")
    q = rng.standard_normal((20, S.D))
    for head in range(2):
        k = kc[:, :, head].reshape(6, 4, 16, S.D).astype(np.float64)
        logits = np.einsum("qd,pbtd->qpbt", q, k).max(-1)
        lo, hi = b[:, head, :, 0].astype(np.float64), b[:, head, :, 1].astype(np.float64)
        score = np.maximum(q[:, None, None] * lo, q[:, None, None] * hi).sum(-1)
        assert (score >= logits - 1e-9).all()


def test_the_plain_selection():
    """Two channels, by hand: scores 5, 9, 9, 1, the last block kept."""
    bounds_ = np.zeros((5, 1, 1, 2, S.D), np.float32)
    bounds_[:, 0, 0, 1, 0] = [5, 9, 9, 1, 0]
    q = np.zeros((1, 1, S.D), np.float32)
    q[0, 0, 0] = 1
    table = np.arange(5, dtype=np.int32)[None]
    assert S.select(q, bounds_, [300], table, 64, 3, 0, 1).tolist() == [[[1, 2, 4]]]
    assert S.select(q, bounds_, [300], table, 64, 2, 0, 1).tolist() == [[[1, 4]]]
    assert S.select(q, bounds_, [100], table, 64, 3, 0, 1).tolist() == [[[0, 1, -1]]]


def test_prototypes_fit_the_header():
    """One argument type for each argument that the header declares."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "fk_b200.h")).read(),
                  flags=re.S)
    kinds = {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "float": ctypes.c_float,
             "size_t": ctypes.c_size_t}
    for name in ("fk_key_bounds", "fk_select_blocks", "fk_selected_attn", "fk_shared_prefix_attn",
                 "fk_shared_prefix_plan",
                 "fk_selected_attn_workspace_bytes", "fk_select_blocks_workspace_bytes",
                 "fk_shared_prefix_workspace_bytes"):
        args = re.search(rf"\b{name}\s*\(([^)]*)\)", text).group(1).split(",")
        want = [ctypes.c_void_p if "*" in a or "fk_stream_t" in a else kinds[a.split()[0]]
                for a in args]
        assert _lib.PROTOTYPES[name][1] == want, name
