"""What the calls of KV caches that take less memory refuse, without a GPU, and their plain statements
against slower ones."""
import ctypes

import numpy as np
import pytest
import torch

import kvcache_oracle as S
from fastkernels_b200 import _lib, ops

L = _lib.lib
INVALID, UNSUPPORTED, WORKSPACE, ALIGNMENT = -1, -2, -3, -4
P = 0x10000          # a non-null, 16-byte aligned stand-in; never dereferenced


def err():
    return L.fk_last_error().decode()


def call(fn, names, defaults, kw):
    names = names.split()
    assert set(kw) <= set(names), kw
    a = dict(defaults, status=None, stream=None)
    a.update(kw)
    return fn(*[a[n] for n in names])


POOL = dict(cache=P, pages=8, page=64, hkv=2, d=128, group=64)
TABLES = dict(lens=P, tables=P, ts=4, cols=4)


def store(**kw):
    return call(L.fk_store_kvcache_q4,
                "k ks v vs cache pages page hkv d group slots wide n status stream",
                dict(POOL, k=P, ks=256, v=P, vs=256, slots=P, wide=0, n=3), kw)


def load(**kw):
    return call(L.fk_load_kvcache_q4, "k v cache pages page hkv d group slots wide n status stream",
                dict(POOL, k=P, v=P, slots=P, wide=1, n=3), kw)


def attend(**kw):
    return call(L.fk_paged_decode_attn_q4,
                "q qs out os cache pages page group lens tables ts cols cu seqs n hq hkv d scale "
                "weights frm longest ws wsb status stream",
                dict(POOL, **TABLES, q=P, qs=1024, out=P, os=1024, cu=None, seqs=3, n=3, hq=8,
                     scale=0.1, weights=None, frm=None, longest=0, ws=P, wsb=1 << 40), kw)


def attend_bf16(**kw):
    return call(L.fk_paged_decode_attn_weights,
                "q qs out os k v pages page stride layout lens tables ts cols cu seqs n hq hkv d "
                "scale weights frm longest splits ws wsb status stream",
                dict(POOL, **TABLES, q=P, qs=1024, out=P, os=1024, k=P, v=P, stride=64 * 256, layout=0,
                     cu=None, seqs=3, n=3, hq=8, scale=0.1, weights=P, frm=None, longest=256,
                     splits=4, ws=P, wsb=1 << 40), kw)


def evict(**kw):
    return call(L.fk_evict_kvcache,
                "k v pages page stride layout hkv d weights lens new tables ts cols seqs budget first "
                "last status stream",
                dict(POOL, **TABLES, k=P, v=P, stride=64 * 256, layout=0, weights=P, new=P + 64,
                     seqs=3, budget=100, first=4, last=20), kw)


def evict_q4(**kw):
    return call(L.fk_evict_kvcache_q4,
                "cache pages page hkv d group weights lens new tables ts cols seqs budget first last "
                "status stream",
                dict(POOL, **TABLES, weights=P, new=P + 64, seqs=3, budget=100, first=4, last=20), kw)


def test_null_pointers_of_a_store():
    for n in ("k", "v", "cache", "slots"):
        assert store(**{n: None}) == INVALID and "null pointer" in err()


@pytest.mark.parametrize("fn", [store, load, attend, evict_q4])
def test_pools_that_no_cache_has(fn):
    assert fn(cache=None) == INVALID and "null pointer" in err()
    assert fn(d=64) == UNSUPPORTED and "head_dim" in err()
    for group in (0, 16, 32, 256):
        assert fn(group=group) == UNSUPPORTED and "groups" in err()
    for page in (0, -16, 8, 24, 48, 80, 100):
        assert fn(page=page) == UNSUPPORTED and "page of" in err()
    assert fn(pages=0) == INVALID and fn(pages=1 << 31) == INVALID and fn(hkv=0) == INVALID
    assert fn(cache=P + 8) == ALIGNMENT


@pytest.mark.parametrize("fn,kw,code", [
    (store, dict(n=-1), INVALID), (store, dict(slots=None), INVALID), (store, dict(ks=255), INVALID),
    (store, dict(ks=260), ALIGNMENT), (store, dict(v=P + 2), ALIGNMENT),
    (store, dict(wide=2), INVALID), (store, dict(n=1 << 31), UNSUPPORTED),
    (load, dict(n=-1), INVALID), (load, dict(k=None), INVALID), (load, dict(v=P + 4), ALIGNMENT),
    (load, dict(slots=None), INVALID),
    (attend, dict(n=-1), INVALID), (attend, dict(seqs=-1), INVALID), (attend, dict(q=None), INVALID),
    (attend, dict(out=None), INVALID), (attend, dict(lens=None), INVALID),
    (attend, dict(tables=None), INVALID), (attend, dict(hq=7), INVALID), (attend, dict(hq=0), INVALID),
    (attend, dict(hq=34, qs=34 * 128, os=34 * 128), UNSUPPORTED), (attend, dict(seqs=2), INVALID),
    (attend, dict(qs=1016), INVALID), (attend, dict(os=1028), ALIGNMENT),
    (attend, dict(q=P + 2), ALIGNMENT), (attend, dict(cols=0), INVALID),
    (attend, dict(ts=-1), INVALID), (attend, dict(longest=-1), INVALID),
    (attend, dict(ws=None, cols=64), WORKSPACE), (attend, dict(wsb=1000, cols=64), WORKSPACE),
    (attend, dict(ws=P + 16, cols=64), WORKSPACE), (attend, dict(ws=None, weights=P), WORKSPACE),
    (attend_bf16, dict(weights=None), INVALID), (attend_bf16, dict(hq=6, qs=768, os=768), UNSUPPORTED),
    (attend_bf16, dict(seqs=2), INVALID), (attend_bf16, dict(layout=2), INVALID),
    (attend_bf16, dict(wsb=1000), WORKSPACE), (attend_bf16, dict(longest=-1), INVALID),
    (attend_bf16, dict(stride=100), INVALID), (attend_bf16, dict(page=48), UNSUPPORTED),
    (attend_bf16, dict(k=None), INVALID), (attend_bf16, dict(cols=0), INVALID),
    (evict, dict(k=None), INVALID), (evict, dict(weights=None), INVALID), (evict, dict(new=None), INVALID),
    (evict, dict(new=P), INVALID), (evict, dict(new=P + 8), INVALID), (evict_q4, dict(new=P - 8), INVALID),
    (evict, dict(lens=None), INVALID), (evict, dict(d=64), UNSUPPORTED),
    (evict, dict(layout=2), INVALID), (evict, dict(stride=100), INVALID),
    (evict, dict(v=P + 8), ALIGNMENT), (evict, dict(page=0), INVALID), (evict, dict(cols=0), INVALID)])
def test_refusals(fn, kw, code):
    assert fn(**kw) == code, err()


@pytest.mark.parametrize("fn", [evict, evict_q4])
def test_budgets_that_cannot_be(fn):
    for kw in (dict(budget=0), dict(first=-1), dict(last=-1), dict(first=101), dict(last=97),
               dict(first=2 ** 31 - 1, last=2 ** 31 - 1), dict(seqs=-1)):
        assert fn(**kw) == INVALID, kw


def test_nothing_to_do_launches_nothing():
    before = L.fk_launch_count()
    assert store(n=0, k=None, slots=None) == 0 and load(n=0, k=None) == 0
    assert attend(n=0, q=None) == 0 and attend(seqs=0, q=None) == 0
    assert attend_bf16(n=0, q=None, weights=None) == 0
    assert evict(seqs=0, weights=None) == 0 and evict_q4(seqs=0, lens=None) == 0
    assert L.fk_launch_count() == before


def test_workspaces():
    def q4(n=4, s=4, hq=32, hkv=8, d=128, w=0, longest=0):
        return ops.paged_decode_attn_q4_workspace_bytes(n, s, hq, hkv, d, w, longest)
    assert q4() > 0 and q4(n=0) == 0 and q4(hq=200) == 0 and q4(d=64) == 0 and q4(longest=-1) == 0
    assert q4(longest=10 ** 6) == q4()                 # only sums of weights grow with it
    assert q4(longest=2048) == 0 and q4(longest=2049) == q4() and q4(w=1, longest=2048) > q4()
    assert q4(w=1, longest=8192) - q4(w=1) == 4 * 8 * 8192 * 4 * 4
    assert q4(n=64, s=4) > q4(n=4, s=4)
    need = ops.paged_decode_attn_weights_workspace_bytes(3, 8, 128, 4, False, 256)
    assert attend_bf16(wsb=need - 1) == WORKSPACE and need % 256 == 0
    need = q4(3, 3, 8, 2)
    assert attend(wsb=need - 1, cols=64) == WORKSPACE


def test_calls_refuse_tensors_on_the_host():
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    cache = torch.zeros((4, 2, 4, 2304), dtype=torch.uint8)
    i = torch.zeros(2, dtype=torch.int32)
    for f in (lambda: ops.store_kvcache_q4(x, x, cache, i), lambda: ops.load_kvcache_q4(cache, i),
              lambda: ops.paged_decode_attn_q4(x, cache, i, i.view(2, 1), 0.1),
              lambda: ops.paged_decode_attn_weights(x, x, x, i, i.view(2, 1), 0.1, x),
              lambda: ops.evict_kvcache(cache, torch.zeros((4, 2, 64)), i, i.view(2, 1), 8)):
        with pytest.raises(_lib.FkError, match="CUDA tensor"):
            f()
    for kw in (dict(head_dim=64), dict(group=32), dict(page_size=24)):
        with pytest.raises(_lib.FkError):
            ops.new_kvcache_q4(**dict(dict(num_pages=2, page_size=64, num_kv_heads=2, device="cpu"), **kw))
    assert ops.new_kvcache_q4(3, 64, 2, device="cpu").shape == (3, 2, 4, 2304)
    assert ops.new_kvcache_q4(3, 64, 2, group=128, device="cpu").shape == (3, 2, 4, 2176)


# --------------------------------------------------------------------- the plain statements
@pytest.mark.parametrize("group", [64, 128])
def test_codes_are_the_nearest_steps(group):
    rng = np.random.default_rng(0)
    x = S.randn(rng, 40, 3, 128)
    lo, s, code = S.quantise(x, group)
    got = S.values(x, group).reshape(40, 3, -1, group)
    g = x.reshape(40, 3, -1, group)
    every = lo[..., None, None] + s[..., None, None] * np.arange(16)
    best = np.abs(every - g[..., None]).min(-1)
    np.testing.assert_array_equal(np.abs(got - g), best)
    # half a step, and what the scale's rounding leaves of the fifteen
    assert (np.abs(got - g) <= s[..., None] * (0.5 + 15 * 2.0 ** -8)).all()
    assert (code.reshape(40, 3, -1, group).min(-1) == 0).all()


def test_packed_units_hold_every_channel_at_its_place():
    """Read one by one, by the layout's words, not the packer's loops."""
    rng = np.random.default_rng(1)
    for group in (64, 128):
        ng = 128 // group
        k, v = S.randn(rng, 32, 1, 128), S.randn(rng, 32, 1, 128)
        pool = S.pool_q4(2, 32, 1, group)
        slots = [32 + i for i in range(32)]
        S.put(pool, k, v, slots, group)
        whole = S.pack(k[:, 0], v[:, 0], group)
        np.testing.assert_array_equal(pool[1, 0], whole)
        assert (pool[0] == 0xFF).all()
        for t in (0, 5, 16, 31):
            u = pool[1, 0, t // 16]
            for kv, x in enumerate((k, v)):
                lo, s, code = S.quantise(x[t, 0], group)
                for c in (0, 1, 7, 8, 63, 64, 100, 127):
                    w = c // 8
                    place = [w % 4 * 4 + w // 4, w % 8 * 2 + w // 8][kv]
                    byte = u[kv * 1024 + t % 16 * 64 + place * 4 + c % 8 // 2]
                    assert (byte >> (4 * (c % 2))) & 15 == code[c]
                    at = 2048 + (kv * 16 + t % 16) * 4 * ng + 4 * (c // group)
                    pair = u[at:at + 4].view(np.uint16).astype(np.uint32) << 16
                    assert pair.view(np.float32)[0] == np.float32(s[c // group])
                    assert pair.view(np.float32)[1] == np.float32(lo[c // group])


def test_eviction_statement():
    w = np.array([9, 1, 5, 7, 3, 8, 2, 6, 4, 0], float)
    # first 1, last 2 of 6: 0 | the best three of 1 .. 7: 5, 3, 7 | 8, 9
    assert S.evict(10, w, 6, 1, 2) == [(5, 1), (7, 2), (8, 4), (9, 5)]
    assert S.evict(6, w[:6], 6, 1, 2) == []
    assert S.evict(5, np.zeros(5), 3, 0, 0) == []
    assert S.evict(5, np.array([np.nan, 1, 1, -np.inf, 1]), 3, 0, 0) == [(4, 0)]


def test_ctypes_take_large_sizes():
    assert ops.paged_decode_attn_q4_workspace_bytes(64, 64, 32, 8, 128, True, 1 << 20) > 1 << 33
    assert isinstance(L.fk_q4_unit_bytes(128, 64), int) and L.fk_q4_unit_bytes(128, 64) == 2304
    assert L.fk_q4_unit_bytes(128, 128) == 2176 and L.fk_q4_unit_bytes(64, 64) == 0
    assert ctypes.sizeof(ctypes.c_size_t) == 8


# ------------------------------------------------------------------------------- the engine
def test_configurations_that_have_no_4_bit_cache():
    from fastkernels_b200.candidate.L4.llama import LlamaConfig
    from fastkernels_b200.models.llama import ServedLlama
    small = dict(hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=4,
                 num_key_value_heads=2, vocab_size=128, max_position_embeddings=64)
    for kw in (dict(kv_bits=8), dict(kv_bits=4, head_dim=64), dict(kv_bits=4, kv_group=32),
               dict(kv_bits=4, kv_block_size=48), dict(kv_bits=4, num_attention_heads=34)):
        with pytest.raises(ValueError):
            ServedLlama(LlamaConfig(**dict(small, **kw)))


def test_slots_of_all_keys_of_a_prefill():
    from types import SimpleNamespace

    from fastkernels_b200.infra.context import key_slots
    lens, page = [5, 0, 130, 64], 64
    tables = torch.tensor([[3, -1, -1], [-1, -1, -1], [7, 1, 0], [2, -1, -1]], dtype=torch.int32)
    cu = torch.tensor(np.cumsum([0, *lens]), dtype=torch.int32)
    want = np.concatenate([S.slots_of(t, n, page) for t, n in zip(tables.numpy(), lens)])
    ctx = SimpleNamespace(cu_seqlens_k=cu, block_tables=tables, spans=None)
    got = key_slots(ctx, page)
    np.testing.assert_array_equal(got.numpy(), want)
    assert key_slots(ctx, page) is got                 # once a forward
    ctx = SimpleNamespace(cu_seqlens_k=cu, block_tables=tables,
                          spans=[SimpleNamespace(total_k=sum(lens))])
    np.testing.assert_array_equal(key_slots(ctx, page).numpy(), want)


def test_command_line_and_folder_options():
    from fastkernels_b200 import engine, generate
    assert generate.parse_args(["--model", "d", "--prompt", "1"]).kv_bits == 16
    assert generate.parse_args(["--model", "d", "--prompt", "1", "--kv-bits", "4"]).kv_bits == 4
    with pytest.raises(SystemExit):
        generate.parse_args(["--model", "d", "--prompt", "1", "--kv-bits", "8"])
    plain = SimpleConfig()
    old = engine.load_folder
    engine.load_folder = lambda folder, dtype: (plain, None)
    try:
        with pytest.raises(ValueError, match="4 bits"):
            engine.DecodeEngine.from_folder("d", max_tokens=8, max_num_seqs=1, kv_bits=4)
    finally:
        engine.load_folder = old


class SimpleConfig:
    """A configuration of a model whose cache is kept in its own type."""
