"""The engine with a KV cache of 4 bits: the same tokens' logits whichever way they come, and those of
an engine whose bf16 pool holds what 4 bits keep."""
import numpy as np
import pytest
import torch

import cases

pytestmark = pytest.mark.gpu
CFG = cases.TINY_QWEN3


def engine(kv_bits, block=64, group=64, layout="NHD", fused=True, seqs=4, max_len=400):
    from fastkernels_b200.candidate.L4.llama import LlamaConfig
    from fastkernels_b200.engine import DecodeEngine
    c = CFG
    cfg = LlamaConfig(hidden_size=c["hidden"], intermediate_size=c["ffn"],
                      num_hidden_layers=c["num_layers"], num_attention_heads=c["num_heads"],
                      num_key_value_heads=c["num_kv_heads"], head_dim=c["head_dim"],
                      vocab_size=c["vocab"], max_position_embeddings=max(c["max_pos"], max_len),
                      rms_norm_eps=c["eps"], rope_theta=c["theta"], qk_norm=c["qk_norm"],
                      kv_block_size=block, kv_layout=layout, fused_attention_prologue=fused,
                      kv_bits=kv_bits, kv_group=group)
    return DecodeEngine(cfg, max_num_seqs=seqs, max_model_len=max_len,
                        num_kv_blocks=seqs * (max_len // block + 2), seed=3, init_scale=0.08)


class Rounding(torch.nn.Module):
    """Stores to the bf16 pool what 4 bits keep of keys and values."""

    def __init__(self, store, group):
        super().__init__()
        self.store, self.group = store, group

    def forward(self, k, v, k_cache, v_cache, slots):
        from fastkernels_b200 import ops
        n, hkv = k.shape[:2]
        tmp = ops.new_kvcache_q4((n + 15) // 16, 16, hkv, group=self.group)
        at = torch.arange(n, device=k.device)
        ops.store_kvcache_q4(k, v, tmp, at)
        self.store(*ops.load_kvcache_q4(tmp, at), k_cache, v_cache, slots)


def rounded_engine(group, block):
    eng = engine(16, block=block, fused=False)
    for layer in eng.model.model.layers:
        layer.self_attn.attn.store_kvcache = Rounding(layer.self_attn.attn.store_kvcache, group)
    return eng


def feed(eng, prompts, cuts):
    """Logits of every prompt's last token and of the tokens behind it, one by one; prompts go in
    portions that end at `cuts`."""
    seqs = [eng.open_sequence() for _ in prompts]
    out = []
    for a, b in zip([0, *cuts], [*cuts, 10 ** 9]):
        part = [(s, p[:-5][a:b]) for s, p in zip(seqs, prompts) if len(p[:-5][a:b])]
        got = eng.feed(part)
    out.append(torch.cat(got))
    for j in range(5):
        out.append(torch.cat(eng.feed([(s, p[len(p) - 5 + j:][:1]) for s, p in zip(seqs, prompts)])))
    for s in seqs:
        eng.finish(s)
    return torch.stack(out)


def prompts(n, length):
    rng = np.random.default_rng(n)
    return [rng.integers(0, CFG["vocab"], length + 17 * i).tolist() for i in range(n)]


@pytest.mark.parametrize("block,group,layout", [(64, 64, "NHD"), (16, 128, "HND"), (256, 64, "NHD")])
def test_logits_are_those_of_a_pool_that_holds_what_4_bits_keep(block, group, layout):
    """bf16 rounds q k and softmax weights elsewhere in the two: as far apart as the engine's own
    bf16 paths are, 8 % RMS of the logits' spread."""
    p = prompts(3, 130)
    got = feed(engine(4, block, group, layout), p, [])
    want = feed(rounded_engine(group, block), p, [])
    err = (got - want).pow(2).mean().sqrt() / want.std()
    assert err < 0.08, err
    assert got.isfinite().all()


def test_portions_and_tokens_see_the_same_cache():
    p = prompts(3, 130)
    eng = engine(4)
    whole = feed(eng, p, [])
    for cuts in ([64], [1, 3, 50, 100], [120]):
        got = feed(eng, p, cuts)
        assert (got - whole).pow(2).mean().sqrt() / whole.std() < 0.08
    assert len(eng.seqs) == 0
    assert eng.device_status() == 0


def test_graphs_and_eager_steps_agree_and_generate():
    p = prompts(4, 60)
    tokens = []
    for graphs in (False, True):
        eng = engine(4)
        first = eng.prefill(p, chunk_tokens=50)
        if graphs:
            eng.capture_cudagraph([4])
        for _ in range(30):
            eng.step(sync=True)
        tokens.append([list(s.output) for s in eng.seqs])
        assert len(first) == 4 and eng.device_status() == 0
    assert tokens[0] == tokens[1]


def test_fused_prologue_and_separate_operators_agree():
    p = prompts(2, 70)
    a, b = (feed(engine(4, fused=f), p, [33]) for f in (True, False))
    assert (a - b).pow(2).mean().sqrt() / a.std() < 0.08


def test_pool_is_smaller_and_filled_at_random():
    small, large = engine(4), engine(16)
    size = sum(x.numel() for x in small.kv_cache)
    assert size * 512 == 144 * large.kv_cache.numel() * 2
    small.fill_kv_random(1)
    small.add_sequences([200, 90], [1, 2])
    assert len(small.step(sync=True)) == 2 and small.device_status() == 0


def test_command_line_of_a_llama_folder(tmp_path):
    import io
    import json
    import pinuvik_oracle
    from fastkernels_b200 import generate
    c = dict(architectures=["LlamaForCausalLM"], hidden_size=256, intermediate_size=256,
             num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
             vocab_size=320, max_position_embeddings=512, rms_norm_eps=1e-6, rope_theta=1e4)
    rng = np.random.default_rng(0)

    def m(*shape):
        return (rng.standard_normal(shape) * 0.1).astype(np.float32)
    w = {"model.embed_tokens.weight": m(320, 256), "model.norm.weight": np.ones(256, np.float32)}
    for i in range(2):
        h = f"model.layers.{i}."
        for n in ("input_layernorm", "post_attention_layernorm"):
            w[h + n + ".weight"] = np.ones(256, np.float32)
        for n, rows in (("q", 512), ("k", 256), ("v", 256)):
            w[f"{h}self_attn.{n}_proj.weight"] = m(rows, 256)
        w[h + "self_attn.o_proj.weight"] = m(256, 512)
        for n in ("gate", "up", "down"):
            w[f"{h}mlp.{n}_proj.weight"] = m(256, 256)
    pinuvik_oracle.write_folder(tmp_path, c, w)
    assert json.loads((tmp_path / "config.json").read_text())["vocab_size"] == 320
    outs = []
    for bits in ("16", "4"):
        out = io.StringIO()
        args = ["--model", str(tmp_path), "--prompt", "5,17,3", "--prompt", "9,8,7,6,5,4",
                "--max-new-tokens", "12", "--kv-bits", bits]
        assert generate.main(args, stdout=out) == 0
        outs.append([[int(t) for t in line.split(",")] for line in out.getvalue().split()])
    assert all(len(line) == 12 for o in outs for line in o) and len(outs[1]) == 2
