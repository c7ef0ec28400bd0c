"""The operators of decode attention that read less of the paged KV cache, and what they are timed on.

  shared   attention of a batch whose sequences begin with the same pages (a system prompt, a
           document that is asked many questions, several answers to one prompt): the common part is
           read once for a whole group
  bounds   the smallest and largest value of every key channel over a block of cached tokens, for
           the blocks that new tokens have touched
  select   per query token and KV head the blocks that can hold the largest logits by those bounds
  attend   attention over selected blocks only
  sparse   bounds, select and attend one after another, as a decode step with sparse attention has it

A case holds the sizes; lengths come from the case alone, values and the order of pages from the
seed.  head_dim is 128 and the type bf16 throughout, as the caches of the framework have it.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
D = 128
SCALE = D ** -0.5
KEEP_FIRST, KEEP_LAST = 1, 2


# ------------------------------------------------------------------------------ cases
def shared(name, batch, groups, hq, hkv, page, layout, prefix, suffix):
    return _named(name, dict(op="shared", batch=batch, groups=groups, hq=hq, hkv=hkv, page=page,
                             layout=layout, prefix_min=prefix[0], prefix_max=prefix[1],
                             suffix_min=suffix[0], suffix_max=suffix[1]))


def sparse(op, name, batch, hq, hkv, page, layout, block, context, queries=1, count=0, new=(1, 1)):
    return _named(name, dict(op=op, batch=batch, hq=hq, hkv=hkv, page=page, layout=layout,
                             block=block, context_min=context[0], context_max=context[1],
                             queries=queries, count=count, new_min=new[0], new_max=new[1]))


def _named(name, c):
    return dict(c, name=name) if name else c


def listed():
    return [
        # a few short answers on a short common instruction: launches count
        shared("shared 8 short", 8, 1, 32, 8, 256, "NHD", (512, 512), (1, 200)),
        # a full chat batch behind one long system prompt
        shared("shared 64 system", 64, 1, 32, 8, 256, "NHD", (8192, 8192), (1, 1024)),
        # several applications' prompts in one batch, on 16-token head-major pages
        shared("shared 128 of 5 HND", 128, 5, 64, 8, 16, "HND", (500, 6000), (16, 2000)),
        # many samples on one document: the products are most of the time
        shared("shared 256 samples", 256, 1, 64, 4, 256, "NHD", (16384, 16384), (64, 512)),
        # a decode step's new keys
        sparse("bounds", "bounds step 64", 64, 32, 8, 64, "NHD", 64, (200, 8000)),
        # prompts that have just been stored
        sparse("bounds", "bounds prompts 7", 7, 32, 8, 256, "NHD", 64, (300, 8192),
               new=(300, 8192)),
        # a small batch with the finest blocks
        sparse("select", "select step 3", 3, 32, 8, 16, "HND", 16, (500, 4000), count=64),
        # a full batch of long documents
        sparse("select", "select step 64 long", 64, 32, 8, 256, "NHD", 64, (8192, 65536), count=64),
        # a prompt's portion: every token selects for itself
        sparse("select", "select portion 1000", 2, 32, 8, 64, "NHD", 64, (9000, 16000),
               queries=500, count=16),
        # one user's few long conversations
        sparse("attend", "attend step 4", 4, 32, 8, 64, "NHD", 64, (3000, 20000), count=32),
        # a full batch of long documents
        sparse("attend", "attend step 64", 64, 32, 8, 256, "NHD", 64, (8192, 32768), count=64),
        # the three in a row, five query heads to a KV head, on 16-token head-major pages
        sparse("sparse", "sparse step 48 HND", 48, 40, 8, 16, "HND", 16, (2000, 24000), count=128),
    ]


def draw(rng):
    def between(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))
    op = rng.choice(["shared", "shared", "bounds", "select", "attend", "sparse"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    page, layout = rng.choice([(16, "HND"), (16, "NHD"), (32, "NHD"), (64, "NHD"), (64, "HND"),
                               (256, "NHD")])
    if op == "shared":
        batch = between(2, 256)
        groups = rng.randint(1, max(1, min(8, batch // 2)))
        longest = between(page, max(page, min(12000, 240000000 // (batch * hq * groups))))
        return shared(None, batch, groups, hq, hkv, page,
                      layout, (max(1, int(longest * rng.uniform(0.2, 1.0))), longest),
                      (1, between(2, 150000 // batch)))
    block = rng.choice([b for b in (16, 32, 64, 128) if page % b == 0])
    queries = 1 if op == "bounds" or rng.random() < 0.7 else between(2, 60)
    tokens = between(1, 64)
    batch = max(1, tokens // queries)
    context = between(queries, 30000)
    count = min(between(4, 128), max(4, 4096 // block))
    new = (1, 1)
    if op == "bounds" and rng.random() < 0.5:
        batch = between(1, 16)
        new = (1, between(1, min(context, 60000 // batch)))
    return sparse(op, None, batch, hq, hkv, page, layout, block,
                  (max(queries, int(context * rng.uniform(0.1, 1.0))), context), queries, count,
                  new)


# ---------------------------------------------------------------- lengths, from the case alone
def _random(c):
    return random.Random(",".join(str(c[k]) for k in sorted(c) if k != "name"))


def _lengths_shared(c):
    """(first row of each group and the end, prefix tokens of each group, tokens of each row)."""
    r = _random(c)
    starts = [0] + sorted(r.sample(range(1, c["batch"]), c["groups"] - 1)) + [c["batch"]]
    prefix = []
    for _ in range(c["groups"]):
        p = r.randint(c["prefix_min"], c["prefix_max"])
        prefix.append(-(-p // c["page"]) * c["page"])
    lens = []
    for g in range(c["groups"]):
        for _ in range(starts[g], starts[g + 1]):
            lens.append(prefix[g] + r.randint(c["suffix_min"], c["suffix_max"]))
    return starts, prefix, lens


def _lengths_sparse(c):
    """(tokens of each sequence, new tokens of each)."""
    r = _random(c)
    lens = [r.randint(c["context_min"], c["context_max"]) for _ in range(c["batch"])]
    return lens, [min(n, r.randint(c["new_min"], c["new_max"])) for n in lens]


def _ceil(a, b):
    return -(-a // b)


# -------------------------------------------------------------------------------- inputs
def _values(gen, *shape):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * 0.5).bfloat16()


def _pool(gen, pages, c, with_values=True):
    """Keys with an offset per head and channel, as trained models have them, and values."""
    tail = (c["page"], c["hkv"], D) if c["layout"] == "NHD" else (c["hkv"], c["page"], D)
    off = torch.randn((c["hkv"], D), generator=gen, device=DEVICE) * 0.5
    off = off if c["layout"] == "NHD" else off[:, None, :]
    keys = torch.empty((pages, *tail), dtype=torch.bfloat16, device=DEVICE)
    values = torch.empty_like(keys) if with_values else None
    piece = max(1, (1 << 27) // (c["page"] * c["hkv"] * D))
    for a in range(0, pages, piece):
        n = min(piece, pages - a)
        keys[a:a + n] = _values(gen, n, *tail) + off
        if with_values:
            values[a:a + n] = _values(gen, n, *tail)
    return keys, values


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(gen, need):
    """Page tables of sequences that need so many pages each, in random order, -1 behind the last."""
    cols = max(need)
    order = torch.randperm(sum(need), generator=gen, device=DEVICE).int()
    at = torch.arange(cols, device=DEVICE)[None, :]
    have = torch.tensor(need, device=DEVICE)[:, None]
    first = torch.cumsum(have, 0) - have
    return torch.where(at < have, order[(first + at).clamp(max=sum(need) - 1)], -1).int()


def prepare(case, seed):
    c = case
    gen = torch.Generator(DEVICE).manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "shared":
        starts, prefix, lens = _lengths_shared(c)
        need = [p // c["page"] for p in prefix] + \
            [_ceil(n, c["page"]) - prefix[g] // c["page"]
             for g in range(c["groups"]) for n in lens[starts[g]:starts[g + 1]]]
        parts = _tables(gen, need)
        cols = max(_ceil(n, c["page"]) for n in lens)
        tables = torch.full((c["batch"], cols + 1), -1, dtype=torch.int32, device=DEVICE)
        for g in range(c["groups"]):
            p = need[g]
            for i in range(starts[g], starts[g + 1]):
                own_pages = need[c["groups"] + i]
                tables[i, :p] = parts[g, :p]
                tables[i, p:p + own_pages] = parts[c["groups"] + i, :own_pages]
        s.update(q=_values(gen, c["batch"], c["hq"], D), lens=_ints(lens), tables=tables,
                 starts=_ints(starts), prefix=_ints(prefix), longest_prefix=max(prefix),
                 longest_suffix=c["suffix_max"],
                 widest=max(b - a for a, b in zip(starts, starts[1:])))
        s["keys"], s["values"] = _pool(gen, sum(need), c)
        return s
    lens, new = _lengths_sparse(c)
    need = [_ceil(n, c["page"]) for n in lens]
    s.update(tables=_tables(gen, need), seq_lens=_ints(lens), longest=max(lens))
    if c["op"] != "select":
        s["keys"], s["values"] = _pool(gen, sum(need), c, c["op"] != "bounds")
    shape = (sum(need), c["hkv"], c["page"] // c["block"], 2, D)
    if c["op"] == "select":
        # bounds as blocks of the same kind of keys have them: around an offset per channel
        off = torch.randn((c["hkv"], 1, D), generator=gen, device=DEVICE) * 0.5
        far = 0.5 * math.sqrt(2 * math.log(c["block"]))
        sides = [off + sign * (far + 0.15 * torch.randn((*shape[:3], D), generator=gen,
                                                        device=DEVICE)) for sign in (-1, 1)]
        s["bounds"] = torch.stack([torch.minimum(*sides), torch.maximum(*sides)], 3).bfloat16()
    else:
        s["bounds"] = torch.zeros(shape, dtype=torch.bfloat16, device=DEVICE)
    if c["op"] in ("bounds", "sparse"):
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s.update(cu_new=_ints(cu) if c["new_max"] > 1 else None, max_new=max(new))
    if c["op"] == "sparse":
        s["bounds"].copy_(_block_bounds(s["keys"], c))     # the steps before have left these
    if c["op"] != "bounds":
        # the last `queries` tokens of every sequence; one each: the rows of the tables
        m = c["queries"]
        s["q"] = _values(gen, c["batch"] * m, c["hq"], D) * 2
        s["lens"] = _ints([n - m + 1 + j for n in lens for j in range(m)])
        s["rows"] = _ints([i for i in range(c["batch"]) for _ in range(m)]) if m > 1 else None
    if c["op"] == "attend":
        n = (s["lens"] + c["block"] - 1) // c["block"]
        at = torch.arange(max(c["count"], _ceil(max(lens), c["block"])), device=DEVICE)
        rank = torch.rand((len(s["lens"]), c["hkv"], len(at)), generator=gen, device=DEVICE)
        rank = torch.where(at == n[:, None, None] - 1, 2.0, rank)
        rank = torch.where(at >= n[:, None, None], -1.0, rank)
        best = rank.topk(c["count"], -1)
        got = torch.where(best.values >= 0, best.indices, len(at)).sort(-1).values
        s["selected"] = torch.where(got < len(at), got, -1).int()
    return s


def _block_bounds(keys, c):
    """Bounds of all blocks of a pool, [pages, heads, blocks of a page, 2, D]."""
    k = keys if c["layout"] == "HND" else keys.transpose(1, 2)
    k = k.reshape(k.shape[0], c["hkv"], c["page"] // c["block"], c["block"], D)
    return torch.stack([k.amin(3), k.amax(3)], 3)


# ------------------------------------------------------------------------------ plain forms
def _gather(pool, pages, offsets, layout):
    """Cached rows at (page, offset) in fp32: [..., heads, D]."""
    if layout == "NHD":
        return pool[pages, offsets].float()
    return pool[pages, :, offsets].float()


def _plain_shared(s):
    c = s["case"]
    b, hkv, g = c["batch"], c["hkv"], c["hq"] // c["hkv"]
    dev = s["q"].device
    q = s["q"].float().view(b, hkv, g, D)
    row = torch.arange(b, device=dev)
    group = torch.searchsorted(s["starts"], row, right=True) - 1
    # the common parts, once per group, for its rows side by side
    width, pmax = s["widest"], s["longest_prefix"]
    t = torch.arange(pmax, device=dev)
    pages = s["tables"][s["starts"][:-1].long()][:, t // c["page"]].clamp(min=0).long()
    off = (t % c["page"]).expand_as(pages)
    member = (s["starts"][:-1, None] + torch.arange(width, device=dev)).clamp(max=b - 1).long()
    q_of = q[member]                                               # [groups, width, hkv, g, D]
    common = torch.einsum("rwhgd,rphd->rwhgp", q_of, _gather(s["keys"], pages, off, c["layout"]))
    place = (row - s["starts"][group]).long()
    common = common[group, place] * SCALE                          # [b, hkv, g, pmax]
    common = common.masked_fill((t >= s["prefix"][group, None])[:, None, None], -math.inf)
    # what every row has for itself
    u = s["prefix"][group, None] + torch.arange(s["longest_suffix"], device=dev)
    live = u < s["lens"][:, None]
    u = torch.where(live, u, 0)
    pages_u = torch.gather(s["tables"], 1, (u // c["page"]).long()).clamp(min=0).long()
    k = _gather(s["keys"], pages_u, u % c["page"], c["layout"])
    alone = torch.einsum("bhgd,bshd->bhgs", q, k) * SCALE
    alone = alone.masked_fill(~live[:, None, None], -math.inf)
    p = torch.softmax(torch.cat([common, alone], -1), -1)
    v = _gather(s["values"], pages_u, u % c["page"], c["layout"])
    out = torch.einsum("bhgs,bshd->bhgd", p[..., pmax:], v)
    p_of = torch.zeros((len(s["prefix"]), width, hkv, g, pmax), device=dev)
    p_of[group, place] = p[..., :pmax]
    v = _gather(s["values"], pages, off, c["layout"])
    out = out + torch.einsum("rwhgp,rphd->rwhgd", p_of, v)[group, place]
    return out.view(b, c["hq"], D).bfloat16()


def _plain_bounds(s):
    c = s["case"]
    dev = s["tables"].device
    lens = s["seq_lens"].long()
    new = (s["cu_new"][1:] - s["cu_new"][:-1]).long() if s["cu_new"] is not None else \
        torch.ones_like(lens)
    first, last = (lens - new) // c["block"], (lens - 1) // c["block"]
    width = (s["max_new"] - 1) // c["block"] + 2
    blocks = torch.minimum(first[:, None] + torch.arange(width, device=dev), last[:, None])
    t = blocks[:, :, None] * c["block"] + torch.arange(c["block"], device=dev)
    live = (t < lens[:, None, None])[..., None, None]
    pages = torch.gather(s["tables"], 1, blocks * c["block"] // c["page"]).long()
    k = _gather(s["keys"], pages[:, :, None].expand_as(t), t % c["page"], c["layout"])
    lo = k.masked_fill(~live, math.inf).amin(2)                    # [batch, width, hkv, D]
    hi = k.masked_fill(~live, -math.inf).amax(2)
    sub = blocks * c["block"] % c["page"] // c["block"]
    s["bounds"][pages, :, sub] = torch.stack([lo, hi], 3).bfloat16()
    return s["bounds"]


def _plain_select(s):
    c = s["case"]
    dev, tokens = s["q"].device, len(s["lens"])
    rows = s["rows"].long() if s["rows"] is not None else torch.arange(tokens, device=dev)
    total = max(c["count"], _ceil(s["longest"], c["block"]))
    at = torch.arange(total, device=dev)
    n = ((s["lens"] + c["block"] - 1) // c["block"]).long()[:, None, None]
    per = c["page"] // c["block"]
    pages = s["tables"][:, (at // per).clamp(max=s["tables"].shape[1] - 1)].clamp(min=0).long()
    # in 64 bits: blocks next to the border must fall on the right side of it
    b = s["bounds"][pages, :, (at % per).expand_as(pages)].double()  # [sequences, total, hkv, 2, D]
    q = s["q"].double().view(tokens, c["hkv"], -1, D)
    q = q.view(c["batch"], c["queries"], c["hkv"], -1, D)
    score = torch.einsum("bmhgd,bnhd->bmhgn", q.clamp(min=0), b[..., 1, :]) + \
        torch.einsum("bmhgd,bnhd->bmhgn", q.clamp(max=0), b[..., 0, :])
    score = score.amax(3).view(tokens, c["hkv"], total)
    kept = (at < KEEP_FIRST) | (at >= n - KEEP_LAST)
    score = torch.where(kept, math.inf, score).masked_fill(at >= n, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True)
    best = order.indices[..., :c["count"]]
    got = torch.where(best < n, best, total).sort(-1).values
    return torch.where(got < total, got, -1).int()


def _plain_attend(s, selected):
    c = s["case"]
    tokens = len(s["lens"])
    dev = s["q"].device
    rows = s["rows"].long() if s["rows"] is not None else torch.arange(tokens, device=dev)
    t = selected.clamp(min=0)[..., None] * c["block"] + torch.arange(c["block"], device=dev)
    live = ((selected >= 0)[..., None] & (t < s["lens"][:, None, None, None])).flatten(2)
    t = torch.where(live, t.flatten(2), 0).long()                  # [tokens, hkv, keys]
    pages = s["tables"][rows[:, None, None], t // c["page"]].long()
    head = torch.arange(c["hkv"], device=dev)[None, :, None]
    where = (pages, t % c["page"], head) if c["layout"] == "NHD" else (pages, head, t % c["page"])
    q = s["q"].float().view(tokens, c["hkv"], -1, D)
    w = torch.einsum("thgd,thnd->thgn", q, s["keys"][where].float()) * SCALE
    p = torch.softmax(w.masked_fill(~live[:, :, None], -math.inf), -1)
    out = torch.einsum("thgn,thnd->thgd", p, s["values"][where].float())
    return out.reshape(tokens, c["hq"], D).bfloat16()


# --------------------------------------------------------------------------------- a pass
def run(state):
    s = state
    c = s["case"]
    if own:
        from fastkernels_b200 import ops
    if c["op"] == "shared":
        if not own:
            return _plain_shared(s)
        return ops.shared_prefix_attn(s["q"], s["keys"], s["values"], s["lens"], s["tables"],
                                      s["starts"], s["prefix"], SCALE, kv_layout=c["layout"])
    outputs = []
    if c["op"] in ("bounds", "sparse"):
        outputs.append(ops.key_bounds(s["keys"], s["bounds"], s["seq_lens"], s["tables"],
                                      cu_new=s["cu_new"], max_new=s["max_new"],
                                      kv_layout=c["layout"]) if own else _plain_bounds(s))
    if c["op"] in ("select", "sparse"):
        outputs.append(ops.select_blocks(s["q"], s["bounds"], s["lens"], s["tables"], c["block"],
                                         c["count"], keep_first=KEEP_FIRST, keep_last=KEEP_LAST,
                                         table_rows=s["rows"]) if own else _plain_select(s))
    if c["op"] in ("attend", "sparse"):
        selected = s["selected"] if c["op"] == "attend" else outputs[-1]
        outputs.append(ops.selected_attn(s["q"], s["keys"], s["values"], s["lens"], s["tables"],
                                         selected, c["block"], SCALE, table_rows=s["rows"],
                                         kv_layout=c["layout"]) if own else
                       _plain_attend(s, selected))
    return outputs[0] if len(outputs) == 1 else outputs


# ------------------------------------------------------------------------- what a pass needs
def work(case):
    c = case
    row = c["hkv"] * D * 2                                # bytes of a token's keys
    if c["op"] == "shared":
        starts, prefix, lens = _lengths_shared(c)
        seen = sum(prefix) + sum(n - prefix[g] for g in range(c["groups"])
                                 for n in lens[starts[g]:starts[g + 1]])
        pages = sum(_ceil(n, c["page"]) for n in lens)
        return {"bytes": seen * 2 * row + 2 * c["batch"] * c["hq"] * D * 2 + 4 * pages,
                "flops": 4 * D * c["hq"] * sum(lens)}
    lens, new = _lengths_sparse(c)
    block, m = c["block"], c["queries"]
    total = {"bytes": 0, "flops": 0}

    def add(bytes_, flops):
        total["bytes"] += bytes_
        total["flops"] += flops
    if c["op"] in ("bounds", "sparse"):
        for n, fresh in zip(lens, new):
            keys = n - (n - fresh) // block * block
            add(keys * row + 2 * row * _ceil(keys, block), 2 * keys * c["hkv"] * D)
    for n in lens:
        blocks = [_ceil(n - m + 1 + j, block) for j in range(m)]
        if c["op"] in ("select", "sparse"):
            add(2 * row * max(0, blocks[-1] - KEEP_FIRST - KEEP_LAST) + m * c["hq"] * D * 2 +
                4 * m * c["hkv"] * c["count"], 4 * D * c["hq"] * sum(blocks))
        if c["op"] in ("attend", "sparse"):
            keys = [(min(b, c["count"]) - 1) * block + (n - m + 1 + j - (b - 1) * block)
                    for j, b in enumerate(blocks)]
            add(min(sum(keys), n) * 2 * row + 2 * m * c["hq"] * D * 2 +
                4 * m * c["hkv"] * c["count"], 4 * D * c["hq"] * sum(keys))
    return total


# ------------------------------------------------------------------- from the definition, 64 bits
def _rows64(pool, table, tokens, c):
    """Cached rows of a sequence's tokens (a range or a tensor) in 64 bits: [tokens, heads, D]."""
    t = torch.as_tensor(tokens, device=DEVICE)
    page = table[t // c["page"]].long()
    got = pool[page, t % c["page"]] if c["layout"] == "NHD" else pool[page, :, t % c["page"]]
    return got.double()


def _attention64(q, k, v):
    """q [heads of a KV head, D] on k, v [keys, D]."""
    z = (k @ q.T) * SCALE
    e = torch.exp(z - z.max(0).values)
    return ((e.T @ v) / e.sum(0)[:, None])


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    g = c["hq"] // c["hkv"]
    tables = s["tables"].cpu()
    on_gpu = s["tables"]
    if c["op"] == "shared":
        lens = s["lens"].tolist()
        if c["batch"] * c["hkv"] > 1100:
            return None
        out = torch.zeros((c["batch"], c["hq"], D), dtype=torch.float64, device=DEVICE)
        for i, n in enumerate(lens):
            k = _rows64(s["keys"], on_gpu[i], torch.arange(n, device=DEVICE), c)
            v = _rows64(s["values"], on_gpu[i], torch.arange(n, device=DEVICE), c)
            for h in range(c["hkv"]):
                out[i, h * g:(h + 1) * g] = _attention64(s["q"][i, h * g:(h + 1) * g].double(),
                                                         k[:, h], v[:, h])
        return out
    outputs = []
    lens, new = _lengths_sparse(c)
    block, m = c["block"], c["queries"]
    if c["op"] in ("bounds", "sparse"):
        for i, (n, fresh) in enumerate(zip(lens, new)):
            for b in range((n - fresh) // block, (n - 1) // block + 1):
                k = _rows64(s["keys"], on_gpu[i],
                            torch.arange(b * block, min(n, (b + 1) * block), device=DEVICE), c)
                page = int(tables[i, b * block // c["page"]])
                sub = b * block % c["page"] // block
                s["bounds"][page, :, sub, 0] = k.min(0).values.bfloat16()
                s["bounds"][page, :, sub, 1] = k.max(0).values.bfloat16()
        outputs.append(s["bounds"].double())
    selected = s.get("selected")
    if c["op"] in ("select", "sparse"):
        selected = torch.full((c["batch"] * m, c["hkv"], c["count"]), -1, dtype=torch.int32)
        for i in range(c["batch"] * m):
            n = _ceil(lens[i // m] - m + 1 + i % m, block)
            b = torch.arange(n, device=DEVICE)
            per = c["page"] // block
            b64 = s["bounds"][on_gpu[i // m][b // per].long(), :, b % per].double()
            q64 = s["q"][i].double().view(c["hkv"], g, 1, D)
            b64 = b64.transpose(0, 1)[:, None]                     # [heads, 1, blocks, 2, D]
            score = torch.maximum(q64 * b64[..., 0, :], q64 * b64[..., 1, :]).sum(-1).amax(1)
            for h, of in enumerate(score.tolist()):
                rank = sorted(range(n), key=lambda x: (x >= KEEP_FIRST and x < n - KEEP_LAST,
                                                       -of[x], x))
                best = sorted(rank[:c["count"]])
                selected[i, h, :len(best)] = torch.tensor(best, dtype=torch.int32)
        outputs.append(selected)
    if c["op"] in ("attend", "sparse"):
        if c["batch"] * m * c["hkv"] > 4000:
            return None if len(outputs) == 0 else outputs + [None]
        chosen = selected.tolist()
        out = torch.zeros((c["batch"] * m, c["hq"], D), dtype=torch.float64, device=DEVICE)
        for i in range(c["batch"] * m):
            n = lens[i // m] - m + 1 + i % m
            for h in range(c["hkv"]):
                t = [x for b in chosen[i][h] if b >= 0
                     for x in range(b * block, min(n, (b + 1) * block))]
                t = torch.tensor(t, device=DEVICE)
                table = on_gpu[i // m]
                page, at = table[t // c["page"]].long(), t % c["page"]
                where = (page, at, h) if c["layout"] == "NHD" else (page, h, at)
                out[i, h * g:(h + 1) * g] = _attention64(
                    s["q"][i, h * g:(h + 1) * g].double(), s["keys"][where].double(),
                    s["values"][where].double())
        outputs.append(out)
    return outputs[0] if len(outputs) == 1 else outputs
