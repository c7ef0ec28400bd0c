"""Read from the kernels' source, without a GPU: what kernels of KV caches load lies in their buffers."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "fastkernels_b200" / "csrc"


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_sums_load_no_logits_behind_a_run():
    """The kernel's expressions for a lane's key and for what it loads, followed for contexts that are no
    whole steps: rows of logits are inside of what the attention before has, 32 a step, heads of a
    token one after another."""
    text = code("fk_sums.cu")
    none = int(re.search(r"SUMS_NONE = (\w+);", text).group(1), 0) if "SUMS_NONE =" in text else None
    inside, behind = re.search(r"key\[j\] = s0 \+ j < end \? ([^:;]*) : ([^:;]*);", text).groups()
    loads = re.findall(r"v\[j\] = ([^?;]*)\?\s*(?:\*reinterpret_cast<const float4\*>\(z|z\[)", text)
    assert len(loads) == 2
    steps_at_once = 4
    for hkv in range(1, 9):
        for lens in ([1], [31], [32], [33], [50], [64], [65], [100], [129], [1, 50, 7], [160, 0, 33],
                     [95, 200]):
            steps = [-(-n // 32) for n in lens]
            first = [sum(steps[:i]) for i in range(len(steps))]
            rows = 32 * hkv * sum(steps)
            total = hkv * sum(steps)
            for run in (4, 5, 7, 16):
                x = 0
                while x < total:
                    entry = max(i for i in range(len(lens)) if first[i] * hkv <= x and steps[i])
                    head, at = divmod(x - first[entry] * hkv, steps[entry])
                    end = min(steps[entry], at + min(total, x // run * run + run) - x)
                    for s0 in range(at, end, steps_at_once):
                        for j in range(steps_at_once):
                            for lane in (0, 31):
                                names = dict(s0=s0, j=j, lane=lane, most=lens[entry], end=end,
                                             SUMS_NONE=none)
                                key = eval(inside if s0 + j < end else behind, {}, names)
                                names.update(key={j: key}, len=32 * steps[entry])
                                base = (first[entry] * hkv + head * steps[entry]) * 32
                                for guard in loads:
                                    if eval(guard.replace("&&", " and ").strip(), {}, names):
                                        assert 0 <= base + (s0 + j) * 32 + lane < rows, (hkv, lens, run)
                    x += max(1, end - at)


def test_warps_have_read_all_places_before_one_changes():
    """Whether a CTA's parts become one is each warp's own reading of all warps' places, and decides who
    meets at the barriers behind: a warp that goes on to its next pair changes its place, so a
    barrier stands between the last such reading and the first change."""
    text = code("fk_q4_attn.cu")
    text = text[text.index("    q4_attn_kernel("):]
    last = max(m.start() for m in re.finditer(r"places\[(?:0|1|w)\]|ends\[w\]",
                                              text[:text.index("auto look_up")]))
    change = text.index("places[warp] = now", last)
    between = text[last:change]
    assert "__syncthreads();" in between
    assert "return" not in between[:between.index("__syncthreads();")]
