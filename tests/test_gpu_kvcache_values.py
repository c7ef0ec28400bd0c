"""4-bit caches on the GPU: values that are no numbers."""
import numpy as np
import pytest

import kvcache_oracle as S
from gpu_util import dev, host_f32
from test_gpu_kvcache_small import Batch, check_sums, ints, weight_error

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
    2^-25 where the largest weight times scale is 2^5 at least; sums of products in fp32, 2^-22 of the
    whole each."""
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
    tol = np.abs(out) * 2.0 ** -8 + low * rel + step * (2.0 ** -11 + rel + keys * 2.0 ** -30)
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
