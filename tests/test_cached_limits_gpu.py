"""Paged attention and the delta-rule walk at the ends of what their documentation allows: any number of query heads
a KV head, any hint, scales of rows that a query may not see, lengths outside the stated bounds.  Bounds as derived
in test_cached_gpu.py; what a test adds to them is derived beside it."""
import pytest
import torch

from oracle import cached as O
from test_cached_gpu import BF, Cache, HEADS, attn_check, cu_of, delta_check, delta_inputs, gen, state_check

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from fastdecisions_b200 import _lib, ops


def attend(c, q, q_lens, max_seqlen=None, max_kv_len=None, code=0):
    """The call into an output of NaN, so that a row nobody wrote shows."""
    dev, kw = c.dev()
    out = torch.full(q.shape, float("nan"), dtype=BF, device="cuda")
    ops.paged_gqa_attention(q.cuda(), *dev, cu_of(q_lens).cuda(), c.kv_lens.cuda(),
                            max(q_lens) if max_seqlen is None else max_seqlen, max_kv_len, out=out, **kw)
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == code
    return out


def oracle(c, q, q_lens):
    return O.paged_attention(q, c.cache[0], c.cache[1], c.table, cu_of(q_lens), c.kv_lens.tolist(), c.scale[0], c.scale[1])


def queries(q_lens, hq, D, seed):
    return torch.randn(sum(q_lens), hq, D, generator=gen(seed)).to(BF)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("group", [65, 80, 128])
def test_attention_one_token_a_tile(group, D, quant):
    # 65 to 128 query heads on one KV head: a tile holds one token (at head_dim 256 a CTA too), in calls that
    # the device sorts, without parts, with parts and with 64 segments
    n = 100 if D == 256 else 200
    for q_lens, kv in (([200], [230]), ([n], [3000]), ([4, 3] * 32, [4 + 17 * i % 200 for i in range(64)])):
        c = Cache(kv, 1, D, 16, quant, group + D)
        q = queries(q_lens, group, D, 1)
        attn_check(attend(c, q, q_lens), oracle(c, q, q_lens), quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("group,D", [(130, 128), (200, 256)])
def test_attention_more_heads_than_a_tile(group, D, quant):
    q_lens, kv = [1, 2, 3], [70, 2, 900]
    c = Cache(kv, 1, D, 16, quant, group)
    q = queries(q_lens, group, D, 2)
    attn_check(attend(c, q, q_lens), oracle(c, q, q_lens), quant)
