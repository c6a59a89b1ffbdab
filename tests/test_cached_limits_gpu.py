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


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("D,n", [(128, 600), (256, 300)])
def test_attention_hint_shorter_than_the_contexts(D, n, quant):
    # 32 heads a KV head, more tiles than SMs: sorted on the device, and too much work for parts to pay
    for q_lens, kv in (([n], [1500]), ([n, 40, 7], [1400, 1500, 900])):
        c = Cache(kv, 2, D, 64, quant, D)
        q = queries(q_lens, 64, D, 3)
        ref = oracle(c, q, q_lens)
        for hint in (1, 750):
            attn_check(attend(c, q, q_lens, max_kv_len=hint), ref, quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:2])
def test_attention_hint_shorter_than_the_contexts_in_parts(hq, hkv, D, quant):
    # parts cut by the host, parts cut by the device, and neither
    for q_lens, kv in (([70, 30], [2500, 60]), ([500, 40, 0, 350, 64, 290, 1, 333], [530, 4500, 9, 3000, 64, 100, 2500, 333])):
        c = Cache(kv, hkv, D, 64, quant, D + 1)
        q = queries(q_lens, hq, D, 4)
        ref = oracle(c, q, q_lens)
        for hint in (1, max(kv) // 2, 100000):
            attn_check(attend(c, q, q_lens, max_kv_len=hint), ref, quant)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_replay_with_contexts_beyond_the_captured_hint(quant):
    q_lens = [600]
    c = Cache([1500], 2, 128, 64, quant, 5)
    dev, kw = c.dev()
    q = queries(q_lens, 64, 128, 5)
    qd, cu, lens = q.cuda(), cu_of(q_lens).cuda(), torch.tensor([640], dtype=torch.int32, device="cuda")
    ops.paged_gqa_attention(qd, *dev, cu, lens, 600, 640, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_gqa_attention(qd, *dev, cu, lens, 600, 640, **kw)
    for kv in (640, 1500, 1000):
        lens.fill_(kv)
        graph.replay()
        torch.cuda.synchronize()
        assert _lib.poll_device_error() == 0
        attn_check(out, O.paged_attention(q, *c.cache, c.table, cu_of(q_lens), [kv], *c.scale), quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D,most,per", [(16, 4, 128, 200, 64), (8, 2, 256, 100, 32)])
def test_attention_segment_longer_than_the_bound(hq, hkv, D, most, per, quant):
    # in a call that the device sorts, the rows of the other segments and its own up to the bound are right, the
    # error bit is set and rows behind the bound's last tile are left as they were
    q_lens = [700] + [most] * 11 + [most // 2] * (0 if D == 128 else 13)
    for kv in ([1600] + [most + 3 * i for i in range(len(q_lens) - 1)], [700 + 3900] + [most + 70 * i for i in range(len(q_lens) - 1)]):
        c = Cache(kv, hkv, D, 64, quant, 12)
        q = queries(q_lens, hq, D, 9)
        o = attend(c, q, q_lens, max_seqlen=most, code=32)
        ref = oracle(c, q, q_lens)
        attn_check(o[700:], ref, quant, rows=slice(700, None))
        attn_check(o[:most], ref, quant, rows=slice(0, most))
        assert o[-(-most // per) * per:700].isnan().all()


@pytest.mark.parametrize("quant", [False, True])
def test_attention_bound_is_exact(quant):
    # a segment of one token more sets the error bit in either kernel, one at the bound does not
    for q_lens, kv in (([2, 1, 2], [60, 5000, 2]), ([9, 70, 1], [80, 70, 4000])):
        c = Cache(kv, 4, 128, 16, quant, 13)
        q = queries(q_lens, 16, 128, 10)
        attn_check(attend(c, q, q_lens), oracle(c, q, q_lens), quant)
        attend(c, q, q_lens, max_seqlen=max(q_lens) - 1, code=32)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_bound_of_zero(quant):
    c = Cache([60, 20], 4, 128, 16, quant, 14)
    q = queries([2, 1], 16, 128, 11)
    attend(c, q, [2, 1], max_seqlen=0, code=32)
    assert attend(c, q, [0, 0], max_seqlen=0).isnan().all()  # padding only


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:2])
@pytest.mark.parametrize("q_lens,kv", [([1, 2, 1], [90, 5, 700]), ([1], [1500]), ([1], [9000]), ([70, 9], [80, 9]), ([70], [6000])])
def test_attention_nan_queries_and_keys_show(q_lens, kv, hq, hkv, D, quant):
    # a query of NaN, and a query that meets a NaN key, give NaN in each kernel and in each join of parts; the others
    # are what they are without
    c = Cache(kv, hkv, D, 64, quant, 19)
    q = queries(q_lens, hq, D, 17)
    ref = oracle(c, q, q_lens)
    T = sum(q_lens)
    q[T - 1, hq - 1] = float("nan")
    q[0, 0, 5] = float("nan")
    o = attend(c, q, q_lens)
    assert o[T - 1, hq - 1].isnan().all() and o[0, 0].isnan().all()
    rest = torch.ones(T, hq, dtype=torch.bool)
    rest[T - 1, hq - 1] = rest[0, 0] = False
    attn_check(o.cpu()[rest], tuple(t[rest] for t in ref), quant)
    q = queries(q_lens, hq, D, 17)
    last = kv[-1] - 1                                     # seen by the last token only
    c.cache[0][int(c.table[-1, last // 64]), 0, last % 64] = float("nan")
    o = attend(c, q, q_lens)
    assert o[T - 1, :hq // hkv].isnan().all()
    rest = torch.ones(T, hq, dtype=torch.bool)
    rest[T - 1, :hq // hkv] = False
    attn_check(o.cpu()[rest], tuple(t[rest] for t in ref), quant)


@pytest.mark.parametrize("q_lens,kv", [([2, 1], [90, 7]), ([1], [1500]), ([1], [9000]), ([60, 50], [90, 70]), ([60, 50], [1900, 70])])
def test_attention_rows_near_the_largest_number(q_lens, kv):
    # V rows of 2^113 times e4m3: sums of weights times V leave float32, their quotients do not
    c = Cache(kv, 4, 128, 16, True, 16)
    for s, length in enumerate(kv):
        pos = torch.arange(length)
        c.scale[1][c.table[s].long()[pos // 16], :, pos % 16] = 240
    q = queries(q_lens, 16, 128, 16)
    attn_check(attend(c, q, q_lens), oracle(c, q, q_lens), True)


def scales_check(o, c, q, q_lens):
    """attn_check's bound and, for an 8-bit cache, one term more.

    More than 32 rows a KV head: V rows are fp16 in units of 2^-7 of the largest scale that the CTA reads.  Where the
    segment's scales lie within 2^31 of each other, an element is off by at most half of fp16's smallest step, 2^-25
    of that unit; else rows of smaller scales may read as zero, elements of at most 448 times 2^-32.  A mean of them is
    off by no more.  Weights are fp16 with the row's largest at 2^6 or above: off by at most half the smallest step,
    2^-31 of the largest weight, each times its |v|.

    Up to 32 rows: P is fp16 times a power of two a row, so that the row's largest contribution p 2^(scale) is at
    least 2^6: a weight is off by at most 2^-31 of that contribution, times the e4m3 value it meets."""
    want, mag, size = oracle(c, q, q_lens)
    if c.quant:
        T, hq, D = q.shape
        rep, cu = hq // c.hkv, cu_of(q_lens)
        tail = torch.zeros(T, hq, D, dtype=torch.float64)
        for s, n in enumerate(q_lens):
            length = int(c.kv_lens[s])
            k = O.cache_rows(c.cache[0], c.scale[0], c.table[s], length)
            v8 = O.cache_rows(c.cache[1], torch.full_like(c.scale[1], 127), c.table[s], length).abs()
            pos = torch.arange(length)
            scale = torch.exp2(c.scale[1][c.table[s].long()[pos // c.page], :, pos % c.page].double() - 127)
            for i in range(n):
                t, seen = int(cu[s]) + i, length - n + i + 1
                for h in range(hq if seen > 0 else 0):
                    sc, v = scale[:, h // rep], v8[:seen, h // rep]
                    p = torch.softmax(k[:seen, h // rep] @ q[t, h].double() * D ** -0.5, 0)
                    if max(q_lens) * rep > 32:
                        lost = 2.0 ** -32 * sc.max() * (1 if sc.max() <= 2 ** 31 * sc.min() else 448)
                        tail[t, h] = lost + 2.0 ** -31 * p.max() * (v * sc[:seen, None]).sum(0)
                    else:
                        tail[t, h] = 2.0 ** -31 * (p * sc[:seen]).max() * v.sum(0)
        mag = mag + tail / 2 ** -11
    attn_check(o, (want, mag, size), c.quant)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("up", [0, 14, 21, 24, 30, 40])
def test_attention_many_rows_behind_large_scales(hq, hkv, D, quant, up):
    # the last token's V row is larger than the others by 2^up; first seen by itself only, then by every row
    n = 33 * hkv // hq + 1
    for q_lens, kv, at in (([n, n + 3, n + 1], [n, n + 90, n + 20], -1), ([n, n], [n + 200, n + 9], 3)):
        c = Cache(kv, hkv, D, 16, quant, D + up)
        for s, length in enumerate(kv):
            pos = at % length
            page = int(c.table[s, pos // 16])
            if quant:
                c.scale[1][page, :, pos % 16] += up
            else:
                c.cache[1][page, :, pos % 16] *= 2.0 ** up
        q = queries(q_lens, hq, D, 15)
        scales_check(attend(c, q, q_lens), c, q, q_lens)


def test_attention_many_rows_smallest_and_largest_scales():
    # scale bytes at both ends of what a write leaves
    for byte in (0, 1, 2, 30, 240):
        for kv in ([90, 70], [1900, 70]):
            c = Cache(kv, 4, 128, 16, True, 16)
            for s, length in enumerate(kv):
                pos = torch.arange(length)
                c.scale[1][c.table[s].long()[pos // 16], :, pos % 16] = byte
            q = queries([60, 50], 16, 128, 16)
            o = attend(c, q, [60, 50])
            want = oracle(c, q, [60, 50])[0]
            # bf16 of this size may be subnormal: half a step of 2^-133 besides the relative bound
            assert ((o.double().cpu() - want).abs() <= 2 ** -7 * want.abs().amax(-1, keepdim=True) + 2.0 ** -134).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("up", [12, 24, 60, 100])
def test_attention_few_rows_behind_hidden_scales(hq, hkv, D, quant, up):
    # the last token's V row, which the others may not see, is larger than theirs by 2^up: their results are
    # what they are without it
    for q_lens, past in (([2, 4, 3, 1], 0), ([2, 8, 1, 5], 70)):
        kv = [n + past for n in q_lens]
        c = Cache(kv, hkv, D, 16, quant, D + up)
        for s, n in enumerate(kv):
            page, off = int(c.table[s, (n - 1) // 16]), (n - 1) % 16
            if quant:
                c.scale[1][page, :, off] += up
            else:
                c.cache[1][page, :, off] *= 2.0 ** up
        q = queries(q_lens, hq, D, 6)
        scales_check(attend(c, q, q_lens), c, q, q_lens)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:3])
@pytest.mark.parametrize("spread", [6.0, 20.0])
def test_attention_few_rows_scales_far_apart(hq, hkv, D, quant, spread):
    # V rows of any size in any order; most of a result may come from keys of small weight and large rows
    for q_lens, kv in (([1, 3, 4, 1], [400, 333, 5, 64]), ([8, 1], [150, 1700]), ([1], [3000])):
        c = Cache(kv, hkv, D, 16, quant, 9, spread=spread, v_only=True)
        q = queries(q_lens, hq, D, 7)
        scales_check(attend(c, q, q_lens), c, q, q_lens)


def test_attention_few_rows_smallest_and_largest_scales():
    # scale bytes at both ends of what a write leaves
    for byte in (0, 1, 2, 240):
        c = Cache([90, 7], 4, 128, 16, True, 11)
        for s, n in enumerate((90, 7)):
            pos = torch.arange(n)
            c.scale[1][c.table[s].long()[pos // 16], :, pos % 16] = byte
            if byte < 240:
                c.scale[1][int(c.table[s, (n - 1) // 16]), :, 3] = byte + 1
        q = queries([2, 1], 16, 128, 8)
        o = attend(c, q, [2, 1])
        want = oracle(c, q, [2, 1])[0]
        # bf16 of this size may be subnormal: half a step of 2^-133 besides the relative bound
        assert ((o.double().cpu() - want).abs() <= 2 ** -7 * want.abs().amax(-1, keepdim=True) + 2.0 ** -134).all()


@pytest.mark.parametrize("q_lens", [[1], [40]])
def test_attention_longest_page_table(q_lens):
    # positions are counted in 32 bits with steps past the last one: tables that reach 2^31 are refused, the longest
    # allowed one works
    c = Cache([70], 4, 128, 256, True, 20)
    (k, v, table), kw = c.dev()
    q = queries(q_lens, 16, 128, 18)
    ref = oracle(c, q, q_lens)
    cu, lens = cu_of(q_lens).cuda(), c.kv_lens.cuda()
    for pages, ok in ((2 ** 23 - 1, False), (2 ** 23 - 2 ** 8 + 1, False), (2 ** 23 - 2 ** 8, True)):
        wide = torch.zeros(1, pages, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        if ok:
            attn_check(ops.paged_gqa_attention(q.cuda(), k, v, wide, cu, lens, q_lens[0], **kw), ref, True)
        else:
            with pytest.raises(ValueError, match="positions"):
                ops.paged_gqa_attention(q.cuda(), k, v, wide, cu, lens, q_lens[0], **kw)
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 0


@pytest.mark.parametrize("quant", [False, True])
def test_one_head_or_one_page_in_any_layout(quant):
    # a dimension of one element has no stride of its own
    c = Cache([100], 1, 128, 16, quant, 15)
    q = queries([3], 6, 128, 12)
    ref = oracle(c, q, [3])
    cu, lens = cu_of([3]).cuda(), c.kv_lens.cuda()

    def lay(t):  # [pages, page size, heads, ..] in memory, heads second as the operators take it
        m = torch.empty_strided(t.shape, (t.stride(0), t.stride(2)) + t.stride()[2:], dtype=t.dtype, device="cuda")
        return m.copy_(t)

    (_, _, table), _ = c.dev()
    k, v = (lay(t.view(torch.uint8)).view(t.dtype) for t in c.cache)
    kw = dict(k_scale=lay(c.scale[0]), v_scale=lay(c.scale[1])) if quant else {}
    attn_check(ops.paged_gqa_attention(q.cuda(), k, v, table, cu, lens, 3, **kw), ref, quant)
    x = torch.randn(3, 1, 128, generator=gen(16)).to(BF).cuda()
    ops.paged_kv_write(x, x, k, v, table, cu, lens, **kw)
    rk, rv = ops.paged_kv_read(k, v, table, cu, lens, 3, **kw)
    want = O.quantise(x.cpu())[1].to(BF) if quant else x.cpu()
    assert torch.equal(rk.cpu(), want) and torch.equal(rv.cpu(), want)
    one = Cache([9], 4, 128, 16, quant, 17)
    (k, v, table), kw = one.dev()
    page = int(one.table[0, 0])
    flat = lambda t: torch.as_strided(t[page:page + 1], t[:1].shape, (1,) + t.stride()[1:], t[page:page + 1].storage_offset())
    kw = {name: flat(t) for name, t in kw.items()}
    q = queries([2], 16, 128, 13)
    o = ops.paged_gqa_attention(q.cuda(), flat(k), flat(v), torch.zeros_like(table[:, :1]), cu_of([2]).cuda(), one.kv_lens.cuda(), 2, **kw)
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 0
    attn_check(o, oracle(one, q, [2]), quant)


def test_truth_value_that_cannot_be_taken():
    c = Cache([10], 4, 128, 16, False, 18)
    dev, _ = c.dev()
    q = queries([1], 16, 128, 14).cuda()
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_gqa_attention(q, *dev, cu_of([1]).cuda(), c.kv_lens.cuda(), 1, gate_interleaved=torch.zeros(2))
    assert torch.isfinite(ops.paged_gqa_attention(q, *dev, cu_of([1]).cuda(), c.kv_lens.cuda(), 1).float()).all()


@pytest.mark.parametrize("n", [1, 3, 8, 9, 21])
@pytest.mark.parametrize("decay", [0.0, -3.0, -30.0, -80.0, -200.0, float("-inf"), 20.0])
def test_delta_decays_of_any_size_and_length(decay, n):
    # walked token by token (up to 8) and in batches: extreme decays among the first eight tokens, several in a row;
    # growth passes 1e18 on the way
    H = 3
    for place in ([0], [0, 1, 2], [1, 2, 4, 5, 7], [2, 7, 8, 20]):
        q, k, v, g, beta = delta_inputs(n, H, H, 90 + n)
        at = [i for i in place if i < n]
        g[0, at[:3] if decay > 0 else at] = decay
        pool = torch.randn(2, H, 128, 128, generator=gen(91)) * 0.5
        d = pool.cuda()
        idx = lambda i: torch.tensor([i], dtype=torch.int32).cuda()
        o = ops.recurrent_gated_delta_rule_(q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), d, idx(0), idx(1))
        torch.cuda.synchronize()
        assert _lib.poll_device_error() == 0
        want, states = O.recurrent_delta(q[0], k[0], v[0], g[0], beta[0], pool[:1], [0, n])
        delta_check(o[0], want)
        state_check(d[1:], states)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("q_lens,kv", [([1] * 20, [700] * 20), ([100], [4500]), ([70, 30, 5], [4500, 60, 900])])
def test_attention_workspace_for_loose_bounds(q_lens, kv, quant):
    # a workspace as the size function gives it serves the call with the same arguments, also where they exceed what
    # the tensors hold
    c = Cache(kv, 4, 128, 64, quant, 21)
    dev, kw = c.dev()
    q = queries(q_lens, 16, 128, 19)
    ref = oracle(c, q, q_lens)
    reach = dev[2].shape[1] * 64
    for max_seqlen in (max(q_lens), 5000, 2 ** 40):
        for hint in (None, 1, max(kv), 10000, 2 ** 20, 2 ** 40):
            need = ops.paged_gqa_workspace_bytes(len(q_lens), max_seqlen, reach if hint is None else hint, sum(q_lens), 16, 4, 128,
                                                 quant)
            ws = torch.empty(need, dtype=torch.uint8, device="cuda")
            o = ops.paged_gqa_attention(q.cuda(), *dev, cu_of(q_lens).cuda(), c.kv_lens.cuda(), max_seqlen, hint, workspace=ws, **kw)
            attn_check(o, ref, quant)
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 0
