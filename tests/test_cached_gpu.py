"""Operators that continue sequences from cached state, against float64 on the CPU.

Tolerances, derived before the first run (half a step of bf16 is 2^-8 of the value, of fp16 2^-11):
* cache rows: exact (the scale is a power of two, the only rounding is the one to e4m3);
* attention: the output's rounding (2^-8 |o|) plus the rounding of the softmax weights (2^-8 of
  sum p |v|; the 8-bit cache rounds them to fp16, 2^-11), plus 2^-10 of sum p |v| for float32: scores
  here stay below 32 in magnitude as sums of 128 or 256 products, so their float32 error is below
  256 * 2^-24 * 32 = 2^-11, and exp2's is 2^-22;
* delta rule: 2^-8 |o|, and 2e-5 of the largest magnitude for float32 sums over 128 terms and up to 70
  steps (70 * 2 * 128 * 2^-24 = 1e-3 if every rounding had one sign; random signs leave its square root
  of the count, 134 * 2^-24 * 2 < 2e-5);
* conv: 2^-8 |y|, and the hardware tanh's 2^-10.9 of |x| / 2 (silu = h + h tanh h, h = x / 2).
"""
import math

import pytest
import torch

from oracle import cached as O

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from fastdecisions_b200 import _lib, ops

BF = torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def no_error():
    torch.cuda.synchronize()
    return _lib.poll_device_error() == 0


def cu_of(lens):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.int64).cumsum(0)), dtype=torch.int32)


class Cache:
    """CPU tensors of a paged cache filled with random rows; unused rows and pages hold NaN."""

    def __init__(self, kv_lens, hkv, D, page, quant, seed, shared=0, spread=0.0, v_only=False):
        g = gen(seed)
        S = len(kv_lens)
        need = [max(0, (x + page - 1) // page - shared) for x in kv_lens]
        total = shared + sum(need) + 2
        order = torch.randperm(total, generator=g)
        self.table = torch.full((S, max([shared + n for n in need] + [1]) + 1), -7, dtype=torch.int32)
        at = shared
        for s in range(S):
            self.table[s, :shared] = order[:shared].int()
            self.table[s, shared:shared + need[s]] = order[at:at + need[s]].int()
            at += need[s]
        used = torch.zeros(total, page, dtype=torch.bool)
        for s, n in enumerate(kv_lens):
            pos = torch.arange(n)
            used[self.table[s].long()[pos // page], pos % page] = True
        self.kv_lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.page, self.D, self.hkv, self.quant = page, D, hkv, quant
        self.scale = [None, None]
        self.cache = []
        for i in range(2):
            x = torch.randn(total, hkv, page, D, generator=g)
            if spread and (i == 1 or not v_only):
                x = x * torch.exp(spread * torch.randn(total, hkv, page, 1, generator=g))
            x = x.to(BF)
            if quant:
                e, val = O.quantise(x)
                q8 = (val / O.power_of_two(e)[..., None]).float().to(torch.float8_e4m3fn)
                q8.view(torch.uint8).masked_fill_(~used[:, None, :, None], 0x7f)
                self.scale[i] = (e + 127).to(torch.uint8).masked_fill(~used[:, None, :], 255)
                self.cache.append(q8)
            else:
                self.cache.append(x.masked_fill(~used[:, None, :, None], float("nan")))

    def dev(self, interleaved=False):
        """Device arguments; ``interleaved`` keeps K and V pages in one pool (page stride twice a page)."""
        kw = {}
        if interleaved:
            pool = torch.stack([c.view(torch.uint8 if self.quant else torch.int16) for c in self.cache], 1).cuda()
            k, v = (pool[:, i].view(self.cache[0].dtype) for i in range(2))
            if self.quant:
                sp = torch.stack(self.scale, 1).cuda()
                kw = dict(k_scale=sp[:, 0], v_scale=sp[:, 1])
        else:
            k, v = (c.cuda() for c in self.cache)
            if self.quant:
                kw = dict(k_scale=self.scale[0].cuda(), v_scale=self.scale[1].cuda())
        return (k, v, self.table.cuda()), kw


def attn_check(o, ref, quant, gate=None, rows=slice(None)):
    want, mag, size = (t[rows] for t in ref)
    sig = 1.0 if gate is None else torch.sigmoid(gate.double())
    # Where scores are not small (rows scaled by many powers of two): a score is a float32 sum of D
    # products, off by at most dz = D * 2^-23 * size, so a weight relative to the sum of weights is off
    # by at most a factor exp(2 dz), and the output by expm1(2 dz) (mag + |o|).  With size <= 32 this is
    # below the 2^-10 of the header.
    dz = want.shape[-1] * 2.0 ** -23 * size
    fp32 = torch.expm1(2 * dz).clamp_max(1e30) * (mag + want.abs())
    bound = 2 ** -8 * want.abs() + (2 ** -11 if quant else 2 ** -8) * mag + torch.maximum(2 ** -10 * mag, fp32)
    want, bound = want * sig, bound * sig
    err = (o.double().cpu() - want).abs()
    assert torch.isfinite(o.float()).all()
    worst = (err - bound).max().item()
    assert worst <= 1e-6, f"error exceeds its bound by {worst}, largest error {err.max().item()}"


def run_attn(q_lens, kv_lens, hq, hkv, D, page, quant, seed=1, gate=False, interleaved=False, shared=0, spread=0.0,
             q_scale=1.0, max_kv_len=None, strided=False, v_only=False, gate_scale=1.0):
    c = Cache(kv_lens, hkv, D, page, quant, seed, shared, spread, v_only)
    T = sum(q_lens)
    g = gen(seed + 1)
    q = (torch.randn(T, hq, D, generator=g) * q_scale).to(BF)
    gt = (torch.randn(T, 2 * hq * D, generator=g) * gate_scale).to(BF) if gate else None
    cu = cu_of(q_lens)
    dev, kw = c.dev(interleaved)
    qd = q.cuda()
    if strided:  # rows inside a wider projection
        wide = torch.full((T, hq * D + 64), float("nan"), dtype=BF, device="cuda")
        wide[:, :hq * D] = qd.reshape(T, -1)
        qd = wide[:, :hq * D].unflatten(1, (hq, D))
    if gate:  # head stride 2 D, as the attention projection holds it
        kw.update(gate=gt.cuda()[:, D:], gate_interleaved=True)
    o = ops.paged_gqa_attention(qd, *dev, cu.cuda(), c.kv_lens.cuda(), max(q_lens + [0]), max_kv_len, **kw)
    ref = O.paged_attention(q, c.cache[0], c.cache[1], c.table, cu, kv_lens, c.scale[0], c.scale[1])
    assert no_error()
    attn_check(o, ref, quant, gt.reshape(T, hq, 2, D)[:, :, 1] if gate else None)


HEADS = [(16, 4, 128), (8, 2, 256), (6, 1, 128), (4, 4, 256), (10, 2, 128)]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("page", [16, 64])
def test_attention_decode(hq, hkv, D, page, quant):
    # one token a sequence: a single key, tile and page borders on both sides, several splits
    kv = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1111]
    run_attn([1] * len(kv), kv, hq, hkv, D, page, quant, seed=hq + page)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:3])
def test_attention_chunks(hq, hkv, D, quant):
    # a few to many new tokens, with and without history, row blocks that end inside a token's heads
    q = [1, 3, 5, 8, 17, 33, 64, 70, 150]
    kv = [1, 3, 300, 9, 17, 200, 64, 71, 700]
    run_attn(q, kv, hq, hkv, D, 32, quant, seed=7, gate=True)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS)
@pytest.mark.parametrize("most", [4, 8, 16])
def test_attention_few_tokens(hq, hkv, D, quant, most):
    # 16, 32 and 64 rows a CTA at four heads a group
    q = [1, most, 2, most - 1, 3]
    run_attn(q, [1, most, 200, 90, 1000], hq, hkv, D, 16, quant, seed=most, gate=True)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS + [(12, 1, 128), (7, 1, 256)])
def test_attention_many_tokens(hq, hkv, D, quant):
    # full and ragged row tiles, a second tile without rows, blocks that end inside a page or at kv_lens
    q = [64, 65, 33, 128, 1, 257, 0]
    run_attn(q, [64, 321, 33, 1000, 700, 260, 9], hq, hkv, D, 16, quant, seed=hq)
    run_attn([200], [201], hq, hkv, D, 128, quant, seed=hq + 1, interleaved=True, strided=True, gate=True)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:2])
def test_attention_many_tokens_split_keys(hq, hkv, D, quant):
    # few row tiles behind a long history: keys split over CTAs, some parts without a visible key
    run_attn([100], [6000], hq, hkv, D, 64, quant, seed=40, gate=True)
    run_attn([70, 30], [4500, 60], hq, hkv, D, 32, quant, seed=41)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:2])
def test_attention_many_tokens_parts_cut_on_the_device(hq, hkv, D, quant):
    # enough tiles for the part size to follow from the lengths, with contexts and tiles far from even;
    # a segment of more tokens than positions, empty ones, and even lengths, where nothing is split
    n = [500, 40, 0, 350, 64, 290, 1, 333]
    run_attn(n, [530, 4500, 9, 3000, 64, 100, 2500, 333], hq, hkv, D, 64, quant, seed=42, gate=True)
    run_attn(n, [500, 40, 0, 350, 64, 290, 1, 333], hq, hkv, D, 32, quant, seed=43)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hq,hkv,D", [(6, 1, 128), (10, 2, 128), (4, 4, 256), (7, 1, 256)])
def test_attention_most_segments_the_device_sorts(hq, hkv, D, quant):
    # 64 segments, groups that do not divide a tile, contexts shorter than the tokens among them
    n = [37 * i % 90 for i in range(64)]
    kv = [max(x + 311 * i % 1300 - 20, 0) for i, x in enumerate(n)]
    run_attn(n, kv, hq, hkv, D, 64, quant, seed=47, gate=hkv == 2)


@pytest.mark.parametrize("n,kv", [([1, 2, 3], [700, 40, 9]), ([1], [5000]), ([80, 33], [90, 333]), ([70], [6000])])
@pytest.mark.parametrize("hq,hkv,D", HEADS[:2])
def test_attention_gates_of_any_size(n, kv, hq, hkv, D):
    # sigmoids from 0 to 1, infinite gates among them, in each kernel and in the join of parts
    run_attn(n, kv, hq, hkv, D, 64, False, seed=45, gate=True, gate_scale=60.0)
    run_attn(n, kv, hq, hkv, D, 64, False, seed=46, gate=True, gate_scale=3e38)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_many_segments_split_keys(quant):
    n = [33 if i % 7 else 1 for i in range(66)]
    run_attn(n, [x + 23 * i for i, x in enumerate(n)], 6, 1, 128, 32, quant, seed=44)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_empty_rows_and_segments(quant):
    # no tokens; no keys; more tokens than positions (the first ones see nothing and give zeros)
    run_attn([0, 4, 0, 6, 1, 2], [10, 0, 0, 3, 0, 2], 16, 4, 128, 16, quant, seed=3)
    run_attn([0, 90, 0, 100], [10, 0, 5, 33], 16, 4, 128, 16, quant, seed=4)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_attention_pages_and_strides(page, quant):
    run_attn([1, 40, 7], [777, 300, 256], 16, 4, 128, page, quant, seed=page, interleaved=True, strided=True, gate=True)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_shared_prefix_pages(quant):
    n = [5, 1, 30, 12]
    run_attn(n, [16 * 20 + 3 + x for x in n], 8, 2, 256, 16, quant, seed=9, shared=20)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_one_long_sequence_many_splits(quant):
    run_attn([1], [9001], 16, 4, 128, 64, quant, seed=12)
    run_attn([3], [5000], 8, 2, 256, 64, quant, seed=13, max_kv_len=1)  # the hint may be wrong


def test_attention_row_scales_far_apart():
    # V rows whose scales differ by many powers of two, in both orders of appearance
    run_attn([1, 9, 40], [400, 333, 500], 16, 4, 128, 16, True, seed=14, spread=6.0)
    for quant in (False, True):  # and with scores that stay small, so that every weight counts
        run_attn([1, 9, 40], [400, 333, 500], 16, 4, 128, 16, quant, seed=16, spread=6.0, v_only=True)


def test_attention_sharp_scores():
    # scores of about +-28: the running maximum moves a lot and most weights vanish
    run_attn([1, 20], [900, 600], 16, 4, 128, 64, False, seed=15, q_scale=6.0)
    run_attn([1, 20], [900, 600], 16, 4, 128, 64, True, seed=15, q_scale=6.0)


def test_attention_rows_behind_the_last_segment_untouched():
    c = Cache([50, 20], 4, 128, 16, False, 21)
    dev, kw = c.dev()
    q = torch.randn(12, 16, 128, generator=gen(2)).to(BF).cuda()
    for max_kv in (50, 4096):  # without and with a split
        out = torch.full((12, 16, 128), 7.0, dtype=BF, device="cuda")
        ops.paged_gqa_attention(q, *dev, torch.tensor([0, 4, 7], dtype=torch.int32).cuda(), c.kv_lens.cuda(), 4,
                                max_kv, out=out)
        assert no_error()
        assert (out[7:] == 7.0).all() and not (out[:7] == 7.0).all()


@pytest.mark.parametrize("quant", [False, True])
def test_attention_bad_metadata_is_contained(quant):
    c = Cache([100, 60, 40], 4, 128, 16, quant, 22)
    dev, kw = c.dev()
    q = torch.randn(9, 16, 128, generator=gen(3)).to(BF)
    ref = O.paged_attention(q, c.cache[0], c.cache[1], c.table, cu_of([3, 3, 3]), [100, 60, 40], *c.scale)

    def call(table=None, cu=(0, 3, 6, 9), lens=(100, 60, 40)):
        o = ops.paged_gqa_attention(q.cuda(), dev[0], dev[1], dev[2] if table is None else table.cuda(),
                                    torch.tensor(cu, dtype=torch.int32).cuda(),
                                    torch.tensor(lens, dtype=torch.int32).cuda(), 3, 100, **kw)
        torch.cuda.synchronize()
        return o, _lib.poll_device_error()

    for bad in (-1, 10 ** 6, 2 ** 31 - 1):  # page ids outside the cache: the other segments are right
        t = c.table.clone()
        t[1, 1] = bad
        o, code = call(table=t)
        assert code == 32
        attn_check(o[:3], ref, quant, rows=slice(0, 3))
        attn_check(o[6:], ref, quant, rows=slice(6, 9))
    o, code = call(lens=(100, -5, 10 ** 9))  # lengths outside the table: no keys
    assert code == 32 and (o[3:] == 0).all()
    attn_check(o[:3], ref, quant, rows=slice(0, 3))
    o, code = call(cu=(0, 3, 2, 9))  # a decreasing range counts as empty
    assert code == 32
    attn_check(o[:2], ref, quant, rows=slice(0, 2))  # row 2 belongs to two ranges here
    assert call()[1] == 0


def test_attention_refusals():
    c = Cache([10], 4, 128, 16, False, 23)
    (k, v, table), _ = c.dev()
    q = torch.zeros(1, 16, 128, dtype=BF, device="cuda")
    cu, lens = torch.tensor([0, 1], dtype=torch.int32).cuda(), c.kv_lens.cuda()
    ok = lambda **kw: ops.paged_gqa_attention(**{**dict(q=q, k_cache=k, v_cache=v, page_table=table, cu_seqlens=cu,
                                                        kv_lens=lens, max_seqlen=1), **kw})
    ok()
    bad = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.cpu()), dict(k_cache=k.float()), dict(k_cache=k[:, :, :8]),
           dict(v_cache=v[:1]), dict(page_table=table.long()), dict(page_table=table[:, :0]), dict(cu_seqlens=cu.long()),
           dict(cu_seqlens=cu[:1]), dict(kv_lens=lens.long()), dict(max_seqlen=-1),
           dict(k_scale=torch.zeros(k.shape[:3], dtype=torch.uint8, device="cuda")),
           dict(k_cache=k.to(torch.float8_e4m3fn), v_cache=v.to(torch.float8_e4m3fn)),
           dict(out=torch.zeros(1, 16, 64, dtype=BF, device="cuda")),
           dict(gate=torch.zeros(1, 16 * 128, dtype=BF, device="cuda"), gate_interleaved=True),
           dict(k_cache=k.transpose(1, 2).contiguous().transpose(1, 2)),
           dict(q=torch.zeros(1, 16, 129, dtype=BF, device="cuda")[:, :, 1:]),
           dict(q=torch.zeros(130 + 16 * 128, dtype=BF, device="cuda")[1:1 + 16 * 128].view(1, 16, 128))]
    for kw in bad:
        with pytest.raises(ValueError):
            ok(**kw)
    big = Cache([5000], 4, 128, 16, False, 23)
    (k2, v2, t2), _ = big.dev()
    with pytest.raises(ValueError, match="workspace"):
        ok(k_cache=k2, v_cache=v2, page_table=t2, kv_lens=big.kv_lens.cuda(),
           workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))


def test_attention_graph_replay_with_other_lengths_and_stream():
    c = Cache([700, 300], 4, 128, 64, True, 31)
    dev, kw = c.dev()
    q = torch.randn(2, 16, 128, generator=gen(5)).to(BF)
    qd, cu, lens = q.cuda(), cu_of([1, 1]).cuda(), c.kv_lens.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_gqa_attention(qd, *dev, cu, lens, 1, 704, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_gqa_attention(qd, *dev, cu, lens, 1, 704, **kw)
    for kv in ([700, 300], [1, 299], [640, 64], [0, 1]):
        lens.copy_(torch.tensor(kv, dtype=torch.int32))
        graph.replay()
        assert no_error()
        attn_check(out, O.paged_attention(q, *c.cache, c.table, cu_of([1, 1]), kv, *c.scale), True)


@pytest.mark.parametrize("quant", [False, True])
def test_attention_graph_replay_of_parts_cut_on_the_device(quant):
    # the part size follows the lengths of each replay; token counts and contexts change, the second stream
    # runs a call of its own meanwhile
    n, kv = [500, 40, 0, 350, 64, 290, 1, 333], [530, 4500, 9, 3000, 64, 100, 2500, 333]
    c = Cache([4600] * 8, 4, 128, 64, quant, 51)
    dev, kw = c.dev()
    T = sum(n)
    q = torch.randn(T, 16, 128, generator=gen(6)).to(BF)
    qd, cu, lens = q.cuda(), cu_of(n).cuda(), torch.tensor(kv, dtype=torch.int32, device="cuda")
    ops.paged_gqa_attention(qd, *dev, cu, lens, 500, 4600, **kw)
    torch.cuda.synchronize()
    graph, other, side = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = ops.paged_gqa_attention(qd, *dev, cu, lens, 500, 4600, **kw)
    with torch.cuda.graph(other):
        out2 = ops.paged_gqa_attention(qd, *dev, cu, lens, 500, 4600, **kw)
    for n2, kv2 in ((n, kv), ([200] * 7 + [178], [4600] * 8), ([500, 500, 500, 78, 0, 0, 0, 0], [501, 500, 499, 4000, 0, 7, 0, 1]),
                    ([1] * 8, [4600, 1, 2, 3, 4, 5, 6, 7])):
        cu.copy_(cu_of(n2))
        lens.copy_(torch.tensor(kv2, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other.replay()
        assert no_error()
        ref = O.paged_attention(q, c.cache[0], c.cache[1], c.table, cu_of(n2), kv2, c.scale[0], c.scale[1])
        rows = slice(0, sum(n2))
        attn_check(out[rows], ref, quant, rows=rows)
        attn_check(out2[rows], ref, quant, rows=rows)


# --------------------------------------------------------------------------- cache write and read
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("hkv,D,page", [(4, 128, 64), (2, 256, 16), (1, 128, 32), (3, 256, 128), (5, 128, 256)])
def test_cache_write_and_read(hkv, D, page, quant):
    q_lens, kv_lens = [1, 0, 70, 5, 33], [40, 17, 70, 261, 600]
    c = Cache(kv_lens, hkv, D, page, quant, seed=hkv * D)
    T = sum(q_lens)
    g = gen(6)
    k = (torch.randn(T, hkv, D, generator=g) * torch.exp(3 * torch.randn(T, hkv, 1, generator=g))).to(BF)
    v = (torch.randn(T, hkv, D, generator=g) * torch.exp(3 * torch.randn(T, hkv, 1, generator=g))).to(BF)
    k[3, 0], v[4, 0], k[7, 0, 1:] = 0, 0, 0          # zero rows, one-element rows
    k[8, 0] = 448.0                                    # exactly at the border of a scale
    v[9, 0, 0], v[10, 0] = 3e38, 2.0 ** -130           # the largest scale, subnormal bf16
    v[9, 0, 1:] = 0
    (kc, vc, table), kw = c.dev(interleaved=True)
    before = [t.view(torch.uint8).clone() for t in (kc, vc)]
    cu = cu_of(q_lens)
    wide = torch.full((T, 2 * hkv * D + 8), float("nan"), dtype=BF, device="cuda")  # v inside a projection
    wide[:, 8:8 + hkv * D] = v.cuda().reshape(T, -1)
    vd = wide[:, 8:8 + hkv * D].unflatten(1, (hkv, D))
    ops.paged_kv_write(k.cuda(), vd, kc, vc, table, cu.cuda(), c.kv_lens.cuda(), **kw)
    rk, rv = ops.paged_kv_read(kc, vc, table, cu.cuda(), c.kv_lens.cuda(), T, **kw)
    assert no_error()
    for x, r in ((k, rk), (v, rv)):
        want = O.quantise(x)[1].to(BF) if quant else x
        assert torch.equal(r.cpu(), want)
    # every other row of the cache is as it was
    touched = torch.zeros(kc.shape[0], page, dtype=torch.bool)
    for s, (n, length) in enumerate(zip(q_lens, kv_lens)):
        pos = torch.arange(length - n, length)
        touched[c.table[s].long()[pos // page], pos % page] = True
    keep = ~touched[:, None, :, None].cuda()
    for t, b in zip((kc, vc), before):
        now = t.view(torch.uint8)
        assert torch.equal(now.masked_fill(~keep, 0), b.masked_fill(~keep, 0))
    # whole contexts
    full = cu_of(kv_lens)
    rk, rv = ops.paged_kv_read(kc, vc, table, full.cuda(), c.kv_lens.cuda(), sum(kv_lens), **kw)
    assert no_error()
    for t, sc, r in ((kc, kw.get("k_scale"), rk), (vc, kw.get("v_scale"), rv)):
        for s, n in enumerate(kv_lens):
            rows = O.cache_rows(t.cpu(), None if sc is None else sc.cpu(), c.table[s], n).to(BF)
            assert torch.equal(r.cpu()[int(full[s]):int(full[s + 1])], rows)


def test_cache_write_non_finite_rows():
    c = Cache([8], 1, 128, 16, True, 41)
    (kc, vc, table), kw = c.dev()
    k = torch.randn(8, 1, 128, generator=gen(7)).to(BF)
    k[1, 0, 5], k[2, 0, 6], k[3, 0, 7] = float("nan"), float("inf"), float("-inf")
    k[4] = float("nan")
    ops.paged_kv_write(k.cuda(), k.cuda(), kc, vc, table, cu_of([8]).cuda(), c.kv_lens.cuda(), **kw)
    rk, _ = ops.paged_kv_read(kc, vc, table, cu_of([8]).cuda(), c.kv_lens.cuda(), 8, **kw)
    rk = rk.cpu().float()
    assert rk[1, 0, 5].isnan() and rk[1].isnan().sum() == 1 and rk[4].isnan().all()
    assert rk[2, 0, 6] == math.inf and rk[3, 0, 7] == -math.inf
    fin = k[1].clone()
    fin[0, 5] = 0
    got = rk[1].clone()
    got[0, 5] = 0
    assert torch.equal(got.to(BF), O.quantise(fin)[1].to(BF))
    assert no_error()


@pytest.mark.parametrize("quant", [False, True])
def test_cache_bad_metadata_is_contained(quant):
    c = Cache([20, 30], 2, 128, 16, quant, 42)
    (kc, vc, table), kw = c.dev()
    k = torch.randn(14, 2, 128, generator=gen(8)).to(BF).cuda()
    lens, cu = c.kv_lens.cuda(), torch.tensor([0, 5, 10], dtype=torch.int32).cuda()

    def case(table=table, cu=cu, lens=lens):
        before = [t.view(torch.uint8).clone() for t in (kc, vc)]
        ops.paged_kv_write(k, k, kc, vc, table, cu, lens, **kw)
        torch.cuda.synchronize()
        code = _lib.poll_device_error()
        ko, vo = (torch.full((14, 2, 128), 7.0, dtype=BF, device="cuda") for _ in range(2))
        ops.paged_kv_read(kc, vc, table, cu, lens, 14, k_out=ko, v_out=vo, **kw)
        torch.cuda.synchronize()
        assert _lib.poll_device_error() == code
        for t, b in zip((kc, vc), before):  # only changes inside the used pages are possible; undo them
            t.view(torch.uint8).copy_(b)
        return ko, code

    def want(rows):
        return (O.quantise(k[rows].cpu())[1].to(BF) if quant else k[rows].cpu())

    ko, code = case()
    assert code == 0 and torch.equal(ko[:10].cpu(), want(slice(0, 10))) and (ko[10:] == 7.0).all()
    t = table.clone()
    t[0, 1] = 99                                        # positions 16..19 of segment 0: rows 1..4
    ko, code = case(table=t)
    assert code == 32 and (ko[1:5] == 0).all() and torch.equal(ko[5:10].cpu(), want(slice(5, 10)))
    for bad in (-1, 10 ** 6):
        ko, code = case(lens=torch.tensor([bad, 30], dtype=torch.int32).cuda())
        assert code == 32 and (ko[:5] == 0).all() and torch.equal(ko[5:10].cpu(), want(slice(5, 10)))
    ko, code = case(lens=torch.tensor([3, 30], dtype=torch.int32).cuda())  # two tokens without a position
    assert code == 0 and (ko[:2] == 0).all() and torch.equal(ko[2:10].cpu(), want(slice(2, 10)))
    ko, code = case(cu=torch.tensor([2, 5, 10], dtype=torch.int32).cuda())  # rows before the first segment
    assert code == 32 and (ko[:2] == 7.0).all() and torch.equal(ko[2:10].cpu(), want(slice(2, 10)))
    ko, code = case(cu=torch.tensor([0, 5, 99], dtype=torch.int32).cuda())  # past the tokens
    assert code == 32 and torch.equal(ko[:5].cpu(), want(slice(0, 5))) and (ko[5:] == 7.0).all()


def test_cache_refusals():
    c = Cache([10], 4, 128, 16, True, 43)
    (k, v, table), kw = c.dev()
    x = torch.zeros(2, 4, 128, dtype=BF, device="cuda")
    cu, lens = torch.tensor([0, 2], dtype=torch.int32).cuda(), c.kv_lens.cuda()
    ops.paged_kv_write(x, x, k, v, table, cu, lens, **kw)
    for a in ((x.float(), x), (x, x[:1]), (x[:, :3], x), (x.cpu(), x), (x.transpose(0, 1), x)):
        with pytest.raises(ValueError):
            ops.paged_kv_write(*a, k, v, table, cu, lens, **kw)
    with pytest.raises(ValueError):
        ops.paged_kv_write(x, x, k, v, table, cu, lens)
    with pytest.raises(ValueError):
        ops.paged_kv_read(k, v, table, cu, lens, -1, **kw)
    with pytest.raises(ValueError):
        ops.paged_kv_read(k, v, table, cu, lens, 2, k_out=x[:1], **kw)


# --------------------------------------------------------------------------- recurrent delta rule
def delta_inputs(T, Hk, H, seed):
    g = gen(seed)
    q = torch.randn(1, T, Hk, 128, generator=g).to(BF)
    k = torch.randn(1, T, Hk, 128, generator=g).to(BF)
    v = torch.randn(1, T, H, 128, generator=g).to(BF)
    gg = -torch.rand(1, T, H, generator=g) * 2
    beta = torch.rand(1, T, H, generator=g).to(BF)
    return q, k, v, gg, beta


def delta_check(o, want):
    err = (o.double().cpu() - want).abs()
    bound = 2 ** -8 * want.abs() + 2e-5 * max(1.0, want.abs().max().item())
    assert (err <= bound).all(), (err - bound).max().item()


def state_check(s, want):
    assert (s.double().cpu() - want).abs().max().item() <= 2e-5 * max(1.0, want.abs().max().item())


@pytest.mark.parametrize("Hk,H", [(16, 16), (5, 5), (2, 6), (1, 1)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [0, 2, 0, 70, 1, 7]])
def test_delta_pool(Hk, H, lens):
    T, S = sum(lens), len(lens)
    q, k, v, g, beta = delta_inputs(T, Hk, H, 50 + S)
    pool = torch.randn(2 * S + 2, H, 128, 128, generator=gen(51)) * 0.5
    first = torch.randperm(S + 1, generator=gen(52))[:S].int()
    first[S - 1] = -1                                    # from zero
    final = (torch.arange(S) + S + 1).int()
    if S > 1:
        final[0] = -3                                    # not kept
    d = pool.cuda()
    cu = cu_of(lens)
    o = ops.recurrent_gated_delta_rule_(q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), d, first.cuda(),
                                        final.cuda(), cu.cuda())
    assert no_error()
    init = torch.stack([pool[i] if i >= 0 else torch.zeros_like(pool[0]) for i in first.tolist()])
    want, states = O.recurrent_delta(q[0], k[0], v[0], g[0], beta[0], init, cu)
    delta_check(o[0], want)
    for s in range(S):
        if final[s] >= 0:
            state_check(d[final[s]], states[s])
    kept = torch.ones(pool.shape[0], dtype=torch.bool)
    kept[final[final >= 0].long()] = False
    assert torch.equal(d.cpu()[kept], pool[kept])


def test_delta_in_place_step_by_step_equals_one_call():
    H, S, n = 16, 3, 6
    q, k, v, g, beta = (t.cuda() for t in delta_inputs(S * n, H, H, 60))
    pool = (torch.randn(S, H, 128, 128, generator=gen(61)) * 0.5).cuda()
    a, b = pool.clone(), pool.clone()
    o1 = ops.recurrent_gated_delta_rule_(*(t.reshape(S, n, *t.shape[2:]) for t in (q, k, v, g, beta)), a)
    outs = []
    for i in range(n):
        step = [t.reshape(S, n, *t.shape[2:])[:, i:i + 1] for t in (q, k, v, g, beta)]
        outs.append(ops.recurrent_gated_delta_rule_(*step, b))
    assert no_error()
    # Not bit-equal: the kernel keeps a segment's decay factored out of its registers and multiplies it in
    # when it stores the state, after every token here and after six there.  Each of the two is within the
    # header's bound of the exact result, so by the triangle inequality they differ by at most twice it.
    assert (a - b).abs().max().item() <= 2 * 2e-5 * max(1.0, a.abs().max().item())
    o2 = torch.cat(outs, 1).float()
    o1 = o1.float()
    assert ((o1 - o2).abs() <= 2 * (2 ** -8 * o1.abs() * (1 + 2 ** -7) + 2e-5 * max(1.0, o1.abs().max().item()))).all()


def test_delta_forks_share_a_slot_and_no_l2norm():
    H, lens = 4, [3, 1, 5]
    T = sum(lens)
    q, k, v, g, beta = delta_inputs(T, H, H, 62)
    q, k = (q * 0.1).to(BF), (k * 0.1).to(BF)
    pool = torch.randn(5, H, 128, 128, generator=gen(63)) * 0.5
    d = pool.cuda()
    cu = cu_of(lens)
    o = ops.recurrent_gated_delta_rule_(q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), d,
                                        torch.tensor([1, 1, 1], dtype=torch.int32).cuda(),
                                        torch.tensor([2, 3, 4], dtype=torch.int32).cuda(), cu.cuda(),
                                        use_qk_l2norm_in_kernel=False)
    want, states = O.recurrent_delta(q[0], k[0], v[0], g[0], beta[0], pool[[1, 1, 1]], cu, l2norm=False)
    assert no_error()
    delta_check(o[0], want)
    state_check(d[2:], states)
    assert torch.equal(d[:2].cpu(), pool[:2])


def test_delta_transformers_signature_and_chunked_agree():
    H, lens = 16, [30, 64, 7]
    T = sum(lens)
    q, k, v, g, beta = (t.cuda() for t in delta_inputs(T, H, H, 64))
    cu = cu_of(lens).cuda()
    init = (torch.randn(3, H, 128, 128, generator=gen(65)) * 0.5).cuda()
    o, s = ops.recurrent_gated_delta_rule(q, k, v, g, beta, initial_state=init, output_final_state=True, cu_seqlens=cu)
    want, states = O.recurrent_delta(q[0].cpu(), k[0].cpu(), v[0].cpu(), g[0].cpu(), beta[0].cpu(), init.cpu(), cu.cpu())
    delta_check(o[0], want)
    state_check(s, states)
    oc, sc = ops.chunk_gated_delta_rule(q, k, v, g, beta, initial_state=init, output_final_state=True, cu_seqlens=cu)
    assert (oc.float() - o.float()).abs().max().item() < 2e-2  # the chunked kernel's own parity bound
    o0, none = ops.recurrent_gated_delta_rule(q.reshape(1, T, H, 128)[:, :10], k[:, :10], v[:, :10], g[:, :10], beta[:, :10])
    assert none is None
    w0, _ = O.recurrent_delta(q[0, :10].cpu(), k[0, :10].cpu(), v[0, :10].cpu(), g[0, :10].cpu(), beta[0, :10].cpu(),
                              torch.zeros(1, H, 128, 128), [0, 10])
    delta_check(o0[0], w0)
    assert no_error()


@pytest.mark.parametrize("decay", [0.0, -3.0, -30.0, -80.0, -200.0, float("-inf"), 20.0])
def test_delta_decays_of_any_size(decay):
    # decays from none to total and growth, mixed with ordinary ones, over several tokens; with growth the
    # state gets large, and bounds are relative to it
    H, n = 3, 21
    q, k, v, g, beta = delta_inputs(n, H, H, 68)
    g[0, 2::3] = decay
    g[0, 10] = decay
    if decay > 0:
        g[0, 2::3], g[0, 5] = 0.0, decay
    pool = torch.randn(2, H, 128, 128, generator=gen(69)) * 0.5
    d = pool.cuda()
    o = ops.recurrent_gated_delta_rule_(q.cuda(), k.cuda(), v.cuda(), g.cuda(), beta.cuda(), d,
                                        torch.tensor([0], dtype=torch.int32).cuda(),
                                        torch.tensor([1], dtype=torch.int32).cuda())
    assert no_error()
    want, states = O.recurrent_delta(q[0], k[0], v[0], g[0], beta[0], pool[:1], [0, n])
    delta_check(o[0], want)
    state_check(d[1:], states)


def test_delta_bad_metadata_and_refusals():
    H = 2
    q, k, v, g, beta = (t.cuda() for t in delta_inputs(6, H, H, 66))
    pool = torch.randn(4, H, 128, 128, generator=gen(67)).cuda()
    idx = lambda *a: torch.tensor(a, dtype=torch.int32).cuda()
    before = pool.clone()
    ops.recurrent_gated_delta_rule_(q, k, v, g, beta, pool, idx(0, 1), idx(9, 2), idx(0, 3, 6))
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 64
    assert torch.equal(pool[[0, 1, 3]], before[[0, 1, 3]]) and not torch.equal(pool[2], before[2])
    pool.copy_(before)
    ops.recurrent_gated_delta_rule_(q, k, v, g, beta, pool, idx(0, 1), idx(2, 3), idx(0, 30, 6))
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 64                # both ranges invalid: states carried over
    assert torch.equal(pool[2], before[0]) and torch.equal(pool[3], before[1])
    bad = [dict(query=q[0]), dict(key=k[:, :3]), dict(value=v[..., :64]), dict(g=g[:, :2]), dict(state=pool.bfloat16()),
           dict(state=pool[:, :1]), dict(state_indices=idx(0, 1, 2)), dict(state_indices=idx(0).long()),
           dict(cu_seqlens=idx(0)), dict(query=q.float()), dict(state=pool.cpu()), dict(out=q.float())]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.recurrent_gated_delta_rule_(**{**dict(query=q, key=k, value=v, g=g, beta=beta, state=pool), **kw})
    with pytest.raises(ValueError):  # two segments, one slot
        ops.recurrent_gated_delta_rule_(q, k, v, g, beta, pool[:1], cu_seqlens=idx(0, 3, 6))


# --------------------------------------------------------------------------- conv with history
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("lens", [[1], [2, 0, 1, 3, 4, 5], [64, 1, 200, 8, 9, 7]])
def test_conv_history(K, lens):
    Hk, Hv = 2, 3
    C, T, S = (2 * Hk + Hv) * 128, sum(lens), len(lens)
    g = gen(70 + K)
    x = torch.randn(1, T, C + 64, generator=g).to(BF)[:, :, :C]
    w = (0.5 * torch.randn(C, K, generator=g)).to(BF)
    pool = torch.randn(S + 3, K - 1, C, generator=g).to(BF)
    first = torch.randperm(S + 3, generator=g)[:S].int()
    in_place = first.clone()
    first[0] = -1
    d = pool.cuda()
    cu = cu_of(lens)
    q, k, v = ops.packed_conv_state_(x.cuda()[:, :, :C], w.cuda(), d, first.cuda(), in_place.cuda(), Hk * 128, Hv * 128,
                                     cu_seqlens=cu.cuda())
    assert no_error()
    hist = torch.stack([pool[i] if i >= 0 else torch.zeros_like(pool[0]) for i in first.tolist()])
    want, pre, finals = O.conv_silu(x[0], w, hist, cu)
    got = torch.cat([t.reshape(T, -1) for t in (q, k, v)], 1).double().cpu()
    bound = 2 ** -8 * want.abs() + 2 ** -10.9 * pre.abs() / 2 + 2e-6
    assert ((got - want).abs() <= bound).all()
    expect = pool.clone()
    expect[in_place.long()] = finals.to(BF)
    assert torch.equal(d.cpu(), expect)


def test_conv_steps_equal_one_call_and_match_the_packed_conv():
    C, n, S = 6144, 11, 2
    g = gen(80)
    x = torch.randn(S, n, C, generator=g).to(BF).cuda()
    w = (0.5 * torch.randn(C, 1, 4, generator=g)).to(BF).cuda()
    a = torch.zeros(S, 3, C, dtype=BF, device="cuda")
    b = a.clone()
    one = ops.packed_conv_state_(x, w, a)
    steps = [ops.packed_conv_state_(x[:, i:j], w, b) for i, j in ((0, 1), (1, 3), (3, 8), (8, 11))]
    assert no_error()
    for i in range(3):
        assert torch.equal(torch.cat([s[i] for s in steps], 1), one[i])
    assert torch.equal(a, b) and torch.equal(a, x[:, -3:])
    plain = ops.packed_conv_qkv(x, w)
    for p, o in zip(plain, one):
        assert (p.float() - o.float()).abs().max().item() <= 2 ** -7 * o.float().abs().max().item()


def test_conv_history_padding_bad_metadata_and_refusals():
    C = 384
    x = torch.randn(1, 10, C, generator=gen(81)).to(BF).cuda()
    w = torch.randn(C, 4, generator=gen(82)).to(BF).cuda()
    pool = torch.randn(3, 3, C, generator=gen(83)).to(BF).cuda()
    idx = lambda *a: torch.tensor(a, dtype=torch.int32).cuda()
    before = pool.clone()
    ops.packed_conv_state_(x, w, pool, idx(0, 5), idx(7, 1), cu_seqlens=idx(0, 4, 6))
    torch.cuda.synchronize()
    assert _lib.poll_device_error() == 64
    assert torch.equal(pool[[0, 2]], before[[0, 2]])
    assert torch.equal(pool[1], torch.cat([torch.zeros(1, C, dtype=BF, device="cuda"), x[0, 4:6]]))
    for kw in (dict(x=x.float()), dict(weight=w[:, :1]), dict(state=pool[:, :2]), dict(state=pool.float()),
               dict(key_dim=100), dict(cu_seqlens=idx(0)), dict(state_indices=idx(0, 1)), dict(x=x.cpu())):
        with pytest.raises(ValueError):
            ops.packed_conv_state_(**{**dict(x=x, weight=w, state=pool), **kw})
