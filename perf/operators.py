"""The cached-continuation operators as workloads: what they compute, in plain torch and through
``fastdecisions_b200.ops``, on seeded inputs.

A decision model that keeps state continues a request from it: the attention layers from a paged
KV cache (written in bf16, or in e4m3 with a power-of-two scale per token and head), the
Gated-DeltaNet layers from a convolution history and a recurrent state.  Kinds of cases:

* ``attn``: attention of the newest tokens of each sequence over its paged cache;
* ``kv``: writing new keys and values into the cache (``quant``: in 8 bits) and reading them back
  (``write`` False: only the read of whole contexts);
* ``delta``: the recurrent gated delta rule from a pool of states;
* ``conv``: the packed causal convolution + SiLU with cached history.

Head layouts are the repository's own: 16 query / 4 KV heads of 128 (the benchmark model) and
8 / 2 of 256 (the reference attention's shape); 16 Gated-DeltaNet heads of 128.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request answering token by token behind a prompt of the benchmark's batch-1 length
        dict(name="attn_decode_one", kind="attn", seqs=1, q_lo=1, q_hi=1, past_lo=1535, past_hi=1535, shared=0,
             hq=16, hkv=4, d=128, page=64, quant=False, gate=True, salt=1),
        # a serving batch, one new token each, contexts from short to the longest request, 8-bit cache
        dict(name="attn_decode_batch_e4m3", kind="attn", seqs=64, q_lo=1, q_hi=1, past_lo=500, past_hi=8192, shared=0,
             hq=16, hkv=4, d=128, page=64, quant=True, gate=True, salt=2),
        # questions of a few dozen tokens asked about one shared document (its pages are shared), wide heads
        dict(name="attn_questions_shared_d256", kind="attn", seqs=48, q_lo=9, q_hi=70, past_lo=0, past_hi=0,
             shared=1490, hq=8, hkv=2, d=256, page=32, quant=False, gate=True, salt=3),
        # ragged chunks behind ragged histories, 8-bit cache, small pages
        dict(name="attn_chunks_e4m3", kind="attn", seqs=8, q_lo=100, q_hi=700, past_lo=600, past_hi=8000, shared=0,
             hq=16, hkv=4, d=128, page=16, quant=True, gate=False, salt=4),
        # two long documents fed in pieces: 2048 new tokens behind 6144 to 14000 cached ones
        dict(name="attn_chunk_long", kind="attn", seqs=2, q_lo=2048, q_hi=2048, past_lo=6144, past_hi=14000, shared=0,
             hq=16, hkv=4, d=128, page=128, quant=False, gate=True, salt=5),
        # the cache update of one decoding step of a serving batch
        dict(name="kv_write_decode", kind="kv", write=True, seqs=64, q_lo=1, q_hi=1, past_lo=100, past_hi=4000,
             hkv=4, d=128, page=64, quant=True, salt=6),
        # the cache update of a packed prompt batch of ragged requests
        dict(name="kv_write_prompts", kind="kv", write=True, seqs=23, q_lo=64, q_hi=8192, past_lo=0, past_hi=333,
             hkv=4, d=128, page=64, quant=True, salt=7),
        # whole contexts read back (to move them, or to hand them to a kernel without pages)
        dict(name="kv_read_contexts", kind="kv", write=False, seqs=19, q_lo=900, q_hi=8191, past_lo=0, past_hi=0,
             hkv=2, d=256, page=32, quant=True, salt=8),
        # one token of one request: 16 heads of 128 x 128 state
        dict(name="delta_decode_one", kind="delta", seqs=1, q_lo=1, q_hi=1, heads=16, shared=False, salt=9),
        # short questions forked from the state of one shared prefix, each keeping a state of its own
        dict(name="delta_questions_shared", kind="delta", seqs=96, q_lo=1, q_hi=24, heads=16, shared=True, salt=10),
        # one token of a serving batch
        dict(name="conv_decode_batch", kind="conv", seqs=64, q_lo=1, q_hi=1, heads=16, shared=False, salt=11),
        # packed questions forked from one shared prefix
        dict(name="conv_questions_shared", kind="conv", seqs=96, q_lo=1, q_hi=200, heads=16, shared=True, salt=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "kv", "delta", "conv"])
    salt = rng.randrange(1 << 20)
    if kind == "attn":
        hq, hkv, d = rng.choice([(16, 4, 128), (8, 2, 256), (8, 8, 128), (6, 1, 128), (10, 2, 128), (4, 4, 256)])
        form = rng.choice(["decode", "few", "chunk", "shared"])
        case = dict(kind=kind, hq=hq, hkv=hkv, d=d, page=rng.choice([16, 32, 64, 128]), quant=rng.random() < 0.5,
                    gate=rng.random() < 0.5, shared=0, past_lo=0, past_hi=0, salt=salt)
        if form == "decode":
            case.update(seqs=_log_int(rng, 1, 64), q_lo=1, q_hi=1)
        elif form == "few":
            case.update(seqs=_log_int(rng, 1, 32), q_lo=1, q_hi=rng.randint(2, 16))
        elif form == "chunk":
            case.update(seqs=_log_int(rng, 1, 8), q_lo=rng.randint(17, 100), q_hi=_log_int(rng, 100, 1000))
        else:
            case.update(seqs=_log_int(rng, 2, 48), q_lo=rng.randint(1, 30), q_hi=rng.randint(30, 100),
                        shared=_log_int(rng, 10, 4000))
        if form != "shared":
            hi = _log_int(rng, 50, 8192)
            case.update(past_lo=rng.randint(0, hi), past_hi=hi)
        return case
    if kind == "kv":
        hkv, d = rng.choice([(4, 128), (2, 256), (8, 128), (1, 128)])
        lo = _log_int(rng, 1, 300)
        return dict(kind=kind, write=rng.random() < 0.6, seqs=_log_int(rng, 1, 48), q_lo=lo,
                    q_hi=lo + _log_int(rng, 1, 2000), past_lo=0, past_hi=_log_int(rng, 1, 500), hkv=hkv, d=d,
                    page=rng.choice([16, 32, 64, 128]), quant=rng.random() < 0.7, salt=salt)
    if kind == "delta":
        lo = rng.randint(1, 8)
        return dict(kind=kind, seqs=_log_int(rng, 1, 96), q_lo=lo, q_hi=lo + rng.randint(0, 20),
                    heads=rng.choice([16, 16, 6, 5]), shared=rng.random() < 0.5, salt=salt)
    lo = rng.randint(1, 64)
    return dict(kind=kind, seqs=_log_int(rng, 1, 96), q_lo=lo, q_hi=lo + rng.randint(0, 200),
                heads=rng.choice([16, 16, 6, 5]), shared=rng.random() < 0.5, salt=salt)


def _lengths(case):
    """New tokens and cached tokens of each sequence: spread over their ranges, the ends included."""
    rng = random.Random(case["salt"])
    n = case["seqs"]

    def spread(lo, hi):
        out = [_log_int(rng, lo + 1, hi + 1) - 1 for _ in range(n)]
        if n > 1:
            out[rng.randrange(n)] = hi
            out[rng.randrange(n)] = lo
        else:
            out[0] = hi
        return out

    new = spread(case["q_lo"], case["q_hi"])
    past = [0] * n
    if case["kind"] in ("attn", "kv"):
        past = spread(case["past_lo"], case["past_hi"])
        if case.get("shared"):
            past = [case["shared"]] * n
    return new, past


def work(case):
    new, past = _lengths(case)
    tokens = sum(new)
    if case["kind"] == "attn":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        context = sum(new) + (case["shared"] if case["shared"] else sum(past))
        per_row = d + 1 if case["quant"] else 2 * d
        rows = 4 * tokens * hq * d + (2 * tokens * hq * d if case["gate"] else 0)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
        return dict(bytes=2 * context * hkv * per_row + rows, flops=4 * pairs * hq * d)
    if case["kind"] == "kv":
        elems = tokens * case["hkv"]
        # write: bf16 in, cached rows (8-bit: and their scales) out; read back: the other way (k and v)
        one_way = 2 * elems * (3 * case["d"] + 1 if case["quant"] else 4 * case["d"])
        return dict(bytes=one_way * (2 if case["write"] else 1), flops=0)
    h = case["heads"]
    if case["kind"] == "delta":
        state = h * 128 * 128 * 4
        reads = 1 if case["shared"] else case["seqs"]
        return dict(bytes=state * (reads + case["seqs"]) + tokens * h * (4 * 256 + 6),
                    flops=tokens * h * 8 * 128 * 128)
    c = 3 * h * 128
    reads = 1 if case["shared"] else case["seqs"]
    return dict(bytes=4 * tokens * c + 6 * c * (reads + case["seqs"]) + 8 * c, flops=tokens * c * 12)


# ----------------------------------------------------------------------------------------- inputs
def _scale_exponent(x):
    """Smallest integer e with max_d |x| <= 448 * 2^e, in [-127, 127] (x: [..., D] float32)."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = e - 9 + (m > 0.875).int()
    return torch.where(m == 0, torch.full_like(e, -127), e).clamp(-127, 127)


def _quantise(x):
    """bf16 [..., D] -> e4m3 values, uint8 exponents (biased by 127)."""
    f = x.float()
    e = _scale_exponent(f)
    return torch.ldexp(f, -e[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed * 1000003 + case["salt"])
    new, past = _lengths(case)
    n, tokens = len(new), sum(new)
    starts = [0]
    for q in new:
        starts.append(starts[-1] + q)
    cu = torch.tensor(starts, dtype=torch.int32, device=dev)
    st = dict(case=case, new=new, past=past, cu=cu)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    if case["kind"] in ("attn", "kv"):
        hkv, d, page = case["hkv"], case["d"], case["page"]
        lens = [q + p for q, p in zip(new, past)]
        shared_pages = (case.get("shared", 0) // page)  # whole pages of a shared prefix exist once
        own_pages = [(x + page - 1) // page - shared_pages for x in lens]
        total = shared_pages + sum(own_pages)
        order = torch.randperm(total + 3, generator=g, device=dev).cpu().tolist()
        width = max(shared_pages + o for o in own_pages) + 1
        table = torch.full((n, width), -1, dtype=torch.int32)
        nxt = shared_pages
        for s, o in enumerate(own_pages):
            table[s, :shared_pages] = torch.tensor(order[:shared_pages], dtype=torch.int32)
            table[s, shared_pages:shared_pages + o] = torch.tensor(order[nxt:nxt + o], dtype=torch.int32)
            nxt += o
        st.update(page_table=table.to(dev), kv_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                  max_seqlen=max(new), max_kv_len=max(lens))
        shape = (total + 3, hkv, page, d)
        for name in ("k", "v"):
            cache = torch.empty(shape, dtype=torch.bfloat16, device=dev)
            for p0 in range(0, shape[0], 1024):
                cache[p0:p0 + 1024] = normal(*cache[p0:p0 + 1024].shape).bfloat16()
            st[name + "_scale"] = None
            if case["quant"]:
                cache, st[name + "_scale"] = _quantise(cache)
            st[name + "_cache"] = cache
        if case["kind"] == "attn":
            st["q"] = normal(tokens, case["hq"], d).bfloat16()
            st["gate"] = normal(tokens, case["hq"] * d).bfloat16() if case["gate"] else None
        else:
            st["k"] = normal(tokens, hkv, d).bfloat16()
            st["v"] = (normal(tokens, hkv, d) * torch.exp(normal(tokens, hkv, 1))).bfloat16()
        return st
    h = case["heads"]
    ids = torch.arange(n, dtype=torch.int32, device=dev)
    first = torch.zeros_like(ids) if case["shared"] else ids
    reads = 1 if case["shared"] else n
    st.update(state_indices=first, final_indices=ids + reads, reads=reads)
    if case["kind"] == "delta":
        st["state"] = normal(reads + n, h, 128, 128) * 0.3
        for name in ("q", "k", "v"):
            st[name] = torch.nn.functional.silu(normal(1, tokens, h, 128)).bfloat16()
        st["g"] = -torch.exp(normal(1, tokens, h) - 1.0)
        st["beta"] = torch.sigmoid(normal(1, tokens, h)).bfloat16()
    else:
        c = 3 * h * 128
        # the convolution reads the leading columns of the layer's wider projection
        st["x"] = normal(1, tokens, c + h * 128 + 32).bfloat16()[:, :, :c]
        st["w"] = (0.5 * normal(c, 4)).bfloat16()
        st["state"] = normal(reads + n, 3, c).bfloat16()
    return st


# ----------------------------------------------------------------------------------- plain forms
def _context(st, s, name, length):
    """Cached rows [0, length) of sequence s, [length, Hkv, D] float32."""
    page = st["case"]["page"]
    ids = st["page_table"][s, :(length + page - 1) // page].long()
    rows = st[name + "_cache"][ids].float()
    if st[name + "_scale"] is not None:
        rows = rows * torch.exp2(st[name + "_scale"][ids].float() - 127.0)[..., None]
    return rows.permute(0, 2, 1, 3).reshape(-1, rows.shape[1], rows.shape[3])[:length]


def _plain_attn(st):
    case = st["case"]
    hkv, d = case["hkv"], case["d"]
    rep = case["hq"] // hkv
    out = torch.empty_like(st["q"])
    t0 = 0
    for s, (n, past) in enumerate(zip(st["new"], st["past"])):
        length = n + past
        k = _context(st, s, "k", length).permute(1, 2, 0)                       # [Hkv, D, L]
        v = _context(st, s, "v", length).permute(1, 0, 2)                       # [Hkv, L, D]
        q = st["q"][t0:t0 + n].float().reshape(n, hkv, rep, d).permute(1, 2, 0, 3)   # [Hkv, rep, n, D]
        hidden = torch.arange(length, device=q.device)[None, :] > torch.arange(past, length, device=q.device)[:, None]
        for h in range(hkv):
            sc = (q[h].reshape(rep * n, d) @ k[h]).reshape(rep, n, length) * d ** -0.5
            sc = sc.masked_fill(hidden, float("-inf"))
            p = torch.exp(sc - sc.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = (p.reshape(rep * n, length) @ v[h]).reshape(rep, n, d).transpose(0, 1)
            if st["gate"] is not None:
                gate = st["gate"][t0:t0 + n].float().reshape(n, hkv, rep, d)[:, h]
                o = o / (1.0 + torch.exp(-gate))
            out[t0:t0 + n, h * rep:(h + 1) * rep] = o.to(out.dtype)
        t0 += n
    return out


def _rows_of_new(st):
    """Page and offset of every new token, in packed order."""
    page = st["case"]["page"]
    seq = torch.repeat_interleave(torch.arange(len(st["new"]), device="cuda"),
                                  torch.tensor(st["new"], device="cuda"))
    t = torch.arange(seq.numel(), device="cuda")
    pos = st["kv_lens"].long()[seq] - (st["cu"].long()[seq + 1] - t)
    return st["page_table"][seq, pos // page].long(), pos % page


def _plain_kv(st):
    page, off = _rows_of_new(st)
    out = []
    for name in ("k", "v"):
        cache, scale = st[name + "_cache"], st[name + "_scale"]
        if scale is None:
            if st["case"]["write"]:
                cache[page, :, off] = st[name]
            out.append(cache[page, :, off])
            continue
        if st["case"]["write"]:
            vals, exps = _quantise(st[name])
            cache.view(torch.uint8)[page, :, off] = vals.view(torch.uint8)
            scale[page, :, off] = exps
        rows = cache.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).float()
        out.append((rows * torch.exp2(scale[page, :, off].float() - 127.0)[..., None]).bfloat16())
    return tuple(out)


def _plain_delta(st):
    new, cu = st["new"], st["cu"].long()
    q, k, v = (st[x][0].float() for x in ("q", "k", "v"))
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * 128 ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    g, beta = st["g"][0], st["beta"][0].float()
    state = st["state"][st["state_indices"].long()].clone()
    out = torch.empty_like(st["v"])
    lens = torch.tensor(new, device="cuda")
    for i in range(max(new)):
        live = torch.nonzero(lens > i).flatten()
        t = cu[live] + i
        s = state[live] * torch.exp(g[t])[..., None, None]
        delta = (v[t] - (s * k[t][..., None]).sum(-2)) * beta[t][..., None]
        s = s + k[t][..., None] * delta[..., None, :]
        state[live] = s
        out[0, t] = (s * q[t][..., None]).sum(-2).bfloat16()
    st["state"][st["final_indices"].long()] = state
    return out, st["state"][st["reads"]:]


def _plain_conv(st):
    new, c = st["new"], st["w"].shape[0]
    cu = st["cu"].long()
    n = len(new)
    x = st["x"][0]
    lens = torch.tensor(new, device="cuda")
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), lens)
    # every segment with its three history rows before it, end to end
    rows = torch.empty(x.shape[0] + 3 * n, c, dtype=torch.float32, device="cuda")
    place = torch.arange(x.shape[0], device="cuda") + 3 * (seq + 1)
    head = cu[:-1] + 3 * torch.arange(n, device="cuda")
    rows[place] = x.float()
    hist = st["state"][st["state_indices"].long()].float()
    for j in range(3):
        rows[head + j] = hist[:, j]
    w = st["w"].float()
    y = rows[place] * w[:, 3]
    for j in range(3):
        y = y + rows[place - 3 + j] * w[:, j]
    y = (y / (1.0 + torch.exp(-y))).bfloat16()
    ends = cu[1:] + 3 * torch.arange(1, n + 1, device="cuda")
    for j in range(3):
        st["state"][st["final_indices"].long(), j] = rows[ends - 3 + j].bfloat16()
    qkv = tuple(part.reshape(1, -1, st["case"]["heads"], 128) for part in y.split(c // 3, dim=1))
    return qkv + (st["state"][st["reads"]:],)


# ------------------------------------------------------------------------------------------- run
def run(state):
    st = state
    kind = st["case"]["kind"]
    if not own:
        return {"attn": _plain_attn, "kv": _plain_kv, "delta": _plain_delta, "conv": _plain_conv}[kind](st)
    from fastdecisions_b200 import ops
    if kind == "attn":
        return ops.paged_gqa_attention(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["cu"],
                                       st["kv_lens"], st["max_seqlen"], st["max_kv_len"], k_scale=st["k_scale"],
                                       v_scale=st["v_scale"], gate=st["gate"])
    if kind == "kv":
        cache = (st["k_cache"], st["v_cache"], st["page_table"], st["cu"], st["kv_lens"])
        if st["case"]["write"]:
            ops.paged_kv_write(st["k"], st["v"], *cache, k_scale=st["k_scale"], v_scale=st["v_scale"])
        return ops.paged_kv_read(*cache, st["k"].shape[0], k_scale=st["k_scale"], v_scale=st["v_scale"])
    if kind == "delta":
        o = ops.recurrent_gated_delta_rule_(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                                            state_indices=st["state_indices"], final_indices=st["final_indices"],
                                            cu_seqlens=st["cu"])
        return o, st["state"][st["reads"]:]
    qkv = ops.packed_conv_state_(st["x"], st["w"], st["state"], state_indices=st["state_indices"],
                                 final_indices=st["final_indices"], cu_seqlens=st["cu"])
    return tuple(qkv) + (st["state"][st["reads"]:],)


# ----------------------------------------------------------------------------------------- exact
def _exact_values(cache, scale, page, off):
    """Rows of the cache in float64, decoded from their bits."""
    if scale is None:
        return cache[page, :, off].double()
    b = cache.view(torch.uint8)[page, :, off].long()
    sign = 1.0 - 2.0 * (b >> 7).double()
    exp, man = (b >> 3) & 15, (b & 7).double()
    mag = torch.where(exp > 0, torch.ldexp(1.0 + man / 8.0, exp - 7), torch.ldexp(man / 8.0, torch.full_like(exp, -6)))
    return sign * mag * torch.ldexp(torch.ones((), device="cuda", dtype=torch.float64),
                                    scale[page, :, off].long() - 127)[..., None]


def _exact_attn(st):
    case, page = st["case"], st["case"]["page"]
    rep, d = case["hq"] // case["hkv"], case["d"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    for s, n in enumerate(st["new"]):
        length = int(st["kv_lens"][s])
        t0 = int(st["cu"][s])
        pos = torch.arange(length, device="cuda")
        pages = st["page_table"][s].long()[pos // page]
        k = _exact_values(st["k_cache"], st["k_scale"], pages, pos % page)
        v = _exact_values(st["v_cache"], st["v_scale"], pages, pos % page)
        for r0 in range(0, n, 512):
            r1 = min(n, r0 + 512)
            seen = (pos[None, :] <= (length - n + torch.arange(r0, r1, device="cuda"))[:, None]).double()
            for h in range(case["hq"]):
                z = st["q"][t0 + r0:t0 + r1, h].double() @ k[:, h // rep].t() / math.sqrt(d)
                z = torch.where(seen > 0, z, torch.full_like(z, -math.inf))
                out[t0 + r0:t0 + r1, h] = torch.softmax(z, -1) @ v[:, h // rep]
    if st["gate"] is not None:
        out *= torch.sigmoid(st["gate"].double()).reshape(out.shape)
    return out


def _exact_kv(st):
    page, off = _rows_of_new(st)
    out = []
    for name in ("k", "v"):
        if not st["case"]["write"]:
            out.append(_exact_values(st[name + "_cache"], st[name + "_scale"], page, off))
            continue
        x = st[name].double()
        if st[name + "_scale"] is None:
            out.append(x)
            continue
        peak = x.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(peak > 0, peak, torch.ones_like(peak)) / E4M3_MAX))
        y = x / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)  # e4m3 spacing at |y|
        out.append(torch.round(y / step) * step * torch.exp2(e))
    return tuple(out)


def _exact_delta(st):
    q, k, v = (st[x][0].double() for x in ("q", "k", "v"))
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) / math.sqrt(128)
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    g, beta = st["g"][0].double(), st["beta"][0].double()
    out = torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    finals = []
    for s in range(len(st["new"])):
        a = st["state"][int(st["state_indices"][s])].double()
        for t in range(int(st["cu"][s]), int(st["cu"][s + 1])):
            a = a * torch.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", a, k[t]))
            a = a + torch.einsum("hk,hv->hkv", k[t], u)
            out[t] = torch.einsum("hkv,hk->hv", a, q[t])
        finals.append(a)
    return out[None], torch.stack(finals)


def _exact_conv(st):
    w = st["w"].double()
    outs, finals = [], []
    for s in range(len(st["new"])):
        x = st["x"][0, int(st["cu"][s]):int(st["cu"][s + 1])].double()
        rows = torch.cat([st["state"][int(st["state_indices"][s])].double(), x])
        y = torch.einsum("tcj,cj->tc", rows.unfold(0, 4, 1), w)
        outs.append(y * torch.sigmoid(y))
        finals.append(rows[-3:])
    y = torch.cat(outs)
    c = y.shape[1]
    return tuple(p.reshape(1, -1, st["case"]["heads"], 128) for p in y.split(c // 3, dim=1)) + (torch.stack(finals),)


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "kv": _exact_kv, "delta": _exact_delta, "conv": _exact_conv}[case["kind"]](st)
