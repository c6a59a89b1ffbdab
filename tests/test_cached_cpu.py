"""Cached-state operators without a GPU: refusals, host-side sizes, installers and the oracle itself."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from fastdecisions_b200 import _lib, ops, patches, workloads as W
from fastdecisions_b200.engine import DecisionEngine, Prefix, StateCache
from oracle import cached as O
from oracle import ops as R


def test_binding_loads_and_has_every_operator():
    b = _lib.binding()
    for name in ("paged_kv_write", "paged_kv_read", "paged_gqa_attention", "recurrent_gated_delta_rule",
                 "packed_conv_state"):
        assert callable(getattr(b, name))
    with pytest.raises(ValueError, match="arguments expected"):
        b.paged_kv_write(1, 2)


def test_cpu_tensors_are_refused():
    bf = torch.bfloat16
    x, cache = torch.zeros(2, 4, 128, dtype=bf), torch.zeros(3, 4, 16, 128, dtype=bf)
    meta = (torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32))
    q = torch.zeros(1, 2, 4, 128, dtype=bf)
    g = torch.zeros(1, 2, 4)
    state = torch.zeros(1, 4, 128, 128)
    calls = [lambda: ops.paged_kv_write(x, x, cache, cache, *meta),
             lambda: ops.paged_kv_read(cache, cache, *meta, 2),
             lambda: ops.paged_gqa_attention(x, cache, cache, *meta, 2),
             lambda: ops.recurrent_gated_delta_rule_(q, q, q, g, g, state),
             lambda: ops.recurrent_gated_delta_rule(q, q, q, g, g, None, False),
             lambda: ops.packed_conv_state_(torch.zeros(1, 2, 384, dtype=bf), torch.zeros(384, 4, dtype=bf),
                                            torch.zeros(1, 3, 384, dtype=bf))]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for wrong in (None, 3, "x"):
        with pytest.raises(ValueError):
            ops.paged_kv_write(wrong, x, cache, cache, *meta)


def test_workspace_size_on_the_host():
    size = ops.paged_gqa_workspace_bytes
    assert size(1, 1, 100, 1, 16, 4, 128) == 0            # one part
    assert size(1, 1, 1535, 1, 16, 4, 128) == 0           # parts joined in a cluster
    for segments, seq, kv, tokens in ((64, 1, 8192, 64), (1, 1, 1 << 20, 1), (2, 100, 8192, 200)):
        need = size(segments, seq, kv, tokens, 16, 4, 128)
        parts, rest = divmod(need, tokens * 16 * (128 * 4 + 8))
        assert rest == 0 and 2 <= parts <= 64
    assert size(1, 1, 100, 1, 16, 5, 128) == 0 and size(0, 1, 1, 1, 16, 4, 128) == 0 and size(1, 1, 1, 1, 16, 4, 64) == 0


def test_state_cache_arguments():
    cfg = W.ModelConfig(num_hidden_layers=4)
    for kw in (dict(tokens=0, prefixes=1), dict(tokens=10, prefixes=0), dict(tokens=10, prefixes=1, page_size=48),
               dict(tokens=10, prefixes=1, kv_dtype="fp8")):
        with pytest.raises(ValueError):
            StateCache(cfg, "cpu", **kw)
    c = StateCache(cfg, "cpu", tokens=100, prefixes=2, page_size=32, kv_dtype="e4m3")
    assert len(c.free_pages) == 4 and len(c.free_slots) == 2
    assert c.layers[3].k.shape == (4, 4, 32, 128) and c.layers[3].ks.shape == (4, 4, 32)
    assert c.layers[0].conv.shape == (2, 3, 6144) and c.layers[0].state.shape == (2, 16, 128, 128)
    with pytest.raises(RuntimeError, match="free"):
        c.take_pages(5)
    c.layers[3].k.view(torch.uint8)[2] = 7
    c.copy_page(2, torch.tensor([0, 3]))
    assert (c.layers[3].k.view(torch.uint8)[[0, 2, 3]] == 7).all() and (c.layers[3].k.view(torch.uint8)[1] == 0).all()


def test_installer_counts_gdn_modules():
    mq = pytest.importorskip("transformers.models.qwen3_5.modeling_qwen3_5")
    cfg = W.ModelConfig(hidden_size=256, num_hidden_layers=8, intermediate_size=256, vocab_size=64)
    model = mq.Qwen3_5TextModel(cfg.to_transformers())
    assert patches.install_recurrent_gated_delta_rule(model) == 6
    assert all(m.recurrent_gated_delta_rule is ops.recurrent_gated_delta_rule
               for m in model.modules() if isinstance(m, mq.Qwen3_5GatedDeltaNet))


def test_oracle_e4m3_is_the_type():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    finite = every[torch.isfinite(every)].sort().values
    assert torch.equal(O.e4m3_round(finite), finite)
    mid = (finite[1:] + finite[:-1]) / 2          # ties and their neighbours
    x = torch.cat([mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20)]).float()
    assert torch.equal(O.e4m3_round(x.double()), x.to(torch.float8_e4m3fn).double())


def test_oracle_scale_is_the_smallest_that_fits():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(2000, 8, generator=g) * torch.exp(8 * torch.randn(2000, 1, generator=g))).bfloat16()
    x[0], x[1] = 0, 448.0
    e, v = O.quantise(x)
    top = x.double().abs().amax(-1)
    assert (top <= 448 * O.power_of_two(e)).all()
    assert (top[1:] > 448 * O.power_of_two(e[1:] - 1)).all()
    assert ((v - x.double()).abs() <= 2 ** -4 * x.double().abs() + 2.0 ** -10 * O.power_of_two(e)[:, None]).all()


def test_oracle_attention_and_recurrences_agree_with_the_uncached_oracle():
    g = torch.Generator().manual_seed(2)
    n, hq, hkv, D, page = 21, 4, 2, 128, 16
    q, k, v = (torch.randn(n, h, D, generator=g).bfloat16() for h in (hq, hkv, hkv))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    kc, vc = (torch.zeros(3, hkv, page, D, dtype=torch.bfloat16) for _ in range(2))
    for p in range(n):
        kc[table[0, p // page], :, p % page], vc[table[0, p // page], :, p % page] = k[p], v[p]
    want = R.gqa_attention_varlen(q, k, v)
    got, mag, size = O.paged_attention(q[5:], kc, vc, table, [0, n - 5], [n])
    assert (got - want[5:]).abs().max() < 1e-5 and (mag >= got.abs() - 1e-9).all() and (size > 0).all()
    H = 2
    dq, dk, dv = (torch.randn(1, n, H, 128, generator=g) for _ in range(3))
    dg, beta = -torch.rand(1, n, H, generator=g), torch.rand(1, n, H, generator=g)
    o, _ = O.recurrent_delta(dq[0], dk[0], dv[0], dg[0], beta[0], torch.zeros(1, H, 128, 128), [0, n])
    assert (o - R.recurrent_gated_delta_rule(dq, dk, dv, dg, beta)[0]).abs().max() < 1e-4
    x, w = torch.randn(1, n, 384, generator=g).bfloat16(), torch.randn(384, 4, generator=g).bfloat16()
    y, _, hist = O.conv_silu(x[0], w, torch.zeros(1, 3, 384), [0, n])
    ref = torch.cat([t.reshape(n, -1) for t in R.packed_conv_silu(x, w)], 1)
    assert (y - ref).abs().max() < 1e-4 and torch.equal(hist[0], x[0, -3:].double())
    assert math.isfinite(float(y.sum()))


def test_prefix_of_another_model_and_failed_extension():
    cfg = W.ModelConfig(num_hidden_layers=4, vocab_size=64)
    eng = object.__new__(DecisionEngine)  # host logic only
    eng.cfg, eng.dev, eng.max_positions = cfg, torch.device("cpu"), 4096
    other = StateCache(W.ModelConfig(num_hidden_layers=8, vocab_size=64), "cpu", 64, 1, 16)
    with pytest.raises(ValueError, match="another model"):
        eng.extend(Prefix(other, 0), [1, 2])
    cache = StateCache(cfg, "cpu", 64, 1, 16)
    with pytest.raises(ValueError, match="another model"):
        eng.score_after(Prefix(other, 0), [W.Request(ids=np.zeros(2, np.int32), slot=1, nopts=2)])

    def fails(*_):
        raise RuntimeError("launch failed")

    eng._run_cached = lambda *_: None
    prefix = eng.cache_prefix(cache, np.zeros(20, np.int32))
    assert prefix.length == 20 and len(cache.free_pages) == 2 and not cache.free_slots
    eng._run_cached = fails
    with pytest.raises(RuntimeError, match="launch failed"):
        eng.extend(prefix, np.zeros(20, np.int32))
    assert prefix.slot is None and len(cache.free_pages) == 4 and len(cache.free_slots) == 1
    with pytest.raises(RuntimeError, match="launch failed"):
        eng.cache_prefix(cache, np.zeros(20, np.int32))
    assert len(cache.free_pages) == 4 and len(cache.free_slots) == 1


def test_prefix_of_another_engine():
    # equal configurations say nothing about the weights (or the device) a cache was filled with
    cfg = W.ModelConfig(num_hidden_layers=4, vocab_size=64)
    a, b = (object.__new__(DecisionEngine) for _ in range(2))  # host logic only
    for eng in (a, b):
        eng.cfg, eng.dev, eng.max_positions = cfg, torch.device("cpu"), 4096
        eng._run_cached = lambda *_: None
    ids = np.zeros(20, np.int32)
    opened = a.open_cache(64, 2, 16)
    prefix = a.cache_prefix(opened, ids)
    own = StateCache(cfg, "cpu", 64, 2, 16)               # belongs to the first engine that uses it
    second = b.cache_prefix(own, ids)
    for eng, other, cache in ((b, prefix, opened), (a, second, own)):
        with pytest.raises(ValueError, match="another engine"):
            eng.score_after(other, [W.Request(ids=ids, slot=1, nopts=2)])
        with pytest.raises(ValueError, match="another engine"):
            eng.extend(other, ids)
        with pytest.raises(ValueError, match="another engine"):
            eng.cache_prefix(cache, ids)
        assert other.length == 20 and len(cache.free_pages) == 2 and len(cache.free_slots) == 1
    a.extend(prefix, ids[:4])
    assert prefix.length == 24


def test_the_c_library_builds_without_torch():
    # in a process where torch cannot be imported; the library here counts as up to date, so nothing is compiled
    code = ("import sys; sys.modules['torch'] = None; sys.path.insert(0, sys.argv[1]); import build; "
            "build._compile = lambda *_: ''; build.os.path.getmtime = lambda _: 0; print(build.build())")
    package = os.path.dirname(os.path.abspath(_lib.__file__))
    r = subprocess.run([sys.executable, "-c", code, package], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    said, path = r.stdout.strip().splitlines()
    assert "_fdk_torch.so is not built" in said and path == _lib.LIB_PATH
