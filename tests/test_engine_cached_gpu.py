"""Requests behind a cached prefix (DecisionEngine.cache_prefix / extend / score_after): the whole run of
the cached operators through a model, against the oracle's float32 forward of the concatenated requests.

Bound: the smoke test's 0.03 on probabilities for a 4-layer bf16 forward against float32, which the
uncached engine is held to as well."""
import numpy as np
import pytest
import torch

from oracle import model as omodel

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from fastdecisions_b200 import _lib, workloads as W
    from fastdecisions_b200.engine import DecisionEngine, pack

BOUND = 0.03


@pytest.fixture(scope="module")
def setup():
    cfg = W.ModelConfig(num_hidden_layers=4, vocab_size=4096)
    weights = W.synthetic_weights(cfg)
    return cfg, weights, DecisionEngine(cfg, weights, "cuda")


def tokens(n, seed):
    return np.random.default_rng(seed).integers(0, 4096, size=n).astype(np.int32)


def questions(spec, seed):
    return [W.Request(ids=tokens(n, seed + i), slot=n - 1 - (i % 2 if n > 1 else 0), nopts=k)
            for i, (n, k) in enumerate(spec)]


def oracle(cfg, weights, prefix, reqs):
    full = [W.Request(ids=np.concatenate([prefix, r.ids]).astype(np.int32), slot=prefix.size + r.slot, nopts=r.nopts)
            for r in reqs]
    b = pack(full)
    probs, _ = omodel.decide(cfg.as_dict(), weights, W.letter_weight(weights), b.ids, b.cu_seqlens,
                             b.slots.astype(np.int64), b.nopts.astype(np.int64))
    return probs.numpy(), full


def check(got, want, bound=BOUND):
    assert got.shape == want.shape and np.isfinite(got).all()
    assert np.allclose(got[want == 0], 0)
    dp = np.abs(got - want).max()
    assert dp < bound, dp


@pytest.mark.parametrize("length", [1, 64, 150, 257])
@pytest.mark.parametrize("spec", [((7, 4), (1, 2), (20, 8)), ((90, 4), (3, 2), (140, 8), (33, 3))])
def test_score_after_prefix(setup, length, spec):
    # short questions take the recurrent delta rule and the few-row attention, long ones the chunked
    # delta rule and the tcgen05 attention; prefixes end at, inside and just behind a page
    cfg, weights, eng = setup
    cache = eng.open_cache(tokens=2048, prefixes=2)
    ids = tokens(length, length)
    prefix = eng.cache_prefix(cache, ids)
    reqs = questions(spec, 100)
    want, full = oracle(cfg, weights, ids, reqs)
    pages = len(cache.free_pages)
    for _ in range(2):  # the prefix is unchanged by its use
        check(eng.score_after(prefix, reqs), want)
    assert len(cache.free_pages) == pages
    check(eng.score(full), want)
    assert _lib.poll_device_error() == 0
    prefix.release()
    assert len(cache.free_pages) == 2048 // 64 and len(cache.free_slots) == 2


def test_extend_in_steps_of_any_size(setup):
    # a prefix grown token by token, by short and by long pieces is the prefix run at once
    cfg, weights, eng = setup
    cache = eng.open_cache(tokens=1024, prefixes=2, page_size=16)
    ids = tokens(200, 9)
    a = eng.cache_prefix(cache, ids)
    b = eng.cache_prefix(cache, ids[:3])
    at = 3
    for n in (1, 1, 2, 5, 1, 30, 100, 1, 56):
        eng.extend(b, ids[at:at + n])
        at += n
    assert at == 200 and a.length == b.length == 200
    reqs = questions(((5, 4), (40, 8)), 300)
    want, _ = oracle(cfg, weights, ids, reqs)
    check(eng.score_after(a, reqs), want)
    check(eng.score_after(b, reqs), want)
    assert _lib.poll_device_error() == 0


def test_small_cache_runs_in_several_batches_and_refuses(setup):
    cfg, weights, eng = setup
    cache = eng.open_cache(tokens=160, prefixes=1, page_size=16)  # ten pages, five of them the prefix's
    ids = tokens(70, 21)
    prefix = eng.cache_prefix(cache, ids)
    reqs = questions(((30, 4), (20, 2), (45, 8), (12, 3), (8, 5)), 400)
    want, _ = oracle(cfg, weights, ids, reqs)
    check(eng.score_after(prefix, reqs), want)
    assert eng.score_after(prefix, []).shape == (0, want.shape[1])
    with pytest.raises(RuntimeError, match="free"):
        eng.score_after(prefix, questions(((90, 4),), 1))
    with pytest.raises(RuntimeError, match="slot"):
        eng.cache_prefix(cache, ids)
    with pytest.raises(RuntimeError, match="pages"):
        eng.extend(prefix, tokens(200, 1))
    with pytest.raises(ValueError):
        eng.extend(prefix, tokens(0, 1))
    with pytest.raises(ValueError):
        eng.open_cache(tokens=10, kv_dtype="int8")
    check(eng.score_after(prefix, reqs), want)  # refusals changed nothing
    prefix.release()
    with pytest.raises(ValueError, match="released"):
        eng.score_after(prefix, reqs)
    assert len(cache.free_pages) == 10


def test_e4m3_cache(setup):
    # One layer of four reads the cache.  Its rows are off by at most 2^-4 each, independently, so
    # attention over more than a hundred rows moves by far less; the bound is doubled for it.
    cfg, weights, eng = setup
    cache = eng.open_cache(tokens=4096, prefixes=1, kv_dtype="e4m3")
    ids = tokens(500, 31)
    prefix = eng.cache_prefix(cache, ids)
    reqs = questions(((6, 4), (25, 2), (70, 8)), 500)
    want, _ = oracle(cfg, weights, ids, reqs)
    check(eng.score_after(prefix, reqs), want, 2 * BOUND)
    assert _lib.poll_device_error() == 0


def test_installed_recurrent_rule_decodes_like_the_models_own(setup):
    """transformers' cached forward, token by token behind a prompt, with the CUDA kernel in place of its
    recurrent delta rule.  The two differ by float32 rounding inside the rule and bf16 rounding of its
    output (2^-8); the framework's layer bound, 2e-2 of the largest output, covers that."""
    mq = pytest.importorskip("transformers.models.qwen3_5.modeling_qwen3_5")
    from fastdecisions_b200 import patches
    cfg, weights, _ = setup
    model = mq.Qwen3_5TextModel(cfg.to_transformers()).to("cuda", torch.bfloat16).eval()
    model.load_state_dict({k: v.to("cuda", torch.bfloat16) for k, v in weights.items()}, strict=False)
    prompt = torch.from_numpy(tokens(12, 77).astype(np.int64)).cuda()[None]

    def run():
        with torch.no_grad():
            out = model(input_ids=prompt[:, :8], use_cache=True)
            hidden = [out.last_hidden_state]
            for i in range(8, 12):
                out = model(input_ids=prompt[:, i:i + 1], past_key_values=out.past_key_values, use_cache=True)
                hidden.append(out.last_hidden_state)
        return torch.cat(hidden, 1).float()

    want = run()
    before = dict(_lib.call_counts)
    assert patches.install_recurrent_gated_delta_rule(model) == 3
    got = run()
    assert _lib.launches_since(before) == 3 * 4
    assert _lib.poll_device_error() == 0
    assert (got - want).abs().max().item() <= 2e-2 * want.abs().max().item()
