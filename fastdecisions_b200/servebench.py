"""Serving-path timing: decision requests scored one call at a time, eager vs bucketed CUDA graphs.

    python -m fastdecisions_b200.servebench [--requests 64] [--per-call 1]

The first ``--requests`` requests of the config-5 mix (synthetic config-4 model) go through
``DecisionEngine.score`` ``--per-call`` at a time, once with eager launches and once with
``graphs=True`` (after one warm-up pass that captures the buckets, then ``seal()``; batches of more
than ``GRAPH_MAX_REQUESTS`` requests launch eagerly either way).  Reports
wall-clock requests/s (host token ids to host probabilities, the synchronising D2H included) and
the device time of the same calls, so the host-dispatch share is visible.  One JSON line per mode.

    python -m fastdecisions_b200.servebench --shared-prefix 1536 [--requests 64] [--suffix 40] [--kv-dtype e4m3]

``--requests`` requests of about ``--suffix`` tokens each behind one prefix: every request run in full
(``score``) against the prefix cached once and the requests' own tokens run behind it
(``cache_prefix`` + ``score_after``; the prefix's own run is timed too).
"""
from __future__ import annotations

import argparse
import json
import time

import numpy as np
import torch

from . import workloads as W
from .engine import DecisionEngine


def shared_prefix(eng, cfg, args):
    rng = np.random.default_rng(17)
    prefix_ids = rng.integers(0, cfg.vocab_size, size=args.shared_prefix).astype(np.int32)
    lens = rng.integers(max(1, args.suffix // 2), args.suffix * 3 // 2 + 1, size=args.requests)
    tails = [W.Request(ids=rng.integers(0, cfg.vocab_size, size=int(n)).astype(np.int32), slot=int(n) - 1, nopts=4)
             for n in lens]
    full = [W.Request(ids=np.concatenate([prefix_ids, r.ids]), slot=prefix_ids.size + r.slot, nopts=4) for r in tails]
    cache = eng.open_cache(args.shared_prefix + args.requests * (3 * args.suffix + 64), 1, kv_dtype=args.kv_dtype)

    def timed(fn, times=5):
        for _ in range(2):
            fn()
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(times):
            fn()
        torch.cuda.synchronize()
        return (time.perf_counter() - t0) / times

    def prefill():
        eng.cache_prefix(cache, prefix_ids).release()

    whole, once = timed(lambda: eng.score(full)), timed(prefill)
    prefix = eng.cache_prefix(cache, prefix_ids)
    after = timed(lambda: eng.score_after(prefix, tails))
    dp = float(np.abs(eng.score_after(prefix, tails) - eng.score(full)).max())
    print(json.dumps({"mode": "shared prefix", "prefix_tokens": args.shared_prefix, "requests": args.requests,
                      "suffix_tokens": int(lens.sum()), "kv_dtype": args.kv_dtype, "full_ms": round(1e3 * whole, 2),
                      "prefix_ms": round(1e3 * once, 2), "after_ms": round(1e3 * after, 2),
                      "speedup": round(whole / (once + after), 2), "max_dp": round(dp, 4)}), flush=True)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--per-call", type=int, default=1)
    ap.add_argument("--max-len", type=int, default=8192)
    ap.add_argument("--shared-prefix", type=int, default=0)
    ap.add_argument("--suffix", type=int, default=40)
    ap.add_argument("--kv-dtype", choices=("bf16", "e4m3"), default="bf16")
    args = ap.parse_args(argv)
    cfg = W.ModelConfig()
    eng = DecisionEngine(cfg, W.synthetic_weights(cfg), "cuda")
    if args.shared_prefix:
        return shared_prefix(eng, cfg, args)
    reqs = [r for r in W.config5_requests(256) if r.ids.size <= args.max_len][:args.requests]
    calls = [reqs[i:i + args.per_call] for i in range(0, len(reqs), args.per_call)]
    for graphs in (False, True):
        for c in calls:  # warm-up (captures every bucket the calls need)
            eng.score(c, graphs=graphs)
        if graphs:
            eng.seal()
        torch.cuda.synchronize()
        dev_ms = 0.0
        t0 = time.perf_counter()
        for c in calls:
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            eng.score(c, graphs=graphs)
            e1.record()
            e1.synchronize()
            dev_ms += e0.elapsed_time(e1)
        wall = time.perf_counter() - t0
        print(json.dumps({"mode": "cuda graphs (bucketed)" if graphs else "eager launches",
                          "requests": len(reqs), "per_call": args.per_call,
                          "tokens": int(sum(r.ids.size for r in reqs)), "requests_per_s": round(len(reqs) / wall, 2),
                          "wall_ms_per_call": round(1000 * wall / len(calls), 3),
                          "stream_ms_per_call": round(dev_ms / len(calls), 3),
                          "graph_captures": eng.stats["graph_captures"]}), flush=True)


if __name__ == "__main__":
    main()
