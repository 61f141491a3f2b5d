"""Several sampled continuations of one prompt on one GPU: the prompt is read once, its cache pages are shared.

    python examples/shared_prompt.py [--streams 8] [--prompt 1000] [--tokens 64] [--layers 4]

A synthetic model (the shapes of bench.py with --layers layers, random NVFP4 weights) reads a random prompt whole, forks
its pages to the streams, samples a token per stream and step, lets half of the streams go on from stream 0 half way, and
compacts the cache at the end.  Prints the times and the pages in use.
"""
import argparse
import importlib.util
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load_package():
    folder = os.path.join(ROOT, "flint-vllm-single-dgx-spark_b200")
    spec = importlib.util.spec_from_file_location("flint_b200", os.path.join(folder, "__init__.py"),
                                                  submodule_search_locations=[folder])
    sys.modules["flint_b200"] = module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)


def timed(what, fn):
    torch.cuda.synchronize()
    t = time.perf_counter()
    fn()
    torch.cuda.synchronize()
    print(f"{what}: {(time.perf_counter() - t) * 1e3:.2f} ms")


def main():
    ap = argparse.ArgumentParser()
    for name, default in (("streams", 8), ("prompt", 1000), ("tokens", 64), ("layers", 4), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=default)
    a = ap.parse_args()
    load_package()
    from flint_b200.model import FlintConfig, FlintModel
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = FlintModel(FlintConfig(layers=a.layers), "cuda", seed=a.seed, max_ctx=a.prompt + a.tokens + 16,
                       max_batch=a.streams, weights="codes")
    dec = SharedPromptDecoder(model, a.streams, sampling=dict(temperature=1.0, top_k=20, top_p=0.95,
                                                              seeds=list(range(a.streams))))
    dec.reserve_history(a.tokens)
    dec.capture()
    prompt = np.random.default_rng(a.seed).integers(0, model.cfg.vocab, size=a.prompt)
    dec.read_prompt(prompt, room=a.tokens)                    # first use: workspaces
    timed(f"prompt of {a.prompt} tokens read and forked to {a.streams} streams",
          lambda: dec.read_prompt(prompt, room=a.tokens))
    half = a.tokens // 2
    step = dec.graphs["step"].replay
    timed(f"{half} steps", lambda: [step() for _ in range(half)])
    late = list(range(a.streams // 2 + 1, a.streams))
    if late:
        timed(f"streams {late} go on from stream 0", lambda: dec.branch(late, [0] * len(late)))
    timed(f"{a.tokens - half} steps", lambda: [step() for _ in range(a.tokens - half)])
    timed("compact", dec.compact)
    dec.check_status()
    alone = a.streams * (-(-(a.prompt + a.tokens) // 16))
    print(f"pages in use: {int(dec.pool.live.item())} (without sharing {alone})")
    print("first tokens:", dec.history[:, :8].tolist())
    dec.close()


if __name__ == "__main__":
    main()
