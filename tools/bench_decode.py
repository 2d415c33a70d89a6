"""Serving benchmark: autoregressive decode throughput of a config (default the flagship GPT-Neo-1.3B; also
ctx32_mixer, whose learned token mixer decodes from per-layer input caches) on one GPU.

Two samplers over the same random-init model and synthetic prompts (``run/infer.py::Sampler``):
  * ``kv``   -- one prefill forward over the prompt, then one single-token forward per generated token over the
                per-layer KV caches (``csrc/kernels/aux_ops.hip::decode_attn_kernel``);
  * ``kv_paged`` -- the same over paged caches (``--page``, ``csrc/kernels/paged.hip``);
  * ``kv_eager`` -- the same without the hipGraph replay of the decode step (``--eager``);
  * ``full`` -- the reference's loop (ref src/run/inference.py:77-97): the whole causal context is recomputed for
                every generated token.
Prints one JSON line per sampler: generated tokens/s over the whole batch, and ms per generated token step.

    python tools/bench_decode.py --batch 32 --prompt 512 --new 128 [--full-new 16]
"""
import argparse
import json
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from homebrewnlp_mtf_amd.config import load_config  # noqa: E402
from homebrewnlp_mtf_amd.models.model import Model  # noqa: E402
from homebrewnlp_mtf_amd.ops import _lib  # noqa: E402
from homebrewnlp_mtf_amd.parallel import state as pstate  # noqa: E402
from homebrewnlp_mtf_amd.run.infer import Sampler  # noqa: E402


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--config", default=os.path.join(os.path.dirname(__file__), "..", "configs", "gpt_neo_1.3b.json"))
    ap.add_argument("--batch", type=int, default=32)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--new", type=int, default=128)
    ap.add_argument("--full-new", type=int, default=16, help="tokens generated by the recompute sampler (0: skip)")
    ap.add_argument("--eager", action="store_true", help="also time KV decoding without the hipGraph")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--page", type=int, default=0, help="kv_page_size: also time decoding over paged caches")
    a = ap.parse_args()
    _lib.lib()
    pstate.set_mesh(pstate.Mesh())
    S = a.prompt + max(a.new, a.full_new)
    p = load_config(a.config, {"sequence_length": S, "train_batch_size": a.batch})
    dev = "cuda:0"
    torch.manual_seed(0)
    model = Model(p, dev)
    x0 = torch.randint(0, p.vocab_size, (a.batch, S, 1), device=dev)
    results = {}
    for name, new in (("kv", a.new), ("kv_paged", a.new if a.page else 0), ("kv_eager", a.new if a.eager else 0),
                      ("full", a.full_new)):
        if new <= 0:
            continue
        p.decode_hip_graphs = name in ("kv", "kv_paged")
        p.kv_page_size = a.page if name == "kv_paged" else 0
        s = Sampler(model, p, dev)
        s.kv_cache = name != "full"
        if name == "kv" and not model.supports_kv_cache():
            raise SystemExit("config is not KV-cache decodable")
        # warmup (prefill + a few steps; paged: the same pages as the timed run, so that its graph stays), then the timed run
        s.sample(x0.clone(), a.prompt, a.temperature, a.prompt + (new if name == "kv_paged" else min(4, new)))
        torch.cuda.synchronize()
        x = x0.clone()
        t0 = time.perf_counter()
        out = s.sample(x, a.prompt, a.temperature, a.prompt + new)
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
        results[name] = out
        cfg_name = os.path.splitext(os.path.basename(a.config))[0]
        line = {"metric": f"decode tokens/s ({name}), {cfg_name}", "sampler": name, "value": round(a.batch * new / dt, 1),
                "unit": "tokens/s", "batch": a.batch, "prompt": a.prompt, "new_tokens": new,
                "ms_per_token_step": round(1e3 * dt / new, 3), "total_s": round(dt, 3), "dtype": "bf16",
                "data": "synthetic prompts, random-init weights", "includes_prefill": True}
        print(json.dumps(line), flush=True)
    if "kv_paged" in results:
        agree = (results["kv"][:, a.prompt:] == results["kv_paged"][:, a.prompt:]).float().mean().item()
        print(json.dumps({"token_agreement_kv_vs_kv_paged": round(agree, 4)}), flush=True)
    if "kv" in results and "full" in results:
        n = a.prompt + min(a.new, a.full_new)
        agree = (results["kv"][:, a.prompt:n] == results["full"][:, a.prompt:n]).float().mean().item()
        print(json.dumps({"token_agreement_kv_vs_full": round(agree, 4), "compared_tokens": n - a.prompt}), flush=True)


if __name__ == "__main__":
    main()
