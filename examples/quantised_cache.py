"""Serving one attention layer from an 8-bit KV cache, with per-head q/k norms.

A batch of sequences of different lengths is prefilled and then decoded token by
token:

* prompt: the projections' packed output goes into ``QuantKVCache.append_qkv`` (norm,
  rotation and quantisation in one launch); the prompt's own attention runs on bf16 rows
  read back from the cache (``read``) with ``ops.gqa_prefill``, as a later chunk of a
  chunked prefill would;
* decode: one CUDA graph per step holds ``kvq_append_qkv`` and ``gqa_decode_kvq`` on
  static buffers.  Lengths live on the device, so the graph is captured once.

    python examples/quantised_cache.py [--fmt int8|fp8_e4m3] [--batch 8] [--prompt 500] [--steps 32]

prints the error of the last step against attention over unquantised K and V.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from lara_b200 import kvquant, ops  # noqa: E402

HQ, HKV, D, HIDDEN = 32, 8, 128, 1024


def run(fmt: str = "int8", batch: int = 8, prompt: int = 500, steps: int = 32, device: str = "cuda:0") -> dict:
    g = torch.Generator(device=device)
    g.manual_seed(0)
    dev = torch.device(device)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev).to(torch.bfloat16)

    w_qkv = randn(HIDDEN, (HQ + 2 * HKV) * D) * HIDDEN ** -0.5
    q_weight, k_weight = randn(D) * 0.1 + 1.0, randn(D) * 0.1 + 1.0
    cos_sin = ops.rope_table(prompt + steps, D, base=500000.0, device=dev)
    norm = dict(cos_sin=cos_sin, q_weight=q_weight, k_weight=k_weight, interleaved=False)

    def project(x):  # [batch, n, hidden] -> q, k, v views [batch, n, heads, D]
        y = (x @ w_qkv).view(*x.shape[:2], HQ + 2 * HKV, D)
        return y[:, :, :HQ], y[:, :, HQ:HQ + HKV], y[:, :, HQ + HKV:]

    # ---- prompts, each of its own length ----
    page = 64
    cache = kvquant.QuantKVCache(num_pages=batch * (-(-(prompt + steps) // page)), page_size=page, n_kv_heads=HKV,
                                 head_dim=D, max_seqs=batch, max_seq_len=prompt + steps, device=dev, fmt=fmt)
    lens = [max(1, prompt - 37 * i) for i in range(batch)]
    slots = [cache.new_sequence() for _ in lens]
    xs = [randn(1, n + steps, HIDDEN) for n in lens]
    for slot, n, x in zip(slots, lens, xs):
        q = cache.append_qkv(*project(x[:, :n]), slots=[slot], **norm)
        k, v = cache.read([slot])
        zero = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.gqa_prefill(q, k, v, zero)  # the prompt's outputs, [1, n, HQ, D]

    # ---- decode: static buffers, one graph for every step ----
    cache.reserve(slots, steps)
    table = cache.block_table[:batch].contiguous()
    starts = cache.lens[:batch].clone()
    now = torch.empty_like(starts)
    ws = kvquant.decode_workspace(batch, HQ, HKV, D, dev)
    status = ops.new_workspace(256, dev)
    qkv = torch.empty((batch, 1, HQ + 2 * HKV, D), dtype=torch.bfloat16, device=dev)
    q_new = torch.empty((batch, 1, HQ, D), dtype=torch.bfloat16, device=dev)
    out = torch.empty((batch, HQ, D), dtype=torch.bfloat16, device=dev)

    def step():
        kvquant.kvq_append_qkv(cache.pool, table, starts, qkv[:, :, :HQ], qkv[:, :, HQ:HQ + HKV],
                               qkv[:, :, HQ + HKV:], new_lens=now, workspace=status, out=q_new, **norm)
        kvquant.gqa_decode_kvq(q_new[:, 0], cache.pool, table, now, workspace=ws, out=out)
        starts.copy_(now)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(steps):
        x = torch.cat([xs[b][:, n + i] for b, n in enumerate(lens)])  # [batch, hidden]
        qkv.copy_((x @ w_qkv).view_as(qkv))
        graph.replay()
    torch.cuda.synchronize(dev)
    bits = ops.workspace_status(status) | ops.workspace_status(ws) | cache.status()

    # ---- the last step against unquantised K and V ----
    worst = 0.0
    for b, n in enumerate(lens):
        q, k, v = project(xs[b])
        pos = torch.arange(n + steps, dtype=torch.int32, device=dev)[None]
        q, k = ops.qk_norm_rope(q, k, positions=pos, **norm)
        kf, vf = (t[0].float().repeat_interleave(HQ // HKV, 1) for t in (k, v))
        p = torch.softmax(torch.einsum("hd,thd->ht", q[0, -1].float(), kf) / math.sqrt(D), -1)
        ref = torch.einsum("ht,thd->hd", p, vf)
        worst = max(worst, ((out[b].float() - ref).norm() / ref.norm()).item())
    return dict(fmt=fmt, batch=batch, cached_tokens=sum(lens) + batch * steps, status=bits, relative_error=worst,
                lens=now.tolist(), expected_lens=[n + steps for n in lens],
                bytes_per_token=2 * HKV * (D + 4), bytes_per_token_bf16=2 * HKV * D * 2)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--fmt", choices=["int8", "fp8_e4m3"], default="int8")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=32)
    r = run(**vars(ap.parse_args()))
    r.pop("lens"), r.pop("expected_lens")
    print(r)


if __name__ == "__main__":
    main()
