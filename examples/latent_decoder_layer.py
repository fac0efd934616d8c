"""One DeepSeek-V3-style decoder layer (latent attention, mixture of experts) serving a small batch.

A prompt step writes the cache, reads it back and attends in the expanded form; every later step
appends one token per request, attends in the absorbed form over the paged cache, and runs the
experts with the few-token kernels. Norms, positions and the dense projections are plain torch.

    python examples/latent_decoder_layer.py --steps 4 --cache e4m3
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import kernelswift_competition_submission_b200 as pkg  # noqa: E402

CACHES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


class Layer:
    """Random weights; hidden, heads and experts as given, latent 512 + rotary 64 as the kernels have them."""

    def __init__(self, hidden=512, heads=16, experts=16, topk=4, groups=4, topk_group=2, inter=256, pages=64,
                 page_size=64, cache="bf16", device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) / math.sqrt(shape[-1])).bfloat16()

        self.heads, self.topk, self.groups, self.topk_group = heads, topk, groups, topk_group
        self.w_q, self.w_c = w(heads * 192, hidden), w(576, hidden)
        self.w_uk, self.w_uv = w(heads, 128, 512), w(heads, 128, 512)
        self.w_o = w(hidden, heads * 128)
        self.gate, self.bias = w(experts, hidden), 0.01 * torch.randn(experts, generator=g, device=device)
        self.w1, self.w2 = w(experts, 2 * inter, hidden), w(experts, hidden, inter)
        self.scale = 1.0 / math.sqrt(192)
        self.page_size = page_size
        self.cache = pkg.latent_cache(pages, page_size, CACHES[cache], device)

    def append(self, x, table, seq, pos):
        """Writes tokens x [n, hidden], token i at position pos[i] of request seq[i]."""
        c = x @ self.w_c.T
        page = table[seq, pos // self.page_size].long()
        pkg.latent_cache_write(self.cache, c[:, :512], c[:, 512:], page * self.page_size + pos % self.page_size)

    def attend_prompt(self, x, table, cu):
        """All tokens of all requests at once: expanded form over what the cache holds."""
        n = x.shape[0]
        q = (x @ self.w_q.T).view(n, self.heads, 192)
        latent, rope = pkg.latent_cache_read(self.cache, table, cu, n)
        up = torch.cat([self.w_uk, self.w_uv], 1)                      # [heads, 256, 512]
        kv = (latent @ up.reshape(-1, 512).T).view(n, self.heads, 256)
        return pkg.latent_attention_prefill(q, kv, rope, cu, cu, self.scale)

    def attend_step(self, x, table, lens):
        """One token per request: absorbed form, the cache's rows are keys and values."""
        q = (x @ self.w_q.T).view(-1, self.heads, 192)
        absorbed = torch.einsum("bhd,hdc->bhc", q[..., :128], self.w_uk)
        q = torch.cat([absorbed, q[..., 128:]], -1)[:, None]
        o = pkg.latent_attention_decode(q, self.cache, table, lens, self.scale)[:, 0]
        return torch.einsum("bhc,hdc->bhd", o, self.w_uv)

    def experts(self, x):
        g = (x @ self.gate.T).float()
        rule = dict(topk=self.topk, renormalize=True, num_expert_group=self.groups, topk_group=self.topk_group,
                    scoring_func="sigmoid", routed_scaling_factor=2.5, e_score_correction_bias=self.bias)
        if x.shape[0] <= pkg.moe_decode_max_tokens(self.topk):
            return pkg.moe_decode(x, g, self.w1, self.w2, **rule)
        weights, ids = pkg.grouped_topk(x, g, **rule)
        return pkg.fused_moe(x, self.w1, self.w2, weights, ids)

    def finish(self, x, attended):
        h = x + attended.reshape(x.shape[0], -1) @ self.w_o.T
        return h + self.experts(torch.nn.functional.rms_norm(h, h.shape[-1:]))


def run(prompts=(70, 1, 200), steps=4, cache="bf16", device="cuda", **sizes):
    """Serves the prompts and ``steps`` tokens each. Returns the layer's last output [requests, hidden] and the
    largest difference, relative to the largest value, of the two attention forms on the prompts' last tokens."""
    device = torch.device("cuda", torch.cuda.current_device()) if device == "cuda" else torch.device(device)
    layer = Layer(cache=cache, device=device, **sizes)
    hidden, B = layer.w_c.shape[1], len(prompts)
    need = [-(-(n + steps) // layer.page_size) for n in prompts]
    table = torch.zeros(B, max(need), dtype=torch.int32, device=device)
    order, o = torch.randperm(layer.cache.shape[0]).to(torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = order[o:o + n].to(device)
        o += n
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(sum(prompts), hidden, generator=g, device=device).bfloat16()
    lens = torch.tensor(prompts, dtype=torch.int32, device=device)
    cu = torch.cat([lens.new_zeros(1), lens.cumsum(0).to(torch.int32)])
    seq = torch.repeat_interleave(torch.arange(B, device=device), lens)
    layer.append(x, table, seq, torch.cat([torch.arange(n, device=device) for n in prompts]))
    attended = layer.attend_prompt(x, table, cu)
    last = cu[1:].long() - 1
    other = layer.attend_step(x[last], table, lens)
    gap = float((other - attended[last]).abs().max() / attended[last].abs().max())
    x = layer.finish(x, attended)[last]
    for _ in range(steps):
        layer.append(x, table, torch.arange(B, device=device), lens.long())
        lens = lens + 1
        x = layer.finish(x, layer.attend_step(x, table, lens))
        x = torch.nn.functional.rms_norm(x, x.shape[-1:])
    pkg.check_device_status(device)
    return x, gap


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--steps", type=int, default=4)
    p.add_argument("--cache", choices=sorted(CACHES), default="bf16")
    a = p.parse_args()
    y, gap = run(steps=a.steps, cache=a.cache)
    print(f"{a.steps} steps of {y.shape[0]} requests; the two attention forms differ by {gap:.4f} of the largest value")
