"""Expanded latent attention, causal: a non-finite value of a later token reaches no row before it, on every run.

The kernel walks 256 query rows as two subtiles of 128 and keys in tiles of 128. Rows of a subtile whose tiles end before
the value have to have the bits of a run without it, and every other row before it its own values: no row may be left
unwritten (the outputs start from a mark) or depend on when a tile lands. Tolerance as in test_latent_attention_gpu.py:
(4 u + 2^-10) sum p |v| for probabilities and results rounded to the type and fp32 scores; 1e-4 (1 + |lse|) for lse.
"""
import math

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

SCALE = 1 / math.sqrt(192)
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}
MARK = 7777.0


def attend(q, kv, kr, cu_q, cu_k):
    out = torch.full((*q.shape[:2], 128), MARK, dtype=q.dtype, device=q.device)
    _, lse = pkg.latent_attention_prefill(q, kv, kr, cu_q, cu_k, SCALE, out=out, return_lse=True)
    return out, lse


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,hist,place", [
    ([256, 200, 129], [0, 0, 0], [140, 199, 128]),          # the second subtile's only tile of its own
    ([511, 700, 300], [0, 70, 1000], [390, 650, 1290]),     # histories: limits inside tiles
])
def test_later_values_reach_no_row(cuda_device, dt, value, new, hist, place):
    heads = 128
    lens = [n + h for n, h in zip(new, hist)]
    g = torch.Generator(device=cuda_device).manual_seed(sum(lens))
    q = torch.randn(sum(new), heads, 192, generator=g, device=cuda_device).to(dt)
    kv = torch.randn(sum(lens), heads, 256, generator=g, device=cuda_device).to(dt)
    kr = torch.randn(sum(lens), 64, generator=g, device=cuda_device).to(dt)
    cu_q = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda_device)
    cu_k = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda_device)
    clean, clean_lse = attend(q, kv, kr, cu_q, cu_k)
    bad = kv.clone()
    for b, p in enumerate(place):
        bad[int(cu_k[b]) + p, :, 128 + 77] = value
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=cuda_device)
    first = None
    for i in range(60):
        if i & 1:
            flush.zero_()
        out, lse = attend(q, bad, kr, cu_q, cu_k)
        if first is None:
            first = out, lse
        assert torch.equal(out.nan_to_num(1e4, 2e4, 3e4), first[0].nan_to_num(1e4, 2e4, 3e4)), f"run {i}"
        assert torch.equal(lse, first[1]), f"run {i}"
    pkg.check_device_status(cuda_device)
    out, lse = first
    for b, (n, h, p) in enumerate(zip(new, hist, place)):
        o, w, at = out[cu_q[b]:cu_q[b + 1]], clean[cu_q[b]:cu_q[b + 1]], p - h   # query `at` is the first to see key p
        s, ws = lse[cu_q[b]:cu_q[b + 1]], clean_lse[cu_q[b]:cu_q[b + 1]]
        # subtiles (row, row + 128) whose last row sees keys of tiles before the value's only
        ends = torch.tensor([-(-(min(r // 128 * 128 + 128, n) + h) // 128) * 128 for r in range(n)])
        apart = (ends <= p).to(cuda_device)
        assert torch.equal(o[apart], w[apart]) and torch.equal(s[apart], ws[apart])
        assert not torch.isfinite(o[at:, :, 77]).any() and not (o == MARK).any()
        # the rows between, and those after in the other values, against 64 bits (a few heads)
        for head in (0, 1, 63, 127):
            k = torch.cat([kv[cu_k[b]:cu_k[b + 1], head, :128], kr[cu_k[b]:cu_k[b + 1]]], 1).double()
            sc = q[cu_q[b]:cu_q[b + 1], head].double() @ k.T * SCALE
            hide = torch.arange(n + h, device=cuda_device) > torch.arange(n, device=cuda_device)[:, None] + h
            sc = sc.masked_fill(hide, float("-inf"))
            pr, v = torch.softmax(sc, -1), kv[cu_k[b]:cu_k[b + 1], head, 128:].double()
            off = (o[:, head].double() - pr @ v).abs() > (4 * U[dt] + 2.0 ** -10) * (pr @ v.abs())
            off[at:, 77] = False
            assert not off.any() and torch.isfinite(o[:at, head]).all()
            want = torch.logsumexp(sc, -1)
            assert ((s[:, head].double() - want).abs() <= 1e-4 * (1 + want.abs())).all()
