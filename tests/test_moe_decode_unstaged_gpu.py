"""moe_decode with e4m3 weights and bf16 tokens: batches whose fp16 copies are kept in shared memory, and batches that are
converted as they are read.

Tolerance as in test_moe_decode_gpu.py: 4 u sum_e w_e |W2| |a|, u = 2^-9. The two ways convert alike (a power of two per row).
"""
import numpy as np
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg
from oracle.grouped_topk import grouped_topk_ref

pytestmark = pytest.mark.gpu

E, TOPK, N = 16, 4, 256


def layer(K, g):
    w1 = (torch.randn(E, 2 * N, K, generator=g, device="cuda") / K ** 0.5).bfloat16()
    w2 = (torch.randn(E, K, N, generator=g, device="cuda") / N ** 0.5).bfloat16()
    (q1, s1), (q2, s2) = pkg.quantize_weights_fp8(w1), pkg.quantize_weights_fp8(w2)
    full = [q.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2) for q, s in ((q1, s1), (q2, s2))]
    return q1, q2, s1, s2, *full


# 160 KB less the kernel's own tables hold 6 rows of 7168, 12 of 4096: both sides of it and beyond
@pytest.mark.parametrize("K,M", [(7168, 6), (7168, 7), (7168, 9), (7168, 10), (7168, 11), (7168, 32), (4096, 12),
                                 (4096, 13), (4096, 16), (4096, 17), (4096, 32)])
def test_layer(cuda_device, K, M):
    g = torch.Generator(device=cuda_device).manual_seed(M)
    q1, q2, s1, s2, d1, d2 = layer(K, g)
    # rows of very different sizes: each has a power of two of its own
    x = torch.randn(M, K, generator=g, device=cuda_device) * torch.exp2(torch.arange(M, device=cuda_device) % 9 - 4.0)[:, None]
    x = x.bfloat16()
    lg = torch.randn(M, E, generator=g, device=cuda_device)
    kw = dict(topk=TOPK, scoring_func="softmax", w1_scale=s1, w2_scale=s2)
    out = pkg.moe_decode(x, lg, q1, q2, **kw)
    assert torch.equal(out, pkg.moe_decode(x, lg, q1, q2, **kw))
    w, ids = grouped_topk_ref(lg.cpu().numpy(), TOPK, True, 1, 1, "softmax", 1.0, None, "max")
    ids = ids.astype(np.int64)
    for t in range(M):
        want = torch.zeros(K, dtype=torch.float64, device=cuda_device)
        mass = torch.zeros_like(want)
        for j in range(TOPK):
            h = d1[ids[t, j]] @ x[t].double()
            a = torch.nn.functional.silu(h[:N]) * h[N:]
            want += float(w[t, j]) * (d2[ids[t, j]] @ a)
            mass += abs(float(w[t, j])) * (d2[ids[t, j]].abs() @ a.abs())
        assert ((out[t].double() - want).abs() <= 4 * 2.0 ** -9 * mass).all(), t


@pytest.mark.parametrize("K,few,many", [(7168, 6, 7), (7168, 9, 10), (4096, 12, 13), (4096, 16, 17)])
def test_either_way(cuda_device, K, few, many):
    """One token more takes the other way; the sums are then cut elsewhere, so two roundings of values of order one."""
    g = torch.Generator(device=cuda_device).manual_seed(K)
    q1, q2, s1, s2, _, _ = layer(K, g)
    x = torch.randn(many, K, generator=g, device=cuda_device).bfloat16()
    x[2, 5], x[3, 9] = float("nan"), float("inf")
    lg = torch.randn(many, E, generator=g, device=cuda_device)
    kw = dict(topk=TOPK, scoring_func="softmax", w1_scale=s1, w2_scale=s2)
    a = pkg.moe_decode(x[:few].contiguous(), lg[:few].contiguous(), q1, q2, **kw)
    b = pkg.moe_decode(x, lg, q1, q2, **kw)[:few]
    keep = [t for t in range(few) if t not in (2, 3)]
    assert torch.isnan(a[2]).all() and torch.isnan(b[2]).all()
    assert not torch.isfinite(a[3]).any() and not torch.isfinite(b[3]).any()
    assert torch.isfinite(a[keep]).all() and torch.allclose(a[keep].float(), b[keep].float(), rtol=2 ** -6, atol=2 ** -6)
