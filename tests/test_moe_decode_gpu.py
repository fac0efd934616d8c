"""moe_decode (a whole MoE layer for a few tokens) against 64-bit torch on the oracle's routing.

Tolerance, derived before any run: a_p is rounded once to the tokens' type (u = 2^-9 bf16, 2^-12 fp16,
taken at 2^-11) and the result once, so with A = sum_e w_e |W2| |a| the error stays under
u (A + |out|) <= 2 u A; fp32 sums of K and N products add at most (K + N) 2^-24 relative to the sums
of magnitudes, below u / 4 here for a_p's own magnitude sum, which the factor 4 u A covers.
"""
import numpy as np
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg
from oracle.grouped_topk import grouped_topk_ref

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}


def weights(E, K, N, kind, dt, g, fmt="ue8m0"):
    w1 = (torch.randn(E, 2 * N, K, generator=g) / K ** 0.5).to(dt).cuda()
    w2 = (torch.randn(E, K, N, generator=g) / N ** 0.5).to(dt).cuda()
    if kind != "e4m3":
        return w1, w2, None, None, w1.double(), w2.double()
    (q1, s1), (q2, s2) = pkg.quantize_weights_fp8(w1, fmt), pkg.quantize_weights_fp8(w2, fmt)
    full = [q.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2) for q, s in ((q1, s1), (q2, s2))]
    return q1, q2, s1, s2, *full


def reference(x, w, ids, d1, d2):
    out = torch.zeros(x.shape[0], d2.shape[1], dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(out)
    n = d2.shape[2]
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            h = d1[ids[t, j]] @ x[t].double()
            a = torch.nn.functional.silu(h[:n]) * h[n:]
            out[t] += float(w[t, j]) * (d2[ids[t, j]] @ a)
            mass[t] += abs(float(w[t, j])) * (d2[ids[t, j]].abs() @ a.abs())
    return out, mass


def run(M, E, topk, groups, tg, K, N, kind="bf16", scoring="sigmoid", bias=True, dt=torch.bfloat16, seed=0,
        fmt="ue8m0", logits=None, spread=1.0, renorm=True):
    g = torch.Generator().manual_seed(seed)
    w1, w2, s1, s2, d1, d2 = weights(E, K, N, kind, dt, g, fmt)
    x = (torch.randn(M, K, generator=g) * spread).to(dt).cuda()
    lg = torch.randn(M, E, generator=g) if logits is None else logits
    b = torch.randn(E, generator=g) * 0.01 if bias else None
    kw = dict(topk=topk, renormalize=renorm, num_expert_group=groups, topk_group=tg, scoring_func=scoring,
              routed_scaling_factor=2.5, e_score_correction_bias=None if b is None else b.cuda(), w1_scale=s1,
              w2_scale=s2)
    out = pkg.moe_decode(x, lg.cuda(), w1, w2, **kw)
    w, ids = grouped_topk_ref(lg.numpy(), topk, renorm, groups, tg, scoring, 2.5, None if b is None else b.numpy(),
                              "top2sum" if bias else "max")
    want, mass = reference(x, w, ids.astype(np.int64), d1, d2)
    tol = 4 * U[dt] * mass
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / tol).max())
    assert torch.equal(out, pkg.moe_decode(x, lg.cuda(), w1, w2, **kw))   # the same bits on every run
    return out, x, lg, w1, w2, kw


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 31, 32])
def test_layer(cuda_device, kind, dt, M):
    run(M, 64, 6, 8, 3, 512, 256, kind=kind, dt=dt, seed=M)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("E,topk,groups,tg,K,N,scoring,bias", [
    (8, 2, 1, 1, 256, 384, "softmax", False), (256, 8, 8, 4, 256, 128, "sigmoid", True),
    (1, 1, 1, 1, 128, 128, "softmax", False), (40, 3, 5, 2, 384, 128, "sigmoid", False),
    (512, 16, 16, 4, 128, 128, "softmax", False), (72, 32, 1, 1, 128, 256, "sigmoid", False)])
def test_layouts(cuda_device, kind, E, topk, groups, tg, K, N, scoring, bias):
    for M in (1, 5, 16):
        run(M, E, topk, groups, tg, K, N, kind=kind, scoring=scoring, bias=bias, seed=M)


def test_sixteen_bit_granularity(cuda_device):
    run(3, 8, 2, 1, 1, 192, 64, scoring="softmax", bias=False)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_crowded_experts(cuda_device, kind):
    """All tokens choose the same two experts: four chunks of eight each."""
    lg = torch.zeros(32, 16) + torch.arange(16).float() * 0.5
    run(32, 16, 2, 1, 1, 256, 128, kind=kind, logits=lg, scoring="softmax", bias=False)


def test_ties_take_the_lowest_expert(cuda_device):
    run(5, 16, 4, 1, 1, 128, 128, logits=torch.zeros(5, 16), scoring="sigmoid", bias=False)


def test_arbitrary_scales_and_large_tokens(cuda_device):
    run(4, 16, 4, 4, 2, 256, 256, kind="e4m3", fmt="fp32")
    run(4, 16, 4, 4, 2, 256, 256, kind="e4m3", spread=2e4)
    run(4, 16, 4, 4, 2, 256, 256, kind="e4m3", spread=1e-6, renorm=False)


def test_agrees_with_the_large_batch_layer(cuda_device):
    out, x, lg, w1, w2, kw = run(8, 64, 6, 8, 3, 512, 256)
    kw = {k: v for k, v in kw.items() if not k.endswith("_scale")}
    other = pkg.moe_layer(x, lg.cuda(), w1, w2, **kw)
    assert torch.allclose(out.float(), other.float(), atol=2e-2, rtol=2e-2)


def test_non_finite(cuda_device):
    out, x, lg, w1, w2, kw = run(5, 64, 6, 8, 3, 512, 256, kind="e4m3")
    bad = lg.clone()
    bad[2] = float("nan")
    got = pkg.moe_decode(x, bad.cuda(), w1, w2, **kw)
    assert torch.isnan(got[2]).all()
    keep = torch.tensor([0, 1, 3, 4], device="cuda")
    assert torch.equal(got[keep], out[keep])
    x2 = x.clone()
    x2[1, 3] = float("nan")
    got = pkg.moe_decode(x2, lg.cuda(), w1, w2, **kw)
    keep = torch.tensor([0, 2, 3, 4], device="cuda")
    assert torch.isnan(got[1]).all() and torch.equal(got[keep], out[keep])
    # a NaN code in one row of a down matrix: that output column of the tokens that chose the expert
    _, ids = pkg.grouped_topk(x, lg.cuda(), 6, True, 8, 3, "sigmoid", 2.5,
                              e_score_correction_bias=kw["e_score_correction_bias"])
    e = int(ids[3, 0])
    w3 = w2.clone()
    w3.view(torch.uint8)[e, 77, 200] = 0xFF
    got = pkg.moe_decode(x, lg.cuda(), w1, w3, **kw)
    hit = (ids == e).any(1)
    assert torch.isnan(got[hit, 77]).all() and torch.isfinite(got[~hit]).all()
    got[:, 77] = out[:, 77]
    assert torch.equal(got, out)


def test_strided_tokens_out_workspace_stream(cuda_device):
    out, x, lg, w1, w2, kw = run(6, 64, 6, 8, 3, 512, 256)
    wide = torch.randn(6, 800, device="cuda").to(x.dtype)
    for off in (0, 16, 3):   # the last is unaligned and copied
        view = wide[:, off:off + 512]
        view.copy_(x)
        o = torch.empty_like(out)
        ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            r = pkg.moe_decode(view, lg.cuda(), w1, w2, out=o, workspace=ws, **kw)
        side.synchronize()
        assert r is o and torch.equal(o, out)


def test_refusals(cuda_device):
    out, x, lg, w1, w2, kw = run(6, 64, 6, 8, 3, 512, 256)
    f, lg = pkg.moe_decode, lg.cuda()
    with pytest.raises(ValueError, match="at most 32 tokens"):
        f(x[:1].expand(33, -1), lg[:1].expand(33, -1), w1, w2, **kw)
    with pytest.raises(TypeError, match="not supported"):
        f(x.float(), lg, w1, w2, **kw)
    with pytest.raises(TypeError, match="dtype of hidden_states"):
        f(x, lg, w1.half(), w2.half(), **kw)
    with pytest.raises(ValueError, match="shape mismatch"):
        f(x, lg, w1, w2[:, :, :128], **kw)
    with pytest.raises(ValueError, match="gating_output"):
        f(x, lg[:5], w1, w2, **kw)
    with pytest.raises(ValueError, match="scoring_func"):
        f(x, lg, w1, w2, **{**kw, "scoring_func": "tanh"})
    with pytest.raises(ValueError, match="need w1_scale"):
        f(x, lg, w1.to(torch.float8_e4m3fn), w2.to(torch.float8_e4m3fn), **kw)
    with pytest.raises(ValueError, match="out must be"):
        f(x, lg, w1, w2, out=out[:, ::2], **kw)
    with pytest.raises(RuntimeError, match="unsupported shape"):
        f(x, lg, w1, w2, **{**kw, "topk_group": 9})
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(x.cpu(), lg, w1, w2, **kw)
    assert f(x[:0], lg[:0], w1, w2, **kw).shape == (0, 512)
    assert pkg.moe_decode_max_tokens(6) == 32 and pkg.moe_decode_max_tokens(32) == 16
