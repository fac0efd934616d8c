"""Latent attention where numbers and offsets are large: scores of 1e5, caches and keys past 2^32 bytes."""
import math

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}
U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}


def src(kind):
    return torch.float16 if kind == "fp16" else torch.bfloat16


def soft(s, v):
    p = torch.softmax(s, -1)
    return p @ v, p @ v.abs(), torch.logsumexp(s, -1)


def close(got, want, mass, dt):
    # probabilities rounded for the second product, the result rounded once, a factor of two over both;
    # the scores here are exact in fp32, their differences too, so exp adds a few 2^-22 only
    assert ((got.double() - want).abs() <= (4 * U[dt] + 2.0 ** -10) * mass + 1e-30).all()


def large(n, sign):
    """Rotary parts whose scores are sign * 130050 + (0, 1, 2 or 3): 255 * 510 has 16 significant bits."""
    k = torch.zeros(n, 64)
    k[:, 0] = 255.0
    k[:, 1] = torch.arange(n) * 7 % 4
    q = torch.zeros(64)
    q[0], q[1] = sign * 510.0, 1.0
    return q, k


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("n", [3, 200, 2000])
def test_decode_large_scores(cuda_device, kind, n, sign):
    """Rows whose scores share 1.3e5 differ by up to 3: the common part has to cancel."""
    dt = src(kind)
    qr, kr = large(n, sign)
    g = torch.Generator().manual_seed(n)
    pages = -(-n // 64)
    cache = pkg.latent_cache(pages, 64, DT[kind], cuda_device)
    pkg.latent_cache_write(cache, torch.randn(n, 512, generator=g).to(dt).to(cuda_device),
                           kr.to(dt).to(cuda_device), torch.arange(n, device=cuda_device))
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    v = pkg.latent_cache_read(cache, table, torch.tensor([0, n], dtype=torch.int32, device=cuda_device), n)[0].double()
    q = torch.zeros(1, 1, 16, 576)
    q[..., 512:] = qr
    out, lse = pkg.latent_attention_decode(q.to(dt).to(cuda_device), cache, table, lens, 1.0, return_lse=True)
    pkg.check_device_status(cuda_device)
    s = (kr.double() @ qr.double()).to(cuda_device)
    want, mass, want_lse = soft(s[None], v)
    close(out[0, 0], want, mass, dt)
    assert ((lse.double() - want_lse).abs() <= 1e-6 * want_lse.abs()).all()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [3, 200, 1000])
def test_prefill_large_scores(cuda_device, dt, n, sign):
    qr, kr = large(n, sign)
    g = torch.Generator().manual_seed(n)
    kv = torch.randn(n, 2, 256, generator=g).to(dt).to(cuda_device)
    q = torch.zeros(5, 2, 192)
    q[..., 128:] = qr
    cu_q = torch.tensor([0, 5], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
    out, lse = pkg.latent_attention_prefill(q.to(dt).to(cuda_device), kv, kr.to(dt).to(cuda_device), cu_q, cu_k, 1.0,
                                            causal=False, return_lse=True)
    pkg.check_device_status(cuda_device)
    s = (kr.double() @ qr.double()).to(cuda_device)
    for h in range(2):
        want, mass, want_lse = soft(s[None], kv[:, h, 128:].double())
        close(out[:, h], want, mass, dt)
        assert ((lse[:, h].double() - want_lse).abs() <= 1e-6 * want_lse.abs()).all()


@pytest.mark.parametrize("kind,pages", [("bf16", 120000), ("e4m3", 105000)])
def test_cache_past_32_bits(cuda_device, kind, pages):
    """Pages on both sides of 2^31 and 2^32 bytes (bf16: of 2^32 elements' bytes too)."""
    dt, n, page = src(kind), 300, 64
    cache = pkg.latent_cache(pages, page, DT[kind], cuda_device)
    assert cache.numel() * cache.element_size() > 2 ** 32
    per = page * cache.shape[2] * cache.element_size()
    ids = [pages - 1, 2 ** 32 // per, 2 ** 31 // per, 1, pages - 2]
    table = torch.tensor([ids], dtype=torch.int32, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(n, 576, generator=g).to(dt).to(cuda_device)
    slots = torch.tensor([ids[j // page] * page + j % page for j in range(n)], device=cuda_device)
    pkg.latent_cache_write(cache, rows[:, :512], rows[:, 512:], slots)
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
    latent, rope = pkg.latent_cache_read(cache, table, cu, n)
    # the same rows in a small cache
    small = pkg.latent_cache(5, page, DT[kind], cuda_device)
    near = torch.arange(5, dtype=torch.int32, device=cuda_device)[None]
    pkg.latent_cache_write(small, rows[:, :512], rows[:, 512:], torch.arange(n, device=cuda_device))
    latent2, rope2 = pkg.latent_cache_read(small, near, cu, n)
    assert torch.equal(latent, latent2) and torch.equal(rope, rope2) and torch.equal(rope, rows[:, 512:])
    q = torch.randn(1, 1, 16, 576, generator=g).to(dt).to(cuda_device)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    far_out = pkg.latent_attention_decode(q, cache, table, lens, 1 / math.sqrt(192))
    assert torch.equal(far_out, pkg.latent_attention_decode(q, small, near, lens, 1 / math.sqrt(192)))
    k = torch.cat([latent, rope], 1).double()
    want, mass, _ = soft(q[0, 0].double() @ k.T / math.sqrt(192), latent.double())
    close(far_out[0, 0], want, mass, dt)
    pkg.check_device_status(cuda_device)


def test_prefill_past_32_bits(cuda_device):
    """The last request's keys begin past 2^31 elements of kv."""
    heads, skip, n, dt = 128, 66000, 500, torch.bfloat16
    kv = torch.zeros(skip + n, heads, 256, dtype=dt, device=cuda_device)
    assert skip * heads * 256 > 2 ** 31
    kv[skip:].normal_()
    kr = torch.zeros(skip + n, 64, dtype=dt, device=cuda_device)
    kr[skip:].normal_()
    q = torch.randn(130, heads, 192, device=cuda_device).to(dt)
    cu_q = torch.tensor([0, 0, 130], dtype=torch.int32, device=cuda_device)
    cu_k = torch.tensor([0, skip, skip + n], dtype=torch.int32, device=cuda_device)
    out = pkg.latent_attention_prefill(q, kv, kr, cu_q, cu_k, 1 / math.sqrt(192))
    alone = torch.tensor([0, 130], dtype=torch.int32, device=cuda_device)
    want = pkg.latent_attention_prefill(q, kv[skip:].clone(), kr[skip:].clone(), alone,
                                        torch.tensor([0, n], dtype=torch.int32, device=cuda_device),
                                        1 / math.sqrt(192))
    assert torch.equal(out, want) and want.float().abs().sum() > 0
    pkg.check_device_status(cuda_device)
