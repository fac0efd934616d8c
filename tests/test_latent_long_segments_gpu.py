"""A non-finite draft token at the end of a very long context: the key-by-key path takes longer than the kernel's waits may
(2 s), and the call still gives its answer and no timeout.

All table entries but the last two name one page, so the context is that page's keys many times over and the softmax is the
one of 128 keys with a count. Two requests per CTA pair, the bad token in every other one. Scores are small, so that the
terms of the fp32 sums over half a million keys are alike. Tolerance as in test_latent_attention_gpu.py, (4 u + 2^-10) sum p |v|.
"""
import time

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

KEYS = 500_000


def test_long_segment(cuda_device):
    n_q, heads, page, B, dt = 2, 64, 128, 148, torch.bfloat16
    width = KEYS // page
    n = width * page
    g = torch.Generator(device=cuda_device).manual_seed(3)
    cache = pkg.latent_cache(3, page, dt, cuda_device)
    rows = torch.randn(3 * page, 576, generator=g, device=cuda_device).to(dt)
    rows[2 * page:] = rows[page:2 * page]
    rows[3 * page - 1, 77] = float("nan")        # page 2: page 1 with a bad last token
    pkg.latent_cache_write(cache, rows[:, :512], rows[:, 512:], torch.arange(3 * page, device=cuda_device))
    table = torch.zeros(B, width, dtype=torch.int32, device=cuda_device)
    table[:, -1] = 1
    table[::2, -1] = 2
    lens = torch.full((B,), n, dtype=torch.int32, device=cuda_device)
    q = (torch.randn(B, n_q, heads, 576, generator=g, device=cuda_device) * 0.01).to(dt)
    torch.cuda.synchronize()
    t0 = time.monotonic()
    out = pkg.latent_attention_decode(q, cache, table, lens, 0.07)
    torch.cuda.synchronize()
    took = time.monotonic() - t0
    pkg.check_device_status(cuda_device)
    assert took > 2.5, f"{took:.2f} s: too short to show anything"
    k = rows[:2 * page].double()
    count = torch.full((2 * page,), 1.0, device=cuda_device, dtype=torch.float64)
    count[:page] = width - 1
    for b in (0, 1, 2, 73, 74, 146, 147):
        for i in range(n_q):
            if b % 2 == 0 and i == 1:
                assert torch.isnan(out[b, i]).all()
                continue
            c = count.clone()
            if i == 0:
                c[-1] = 0   # token 0 does not see the last position
            e = c * torch.exp(q[b, i].double() @ k.T * 0.07)
            p = e / e.sum(-1, keepdim=True)
            want, mass = p @ k[:, :512], p @ k[:, :512].abs()
            assert ((out[b, i].double() - want).abs() <= (4 * 2.0 ** -9 + 2.0 ** -10) * mass).all()
