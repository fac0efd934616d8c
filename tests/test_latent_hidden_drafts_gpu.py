"""Absorbed latent attention: a draft token's non-finite row is kept from the rows before it in both CTAs of a pair, on
every run.

Four draft tokens of 32 heads fill the 128 rows of a pair: tokens 0 and 1 are the first CTA's, 2 and 3 the second's. Each CTA
brings in half of the values' columns, and either may be the one that finds the bad one. Tolerance as in
test_latent_attention_gpu.py: (4 u + 2^-10) sum p |v|.
"""
import math

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}
SCALE = 1 / math.sqrt(192)


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("column", [5, 200, 300, 511])
def test_both_ctas_are_told(cuda_device, kind, column):
    n_q, heads, page, lens = 4, 32, 64, [140 + 13 * i for i in range(90)]
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    pages = max(-(-n // page) for n in lens)
    cache = pkg.latent_cache(pages * len(lens), page, torch.float8_e4m3fn if kind == "e4m3" else dt, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(column)
    rows = torch.randn(len(lens), pages * page, 576, generator=g, device=cuda_device).to(dt)
    for b, n in enumerate(lens):
        rows[b, n - 1, column] = float("nan")   # the last draft token: tokens 0, 1 and 2 do not see it
    flat = rows.view(-1, 576)
    pkg.latent_cache_write(cache, flat[:, :512], flat[:, 512:], torch.arange(flat.shape[0], device=cuda_device))
    table = torch.arange(pages * len(lens), dtype=torch.int32, device=cuda_device).view(len(lens), pages)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    q = torch.randn(len(lens), n_q, heads, 576, generator=g, device=cuda_device).to(dt)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=cuda_device)
    first = None
    for i in range(60):
        if i & 1:
            flush.zero_()
        out = torch.full((len(lens), n_q, heads, 512), 7777.0, dtype=dt, device=cuda_device)
        _, lse = pkg.latent_attention_decode(q, cache, table, lens_t, SCALE, out=out, return_lse=True)
        if first is None:
            first = out, lse
        assert torch.isfinite(out[:, :3]).all(), f"run {i}"
        assert torch.equal(out[:, :3], first[0][:, :3]) and torch.equal(lse[:, :3], first[1][:, :3]), f"run {i}"
    pkg.check_device_status(cuda_device)
    assert torch.isnan(first[0][:, 3]).all()
    for b in (0, 1, 44, 89):
        n = lens[b]
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda_device)
        latent, rope = pkg.latent_cache_read(cache, table[b:b + 1], cu, n)
        k = torch.cat([latent, rope], 1).double()
        for i in range(3):
            seen = n - n_q + 1 + i
            p = torch.softmax(q[b, i].double() @ k[:seen].T * SCALE, -1)
            want, mass = p @ k[:seen, :512], p @ k[:seen, :512].abs()
            assert ((first[0][b, i].double() - want).abs() <= (4 * U[dt] + 2.0 ** -10) * mass).all()
