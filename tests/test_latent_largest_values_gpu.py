"""e4m3 pages at the top of bf16's range: what is finite stays finite."""
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

TOP = float(torch.finfo(torch.bfloat16).max)   # 255 * 2^120


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_finite_values_read_back_finite(cuda_device, sign):
    """All bf16 values from 2^127 up beside smaller ones: the code nearest to x / 2^120 that is finite when read back."""
    x = torch.zeros(4, 512)
    x[:, :128] = sign * (torch.arange(128) + 128) * 2.0 ** 120   # 128 .. 255
    x[1, 128:256] = sign * 2.0 ** 119
    x[1, 200] = sign * TOP
    x[2, 384:] = 223 * 2.0 ** 120                                # the largest block under scale 2^119
    x = x.bfloat16().to(cuda_device)
    cache = pkg.latent_cache(1, 16, torch.float8_e4m3fn, cuda_device)
    rope = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda_device)
    pkg.latent_cache_write(cache, x, rope, torch.arange(4, device=cuda_device))
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    got, _ = pkg.latent_cache_read(cache, table, torch.tensor([0, 4], dtype=torch.int32, device=cuda_device), 4)
    b = x.double().cpu().view(4, 4, 128)
    amax = b.abs().amax(-1, keepdim=True)
    s = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp_min(-126)), torch.ones_like(amax))
    q = (b / s).float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    back = q * s
    back = torch.where(back.abs() >= 2.0 ** 128, back * (15 / 16), back)
    assert torch.isfinite(got).all()
    assert torch.equal(got.double().cpu().view(4, 4, 128), back)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("byte", [247, 254])
def test_hidden_codes_that_widen_to_infinity(cuda_device, page, byte):
    """A draft token whose code is infinite under its scale (pages that another program wrote) reaches no row before it."""
    n, n_q, heads, place = 140, 3, 16, 138   # query 0 sees other keys of the tile
    pages = -(-n // page)
    cache = pkg.latent_cache(pages, page, torch.float8_e4m3fn, cuda_device)
    g = torch.Generator().manual_seed(byte)
    rows = torch.randn(n, 576, generator=g).bfloat16().to(cuda_device)
    pkg.latent_cache_write(cache, rows[:, :512], rows[:, 512:], torch.arange(n, device=cuda_device))
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    q = torch.randn(1, n_q, heads, 576, generator=g).bfloat16().to(cuda_device)
    want = pkg.latent_attention_decode(q, cache, table, lens, 0.07)
    flat, at = cache.view(pages, -1)[place // page], place % page
    flat[at * 512 + 300] = 0x7E                                 # 448
    flat[page * 640 + at * 4 + 2] = byte                        # the scale of values 256 .. 383
    for i in range(256, 384):
        if i != 300:
            flat[at * 512 + i] = 0
    out = pkg.latent_attention_decode(q, cache, table, lens, 0.07)
    pkg.check_device_status(cuda_device)
    # query 0 sees positions up to 137, which are as before; the key-by-key path rounds elsewhere (16-bit P: 2^-9 of
    # values of order one)
    assert torch.isfinite(out[0, 0]).all() and (out[0, 0].float() - want[0, 0].float()).abs().max() <= 0.05
    assert not torch.isfinite(out[0, 1:, :, 300]).any()
