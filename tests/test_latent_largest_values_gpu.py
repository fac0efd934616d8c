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
