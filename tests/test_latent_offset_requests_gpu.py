"""Prefix sums that do not start at zero, as a slice of a larger batch's: the rows before them belong to no request."""
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("first", [1, 17, 200])
def test_cache_read(cuda_device, kind, first):
    lens, page = [40, 0, 65], 16
    need = [-(-n // page) for n in lens]
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    cache = pkg.latent_cache(sum(need), page, DT[kind], cuda_device)
    rows = torch.randn(sum(need) * page, 576, device=cuda_device).to(dt)
    pkg.latent_cache_write(cache, rows[:, :512], rows[:, 512:], torch.arange(rows.shape[0], device=cuda_device))
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(o, o + n)
        o += n
    table = table.to(cuda_device)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda_device)
    want, want_r = pkg.latent_cache_read(cache, table, cu, sum(lens))
    got, got_r = pkg.latent_cache_read(cache, table, cu + first, first + sum(lens) + 2)
    pkg.check_device_status(cuda_device)
    end = first + sum(lens)
    assert torch.equal(got[first:end], want) and torch.equal(got_r[first:end], want_r)
    for t in (got, got_r):
        assert not t[:first].any() and not t[end:].any()
    none, none_r = pkg.latent_cache_read(cache, table[:0], cu[:1] + first, first + 2)
    assert not none.any() and not none_r.any()
