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


@pytest.mark.parametrize("first", [1, 130, 300])
@pytest.mark.parametrize("new", [[40, 0, 300], [256], []])
def test_prefill(cuda_device, first, new):
    """Queries before cu_q[0] and past cu_q[-1] get zeros and -inf, the requests what they get alone."""
    heads, dt, n = 3, torch.bfloat16, sum(new)
    q = torch.randn(first + n + 5, heads, 192, device=cuda_device).to(dt)
    kv = torch.randn(n + 9, heads, 256, device=cuda_device).to(dt)
    kr = torch.randn(n + 9, 64, device=cuda_device).to(dt)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(cuda_device)
    out = torch.full((q.shape[0], heads, 128), 7777.0, dtype=dt, device=cuda_device)
    _, lse = pkg.latent_attention_prefill(q, kv, kr, cu + first, cu + 4, 0.07, out=out, return_lse=True)
    want, want_lse = pkg.latent_attention_prefill(q[first:first + n], kv[4:4 + n], kr[4:4 + n], cu, cu, 0.07,
                                                  return_lse=True)
    pkg.check_device_status(cuda_device)
    assert torch.equal(out[first:first + n], want) and torch.equal(lse[first:first + n], want_lse)
    rest = torch.cat([torch.arange(first), torch.arange(first + n, q.shape[0])]).to(cuda_device)
    assert not out[rest].any() and torch.isneginf(lse[rest]).all()
