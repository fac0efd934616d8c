"""Paged latent cache: rows written and read back, against the definition computed with torch."""
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


def src_dtype(kind):
    return torch.float16 if kind == "fp16" else torch.bfloat16


def quantised(x):
    """e4m3 values of x [n, 512] under the smallest power-of-two scale >= amax / 448 of each 128."""
    b = x.double().view(-1, 4, 128)
    amax = torch.where(torch.isfinite(b), b.abs(), torch.zeros_like(b)).amax(-1, keepdim=True)
    s = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / 448)).clamp_min(-126)), torch.ones_like(amax))
    q = (b / s).float().clamp(-448, 448).to(torch.float8_e4m3fn).double() * s
    q = torch.where(torch.isfinite(b), q, torch.full_like(q, float("nan")))
    return q.view(-1, 512).to(torch.bfloat16)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [0, 5, 0], [17, 16, 64, 129, 1], [300, 0, 63]])
def test_round_trip(cuda_device, kind, page, lens):
    g = torch.Generator().manual_seed(page + len(lens))
    n = sum(lens)
    need = [max(1, -(-v // page)) for v in lens]
    perm = torch.randperm(sum(need) + 3, generator=g).tolist()
    table = torch.full((len(lens), max(need)), -7, dtype=torch.int32)
    slots, o = [], 0
    for b, v in enumerate(lens):
        table[b, :need[b]] = torch.tensor(perm[o:o + need[b]], dtype=torch.int32)
        o += need[b]
        slots += [int(table[b, j // page]) * page + j % page for j in range(v)]
    dt = src_dtype(kind)
    latent = (torch.randn(n, 512, generator=g) * torch.exp2(torch.randint(-20, 14, (n, 1), generator=g).float())).to(dt)
    rope = torch.randn(n, 64, generator=g).to(dt)
    cache = pkg.latent_cache(sum(need) + 3, page, DT[kind], cuda_device)
    order = torch.randperm(n, generator=g)
    pkg.latent_cache_write(cache, latent[order].to(cuda_device), rope[order].to(cuda_device),
                           torch.tensor(slots, dtype=torch.int64)[order].to(cuda_device))
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(cuda_device)
    got, got_r = pkg.latent_cache_read(cache, table.to(cuda_device), cu, n)
    want = quantised(latent) if kind == "e4m3" else latent
    assert same(got.cpu(), want) and torch.equal(got_r.cpu(), rope)
    # rows past the last request are zeros
    more, more_r = pkg.latent_cache_read(cache, table.to(cuda_device), cu, n + 3)
    assert torch.equal(more[:n], got) and not more[n:].any() and not more_r[n:].any()
    pkg.check_device_status(cuda_device)


def test_codes_are_the_row_quantisers(cuda_device):
    x = torch.randn(70, 512, device=cuda_device).bfloat16()
    x[3, :128] = 0
    cache = pkg.latent_cache(2, 64, torch.float8_e4m3fn, cuda_device)
    slots = torch.arange(70, device=cuda_device)
    pkg.latent_cache_write(cache, x, torch.zeros(70, 64, device=cuda_device, dtype=torch.bfloat16), slots)
    q, s = pkg.quantize_rows_fp8(x)
    flat = cache.view(2, -1)
    codes = flat[:, :64 * 512].reshape(128, 512)[:70]
    exps = flat[:, 64 * 640:].reshape(128, 4)[:70]
    assert torch.equal(codes, q.view(torch.uint8))
    assert torch.equal(torch.exp2(exps.float() - 127), s)


def test_non_finite_values_stay_in_their_place(cuda_device):
    x = torch.randn(4, 512, device=cuda_device).bfloat16()
    clean = x.clone()
    x[0, 5], x[1, 200], x[2, 511] = float("inf"), float("-inf"), float("nan")
    x[3, :128] = float("inf")
    cache = pkg.latent_cache(1, 16, torch.float8_e4m3fn, cuda_device)
    pkg.latent_cache_write(cache, x, x[:, :64].contiguous(), torch.arange(4, device=cuda_device))
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    got, rope = pkg.latent_cache_read(cache, table, torch.tensor([0, 4], dtype=torch.int32, device=cuda_device), 4)
    assert same(got.cpu(), quantised(x.cpu()))
    assert same(rope, x[:, :64])
    assert int(torch.isnan(got).sum()) == 3 + 128
    assert same(got[3, 128:].cpu(), quantised(clean.cpu())[3, 128:])


@pytest.mark.parametrize("value", [1e-38, 1e-40, 3e38, 448.0, 449.0, 0.0])
def test_extreme_blocks(cuda_device, value):
    x = torch.full((2, 512), value).bfloat16()
    x[1, ::2] = -x[1, ::2] / 3
    cache = pkg.latent_cache(1, 16, torch.float8_e4m3fn, cuda_device)
    rope = torch.zeros(2, 64, dtype=torch.bfloat16, device=cuda_device)
    pkg.latent_cache_write(cache, x.to(cuda_device), rope, torch.arange(2, device=cuda_device))
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda_device)
    got, _ = pkg.latent_cache_read(cache, table, torch.tensor([0, 2], dtype=torch.int32, device=cuda_device), 2)
    assert same(got.cpu(), quantised(x))


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("offset", [0, 1, 3, 8])
def test_strided_and_unaligned_sources(cuda_device, kind, offset):
    wide = torch.randn(9, 1000, device=cuda_device).bfloat16()
    latent, rope = wide[:, offset:offset + 512], wide[:, 600 + offset:664 + offset]
    a, b = (pkg.latent_cache(2, 16, DT[kind], cuda_device) for _ in range(2))
    slots = torch.tensor([4, 31, 0, -1, 17, 9, -5, 2, 30], device=cuda_device, dtype=torch.int32)
    pkg.latent_cache_write(a, latent, rope, slots)
    keep = slots >= 0
    pkg.latent_cache_write(b, latent[keep].contiguous(), rope[keep].contiguous(), slots[keep].long())
    assert torch.equal(a, b)   # negative slots write nothing


def test_bad_slot_and_bad_page_are_reported(cuda_device):
    cache = pkg.latent_cache(2, 16, torch.bfloat16, cuda_device)
    row = torch.ones(1, 512, device=cuda_device, dtype=torch.bfloat16)
    pkg.latent_cache_write(cache, row, row[:, :64], torch.tensor([32], device=cuda_device))
    with pytest.raises(RuntimeError, match="device status"):
        pkg.check_device_status(cuda_device)
    assert not cache.any()
    table = torch.tensor([[2]], dtype=torch.int32, device=cuda_device)
    got, rope = pkg.latent_cache_read(cache, table, torch.tensor([0, 2], dtype=torch.int32, device=cuda_device), 2)
    assert torch.isnan(got).all() and torch.isnan(rope).all()
    with pytest.raises(RuntimeError, match="device status"):
        pkg.check_device_status(cuda_device)
    pkg.check_device_status(cuda_device)


def test_refusals(cuda_device):
    cache = pkg.latent_cache(2, 16, torch.bfloat16, cuda_device)
    row = torch.ones(3, 512, device=cuda_device, dtype=torch.bfloat16)
    slots = torch.arange(3, device=cuda_device)
    with pytest.raises(ValueError, match="page_size"):
        pkg.latent_cache(1, 48)
    with pytest.raises(TypeError, match="not supported"):
        pkg.latent_cache(1, 16, torch.float32)
    with pytest.raises(TypeError, match="must be"):
        pkg.latent_cache_write(cache, row.half(), row[:, :64].half(), slots)
    with pytest.raises(ValueError, match="same number"):
        pkg.latent_cache_write(cache, row, row[:2, :64], slots)
    with pytest.raises(ValueError, match="latent must be"):
        pkg.latent_cache_write(cache, row[:, :500], row[:, :64], slots)
    with pytest.raises(ValueError, match="latent_cache"):
        pkg.latent_cache_write(cache[:, ::2], row, row[:, :64], slots)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pkg.latent_cache_write(cache, row.cpu(), row[:, :64], slots)
    with pytest.raises(ValueError, match="block_table"):
        pkg.latent_cache_read(cache, torch.zeros(3, 1, dtype=torch.int32, device=cuda_device),
                              torch.zeros(2, dtype=torch.int32, device=cuda_device), 0)
