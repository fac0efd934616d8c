"""A caller's workspace goes to the kernels by its address: one that they cannot use is refused, a small one replaced."""
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu


def check(call, need):
    want = call(None)
    for bad in (torch.empty(need, dtype=torch.uint8), torch.empty(2 * need, dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(ValueError, match="workspace must be"):
            call(bad)
    with pytest.raises(RuntimeError):   # off 16 bytes
        call(torch.empty(need + 1, dtype=torch.uint8, device="cuda")[1:])
    for good in (torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(need // 4 + 1, device="cuda"),
                 torch.empty(8, dtype=torch.uint8, device="cuda")):
        assert torch.equal(call(good), want)


def test_decode(cuda_device):
    cache = pkg.latent_cache(2, 64, torch.bfloat16, cuda_device)
    cache.normal_()
    q = torch.randn(2, 1, 16, 576, device=cuda_device).bfloat16()
    table = torch.arange(2, dtype=torch.int32, device=cuda_device)[:, None]
    lens = torch.tensor([64, 3], dtype=torch.int32, device=cuda_device)
    check(lambda w: pkg.latent_attention_decode(q, cache, table, lens, 0.07, workspace=w),
          pkg.latent_attention_decode_workspace_bytes(2, 1, 16))


def test_moe_decode(cuda_device):
    x, lg = torch.randn(3, 256, device=cuda_device).bfloat16(), torch.randn(3, 8, device=cuda_device)
    w1, w2 = (torch.randn(8, *s, device=cuda_device).bfloat16() / 16 for s in ((256, 256), (256, 128)))
    check(lambda w: pkg.moe_decode(x, lg, w1, w2, topk=2, workspace=w), 1 << 16)
