"""The cache's calls, the expanded form and moe_decode in CUDA graphs: replays follow the inputs on the device."""
import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu


def captured(f):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        f()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
def test_cache(cuda_device, kind):
    dt = torch.float16 if kind == torch.float16 else torch.bfloat16
    cache, other = (pkg.latent_cache(6, 32, kind, cuda_device) for _ in range(2))
    latent, rope = torch.randn(70, 512, device=cuda_device).to(dt), torch.randn(70, 64, device=cuda_device).to(dt)
    slots = torch.randperm(6 * 32, device=cuda_device)[:70]
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=cuda_device)
    cu = torch.tensor([0, 80, 150], dtype=torch.int32, device=cuda_device)

    def step():
        pkg.latent_cache_write(cache, latent, rope, slots)
        return pkg.latent_cache_read(cache, table, cu, 150)

    graph, out = captured(step)
    for seed in range(3):
        torch.manual_seed(seed)
        latent.normal_()
        rope.normal_()
        slots.copy_(torch.randperm(6 * 32, device=cuda_device)[:70])
        table.copy_(torch.randperm(6, device=cuda_device).view(2, 3))
        cu[1] = 60 + 15 * seed   # up to three pages a request
        other.copy_(cache)
        graph.replay()
        pkg.latent_cache_write(other, latent, rope, slots)
        want = pkg.latent_cache_read(other, table, cu, 150)
        assert torch.equal(cache, other)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    pkg.check_device_status(cuda_device)


def test_prefill(cuda_device):
    q, kv, kr = (torch.randn(400, *s, device=cuda_device).bfloat16() for s in ((3, 192), (3, 256), (64,)))
    cu = torch.tensor([0, 100, 400], dtype=torch.int32, device=cuda_device)
    graph, out = captured(lambda: pkg.latent_attention_prefill(q, kv, kr, cu, cu, 0.07, return_lse=True))
    for cut in (100, 0, 399):
        q.normal_()
        cu[1] = cut
        graph.replay()
        want = pkg.latent_attention_prefill(q, kv, kr, cu, cu, 0.07, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    pkg.check_device_status(cuda_device)


@pytest.mark.parametrize("f8", [False, True])
def test_moe_decode(cuda_device, f8):
    w1 = (torch.randn(16, 512, 512, device=cuda_device) / 22).bfloat16()
    w2 = (torch.randn(16, 512, 256, device=cuda_device) / 16).bfloat16()
    kw = dict(topk=4)
    if f8:
        (w1, s1), (w2, s2) = pkg.quantize_weights_fp8(w1), pkg.quantize_weights_fp8(w2)
        kw.update(w1_scale=s1, w2_scale=s2)
    x, lg = torch.randn(5, 512, device=cuda_device).bfloat16(), torch.randn(5, 16, device=cuda_device)
    graph, out = captured(lambda: pkg.moe_decode(x, lg, w1, w2, **kw))
    for scale in (1.0, 100.0, 1e-3):
        x.normal_(std=scale)
        lg.normal_()
        graph.replay()
        assert torch.equal(out, pkg.moe_decode(x, lg, w1, w2, **kw))
