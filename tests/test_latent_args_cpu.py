"""CPU: host-side refusals of the latent cache, latent attention and few-token MoE entries (nothing is launched)."""
import ctypes

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg
from kernelswift_competition_submission_b200 import _lib, build

P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(258)
BF16, FP16, E4M3 = _lib.MOE_DTYPE_BF16, _lib.MOE_DTYPE_FP16, _lib.MOE_CACHE_E4M3


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def call(f, defaults, **change):
    assert set(change) <= set(defaults)
    return f(*{**defaults, **change}.values())


def test_page_bytes(lib):
    f = lib.moe_latent_cache_page_bytes
    assert [f(BF16, p) for p in (16, 32, 64, 128)] == [p * 1152 for p in (16, 32, 64, 128)]
    assert f(E4M3, 64) == 64 * 644 and f(BF16, 48) == -1 and f(77, 64) == -1


def test_cache_write(lib):
    d = dict(dtype=BF16, latent=P, ldl=512, rope=P, ldr=64, slots=P, n=4, fmt=BF16, cache=P, pages=2, page=64,
             status=None, stream=None)
    f = lib.moe_latent_cache_write
    assert call(f, d, n=0, latent=None) == _lib.MOE_OK
    for bad in (dict(fmt=FP16), dict(dtype=FP16, fmt=E4M3), dict(fmt=9), dict(dtype=9)):
        assert call(f, d, **bad) == _lib.MOE_ERR_UNSUPPORTED
    for bad in (dict(page=48), dict(page=0), dict(pages=2 ** 31), dict(n=2 ** 31)):
        assert call(f, d, **bad) == _lib.MOE_ERR_BAD_SHAPE
    for bad in (dict(n=-1), dict(pages=-1), dict(latent=None), dict(rope=None), dict(slots=None), dict(cache=None),
                dict(cache=ODD), dict(slots=ODD), dict(latent=ctypes.c_void_p(257)), dict(ldl=-1)):
        assert call(f, d, **bad) == _lib.MOE_ERR_INVALID_ARG


def test_cache_read(lib):
    d = dict(fmt=BF16, cache=P, pages=2, page=64, table=P, ldt=1, width=1, cu=P, seqs=1, total=4, latent=P, rope=P,
             status=None, stream=None)
    f = lib.moe_latent_cache_read
    assert call(f, d, total=0, cache=None) == _lib.MOE_OK
    assert call(f, d, fmt=9) == _lib.MOE_ERR_UNSUPPORTED
    assert call(f, d, page=17) == _lib.MOE_ERR_BAD_SHAPE
    for bad in (dict(total=-1), dict(seqs=-1), dict(cu=None), dict(table=None), dict(latent=ODD), dict(rope=None)):
        assert call(f, d, **bad) == _lib.MOE_ERR_INVALID_ARG


def test_decode(lib):
    need = lib.moe_latent_decode_workspace_bytes(2, 1, 16)
    assert need > 0 and lib.moe_latent_decode_workspace_bytes(2, 0, 16) == 0
    d = dict(dtype=BF16, q=P, seqs=2, n_q=1, heads=16, fmt=BF16, cache=P, pages=2, page=64, table=P, ldt=1, width=1,
             lens=P, scale=1.0, out=P, lse=None, ws=P, ws_bytes=need, status=None, stream=None)
    f = lib.moe_latent_decode
    assert call(f, d, seqs=0, q=None) == _lib.MOE_OK
    for bad in (dict(fmt=FP16), dict(dtype=FP16, fmt=E4M3), dict(dtype=5)):
        assert call(f, d, **bad) == _lib.MOE_ERR_UNSUPPORTED
    for bad in (dict(page=1), dict(heads=65536, n_q=2), dict(seqs=65536), dict(width=2 ** 25)):
        assert call(f, d, **bad) == _lib.MOE_ERR_BAD_SHAPE
    for bad in (dict(n_q=0), dict(heads=0), dict(pages=0), dict(q=ODD), dict(out=ODD), dict(cache=ODD), dict(lens=None),
                dict(table=None), dict(width=-1)):
        assert call(f, d, **bad) == _lib.MOE_ERR_INVALID_ARG
    for bad in (dict(ws=None), dict(ws=ODD), dict(ws_bytes=need - 1)):
        assert call(f, d, **bad) == _lib.MOE_ERR_WORKSPACE


def test_prefill(lib):
    d = dict(dtype=BF16, q=P, qt=384, qh=192, kv=P, kt=512, kh=256, kr=P, krt=64, cu_q=P, cu_k=P, seqs=1, tq=4, tk=4,
             heads=2, scale=1.0, causal=1, out=P, lse=None, status=None, stream=None)
    f = lib.moe_latent_prefill
    assert call(f, d, tq=0, q=None) == _lib.MOE_OK
    assert call(f, d, dtype=9) == _lib.MOE_ERR_UNSUPPORTED
    for bad in (dict(qt=0), dict(qh=12), dict(kt=-8), dict(krt=4), dict(tq=2 ** 31), dict(heads=65536),
                dict(seqs=65536)):
        assert call(f, d, **bad) == _lib.MOE_ERR_BAD_SHAPE
    for bad in (dict(tq=-1), dict(heads=0), dict(q=ODD), dict(kv=None), dict(kr=ODD), dict(cu_q=None), dict(out=None)):
        assert call(f, d, **bad) == _lib.MOE_ERR_INVALID_ARG


def test_few_tokens(lib):
    assert [lib.moe_few_max_tokens(k) for k in (0, 1, 8, 16, 32)] == [0, 32, 32, 32, 16]
    need = lib.moe_few_workspace_bytes(4, 2, 128)
    d = dict(dtype=BF16, x=P, ld=256, g=P, bias=None, f8=0, w1=P, s1=None, w2=P, s2=None, m=4, e=8, k=2, rn=1, ng=1,
             tg=1, sc=0, gm=0, s=1.0, K=256, N=128, out=P, ws=P, ws_bytes=need, stream=None)
    f = lib.moe_few_tokens
    assert call(f, d, m=0, x=None) == _lib.MOE_OK
    assert call(f, d, dtype=9) == _lib.MOE_ERR_UNSUPPORTED
    for bad in (dict(K=250), dict(N=96), dict(f8=1, s1=P, s2=P, K=192), dict(m=33), dict(e=7, ng=2), dict(k=9),
                dict(tg=2), dict(ng=8, gm=1)):
        assert call(f, d, **bad) == _lib.MOE_ERR_BAD_SHAPE
    for bad in (dict(m=-1), dict(sc=5), dict(gm=5), dict(x=ODD), dict(ld=252), dict(w1=None), dict(f8=1), dict(out=None),
                dict(w2=ODD)):
        assert call(f, d, **bad) == _lib.MOE_ERR_INVALID_ARG
    assert call(f, d, ws_bytes=need - 1) == _lib.MOE_ERR_WORKSPACE


def test_python_refuses_without_a_gpu():
    cache = pkg.latent_cache(2, 16, device="cpu")
    assert cache.shape == (2, 16, 576) and pkg.latent_cache(2, 16, torch.float8_e4m3fn, "cpu").shape == (2, 16, 644)
    with pytest.raises(ValueError):
        pkg.latent_cache(2, 48, device="cpu")
    with pytest.raises(TypeError):
        pkg.latent_cache(2, 16, torch.float32, "cpu")
    z, i = torch.zeros(1, 512, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: pkg.latent_cache_write(cache, z, z[:, :64], i),
              lambda: pkg.latent_cache_read(cache, i[None], torch.zeros(2, dtype=torch.int32), 1),
              lambda: pkg.latent_attention_decode(torch.zeros(1, 1, 2, 576), cache, i[None], i, 1.0),
              lambda: pkg.moe_decode(z, z[:, :8].float(), z, z, topk=2)):
        with pytest.raises((RuntimeError, ValueError), match="CUDA|cuda|GPU"):
            f()
