"""Latent attention, absorbed over the paged cache and expanded, against 64-bit torch.

Tolerance, derived before any run. With A = sum_j p_j |v_j| per output value: the probabilities may
be rounded to the value type for the second product (u A, u the unit roundoff: 2^-9 bf16, 2^-12
fp16 taken at 2^-11), the result is rounded once (u |o| <= u A), and fp32 scores of up to 576
products are off by at most 576 * 2^-24 * scale * sum |q k| < 2^-11 for these inputs, which moves
each p by that share and the normalised result by twice it. Together (4 u + 2^-10) A bounds the
error with a factor of two over the roundings.
"""
import math

import pytest
import torch

import kernelswift_competition_submission_b200 as pkg

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -9, torch.float16: 2.0 ** -11}
SCALE = 1.0 / math.sqrt(192)


def check(got, want, mass, dt, name=""):
    got, tol = got.double(), (4 * U[dt] + 2.0 ** -10) * mass + 1e-30
    bad = ~((got - want).abs() <= tol)
    bad &= ~(torch.isnan(got) & torch.isnan(want))
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst " \
                          f"{float(((got - want).abs() / tol).nan_to_num(9e9).max()):.3g} of the tolerance"


def soft(s, v):
    """softmax(s) v, sum p |v| and log-sum-exp in 64 bits; rows of -inf give zeros and -inf."""
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((*s.shape[:-1], 1), float("-inf"))
    e = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    z = e.sum(-1, keepdim=True)
    p = torch.where(z > 0, e / z, torch.zeros_like(e))
    lse = torch.where(z > 0, top + torch.log(z), torch.full_like(top, float("-inf")))
    return p @ v, p @ v.abs(), lse[..., 0]


# ------------------------------------------------------------------ absorbed form
def make_cache(lens, page, kind, seed=0, spread=1.0, device="cuda"):
    """A cache with shuffled pages whose slots past every length hold NaN, its table, and the rows."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 2
    perm = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(lens), max(need + [1])), n_pages + 99, dtype=torch.int32)
    dt = torch.float16 if kind == "fp16" else torch.bfloat16
    cache = pkg.latent_cache(n_pages, page, torch.float8_e4m3fn if kind == "e4m3" else dt, device)
    if kind == "e4m3":
        cache.fill_(0x7F)
    else:
        cache.fill_(float("nan"))
    slots, o = [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = torch.tensor(perm[o:o + need[b]], dtype=torch.int32)
        o += need[b]
        slots += [int(table[b, j // page]) * page + j % page for j in range(n)]
    total = sum(lens)
    rows = (torch.randn(total, 576, generator=g) * spread).to(dt).to(device)
    pkg.latent_cache_write(cache, rows[:, :512], rows[:, 512:], torch.tensor(slots, dtype=torch.int64, device=device))
    table = table.to(device)
    cu = torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).to(device)
    if total:
        latent, rope = pkg.latent_cache_read(cache, table, cu, total)
        rows = torch.cat([latent, rope], 1)
    pkg.check_device_status()
    return cache, table, rows.split(list(lens)), dt


def decode_ref(q, rows, scale):
    B, n_q, heads, _ = q.shape
    out = torch.zeros(B, n_q, heads, 512, dtype=torch.float64, device=q.device)
    mass, lse = torch.zeros_like(out), torch.full(out.shape[:3], float("-inf"), dtype=torch.float64, device=q.device)
    for b in range(B):
        for i in range(n_q):
            k = rows[b][:max(0, rows[b].shape[0] - n_q + 1 + i)].double()
            if k.shape[0]:
                out[b, i], mass[b, i], lse[b, i] = soft(q[b, i].double() @ k.T * scale, k[:, :512])
    return out, mass, lse


def run_decode(lens, page, kind, heads, n_q, seed=0, scale=SCALE, spread=1.0, q_spread=1.0):
    cache, table, rows, dt = make_cache(lens, page, kind, seed, spread)
    g = torch.Generator().manual_seed(seed + 100)
    q = (torch.randn(len(lens), n_q, heads, 576, generator=g) * q_spread).to(dt).cuda()
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, lse = pkg.latent_attention_decode(q, cache, table, lens_t, scale, return_lse=True)
    pkg.check_device_status()
    want, mass, want_lse = decode_ref(q, rows, scale)
    check(out, want, mass, dt, "out")
    fin = torch.isfinite(want_lse)
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want_lse))
    assert ((lse.double() - want_lse)[fin].abs() <= 1e-4 * (1 + want_lse[fin].abs())).all()
    again = pkg.latent_attention_decode(q, cache, table, lens_t, scale)
    assert torch.equal(again, out)   # the same bits on every run
    return out


@pytest.mark.parametrize("kind", ["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,n_q", [(128, 1), (16, 1), (12, 3)])
def test_decode_ragged(cuda_device, kind, page, heads, n_q):
    run_decode([1000, 0, 1, 63, 64, 65, 127, 128, 129, 513], page, kind, heads, n_q, seed=page + heads)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads,n_q", [(1, 1), (7, 1), (40, 2), (64, 1), (65, 1), (100, 2), (128, 4), (200, 1)])
def test_decode_heads(cuda_device, kind, heads, n_q):
    run_decode([777, 130, 3], 64, kind, heads, n_q, seed=heads)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lens", [[20011], [4097, 1], [1], [0], [0, 0, 0], [2] * 37, [128] * 5, [9999, 0, 9999]])
def test_decode_lengths(cuda_device, kind, lens):
    run_decode(lens, 64, kind, 128, 1, seed=len(lens))


@pytest.mark.parametrize("n_q", [2, 4, 9])
@pytest.mark.parametrize("lens", [[1, 0, 2, 3, 8, 9, 10, 130], [129, 135]])
def test_decode_draft_rows_that_see_nothing(cuda_device, n_q, lens):
    run_decode(lens, 16, "bf16", 16, n_q)


@pytest.mark.parametrize("scale", [0.0, -0.07, 3.0])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_decode_scales(cuda_device, scale, kind):
    """Flat, negated and one-hot softmax; at 3.0 the running maximum moves by hundreds."""
    run_decode([900, 130], 64, kind, 32, 1, scale=scale, q_spread=0.3 if scale == 3.0 else 1.0)


def test_decode_growing_scores(cuda_device):
    """Scores that rise along the context: every tile moves the maximum."""
    cache, table, rows, dt = make_cache([1500], 64, "bf16")
    ramp = torch.linspace(0, 30, 1500, device="cuda")[:, None].expand(1500, 576)
    new = (rows[0].float() * 0.05 + ramp * 0.05).to(dt)
    slots = (table[0].long()[:, None] * 64 + torch.arange(64, device="cuda")).view(-1)[:1500]
    pkg.latent_cache_write(cache, new[:, :512], new[:, 512:], slots)
    q = torch.rand(1, 1, 128, 576, device="cuda").to(dt)
    lens = torch.tensor([1500], dtype=torch.int32, device="cuda")
    out = pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    want, mass, _ = decode_ref(q, [new], SCALE)
    check(out, want, mass, dt)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("place", [99, 130, 201])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_decode_hidden_and_seen_non_finite(cuda_device, kind, place, value):
    """A draft token's non-finite row reaches the queries that see it and no other."""
    cache, table, rows, dt = make_cache([202, 150], 32, kind)
    bad = rows[0][place:place + 1].clone()
    bad[0, 7] = value
    slot = int(table[0, place // 32]) * 32 + place % 32
    pkg.latent_cache_write(cache, bad[:, :512], bad[:, 512:], torch.tensor([slot], device="cuda"))
    if kind == "e4m3":
        bad[0, 7] = float("nan")   # an e4m3 page keeps both as NaN
    rows = [torch.cat([rows[0][:place], bad, rows[0][place + 1:]]), rows[1]]
    q = torch.randn(2, 4, 16, 576, device="cuda").to(dt)
    lens = torch.tensor([202, 150], dtype=torch.int32, device="cuda")
    out = pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    want, mass, _ = decode_ref(q, rows, SCALE)
    sees = torch.tensor([202 - 4 + i >= place for i in range(4)], device="cuda")
    check(out[1], want[1], mass[1], dt, "other request")
    if (~sees).any():
        check(out[0][~sees], want[0][~sees], mass[0][~sees], dt, "rows before")
    if value != value:
        assert torch.isnan(out[0][sees]).all()
    else:
        assert not torch.isfinite(out[0][sees]).all(-1).any()


def test_decode_other_stream_and_out(cuda_device):
    cache, table, rows, dt = make_cache([700, 31], 64, "bf16")
    q = torch.randn(2, 1, 128, 576, device="cuda").to(dt)
    lens = torch.tensor([700, 31], dtype=torch.int32, device="cuda")
    plain = pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    need = pkg.latent_attention_decode_workspace_bytes(2, 1, 128)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda").fill_(255)
    out = torch.full_like(plain, float("nan"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.latent_attention_decode(q, cache, table, lens, SCALE, out=out, workspace=ws)
    side.synchronize()
    assert got is out and torch.equal(out, plain)


def test_decode_graph(cuda_device):
    """Lengths are read on the device: a captured call follows them."""
    cache, table, rows, dt = make_cache([700, 310], 64, "bf16")
    q = torch.randn(2, 1, 16, 576, device="cuda").to(dt)
    lens = torch.tensor([700, 310], dtype=torch.int32, device="cuda")
    pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.latent_attention_decode(q, cache, table, lens, SCALE)
    for new in ([700, 310], [5, 0], [641, 1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, mass, _ = decode_ref(q, [rows[0][:new[0]], rows[1][:new[1]]], SCALE)
        check(out, want, mass, dt)


def test_decode_bad_lengths_and_pages_are_reported(cuda_device):
    cache, table, rows, dt = make_cache([100], 64, "bf16")
    q = torch.randn(1, 1, 16, 576, device="cuda").to(dt)
    pkg.latent_attention_decode(q, cache, table, torch.tensor([999], dtype=torch.int32, device="cuda"), SCALE)
    with pytest.raises(RuntimeError, match="device status"):
        pkg.check_device_status()
    bad = table.clone()
    bad[0, 1] = -1
    out = pkg.latent_attention_decode(q, cache, bad, torch.tensor([100], dtype=torch.int32, device="cuda"), SCALE)
    with pytest.raises(RuntimeError, match="device status"):
        pkg.check_device_status()
    want, mass, _ = decode_ref(q, [rows[0][:64]], SCALE)   # the page is left out
    check(out, want, mass, dt)


def test_decode_refusals(cuda_device):
    cache, table, rows, dt = make_cache([100], 64, "bf16")
    q = torch.randn(1, 1, 16, 576, device="cuda").to(dt)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    f = pkg.latent_attention_decode
    with pytest.raises(TypeError, match="q must be"):
        f(q.half(), cache, table, lens, SCALE)
    with pytest.raises(ValueError, match="q must be"):
        f(q[..., :512], cache, table, lens, SCALE)
    with pytest.raises(ValueError, match="cache_lens"):
        f(q, cache, table, lens.repeat(2), SCALE)
    with pytest.raises(ValueError, match="cache_lens"):
        f(q, cache, table, lens.float(), SCALE)
    with pytest.raises(ValueError, match="block_table"):
        f(q, cache, table.repeat(2, 1), lens, SCALE)
    with pytest.raises(ValueError, match="latent_cache"):
        f(q, cache.view(-1, 576), table, lens, SCALE)
    with pytest.raises(ValueError, match="out must be"):
        f(q, cache, table, lens, SCALE, out=torch.empty(1, 1, 16, 512, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(q.cpu(), cache, table, lens, SCALE)
    assert f(q[:0], cache, table[:0], lens[:0], SCALE).shape == (0, 1, 16, 512)
    with pytest.raises(RuntimeError, match="unsupported shape"):
        f(torch.empty(1, 513, 128, 576, device="cuda", dtype=dt), cache, table, lens, SCALE)


# ------------------------------------------------------------------ expanded form
def prefill_ref(q, kv, kr, new, lens, scale, causal):
    heads = q.shape[1]
    out = torch.zeros(q.shape[0], heads, 128, dtype=torch.float64, device=q.device)
    mass, lse = torch.zeros_like(out), torch.full(out.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    a = c = 0
    for n, m in zip(new, lens):
        for h in range(heads):
            s = q[a:a + n, h, :128].double() @ kv[c:c + m, h, :128].double().T
            s = (s + q[a:a + n, h, 128:].double() @ kr[c:c + m].double().T) * scale
            v = kv[c:c + m, h, 128:].double()
            if causal:
                hide = torch.arange(m, device=q.device)[None] > (m - n + torch.arange(n, device=q.device))[:, None]
                s = s.masked_fill(hide, float("-inf"))
            if m and n:
                out[a:a + n, h], mass[a:a + n, h], lse[a:a + n, h] = soft(s, v)
        a, c = a + n, c + m
    return out, mass, lse


def cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def run_prefill(new, lens, heads, dt, causal, seed=0, scale=SCALE):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(new), heads, 192, generator=g).to(dt).cuda()
    kv = torch.randn(sum(lens), heads, 256, generator=g).to(dt).cuda()
    kr = torch.randn(sum(lens), 64, generator=g).to(dt).cuda()
    out, lse = pkg.latent_attention_prefill(q, kv, kr, cu(new), cu(lens), scale, causal=causal, return_lse=True)
    want, mass, want_lse = prefill_ref(q, kv, kr, new, lens, scale, causal)
    check(out, want, mass, dt, "out")
    fin = torch.isfinite(want_lse)
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want_lse))
    assert ((lse.double() - want_lse)[fin].abs() <= 1e-4 * (1 + want_lse[fin].abs())).all()
    pkg.check_device_status()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 127, 128, 129, 255, 256, 257, 385, 700])
def test_prefill_lengths(cuda_device, dt, causal, n):
    run_prefill([n], [n], 3, dt, causal, seed=n)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [5, 129, 1]), ([5, 0, 300, 17], [5, 40, 900, 17]),
                                      ([130, 257], [0, 400]), ([64, 200, 3], [10, 100, 1]), ([0], [0]),
                                      ([7] * 20, [300] * 20), ([513, 1, 255], [1500, 700, 255])])
def test_prefill_ragged(cuda_device, causal, new, lens):
    """Histories, empty requests, and queries that see no key (more queries than keys)."""
    run_prefill(new, lens, 4, torch.bfloat16, causal, seed=sum(new))


@pytest.mark.parametrize("scale", [0.0, -0.07, 2.0])
def test_prefill_scales(cuda_device, scale):
    run_prefill([300], [300], 2, torch.bfloat16, True, scale=scale)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_non_finite_neighbours(cuda_device, causal, value):
    """Another request's values, and with a mask later tokens' values, reach no row."""
    dt, new, h = torch.bfloat16, [200, 300, 77], 2
    q, kv, kr = (torch.randn(577, *s, device="cuda").to(dt) for s in ((h, 192), (h, 256), (64,)))
    want, mass, _ = prefill_ref(q, kv, kr, new, new, SCALE, causal)
    kv2, kr2 = kv.clone(), kr.clone()
    kv2[200:500] = value
    kr2[200:500] = value
    out = pkg.latent_attention_prefill(q, kv2, kr2, cu(new), cu(new), SCALE, causal=causal)
    keep = torch.cat([torch.arange(200), torch.arange(500, 577)]).cuda()
    check(out[keep], want[keep], mass[keep], dt)
    assert not torch.isfinite(out[200:500]).any()
    if causal:
        for place in (37, 150):   # a later token of the same request, in values only, then in keys too
            kv3, kr3 = kv.clone(), kr.clone()
            kv3[place, 1, 128 + 9] = value
            if place == 150:
                kr3[place, 0] = value
            out = pkg.latent_attention_prefill(q, kv3, kr3, cu(new), cu(new), SCALE)
            check(out[:place], want[:place], mass[:place], dt, f"rows before {place}")
            check(out[200:], want[200:], mass[200:], dt, "other requests")
            assert not torch.isfinite(out[place:200, 1, 9]).any()
            if place == 37:
                check(out[:, 0], want[:, 0], mass[:, 0], dt, "other head")
                check(out[:, 1, :9], want[:, 1, :9], mass[:, 1, :9], dt, "other values")


def test_prefill_strides(cuda_device):
    """Views into wider projections: head slices, sliced rows and a rotary slice."""
    dt = torch.bfloat16
    big_q = torch.randn(333, 6, 256, device="cuda").to(dt)
    big_kv = torch.randn(333, 5, 512, device="cuda").to(dt)
    big_kr = torch.randn(333, 576, device="cuda").to(dt)
    q, kv, kr = big_q[:, 1:4, 64:], big_kv[:, 2:5, 128:384], big_kr[:, 512:]
    out = pkg.latent_attention_prefill(q, kv, kr, cu([333]), cu([333]), SCALE)
    want, mass, _ = prefill_ref(q, kv, kr, [333], [333], SCALE, True)
    check(out, want, mass, dt)
    odd = torch.randn(333, 3, 193, device="cuda").to(dt)[..., 1:]   # unaligned: copied, then read
    out = pkg.latent_attention_prefill(odd, kv, kr, cu([333]), cu([333]), SCALE)
    want, mass, _ = prefill_ref(odd, kv, kr, [333], [333], SCALE, True)
    check(out, want, mass, dt)


def test_prefill_pieces_join(cuda_device):
    """A context attended in two pieces without a mask, joined by log-sum-exp, is the whole."""
    dt, h = torch.bfloat16, 4
    q = torch.randn(50, h, 192, device="cuda").to(dt)
    kv, kr = torch.randn(900, h, 256, device="cuda").to(dt), torch.randn(900, 64, device="cuda").to(dt)
    parts = []
    for a, b in ((0, 411), (411, 900)):
        parts.append(pkg.latent_attention_prefill(q, kv[a:b], kr[a:b], cu([50]), cu([b - a]), SCALE, causal=False,
                                                  return_lse=True))
    z = torch.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o.double() * torch.exp(s - z).double()[..., None] for o, s in parts)
    want, mass, _ = prefill_ref(q, kv, kr, [50], [900], SCALE, False)
    check(joined, want, mass, dt)


def test_prefill_rows_past_the_requests_and_stream(cuda_device):
    dt = torch.bfloat16
    q, kv, kr = (torch.randn(200, *s, device="cuda").to(dt) for s in ((2, 192), (2, 256), (64,)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = pkg.latent_attention_prefill(q, kv, kr, cu([90, 40]), cu([90, 40]), SCALE, return_lse=True)
    side.synchronize()
    want, mass, _ = prefill_ref(q, kv, kr, [90, 40], [90, 40], SCALE, True)
    check(out, want, mass, dt)
    assert not out[130:].any() and torch.isneginf(lse[130:]).all()


def test_prefill_refusals(cuda_device):
    dt = torch.bfloat16
    q, kv, kr = (torch.randn(20, *s, device="cuda").to(dt) for s in ((2, 192), (2, 256), (64,)))
    c = cu([20])
    f = pkg.latent_attention_prefill
    with pytest.raises(TypeError, match="dtype"):
        f(q.float(), kv, kr, c, c, SCALE)
    with pytest.raises(TypeError, match="dtype of q"):
        f(q, kv.half(), kr, c, c, SCALE)
    with pytest.raises(ValueError, match="q must be"):
        f(q[..., :128], kv, kr, c, c, SCALE)
    with pytest.raises(ValueError, match="kv must be"):
        f(q, kv[:, :1], kr, c, c, SCALE)
    with pytest.raises(ValueError, match="k_rope must be"):
        f(q, kv, kr[:10], c, c, SCALE)
    with pytest.raises(ValueError, match="same length"):
        f(q, kv, kr, c, cu([10, 10]), SCALE)
    with pytest.raises(ValueError, match="out must be"):
        f(q, kv, kr, c, c, SCALE, out=torch.empty(20, 2, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        f(q.cpu(), kv, kr, c, c, SCALE)
    assert f(q[:0], kv, kr, cu([0]), c, SCALE).shape == (0, 2, 128)


# ------------------------------------------------------------------ the two forms together
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_forms_agree(cuda_device, kind):
    """One request's last token: absorbed over the cache, and expanded from the rows read back."""
    n, h = 391, 16
    cache, table, rows, dt = make_cache([n], 64, kind)
    wk = (torch.randn(h, 128, 512, device="cuda") / 512 ** 0.5)
    wv = (torch.randn(h, 128, 512, device="cuda") / 512 ** 0.5)
    qn, qr = torch.randn(h, 128, device="cuda"), torch.randn(h, 64, device="cuda").to(dt)
    latent, rope = pkg.latent_cache_read(cache, table, cu([n]), n)
    kv = torch.cat([torch.einsum("hdc,nc->nhd", w, latent.float()) for w in (wk, wv)], -1).to(dt)
    q = torch.cat([qn.to(dt), qr], -1)[None]
    a = pkg.latent_attention_prefill(q, kv, rope, cu([1]), cu([n]), SCALE)[0].float()
    qa = torch.cat([torch.einsum("hd,hdc->hc", qn, wk).to(dt), qr], -1)[None, None]
    o = pkg.latent_attention_decode(qa, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), SCALE)
    b = torch.einsum("hc,hdc->hd", o[0, 0].float(), wv)
    # 16-bit queries, keys, values and latent outputs: roundings of 2^-9 on values of order one
    assert (a - b).abs().max() <= 0.05 * b.abs().max()
