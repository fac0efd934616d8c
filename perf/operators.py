"""Cases, plain forms and 64-bit references of the latent-attention and few-token MoE operators.

Four operators of one decoder layer's serving step are measured here:

* ``cache``    tokens written into a paged latent cache (16-bit, or e4m3 with power-of-two block
               scales) and the contexts read back for the expanded form;
* ``decode``   latent attention over that cache in the absorbed form (all heads share the cached
               512 + 64 vector of a token);
* ``prefill``  latent attention in the expanded form (per-head keys and values, one rotary key
               shared by all heads), variable lengths;
* ``moe``      routing and experts of one mixture-of-experts layer for a few tokens.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own``, through the
package's entry points. ``exact`` computes them in 64 bits from the definitions.
"""

import math
import random

import torch

own = False

DC = 512    # latent values of a cached token
DR = 64     # rotary key values of a cached token
DN = 128    # per-head key part without position, and per-head value, of the expanded form
ROW8 = DC + 2 * DR + DC // 128   # bytes of a token in an 8-bit page

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.bfloat16}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 48 running requests appends its tokens to the cache (latency)
        dict(name="cache_append_bf16", op="cache", dtype="bf16", page=64, n_seq=48, max_new=1, history=700,
             read=False, len_seed=1),
        # chunked prefill: two chunks are quantised into the cache, then their whole contexts
        # (history and chunk) are read back for the expanded form
        dict(name="cache_chunk_fp8", op="cache", dtype="fp8", page=64, n_seq=2, max_new=1531, history=24011,
             read=True, len_seed=2),
        # a single request, all heads on this GPU (latency)
        dict(name="decode_one_bf16", op="decode", dtype="bf16", page=64, n_seq=1, heads=128, n_q=1, max_len=1237,
             empty=False, lse=False, len_seed=3),
        # a serving batch with ragged contexts, all heads on this GPU
        dict(name="decode_batch_bf16", op="decode", dtype="bf16", page=64, n_seq=40, heads=128, n_q=1, max_len=9000,
             empty=True, lse=False, len_seed=4),
        # heads split over 8 GPUs, 8-bit cache, a large ragged batch in small pages
        dict(name="decode_shard_fp8", op="decode", dtype="fp8", page=32, n_seq=120, heads=16, n_q=1, max_len=7001,
             empty=True, lse=False, len_seed=5),
        # three draft tokens a request are scored in one call, heads split over 4 GPUs
        dict(name="decode_draft_fp16", op="decode", dtype="fp16", page=16, n_seq=7, heads=32, n_q=3, max_len=3301,
             empty=False, lse=True, len_seed=6),
        # a batch of ragged prompts, heads split over 8 GPUs
        dict(name="prefill_ragged_bf16", op="prefill", dtype="bf16", n_seq=9, heads=16, max_q=1777, history=0,
             causal=True, lse=False, len_seed=7),
        # one piece of a long context attended without a mask, to be joined by its log-sum-exp
        dict(name="prefill_piece_fp16", op="prefill", dtype="fp16", n_seq=3, heads=24, max_q=611, history=4007,
             causal=False, lse=True, len_seed=8),
        # a long prompt, all heads on this GPU
        dict(name="prefill_long_bf16", op="prefill", dtype="bf16", n_seq=1, heads=128, max_q=7993, history=0,
             causal=True, lse=False, len_seed=9),
        # DeepSeek-V3 layer, one token, e4m3 weights (latency)
        dict(name="moe_one_fp8", op="moe", dtype="fp8", tokens=1, experts=256, topk=8, groups=8, topk_group=4,
             hidden=7168, inter=2048, scoring="sigmoid", bias=True),
        # the same layer for the tokens of a small decode batch
        dict(name="moe_few_fp8", op="moe", dtype="fp8", tokens=11, experts=256, topk=8, groups=8, topk_group=4,
             hidden=7168, inter=2048, scoring="sigmoid", bias=True),
        # Mixtral-style layer, few tokens, 16-bit weights: experts with several tokens each
        dict(name="moe_mixtral_bf16", op="moe", dtype="bf16", tokens=6, experts=8, topk=2, groups=1, topk_group=1,
             hidden=4096, inter=14336, scoring="softmax", bias=False),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["cache", "decode", "decode", "prefill", "moe"])
    seed = rng.randrange(1 << 30)
    if op == "cache":
        dtype = rng.choice(["bf16", "fp16", "fp8"])
        c = dict(op=op, dtype=dtype, page=rng.choice([16, 32, 64, 128]), n_seq=_log_int(rng, 1, 160),
                 max_new=_log_int(rng, 1, 4096), history=rng.choice([0, _log_int(rng, 1, 20000)]),
                 read=True if dtype == "fp8" else rng.random() < 0.5, len_seed=seed)
        shrink = ("max_new", "history", "n_seq")
    elif op == "decode":
        c = dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp8"]), page=rng.choice([16, 32, 64, 128]),
                 n_seq=_log_int(rng, 1, 160), heads=rng.choice([8, 12, 16, 32, 40, 64, 128]),
                 n_q=rng.choice([1, 1, 1, 2, 3, 4]), max_len=_log_int(rng, 5, 40000), empty=False,
                 lse=rng.random() < 0.5, len_seed=seed)
        c["empty"] = not c["lse"] and c["n_seq"] > 4
        shrink = ("max_len", "n_seq")
    elif op == "prefill":
        c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), n_seq=_log_int(rng, 1, 24),
                 heads=rng.choice([4, 8, 16, 20, 32, 64, 128]), max_q=_log_int(rng, 1, 8000),
                 history=rng.choice([0, 0, _log_int(rng, 1, 6000)]), causal=rng.random() < 0.75,
                 lse=rng.random() < 0.5, len_seed=seed)
        shrink = ("max_q", "history", "n_seq")
    else:
        experts, topk, groups, tg, hidden, inter, scoring, bias = rng.choice([
            (256, 8, 8, 4, 7168, 2048, "sigmoid", True), (8, 2, 1, 1, 4096, 14336, "softmax", False),
            (64, 6, 8, 3, 2048, 1024, "sigmoid", True), (64, 6, 8, 3, 512, 256, "sigmoid", True)])
        dtype = rng.choice(["bf16", "fp16", "fp8"])
        return dict(op=op, dtype=dtype, tokens=_log_int(rng, 1, 32), experts=experts, topk=topk, groups=groups,
                    topk_group=tg, hidden=hidden, inter=inter, scoring=scoring, bias=bias)
    limit = {}
    for k in listed():
        w = work(k)
        for f in w:
            limit[(k["op"], f)] = max(limit.get((k["op"], f), 0), w[f])
    i = 0
    while any(v > limit[(op, f)] for f, v in work(c).items()):
        k = shrink[i % len(shrink)]
        c[k] = max(c[k] * 2 // 3, 0 if k == "history" else 1)
        if c[k] == 3072:
            c[k] -= 1
        i += 1
    return c


def _lens(case):
    """Lengths of a case's requests, the same for every seed: the first has the full length, the
    second one token, every seventh none where the case says so, the rest spread over the range."""
    rng = random.Random(case["len_seed"])
    n = case["n_seq"]
    if case["op"] == "decode":
        top, low = case["max_len"], min(case["n_q"], case["max_len"])
        out = [rng.randint(low + (top - low) // 8, top) for _ in range(n)]
        out[0] = top
        if n > 1:
            out[1] = low
        if case["empty"]:
            out = [0 if i % 7 == 3 else v for i, v in enumerate(out)]
        return out
    top = case["max_new"] if case["op"] == "cache" else case["max_q"]
    new = [_log_int(rng, 1, top) for _ in range(n)]
    new[0] = top
    hist = [rng.randint(case["history"] // 2, case["history"]) for _ in range(n)]
    return new, hist


def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    op = case["op"]
    item = {"bf16": 2 * (DC + DR), "fp16": 2 * (DC + DR), "fp8": ROW8}[case["dtype"]]
    if op == "cache":
        new, hist = _lens(case)
        n, total = sum(new), sum(new) + sum(hist)
        b = n * (2 * (DC + DR) + item + 8)
        if case["read"]:
            b += total * (item + 2 * (DC + DR))
        return {"bytes": b, "flops": 4 * n * DC if case["dtype"] == "fp8" else 0}
    if op == "decode":
        lens = _lens(case)
        rows = case["n_q"] * case["heads"]
        b = sum(lens) * item + len(lens) * rows * 2 * (DC + DR + DC)
        return {"bytes": b, "flops": 2 * rows * sum(lens) * (DC + DR + DC)}
    if op == "prefill":
        new, hist = _lens(case)
        tq, tk, h = sum(new), sum(new) + sum(hist), case["heads"]
        pairs = sum(n * (n + p) - (n * (n - 1) // 2 if case["causal"] else 0) for n, p in zip(new, hist))
        b = 2 * (tq * h * (DN + DR + DN) + tk * h * 2 * DN + tk * DR)
        return {"bytes": b, "flops": 2 * h * pairs * (DN + DR + DN)}
    m, e, k = case["tokens"], case["experts"], case["topk"]
    kk, nn = case["hidden"], case["inter"]
    hit = e * (1.0 - (1.0 - k / e) ** m)   # experts that m tokens reach on average
    wbytes = 3 * kk * nn * (1 if case["dtype"] == "fp8" else 2)
    return {"bytes": int(hit * wbytes + m * (4 * kk + 4 * e)), "flops": 6 * m * k * kk * nn}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(lens, page, gen):
    """A block table over shuffled pages, with a few pages that no request holds."""
    need = [max(1, -(-n // page)) for n in lens]
    width = max(need)
    perm = torch.randperm(sum(need) + 5, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), int(perm[0]), dtype=torch.int32)
    host, o = perm.cpu(), 0
    for i, n in enumerate(need):
        table[i, :n] = host[o:o + n]
        o += n
    return table.cuda(), sum(need) + 5


def _slot_ids(table, page, first, last):
    """Cache slots of positions first[b] .. last[b] - 1 of every request, in order."""
    host, out = table.cpu().long(), []
    for b, (p, n) in enumerate(zip(first, last)):
        pos = torch.arange(p, n)
        out.append(host[b][pos // page] * page + pos % page)
    return torch.cat(out).cuda()


def _filled_cache(case, lens, table, n_pages, gen):
    """A cache whose first lens[b] positions hold tokens; its other slots hold NaN where only
    tokens are read, zeros where the whole cache is an output."""
    page = case["page"]
    rest = 0.0 if case["op"] == "cache" and not case["read"] else float("nan")
    live = _slot_ids(table, page, [0] * len(lens), lens)
    if case["dtype"] == "fp8":
        cache = torch.full((n_pages, page, ROW8), 0x7F, dtype=torch.uint8, device="cuda")
        codes, rope, scale = _views8(cache)
        x = torch.randn(live.numel(), DC, generator=gen, device="cuda") * 150
        codes[live // page, live % page] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        rope.fill_(float("nan"))
        rope[live // page, live % page] = torch.randn(live.numel(), DR, generator=gen, device="cuda").bfloat16()
        scale[live // page, live % page] = torch.randint(118, 121, (live.numel(), DC // 128), generator=gen,
                                                         device="cuda", dtype=torch.uint8)
        return cache
    cache = torch.full((n_pages, page, DC + DR), rest, dtype=_DT[case["dtype"]], device="cuda")
    rows = torch.randn(live.numel(), DC + DR, generator=gen, device="cuda").to(cache.dtype)
    cache.view(-1, DC + DR)[live] = rows
    return cache


def _views8(cache):
    """The three parts of 8-bit pages: codes [P, page, 512], rotary keys bf16 [P, page, 64] and
    the exponent bytes of the block scales [P, page, 4]."""
    n, page, _ = cache.shape
    flat = cache.view(n, page * ROW8)
    a, b = page * DC, page * (DC + 2 * DR)
    return (flat[:, :a].view(n, page, DC), flat[:, a:b].view(torch.bfloat16).view(n, page, DR),
            flat[:, b:].view(n, page, DC // 128))


def prepare(case, seed):
    gen = _gen(seed)
    op, dt = case["op"], _DT[case["dtype"]]
    st = {"case": case}
    if op == "cache":
        new, hist = _lens(case)
        lens = [a + b for a, b in zip(new, hist)]
        table, n_pages = _pages(lens, case["page"], gen)
        st["cache"] = _filled_cache(case, hist, table, n_pages, gen)
        st["latent"] = torch.randn(sum(new), DC, generator=gen, device="cuda").to(dt)
        # the rotary key is a column slice of a wider projection's output
        st["k_rope"] = torch.randn(sum(new), DR + 192, generator=gen, device="cuda").to(dt)[:, 192:]
        st["slots"] = _slot_ids(table, case["page"], hist, lens)
        st["table"], st["total"] = table, sum(lens)
        st["cu"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
        st["all_slots"] = _slot_ids(table, case["page"], [0] * len(lens), lens)
    elif op == "decode":
        lens = _lens(case)
        table, n_pages = _pages(lens, case["page"], gen)
        st["cache"] = _filled_cache(case, lens, table, n_pages, gen)
        st["q"] = torch.randn(len(lens), case["n_q"], case["heads"], DC + DR, generator=gen, device="cuda").to(dt)
        st["table"], st["host_lens"] = table, lens
        st["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
        st["scale"] = 1.0 / math.sqrt(DN + DR)
    elif op == "prefill":
        new, hist = _lens(case)
        lens = [a + b for a, b in zip(new, hist)]
        h = case["heads"]
        st["q"] = torch.randn(sum(new), h, DN + DR, generator=gen, device="cuda").to(dt)
        st["kv"] = torch.randn(sum(lens), h, 2 * DN, generator=gen, device="cuda").to(dt)
        st["k_rope"] = torch.randn(sum(lens), DR, generator=gen, device="cuda").to(dt)
        st["new"], st["host_lens"] = new, lens
        st["cu_q"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        st["cu_k"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
        st["scale"] = 1.0 / math.sqrt(DN + DR)
    else:
        m, e, kk, nn = case["tokens"], case["experts"], case["hidden"], case["inter"]
        st["x"] = torch.randn(m, kk, generator=gen, device="cuda").to(dt)
        st["logits"] = torch.randn(m, e, generator=gen, device="cuda")
        st["bias"] = torch.randn(e, generator=gen, device="cuda") * 0.01 if case["bias"] else None
        for name, rows, cols in (("w1", 2 * nn, kk), ("w2", kk, nn)):
            if case["dtype"] == "fp8":
                w = torch.empty(e, rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
                for i in range(e):
                    w[i] = (torch.randn(rows, cols, generator=gen, device="cuda") * 100).clamp(-448, 448).to(w.dtype)
                mid = round(math.log2(1.0 / math.sqrt(cols) / 100))
                ex = torch.randint(mid - 1, mid + 1, (e, rows // 128, cols // 128), generator=gen, device="cuda")
                st[name + "_scale"] = torch.exp2(ex.float())
            else:
                w = torch.empty(e, rows, cols, dtype=dt, device="cuda")
                for i in range(e):
                    w[i] = (torch.randn(rows, cols, generator=gen, device="cuda") / math.sqrt(cols)).to(dt)
                st[name + "_scale"] = None
            st[name] = w
    return st


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_cache(st):
    import kernelswift_competition_submission_b200 as pkg
    pkg.latent_cache_write(st["cache"], st["latent"], st["k_rope"], st["slots"])
    if not st["case"]["read"]:
        return st["cache"]
    return pkg.latent_cache_read(st["cache"], st["table"], st["cu"], st["total"])


def _own_decode(st):
    import kernelswift_competition_submission_b200 as pkg
    return pkg.latent_attention_decode(st["q"], st["cache"], st["table"], st["lens"], st["scale"],
                                       return_lse=st["case"]["lse"])


def _own_prefill(st):
    import kernelswift_competition_submission_b200 as pkg
    return pkg.latent_attention_prefill(st["q"], st["kv"], st["k_rope"], st["cu_q"], st["cu_k"], st["scale"],
                                        causal=st["case"]["causal"], return_lse=st["case"]["lse"])


def _own_moe(st):
    import kernelswift_competition_submission_b200 as pkg
    c = st["case"]
    return pkg.moe_decode(st["x"], st["logits"], st["w1"], st["w2"], topk=c["topk"], renormalize=True,
                          num_expert_group=c["groups"], topk_group=c["topk_group"], scoring_func=c["scoring"],
                          routed_scaling_factor=2.5, e_score_correction_bias=st["bias"],
                          w1_scale=st["w1_scale"], w2_scale=st["w2_scale"])


def _plain_cache(st):
    cache, page = st["cache"], st["case"]["page"]
    slots = st["slots"]
    if st["case"]["dtype"] != "fp8":
        rows = cache.view(-1, DC + DR)
        rows[slots] = torch.cat([st["latent"], st["k_rope"]], 1)
        if not st["case"]["read"]:
            return cache
        got = rows[st["all_slots"]]
        return got[:, :DC].contiguous(), got[:, DC:].contiguous()
    codes, rope, scale = _views8(cache)
    x = st["latent"].float().view(-1, DC // 128, 128)
    t = x.abs().amax(-1) / 448.0
    bits = t.view(torch.int32)
    up = torch.where((bits & 0x7FFFFF) != 0, (bits >> 23) + 1, bits >> 23)
    up = torch.where(t > 0, up, torch.full_like(up, 127))   # an all-zero block takes the scale 1
    s = (up << 23).view(torch.float32)
    q = (x / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    page_of, off = slots // page, slots % page
    codes[page_of, off] = q.view(-1, DC)
    rope[page_of, off] = st["k_rope"]
    scale[page_of, off] = up.to(torch.uint8)
    return _read8(st["cache"], st["all_slots"])


def _read8(cache, slots):
    codes, rope, scale = _views8(cache)
    page = cache.shape[1]
    page_of, off = slots // page, slots % page
    c = codes[page_of, off].view(torch.float8_e4m3fn).float().view(-1, DC // 128, 128)
    s = (scale[page_of, off].int() << 23).view(torch.float32)
    return (c * s[..., None]).view(-1, DC).bfloat16(), rope[page_of, off]


def _context(st, b, n):
    """The n cached rows of request b, in 32 bits."""
    page = st["case"]["page"]
    pages = st["table"][b, :-(-n // page)].long()
    if st["case"]["dtype"] != "fp8":
        return st["cache"][pages].view(-1, DC + DR)[:n].float()
    codes, rope, scale = _views8(st["cache"])
    c = codes[pages].reshape(-1, DC)[:n].view(torch.float8_e4m3fn).float().view(n, DC // 128, 128)
    s = (scale[pages].reshape(-1, DC // 128)[:n].int() << 23).view(torch.float32)
    return torch.cat([(c * s[..., None]).view(n, DC), rope[pages].reshape(-1, DR)[:n].float()], 1)


def _plain_decode(st):
    c = st["case"]
    q, nq, h = st["q"], c["n_q"], c["heads"]
    out = torch.zeros(q.shape[0], nq, h, DC, dtype=q.dtype, device=q.device)
    lse = torch.full((q.shape[0], nq, h), float("-inf"), device=q.device)
    for b, n in enumerate(st["host_lens"]):
        if n == 0:
            continue
        kv = _context(st, b, n)
        s = (q[b].float().view(nq * h, DC + DR) @ kv.T).view(nq, h, n) * st["scale"]
        if nq > 1:   # draft token i sees the context up to and with itself
            last = n - nq + torch.arange(nq, device=q.device)
            hide = torch.arange(n, device=q.device)[None, :] > last[:, None]
            s = s.masked_fill(hide[:, None, :], float("-inf"))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        z = p.sum(-1, keepdim=True)
        out[b] = ((p.view(nq * h, n) @ kv[:, :DC]).view(nq, h, DC) / z).to(q.dtype)
        lse[b] = (top + torch.log(z))[..., 0]
    return (out, lse) if c["lse"] else out


def _plain_prefill(st):
    c = st["case"]
    q, kv, kr, h = st["q"], st["kv"], st["k_rope"], c["heads"]
    out = torch.zeros(q.shape[0], h, DN, dtype=q.dtype, device=q.device)
    lse = torch.full((q.shape[0], h), float("-inf"), device=q.device)
    oq = ok = 0
    for n, m in zip(st["new"], st["host_lens"]):
        step = max(1, (1 << 28) // (n * m))   # heads at a time: score tables of about a gigabyte
        rope = kr[ok:ok + m].float()
        for h0 in range(0, h, step):
            qs = q[oq:oq + n, h0:h0 + step].float().transpose(0, 1)
            ks = kv[ok:ok + m, h0:h0 + step, :DN].float().transpose(0, 1)
            vs = kv[ok:ok + m, h0:h0 + step, DN:].float().transpose(0, 1)
            s = (qs[..., :DN] @ ks.transpose(1, 2) + qs[..., DN:] @ rope.T) * st["scale"]
            if c["causal"]:
                last = m - n + torch.arange(n, device=q.device)
                s.masked_fill_((torch.arange(m, device=q.device)[None, :] > last[:, None])[None], float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = s.sub_(top).exp_()
            z = p.sum(-1, keepdim=True)
            out[oq:oq + n, h0:h0 + step] = ((p @ vs) / z).transpose(0, 1).to(q.dtype)
            lse[oq:oq + n, h0:h0 + step] = (top + torch.log(z))[..., 0].T
        oq, ok = oq + n, ok + m
    return (out, lse) if c["lse"] else out


def _plain_moe(st):
    c = st["case"]
    e, g, k = c["experts"], c["groups"], c["topk"]
    logits = st["logits"].float()
    m = logits.shape[0]
    if c["scoring"] == "sigmoid":
        scores = 1.0 / (1.0 + torch.exp(-logits))
    else:
        ex = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = ex / ex.sum(-1, keepdim=True)
    rank = scores if st["bias"] is None else scores + st["bias"]
    groups = rank.view(m, g, e // g)
    if st["bias"] is None:
        gs = groups.amax(-1)
    else:
        gs = groups.sort(-1, descending=True)[0][..., :2].sum(-1)
    keep = gs.sort(dim=-1, descending=True, stable=True)[1][:, :c["topk_group"]]
    kept = torch.zeros_like(gs, dtype=torch.bool).scatter_(1, keep, True)
    rank = groups.masked_fill(~kept[..., None], float("-inf")).view(m, e)
    ids = rank.sort(dim=-1, descending=True, stable=True)[1][:, :k]
    wt = scores.gather(1, ids)
    wt = wt / wt.sum(-1, keepdim=True) * 2.5
    x, nn = st["x"].float(), c["inter"]
    out = torch.zeros(m, c["hidden"], device=x.device)
    for j in range(k):
        h = torch.bmm(_weights(st, "w1", ids[:, j]), x[:, :, None])[..., 0]
        a = h[:, :nn] / (1.0 + torch.exp(-h[:, :nn])) * h[:, nn:]
        out += wt[:, j:j + 1] * torch.bmm(_weights(st, "w2", ids[:, j]), a[:, :, None])[..., 0]
    return out.to(st["x"].dtype)


def _weights(st, name, ids):
    w = st[name][ids] if st[name].element_size() > 1 else st[name].view(torch.uint8)[ids].view(torch.float8_e4m3fn)
    w = w.float()
    if st[name + "_scale"] is None:
        return w
    n, r, c = w.shape
    w.view(n, r // 128, 128, c // 128, 128).mul_(st[name + "_scale"][ids][:, :, None, :, None])
    return w


_OWN = {"cache": _own_cache, "decode": _own_decode, "prefill": _own_prefill, "moe": _own_moe}
_PLAIN = {"cache": _plain_cache, "decode": _plain_decode, "prefill": _plain_prefill, "moe": _plain_moe}


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    st = prepare(case, seed)
    return {"cache": _exact_cache, "decode": _exact_decode, "prefill": _exact_prefill,
            "moe": _exact_moe}[case["op"]](case, st)


def _e4m3_values(codes):
    """Values of e4m3 bytes from the format: sign, 4 exponent bits (bias 7), 3 fraction bits."""
    c = codes.long()
    e, f = (c >> 3) & 15, (c & 7).double()
    mag = torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * torch.exp2((e - 7).double()))
    mag = torch.where((c & 127) == 127, torch.full_like(mag, float("nan")), mag)
    return torch.where(c >= 128, -mag, mag)


def _e4m3_round(v):
    """v (|v| <= 448, float64) rounded to the nearest e4m3 value, ties to the even fraction."""
    ex = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    ex = torch.where(torch.exp2(ex) > v.abs().clamp_min(2.0 ** -6), ex - 1, ex)
    step = torch.exp2(ex - 3)
    return torch.round(v / step) * step


def _cache_rows64(case, cache, slots):
    page = case["page"]
    if case["dtype"] != "fp8":
        return cache.reshape(-1, DC + DR)[slots].double()
    flat = cache.reshape(cache.shape[0], -1)
    pg, off = (slots // page)[:, None], (slots % page)[:, None]
    col = torch.arange(DC, device=cache.device)[None]
    lat = _e4m3_values(flat[pg, off * DC + col])
    rcol = torch.arange(2 * DR, device=cache.device)[None]
    rope = flat[pg, page * DC + off * 2 * DR + rcol].view(torch.bfloat16).double()
    sc = flat[pg, page * (DC + 2 * DR) + off * 4 + col // 128].double()
    return torch.cat([lat * torch.exp2(sc - 127), rope], 1)


def _exact_cache(case, st):
    lat, rope = st["latent"].double(), st["k_rope"].double()
    if case["dtype"] == "fp8":
        amax = lat.view(-1, 4, 128).abs().amax(-1)
        s = torch.exp2(torch.ceil(torch.log2(amax / 448)))
        s = torch.where(amax > 0, s, torch.ones_like(s)).repeat_interleave(128, 1)
        lat = _e4m3_round(lat / s) * s
    new = torch.cat([lat, rope], 1)
    if not case["read"]:
        whole = st["cache"].double()
        whole.view(-1, DC + DR)[st["slots"]] = new
        return whole
    n_slots = st["cache"].shape[0] * case["page"]
    where = torch.full((n_slots,), -1, dtype=torch.long, device="cuda")
    where[st["slots"]] = torch.arange(new.shape[0], device="cuda")
    pick = where[st["all_slots"]]
    rows = _cache_rows64(case, st["cache"], st["all_slots"])
    rows = torch.where((pick >= 0)[:, None], new[pick.clamp_min(0)], rows)
    return rows[:, :DC], rows[:, DC:]


def _exact_decode(case, st):
    nq, h = case["n_q"], case["heads"]
    lens = st["lens"].tolist()
    out = torch.zeros(len(lens), nq, h, DC, dtype=torch.float64, device="cuda")
    lse = torch.full((len(lens), nq, h), float("-inf"), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if n == 0:
            continue
        rows = _cache_rows64(case, st["cache"], _slot_ids(st["table"][b:b + 1], case["page"], [0], [n]))
        for i in range(nq):
            m = n - nq + 1 + i
            s = torch.einsum("hd,nd->hn", st["q"][b, i].double(), rows[:m]) * st["scale"]
            lse[b, i] = torch.logsumexp(s, -1)
            out[b, i] = torch.exp(s - lse[b, i][:, None]) @ rows[:m, :DC]
    return (out, lse) if case["lse"] else out


def _exact_prefill(case, st):
    h = case["heads"]
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    out = torch.zeros(cq[-1], h, DN, dtype=torch.float64, device="cuda")
    lse = torch.full((cq[-1], h), float("-inf"), dtype=torch.float64, device="cuda")
    for b in range(len(cq) - 1):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        rope = st["k_rope"][ck[b]:ck[b + 1]].double()
        for j in range(h):
            key = torch.cat([st["kv"][ck[b]:ck[b + 1], j, :DN].double(), rope], 1)
            val = st["kv"][ck[b]:ck[b + 1], j, DN:].double()
            for r0 in range(0, n, 2048):
                r1 = min(n, r0 + 2048)
                seen = m - n + r1 if case["causal"] else m
                s = (st["q"][cq[b] + r0:cq[b] + r1, j].double() @ key[:seen].T) * st["scale"]
                if case["causal"]:
                    s += torch.full_like(s, float("-inf")).triu(m - n + r0 + 1)
                z = torch.logsumexp(s, -1)
                lse[cq[b] + r0:cq[b] + r1, j] = z
                out[cq[b] + r0:cq[b] + r1, j] = torch.exp(s - z[:, None]) @ val[:seen]
    return (out, lse) if case["lse"] else out


def _exact_moe(case, st):
    e, g, k, nn = case["experts"], case["groups"], case["topk"], case["inter"]
    z = st["logits"].double()
    scores = torch.sigmoid(z) if case["scoring"] == "sigmoid" else torch.softmax(z, -1)
    x = st["x"].double()
    out = torch.zeros(z.shape[0], case["hidden"], dtype=torch.float64, device="cuda")
    pairs = {}
    bias = torch.zeros(e) if st["bias"] is None else st["bias"].double().cpu()
    for t, row in enumerate(scores.cpu()):
        val = (row + bias).tolist()
        per = [val[i * (e // g):(i + 1) * (e // g)] for i in range(g)]
        gsc = [max(p) if st["bias"] is None else sum(sorted(p)[-2:]) for p in per]
        best = sorted(range(g), key=lambda i: (-gsc[i], i))[:case["topk_group"]]
        cand = [i for i in range(e) if i // (e // g) in best]
        ids = sorted(cand, key=lambda i: (-val[i], i))[:k]
        tot = sum(float(row[i]) for i in ids)
        for i in ids:
            pairs.setdefault(i, []).append((t, 2.5 * float(row[i]) / tot))
    for i, toks in pairs.items():
        mats = []
        for name in ("w1", "w2"):
            if case["dtype"] == "fp8":
                s = st[name + "_scale"][i].double().repeat_interleave(128, 0).repeat_interleave(128, 1)
                mats.append(_e4m3_values(st[name][i].view(torch.uint8)) * s)
            else:
                mats.append(st[name][i].double())
        rows = torch.tensor([t for t, _ in toks], device="cuda")
        h = x[rows] @ mats[0].T
        act = torch.nn.functional.silu(h[:, :nn]) * h[:, nn:]
        wt = torch.tensor([w for _, w in toks], dtype=torch.float64, device="cuda")
        out[rows] += wt[:, None] * (act @ mats[1].T)
    return out
