"""What is measured of the ragged-serving operators: per-head query/key norms with the rotation, written to a page pool;
attention of new tokens over the paged cache; log probabilities of given tokens with entropy and top alternatives.

`own` False: plain torch in 32 bits, rounded once at the end.  `own` True: the calls a user makes of nnzap_b200.paged.
Head layouts and sizes are the Bonsai preset's (16 query / 8 key-value heads of 128, vocabulary 151936 or the trimmed
151669, prompt chunks of 512, context up to 32768) and those of the package's head_dim 64 kernels (8 / 2 heads)."""
import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-6


def listed():
    return [
        # one decode step of one sequence: a launch-latency case
        {"name": "norm_rope_1", "op": "norm_rope", "tokens": 1, "n_q": 16, "n_kv": 8, "hd": 128, "page": 16,
         "dtype": "f16", "style": "pairwise", "token_major": False, "start": 515},
        # one prefill chunk of the engine's maximum length
        {"name": "norm_rope_512", "op": "norm_rope", "tokens": 512, "n_q": 16, "n_kv": 8, "hd": 128, "page": 16,
         "dtype": "f16", "style": "pairwise", "token_major": False, "start": 4096},
        # a long prompt in one pass, odd length, half-split rotation, pages stored token by token
        {"name": "norm_rope_8191", "op": "norm_rope", "tokens": 8191, "n_q": 16, "n_kv": 8, "hd": 128, "page": 64,
         "dtype": "bf16", "style": "half_split", "token_major": True, "start": 0},
        # one token of one conversation: latency
        {"name": "attn_1x515", "op": "attn", "seqs": 1, "singles": 1, "chunk": 0, "kv_min": 515, "kv_max": 515,
         "n_q": 16, "n_kv": 8, "hd": 128, "page": 16, "dtype": "f16", "token_major": False},
        # a decode batch of 64 conversations of different lengths
        {"name": "attn_64x4032", "op": "attn", "seqs": 64, "singles": 64, "chunk": 0, "kv_min": 2017, "kv_max": 4032,
         "n_q": 16, "n_kv": 8, "hd": 128, "page": 16, "dtype": "f16", "token_major": False},
        # one token over a full context: few rows, a long axis
        {"name": "attn_1x32767", "op": "attn", "seqs": 1, "singles": 1, "chunk": 0, "kv_min": 32767, "kv_max": 32767,
         "n_q": 16, "n_kv": 8, "hd": 128, "page": 64, "dtype": "bf16", "token_major": True},
        # a prompt chunk behind 4096 cached tokens
        {"name": "attn_chunk512", "op": "attn", "seqs": 1, "singles": 0, "chunk": 512, "kv_min": 4608, "kv_max": 4608,
         "n_q": 16, "n_kv": 8, "hd": 128, "page": 16, "dtype": "f16", "token_major": False},
        # a mixed serving step: 31 single tokens and one odd prompt chunk, head_dim 64
        {"name": "attn_mixed", "op": "attn", "seqs": 32, "singles": 31, "chunk": 449, "kv_min": 601, "kv_max": 4001,
         "n_q": 8, "n_kv": 2, "hd": 64, "page": 24, "dtype": "bf16", "token_major": False},
        # a long prompt's second half: bound by the tensor cores
        {"name": "attn_chunk4096", "op": "attn", "seqs": 1, "singles": 0, "chunk": 4096, "kv_min": 8192, "kv_max": 8192,
         "n_q": 16, "n_kv": 8, "hd": 128, "page": 64, "dtype": "bf16", "token_major": False},
        # the sampled token's log probability in single-row decoding
        {"name": "logprobs_1", "op": "logprobs", "rows": 1, "vocab": 151936, "pad": 0, "top_k": 5, "dtype": "f32"},
        # a decode batch, trimmed odd vocabulary in padded rows, some tokens disallowed
        {"name": "logprobs_64", "op": "logprobs", "rows": 64, "vocab": 151669, "pad": 267, "top_k": 20, "dtype": "bf16"},
        # scoring one prompt chunk
        {"name": "logprobs_512", "op": "logprobs", "rows": 512, "vocab": 151936, "pad": 0, "top_k": 20, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "attn", "attn", "logprobs"])
    if op == "logprobs":
        rows = _log_int(rng, 1, 512)
        vocab = _log_int(rng, 500, 151936)
        return {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 3, 64]), "top_k": rng.choice([0, 1, 5, 20, 32]),
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    n_q, n_kv, hd = rng.choice([(16, 8, 128), (16, 8, 128), (8, 2, 64), (8, 8, 128), (32, 8, 128), (4, 2, 128), (6, 2, 64)])
    base = {"op": op, "n_q": n_q, "n_kv": n_kv, "hd": hd, "page": rng.choice([8, 16, 16, 24, 64, 128]),
            "dtype": rng.choice(["f16", "bf16"]), "token_major": rng.random() < 0.5}
    if op == "norm_rope":
        return dict(base, tokens=_log_int(rng, 1, 4096), style=rng.choice(["pairwise", "half_split"]), start=rng.randrange(0, 8192))
    kind = rng.choice(["single", "batch", "chunk", "mixed"])
    if kind == "single":
        kv = _log_int(rng, 1, 32767)
        return dict(base, seqs=1, singles=1, chunk=0, kv_min=kv, kv_max=kv)
    if kind == "batch":
        seqs = _log_int(rng, 2, 64)
        hi = _log_int(rng, 16, 4032)
        return dict(base, seqs=seqs, singles=seqs, chunk=0, kv_min=rng.randint(1, hi), kv_max=hi)
    chunk = _log_int(rng, 2, 2048)
    if kind == "chunk":
        kv = chunk + _log_int(rng, 1, 4096) - 1
        return dict(base, seqs=1, singles=0, chunk=chunk, kv_min=kv, kv_max=kv)
    seqs = _log_int(rng, 2, 24)
    chunk = min(chunk, 512)
    return dict(base, seqs=seqs, singles=seqs - 1, chunk=chunk, kv_min=chunk + rng.randint(0, 200), kv_max=chunk + 200 + _log_int(rng, 1, 2048))


def _pool(g, pages, c, dt):
    """K or V page pool, indexed [page][kv head][slot in page][d]; stored head by head, or token by token."""
    n_kv, page, hd = c["n_kv"], c["page"], c["hd"]
    if c["token_major"]:
        return torch.randn(pages, page, n_kv, hd, device="cuda", generator=g, dtype=torch.float32).to(dt).transpose(1, 2)
    return torch.randn(pages, n_kv, page, hd, device="cuda", generator=g, dtype=torch.float32).to(dt)


def _lens(case):
    """(new tokens, keys) of every sequence: the chunk first, then the single tokens, lengths spread over the range."""
    n, lo, hi = case["seqs"], case["kv_min"], case["kv_max"]
    new = [case["chunk"]] * (n - case["singles"]) + [1] * case["singles"]
    kv = [hi if n == 1 else lo + (hi - lo) * ((i * 7919) % n) // max(1, n - 1) for i in range(n)]
    return new, [max(a, b) for a, b in zip(kv, new)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    if case["op"] == "logprobs":
        R, V = case["rows"], case["vocab"]
        full = torch.randn(R, V + case["pad"], device="cuda", generator=g) * 3
        if case["pad"]:  # padded vocabularies come with rows that disallow some tokens
            full[torch.rand(R, V + case["pad"], device="cuda", generator=g) < 0.01] = -math.inf
        tokens = torch.randint(0, V, (R,), device="cuda", generator=g)
        full[torch.arange(R, device="cuda"), tokens] = 2.0   # a given token is an allowed one
        return {"case": case, "logits": full.to(dt)[:, :V], "tokens": tokens.to(torch.int32)}
    n_q, n_kv, hd, page = case["n_q"], case["n_kv"], case["hd"], case["page"]
    s = {"case": case}
    if case["op"] == "norm_rope":
        T = case["tokens"]
        pages = (T + page - 1) // page + 3
        s["k"], s["v"] = _pool(g, pages, case, dt), _pool(g, pages, case, dt)
        s["qkv"] = torch.randn(T, (n_q + 2 * n_kv) * hd, device="cuda", generator=g).to(dt)
        s["q_norm"] = 1 + 0.2 * torch.randn(hd, device="cuda", generator=g)
        s["k_norm"] = 1 + 0.2 * torch.randn(hd, device="cuda", generator=g)
        s["positions"] = torch.arange(case["start"], case["start"] + T, device="cuda", dtype=torch.int32)
        order = torch.randperm(pages, device="cuda", generator=g)
        t = torch.arange(T, device="cuda")
        s["slots"] = order[t // page] * page + t % page
        ang = torch.arange(case["start"] + T, device="cuda", dtype=torch.float64)[:, None] * (
            1e6 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))
        s["table"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s["q"] = torch.empty(T, n_q * hd, device="cuda", dtype=dt)
        if own:
            from nnzap_b200 import paged
            s["kv"] = paged.PagedKV(s["k"], s["v"])
            s["op"] = paged.QKNormRope(s["kv"], n_q, s["q_norm"], s["k_norm"], s["table"], eps=_EPS, rope_style=case["style"])
        return s
    new, kv = _lens(case)
    need = [(L + page - 1) // page for L in kv]
    pages = sum(need) + 1
    s["k"], s["v"] = _pool(g, pages, case, dt), _pool(g, pages, case, dt)
    s["qf"] = torch.randn(sum(new), n_q * hd, device="cuda", generator=g).to(dt)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed), dtype=torch.int64).to(torch.int32)
    table, at = torch.full((len(kv), max(need)), -1, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["page_table"] = table.cuda()
    s["q_start"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    s["max_new"] = max(new)
    s["out"] = torch.empty_like(s["qf"])
    if own:
        from nnzap_b200 import paged
        s["kv"] = paged.PagedKV(s["k"], s["v"])
        s["op"] = paged.PagedAttention(s["kv"], n_q)
    return s


def _plain_norm_rope(s):
    c = s["case"]
    n_q, n_kv, hd = c["n_q"], c["n_kv"], c["hd"]
    x = s["qkv"].float().view(c["tokens"], n_q + 2 * n_kv, hd)
    qk = x[:, :n_q + n_kv]
    w = torch.cat([s["q_norm"].expand(n_q, hd), s["k_norm"].expand(n_kv, hd)])
    y = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + _EPS) * w
    cs = s["table"][s["positions"].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    if c["style"] == "pairwise":
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    s["q"].copy_(y[:, :n_q].reshape(c["tokens"], n_q * hd))
    pg, at = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k"][pg, :, at] = y[:, n_q:].to(s["k"].dtype)
    s["v"][pg, :, at] = x[:, n_q + n_kv:].to(s["v"].dtype)
    return s["q"], s["k"], s["v"]


def _plain_attn(s):
    c = s["case"]
    n_q, n_kv, hd, page, N = c["n_q"], c["n_kv"], c["hd"], c["page"], s["max_new"]
    S, W = s["page_table"].shape
    pt = s["page_table"].long()
    j = torch.arange(W * page, device="cuda")
    here = (pt >= 0).repeat_interleave(page, 1) & (j < s["kv_len"][:, None])             # [S][keys]
    k = s["k"][pt.clamp(min=0)].float().transpose(2, 3).reshape(S, W * page, n_kv, hd)
    v = s["v"][pt.clamp(min=0)].float().transpose(2, 3).reshape(S, W * page, n_kv, hd) * here[..., None, None]
    start = s["q_start"][:-1].long()
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(N, device="cuda")
    live = i < n[:, None]                                                                  # [S][new]
    at = torch.where(live, start[:, None] + i, 0)
    q = s["qf"][at].float().view(S, N, n_kv, n_q // n_kv, hd)
    see = here[:, None] & (j <= (s["kv_len"] - n)[:, None, None] + i[:, None])             # [S][new][keys]
    p = torch.einsum("snkgd,sjkd->skgnj", q, k).mul_(1 / math.sqrt(hd))
    p.masked_fill_(~see[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    o = torch.einsum("skgnj,sjkd->snkgd", p, v)
    o = o / p.sum(-1).permute(0, 3, 1, 2)[..., None].clamp(min=1e-30)
    s["out"][at[live]] = o.reshape(S, N, n_q * hd)[live].to(s["out"].dtype)
    return s["out"]


def _plain_logprobs(s):
    k = s["case"]["top_k"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lp = x - m - z.log()
    p = e / z
    out = {"logprob": lp.gather(1, s["tokens"].long()[:, None])[:, 0],
           "entropy": -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)}
    if k:
        val, idx = lp.sort(dim=-1, descending=True, stable=True)
        out["top_logprobs"], out["top_ids"] = val[:, :k].contiguous(), idx[:, :k].to(torch.int32)
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm_rope": _plain_norm_rope, "attn": _plain_attn, "logprobs": _plain_logprobs}[op](state)
    if op == "norm_rope":
        q = state["op"](state["qkv"], state["positions"], state["slots"], out=state["q"])
        return q, state["k"], state["v"]
    if op == "attn":
        return state["op"](state["qf"], state["page_table"], state["q_start"], state["kv_len"], state["max_new"], out=state["out"])
    from nnzap_b200 import paged
    r = paged.token_logprobs(state["logits"], state["tokens"], top_k=state["case"]["top_k"])
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if state["case"]["top_k"]:
        out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
    return out


def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * b + case["rows"] * (12 + 8 * case["top_k"]), "flops": 5 * n}
    n_q, n_kv, hd = case["n_q"], case["n_kv"], case["hd"]
    if case["op"] == "norm_rope":
        T = case["tokens"]
        return {"bytes": 2 * T * (n_q + 2 * n_kv) * hd * b + T * (hd * 4 + 12) + hd * 8, "flops": 8 * T * (n_q + n_kv) * hd}
    new, kv = _lens(case)
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, kv))
    return {"bytes": 2 * sum(kv) * n_kv * hd * b + 2 * sum(new) * n_q * hd * b, "flops": 4 * seen * n_q * hd}


def exact(case, seed):
    """The definitions in 64 bits, one sequence or head at a time."""
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "logprobs":
        x = s["logits"].to(f)
        lse = torch.logsumexp(x, -1)
        t = s["tokens"].long()
        p = torch.exp(x - lse[:, None])
        out = {"logprob": x[torch.arange(len(t), device="cuda"), t] - lse,
               "entropy": -torch.special.xlogy(p, p).sum(-1)}
        if case["top_k"]:
            # value descending, index ascending: the k largest of (value, -index)
            val, idx = torch.sort(-x, dim=-1, stable=True)
            out["top_logprobs"] = -val[:, :case["top_k"]] - lse[:, None]
            out["top_ids"] = idx[:, :case["top_k"]].to(torch.int32)
        return out
    n_q, n_kv, hd, page = case["n_q"], case["n_kv"], case["hd"], case["page"]
    if case["op"] == "norm_rope":
        z = torch.view_as_complex(s["table"].to(f))[s["positions"].long()]                  # [T][hd/2]
        heads = s["qkv"].to(f).view(-1, n_q + 2 * n_kv, hd)
        k, v, q = s["k"].to(f), s["v"].to(f), torch.empty(case["tokens"], n_q, hd, device="cuda", dtype=f)
        for h in range(n_q + 2 * n_kv):
            x = heads[:, h]
            if h < n_q + n_kv:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + _EPS) * (s["q_norm"] if h < n_q else s["k_norm"]).to(f)
                if case["style"] == "pairwise":
                    x = torch.view_as_real(torch.view_as_complex(x.view(-1, hd // 2, 2)) * z).reshape(-1, hd)
                else:
                    y = torch.complex(x[:, :hd // 2], x[:, hd // 2:]) * z
                    x = torch.cat([y.real, y.imag], -1)
            if h < n_q:
                q[:, h] = x
            else:
                (k if h < n_q + n_kv else v)[s["slots"] // page, (h - n_q) % n_kv, s["slots"] % page] = x
        return q.reshape(case["tokens"], -1), k, v
    new, kv = _lens(case)
    out, at = torch.zeros(sum(new), n_q, hd, device="cuda", dtype=f), 0
    for i, (n, L) in enumerate(zip(new, kv)):
        rows = s["page_table"][i, :(L + page - 1) // page].long()
        for h in range(n_q):
            kh = s["k"][rows, h // (n_q // n_kv)].reshape(-1, hd)[:L].to(f)
            vh = s["v"][rows, h // (n_q // n_kv)].reshape(-1, hd)[:L].to(f)
            qh = s["qf"][at:at + n, h * hd:(h + 1) * hd].to(f)
            sc = (qh @ kh.T) / math.sqrt(hd)
            mask = torch.ones(n, L, device="cuda", dtype=torch.bool).tril(L - n)
            out[at:at + n, h] = torch.softmax(sc.masked_fill(~mask, -math.inf), -1) @ vh
        at += n
    return out.reshape(sum(new), n_q * hd)
