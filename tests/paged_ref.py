"""Plain 64-bit implementations of the ragged-serving operators, and the error bounds that their tests allow."""
import numpy as np
import torch

F = torch.float64
# half a unit in the last place, relative, of the 16-bit types
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def norm_rope(x, w, table_rows, eps, style):
    """x [T][heads][hd] -> normed and rotated, and sum |a| + |b| of each pair (for the bound)."""
    x = x.to(F)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(F)
    cos, sin = table_rows[:, None, :, 0].to(F), table_rows[:, None, :, 1].to(F)
    hd = x.shape[-1]
    i = torch.arange(hd // 2, device=x.device)
    ia, ib = (2 * i, 2 * i + 1) if style == "pairwise" else (i, i + hd // 2)
    a, b = y[..., ia], y[..., ib]
    out, mag = torch.empty_like(y), torch.empty_like(y)
    out[..., ia], out[..., ib] = a * cos - b * sin, a * sin + b * cos
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return out, mag


def norm_rope_bound(want, mag, dtype):
    # one rounding of the result, a few f32 operations on |a| + |b| (norm sum of
    # 128 squares, rsqrt, two products, one sum: under 2^-18), fp16 subnormals
    return UNIT[dtype] * want.abs() + 2.0 ** -18 * mag + 2.0 ** -25


def attention(q, k, v, page_table, q_start, kv_len, scale, before):
    """`before` [T][n_q * hd] are the output rows as they were.  Returns the
    result and the bound of its error, both [T][n_q][hd]."""
    P, n_kv, page, hd = k.shape
    T = q.shape[0]
    n_q = q.shape[1] // hd
    G = n_q // n_kv
    u = UNIT[q.dtype]
    qd = q.to(F).view(T, n_q, hd)
    out = before.to(F).view(T, n_q, hd).clone()
    tol = torch.zeros_like(out)
    for s in range(len(kv_len)):
        a, b = int(q_start[s]), int(q_start[s + 1])
        n, L = b - a, int(kv_len[s])
        if n == 0:
            continue
        j = torch.arange(max(L, 0), device=q.device)
        j = j[: page_table.shape[1] * page]
        pg = page_table[s].long()[j // page]
        ok = (pg >= 0) & (pg < P)
        j, pg = j[ok], pg[ok]
        kk, vv = k[pg, :, j % page].to(F), v[pg, :, j % page].to(F)          # [keys][n_kv][hd]
        kk, vv = kk.repeat_interleave(G, 1), vv.repeat_interleave(G, 1)
        sc = torch.einsum("ihd,jhd->hij", qd[a:b], kk) * scale
        see = j[None, :] <= (L - n + torch.arange(n, device=q.device))[:, None]
        sc = sc.masked_fill(~see, -torch.inf)
        p = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0) if j.numel() else sc
        out[a:b] = torch.einsum("hij,jhd->ihd", p, vv)
        # probabilities and result rounded once each to the 16-bit type; f32
        # scores of hd products of |q||k| (2^-24 hd |s|max, under 2e-4 here);
        # probabilities below the normal fp16 range: 2^-25 of the row's largest
        w = torch.einsum("hij,jhd->ihd", p, vv.abs())
        low = torch.einsum("hij,jhd->ihd", see[None].to(F) * p.amax(-1, keepdim=True), vv.abs()) if j.numel() else w
        tol[a:b] = (2 * u + 2e-4) * w + 2.0 ** -25 * low + 2.0 ** -24
    return out, tol


def logprobs(x, tokens, k):
    """x [rows][n]; tokens [rows][m].  Rows of -infinity: -infinity, entropy 0."""
    x = x.to(F)
    n = x.shape[1]
    empty = torch.isinf(x).all(-1) & (x < 0).all(-1)
    # from the maximum down: x - lse itself would lose ln(sum) for |x| over 2^52
    m = torch.where(empty, torch.zeros_like(x[:, 0]), x.amax(-1))
    ls = torch.logsumexp(x - m[:, None], -1)
    lse = m + ls
    lp = torch.where(empty[:, None], torch.full_like(x, -torch.inf), x - m[:, None] - ls[:, None])
    p = lp.exp()
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(-1)
    t = tokens.long()
    got = lp.gather(1, t.clamp(0, n - 1))
    got = torch.where(t < 0, torch.zeros_like(got), torch.where(t >= n, torch.full_like(got, torch.nan), got))
    # value descending, id ascending, disallowed tokens never
    order = torch.sort(torch.where(torch.isnan(x), torch.full_like(x, -torch.inf), x), dim=-1, descending=True, stable=True)
    ids = torch.nn.functional.pad(order.indices, (0, max(0, k - n)), value=-1)[:, :k].clone()
    val = torch.nn.functional.pad(order.values, (0, max(0, k - n)), value=-torch.inf)[:, :k]
    none = val == -torch.inf
    top = torch.where(none, val, val - m[:, None] - ls[:, None])
    top[none & torch.isnan(lse)[:, None]] = torch.nan
    ids[none] = -1
    return got, ent, lse, ids.to(torch.int32), top


def pool(rng, pages, n_kv, page, hd, dtype, layout):
    """Equal K and V page pools of an interesting stride: "head" by head, "token" by token, "both" in one allocation."""
    def r(*shape):
        return torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).cuda().to(dtype)
    if layout == "head":
        return r(pages, n_kv, page, hd), r(pages, n_kv, page, hd)
    if layout == "token":
        return r(pages, page, n_kv, hd).transpose(1, 2), r(pages, page, n_kv, hd).transpose(1, 2)
    both = r(pages, 2, n_kv, page, hd)
    return both[:, 0], both[:, 1]
