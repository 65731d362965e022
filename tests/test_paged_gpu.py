"""GPU parity of the ragged-serving operators (nnzap_b200.paged) with plain
64-bit implementations: page sizes, strides, head layouts, ragged lengths,
absent pages, empty rows, non-finite values where nothing may look."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(autouse=True)
def _gpu(cuda, built_lib):
    yield


def P():
    from nnzap_b200 import paged
    return paged


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def within(got, want, tol, what):
    err = (got.to(R.F) - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off; worst {float((err / tol).nan_to_num(1e9).max()):.2f} of the bound"


# ---- rotation table ---------------------------------------------------------
@pytest.mark.parametrize("hd,theta,n", [(128, 1e6, 32768), (64, 1e4, 33)])
def test_rope_table(hd, theta, n):
    t = P().rope_table(theta, hd, n)
    f = float(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd)
    ang = np.arange(n)[:, None] * f
    want = np.stack([np.cos(ang), np.sin(ang)], -1)
    # f32 rounding of the cosine, and the angle's f64 error (2^-52 of up to 32768 radians)
    assert np.abs(t.cpu().numpy() - want).max() <= 2.0 ** -24


# ---- norm + rotation into pages ----------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("style", ["pairwise", "half_split"])
@pytest.mark.parametrize("n_q,n_kv,hd,page,layout,T", [
    (16, 8, 128, 16, "head", 1), (16, 8, 128, 16, "token", 77), (4, 2, 128, 24, "both", 130), (2, 2, 64, 8, "head", 5),
    (8, 2, 64, 5, "token", 300), (3, 1, 128, 1, "head", 9), (6, 3, 64, 64, "both", 33)])
def test_qk_norm_rope(dtype, style, n_q, n_kv, hd, page, layout, T):
    rng = np.random.default_rng(T + hd)
    dt, H = DT[dtype], n_q + 2 * n_kv
    pages = T // page + 3
    k, v = R.pool(rng, pages, n_kv, page, hd, dt, layout)
    k0, v0 = k.clone(), v.clone()
    wide = dev(rng.standard_normal((T, H * hd + 24), dtype=np.float32) * 2, dt)      # rows of a wider matrix
    qkv = wide[:, 8:8 + H * hd]
    qkv[T // 2] = 0                                                                     # a zero row: eps only
    qn, kn = (dev(1 + 0.3 * rng.standard_normal(hd), torch.float32) for _ in range(2))
    table = P().rope_table(1e6, hd, 5000)
    pos = dev(rng.integers(0, 5000, T).astype(np.int32))
    slots = dev(rng.permutation(pages * page)[:T].astype(np.int64))
    if T > 2:
        slots[1] = -1                                                                   # computed, not written
    out = torch.full((T, n_q * hd + 16), 7.0, dtype=dt, device="cuda")
    got = P().QKNormRope(P().PagedKV(k, v), n_q, qn, kn, table, eps=1e-6, rope_style=style)(qkv, pos, slots, out=out[:, 8:8 + n_q * hd])
    P().stream_check()
    assert (out[:, :8] == 7).all() and (out[:, 8 + n_q * hd:] == 7).all()
    x = qkv.reshape(T, H, hd)
    rows = table[pos.long()]
    want, mag = R.norm_rope(x[:, :n_q], qn, rows, 1e-6, style)
    within(got.reshape(T, n_q, hd), want, R.norm_rope_bound(want, mag, dt), "q")
    wk, mk = R.norm_rope(x[:, n_q:n_q + n_kv], kn, rows, 1e-6, style)
    live = slots >= 0
    pg, at = slots[live] // page, slots[live] % page
    within(k[pg, :, at], wk[live], R.norm_rope_bound(wk, mk, dt)[live], "k")
    assert torch.equal(v[pg, :, at], x[live, n_q + n_kv:])
    k0[pg, :, at], v0[pg, :, at] = k[pg, :, at], v[pg, :, at]
    assert torch.equal(k, k0) and torch.equal(v, v0), "slots that no token names are left alone"


def test_qk_norm_rope_in_place_and_bad_tokens():
    """q over its own projections; a position or slot out of range is reported, its token zeroed and not written."""
    from nnzap_b200._capi import NNZ_EDEVICE, NnzError
    rng = np.random.default_rng(5)
    kv = P().PagedKV.empty(4, 2, 8, 128)
    table = P().rope_table(1e4, 128, 64)
    one = torch.ones(128, device="cuda")
    op = P().QKNormRope(kv, 4, one, one, table)
    qkv = dev(rng.standard_normal((4, 8 * 128), dtype=np.float32), torch.float16)
    src = qkv.clone()
    pos = dev(np.array([0, 63, 64, 3], np.int32))
    slots = dev(np.array([0, 9, 5, 32], np.int64))
    ref = op(src, pos, slots)
    with pytest.raises(NnzError) as e:
        P().stream_check()
    assert e.value.code == NNZ_EDEVICE
    P().stream_check()                                   # reported once
    assert (ref[2:] == 0).all() and (ref[:2] != 0).any()
    assert (kv.k[0, :, 5] == 0).all() and (kv.v[0, :, 5] == 0).all()
    assert torch.equal(kv.v[0, :, 0], src[0, 768:].view(2, 128)) and torch.equal(kv.v[1, :, 1], src[1, 768:].view(2, 128))
    op(qkv, pos, slots, out=qkv[:, :512])
    with pytest.raises(NnzError):
        P().stream_check()
    assert torch.equal(qkv[:, :512], ref) and torch.equal(qkv[:, 512:], src[:, 512:])


# more heads than a thread asks for at once: 32 of 128, 64 of 64
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("style", ["pairwise", "half_split"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n_q,n_kv,hd,T", [(32, 8, 128, 19), (64, 8, 64, 7), (70, 35, 64, 3), (128, 1, 128, 2)])
def test_qk_norm_rope_many_heads(dtype, style, in_place, n_q, n_kv, hd, T):
    rng = np.random.default_rng(n_q + hd)
    dt, H = DT[dtype], n_q + 2 * n_kv
    kv = P().PagedKV.empty(3, n_kv, 8, hd, dtype=dt)
    qkv = dev(rng.standard_normal((T, H * hd), dtype=np.float32) * 2, dt)
    src = qkv.clone().view(T, H, hd)
    qn, kn = (dev(1 + 0.3 * rng.standard_normal(hd), torch.float32) for _ in range(2))
    table = P().rope_table(1e6, hd, 5000)
    pos, slots = dev(rng.integers(0, 5000, T).astype(np.int32)), dev(rng.permutation(24)[:T].astype(np.int64))
    op = P().QKNormRope(kv, n_q, qn, kn, table, eps=1e-6, rope_style=style)
    got = op(qkv, pos, slots, out=qkv[:, :n_q * hd] if in_place else None)
    P().stream_check()
    rows = table[pos.long()]
    want, mag = R.norm_rope(src[:, :n_q], qn, rows, 1e-6, style)
    within(got.reshape(T, n_q, hd), want, R.norm_rope_bound(want, mag, dt), "q")
    wk, mk = R.norm_rope(src[:, n_q:n_q + n_kv], kn, rows, 1e-6, style)
    within(kv.k[slots // 8, :, slots % 8], wk, R.norm_rope_bound(wk, mk, dt), "k")
    assert torch.equal(kv.v[slots // 8, :, slots % 8], src[:, n_q + n_kv:])
    assert torch.equal(qkv.view(T, H, hd)[:, n_q:], src[:, n_q:])


# ---- attention over pages ------------------------------------------------------
def attn_case(seed, lens, n_q, n_kv, hd, page, dtype, layout, absent=0.0, gap=0, poison=True, scale=None, extra_cols=1):
    """lens: [(new, keys)].  Slots that no sequence owns hold NaN and infinities."""
    rng = np.random.default_rng(seed)
    dt = DT[dtype]
    need = [-(-L // page) for _, L in lens]
    pages = sum(need) + 2
    k, v = R.pool(rng, pages, n_kv, page, hd, dt, layout)
    order = rng.permutation(pages)
    table, at = np.full((len(lens), max(need) + extra_cols), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    if poison:
        used = torch.zeros(pages, page, dtype=torch.bool)
        for s, (_, L) in enumerate(lens):
            j = np.arange(L)
            used[table[s, j // page], j % page] = True
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")], dtype=dt, device="cuda")
        pg, sl = torch.nonzero(~used, as_tuple=True)
        k[pg.cuda(), :, sl.cuda()] = bad[torch.arange(hd, device="cuda") % 3]
        v[pg.cuda(), :, sl.cuda()] = bad[torch.arange(hd, device="cuda") % 3]
    if absent:
        gone = rng.random(table.shape) < absent
        for pg in table[gone & (table >= 0)]:
            k[int(pg)], v[int(pg)] = float("nan"), float("inf")
        table[gone] = -1
    new = np.array([n for n, _ in lens])
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + gap
    T = int(new.sum()) + 2 * gap
    wide = dev(rng.standard_normal((T, n_q * hd + 8), dtype=np.float32), dt)
    return {"q": wide[:, :n_q * hd], "k": k, "v": v, "table": dev(table), "q_start": dev(q_start),
            "kv_len": dev(np.array([L for _, L in lens], np.int32)), "max_new": int(new.max()), "n_q": n_q, "scale": scale}


def check_attn(c, what=""):
    out = torch.full((c["q"].shape[0], c["q"].shape[1] + 8), 3.0, dtype=c["q"].dtype, device="cuda")
    o = out[:, :c["q"].shape[1]]
    kv = P().PagedKV(c["k"], c["v"])
    op = P().PagedAttention(kv, c["n_q"], scale=c["scale"])
    before = o.clone()
    got = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"], out=o)
    P().stream_check()
    scale = c["scale"] if c["scale"] is not None else kv.head_dim ** -0.5
    want, tol = R.attention(c["q"], c["k"], c["v"], c["table"], c["q_start"].tolist(), c["kv_len"].tolist(), scale, before)
    within(got.reshape(want.shape), want, tol, what)
    assert (out[:, c["q"].shape[1]:] == 3).all()
    again = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
    assert torch.equal(again[int(c["q_start"][0]):int(c["q_start"][-1])], got[int(c["q_start"][0]):int(c["q_start"][-1])]), "same call, same bits"
    return got


# one token each: lengths around every tile and page edge, one key, no key
SINGLE = [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 127), (1, 128), (1, 129), (1, 515), (1, 0), (1, 1000)]
# chunks around the row tiles, with and without cached tokens, an empty sequence, rows without keys
CHUNK = [(1, 1), (2, 2), (5, 9), (64, 64), (63, 200), (0, 40), (65, 65), (127, 300), (129, 129), (1, 700), (257, 400), (7, 3), (300, 811)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", ["single", "chunk"])
@pytest.mark.parametrize("n_q,n_kv,hd,page,layout", [
    (16, 8, 128, 16, "head"), (8, 2, 64, 24, "token"), (4, 4, 128, 8, "both"), (6, 2, 64, 16, "head"), (16, 1, 128, 64, "token"),
    (2, 2, 64, 128, "head"), (5, 1, 128, 40, "head"), (32, 1, 64, 256, "both"), (4, 2, 128, 1, "head"), (8, 2, 64, 5, "token"),
    (40, 2, 128, 16, "head")])
def test_paged_attention(dtype, lens, n_q, n_kv, hd, page, layout):
    check_attn(attn_case(n_q * page, SINGLE if lens == "single" else CHUNK, n_q, n_kv, hd, page, dtype, layout))


@pytest.mark.parametrize("dtype,page,absent", [("f16", 16, 0.3), ("bf16", 24, 0.6), ("f16", 5, 0.4), ("f16", 64, 1.0)])
@pytest.mark.parametrize("lens", [SINGLE, CHUNK, [(3, 2000), (200, 1500), (1, 900)]])
def test_paged_attention_absent_pages(dtype, page, absent, lens):
    """Pages that were evicted are not looked at; rows with none left are zero."""
    check_attn(attn_case(11, lens, 8, 4, 128, page, dtype, "head", absent=absent))


@pytest.mark.parametrize("lens", [[(1, 20000)], [(1, 9001), (1, 3), (1, 4097)], [(4, 7000), (2, 130)], [(700, 4000), (1, 5)],
                                  [(1, 300)] * 33, [(512, 512), (512, 1024)]])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 32)])
def test_paged_attention_long_and_many(lens, hd, page):
    check_attn(attn_case(3, lens, 8, 4, hd, page, "f16", "head"))


# one sequence: its heads' keys are cut over clusters whose shape follows the page table's length
@pytest.mark.parametrize("new,keys", [(1, 0), (1, 1), (1, 16), (1, 17), (1, 130), (1, 515), (2, 1), (4, 4), (3, 2049), (1, 4095), (2, 4097), (1, 9000)])
@pytest.mark.parametrize("n_q,n_kv,hd,page,dtype,cols", [
    (16, 8, 128, 16, "f16", 0), (16, 8, 128, 16, "bf16", 300), (8, 2, 64, 24, "bf16", 0), (4, 1, 64, 64, "f16", 80), (32, 32, 128, 8, "f16", 1),
    (40, 40, 64, 16, "bf16", 300)])
def test_paged_attention_one_sequence(new, keys, n_q, n_kv, hd, page, dtype, cols):
    check_attn(attn_case(new + keys, [(new, keys)], n_q, n_kv, hd, page, dtype, "head", extra_cols=max(cols, 1 - keys)))


@pytest.mark.parametrize("cols", [1, 300])
@pytest.mark.parametrize("keys,absent", [(515, 0.5), (5000, 0.3), (5000, 1.0)])
def test_paged_attention_one_sequence_with_absent_pages(keys, absent, cols):
    check_attn(attn_case(21, [(2, keys)], 8, 4, 128, 16, "f16", "head", absent=absent, extra_cols=cols))


# few rows over lengths that are split within a CTA, over two and over many, next to short ones
@pytest.mark.parametrize("lens", [[(1, 515)] * 2, [(2, 2048)] * 4, [(1, 1), (1, 6000), (1, 17)], [(4, 33 * i) for i in range(1, 32)],
                                  [(1, 61 * i) for i in range(70)], [(8, 900), (1, 901), (5, 5)]])
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(16, 8, 128, 16), (8, 4, 64, 40)])
def test_paged_attention_small_batches(lens, n_q, n_kv, hd, page):
    check_attn(attn_case(5, lens, n_q, n_kv, hd, page, "bf16", "both"))


def test_paged_attention_short_tails_after_long_epilogues():
    """Tasks of one row tile (its partner's warps have nothing to do in them) next to tasks of two, several to a CTA."""
    lens = [(7 + i % 11, 600 + 131 * (i % 7)) for i in range(90)]
    c = attn_case(13, lens, 40, 2, 128, 16, "f16", "head")
    first = check_attn(c).clone()
    op = P().PagedAttention(P().PagedKV(c["k"], c["v"]), c["n_q"])
    for _ in range(20):
        assert torch.equal(op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"]), first)
    P().stream_check()


# chunks whose tiles end one short of, on and past the edges of 64 and 128 keys
@pytest.mark.parametrize("new,keys", [(17, 17), (64, 65), (127, 128), (128, 1024), (129, 191), (255, 4099), (513, 513), (1025, 1153)])
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(16, 8, 128, 16), (8, 2, 64, 64)])
def test_paged_attention_one_chunk(new, keys, n_q, n_kv, hd, page):
    check_attn(attn_case(new, [(new, keys)], n_q, n_kv, hd, page, "f16", "token"))


def test_paged_attention_padding_rows_and_scale():
    c = attn_case(9, [(3, 50), (9, 80)], 4, 2, 128, 16, "bf16", "head", gap=5, scale=0.25)
    got = check_attn(c)
    assert (got[:5] == 3).all() and (got[-5:] == 3).all(), "rows outside every sequence are left alone"


def test_paged_attention_peaked_and_rising_scores():
    """Score maxima that grow along the keys (every tile rescales), and one key that takes all the weight."""
    for n in (1, 40, 200):
        c = attn_case(21, [(n, 1500)], 4, 2, 128, 16, "f16", "head")
        j = torch.arange(1500, device="cuda")
        pg, at = c["table"][0].long()[j // 16], j % 16
        c["q"][:] = 0
        c["q"].view(n, 4, 128)[..., 0] = 8.0
        ramp = torch.zeros(1500, 128, device="cuda")
        ramp[:, 0] = j / 1500 * 40
        ramp[700, 0] = 60
        c["k"][pg, :, at] = ramp[:, None].half().expand(-1, 2, -1)
        check_attn(c, f"{n} rows")


@pytest.mark.parametrize("n", [5, 200])
def test_paged_attention_nonfinite_values_stay_in_their_rows(n):
    """A new token whose key and value overflowed reaches itself and later tokens, not earlier ones."""
    L = 333
    c = attn_case(31, [(n, L)], 4, 2, 128, 16, "f16", "head", poison=False)
    at = L - 3                                            # the token of row n - 3
    clean = check_attn(c).clone()
    pg = int(c["table"][0, at // 16])
    c["k"][pg, :, at % 16] = float("inf")
    c["v"][pg, :, at % 16] = float("nan")
    op = P().PagedAttention(P().PagedKV(c["k"], c["v"]), 4)
    got = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
    assert torch.equal(got[:n - 3], clean[:n - 3])
    assert torch.isnan(got[n - 3:]).all()


@pytest.mark.parametrize("n", [1, 200])
def test_paged_attention_low_scores_and_nan_keys(n):
    """Rows whose scores all lie far below zero keep their precision; a NaN key, wherever it is, shows in every row that sees it."""
    L = 700
    c = attn_case(81, [(n, L)], 4, 2, 128, 16, "f16", "head")
    j = torch.arange(L, device="cuda")
    pg, at = c["table"][0].long()[j // 16], j % 16
    c["q"].view(n, 4, 128)[..., 0] = 30.0
    keep = c["k"][pg, :, at].clone()
    for low in (-20.0, -60.0, -400.0):                      # scores near -53, -160, -1060
        k = keep.clone()
        k[..., 0] = low
        c["k"][pg, :, at] = k
        check_attn(c, f"low {low}")
    c["k"][pg, :, at] = keep
    op = P().PagedAttention(P().PagedKV(c["k"], c["v"]), 4)
    for key in list(range(8)) + [L - n, L - 1]:
        k = keep.clone()
        k[key] = float("nan")
        c["k"][pg, :, at] = k
        got = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
        sees = torch.arange(n, device="cuda") + L - n >= key
        assert torch.isnan(got[sees]).all() and torch.isfinite(got[~sees]).all(), key


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("first,rest", [(-7.9, -24.92), (-7.9, -22.6), (-5.9, -24.4), (-39.9, -56.92), (0.1, -16.92)])
@pytest.mark.parametrize("zero_first", [True, False])
def test_paged_attention_many_keys_far_below_the_first(dtype, first, rest, zero_first):
    """128 keys of 2^first, then 32000 of 2^rest, which together weigh a few
    thousandths of them: a sequence for every SM, all alike, so that one CTA
    has all keys of its rows.  With values of 0 for the first keys only the
    others' probabilities are seen, within the bound that holds everywhere.
    With values near 1 for all, the products of the others meet a sum 2^24 times
    their size, of which the tensor cores keep 2^-25: that much more a key."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n, G, hd, page, L = 16, 16, 64, 64, 128 + 32000
    dt, ln2 = DT[dtype], float(np.log(2))
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.zeros(L // page, 1, page, hd, device="cuda")
    k[..., 0] = rest * ln2
    k[:2, ..., 0] = first * ln2
    v = 1 + 0.01 * torch.randn(L // page, 1, page, hd, device="cuda", generator=g)
    if zero_first:
        v[:2] = 0
    k, v = k.to(dt), v.to(dt)
    q = torch.zeros(n, G, hd, device="cuda", dtype=dt)
    q[..., 0] = 8.0                                          # times 1 / 8: the score is the key's first element
    q = q.view(n, G * hd)
    table = torch.arange(L // page, dtype=torch.int32, device="cuda")[None]
    want, tol = R.attention(q, k, v, table, [0, n], [L], hd ** -0.5, q)
    if not zero_first:
        tol = tol + L * 2.0 ** -25 * want.abs()
    i32 = dict(dtype=torch.int32, device="cuda")
    got = P().PagedAttention(P().PagedKV(k, v), G)(q.repeat(sms, 1), table.repeat(sms, 1), torch.arange(sms + 1, **i32) * n,
                                                   torch.full((sms,), L, **i32), n)
    P().stream_check()
    got = got.view(sms, n, G, hd)
    assert torch.equal(got, got[:1].expand_as(got))
    within(got[0], want, tol, f"{first} {rest}")


def test_paged_attention_far_pages():
    """Element offsets beyond 32 bits: the last pages of a pool of 2^32 + elements."""
    page, n_kv, hd = 16, 8, 128
    pages = (1 << 32) // (page * n_kv * hd) + 40
    k = torch.zeros(pages, n_kv, page, hd, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    c = attn_case(41, [(1, 333), (30, 100)], 16, n_kv, hd, page, "f16", "head", poison=False)
    m = c["k"].shape[0]
    k[-m:], v[-m:] = c["k"], c["v"]
    near = check_attn(c).clone()
    c["k"], c["v"], c["table"] = k, v, torch.where(c["table"] >= 0, c["table"] + (pages - m), c["table"])
    got = P().PagedAttention(P().PagedKV(k, v), 16)(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
    P().stream_check()
    assert torch.equal(got, near)
    # and the writer of those pages
    table = P().rope_table(1e6, hd, 8)
    one = torch.ones(hd, device="cuda")
    slots = torch.tensor([pages * page - 1], dtype=torch.int64, device="cuda")
    qkv = torch.randn(1, 32 * hd, device="cuda").half()
    P().QKNormRope(P().PagedKV(k, v), 16, one, one, table)(qkv, torch.zeros(1, dtype=torch.int32, device="cuda"), slots)
    P().stream_check()
    assert torch.equal(v[-1, :, -1], qkv.view(32, hd)[24:])


def test_paged_attention_bad_tables_are_reported():
    from nnzap_b200._capi import NNZ_EDEVICE, NnzError
    for page in (16, 5):
        for lens in ([(1, 300), (1, 40)], [(70, 300), (30, 40)]):
            for what in ("page", "length", "rows", "new"):
                c = attn_case(51, lens, 4, 2, 128, page, "f16", "head", poison=False, extra_cols=0)
                kv = P().PagedKV(c["k"], c["v"])
                table, q_start, kv_len, max_new = c["table"], c["q_start"], c["kv_len"], c["max_new"]
                if what == "page":
                    table[0, 1] = kv.num_pages
                elif what == "length":
                    kv_len[0] = table.shape[1] * page + 7
                elif what == "rows":
                    q_start[-1] += 3
                    max_new += 3
                else:
                    max_new -= 1
                if max_new == 0:
                    continue
                out = torch.zeros_like(c["q"])
                P().PagedAttention(kv, 4)(c["q"], table, q_start, kv_len, max_new, out=out)
                with pytest.raises(NnzError) as e:
                    P().stream_check()
                assert e.value.code == NNZ_EDEVICE, what
                assert torch.isfinite(out).all()
                P().stream_check()


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what", ["empty sequence", "descending", "past the end", "negative length"])
def test_paged_attention_bad_sequences_without_rows_are_reported(page, new, what):
    """Ranges and lengths that no row of the output comes across, in every kernel."""
    from nnzap_b200._capi import NNZ_EDEVICE, NnzError
    c = attn_case(53, [(new, 300), (new, 200), (new, 100)], 4, 2, 128, page, "f16", "head", poison=False, extra_cols=0)
    q_start, kv_len = c["q_start"].tolist(), c["kv_len"].tolist()
    if what == "empty sequence":
        q_start, kv_len = [0, new, new, 2 * new], [300, c["table"].shape[1] * page + 1, 100]
    elif what == "descending":
        q_start = [0, new, 0, 2 * new]
    elif what == "past the end":
        q_start = [0, new, 3 * new, 4 * new]
    else:
        q_start, kv_len = [0, new, new, 2 * new], [300, -1, 100]
    out = torch.full_like(c["q"], 3.0)
    i32 = dict(dtype=torch.int32, device="cuda")
    P().PagedAttention(P().PagedKV(c["k"], c["v"]), 4)(c["q"], c["table"], torch.tensor(q_start, **i32), torch.tensor(kv_len, **i32), 2 * new, out=out)
    with pytest.raises(NnzError) as e:
        P().stream_check()
    assert e.value.code == NNZ_EDEVICE and torch.isfinite(out).all()
    P().stream_check()


def test_paged_ops_on_another_stream():
    """Calls go to torch's current stream: a long-running producer on it is waited for."""
    c = attn_case(61, [(40, 400), (1, 90)], 8, 4, 128, 16, "f16", "head")
    want = check_attn(c)
    op = P().PagedAttention(P().PagedKV(c["k"], c["v"]), 8)
    q = c["q"].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        big = torch.randn(4096, 4096, device="cuda")
        late = torch.zeros_like(q)
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(q)
        got = op(late, c["table"], c["q_start"], c["kv_len"], c["max_new"])
        lp = P().token_logprobs(got.float(), top_k=3)
    st.synchronize()
    a, b = int(c["q_start"][0]), int(c["q_start"][-1])
    assert torch.equal(got[a:b], want[a:b])
    assert torch.equal(lp.top_ids, P().token_logprobs(got.float(), top_k=3).top_ids)


def test_errors_raised_while_others_are_collected_are_kept():
    """Two streams raise an error of their own kind while a thread collects
    errors on a third: every one of them is reported."""
    import threading
    from nnzap_b200._capi import NnzError
    kv = P().PagedKV.empty(4, 2, 8, 128)
    one = torch.ones(128, device="cuda")
    op = P().QKNormRope(kv, 4, one, one, P().rope_table(1e4, 128, 64))
    qkv = torch.zeros(1, 8 * 128, dtype=torch.float16, device="cuda")
    i32, i64 = dict(dtype=torch.int32, device="cuda"), dict(dtype=torch.int64, device="cuda")
    position = (torch.tensor([64], **i32), torch.tensor([0], **i64))
    page = (torch.tensor([0], **i32), torch.tensor([32], **i64))
    outs = [torch.zeros(1, 4 * 128, dtype=torch.float16, device="cuda") for _ in range(2)]
    a, b, c = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    seen, checks, stop = set(), [0], threading.Event()

    def collect():
        with torch.cuda.stream(c):
            while not stop.is_set():
                try:
                    P().stream_check()
                except NnzError as e:
                    seen.update(w for w in ("position", "page") if w in str(e))
                checks[0] += 1
    t = threading.Thread(target=collect)
    t.start()
    lost = 0
    try:
        for _ in range(500):
            seen.clear()
            for st, bad, out in ((a, position, outs[0]), (b, page, outs[1])):
                with torch.cuda.stream(st):
                    op(qkv, *bad, out=out)
            a.synchronize()
            b.synchronize()
            done = checks[0] + 2                        # a check that began after this
            while checks[0] < done and t.is_alive():
                pass
            lost += seen != {"position", "page"}
    finally:
        stop.set()
        t.join()
    assert lost == 0


@pytest.mark.parametrize("lens", [[(1, 9000), (1, 3)], [(200, 4000)]])
def test_paged_attention_workspace_made_on_another_stream(lens):
    """An operator whose workspace is still to be zeroed, behind other work on
    the stream it was made on and in memory that held ones, called at once on
    two more streams: split tasks meet in the workspace."""
    c = attn_case(91, lens, 8, 4, 128, 16, "f16", "head")
    want = check_attn(c)
    kv = P().PagedKV(c["k"], c["v"])
    n = P().PagedAttention(kv, 8).workspace.buf.numel()
    made, used = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(made):
        torch.full((n,), 255, dtype=torch.uint8, device="cuda")       # the next block of this size and stream
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        op = P().PagedAttention(kv, 8)
    with torch.cuda.stream(used):
        first = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
    second = op(c["q"], c["table"], c["q_start"], c["kv_len"], c["max_new"])
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)
    P().stream_check()


def test_paged_ops_in_a_cuda_graph():
    """Lengths, tables and tokens are read on the device: one captured step serves every later one."""
    c = attn_case(71, [(1, 1), (1, 1), (1, 1)], 8, 4, 128, 16, "f16", "head", poison=False)
    k, v = (torch.randn(40, 4, 16, 128, device="cuda").half() for _ in range(2))
    table = torch.randperm(40, device="cuda")[:39].view(3, 13).to(torch.int32)
    kv_len = torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda")
    op = P().PagedAttention(P().PagedKV(k, v), 8)
    out = torch.zeros_like(c["q"])
    args = (c["q"], table, c["q_start"], kv_len, 1)
    op(*args, out=out)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        op(*args, out=out)
    for lens in ([1, 17, 200], [208, 64, 65]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        want, tol = R.attention(c["q"], k, v, table, [0, 1, 2, 3], lens, 128 ** -0.5, out)
        within(out.view(want.shape), want, tol, str(lens))


# ---- log probabilities -----------------------------------------------------------
def check_lp(x, tokens, k):
    r = P().token_logprobs(x, tokens, top_k=k)
    P().stream_check()
    got, ent, lse, ids, top = R.logprobs(x, tokens if tokens.dim() == 2 else tokens[:, None], k)
    # f32 sums: up to a few hundred terms one after the other (2^-24 each),
    # 2-ulp exponentials, x - M to 2^-24 of itself
    def near(a, b, what):
        same = (a.to(R.F) == b) | (torch.isnan(a) & torch.isnan(b))
        ok = same | ((a.to(R.F) - b).abs() <= 3e-5 + 1e-6 * b.abs())
        assert ok.all(), f"{what}: worst {float(torch.where(same, torch.zeros_like(b), (a.to(R.F) - b).abs()).max()):.2e}"
    near(r.logprob.view(got.shape), got, "logprob")
    near(r.entropy, ent, "entropy")
    near(r.logsumexp, lse, "logsumexp")
    if k:
        assert torch.equal(r.top_ids, ids)
        near(r.top_logprobs, top, "top")
    return r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,n,pad,k", [(1, 1, 0, 1), (2, 3, 1, 5), (1, 32, 0, 32), (3, 33, 2, 32), (5, 1000, 3, 20), (7, 4097, 1, 1),
                                           (2, 151936, 0, 20), (4, 151669, 267, 5), (1, 151669, 0, 32), (300, 5001, 7, 8), (3, 70000, 1, 0)])
def test_token_logprobs(dtype, rows, n, pad, k):
    g = torch.Generator(device="cuda").manual_seed(n)
    full = (torch.randn(rows, n + pad, device="cuda", generator=g) * 4).to(DT[dtype])
    full[:, n:] = float("nan")                      # padding is never looked at
    tok = torch.randint(0, n, (rows, 3), device="cuda", generator=g).to(torch.int32)
    tok[:, 1] = -1
    before = full.clone()
    check_lp(full[:, :n], tok, k)
    assert torch.equal(full[:, :n], before[:, :n])


@pytest.mark.parametrize("dtype,n", [("f32", 100001), ("f32", 151936), ("f32", 200001), ("bf16", 200003), ("f16", 420001)])
@pytest.mark.parametrize("k", [20, 32])
def test_token_logprobs_long_rows_of_many(dtype, n, k):
    """A row to a CTA, whose steps (4096 f32, 8192 16-bit elements) share the 24
    slots of step maxima by two or more: the best values lie in the first,
    second, third and last steps, several to a step."""
    rows, step = 150, 4096 if dtype == "f32" else 8192
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, device="cuda", generator=g)
    at = torch.tensor([step + 5, step + 900, 3 * step - 1, 2 * step, 7, step - 1, n - 1, n - n % step, 5 * step + 2], device="cuda")
    x[:, at] = 20 + torch.arange(len(at), device="cuda") % 4 * 0.5
    x[1::2] = x[1::2].roll(step, -1)
    tok = torch.randint(0, n, (rows,), device="cuda", generator=g).to(torch.int32)
    check_lp(x.to(DT[dtype]), tok, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "ties", "zeros", "masked", "few", "huge", "tail", "lowest"])
def test_token_logprobs_orders_and_masks(dtype, kind):
    n, rows = 20011, 3
    i = torch.arange(n, device="cuda", dtype=torch.float32)
    x = {"equal": torch.full((n,), -2.5, device="cuda"), "rising": i / 100, "falling": -i / 100, "ties": torch.floor((i * 37) % 50) / 7,
         "zeros": torch.where(i % 3 == 0, -torch.zeros_like(i), torch.zeros_like(i)), "masked": torch.where(i % 7 == 3, i * 0 + 1, -torch.inf * torch.ones_like(i)),
         "few": torch.full((n,), -torch.inf, device="cuda"), "huge": (i % 91) * 1e36, "tail": torch.where(i >= n - 3, i, i * 0 - 50),
         "lowest": torch.where(i % 5 > 0, torch.full_like(i, torch.finfo(DT[dtype]).min), (i % 11) / 3)}[kind].clone()
    if kind == "few":
        x[[5, 9000, n - 1]] = torch.tensor([1.0, 2.0, 1.0], device="cuda")
    xx = x.to(DT[dtype]).repeat(rows, 1)
    if kind == "few":
        xx[1] = -torch.inf                            # nothing is allowed
    tok = torch.tensor([[0, n - 1, 9000]] * rows, dtype=torch.int32, device="cuda")
    r = check_lp(xx, tok, 32)
    if kind == "few":
        assert (r.top_ids[1] == -1).all() and r.entropy[1] == 0 and (r.logprob[1] == -torch.inf).all()


def test_token_logprobs_nonfinite_and_bad_tokens():
    from nnzap_b200._capi import NNZ_EDEVICE, NnzError
    x = torch.randn(4, 5000, device="cuda")
    x[1, 77], x[2, 4999] = float("nan"), float("inf")
    tok = torch.tensor([3, 3, 3, 4999], dtype=torch.int32, device="cuda")
    r = P().token_logprobs(x, tok, top_k=4)
    P().stream_check()
    assert torch.isfinite(r.logprob[[0, 3]]).all() and torch.isnan(r.logprob[[1, 2]]).all() and torch.isnan(r.entropy[[1, 2]]).all()
    assert torch.equal(r.top_ids[1], R.logprobs(x[1:2], tok[1:2, None], 4)[3][0]) and int(r.top_ids[2, 0]) == 4999
    tok[0] = 5000
    r = P().token_logprobs(x, tok)
    with pytest.raises(NnzError) as e:
        P().stream_check()
    assert e.value.code == NNZ_EDEVICE and torch.isnan(r.logprob[0]) and torch.isfinite(r.logprob[3])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("off", [1, 2, 3, 5])
def test_token_logprobs_unaligned_rows(dtype, off):
    buf = torch.randn(9 * 1237 + 16, device="cuda").to(DT[dtype])
    x = buf[off:off + 9 * 1237].view(9, 1237)
    check_lp(x, torch.arange(9, device="cuda", dtype=torch.int32), 7)


def test_empty_calls():
    kv = P().PagedKV.empty(2, 2, 8, 64)
    z = torch.zeros(0, 128, dtype=torch.float16, device="cuda")
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert P().PagedAttention(kv, 2)(z, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), i32, 0).shape == (0, 128)
    table = P().rope_table(1e4, 64, 4)
    one = torch.ones(64, device="cuda")
    assert P().QKNormRope(kv, 2, one, one, table)(torch.zeros(0, 384, dtype=torch.float16, device="cuda"), i32, i32.long()).shape == (0, 128)
    r = P().token_logprobs(torch.zeros(0, 10, device="cuda"), i32, top_k=2)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 2)
    P().stream_check()
