"""CPU tests of what the ragged-serving entry points refuse (before any device call)."""
import ctypes as C

import pytest


def capi():
    from nnzap_b200 import _capi
    return _capi


@pytest.fixture(autouse=True)
def _lib(built_lib):
    yield


def pool(**kw):
    k = capi().NnzPagedKv(k=0x1000, v=0x2000, dtype=capi().NNZ_DT_F16, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128,
                          page_stride=4096, head_stride=2048, token_stride=128)
    for n, v in kw.items():
        setattr(k, n, v)
    return k


def norm_args(**kw):
    a = capi().NnzNormRopeArgs(qkv=0x1000, qkv_stride=1024, tokens=3, num_query_heads=4, q_norm=0x1000, k_norm=0x1000, eps=1e-6,
                               rope_style=0, rope_table=0x1000, table_positions=8, positions=0x1000, slots=0x1000, q_out=0x1000, q_stride=512)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def attn_args(**kw):
    a = capi().NnzPagedAttnArgs(q=0x1000, q_stride=512, tokens=3, num_query_heads=4, num_seqs=1, max_new=3, q_start=0x1000, kv_len=0x1000,
                                page_table=0x1000, table_stride=4, scale=0.0, out=0x1000, out_stride=512, workspace=0x1000,
                                workspace_bytes=1 << 30)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def lp_args(**kw):
    a = capi().NnzLogprobsArgs(logits=0x1000, dtype=capi().NNZ_DT_F32, rows=2, n=100, stride=100, tokens=0x1000, num_tokens=1, top_k=4,
                               logprob=0x1000, entropy=0x1000, logsumexp=0x1000, top_ids=0x1000, top_logprobs=0x1000)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD_POOL = [dict(k=None), dict(v=None), dict(dtype=4), dict(dtype=0), dict(head_dim=96), dict(num_kv_heads=0), dict(num_pages=0),
            dict(page_size=0), dict(page_size=65537), dict(page_stride=4097), dict(head_stride=2044), dict(token_stride=120),
            dict(token_stride=-128), dict(page_stride=0), dict(head_stride=0), dict(k=0x1008), dict(v=0x2002)]


@pytest.mark.parametrize("bad", BAD_POOL)
def test_pool_refusals(bad):
    c, L = capi(), capi().lib()
    k = pool(**bad)
    assert L.nnz_qk_norm_rope_paged(C.byref(k), C.byref(norm_args()), None) == c.NNZ_EINVAL
    assert L.nnz_paged_attn(C.byref(k), C.byref(attn_args()), None) == c.NNZ_EINVAL
    assert L.nnz_last_error().startswith(b"paged kv")
    assert L.nnz_paged_attn_workspace(C.byref(k), 4) == 0


@pytest.mark.parametrize("bad", [dict(qkv=None), dict(q_norm=None), dict(k_norm=None), dict(rope_table=None), dict(positions=None),
                                 dict(slots=None), dict(q_out=None), dict(qkv_stride=1016), dict(qkv_stride=1028), dict(q_stride=504),
                                 dict(q_stride=516), dict(num_query_heads=0), dict(table_positions=0), dict(rope_style=2),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(qkv=0x1002), dict(q_out=0x1008), dict(q_norm=0x1004),
                                 dict(rope_table=0x1004)])
def test_norm_rope_refusals(bad):
    L = capi().lib()
    assert L.nnz_qk_norm_rope_paged(C.byref(pool()), C.byref(norm_args(**bad)), None) == capi().NNZ_EINVAL
    assert L.nnz_qk_norm_rope_paged(C.byref(pool()), None, None) == capi().NNZ_EINVAL
    assert L.nnz_qk_norm_rope_paged(None, C.byref(norm_args()), None) == capi().NNZ_EINVAL


@pytest.mark.parametrize("bad", [dict(q=None), dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(out=None),
                                 dict(workspace=None), dict(workspace=0x1010), dict(workspace_bytes=8), dict(q_stride=504),
                                 dict(q_stride=516), dict(out_stride=504), dict(num_query_heads=0), dict(num_query_heads=3),
                                 dict(num_query_heads=130), dict(table_stride=0), dict(table_stride=1 << 28), dict(scale=-1.0),
                                 dict(scale=float("nan")), dict(q=0x1004), dict(out=0x1008)])
def test_paged_attn_refusals(bad):
    L = capi().lib()
    assert L.nnz_paged_attn(C.byref(pool()), C.byref(attn_args(**bad)), None) == capi().NNZ_EINVAL
    assert L.nnz_paged_attn(C.byref(pool()), None, None) == capi().NNZ_EINVAL


@pytest.mark.parametrize("bad", [dict(logits=None), dict(logits=0x1002), dict(dtype=0), dict(dtype=7), dict(n=0), dict(stride=99),
                                 dict(top_k=33), dict(top_ids=None), dict(top_logprobs=None), dict(logprob=None), dict(tokens=None)])
def test_logprobs_refusals(bad):
    L = capi().lib()
    assert L.nnz_token_logprobs(C.byref(lp_args(**bad)), None) == capi().NNZ_EINVAL
    assert L.nnz_token_logprobs(None, None) == capi().NNZ_EINVAL


def test_nothing_to_do_is_no_error():
    L = capi().lib()
    assert L.nnz_qk_norm_rope_paged(C.byref(pool()), C.byref(norm_args(tokens=0)), None) == 0
    for none in (dict(tokens=0), dict(num_seqs=0), dict(max_new=0)):
        assert L.nnz_paged_attn(C.byref(pool()), C.byref(attn_args(**none)), None) == 0
    assert L.nnz_token_logprobs(C.byref(lp_args(rows=0)), None) == 0


@pytest.mark.parametrize("theta,hd,n,ptr", [(0.0, 128, 4, 0x1000), (float("nan"), 128, 4, 0x1000), (1e4, 0, 4, 0x1000), (1e4, 63, 4, 0x1000),
                                            (1e4, 64, 0, 0x1000), (1e4, 64, 4, None), (1e4, 64, 4, 0x1004)])
def test_rope_table_refusals(theta, hd, n, ptr):
    assert capi().lib().nnz_rope_table(theta, hd, n, ptr, None) == capi().NNZ_EINVAL


def test_workspace_needs_whole_groups():
    L = capi().lib()
    assert L.nnz_paged_attn_workspace(C.byref(pool()), 4) > 0
    assert L.nnz_paged_attn_workspace(C.byref(pool()), 3) == 0 and L.nnz_paged_attn_workspace(C.byref(pool()), 0) == 0


def test_python_argument_checks():
    torch = pytest.importorskip("torch")
    from nnzap_b200 import paged
    k = torch.zeros(2, 2, 8, 64, dtype=torch.float16)
    for a, b in [(k, k), (k, k[:1]), (k.float(), k.float()), (k[0], k[0]), (k, k.transpose(1, 2).contiguous().transpose(1, 2))]:
        with pytest.raises(ValueError):
            paged.PagedKV(a, b)                 # host tensors, unequal shapes, strides or types
    for bad in [torch.zeros(3, 4), torch.zeros(4), torch.zeros(3, 4, dtype=torch.int32)]:
        with pytest.raises(ValueError):
            paged.token_logprobs(bad)
    with pytest.raises(ValueError):
        paged.rope_table(1e4, 64, 0)
