"""CPU tests of the host side of nnzap_b200.paged: the library's functions are
replaced by stubs that look at what they are given."""
import ctypes as C
import threading

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _lib(built_lib):
    yield


@pytest.fixture
def paged(monkeypatch):
    from nnzap_b200 import paged
    monkeypatch.setattr(paged, "_stream", lambda device=None: 0)
    return paged


def host_kv(paged, n_kv=2, page=16, hd=64, pages=4):
    """A page pool in host memory, which the constructor does not take."""
    from nnzap_b200 import _capi as capi
    kv = object.__new__(paged.PagedKV)
    kv.k, kv.v = torch.zeros(pages, n_kv, page, hd, dtype=torch.float16), torch.zeros(pages, n_kv, page, hd, dtype=torch.float16)
    kv.dtype, kv.device, kv.index = torch.float16, torch.device("cpu"), 0
    kv.num_pages, kv.num_kv_heads, kv.page_size, kv.head_dim = kv.k.shape
    kv.c = capi.NnzPagedKv(k=0x1000, v=0x2000, dtype=capi.NNZ_DT_F16, num_pages=pages, page_size=page, num_kv_heads=n_kv, head_dim=hd,
                           page_stride=n_kv * page * hd, head_stride=page * hd, token_stride=hd)
    kv._ref = C.byref(kv.c)
    return kv


def norm_rope(paged):
    one = torch.ones(64)
    return paged.QKNormRope(host_kv(paged), 4, one, one, torch.zeros(8, 32, 2))


def norm_rope_inputs(n):
    return torch.zeros(n, 8 * 64, dtype=torch.float16), torch.zeros(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int64)


def attn_inputs(n):
    return (torch.zeros(n, 4 * 64, dtype=torch.float16), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
            torch.zeros(1, dtype=torch.int32), n)


def struct_of(ref):
    return ref._obj


# ---- threads ---------------------------------------------------------------------
@pytest.mark.parametrize("which", ["norm_rope", "attention"])
def test_two_threads_share_an_operator(paged, which):
    """While one thread's call is inside the library, which runs without the
    GIL, another thread calls the same object: each call's arguments stay its
    own, and calls that use one workspace do not overlap."""
    from nnzap_b200 import _capi as capi
    if which == "norm_rope":
        op, inputs, src, T = norm_rope(paged), norm_rope_inputs, "qkv", capi.NnzNormRopeArgs
    else:
        op, inputs, src, T = paged.PagedAttention(host_kv(paged), 4), attn_inputs, "q", capi.NnzPagedAttnArgs
    first_in, second_in = threading.Event(), threading.Event()
    seen, inside, overlap = {}, [], []

    def stub(kv, ref, stream):
        a = struct_of(ref)
        assert isinstance(a, T)
        me = threading.current_thread().name
        overlap.append(len(inside))
        inside.append(me)
        if me == "first":
            first_in.set()
            second_in.wait(0.5)
        else:
            second_in.set()
        seen[me] = (getattr(a, src), a.tokens)
        inside.remove(me)
        return 0
    op._fn = stub
    x = {"first": inputs(3), "second": inputs(5)}

    def second():
        first_in.wait(5)
        op(*x["second"])
    t = [threading.Thread(target=lambda: op(*x["first"]), name="first"), threading.Thread(target=second, name="second")]
    for i in t:
        i.start()
    for i in t:
        i.join(20)
    assert seen == {n: (v[0].data_ptr(), len(v[0])) for n, v in x.items()}
    if which == "attention":
        assert max(overlap) == 0
