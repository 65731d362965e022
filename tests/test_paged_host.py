"""CPU tests of the host side of nnzap_b200.paged: the library's functions are
replaced by stubs that look at what they are given."""
import ctypes as C
import threading

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _lib(built_lib):
    yield


class Stream:
    """A stream that notes what it waits for."""
    def __init__(self, handle, log):
        self.cuda_stream, self.log = handle, log

    def wait_stream(self, other):
        self.log.append(("wait", self.cuda_stream, other.cuda_stream))


class Devices:
    """Two devices that are not there: which one is current."""
    current = 0

    def guard(self, device):
        class Guard:
            def __enter__(g):
                g.back, want = self.current, torch.device(device) if isinstance(device, str) else device
                want = getattr(want, "index", want)
                self.current = g.back if want is None else want

            def __exit__(g, *exc):
                self.current = g.back
        return Guard()


@pytest.fixture
def devices(monkeypatch):
    from nnzap_b200 import paged
    d = Devices()
    # (raising=False: also where the module does not look at the device)
    monkeypatch.setattr(paged, "_current_device", lambda: d.current, raising=False)
    monkeypatch.setattr(paged, "_device", d.guard, raising=False)
    monkeypatch.setattr(paged, "_stream", lambda device=None: 100 + (d.current if device is None else device))
    monkeypatch.setattr(paged, "_current_stream", lambda device=None: Stream(100 + d.current, []), raising=False)
    monkeypatch.setattr(paged, "_capturing", lambda: False, raising=False)
    return d


@pytest.fixture
def paged(devices):
    from nnzap_b200 import paged
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


# ---- devices ---------------------------------------------------------------------
def test_operators_run_on_the_device_of_their_tensors(paged, devices):
    """Called while another device is current, an operator launches on its
    tensors' device and that device's stream, and leaves the current one as it was."""
    devices.current = 1
    for op, inputs in ((norm_rope(paged), norm_rope_inputs), (paged.PagedAttention(host_kv(paged), 4), attn_inputs)):
        seen = []
        op._fn = lambda kv, ref, stream: seen.append((devices.current, stream)) or 0
        op(*inputs(3))
        assert seen == [(0, 100)] and devices.current == 1


class Lib:
    """The library's functions, which note the current device and their last argument."""
    def __init__(self, devices, result=0):
        self.devices, self.result, self.calls = devices, result, []

    def __getattr__(self, name):
        def f(*args):
            self.calls.append((name, self.devices.current, args[-1]))
            return self.result
        return f


def test_workspace_is_sized_on_the_pools_device(paged, devices, monkeypatch):
    devices.current, lib = 1, Lib(devices, 512)
    monkeypatch.setattr(paged, "lib", lambda: lib)
    paged.PagedAttention(host_kv(paged), 4)
    assert [c[:2] for c in lib.calls if c[0] == "nnz_paged_attn_workspace"] == [("nnz_paged_attn_workspace", 0)]


def test_rope_table_and_checks_follow_the_device_argument(paged, devices, monkeypatch):
    lib, empty = Lib(devices), torch.empty

    class OnOne(torch.Tensor):
        device = torch.device("cuda", 1)
    monkeypatch.setattr(paged, "lib", lambda: lib)
    monkeypatch.setattr(paged.torch, "empty", lambda *shape, dtype, device: empty(*shape, dtype=dtype).as_subclass(OnOne))
    paged.rope_table(1e4, 64, 8, device="cuda:1")
    paged.stream_check("cuda:1")
    paged.stream_check()
    assert lib.calls == [("nnz_rope_table", 1, 101), ("nnz_stream_check", 1, 101), ("nnz_stream_check", 0, 100)]
    assert devices.current == 0


def test_token_logprobs_on_another_device(paged, devices, monkeypatch):
    lib, empty = Lib(devices), torch.empty

    class OnOne(torch.Tensor):
        device, is_cuda = torch.device("cuda", 1), True
    monkeypatch.setattr(paged, "lib", lambda: lib)
    monkeypatch.setattr(paged.torch, "empty", lambda *shape, dtype, device: empty(*shape, dtype=dtype))
    paged.token_logprobs(torch.zeros(2, 8).as_subclass(OnOne), top_k=2)
    assert lib.calls == [("nnz_token_logprobs", 1, 101)] and devices.current == 0


def test_a_models_step_runs_on_its_device(paged, devices):
    from nnzap_b200.score import PagedModel
    seen = []

    class Weights:
        M = 10

        def rows(self, ids):
            seen.append(devices.current)
            return torch.zeros(len(ids), 4)

        def gemm(self, x, out=None, dtype=None):
            seen.append(devices.current)
            return out
    m = object.__new__(PagedModel)
    m.device, m.layers, m.embed, m.lm_head, m.final_norm = torch.device("cuda", 1), [], Weights(), Weights(), torch.ones(4)
    m.config = type("Config", (), {"eps": 1e-6})
    m.step(torch.zeros(3, dtype=torch.int32), None, None, None, None, None, 1)
    assert seen == [1, 1] and devices.current == 0


# ---- streams ---------------------------------------------------------------------
def test_a_workspace_follows_its_calls_from_stream_to_stream(paged, monkeypatch):
    """Zeroed on stream 1, used on 2, 2, 3 and 3 (in a graph's capture on 4
    between them): a stream that is not the last use's waits for it, before the
    launch, and the memory is marked as used there."""
    log, zeros, now = [], torch.zeros, [1]

    class Buffer(torch.Tensor):
        def record_stream(self, stream):
            log.append(("record", stream.cuda_stream))
    monkeypatch.setattr(paged.torch, "zeros", lambda *a, **k: zeros(*a, **k).as_subclass(Buffer))
    monkeypatch.setattr(paged, "_stream", lambda device=None: now[0])
    monkeypatch.setattr(paged, "_current_stream", lambda device=None: Stream(now[0], log), raising=False)
    monkeypatch.setattr(paged, "_capturing", lambda: now[0] == 4, raising=False)
    op = paged.PagedAttention(host_kv(paged), 4)
    op._fn = lambda kv, ref, stream: log.append(("launch", stream)) or 0
    for now[0] in (2, 2, 4, 3, 3):
        op(*attn_inputs(3))
    assert log == [("wait", 2, 1), ("record", 2), ("launch", 2), ("launch", 2), ("launch", 4),
                   ("wait", 3, 2), ("record", 3), ("launch", 3), ("launch", 3)]


def test_operators_share_a_workspace(paged):
    """One after the other, from two threads too; a workspace that is too small or elsewhere is refused."""
    first = paged.PagedAttention(host_kv(paged, hd=128), 4)
    second = paged.PagedAttention(host_kv(paged), 4, workspace=first.workspace)
    inside, overlap, where = [], [], []

    def stub(kv, ref, stream):
        overlap.append(len(inside))
        inside.append(1)
        where.append(struct_of(ref).workspace)
        threading.Event().wait(0.05)
        inside.pop()
        return 0
    first._fn = second._fn = stub
    hd128 = (torch.zeros(3, 4 * 128, dtype=torch.float16), *attn_inputs(3)[1:])
    t = [threading.Thread(target=lambda: first(*hd128)), threading.Thread(target=lambda: second(*attn_inputs(3)))]
    for i in t:
        i.start()
    for i in t:
        i.join(20)
    assert overlap == [0, 0] and where == [first.workspace.buf.data_ptr()] * 2
    small = paged.PagedAttention(host_kv(paged), 4).workspace
    with pytest.raises(ValueError):
        paged.PagedAttention(host_kv(paged, hd=128), 4, workspace=small)
    small.buf = torch.empty(first.workspace.buf.numel(), dtype=torch.uint8, device="meta")
    with pytest.raises(ValueError):
        paged.PagedAttention(host_kv(paged), 4, workspace=small)


# ---- numbers -----------------------------------------------------------------------
@pytest.mark.parametrize("scale", [0.0, 1e-60, -1.0, 1e60, float("inf"), float("nan")])
def test_scales_that_are_none(paged, scale):
    """0 would be taken for the default, an infinite one makes every row NaN."""
    with pytest.raises(ValueError):
        paged.PagedAttention(host_kv(paged), 4, scale=scale)


@pytest.mark.parametrize("max_new", [-1, 1 << 31, 1 << 32])
def test_counts_that_do_not_fit(paged, max_new):
    op = paged.PagedAttention(host_kv(paged), 4)
    op._fn = lambda *a: pytest.fail("called")
    with pytest.raises(ValueError):
        op(*attn_inputs(3)[:4], max_new)


def test_the_library_refuses_an_infinite_scale():
    from nnzap_b200 import _capi as capi
    kv = capi.NnzPagedKv(k=0x1000, v=0x2000, dtype=capi.NNZ_DT_F16, num_pages=4, page_size=16, num_kv_heads=2, head_dim=128,
                         page_stride=4096, head_stride=2048, token_stride=128)
    a = capi.NnzPagedAttnArgs(q=0x1000, q_stride=512, tokens=3, num_query_heads=4, num_seqs=1, max_new=3, q_start=0x1000, kv_len=0x1000,
                              page_table=0x1000, table_stride=4, scale=float("inf"), out=0x1000, out_stride=512, workspace=0x1000,
                              workspace_bytes=1 << 30)
    assert capi.lib().nnz_paged_attn(C.byref(kv), C.byref(a), None) == capi.NNZ_EINVAL
