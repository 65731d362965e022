"""CPU tests of what the library's host code keeps for each device: its objects
linked with a pretended CUDA runtime of two devices (fake_cudart.cpp)."""
import ctypes as C
import subprocess
from collections import namedtuple
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
Launch = namedtuple("Launch", "device grid cluster smem")


@pytest.fixture
def runtime(built_lib, tmp_path):
    """make(sources): a fresh copy of those objects over the pretended runtime."""
    from nnzap_b200 import build

    def make(*names):
        so = tmp_path / f"fake_{len(list(tmp_path.iterdir()))}.so"
        cuda = Path(build._nvcc()).resolve().parent.parent / "include"
        subprocess.run(["g++", "-O1", "-std=c++20", "-shared", "-fPIC", "-w", "-I", str(cuda), str(HERE / "fake_cudart.cpp"),
                        *[str(build.BUILD / f"{n}.cu.o") for n in names], "-Wl,-Bsymbolic", "-Wl,-z,defs", "-lm", "-o", str(so)], check=True)
        lib = C.CDLL(str(so))
        lib.fake_message.restype = C.c_char_p

        def launches():
            out = []
            for i in range(lib.fake_launches()):
                v = (C.c_uint * 4)()
                lib.fake_launch(i, v)
                out.append(Launch(*v))
            return out
        lib.launches = launches
        return lib
    return make


def logprobs(lib):
    from nnzap_b200 import _capi as capi
    a = capi.NnzLogprobsArgs(logits=0x1000, dtype=capi.NNZ_DT_F32, rows=1, n=151936, stride=151936, top_k=4, entropy=0x1000,
                             top_ids=0x1000, top_logprobs=0x1000)
    return lib.nnz_token_logprobs(C.byref(a), None)


def attention(lib, workspace=1 << 30, new=1, keys=32768):
    from nnzap_b200 import _capi as capi
    kv = capi.NnzPagedKv(k=0x1000, v=0x2000, dtype=capi.NNZ_DT_F16, num_pages=4, page_size=16, num_kv_heads=8, head_dim=128,
                         page_stride=16384, head_stride=2048, token_stride=128)
    a = capi.NnzPagedAttnArgs(q=0x1000, q_stride=2048, tokens=new, num_query_heads=16, num_seqs=1, max_new=new, q_start=0x1000, kv_len=0x1000,
                              page_table=0x1000, table_stride=keys // 16, out=0x1000, out_stride=2048, workspace=0x1000, workspace_bytes=workspace)
    return lib.nnz_paged_attn(C.byref(kv), C.byref(a), None)


def test_wide_clusters_are_allowed_on_every_device(runtime):
    lib = runtime("logprobs")
    for dev in (0, 1, 0):
        lib.fake_use(dev)
        assert logprobs(lib) == 0, lib.fake_message()
    assert [(x.device, x.cluster) for x in lib.launches()] == [(0, 16), (1, 16), (0, 16)]


def test_log_probabilities_without_wide_clusters(runtime):
    """A device that takes no cluster of 16 gets 8 CTAs a row; the other one its 16."""
    lib = runtime("logprobs")
    lib.fake_device(1, 148, 148, 0)
    for dev in (1, 0, 1):
        lib.fake_use(dev)
        assert logprobs(lib) == 0, lib.fake_message()
    assert [(x.device, x.cluster) for x in lib.launches()] == [(1, 8), (0, 16), (1, 8)]


def test_one_sequence_over_the_clusters_of_each_device(runtime):
    """Clusters of 4 CTAs, as many of each of the 8 heads as run at once: 4 on
    one device, 1 on the other."""
    lib = runtime("paged", "paged_stream", "paged_umma")
    lib.fake_device(1, 40, 39, 1)
    for dev in (0, 1, 0):
        lib.fake_use(dev)
        assert attention(lib) == 0, lib.fake_message()
    assert [(x.device, x.grid, x.cluster) for x in lib.launches()] == [(0, 128, 4), (1, 32, 4), (0, 128, 4)]


def test_chunks_on_every_device(runtime):
    lib = runtime("paged", "paged_stream", "paged_umma")
    for dev in (0, 1, 0):
        lib.fake_use(dev)
        assert attention(lib, new=64) == 0, lib.fake_message()
    assert [x.device for x in lib.launches() if x.smem] == [0, 1, 0]


def test_quantized_gemms_on_every_device(runtime):
    class Args(C.Structure):
        _fields_ = [("M", C.c_uint32), ("K", C.c_uint32), ("N", C.c_uint32), ("fmt", C.c_int), ("gs", C.c_int), ("bf16s", C.c_int),
                    ("bf16r", C.c_int), *[(n, C.c_void_p) for n in ("w", "s", "b", "w2", "s2", "b2")], ("epi", C.c_int), ("acc", C.c_void_p),
                    ("acc_floats", C.c_size_t), ("out", C.c_void_p), ("ldo", C.c_uint32), ("err", C.c_void_p), ("prof", C.c_int), ("pdl", C.c_int)]
    lib = runtime("gemm")
    a = Args(M=64, K=256, N=512, gs=128, w=0x1000, s=0x1000, out=0x1000, ldo=512)
    launch = lib._ZN3nnz11gemm_launchERKNS_8GemmArgsEPK6__halfP11CUstream_st
    for dev in (0, 1, 0):
        lib.fake_use(dev)
        assert launch(C.byref(a), C.c_void_p(0x1000), None) == 0
    assert [x.device for x in lib.launches()] == [0, 1, 0]
