"""The paged 4-bit cache's and the packed prompt attention's entry points on a host without a GPU:
argument errors come back before anything is launched, CPU tensors are refused."""
import ctypes
import pathlib
import re

import pytest
import torch

from halftone_quantizedkvcache_b200 import _lib, kernels

HEADER = pathlib.Path(__file__).parents[1] / "include" / "halftone_b200.h"
S2, C2, SC2 = (512, 128), (16 * 64 * 2, 16 * 64), (16 * 4 * 2, 16 * 4)


def struct_of(name):
    """The C struct of an entry's arguments, as the header declares it."""
    body = re.search(r"typedef struct %s_args \{(.*?)\}" % name, HEADER.read_text(), re.S).group(1)
    kinds = {"int": ctypes.c_int, "float": ctypes.c_float, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t,
             "hq_stream_t": ctypes.c_void_p}
    fields = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        kind = kinds.get(line.removeprefix("const ").split()[0])
        for part in line.split(","):
            field, two = re.search(r"(\w+)(\[2\])?$", part.strip()).groups()
            f = ctypes.c_void_p if "*" in part else kind
            fields.append((field, f * 2 if two else f))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


def call(name, base, **at):
    s = struct_of(name)()
    names = [f for f, _ in s._fields_ if f != "pad"]
    assert set(base) == set(names) and set(at) <= set(names)
    for k, v in {**base, **at}.items():
        setattr(s, k, type(getattr(s, k))(*v) if isinstance(v, tuple) else v)
    return getattr(_lib.lib(), name)(bytes(s))


def refused(name, base, cases):
    for code, at in cases:
        assert call(name, base, **at) == code, at


@pytest.mark.parametrize("name,plan", [("hq_paged4_append", "q_strides"), ("hq_paged4_decode", "code_strides"),
                                       ("hq_paged4_gather", "code_strides"), ("hq_packed_prefill", "workspace_bytes")])
def test_argument_structs_are_the_headers(name, plan):
    s, (head, tail) = struct_of(name), _lib.ARGS[name]
    assert getattr(s, plan).offset == head.size and ctypes.sizeof(s) == head.size + tail.size
    assert getattr(_lib.lib(), name)(None) == -1


def test_append_argument_errors():
    base = dict(q=256, k_new=256, v_new=256, x_dtype=1, q_strides=S2, k_strides=S2, v_strides=S2, T=3, B=2, Hq=4, Hkv=2, D=128,
                cu_seqlens=256, lens=256, pos_offset=None, q_weight=None, k_weight=None, w_dtype=1, eps=1e-6, inv_freq=256,
                rotary_dim=128, interleaved=0, factor=1.0, k_codes=256, v_codes=256, code_strides=C2, k_scale=256,
                v_scale=256, scale_strides=SC2, n_pages=5, page_size=16, tables=256, table_stride=4, max_pages=4, q_out=256,
                qo_strides=S2, k_out=None, ko_strides=S2, copy_rest=0, status=None, stream=None)
    refused("hq_paged4_append", base, [
        (-1, dict(q=None)), (-1, dict(k_new=None)), (-1, dict(v_new=None)), (-1, dict(lens=None)), (-1, dict(q_out=None)),
        (-1, dict(T=-1)), (-1, dict(B=-1)), (-1, dict(Hq=0)), (-1, dict(Hkv=0)), (-1, dict(cu_seqlens=None)),
        (-1, dict(inv_freq=None)), (-1, dict(rotary_dim=144)), (-1, dict(eps=-1.0)), (-1, dict(eps=float("nan"))),
        (-1, dict(q=264)), (-1, dict(q_strides=(512, 100))), (-1, dict(qo_strides=(0, 128))),
        (-1, dict(k_codes=None)), (-1, dict(k_codes=264)), (-1, dict(code_strides=(100, 1024))),
        (-1, dict(code_strides=(1024, 512))), (-1, dict(scale_strides=(32, 64))), (-1, dict(tables=None)),
        (-1, dict(k_out=256)),                             # k_out is k_new
        (-2, dict(x_dtype=0)), (-2, dict(D=64, rotary_dim=64)), (-2, dict(rotary_dim=24)), (-2, dict(w_dtype=2)),
        (-2, dict(page_size=48)), (-2, dict(page_size=8)), (-2, dict(page_size=512)), (-2, dict(max_pages=1 << 28)),
        (-2, dict(code_strides=(1 << 31, 1024))),
    ])
    assert call("hq_paged4_append", base, T=0) == 0


def test_decode_argument_errors():
    L = _lib.lib()
    nb = L.hq_paged4_decode_workspace_bytes(2, 4, 2, 16, 128, 128)
    assert nb > 1 == L.hq_paged4_decode_workspace_bytes(2, 4, 2, 16, 64, 128)   # 1024 tokens: none is needed
    base = dict(q=256, q_dtype=1, q_strides=S2, k_codes=256, v_codes=256, code_strides=C2, k_scale=256, v_scale=256,
                scale_strides=SC2, n_pages=5, page_size=16, tables=256, table_stride=128, max_pages=128, lens=256, B=2, Hq=4,
                Hkv=2, D=128, sm_scale=0.1, out=256, out_strides=S2, workspace=256, workspace_bytes=nb, status=None, stream=None)
    refused("hq_paged4_decode", base, [
        (-1, dict(q=None)), (-1, dict(lens=None)), (-1, dict(out=None)), (-1, dict(q=264)), (-1, dict(B=-1)),
        (-1, dict(Hq=0)), (-1, dict(q_strides=(512, 4))), (-1, dict(out_strides=(0, 128))),
        (-1, dict(out_strides=(512, 0))), (-1, dict(k_codes=None)), (-1, dict(tables=None)), (-1, dict(n_pages=-1)),
        (-2, dict(q_dtype=0)), (-2, dict(D=64)), (-2, dict(Hq=5)), (-2, dict(B=1025)), (-2, dict(page_size=20)),
        (-3, dict(workspace=None)), (-3, dict(workspace=264)), (-3, dict(workspace_bytes=nb - 1)),
    ])
    assert call("hq_paged4_decode", base, B=0) == 0
    for bad in ((0, 4, 2, 16, 4, 128), (2, 5, 2, 16, 4, 128), (2, 4, 2, 16, 4, 64), (1025, 4, 2, 16, 4, 128),
                (2, 258, 2, 16, 4, 128)):
        assert L.hq_paged4_decode_workspace_bytes(*bad) == 0


def test_gather_argument_errors():
    base = dict(k_codes=256, v_codes=256, code_strides=C2, k_scale=256, v_scale=256, scale_strides=SC2, n_pages=5, page_size=16,
                tables=256, table_stride=4, max_pages=4, lens=256, first=None, cu_seqlens=256, T=7, B=2, Hkv=2, D=128,
                k_out=256, v_out=512, out_dtype=1, k_strides=S2, v_strides=S2, zero_rest=0, status=None, stream=None)
    refused("hq_paged4_gather", base, [
        (-1, dict(k_codes=None)), (-1, dict(lens=None)), (-1, dict(cu_seqlens=None)), (-1, dict(T=-1)), (-1, dict(Hkv=0)),
        (-1, dict(k_out=None)), (-1, dict(v_out=264)), (-1, dict(v_out=256)), (-1, dict(k_strides=(0, 128))),
        (-1, dict(v_strides=(512, 4))), (-2, dict(D=64)), (-2, dict(out_dtype=0)), (-2, dict(page_size=17)),
    ])
    assert call("hq_paged4_gather", base, T=0) == 0


def test_prefill_argument_errors():
    L = _lib.lib()
    nb = L.hq_packed_prefill_workspace_bytes(16, 1 << 20, 1, 4, 2, 128)
    assert nb > 256                                        # few rows, many keys: split
    assert L.hq_packed_prefill_workspace_bytes(512, 512, 1, 16, 8, 128) == 1    # none is needed
    base = dict(q=256, k=256, v=256, dtype=1, q_strides=S2, k_strides=S2, v_strides=S2, cu_q=256, cu_k=256, T=16, Tk=1 << 20, B=1,
                Hq=4, Hkv=2, D=128, causal=1, sm_scale=0.1, out=256, out_strides=S2, zero_rest=0, workspace=256,
                workspace_bytes=nb, status=None, stream=None)
    refused("hq_packed_prefill", base, [
        (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(cu_q=None)), (-1, dict(cu_k=None)), (-1, dict(out=None)),
        (-1, dict(T=-1)), (-1, dict(Tk=-1)), (-1, dict(Hq=0)), (-1, dict(sm_scale=0.0)), (-1, dict(sm_scale=-0.1)),
        (-1, dict(sm_scale=float("nan"))), (-1, dict(sm_scale=float("inf"))), (-1, dict(q=264)), (-1, dict(v=264)),
        (-1, dict(k_strides=(0, 128))), (-1, dict(v_strides=(512, 0))),
        (-1, dict(k_strides=(128, 1 << 20))),              # K's larger stride elsewhere than V's
        (-1, dict(out_strides=(0, 128))), (-2, dict(dtype=0)), (-2, dict(D=64)), (-2, dict(Hq=5)),
        (-3, dict(workspace=None)), (-3, dict(workspace_bytes=nb - 1)), (-3, dict(workspace=264)),
    ])
    assert call("hq_packed_prefill", base, T=0) == 0
    assert call("hq_packed_prefill", base, B=0) == 0
    assert L.hq_packed_prefill_workspace_bytes(0, 5, 1, 4, 2, 128) == 0
    assert L.hq_packed_prefill_workspace_bytes(1 << 30, 5, 1, 4, 2, 128) == 0


def test_cpu_tensors_are_refused():
    cache = kernels.paged4_alloc(3, 2, page_size=16, device="cpu")
    assert cache["k"].shape == (3, 2, 16, 64) and cache["v_scale"].shape == (3, 2, 16, 4)
    q, k = torch.zeros(4, 4, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    tables, lens, cu = torch.zeros(4, 1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
    for call in (lambda: kernels.paged4_append(q, k, k, cache, tables, lens),
                 lambda: kernels.paged4_decode_attn(q, cache, tables, lens),
                 lambda: kernels.paged4_gather(cache, tables, lens, cu, 4),
                 lambda: kernels.packed_prefill_attn(q, k, k, cu)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()


def test_alloc_and_arguments_of_the_wrong_kind():
    for bad in (dict(page_size=48), dict(page_size=0), dict(head_dim=64)):
        with pytest.raises(ValueError):
            kernels.paged4_alloc(3, 2, device="cpu", **bad)
    with pytest.raises(ValueError):
        kernels.paged4_alloc(0, 2, device="cpu")
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    lens = torch.zeros(4, dtype=torch.int32)
    cache = kernels.paged4_alloc(3, 2, page_size=16, device="cpu")
    with pytest.raises(ValueError):
        kernels.paged4_decode_attn(q, {"k": 1}, lens[:, None], lens)
    with pytest.raises(ValueError):
        kernels.paged4_decode_attn(q, None, lens[:, None], lens)
    with pytest.raises(ValueError):
        kernels.paged4_decode_attn([1], cache, lens[:, None], lens)
    with pytest.raises(ValueError):
        kernels.paged4_append(q, q, q, cache, lens[:, None], [0])
    with pytest.raises(ValueError):
        kernels.paged4_append(q, q, q, cache, lens[:, None], lens, inv_freq=[0.5])
    with pytest.raises(ValueError):
        kernels.paged4_gather(cache, None, lens, lens, 4)
    with pytest.raises(ValueError):
        kernels.packed_prefill_attn(q, q, None, lens)


# ---- outputs that share memory with one another or with what a call reads
def test_outputs_that_overlap_are_refused():
    M = 1 << 20
    st = (512, 128)                                        # [T, 4, 128]; two heads of it: half a token's row
    append = dict(q=1 * M, k_new=2 * M, v_new=3 * M, x_dtype=1, q_strides=st, k_strides=(256, 128), v_strides=(256, 128), T=30, B=2,
                  Hq=4, Hkv=2, D=128, cu_seqlens=256, lens=256, pos_offset=None, q_weight=None, k_weight=None, w_dtype=1, eps=1e-6,
                  inv_freq=256, rotary_dim=128, interleaved=0, factor=1.0, k_codes=4 * M, v_codes=5 * M, code_strides=C2,
                  k_scale=6 * M, v_scale=7 * M, scale_strides=SC2, n_pages=5, page_size=16, tables=256, table_stride=4, max_pages=4,
                  q_out=8 * M, qo_strides=st, k_out=9 * M, ko_strides=(256, 128), copy_rest=0, status=None, stream=None)
    refused("hq_paged4_append", append, [
        (-1, dict(k_out=2 * M)), (-1, dict(k_out=2 * M + 512)), (-1, dict(k_out=2 * M + 16)), (-1, dict(k_out=2 * M - 29 * 512)),
        (-1, dict(k_out=3 * M + 512)), (-1, dict(k_out=1 * M)), (-1, dict(k_out=8 * M + 1024 * 29)),
        (-1, dict(k_out=2 * M + 256, ko_strides=(512, 128))),
        (-1, dict(k_out=9 * M, ko_strides=(128, 128))),     # tokens that share heads
        (-1, dict(q_out=1 * M + 1024)), (-1, dict(q_out=1 * M, qo_strides=(1024, 128))), (-1, dict(q_out=2 * M)), (-1, dict(q_out=3 * M - 16)),
        (-1, dict(q_out=8 * M, qo_strides=(512, 64))), (-1, dict(q_out=8 * M, qo_strides=(128, 128))),
        (-1, dict(v_codes=4 * M)), (-1, dict(v_codes=4 * M + 1024)), (-1, dict(code_strides=(1024, 1024))),
        (-1, dict(v_scale=6 * M + 128 * 9)), (-1, dict(scale_strides=(64, 64))),
    ])
    decode = dict(q=1 * M, q_dtype=1, q_strides=st, k_codes=2 * M, v_codes=3 * M, code_strides=C2, k_scale=4 * M, v_scale=5 * M,
                  scale_strides=SC2, n_pages=5, page_size=16, tables=256, table_stride=4, max_pages=4, lens=256, B=20, Hq=4, Hkv=2,
                  D=128, sm_scale=0.1, out=6 * M, out_strides=st, workspace=None, workspace_bytes=0, status=None, stream=None)
    refused("hq_paged4_decode", decode, [
        (-1, dict(out=1 * M + 1024)), (-1, dict(out=1 * M + 8)), (-1, dict(out=1 * M, out_strides=(256, 128))),
        (-1, dict(out_strides=(128, 128))), (-1, dict(out_strides=(512, 64))), (-1, dict(out_strides=(0, 128))),
    ])
    gather = dict(k_codes=2 * M, v_codes=3 * M, code_strides=C2, k_scale=4 * M, v_scale=5 * M, scale_strides=SC2, n_pages=5,
                  page_size=16, tables=256, table_stride=4, max_pages=4, lens=256, first=None, cu_seqlens=256, T=70, B=2, Hkv=2,
                  D=128, k_out=6 * M, v_out=7 * M, out_dtype=1, k_strides=(256, 128), v_strides=(256, 128), zero_rest=0, status=None,
                  stream=None)
    refused("hq_paged4_gather", gather, [
        (-1, dict(v_out=6 * M)), (-1, dict(v_out=6 * M + 512)), (-1, dict(v_out=6 * M + 256)), (-1, dict(v_out=6 * M - 69 * 512)),
        (-1, dict(k_strides=(512, 128), v_strides=(512, 128), v_out=6 * M + 256)),
        (-1, dict(k_strides=(128, 128))), (-1, dict(v_strides=(128, 256))), (-1, dict(v_strides=(256, 0))),
    ])
    prefill = dict(q=1 * M, k=2 * M, v=3 * M, dtype=1, q_strides=st, k_strides=(256, 128), v_strides=(256, 128), cu_q=256, cu_k=256,
                   T=160, Tk=160, B=1, Hq=4, Hkv=2, D=128, causal=1, sm_scale=0.1, out=6 * M, out_strides=st, zero_rest=0,
                   workspace=16 * M, workspace_bytes=1 << 30, status=None, stream=None)
    refused("hq_packed_prefill", prefill, [
        (-1, dict(out=2 * M)), (-1, dict(out=3 * M + 159 * 512)), (-1, dict(out=1 * M + 1024)), (-1, dict(out=1 * M, out_strides=(1024, 128))),
        (-1, dict(out_strides=(128, 128))), (-1, dict(out_strides=(0, 128))), (-1, dict(out_strides=(512, 0))),
    ])
