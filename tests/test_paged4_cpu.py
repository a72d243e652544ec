"""The paged 4-bit cache's and the packed prompt attention's entry points on a host without a GPU:
argument errors come back before anything is launched, CPU tensors are refused."""
import pytest
import torch

from halftone_quantizedkvcache_b200 import _lib, kernels

S2 = _lib.strides((512, 128), 2)
C2 = _lib.strides((16 * 64 * 2, 16 * 64), 2)
SC2 = _lib.strides((16 * 4 * 2, 16 * 4), 2)


def changed(args, **at):
    a = list(args)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def refused(fn, base, cases):
    for code, at in cases:
        assert fn(*changed(base, **at)) == code, at


def test_append_argument_errors():
    # q k v dt qs ks vs T B Hq Hkv D cu lens off qw kw wdt eps inv rot inter factor k v cs ks vs ss n page
    # tables ts max qo qos ko kos rest status stream
    base = [256, 256, 256, 1, S2, S2, S2, 3, 2, 4, 2, 128, 256, 256, None, None, None, 1, 1e-6, 256, 128, 0, 1.0,
            256, 256, C2, 256, 256, SC2, 5, 16, 256, 4, 4, 256, S2, None, None, 0, None, None]
    fn = _lib.lib().hq_paged4_append
    refused(fn, base, [
        (-1, dict(_0=None)), (-1, dict(_1=None)), (-1, dict(_2=None)), (-1, dict(_13=None)), (-1, dict(_34=None)),
        (-1, dict(_7=-1)), (-1, dict(_8=-1)), (-1, dict(_9=0)), (-1, dict(_10=0)), (-1, dict(_12=None)),
        (-1, dict(_19=None)), (-1, dict(_20=144)), (-1, dict(_18=-1.0)), (-1, dict(_18=float("nan"))),
        (-1, dict(_0=264)), (-1, dict(_4=_lib.strides((512, 100), 2))), (-1, dict(_35=_lib.strides((0, 128), 2))),
        (-1, dict(_23=None)), (-1, dict(_23=264)), (-1, dict(_25=_lib.strides((100, 1024), 2))),
        (-1, dict(_25=_lib.strides((1024, 512), 2))), (-1, dict(_28=_lib.strides((32, 64), 2))), (-1, dict(_31=None)),
        (-1, dict(_36=256, _37=S2)),                       # k_out is k_new
        (-2, dict(_3=0)), (-2, dict(_11=64, _20=64)), (-2, dict(_20=24)), (-2, dict(_17=2)), (-2, dict(_30=48)), (-2, dict(_30=8)),
        (-2, dict(_30=512)), (-2, dict(_33=1 << 28)), (-2, dict(_25=_lib.strides((1 << 31, 1024), 2))),
    ])


def test_decode_argument_errors():
    L = _lib.lib()
    nb = L.hq_paged4_decode_workspace_bytes(2, 4, 2, 16, 128, 128)
    assert nb > 1 == L.hq_paged4_decode_workspace_bytes(2, 4, 2, 16, 64, 128)   # 1024 tokens: none is needed
    base = [256, 1, S2, 256, 256, C2, 256, 256, SC2, 5, 16, 256, 128, 128, 256, 2, 4, 2, 128, 0.1, 256, S2, 256, nb, None, None]
    refused(L.hq_paged4_decode, base, [
        (-1, dict(_0=None)), (-1, dict(_14=None)), (-1, dict(_20=None)), (-1, dict(_0=264)), (-1, dict(_15=-1)),
        (-1, dict(_16=0)), (-1, dict(_2=_lib.strides((512, 4), 2))), (-1, dict(_21=_lib.strides((0, 128), 2))),
        (-1, dict(_21=_lib.strides((512, 0), 2))), (-1, dict(_3=None)), (-1, dict(_11=None)), (-1, dict(_9=-1)),
        (-2, dict(_1=0)), (-2, dict(_18=64)), (-2, dict(_16=5)), (-2, dict(_15=1025)), (-2, dict(_10=20)),
        (-3, dict(_22=None)), (-3, dict(_22=264)), (-3, dict(_23=nb - 1)),
    ])
    assert L.hq_paged4_decode(*changed(base, _15=0)) == 0
    for bad in ((0, 4, 2, 16, 4, 128), (2, 5, 2, 16, 4, 128), (2, 4, 2, 16, 4, 64), (1025, 4, 2, 16, 4, 128),
                (2, 258, 2, 16, 4, 128)):
        assert L.hq_paged4_decode_workspace_bytes(*bad) == 0


def test_gather_argument_errors():
    base = [256, 256, C2, 256, 256, SC2, 5, 16, 256, 4, 4, 256, None, 256, 7, 2, 2, 128, 256, 512, 1, S2, S2, 0, None, None]
    refused(_lib.lib().hq_paged4_gather, base, [
        (-1, dict(_0=None)), (-1, dict(_11=None)), (-1, dict(_13=None)), (-1, dict(_14=-1)), (-1, dict(_16=0)),
        (-1, dict(_18=None)), (-1, dict(_19=264)), (-1, dict(_19=256)), (-1, dict(_21=_lib.strides((0, 128), 2))),
        (-1, dict(_22=_lib.strides((512, 4), 2))), (-2, dict(_17=64)), (-2, dict(_20=0)), (-2, dict(_7=17)),
    ])
    assert _lib.lib().hq_paged4_gather(*changed(base, _14=0)) == 0


def test_prefill_argument_errors():
    L = _lib.lib()
    nb = L.hq_packed_prefill_workspace_bytes(16, 1 << 20, 1, 4, 2, 128)
    assert nb > 256                                        # few rows, many keys: split
    base = [256, 256, 256, 1, S2, S2, S2, 256, 256, 16, 1 << 20, 1, 4, 2, 128, 1, 0.1, 256, S2, 0, 256, nb, None, None]
    refused(L.hq_packed_prefill, base, [
        (-1, dict(_0=None)), (-1, dict(_1=None)), (-1, dict(_7=None)), (-1, dict(_8=None)), (-1, dict(_17=None)),
        (-1, dict(_9=-1)), (-1, dict(_10=-1)), (-1, dict(_12=0)), (-1, dict(_16=0.0)), (-1, dict(_16=-0.1)),
        (-1, dict(_16=float("nan"))), (-1, dict(_16=float("inf"))), (-1, dict(_0=264)), (-1, dict(_2=264)),
        (-1, dict(_5=_lib.strides((0, 128), 2))), (-1, dict(_6=_lib.strides((512, 0), 2))),
        (-1, dict(_5=_lib.strides((128, 1 << 20), 2))),    # K's larger stride elsewhere than V's
        (-1, dict(_18=_lib.strides((0, 128), 2))), (-2, dict(_3=0)), (-2, dict(_14=64)), (-2, dict(_12=5)),
        (-3, dict(_20=None)), (-3, dict(_21=nb - 1)), (-3, dict(_20=264)),
    ])
    assert L.hq_packed_prefill(*changed(base, _9=0)) == 0
    assert L.hq_packed_prefill(*changed(base, _11=0)) == 0
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
