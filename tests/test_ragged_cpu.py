"""Host side of the ragged-batch operators: what the C entries and the wrappers refuse (before
anything touches a device), scratch sizes, and the rotary frequencies."""
import ctypes
import math

import pytest
import torch

from halftone_quantizedkvcache_b200 import _lib, kernels

F32, BF16, F16 = (kernels._DT[t] for t in (torch.float32, torch.bfloat16, torch.float16))
INVALID, UNSUPPORTED, WORKSPACE = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE
B, HQ, HKV, S, D = 2, 8, 2, 640, 128
PTR = 1 << 20          # aligned and never read: every call here ends on the host
CODES = (HKV * S * D, S * D, D)


def decode_args(**change):
    a = dict(q=PTR, q_dt=BF16, qs=(HQ * D, D, 1), k=PTR, v=PTR, kvs=CODES, ksc=PTR, vsc=PTR, sdt=F16,
             kss=(HKV * D, D, 1), vss=(HKV * S, S, 1), lens=PTR, B=B, Hq=HQ, Hkv=HKV, S=S, D=D,
             window=0, sinks=0, sm=0.1, qq=0, out=PTR, os=(HQ * D, D, 1), ws=PTR, nws=0, status=None,
             stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return [_lib.strides(x, 3) if isinstance(x, tuple) else x for x in a.values()]


@pytest.mark.parametrize("change,code", [
    (dict(), WORKSPACE),                       # all else in order: the scratch is too small
    (dict(nws=1 << 30, ws=PTR + 16), WORKSPACE),
    (dict(nws=1 << 30, ws=None), WORKSPACE),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(q=PTR + 8), INVALID),
    (dict(out=PTR + 4), INVALID), (dict(k=PTR + 8), INVALID), (dict(v=PTR + 1), INVALID),
    (dict(k=None), INVALID), (dict(ksc=None), INVALID), (dict(vsc=None), INVALID),
    (dict(qs=(HQ * D, D, 2)), INVALID), (dict(qs=(HQ * D + 4, D, 1)), INVALID),
    (dict(os=(HQ * D, D + 2, 1)), INVALID), (dict(kvs=(HKV * S * D, S * D, D + 8)), INVALID),
    (dict(B=-1), INVALID), (dict(S=-1), INVALID), (dict(window=-1), INVALID), (dict(sinks=-1), INVALID),
    (dict(Hq=0), INVALID), (dict(Hkv=0), INVALID),
    (dict(Hkv=3), UNSUPPORTED), (dict(Hq=2 * 129), UNSUPPORTED), (dict(D=64), UNSUPPORTED),
    (dict(q_dt=F32), UNSUPPORTED), (dict(q_dt=17), UNSUPPORTED), (dict(sdt=BF16), UNSUPPORTED),
    (dict(B=1025), UNSUPPORTED), (dict(S=(1 << 30) + 1), UNSUPPORTED),
    (dict(B=0), _lib.OK),
])
def test_window_decode_c_entry(change, code):
    assert _lib.lib().hq_window_decode_int8(*decode_args(**change)) == code


def prefill_args(**change):
    a = dict(q=PTR, q_dt=BF16, qs=(HQ * 40 * D, 40 * D, D, 1), k=PTR, v=PTR, kvs=CODES, ksc=PTR,
             vsc=PTR, sdt=F16, kss=(HKV * D, D, 1), vss=(HKV * S, S, 1), lens=PTR, q_lens=None, B=B,
             Hq=HQ, Hkv=HKV, Sq=40, S=S, D=D, window=0, sinks=0, sm=0.1, qq=0, out=PTR,
             os=(HQ * 40 * D, D, HQ * D, 1), ws=PTR, nws=0, status=None, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return [_lib.strides(x, len(x)) if isinstance(x, tuple) else x for x in a.values()]


@pytest.mark.parametrize("change,code", [
    (dict(), WORKSPACE),                       # few rows: the keys are split, which takes scratch
    (dict(Sq=-1), INVALID), (dict(qs=(HQ * 40 * D, 40 * D, D, 2)), INVALID),
    (dict(qs=(HQ * 40 * D, 40 * D, D + 1, 1)), INVALID), (dict(q=PTR + 2), INVALID),
    (dict(B=65536), UNSUPPORTED), (dict(Sq=1 << 30), UNSUPPORTED), (dict(Sq=1 << 22), UNSUPPORTED),
    (dict(D=256), UNSUPPORTED), (dict(q_dt=F32), UNSUPPORTED), (dict(Hq=7), UNSUPPORTED),
    (dict(B=0), _lib.OK), (dict(Sq=0), _lib.OK),
])
def test_window_prefill_c_entry(change, code):
    assert _lib.lib().hq_window_prefill_int8(*prefill_args(**change)) == code


def prefix_args(**change):
    a = dict(q=PTR, q_dt=BF16, qs=(HQ * D, D, 1), pk=PTR, pv=PTR, pkvs=CODES, pksc=PTR, pvsc=PTR,
             pkss=(HKV * D, D, 1), pvss=(HKV * S, S, 1), plens=None, G=1, P=S, k=PTR, v=PTR,
             kvs=CODES, ksc=PTR, vsc=PTR, kss=(HKV * D, D, 1), vss=(HKV * S, S, 1), lens=PTR, S=S,
             sdt=F16, B=B, Hq=HQ, Hkv=HKV, D=D, sm=0.1, qq=0, out=PTR, os=(HQ * D, D, 1), ws=PTR,
             nws=0, status=None, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return [_lib.strides(x, 3) if isinstance(x, tuple) else x for x in a.values()]


@pytest.mark.parametrize("change,code", [
    (dict(), WORKSPACE), (dict(G=0), INVALID), (dict(G=3), INVALID), (dict(pk=None), INVALID),
    (dict(pv=PTR + 8), INVALID), (dict(pkvs=(HKV * S * D, S * D, D + 1)), INVALID),
    (dict(P=-1), INVALID), (dict(B=1026, G=2), UNSUPPORTED), (dict(D=64), UNSUPPORTED),
    (dict(sdt=BF16), UNSUPPORTED), (dict(P=(1 << 30) + 1), UNSUPPORTED), (dict(B=0), _lib.OK),
])
def test_prefix_decode_c_entry(change, code):
    assert _lib.lib().hq_prefix_decode_int8(*prefix_args(**change)) == code


def rope_args(**change):
    q4, k4 = (HQ * 3 * D, 3 * D, D, 1), (HKV * 3 * D, 3 * D, D, 1)
    a = dict(q=PTR, k=PTR, v=PTR, dt=BF16, qs=q4, ks=k4, vs=k4, B=B, Hq=HQ, Hkv=HKV, S=3, D=D,
             freq=PTR, rot=64, inter=0, factor=1.0, lens=PTR, n_new=None, off=None, ksc=PTR, sdt=F16,
             kss=(0, D, 1), kc=PTR, vc=PTR, cs=CODES, vsc=PTR, vss=(HKV * S, S, 1), cap=S, qo=PTR,
             qos=q4, status=None, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return [_lib.strides(x, len(x)) if isinstance(x, tuple) else x for x in a.values()]


@pytest.mark.parametrize("change,code", [
    (dict(q=None), INVALID), (dict(lens=None), INVALID), (dict(freq=None), INVALID),
    (dict(rot=63), INVALID), (dict(rot=130), INVALID), (dict(rot=-2), INVALID), (dict(B=-1), INVALID),
    (dict(Hkv=0), INVALID), (dict(cap=-1), INVALID), (dict(kc=PTR + 8), INVALID),
    (dict(q=PTR + 2), INVALID), (dict(qs=(HQ * 3 * D, 3 * D, D + 4, 1)), INVALID),
    (dict(ks=(HKV * 3 * D, 3 * D, D, 2)), INVALID), (dict(cs=(HKV * S * D, S * D, D + 8)), INVALID),
    (dict(D=96, rot=32), UNSUPPORTED), (dict(dt=17), UNSUPPORTED), (dict(sdt=BF16), UNSUPPORTED),
    (dict(B=1 << 20, S=1 << 20), UNSUPPORTED),
    (dict(B=0), _lib.OK), (dict(S=0), _lib.OK),
])
def test_rope_append_c_entry(change, code):
    assert _lib.lib().hq_rope_append_kv(*rope_args(**change)) == code


def test_scratch_sizes():
    """Zero where a shape is not supported, and never below what a smaller batch takes."""
    L = _lib.lib()
    size = L.hq_window_workspace_bytes
    assert size(BF16, 4, 8, 2, 0, 4096, 128, 0, 0) % 4 == 0
    for bad in ((BF16, 0, 8, 2, 0, 64, 128, 0, 0), (BF16, 2, 8, 3, 0, 64, 128, 0, 0),
                (BF16, 2, 8, 2, 0, 64, 64, 0, 0), (BF16, 2, 8, 2, -1, 64, 128, 0, 0),
                (BF16, 2, 8, 2, 0, 64, 128, -1, 0), (BF16, 1025, 8, 2, 0, 64, 128, 0, 0),
                (BF16, 2, 2 * 129, 2, 0, 64, 128, 0, 0)):
        assert size(*bad) == 0
    sizes = [size(BF16, b, 8, 2, 0, 4096, 128, 256, 4) for b in range(1, 65)]
    assert sizes == sorted(sizes)
    assert size(BF16, 1, 8, 8, 8192, 8192, 128, 0, 0) == 256   # a block per row tile: none
    pre = L.hq_prefix_decode_workspace_bytes
    assert pre(F16, 2, 8, 8, 2, 512, 64, 128) > 0
    for bad in ((F16, 3, 8, 8, 2, 512, 64, 128), (F16, 2, 8, 8, 2, 512, 64, 256),
                (F16, 0, 8, 8, 2, 512, 64, 128), (F16, 2, 8, 8, 2, -1, 64, 128)):
        assert pre(*bad) == 0


def test_entries_end_in_status_codes():
    """The entries are plain C: a null stride array or a null everything is a code, no abort."""
    L = _lib.lib()
    for fn in (L.hq_window_decode_int8, L.hq_window_prefill_int8, L.hq_prefix_decode_int8,
               L.hq_rope_append_kv):
        args = [0.0 if t is ctypes.c_float else None if t is ctypes.c_void_p or hasattr(t, "_type_")
                and not isinstance(t._type_, str) else 0 for t in fn.argtypes]
        assert fn(*args) == INVALID


def test_wrappers_refuse_host_tensors_and_wrong_kinds():
    q = torch.zeros(2, 8, 1, 128, dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 64, 128, dtype=torch.int8)
    ksc, vsc = torch.ones(2, 2, 1, 128, dtype=torch.float16), torch.ones(2, 2, 64, 1, dtype=torch.float16)
    n = torch.zeros(2, dtype=torch.int32)
    kn = torch.zeros(2, 2, 1, 128, dtype=torch.bfloat16)
    f = torch.ones(64)
    for call in (lambda q, n: kernels.int8_window_decode_attn(q, k, ksc, k, vsc, n),
                 lambda q, n: kernels.int8_window_prefill_attn(q, k, ksc, k, vsc, n),
                 lambda q, n: kernels.int8_window_prefill_attn(q, k, ksc, k, vsc, n, q_lens=n),
                 lambda q, n: kernels.int8_prefix_decode_attn(q, k[:1], ksc[:1], k[:1], vsc[:1], k, ksc,
                                                              k, vsc, n, prefix_lens=n),
                 lambda q, n: kernels.rope_append_kv(q, kn, kn, f, k, k, ksc, vsc, n, n_new=n)):
        with pytest.raises(ValueError):    # host tensors
            call(q, n)
        with pytest.raises(ValueError):    # lengths that are no tensor
            call(q, [1, 2])
        with pytest.raises(ValueError):
            call(None, n)


def test_rope_inv_freq():
    f, m = kernels.rope_inv_freq(64, 500000.0, device="cpu")
    j = torch.arange(32, dtype=torch.float64)
    # a float64 power rounded once to float32
    assert m == 1.0 and f.dtype == torch.float32
    assert torch.equal(f, (500000.0 ** (-2 * j / 64)).float())
    lin, m = kernels.rope_inv_freq(64, 500000.0, scaling="linear", factor=4.0, device="cpu")
    assert m == 1.0 and torch.equal(lin, f / 4)          # a power of two: exact
    ntk, m = kernels.rope_inv_freq(64, 10000.0, scaling="ntk", factor=8.0, device="cpu")
    one, _ = kernels.rope_inv_freq(64, 10000.0, device="cpu")
    assert m == 1.0 and ntk[0] == 1.0
    # the slowest pair is divided by the factor: one rounding on each side, and the power's
    assert abs(ntk[-1].item() * 8 / one[-1].item() - 1) <= 4 * 2.0 ** -24
    assert (ntk <= one).all()
    yarn, m = kernels.rope_inv_freq(128, 10000.0, scaling="yarn", factor=16.0, original_len=4096,
                                    device="cpu")
    base, _ = kernels.rope_inv_freq(128, 10000.0, device="cpu")
    assert abs(m - (0.1 * math.log(16.0) + 1)) < 1e-12
    turns = 4096 * base.double() / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], base[turns > 40])     # well above beta_fast: unchanged
    slow = turns < 0.8
    assert slow.any() and torch.equal(yarn[slow], base[slow] / 16)
    ratio = yarn / base
    assert (ratio[1:] <= ratio[:-1] + 2.0 ** -22).all()        # the ramp falls
    same, m = kernels.rope_inv_freq(128, 10000.0, scaling="yarn", factor=1.0, original_len=4096,
                                    device="cpu")
    assert m == 1.0 and torch.equal(same, base)
    for bad in (dict(rotary_dim=63), dict(rotary_dim=0), dict(rotary_dim=64, theta=0.0),
                dict(rotary_dim=64, factor=0.5), dict(rotary_dim=64, scaling="other"),
                dict(rotary_dim=2, scaling="ntk", factor=2.0), dict(rotary_dim=64, scaling="yarn")):
        with pytest.raises(ValueError):
            kernels.rope_inv_freq(device="cpu", **bad)
