"""Attention over ragged int8 caches on the GPU: sliding window with sinks (decode, prefill)
and shared-prefix decode, against the definitions in float64.

Tolerance, derived from the arithmetic.  Write z_j for the scores, p_j for the softmax, v_j for
the dequantized values, u = 2^-11 (half a step of float16).  The kernel rounds P to float16
once (u P); float16 models keep q' in two float16 parts (|dz_j| <= u^2 sum_d |q_d k_jd|
sm_scale) and V exact, bf16 models q' in one (u in place of u^2) and V as a float16 product of
the code and a float16 scale (2 u).  Weights off by a relative dz change a normalised sum by
2 dz at most, so
    |out - ref| <= eps_out / 2 |ref| + A (r u + 2 Z dq + 2^-16 (1 + Z)),
A = sum_j p_j |v_j|, Z = max_j sum_d |q_d k_jd| sm_scale, r = 1 or 3, dq = u^2 or u; the last
term covers float32 accumulation (128 products, up to 2^13 keys) and the approximate exp2
(2^-22 each).
"""
import math

import pytest
import torch

from halftone_quantizedkvcache_b200 import kernels

pytestmark = pytest.mark.gpu
TDT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
D = 128
U = 2.0 ** -11


def make_cache(g, B, Hkv, S, sdt, v_spread=False):
    k = torch.randint(-127, 128, (B, Hkv, S, D), generator=g, device="cuda", dtype=torch.int8)
    v = torch.randint(-127, 128, (B, Hkv, S, D), generator=g, device="cuda", dtype=torch.int8)
    ksc = torch.rand((B, Hkv, 1, D), generator=g, device="cuda") * 0.03 + 0.01
    ksc[..., ::37] *= 20
    vsc = torch.rand((B, Hkv, S, 1), generator=g, device="cuda") * 0.02 + 0.01
    if v_spread:  # V scales over many powers of two, some exactly zero
        vsc = vsc * 2.0 ** torch.randint(-12, 13, vsc.shape, generator=g, device="cuda").float()
        vsc[:, :, ::5] = 0.0
    return k, (ksc / 4).to(TDT[sdt]), v, vsc.to(TDT[sdt])


def fake_quant(q):
    x = q.float()
    s = x.abs().amax(-1, keepdim=True).clamp(min=1e-8) / torch.full((), 127.0, device="cuda")
    return ((x / s).round().clamp(-127, 127) * s).to(q.dtype)


def ref_rows(q, k, v, seen, dt):
    """float64 attention of q [R,D] over k, v [S,D] with seen [R,S]: (out, bound)."""
    q = q.double()
    sm = 1.0 / math.sqrt(D)
    z = (q @ k.T) * sm
    z = torch.where(seen, z, torch.full_like(z, -math.inf))
    top = z.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(z - top)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    out = p @ v
    a = p @ v.abs()
    zabs = torch.where(seen, (q.abs() @ k.abs().T) * sm, torch.zeros_like(z)).amax(-1, keepdim=True)
    dq, r = (U, 3) if dt == "bf16" else (U * U, 1)
    tol = torch.finfo(TDT[dt]).eps / 2 * out.abs() + a * (r * U + 2 * zabs * dq + 2.0 ** -16 * (1 + zabs))
    return out, tol + 1e-30


def check(got, ref, tol, what):
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = err > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst ratio "
                           f"{(err / tol).max().item():.2f}, max err {err.max().item():.3e}")


def window_ref(q, cache, lens, q_lens, window, sinks, dt):
    """[B,Sq,Hq,D] reference and bound (rows past q_lens: zeros, no error allowed)."""
    k8, ksc, v8, vsc = cache
    B, Hq, Sq, _ = q.shape
    rep = Hq // k8.shape[1]
    out = torch.zeros((B, Sq, Hq, D), dtype=torch.float64, device="cuda")
    tol = torch.full_like(out, 1e-30)
    for b in range(B):
        n, m = min(max(lens[b], 0), k8.shape[2]), q_lens[b]
        pos = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        seen = (j <= pos) & ((j > pos - (window or 1 << 40)) | (j < sinks))
        if n == 0 or m == 0:
            continue
        for h in range(Hq):
            k = k8[b, h // rep, :n].double() * ksc[b, h // rep].double()
            v = v8[b, h // rep, :n].double() * vsc[b, h // rep, :n].double()
            out[b, :m, h], tol[b, :m, h] = ref_rows(q[b, h, :m], k, v, seen, dt)
    return out, tol


def poison_past(cache, lens):
    """What lies past a sequence's length must not matter."""
    k8, _, v8, vsc = cache
    for b, n in enumerate(lens):
        n = max(n, 0)
        vsc[b, :, n:] = float("nan")
        k8[b, :, n:] = 127
        v8[b, :, n:] = -128


@pytest.mark.parametrize("B,Hkv,rep,cap,lens,window,sinks,dt,sdt", [
    (1, 1, 1, 1, [1], None, 0, "bf16", "f16"),                  # one token
    (3, 2, 2, 64, [0, 1, 64], 1, 0, "bf16", "f16"),             # empty, window of one
    (2, 8, 2, 700, [700, 129], 128, 4, "bf16", "f32"),          # tiles cut by the window
    (4, 2, 4, 1111, [5, 300, 1000, 1111], 256, 200, "f16", "f16"),  # sinks past one tile
    (5, 1, 7, 513, [0, 127, 128, 129, 513], 130, 1, "bf16", "f32"),  # odd group
    (2, 2, 16, 400, [400, 399], None, 0, "f16", "f32"),
    (1, 1, 128, 300, [300], 77, 3, "bf16", "f16"),              # one kv head for all
    (1, 8, 2, 9000, [9000], 4096, 4, "bf16", "f16"),            # cut over many blocks
    (200, 2, 2, 300, None, 100, 2, "bf16", "f16"),              # more units than blocks
    (2, 2, 2, 200, [999, -3], 50, 2, "bf16", "f16"),            # lengths out of range clamp
    (2, 1, 3, 256, [200, 256], 1 << 20, 1 << 20, "f16", "f16"),
])
def test_window_decode(B, Hkv, rep, cap, lens, window, sinks, dt, sdt):
    g = torch.Generator(device="cuda").manual_seed(B * 7 + cap)
    if lens is None:
        lens = [(37 * b) % (cap + 1) for b in range(B)]
    cache = make_cache(g, B, Hkv, cap, sdt)
    poison_past(cache, lens)
    q = torch.randn((B, Hkv * rep, 1, D), generator=g, device="cuda").to(TDT[dt])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = kernels.int8_window_decode_attn(q, *cache, n, window=window, sinks=sinks)
    assert got.shape == q.shape and got.dtype == q.dtype
    ref, tol = window_ref(q, cache, lens, [1] * B, window, sinks, dt)
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "window decode")
    again = kernels.int8_window_decode_attn(q[:, :, 0], *cache, n, window=window, sinks=sinks)
    assert torch.equal(again, got[:, :, 0]), "the same call twice"
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("B,Hkv,rep,Sq,cap,lens,q_lens,window,sinks,dt,sdt", [
    (1, 1, 1, 1, 1, [1], None, None, 0, "bf16", "f16"),
    (1, 8, 2, 512, 512, [512], None, 256, 4, "bf16", "f16"),
    (2, 2, 2, 300, 300, [300, 300], None, None, 0, "bf16", "f32"),      # plain causal
    (3, 2, 6, 77, 1500, [200, 900, 1500], [1, 40, 77], 400, 3, "f16", "f32"),
    (4, 1, 3, 50, 130, [50, 130, 0, 64], [50, 0, 0, 17], 20, 1, "bf16", "f16"),
    (1, 2, 4, 700, 2000, [2000], None, 64, 130, "bf16", "f16"),         # sinks longer than a tile
    (2, 1, 16, 129, 400, [400, 300], None, 1, 0, "f16", "f16"),         # each sees itself
    (1, 4, 1, 5, 8000, [8000], None, None, 0, "bf16", "f16"),           # few rows, split keys
    (2, 16, 2, 600, 600, [600, 500], [600, 500], 300, 0, "bf16", "f16"),  # two row tiles a block
    (1, 1, 2, 40, 100, [25], None, None, 0, "bf16", "f16"),             # queries before position 0
])
def test_window_prefill(B, Hkv, rep, Sq, cap, lens, q_lens, window, sinks, dt, sdt):
    g = torch.Generator(device="cuda").manual_seed(Sq * 3 + cap)
    cache = make_cache(g, B, Hkv, cap, sdt)
    poison_past(cache, lens)
    q = torch.randn((B, Hkv * rep, Sq, D), generator=g, device="cuda").to(TDT[dt])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ql = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device="cuda")
    got = kernels.int8_window_prefill_attn(q, *cache, n, window=window, sinks=sinks, q_lens=ql)
    assert got.shape == (B, Sq, Hkv * rep, D) and got.dtype == q.dtype
    ref, tol = window_ref(q, cache, lens, q_lens or [Sq] * B, window, sinks, dt)
    check(got, ref, tol, "window prefill")
    if q_lens is not None:  # rows past q_lens stay as they were
        out = torch.full_like(got, 3.0)
        kernels.int8_window_prefill_attn(q, *cache, n, window=window, sinks=sinks, q_lens=ql, out=out)
        for b, m in enumerate(q_lens):
            assert (out[b, m:] == 3.0).all()
            assert torch.equal(out[b, :m], got[b, :m])
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("G,U,Hkv,rep,P,plens,cap,lens,dt,sdt", [
    (1, 1, 1, 1, 1, [1], 1, [1], "bf16", "f16"),
    (1, 4, 8, 2, 512, None, 256, [1, 100, 256, 0], "bf16", "f16"),
    (3, 5, 2, 8, 700, [700, 0, 333], 333, None, "f16", "f32"),
    (1, 64, 2, 2, 5000, None, 40, None, "bf16", "f16"),        # 128 rows
    (1, 65, 2, 3, 1500, None, 40, None, "bf16", "f16"),        # 195 rows: two row tiles
    (2, 70, 1, 8, 600, [555, 600], 17, None, "bf16", "f32"),   # 560 rows: three blocks' worth
    (2, 33, 1, 8, 300, [0, 0], 30, None, "f16", "f16"),        # no prefix at all
    (1, 3, 2, 2, 300, None, 64, [0, 0, 0], "bf16", "f16"),     # nothing of their own
    (1, 2, 2, 2, 64, [0], 64, [0, 7], "bf16", "f16"),          # one sequence sees nothing
])
def test_prefix_decode(G, U, Hkv, rep, P, plens, cap, lens, dt, sdt):
    g = torch.Generator(device="cuda").manual_seed(G * 100 + U + P)
    B = G * U
    if lens is None:
        lens = [(29 * b) % (cap + 1) for b in range(B)]
    pre, own = make_cache(g, G, Hkv, P, sdt), make_cache(g, B, Hkv, cap, sdt)
    poison_past(own, lens)
    pl = plens or [P] * G
    poison_past(pre, pl)
    q = torch.randn((B, Hkv * rep, 1, D), generator=g, device="cuda").to(TDT[dt])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pn = None if plens is None else torch.tensor(plens, dtype=torch.int32, device="cuda")
    got = kernels.int8_prefix_decode_attn(q, *pre, *own, n, prefix_lens=pn)
    for b in range(B):
        gr = b // U
        for h in range(Hkv * rep):
            kh = h // rep
            k = torch.cat([pre[0][gr, kh, :pl[gr]].double() * pre[1][gr, kh].double(),
                           own[0][b, kh, :lens[b]].double() * own[1][b, kh].double()])
            v = torch.cat([pre[2][gr, kh, :pl[gr]].double() * pre[3][gr, kh, :pl[gr]].double(),
                           own[2][b, kh, :lens[b]].double() * own[3][b, kh, :lens[b]].double()])
            if len(k) == 0:
                assert (got[b, h] == 0).all()
                continue
            seen = torch.ones((1, len(k)), dtype=torch.bool, device="cuda")
            ref, tol = ref_rows(q[b, h], k, v, seen, dt)
            check(got[b, h], ref, tol, f"prefix decode b={b} h={h}")
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_v_scales_over_many_powers_of_two(dt):
    """V scales from 2^-19 to 2^7 and exact zeros in one cache: neither side of the softmax
    loses what the other holds."""
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = make_cache(g, 2, 2, 600, "f32", v_spread=True)
    lens = [600, 77]
    q = torch.randn((2, 4, 1, D), generator=g, device="cuda").to(TDT[dt])
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = kernels.int8_window_decode_attn(q, *cache, n)
    ref, tol = window_ref(q, cache, lens, [1, 1], None, 0, dt)
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "v scales")
    cache[3].zero_()  # all values zero
    got = kernels.int8_window_decode_attn(q, *cache, n)
    assert (got == 0).all()


def test_one_heavy_sink_with_zero_values():
    """A first token that takes nearly all of the softmax and holds zeros, as sinks do."""
    g = torch.Generator(device="cuda").manual_seed(6)
    cache = make_cache(g, 1, 1, 500, "f16")
    cache[3][:, :, 0] = 0.0
    q = torch.randn((1, 2, 1, D), generator=g, device="cuda").to(torch.bfloat16)
    cache[0][0, 0, 0] = (q[0, 0, 0].sign() * 100).to(torch.int8)
    n = torch.tensor([500], dtype=torch.int32, device="cuda")
    got = kernels.int8_window_decode_attn(q, *cache, n, window=100, sinks=1)
    ref, tol = window_ref(q, cache, [500], [1], 100, 1, "bf16")
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "zero-valued sink")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_q_quant_and_strides(dt):
    """q fake-quantized in the call; q, cache and out as strided views."""
    g = torch.Generator(device="cuda").manual_seed(7)
    B, Hkv, rep, cap = 2, 2, 2, 200
    k8, ksc, v8, vsc = make_cache(g, B, Hkv, cap, "f16")
    lens = [150, 200]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # token-major cache [B, cap, Hkv, D] and scales, q from [B, Sq, Hq, D]
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k8, v8))
    kst = ksc.expand(B, Hkv, 1, D)
    vst = vsc.transpose(1, 2).contiguous().transpose(1, 2)
    q = torch.randn((B, 9, Hkv * rep, D), generator=g, device="cuda").to(TDT[dt]).transpose(1, 2)
    want = kernels.int8_window_prefill_attn(fake_quant(q), k8, ksc, v8, vsc, n, window=60, sinks=2)
    big = torch.zeros((B, 9, Hkv * rep, 2 * D), dtype=TDT[dt], device="cuda")
    out = big[..., D:]
    got = kernels.int8_window_prefill_attn(q, kt, kst, vt, vst, n, window=60, sinks=2, q_quant=True,
                                           out=out)
    assert got is out and torch.equal(out, want) and (big[..., :D] == 0).all()
    d = kernels.int8_window_decode_attn(q[:, :, -1], kt, kst, vt, vst, n, window=60, sinks=2,
                                        q_quant=True)
    ref, tol = window_ref(fake_quant(q)[:, :, -1:], (k8, ksc, v8, vsc), lens, [1, 1], 60, 2, dt)
    check(d, ref[:, 0], tol[:, 0], "decode, strided")
