"""Decode with up to 4 query rows per kv head, on the GPU, held to its own arithmetic: q' and P v_scale
in 24-bit fixed point (three int8 digits), exact integer sums, float32 for the rest.

Tolerance.  With c_jd the K codes, q'_d = q_d k_scale_d / sqrt(D) / ln 2, Q its largest |q'_d|, a score
z_j (in powers of two) is off by sum_d |c_jd| Q / (2 * 8355711) (q' held in 8355711 steps to Q, zeros
exactly), by q' itself (its three float32 products: 2^-22 sum_d |q'_d c_jd|) and by its float32 sums
(as much again); exp2 adds a relative 2^-22 and z - m's rounding 2^-24 |z|.  A normalised sum moves by at
most 2 ln 2 max_j dz_j A, A = sum_j p_j |v_j|.  w_j = p_j v_scale_j is held in steps of 2 max w / 8355711,
so off by half of that times |code_j|; float32 sums of O and l: 2^-20 A.  The output adds half a step of
its type (float16: no less than 2^-25).  In channels where the output nearly cancels this is far below
the 2^-11 A of the float16 kernel, and a lost digit shows."""
import math

import pytest
import torch

from halftone_quantizedkvcache_b200 import kernels

TDT = {"bf16": torch.bfloat16, "f16": torch.float16}
D = 128
STEPS = 8355711


def reference(q, k8, ksc, v8, vsc, dt):
    """float64 output and bound of rows q [R,D] over one head's codes [S,D] and scales [D], [S]."""
    qs = q.double() * ksc.double() / (math.sqrt(D) * math.log(2))
    k, v = k8.double(), v8.double()
    z = qs @ k.T
    p = torch.exp2(z - z.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    w = p * vsc.double()
    out, a = w @ v, w @ v.abs()
    big = qs.abs().amax(-1, keepdim=True)
    dz = big / (2 * STEPS) * ((qs != 0).double() @ k.abs().T) + 2.0 ** -21 * (qs.abs() @ k.abs().T)
    dz = (dz + 2.0 ** -24 * z.abs()).amax(-1, keepdim=True) + 2.0 ** -22
    tol = 2 * math.log(2) * dz * a + w.amax(-1, keepdim=True) / STEPS * v.abs().sum(0) + 2.0 ** -20 * a
    tol = tol + torch.finfo(TDT[dt]).eps / 2 * out.abs() + (2.0 ** -25 if dt == "f16" else 0.0)
    return out, tol


def inputs(dev, S, rep, dt, flat, B=16, Hkv=4):
    g = torch.Generator(device=dev).manual_seed(S + rep)
    k8, v8 = (torch.randint(-127, 128, (B, Hkv, S, D), generator=g, device=dev, dtype=torch.int8)
              for _ in range(2))
    ksc = torch.rand((B, Hkv, 1, D), generator=g, device=dev) * 0.02 + 0.01
    vsc = torch.rand((B, Hkv, S, 1), generator=g, device=dev) * 0.02 + 0.01
    q = torch.randn((B, Hkv * rep, 1, D), generator=g, device=dev).to(TDT[dt])
    return torch.zeros_like(q) if flat else q, k8, ksc, v8, vsc


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rep", [1, 2, 3, 4])
@pytest.mark.parametrize("S,flat", [(2, False), (2, True), (64, False), (64, True), (300, True), (700, False)])
def test_digits(S, rep, dt, flat):
    """flat: a query of zeros, whose weights are the V scales alone."""
    q, k8, ksc, v8, vsc = inputs("cuda", S, rep, dt, flat)
    B, Hkv = k8.shape[:2]
    n = torch.full((B,), S, dtype=torch.int32, device="cuda")
    got = kernels.int8_window_decode_attn(q, k8, ksc, v8, vsc, n)
    shared = kernels.int8_prefix_decode_attn(q[:1], k8[:1], ksc[:1], v8[:1], vsc[:1], k8[:1, :, :0], ksc[:1],
                                             v8[:1, :, :0], vsc[:1, :, :0], n[:1] * 0)
    for b in range(B):
        for h in range(Hkv):
            rows = slice(h * rep, (h + 1) * rep)
            ref, tol = reference(q[b, rows, 0], k8[b, h], ksc[b, h, 0], v8[b, h], vsc[b, h, :, 0], dt)
            for x in [got[b, rows, 0]] + ([shared[0, rows, 0]] if b == 0 else []):
                err = (x.double() - ref).abs()
                assert (err <= tol).all(), (b, h, (err / tol).max().item())


def fixed_point(q, k8, ksc, v8, vsc, steps_q, steps_p):
    """The kernel's arithmetic with q' and w in the given numbers of steps, the rest exact."""
    qs = q.double() * ksc.double() / (math.sqrt(D) * math.log(2))
    big = qs.abs().amax(-1, keepdim=True).clamp(min=1e-300)
    z = ((qs / big * steps_q).round() / steps_q * big) @ k8.double().T
    p = torch.exp2(z - z.amax(-1, keepdim=True))
    w = p * vsc.double()
    top = 2 * w.amax(-1, keepdim=True)
    return ((w / top * steps_p).round() / steps_p * top) @ v8.double() / p.sum(-1, keepdim=True)


@pytest.mark.parametrize("rep", [1, 4])
def test_the_bound_sees_a_lost_digit(rep):
    """On the CPU: 24 bits keep the bound, 16 on either side do not."""
    lost = {"q": 0.0, "p": 0.0}
    for S, flat in ((2, False), (64, True)):
        q, k8, ksc, v8, vsc = inputs("cpu", S, rep, "f16", flat)
        for b in range(k8.shape[0]):
            for h in range(k8.shape[1]):
                at = (q[b, h * rep:(h + 1) * rep, 0], k8[b, h], ksc[b, h, 0], v8[b, h], vsc[b, h, :, 0])
                ref, tol = reference(*at, "f16")
                worst = lambda a, c: ((fixed_point(*at, a, c).half().double() - ref).abs() / tol).max().item()  # noqa: E731
                assert worst(STEPS, STEPS) <= 1
                lost["q"] = max(lost["q"], worst(STEPS >> 8, STEPS))
                lost["p"] = max(lost["p"], worst(STEPS, STEPS >> 8))
    assert lost["q"] > 1 and lost["p"] > 1, lost
