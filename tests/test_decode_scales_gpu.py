"""Decode over int8 caches whose V scales differ by many powers of two, on the GPU, against the
definition in float64.

Tolerance, from the arithmetic of the int8 tensor-core kernels.  Write z_j for the scores in powers
of two, p_j for the softmax (its largest divided out), w_j = p_j v_scale_j.  q' is held in 24 bits
(8355711 steps to its largest value Q): scores are off by 128 * 127 * Q / (2 * 8355711) <= Q 2^-10,
and by four float32 roundings of z and exp2's 2^-22, so p_j by a relative
dz = Q 2^-10 + 2^-22 (1 + max |z|), and a normalised sum by 2 dz A, A = sum p_j |v_j|.  w_j is held
in steps of at most 2^-18 of the largest w seen at the same maximum (a scale chosen at twice the
largest w, kept while that falls to a sixteenth): off by min(w_j, 2^-19 max w), times codes up to
127.  The output adds half a step of its type, float16 no less than 2^-25.
"""
import math

import pytest
import torch

from halftone_quantizedkvcache_b200 import kernels

pytestmark = pytest.mark.gpu
TDT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
D, B, HKV, S = 128, 200, 2, 512     # 400 (sequence, kv head) units: each block walks whole sequences


def late_leader(at, rise):
    """Early keys (the first 128) at score 0 with V scales of 2^7, and key ``at``, whose score for a
    query of ones is higher by ``rise`` (powers of two), with the V scale of all others, 2^-19."""
    g = torch.Generator(device="cuda").manual_seed(at)
    k = torch.zeros((B, HKV, S, D), dtype=torch.int8, device="cuda")
    k[:, :, at] = 127
    ksc = torch.full((B, HKV, 1, D), rise * math.log(2) * math.sqrt(D) / (127 * D), device="cuda")
    v = torch.randint(-127, 128, (B, HKV, S, D), generator=g, device="cuda", dtype=torch.int8)
    vsc = torch.full((B, HKV, S, 1), 2.0 ** -19, device="cuda")
    vsc[:, :, :128] = 2.0 ** 7
    return k, ksc, v, vsc


def check(got, cache, rep, dt, rise):
    """got [B,Hq,D] against float64; every query row is ones."""
    k, ksc, v, vsc = cache
    z = (k[0, 0].double() * ksc[0, 0].double()).sum(-1) / (math.sqrt(D) * math.log(2))  # all units alike
    p = torch.exp2(z - z.max())
    for b in (0, 1, 57, 198, 199):
        for h in range(HKV):
            w = (p / p.sum()) * vsc[b, h, :, 0].double()
            ref = w @ v[b, h].double()
            a = w @ v[b, h].double().abs()
            dz = rise / (127 * D) * 2.0 ** -10 + 2.0 ** -22 * (1 + rise)
            step = torch.minimum(w, 2.0 ** -19 * w.max()).sum() * 127
            tol = (torch.finfo(TDT[dt]).eps / 2 * ref.abs() + 2 * dz * a + step
                   + (2.0 ** -25 if dt == "f16" else 0.0))
            err = (got[b, h * rep:(h + 1) * rep].double() - ref).abs()
            assert (err <= tol).all(), (b, h, (err / tol).max().item())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rep", [1, 2, 4])
@pytest.mark.parametrize("at,rise", [(130, 40.0), (300, 40.0), (261, 60.0), (259, 30.0)])
def test_a_late_key_with_small_values_takes_the_lead(rep, dt, at, rise):
    """Keys of large values at low scores, then one of tiny values at a far higher score, in the
    same block: what the early ones needed must not decide how finely the late one is held."""
    cache = late_leader(at, rise)
    q = torch.ones((B, HKV * rep, D), device="cuda").to(TDT[dt])
    check(kernels.int8_decode_attn(q, *cache), cache, rep, dt, rise)
    check(kernels.int8_decode_attn(q, *cache, dynamic_tiles=True), cache, rep, dt, rise)
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    check(kernels.int8_decode_attn(q, *cache, seq_len=n), cache, rep, dt, rise)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rep", [1, 2, 4])
@pytest.mark.parametrize("at,rise", [(130, 40.0), (300, 40.0), (261, 60.0), (259, 30.0)])
def test_the_same_in_the_block_wise_layout(rep, dt, at, rise):
    cache = late_leader(at, rise)
    k, ksc, v, vsc = cache
    blocks = kernels.kblock_alloc(B, HKV, S, D, dtype=TDT[dt], v_scale_dtype=torch.float32)
    blocks["k"].copy_(k)
    blocks["k_scale"].copy_(ksc.expand(B, HKV, S // 128, D))
    blocks["v"].copy_(v)
    blocks["v_scale"].copy_(vsc[..., 0])
    q = torch.ones((B, HKV * rep, D), device="cuda").to(TDT[dt])
    check(kernels.kblock_decode(q, blocks, S), cache, rep, dt, rise)
    n = torch.tensor([S], dtype=torch.int32, device="cuda")
    check(kernels.kblock_decode(q, blocks, S, seq_len=n), cache, rep, dt, rise)
