"""Calls of the ragged-batch operators at the edges of what their documentation allows, on the
GPU.  Bounds as in test_ragged_gpu."""
import math

import pytest
import torch

from halftone_quantizedkvcache_b200 import kernels
from test_ragged_gpu import D, TDT, check, ref_rows

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def late_leader(g, B, Hkv, S, at, rise):
    """Codes and float32 scales of a cache whose early keys (the first 128) have score 0 and V
    scales of 2^7 and whose key ``at`` has, for a query of ones, a score higher by ``rise`` (in
    powers of two) and the V scale of all others, 2^-19."""
    k = torch.zeros((B, Hkv, S, D), dtype=torch.int8, device="cuda")
    k[:, :, at] = 127
    ksc = torch.full((B, Hkv, 1, D), rise * math.log(2) * math.sqrt(D) / (127 * D), device="cuda")
    v = torch.randint(-127, 128, (B, Hkv, S, D), generator=g, device="cuda", dtype=torch.int8)
    vsc = torch.full((B, Hkv, S, 1), 2.0 ** -19, device="cuda")
    vsc[:, :, :128] = 2.0 ** 7
    return k, ksc, v, vsc


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rep", [1, 2, 4, 8])
@pytest.mark.parametrize("at,rise", [(130, 40.0), (300, 40.0), (261, 60.0), (259, 30.0)])
def test_a_late_key_with_small_values_takes_the_lead(rep, dt, at, rise):
    """Keys of large values at low scores, then one of tiny values at a far higher score, in the
    same block: what the early ones needed must not decide how finely the late one is held.
    Float16 outputs below 2^-14, which values this small give, are multiples of 2^-24: rounding
    takes up to 2^-25 there, whatever the value (the bound's eps / 2 |ref| holds above)."""
    g = torch.Generator(device="cuda").manual_seed(rep)
    B, Hkv, S = 200, 2, 512        # 1600 tiles: several of one sequence to a block
    cache = late_leader(g, B, Hkv, S, at, rise)
    q = torch.ones((B, Hkv * rep, 1, D), device="cuda").to(TDT[dt])
    got = kernels.int8_window_decode_attn(q, *cache, i32([S] * B))
    k8, ksc, v8, vsc = (x[:, :, :].double() for x in cache)
    seen = torch.ones((1, S), dtype=torch.bool, device="cuda")
    step = 2.0 ** -25 if dt == "f16" else 0.0
    for b in (0, 1, 57, 198, 199):
        for h in range(Hkv):
            ref, tol = ref_rows(q[b, h * rep], k8[b, h] * ksc[b, h], v8[b, h] * vsc[b, h], seen, dt)
            check(got[b, h * rep:(h + 1) * rep, 0], ref.expand(rep, D), tol.expand(rep, D) + step,
                  f"b={b} h={h}")
    assert kernels.ragged_status() == 0
