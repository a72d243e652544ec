"""Rotary positions with the write to an int8 cache, against the definition in float64.

Codes and V scales are whole-number results of one rounding and must be equal: the reference
forms the same quotients in float64.  q is the rotation rounded to its type: off by half a step
of the value, eps / 2 |q|, plus the error of the rotation itself, 2^-45 of the pair's size in
float64 (float32 inputs) and 2^-21 in float32 (16-bit inputs: cos and sin to 2^-23, two
products and a sum to 2^-24 each, of values up to the pair's size times the factor)."""
import pytest
import torch

from halftone_quantizedkvcache_b200 import kernels

pytestmark = pytest.mark.gpu
TDT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def rotate64(x, pos, inv_freq, inter, factor):
    """x [H, n, D] float64 at positions pos [n]."""
    rot = 2 * len(inv_freq)
    ang = pos.double()[:, None] * inv_freq.double()
    c, s = ang.cos() * factor, ang.sin() * factor
    y = x.clone()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.parametrize("B,Hq,Hkv,S,D,rot,inter,lens,n_new,off,dt,sdt", [
    (1, 16, 8, 1, 128, 128, False, [4000], None, None, "bf16", "f16"),
    (3, 4, 2, 7, 128, 64, True, [0, 100, 57], [7, 0, 3], None, "f16", "f32"),
    (2, 6, 2, 33, 64, 64, False, [1, 0], [33, 20], [1000003, 131072], "f32", "f32"),
    (2, 2, 1, 5, 256, 96, False, [10, 3], None, [7, 0], "bf16", "f32"),
    (1, 3, 3, 4, 128, 20, False, [9], None, None, "f16", "f16"),   # a rotated part off the lanes' grid
    (1, 3, 3, 4, 128, 2, True, [9], None, None, "bf16", "f16"),
    (2, 4, 4, 3, 128, 0, False, [5, 6], None, None, "bf16", "f16"),  # nothing turned
    (40, 2, 1, 50, 128, 128, False, None, None, None, "bf16", "f16"),
])
def test_rope_append(B, Hq, Hkv, S, D, rot, inter, lens, n_new, off, dt, sdt):
    g = torch.Generator(device="cuda").manual_seed(S * 11 + D + rot)
    lens = lens or [(13 * b) % 60 for b in range(B)]
    cap = max(lens) + S + 3
    mk = lambda h: torch.randn((B, h, S, D), generator=g, device="cuda").to(TDT[dt])  # noqa: E731
    q, kn, vn = mk(Hq), mk(Hkv), mk(Hkv)
    vn[:, :, 0] = 0  # an all-zero row
    kc, vc = (torch.full((B, Hkv, cap, D), 77, dtype=torch.int8, device="cuda") for _ in range(2))
    vs = torch.full((B, Hkv, cap, 1), 9.0, device="cuda").to(TDT[sdt])
    ks = (torch.rand((B, Hkv, 1, D), generator=g, device="cuda") * 0.02 + 0.015).to(TDT[sdt])
    inv, factor = kernels.rope_inv_freq(max(rot, 2), 1e6, scaling="linear", factor=2.0)
    inv = inv[:rot // 2].contiguous()
    factor = 1.25
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = kernels.rope_append_kv(q, kn, vn, inv, kc, vc, ks, vs, i32(lens), n_new=i32(n_new),
                                 pos_offset=i32(off), interleaved=inter, factor=factor)
    eps = torch.finfo(TDT[dt]).eps
    for b in range(B):
        n, r0 = (S if n_new is None else n_new[b]), lens[b]
        pos = torch.arange(r0, r0 + n, device="cuda") + (off[b] if off else 0)
        want = rotate64(q[b, :, :n].double(), pos, inv, inter, factor)
        big = q[b, :, :n].double().abs().amax(-1, keepdim=True) * 4
        err = (got[b, :, :n].double() - want).abs()
        assert (err <= eps / 2 * want.abs() + (2.0 ** -45 if dt == "f32" else 2.0 ** -21) * big + torch.finfo(TDT[dt]).tiny).all()
        assert torch.equal(got[b, :, n:], q[b, :, n:])
        kr = rotate64(kn[b, :, :n].double(), pos, inv, inter, factor)
        kw = (kr / ks[b].double()).round().clamp(-127, 127).to(torch.int8)
        assert torch.equal(kc[b, :, r0:r0 + n], kw)
        x = vn[b, :, :n].float()
        sc = x.abs().amax(-1, keepdim=True).clamp(min=1e-8) / torch.full((), 127.0, device="cuda")
        assert torch.equal(vc[b, :, r0:r0 + n], (x / sc).round().clamp(-127, 127).to(torch.int8))
        assert torch.equal(vs[b, :, r0:r0 + n], sc.to(TDT[sdt]))
        for t, fill in ((kc, 77), (vc, 77), (vs, 9.0)):  # other rows stay as they were
            assert (t[b, :, :r0] == fill).all() and (t[b, :, r0 + n:] == fill).all()
    assert kernels.ragged_status() == 0


def test_rope_in_place_broadcast_scale_and_views():
    """q_out = q, one K scale for every sequence, q / k / v as views of one projection."""
    g = torch.Generator(device="cuda").manual_seed(3)
    B, Hq, Hkv, S, D = 2, 4, 2, 5, 128
    x = torch.randn((B, S, Hq + 2 * Hkv, D), generator=g, device="cuda").to(torch.bfloat16)
    q, kn, vn = (t.transpose(1, 2) for t in x.split([Hq, Hkv, Hkv], 2))
    ks = torch.rand((1, Hkv, 1, D), generator=g, device="cuda") * 0.02 + 0.015
    inv, _ = kernels.rope_inv_freq(D)
    lens = torch.tensor([3, 0], dtype=torch.int32, device="cuda")

    def bufs():
        return (torch.zeros((B, 9, Hkv, D), dtype=torch.int8, device="cuda").transpose(1, 2),
                torch.zeros((B, 9, Hkv, D), dtype=torch.int8, device="cuda").transpose(1, 2),
                torch.zeros((B, 9, Hkv, 1), device="cuda").transpose(1, 2))

    a, c = bufs(), bufs()
    want = kernels.rope_append_kv(q.contiguous(), kn.contiguous(), vn.contiguous(), inv, a[0], a[1],
                                  ks.expand(B, Hkv, 1, D).contiguous(), a[2], lens)
    got = kernels.rope_append_kv(q, kn, vn, inv, c[0], c[1], ks, c[2], lens, q_out=q)
    assert got is q and torch.equal(q, want)
    assert all(torch.equal(s, t) for s, t in zip(a, c))


def test_rope_full_sequence_writes_nothing_and_reports():
    B, H, S, D, cap = 3, 1, 4, 128, 8
    q = torch.randn((B, H, S, D), device="cuda").to(torch.bfloat16)
    kc, vc = (torch.full((B, H, cap, D), 5, dtype=torch.int8, device="cuda") for _ in range(2))
    vs = torch.ones((B, H, cap, 1), device="cuda")
    ks = torch.ones((B, H, 1, D), device="cuda") * 0.03
    inv, _ = kernels.rope_inv_freq(D)
    lens = torch.tensor([5, 4, -1], dtype=torch.int32, device="cuda")
    kernels.reset_ragged_status()
    kernels.rope_append_kv(q, q, q, inv, kc, vc, ks, vs, lens)
    assert kernels.ragged_status() == -1
    kernels.reset_ragged_status()
    assert kernels.ragged_status() == 0
    for b in (0, 2):
        assert (kc[b] == 5).all() and (vc[b] == 5).all() and (vs[b] == 1).all()
    assert (kc[1, :, 4:] != 5).any() and (kc[1, :, :4] == 5).all()
