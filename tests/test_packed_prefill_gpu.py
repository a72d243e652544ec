"""Attention of packed sequences over 16-bit K and V on a GPU, against the formula in float64."""
import math

import pytest
import torch

import paged4_plain as plain

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
D = 128


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cum(v):
    return ints([0] + torch.tensor(v).cumsum(0).tolist())


def seen_of(n, m, causal):
    i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")
    return (j <= m - n + i) if causal else (j >= 0).expand(n, m)


def check(out, q, k, v, nq, nk, causal=True, scale=None):
    rep = q.shape[1] // k.shape[1]
    half = torch.finfo(out.dtype).eps / 2
    a = c = 0
    for n, m in zip(nq, nk):
        qq, kk, vv = (x.transpose(0, 1) for x in (q[a:a + n], k[c:c + m], v[c:c + m]))
        ref, mag = plain.attend(qq, kk.repeat_interleave(rep, 0), vv.repeat_interleave(rep, 0), seen_of(n, m, causal), scale)
        # each weight is rounded to the type (half a step of itself), the output once more; float32
        # scores are off by 2^-21 of sum |q k| <= 16 x 11, the weights twice that: 2^-13 at most.
        err = (out[a:a + n].transpose(0, 1).double() - ref).abs()
        bad = ~(err <= half * ref.abs() * 1.01 + (half + 2.0 ** -13) * mag)
        assert not bad.any(), (n, m, int(bad.sum()), float(err.max()))
        a, c = a + n, c + m


def make(nq, nk, Hkv, rep, dt, seed, extra=0):
    g = gen(seed)
    q = torch.randn((sum(nq) + extra, Hkv * rep, D), generator=g, device="cuda").to(dt)
    k, v = (torch.randn((sum(nk) + extra, Hkv, D), generator=g, device="cuda").to(dt) for _ in range(2))
    return q, k, v


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nq,nk,Hkv,rep", [
    ([1], None, 1, 1), ([128], None, 2, 1), ([129, 1], None, 1, 2), ([512], None, 8, 2),
    ([5, 0, 300, 77, 1], None, 2, 3), ([1000], None, 1, 8), ([64, 65, 63], None, 2, 4),
    ([20, 48, 77], [1020, 2600, 4099], 2, 6), ([1, 1, 1], [1, 700, 129], 4, 2), ([257, 30], [600, 30], 1, 1),
    ([40, 10], [8, 0], 2, 2), ([0, 0, 3], [5, 0, 3], 1, 2), ([2100, 900], None, 2, 2), ([3], [3], 1, 100),
])
def test_causal(dtype, nq, nk, Hkv, rep):
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v = make(nq, nk or nq, Hkv, rep, DT[dtype], 31)
    out = kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk) if nk else None)
    check(out, q, k, v, nq, nk or nq)
    assert kernels.ragged_status() == 0
    assert torch.equal(out, kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk) if nk else None))


@pytest.mark.parametrize("nq,nk,Hkv,rep", [([100, 7], [50, 700], 2, 2), ([300], [300], 1, 3), ([9], [0], 1, 1)])
def test_without_mask_and_with_a_scale(nq, nk, Hkv, rep):
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v = make(nq, nk, Hkv, rep, torch.bfloat16, 5)
    check(kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk), causal=False, sm_scale=0.03), q, k, v, nq, nk, False, 0.03)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_scores_and_a_maximum_that_keeps_growing(dtype):
    """Scores that rise from key to key, so that every tile moves the maximum; then ones that fall."""
    from halftone_quantizedkvcache_b200 import kernels
    n = 700
    q, k, v = make([n], [n], 1, 2, DT[dtype], 6)
    for ramp in (torch.linspace(-30, 30, n, device="cuda"), torch.linspace(30, -30, n, device="cuda")):
        k2 = k.clone()
        k2[:, 0, 0] = ramp.to(k.dtype)
        q2 = q.clone()
        q2[..., 0] = 20.0
        out = kernels.packed_prefill_attn(q2, k2, v, cum([n]))
        rows = plain.attend(q2.transpose(0, 1), k2.transpose(0, 1).repeat_interleave(2, 0), v.transpose(0, 1).repeat_interleave(2, 0), seen_of(n, n, True))
        half = torch.finfo(out.dtype).eps / 2
        err = (out.transpose(0, 1).double() - rows[0]).abs()
        # sum |q k| up to 700 here: 2^-21 x 700 / 11 x 2 of the weights, 2^-14
        assert (err <= half * rows[0].abs() * 1.01 + (half + 2.0 ** -13) * rows[1]).all()


def test_rows_behind_the_last_sequence_and_out():
    from halftone_quantizedkvcache_b200 import kernels
    nq = [70, 33]
    q, k, v = make(nq, nq, 2, 2, torch.bfloat16, 4, extra=9)
    q[103:], k[103:], v[103:] = math.nan, math.nan, math.inf
    out = kernels.packed_prefill_attn(q, k, v, cum(nq))
    assert (out[103:] == 0).all()
    check(out, q, k, v, nq, nq)
    buf = torch.full((112, 8, D), 2.5, dtype=torch.bfloat16, device="cuda")
    kernels.packed_prefill_attn(q, k, v, cum(nq), out=buf[:, ::2])
    assert torch.equal(buf[:103, ::2], out[:103]) and (buf[103:] == 2.5).all() and (buf[:, 1::2] == 2.5).all()
    assert (kernels.packed_prefill_attn(q, k, v, ints([0])) == 0).all()
    # rows before the first sequence
    ahead = kernels.packed_prefill_attn(q, k, v, ints([70, 103]), ints([70, 103]))
    assert (ahead[:70] == 0).all() and (ahead[103:] == 0).all() and torch.equal(ahead[70:103], out[70:103])
    assert kernels.packed_prefill_attn(q[:0], k, v, ints([0, 0]), ints([0, 5])).shape == (0, 4, D)
    assert (kernels.packed_prefill_attn(q, k[:0], v[:0], cum(nq), ints([0, 0, 0])) == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_that_are_no_numbers_stay_with_the_rows_that_see_them(dtype):
    from halftone_quantizedkvcache_b200 import kernels
    nq = [200, 300]
    q, k, v = make(nq, nq, 2, 2, DT[dtype], 14)
    ref = kernels.packed_prefill_attn(q, k, v, cum(nq))
    for where, bad in (("k", math.nan), ("v", math.nan), ("v", math.inf), ("v", -math.inf)):
        k2, v2 = k.clone(), v.clone()
        (k2 if where == "k" else v2)[150, 1, 77] = bad       # sequence 0, key 150, head 1
        (k2 if where == "k" else v2)[200 + 260, 0, 5] = bad  # sequence 1, key 260, head 0
        out = kernels.packed_prefill_attn(q, k2, v2, cum(nq))
        hit = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
        hit[150:200, 2:], hit[460:, :2] = True, True
        assert out[hit].isnan().any(-1).all() if where == "v" else out[hit].isnan().all()
        assert torch.equal(out[~hit], ref[~hit]), where


def test_strides():
    from halftone_quantizedkvcache_b200 import kernels
    nq = [130, 61]
    g = gen(17)
    qkv = torch.randn((191, 8 * D), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([4 * D, 2 * D, 2 * D], 1))
    dense = [x.contiguous() for x in (q, k, v)]
    ref = kernels.packed_prefill_attn(*dense, cum(nq))
    assert torch.equal(kernels.packed_prefill_attn(q, k, v, cum(nq)), ref)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in dense]
    assert torch.equal(kernels.packed_prefill_attn(*heads_first, cum(nq)), ref)
    assert torch.equal(kernels.packed_prefill_attn(dense[0], heads_first[1], dense[2], cum(nq)), ref)
    wide = torch.randn((191, 2, 2 * D + 4), generator=g, device="cuda").to(torch.bfloat16)
    wide[..., 4:D + 4] = dense[1]
    assert torch.equal(kernels.packed_prefill_attn(dense[0], wide[..., 4:D + 4], dense[2], cum(nq)), ref)
    one = dense[1][:, :1].expand(191, 2, D)
    assert torch.equal(kernels.packed_prefill_attn(dense[0], one, dense[2], cum(nq)),
                       kernels.packed_prefill_attn(dense[0], one.contiguous(), dense[2], cum(nq)))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,m", [(1, 4096), (64, 900), (300, 9000)])
def test_many_small_weights_beside_a_large_one(dtype, n, m):
    # key 0 has weight 1, each other 2^-25.4, which float16 would round to nothing: together they carry
    # V.  float16's weights lose at most 2^-32 of the largest each.
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v = (torch.zeros((x, 1, D), device="cuda") for x in (n, m, m))
    q[:, :, 3], k[0, :, 3] = 16.0, 25.4 * math.log(2.0) / 16.0 * math.sqrt(D)
    v[1:] = 4096.0
    q, k, v = (x.to(DT[dtype]) for x in (q, k, v))
    out = kernels.packed_prefill_attn(q, k, v, cum([n]), cum([m]), causal=False)
    ref, mag = plain.attend(*(x.transpose(0, 1) for x in (q, k, v)), seen_of(n, m, False), None)
    half = torch.finfo(DT[dtype]).eps / 2
    err = (out.transpose(0, 1).double() - ref).abs()
    assert float(ref.min()) > 0.05
    assert not (~(err <= half * ref.abs() * 1.01 + (half + 2.0 ** -13) * mag + 2.0 ** -32 * m * 4096)).any(), float(err.max())


def test_queries_that_share_memory_and_neighbours_that_are_no_numbers():
    from halftone_quantizedkvcache_b200 import kernels
    nq = [5, 130, 60]
    for rep in (2, 3, 128):
        q, k, v = make(nq, nq, 1, rep, torch.bfloat16, 9)
        for shared in (q[:, :1].expand_as(q), q[:1].expand_as(q)):
            out = kernels.packed_prefill_attn(shared, k, v, cum(nq))
            assert torch.equal(out, kernels.packed_prefill_attn(shared.contiguous(), k, v, cum(nq)))
        out = kernels.packed_prefill_attn(q, k, v, cum(nq))
        q[5:135], k[5:135], v[5:135] = math.nan, math.inf, math.nan
        bad = kernels.packed_prefill_attn(q, k, v, cum(nq))
        assert torch.equal(bad[:5], out[:5]) and torch.equal(bad[135:], out[135:]) and bad[5:135].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,m", [(250, 250), (4, 1024), (5, 1000), (256, 1024)])
def test_short_sequences_with_a_maximum_that_keeps_growing(dtype, n, m):
    # blocks of one row tile, a row's keys shared by two threads; their keys split over blocks or not
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v = make([n], [m], 1, 2, DT[dtype], 26)
    for ramp in (torch.linspace(-30, 30, m, device="cuda"), torch.linspace(30, -30, m, device="cuda")):
        k[:, 0, 0] = ramp.to(k.dtype)
        q[..., 0] = 20.0
        # (sum |q k| up to 700, as above)
        check(kernels.packed_prefill_attn(q, k, v, cum([n]), cum([m])), q, k, v, [n], [m])
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nq,nk,Hkv,rep", [
    ([600], [500], 8, 2), ([1100, 600], [700, 470], 8, 1), ([2010], [100], 4, 8), ([700, 900, 3], [532, 0, 3], 2, 4),
    ([650], [500], 3, 3),
])
def test_blocks_whose_first_row_tile_sees_no_key(dtype, nq, nk, Hkv, rep):
    # More queries than keys: in some block of two row tiles the first one's rows see nothing, the second's do.
    # The zeros of the first leave by the memory that its Q is copied to.
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v = make(nq, nk, Hkv, rep, DT[dtype], 37)
    blind = torch.cat([torch.arange(n, device="cuda") < n - m for n, m in zip(nq, nk)])
    first = kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk))
    check(first, q, k, v, nq, nk)
    for _ in range(50):
        out = kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk))
        assert (out[blind] == 0).all()
        assert torch.equal(out, first)
    assert kernels.ragged_status() == 0
