"""The paged 4-bit cache on a GPU against plain float64 forms: append (norms, rotation, codes), decode,
gather."""
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


def near(got, ref, extra):
    """Half a step of the output's type, and `extra` for the arithmetic before it."""
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bad = ~(err <= half * ref.abs() * 1.01 + extra)
    assert not bad.any(), (int(bad.sum()), float((err - half * ref.abs()).max()))


# ---------------------------------------------------------------- append
def append_case(new, past, Hkv, rep, dt, page, seed, fused=True):
    g = gen(seed)
    T, B = sum(new), len(new)
    x = torch.randn((T, (rep + 2) * Hkv * D), generator=g, device="cuda").to(dt)
    q, k, v = (y.unflatten(1, (-1, D)) for y in x.split([rep * Hkv * D, Hkv * D, Hkv * D], 1))
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    from halftone_quantizedkvcache_b200 import kernels
    per = max(1, -(-max(a + b for a, b in zip(new, past)) // page))
    cache = plain.random_cache(kernels, B * per + 3, Hkv, page, g)
    tables = plain.random_tables(B, per, B * per + 3, g)
    return q, k, v, cache, tables


def check_append(q, k, v, cache, tables, new, past, before, q_got, k_got, inv, weights, inter=False,
                 factor=1.0, offset=None, eps=1e-6):
    """Every byte of the cache and every row of q and k."""
    dev, page = q.device, cache["k"].shape[2]
    b = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
    i = torch.cat([torch.arange(n, device=dev) for n in new]) if sum(new) else torch.zeros(0, dtype=torch.long, device=dev)
    at = torch.tensor(past, device=dev)[b] + i
    pos = at + (offset.long()[b] if offset is not None else 0)
    qw, kw = weights if weights is not None else (None, None)
    n = len(at)
    q64 = plain.turned(q[:n], qw, pos, inv, inter, factor, eps)
    k64 = plain.turned(k[:n], kw, pos, inv, inter, factor, eps)
    # the float32 route: 2^-20 of |x w| + |o w_o| (paged4_append.cu), normed rows below 12 x 2 x 2
    size = 48.0 if weights is not None else 2.0 * float(k.abs().max()) + 2.0 * float(q.abs().max())
    near(q_got[:n], q64, 1e-6 * size * abs(factor))
    if k_got is not None:
        near(k_got[:n], k64, 1e-6 * size * abs(factor))
    pg, t = tables.long()[b, at // page], at % page
    for name, x in (("k", k64), ("v", v[:n].double())):
        codes, sc = plain.coded(x)
        rows = before[name].clone()
        scales = before[name + "_scale"].clone()
        byte, sh = plain.byte_of(t, dev)
        row = torch.zeros((n, x.shape[1], 64), dtype=torch.int64, device=dev)
        row.scatter_add_(2, byte[:, None].expand(-1, x.shape[1], -1), (codes + 8) << sh)
        rows[pg, :, t], scales[pg, :, t] = row.to(torch.uint8), sc
        assert torch.equal(cache[name + "_scale"].view(torch.int16), scales.view(torch.int16)), name
        assert torch.equal(cache[name], rows), (name, int((cache[name] != rows).sum()))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new,past,Hkv,rep,page,rot,inter,norm", [
    ([1], [0], 8, 2, 64, 128, False, True),
    ([1], [4001], 1, 1, 16, 128, True, True),
    ([1, 1, 1], [63, 64, 65], 2, 4, 64, 64, False, False),
    ([5, 0, 17, 1], [0, 9, 31, 254], 4, 3, 32, 96, True, True),
    ([300, 211], [7, 1000], 8, 2, 128, 128, False, True),
    ([77, 33], [3, 0], 2, 6, 256, 32, False, False),
    ([40, 9], [3, 0], 3, 1, 16, 0, False, True),
    ([40, 9], [3, 0], 3, 1, 16, 0, False, False),
    ([2000], [0], 4, 2, 64, 128, False, True),
])
def test_append(dtype, new, past, Hkv, rep, page, rot, inter, norm):
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v, cache, tables = append_case(new, past, Hkv, rep, DT[dtype], page, 11)
    before = {n: x.clone() for n, x in cache.items()}
    inv = kernels.rope_inv_freq(rot, 1e6)[0] if rot else None
    g = gen(5)
    w = [torch.empty(D, device="cuda").uniform_(0.2, 2.0, generator=g).to(DT[dtype]) for _ in range(2)] if norm else None
    k_out = torch.zeros_like(k, memory_format=torch.contiguous_format)
    got = kernels.paged4_append(q, k, v, cache, tables, ints(past), cu_seqlens=cum(new), inv_freq=inv,
                                interleaved=inter, q_weight=w and w[0], k_weight=w and w[1], k_out=k_out)
    check_append(q, k, v, cache, tables, new, past, before, got, k_out, inv, w, inter)
    assert kernels.ragged_status() == 0


def test_append_without_starts_far_positions_and_float32_weights():
    from halftone_quantizedkvcache_b200 import kernels
    new, past = [1] * 7, [0, 5, 100, 3, 64, 63, 1]
    q, k, v, cache, tables = append_case(new, past, 4, 2, torch.bfloat16, 16, 3, fused=False)
    before = {n: x.clone() for n, x in cache.items()}
    inv, factor = kernels.rope_inv_freq(128, 1e4, scaling="yarn", factor=4.0, original_len=4096)
    off = ints([0, 1 << 20, 999_983, 131_072, 1, 2, 2_000_003])
    w = [torch.rand(D, device="cuda", generator=gen(1)) + 0.5 for _ in range(2)]
    q0 = q.clone()
    got = kernels.paged4_append(q, k, v, cache, tables, ints(past), inv_freq=inv, factor=factor,
                                pos_offset=off, q_weight=w[0], k_weight=w[1], eps=1e-5, q_out=q)
    assert got is q
    check_append(q0, k, v, cache, tables, new, past, before, got, None, inv, w, False, factor, off, 1e-5)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_append_values_of_every_kind(dtype):
    """Zeros, subnormals, the largest values, exact ties of x / s: all as the float64 form has them."""
    from halftone_quantizedkvcache_b200 import kernels
    dt = DT[dtype]
    q, k, v, cache, tables = append_case([64], [0], 2, 1, dt, 64, 4, fused=False)
    for x in (k, v):
        x[0] = 0
        x[1] *= torch.finfo(dt).tiny
        x[2] = (x[2].sign() * 60000.0 * torch.rand_like(x[2].float())).to(dt)
        x[3] *= 1e-6
        # s = 2^-3 exactly, every quotient k / 2: ties at the odd ones
        x[4] = (torch.arange(D, device="cuda") % 31 - 15).to(dt) / 16
        x[4, :, ::32] = 7.5 / 8
        x[5] = x[4] * 1024
        x[6, :, 32:64] = 0
        x[7, :, 3] *= 300
    before = {n: x.clone() for n, x in cache.items()}
    got = kernels.paged4_append(q, k, v, cache, tables, ints([0]), cu_seqlens=ints([0, 64]))
    assert torch.equal(got, q)
    check_append(q, k, v, cache, tables, [64], [0], before, got, None, None, None)


def test_append_scale_beyond_float16_saturates():
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v, cache, tables = append_case([2], [0], 1, 1, torch.bfloat16, 16, 4, fused=False)
    v[0] = 1e6 * v[0].sign()
    v[1, 0, 40] = math.inf
    k[1, 0, 100] = math.nan
    kernels.paged4_append(q, k, v, cache, tables, ints([0]), cu_seqlens=ints([0, 2]))
    kv, vv = kernels.paged4_gather(cache, tables, ints([2]), ints([0, 2]), 2, dtype=torch.bfloat16)
    assert torch.equal(vv[0], (torch.where(v[0] < 0, -8.0, 7.0) * 65504.0).to(torch.bfloat16))
    # a group that holds no number says so, the others of its row do not care
    assert vv[1, 0, 32:64].isnan().all() and vv[1, 0, :32].isfinite().all() and vv[1, 0, 64:].isfinite().all()
    assert kv[1, 0, 96:].isnan().all() and kv[1, 0, :96].isfinite().all()


def test_append_that_does_not_fit_writes_nothing():
    from halftone_quantizedkvcache_b200 import kernels
    new, past = [4, 3, 2], [13, 0, 5]
    q, k, v, cache, tables = append_case(new, [0, 0, 0], 2, 2, torch.bfloat16, 16, 9)   # 16 places each
    before = {n: x.clone() for n, x in cache.items()}
    kernels.reset_ragged_status()
    tables[2, 0] = cache["k"].shape[0]           # no page of the cache
    got = kernels.paged4_append(q, k, v, cache, tables, ints(past), cu_seqlens=cum(new))
    assert kernels.ragged_status() == -1
    kernels.reset_ragged_status()
    assert torch.equal(got, q)                   # q is served all the same
    kept = dict(before)
    page = int(tables[1, 0])
    for n in cache:
        other = torch.ones(cache[n].shape[0], dtype=torch.bool, device="cuda")
        other[page] = False
        assert torch.equal(cache[n][other], kept[n][other]), n
        assert not torch.equal(cache[n][page, :, :3], kept[n][page, :, :3])


def test_append_rows_behind_the_last_sequence():
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v, cache, tables = append_case([6, 5], [0, 0], 2, 2, torch.float16, 16, 2)
    inv = kernels.rope_inv_freq(128)[0]
    k_out, q_out = torch.full((11, 2, D), 3.0, dtype=torch.float16, device="cuda"), torch.full((11, 4, D), 5.0, dtype=torch.float16, device="cuda")
    before = {n: x.clone() for n, x in cache.items()}
    kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=ints([0, 6, 9]), inv_freq=inv,
                          q_out=q_out, k_out=k_out)
    assert (q_out[9:] == 5).all() and (k_out[9:] == 3).all()
    check_append(q, k, v, cache, tables, [6, 3], [0, 0], before, q_out, k_out, inv, None)
    got = kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=ints([0, 6, 9]), inv_freq=inv)
    assert torch.equal(got[9:], q[9:]) and torch.equal(got[:9], q_out[:9])
    # and before the first
    q_out.fill_(5)
    kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=ints([4, 4, 9]), inv_freq=inv, q_out=q_out)
    assert (q_out[:4] == 5).all() and (q_out[9:] == 5).all() and not (q_out[4:9] == 5).all()
    assert kernels.ragged_status() == 0
    assert kernels.paged4_append(q[:0], k[:0], v[:0], cache, tables, ints([0, 0]), cu_seqlens=ints([0, 0, 0])).shape == (0, 4, D)


# ---------------------------------------------------------------- decode
def rounded_weights(q, cache, tables, b, n, scale=None):
    """What rounding p x scale to a 16-bit whole number of its tile's largest can do to the output: per
    tile of 64 tokens half a step, 1 / (2 x 32512), of the largest p times the group's largest scale,
    times sum |code|.  q [Hkv, rep, D] -> [Hkv, rep, D]."""
    Hkv, page = cache["k"].shape[1:3]
    k = plain.values(cache, "k", tables, b, n).transpose(0, 1)
    p = torch.softmax(q.double() @ k.transpose(1, 2) * (scale if scale is not None else 1 / math.sqrt(D)), -1)
    codes, sc = plain.read_codes(cache, "v", *plain.slots(tables, page, b, n))
    pad = -n % 64
    p = torch.nn.functional.pad(p, (0, pad)).unflatten(-1, (-1, 64)).amax(-1)                 # [Hkv, rep, tiles]
    sc = torch.nn.functional.pad(sc.abs().permute(1, 2, 0), (0, pad)).unflatten(-1, (-1, 64)).amax(-1)  # [Hkv, 4, tiles]
    codes = torch.nn.functional.pad(codes.double().abs().permute(1, 2, 0), (0, pad)).unflatten(-1, (-1, 64)).sum(-1)
    return torch.einsum("hrt,hdt,hdt->hrd", p, sc.repeat_interleave(32, 1), codes) / (2 * 32512)


def check_decode(out, q, cache, tables, lens, scale=None):
    Hkv = cache["k"].shape[1]
    for b, n in enumerate(lens):
        k, v = (plain.values(cache, x, tables, b, n).transpose(0, 1) for x in ("k", "v"))
        qq = q[b].view(Hkv, -1, D)
        ref, mag = plain.attend(qq, k, v, torch.ones((1, n), dtype=torch.bool, device="cuda"), scale)
        # Scores: q in steps of 2^-21 of the row's largest |q| (below 5), times sum |k| (below 128 x 1.6),
        # and float32 roundings of sums below 16 x 11: 2^-14 of a weight at most, twice, against sum p |v|.
        near(out[b].view(ref.shape), ref, mag * 2.0 ** -12 + 1.01 * rounded_weights(qq, cache, tables, b, n, scale) if n else mag)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,Hkv,rep,page", [
    ([1], 8, 2, 64), ([31], 1, 1, 16), ([32, 33, 0, 64], 2, 4, 16), ([512], 8, 2, 64),
    ([5, 777, 1300, 2, 0, 129], 4, 3, 32), ([2501, 40, 1], 2, 8, 128), ([300, 301], 1, 5, 256),
    ([100, 17], 2, 16, 64), ([90, 3], 1, 40, 16), ([0, 0], 2, 2, 16), ([9000], 1, 2, 64),
])
def test_decode(dtype, lens, Hkv, rep, page):
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(21)
    per = max(1, -(-max(lens) // page))
    cache = plain.random_cache(kernels, len(lens) * per + 2, Hkv, page, g)
    tables = plain.random_tables(len(lens), per, len(lens) * per + 2, g)
    q = torch.randn((len(lens), Hkv * rep, D), generator=g, device="cuda").to(DT[dtype])
    out = kernels.paged4_decode_attn(q, cache, tables, ints(lens))
    check_decode(out, q, cache, tables, lens)
    assert kernels.ragged_status() == 0
    # the same, bit by bit, on a second run, and as [B, H, 1, D]
    again = kernels.paged4_decode_attn(q[:, :, None], cache, tables, ints(lens))
    assert torch.equal(again[:, :, 0], out)


def test_decode_many_short_sequences():
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(2)
    lens = [(7 * i) % 130 for i in range(1000)]
    cache = plain.random_cache(kernels, 9010, 2, 16, g)
    tables = plain.random_tables(1000, 9, 9010, g)
    q = torch.randn((1000, 4, D), generator=g, device="cuda").to(torch.bfloat16)
    out = kernels.paged4_decode_attn(q, cache, tables, ints(lens))
    check_decode(out[::37], q[::37], cache, tables[::37], lens[::37])
    assert (out[0] == 0).all()


def test_decode_ignores_what_no_token_wrote():
    """Scales behind the last token NaN or infinite, table entries behind the last page no pages."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(8)
    lens, page = [37, 70, 0], 32
    cache = plain.random_cache(kernels, 14, 2, page, g)
    tables = plain.random_tables(3, 4, 14, g)
    q = torch.randn((3, 4, D), generator=g, device="cuda").to(torch.bfloat16)
    ref = kernels.paged4_decode_attn(q, cache, tables, ints(lens))
    for b, n in enumerate(lens):
        pg, t = plain.slots(tables, page, b, 4 * page)
        for name, x in (("k_scale", math.nan), ("v_scale", math.nan), ("k_scale", math.inf), ("v_scale", -math.inf)):
            cache[name][pg[n:], :, t[n:]] = x
            assert torch.equal(kernels.paged4_decode_attn(q, cache, tables, ints(lens)), ref)
    tables[0, 2:], tables[1, 3:], tables[2] = -5, 1 << 30, 99
    assert torch.equal(kernels.paged4_decode_attn(q, cache, tables, ints(lens)), ref)
    assert kernels.ragged_status() == 0
    # lengths past what the table holds end with it
    long = kernels.paged4_decode_attn(q[:1], cache, tables[:1, :1], ints([10 ** 9]))
    assert torch.equal(long, kernels.paged4_decode_attn(q[:1], cache, tables[:1, :1], ints([32])))
    assert (kernels.paged4_decode_attn(q[:1], cache, tables[:1, :0], ints([5])) == 0).all()


def test_decode_seen_scales_that_are_no_numbers_reach_the_output():
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(8)
    cache = plain.random_cache(kernels, 8, 2, 64, g)
    tables = plain.random_tables(2, 3, 8, g)
    q = torch.randn((2, 4, D), generator=g, device="cuda").to(torch.bfloat16)
    cache["k_scale"][int(tables[0, 1]), 0, 5, 2] = math.nan
    cache["v_scale"][int(tables[1, 0]), 1, 9, 1] = math.nan
    out = kernels.paged4_decode_attn(q, cache, tables, ints([150, 150]))
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all()
    assert out[1, 2:, 32:64].isnan().all() and out[1, 2:, :32].isfinite().all() and out[1, :2].isfinite().all()


def test_decode_extremes():
    """Scores far apart (one key takes all), V scales from 2^-24 to 65504, a page that is none."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(13)
    cache = plain.random_cache(kernels, 12, 1, 64, g)
    tables = plain.random_tables(2, 4, 12, g)
    q = (torch.randn((2, 2, D), generator=g, device="cuda") * 40).to(torch.float16)
    cache["v_scale"].copy_(2.0 ** torch.randint(-24, 16, cache["v_scale"].shape, generator=g, device="cuda").float())
    cache["v_scale"].clamp_(max=65504)
    out = kernels.paged4_decode_attn(q, cache, tables, ints([256, 200])).float()
    for b, n in enumerate([256, 200]):
        k, v = (plain.values(cache, x, tables, b, n).transpose(0, 1) for x in ("k", "v"))
        ref, mag = plain.attend(q[b].view(1, 2, D), k, v, torch.ones((1, n), dtype=torch.bool, device="cuda"))
        # 40 times the scores: 40 times the weights' errors.  Below 2^-14 float16's steps are 2^-24 whatever
        # the value, so its rounding is off by up to 2^-25 there.
        err = (out[b].view(ref.shape).double() - ref.clamp(-65504, 65504)).abs()
        extra = mag * 40 * 2.0 ** -12 + 1.01 * rounded_weights(q[b].view(1, 2, D), cache, tables, b, n)
        bad = ~(err <= 2.0 ** -11 * ref.abs() + extra + 2.0 ** -25) & (ref.abs() < 60000)
        assert not bad.any(), (float(err[bad].max()), ref[bad][:4].tolist())
    kernels.reset_ragged_status()
    tables[1, 1] = -1
    ok = kernels.paged4_decode_attn(q, cache, tables, ints([256, 200]))
    assert kernels.ragged_status() == -1
    kernels.reset_ragged_status()
    assert torch.equal(ok[0].float(), out[0])


def test_decode_strides_out_and_scale():
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(3)
    big = plain.random_cache(kernels, 20, 4, 32, g)
    cache = {n: x[4:, 1:3] for n, x in big.items()}      # a slice of a larger pool: other strides
    tables = plain.random_tables(2, 8, 16, g).flip(0)[[0, 1, 0], :5]   # two sequences share their pages
    tables = torch.cat([tables, tables], 1)[:, :5]
    lens = [150, 31, 97]
    q = torch.randn((3, 12, D), generator=g, device="cuda").to(torch.bfloat16)[:, ::2][:, :4]
    out = torch.full((3, 4, 2 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    got = kernels.paged4_decode_attn(q, cache, tables, ints(lens), out=out[..., :D], sm_scale=-0.05)
    assert got.data_ptr() == out.data_ptr() and (out[..., D:] == 7).all()
    check_decode(out[..., :D].contiguous(), q.contiguous(), cache, tables, lens, -0.05)
    odd = torch.randn((3, 4 * D + 1), generator=g, device="cuda").to(torch.bfloat16)[:, 1:].unflatten(1, (4, D))
    assert torch.equal(kernels.paged4_decode_attn(odd, cache, tables, ints(lens)),
                       kernels.paged4_decode_attn(odd.contiguous(), cache, tables, ints(lens)))


# ---------------------------------------------------------------- gather
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,Hkv,page", [([1], 1, 16), ([0, 33, 200], 2, 32), ([700, 5], 8, 64), ([300], 3, 256)])
def test_gather(dtype, lens, Hkv, page):
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(6)
    per = max(1, -(-max(lens) // page))
    cache = plain.random_cache(kernels, len(lens) * per + 2, Hkv, page, g)
    tables = plain.random_tables(len(lens), per, len(lens) * per + 2, g)
    n = sum(lens)
    k, v = kernels.paged4_gather(cache, tables, ints(lens), cum(lens), n + 3, dtype=DT[dtype])
    for got, name in ((k, "k"), (v, "v")):
        ref = torch.cat([plain.values(cache, name, tables, b, m) for b, m in enumerate(lens)])
        # the product of a 4-bit and an 11-bit number is exact in float32, and rounded once
        assert torch.equal(got[:n], ref.float().to(DT[dtype]))
        assert (got[n:] == 0).all()
    # from the second half on, into rows of a larger buffer
    first = [m // 2 for m in lens]
    rows = [m - f for m, f in zip(lens, first)]
    out = [torch.full((n + 3, 2 * Hkv, D), 9.0, dtype=DT[dtype], device="cuda")[:, :Hkv] for _ in range(2)]
    kernels.paged4_gather(cache, tables, ints(lens), cum(rows), n + 3, first=ints(first), k_out=out[0], v_out=out[1])
    for got, name in ((out[0], "k"), (out[1], "v")):
        ref = torch.cat([plain.values(cache, name, tables, b, m)[f:] for b, (m, f) in enumerate(zip(lens, first))])
        assert torch.equal(got[:sum(rows)], ref.float().to(DT[dtype])) and (got[sum(rows):] == 9).all()
    assert kernels.ragged_status() == 0


def test_gather_bad_pages_and_short_rows():
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(6)
    cache = plain.random_cache(kernels, 9, 2, 16, g)
    tables = plain.random_tables(2, 4, 9, g)
    ref = [plain.values(cache, "k", tables, b, 64).float().to(torch.bfloat16) for b in range(2)]
    # fewer rows than tokens: the first ones; more rows than tokens: the others empty
    k, _ = kernels.paged4_gather(cache, tables, ints([64, 10]), ints([0, 20, 50]), 50)
    assert torch.equal(k[:20], ref[0][:20]) and torch.equal(k[20:30], ref[1][:10]) and (k[30:] == 0).all()
    kernels.reset_ragged_status()
    tables[0, 1] = 9
    k, _ = kernels.paged4_gather(cache, tables, ints([40, 10]), ints([0, 40, 50]), 50)
    assert kernels.ragged_status() == -1
    kernels.reset_ragged_status()
    assert torch.equal(k[:16], ref[0][:16]) and (k[16:32] == 0).all() and torch.equal(k[32:40], ref[0][32:40])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("inter,rot", [(False, 128), (True, 128), (False, 96)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_turned_rows_that_hold_no_number(dtype, inter, rot, bad):
    """A channel of K that is no number, in many turned rows (one in 60 is formed in float64 too): its group
    and its partner's have scales that are none, the others what they would have."""
    from halftone_quantizedkvcache_b200 import kernels
    new, page = [2000, 1100], 64
    q, k, v, cache, tables = append_case(new, [0, 0], 4, 1, DT[dtype], page, 15, fused=False)
    g = gen(16)
    T, H = k.shape[:2]
    at = torch.randint(0, D, (T, H), generator=g, device="cuda")
    k.scatter_(2, at[..., None], bad)
    inv = kernels.rope_inv_freq(rot, 1e6)[0]
    kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=cum(new), inv_freq=inv, interleaved=inter)
    half = rot // 2
    other = torch.where(at >= rot, at, at ^ 1 if inter else torch.where(at < half, at + half, at - half))
    hit = torch.zeros((T, H, 4), dtype=torch.bool, device="cuda")
    hit.scatter_(2, at[..., None] // 32, True).scatter_(2, other[..., None] // 32, True)
    b = torch.repeat_interleave(torch.arange(2, device="cuda"), torch.tensor(new, device="cuda"))
    i = torch.cat([torch.arange(n, device="cuda") for n in new])
    codes, sc = plain.read_codes(cache, "k", tables.long()[b, i // page], i % page)
    assert sc[hit].isnan().all(), int((~sc[hit].isnan()).sum())
    # a group's codes are its own affair: zeros in the place of the channels that are no numbers
    k.scatter_(2, at[..., None], 0.0)
    want, wsc = plain.coded(plain.turned(k, None, i, inv, inter, 1.0, 0.0))
    assert torch.equal(sc[~hit], wsc.double()[~hit])
    assert torch.equal(codes.unflatten(-1, (4, 32))[~hit], want.unflatten(-1, (4, 32))[~hit])


def lost_weights(q, cache, tables, b, n, scale=None):
    """What rounding p x scale to a 16-bit whole number does to the output at most: per row, group and tile of
    64 tokens half a step, 1 / (2 x 32512), of the largest p x scale (taken to 2^-8 of itself), times
    sum |code|.  q [Hkv, rep, D] -> [Hkv, rep, D]."""
    page = cache["k"].shape[2]
    k = plain.values(cache, "k", tables, b, n).transpose(0, 1)
    p = torch.softmax(q.double() @ k.transpose(1, 2) * (scale if scale is not None else 1 / math.sqrt(D)), -1)
    codes, sc = plain.read_codes(cache, "v", *plain.slots(tables, page, b, n))
    pad = -n % 64
    top = p[:, :, None] * sc.abs().permute(1, 2, 0)[:, None]                                   # [Hkv, rep, 4, n]
    top = torch.nn.functional.pad(top, (0, pad)).unflatten(-1, (-1, 64)).amax(-1)
    codes = torch.nn.functional.pad(codes.double().abs().permute(1, 2, 0), (0, pad)).unflatten(-1, (-1, 64)).sum(-1)
    return torch.einsum("hrdt,hdt->hrd", top.repeat_interleave(32, 2), codes) * (1 + 2.0 ** -8) / (2 * 32512)


def scored_cache(scores, Hkv, page, seed):
    """One sequence whose token t has the score x scores[t] for a row of q that holds x throughout: all
    codes of K are 7.  V: random codes, scales 0.1 .. 0.4."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(seed)
    n = len(scores)
    per = -(-n // page)
    cache = plain.random_cache(kernels, per + 1, Hkv, page, g)
    tables = plain.random_tables(1, per, per + 1, g)
    cache["k"].fill_(0xff)
    pg, t = plain.slots(tables, page, 0, n)
    cache["k_scale"][pg, :, t] = (torch.tensor(scores, device="cuda").double() / (7 * math.sqrt(D))).half()[:, None, None]
    return cache, tables, pg, t


def check_scored(cache, tables, n, dt, rows):
    """Rows of q that hold one number each, against the formula.  K's scales are the scores' only source."""
    from halftone_quantizedkvcache_b200 import kernels
    Hkv = cache["k"].shape[1]
    q = torch.tensor(rows, device="cuda")[None, None, :, None].expand(1, Hkv, len(rows), D).reshape(1, -1, D).to(dt).contiguous()
    out = kernels.paged4_decode_attn(q, cache, tables, ints([n]))
    k, v = (plain.values(cache, x, tables, 0, n).transpose(0, 1) for x in ("k", "v"))
    qq = q[0].view(Hkv, -1, D)
    ref, mag = plain.attend(qq, k, v, torch.ones((1, n), dtype=torch.bool, device="cuda"))
    # q is a whole number of steps here but for 2^-22 of itself; scores below 80: 2^-13 of a weight at most,
    # twice.  Below its smallest normal number float16's step is 2^-24 whatever the value.
    extra = mag * 2.0 ** -12 + lost_weights(qq, cache, tables, 0, n) + (2.0 ** -25 if dt == torch.float16 else 0.0)
    near(out[0].view(ref.shape), ref, extra)
    assert kernels.ragged_status() == 0
    return out, ref


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Hkv,rows,page", [(1, [1.0], 64), (2, [1.0, 0.5], 16), (1, [1.0, 0.75, 0.5, 0.25, 1.5], 128)])
@pytest.mark.parametrize("ratio", [1e2, 1e3, 1e4, 2.0 ** 18])
def test_decode_a_large_scale_without_weight_takes_no_bits(dtype, Hkv, rows, page, ratio):
    """Tokens that no row heeds (p of 1e-12 and less for x = 1) with V scales `ratio` times those of the token
    that all of them do."""
    n = 200
    scores = [0.0] * n
    heeded = [7, 100, 150, 199]                 # one of each tile
    for t in heeded:
        scores[t] = 28.0
    cache, tables, pg, t = scored_cache(scores, Hkv, page, 41)
    v_scale = torch.full((n,), 2.0 ** -4 if ratio < 2e4 else 2.0 ** -10, device="cuda")
    light = torch.ones(n, dtype=torch.bool, device="cuda")
    light[heeded] = False
    v_scale[light] *= ratio
    cache["v_scale"][pg, :, t] = v_scale.half()[:, None, None]
    check_scored(cache, tables, n, DT[dtype], rows)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Hkv,rows,page", [(1, [1.0], 64), (2, [1.0, 0.5], 16), (1, [1.0, 0.75, 0.5, 0.25, 1.5], 128)])
@pytest.mark.parametrize("sink", [0.0, 2.0 ** -24, 0.002])
@pytest.mark.parametrize("n,far", [(64, 8.0), (500, 12.0), (3000, 20.0)])
def test_decode_beside_a_token_that_takes_the_weight_and_has_no_values(dtype, Hkv, rows, page, sink, n, far):
    """A first token with most of the softmax and V next to nothing, as sinks have it: the others' V is
    what goes out, each with a weight of e^-far."""
    cache, tables, pg, t = scored_cache([40.0] + [40.0 - far] * (n - 1), Hkv, page, 43)
    cache["v_scale"][pg[0], :, t[0]] = sink
    out, ref = check_scored(cache, tables, n, DT[dtype], rows)
    assert float(ref.abs().max()) > 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [64, 1000, 5000])
def test_decode_many_small_weights_beside_a_large_one(dtype, n):
    """Key 0 has weight 1 and codes of zero under a scale like the others', each other key a weight of 2^-11:
    one step in 32512 of 64 tokens' largest is what each may lose, and together they carry V."""
    cache, tables, pg, t = scored_cache([40.0] + [40.0 - 11 * math.log(2.0)] * (n - 1), 1, 64, 44)
    cache["v"][pg[0], :, t[0]] = 0x88
    check_scored(cache, tables, n, DT[dtype], [1.0, 0.5])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_decode_scales_of_all_sizes(dtype):
    """V scales from 2^-24 to 2^8 and scores within ten of each other, all at random."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(45)
    lens = [900, 64, 1, 333]
    cache = plain.random_cache(kernels, 70, 2, 64, g)
    tables = plain.random_tables(4, 15, 70, g)
    cache["v_scale"].copy_(2.0 ** torch.randint(-24, 9, cache["v_scale"].shape, generator=g, device="cuda").float())
    q = torch.randn((4, 6, D), generator=g, device="cuda").to(DT[dtype])
    out = kernels.paged4_decode_attn(q, cache, tables, ints(lens))
    for b, n in enumerate(lens):
        k, v = (plain.values(cache, x, tables, b, n).transpose(0, 1) for x in ("k", "v"))
        qq = q[b].view(2, -1, D)
        ref, mag = plain.attend(qq, k, v, torch.ones((1, n), dtype=torch.bool, device="cuda"))
        near(out[b].view(ref.shape), ref, mag * 2.0 ** -12 + lost_weights(qq, cache, tables, b, n) + 2.0 ** -25)


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30, 1e-6])
@pytest.mark.parametrize("inter,f32", [(False, True), (True, False)])
def test_append_norms_of_rows_whose_squares_float32_does_not_hold(eps, inter, f32):
    """Rows from bf16's smallest numbers to its largest, normed and turned: q, k, codes and scales are the
    float64 form's."""
    from halftone_quantizedkvcache_b200 import kernels
    new = [1500]
    q, k, v, cache, tables = append_case(new, [5], 2, 2, torch.bfloat16, 64, 51, fused=False)
    g = gen(52)
    powers = torch.tensor([-126, -100, -75, -62, -50, -49, 0, 49, 50, 59, 60, 62, 64, 100, 120, 124], device="cuda")
    for x in (q, k):
        by = powers[torch.randint(0, len(powers), x.shape[:2], generator=g, device="cuda")]
        x.copy_((x.double() * 2.0 ** by.double()[..., None]).to(torch.bfloat16))
    x[7, :, ::3] = 0                                     # (and some channels much smaller than their row's)
    x[8, :, 1:] *= 2.0 ** -60
    assert x.isfinite().all() and (x[:, :, 0] != 0).any()
    before = {n: y.clone() for n, y in cache.items()}
    inv = kernels.rope_inv_freq(128, 1e6)[0]
    w = [torch.empty(D, device="cuda").uniform_(0.2, 2.0, generator=g).to(torch.float32 if f32 else torch.bfloat16) for _ in range(2)]
    k_out = torch.zeros_like(k)
    got = kernels.paged4_append(q, k, v, cache, tables, ints([5]), cu_seqlens=cum(new), inv_freq=inv, interleaved=inter,
                                q_weight=w[0], k_weight=w[1], eps=eps, k_out=k_out)
    eps32 = float(torch.tensor(eps, dtype=torch.float32))
    check_append(q, k, v, cache, tables, new, [5], before, got, k_out, inv, w, inter, eps=eps32)


def test_append_norm_without_eps_of_rows_that_are_zero_or_no_number():
    from halftone_quantizedkvcache_b200 import kernels
    q, k, v, cache, tables = append_case([4], [0], 1, 1, torch.bfloat16, 16, 53, fused=False)
    k[1] = 0                                             # 0 / 0
    k[2, 0, 40] = math.nan
    w = torch.ones(D, device="cuda")
    kernels.paged4_append(q, k, v, cache, tables, ints([0]), cu_seqlens=ints([0, 4]), q_weight=w, k_weight=w, eps=0.0)
    kv, _ = kernels.paged4_gather(cache, tables, ints([4]), ints([0, 4]), 4)
    assert kv[1:3].isnan().all() and kv[0].isfinite().all() and kv[3].isfinite().all()
    kernels.paged4_append(q, k, v, cache, tables, ints([0]), cu_seqlens=ints([0, 4]), q_weight=w, k_weight=w, eps=1e-6)
    kv, _ = kernels.paged4_gather(cache, tables, ints([4]), ints([0, 4]), 4)
    assert (kv[1] == 0).all() and kv[2].isnan().all()


def test_append_norms_in_place_over_many_heads_and_rows_behind_the_last_sequence():
    """As above, 40 q heads a token in one block, q turned in its own memory; rows of no sequence stay."""
    from halftone_quantizedkvcache_b200 import kernels
    new = [9000, 597]
    q, k, v, cache, tables = append_case(new + [3], [0, 0, 0], 2, 20, torch.bfloat16, 64, 54, fused=True)
    tables = tables[:2].contiguous()
    g = gen(55)
    for x in (q, k):
        x.mul_(torch.where(torch.rand(x.shape[:2], generator=g, device="cuda") < 0.1, 2.0 ** 70, 1.0).to(torch.bfloat16)[..., None])
    before = {n: y.clone() for n, y in cache.items()}
    inv = kernels.rope_inv_freq(128, 1e6)[0]
    w = [torch.empty(D, device="cuda").uniform_(0.2, 2.0, generator=g) for _ in range(2)]
    q0 = q.clone()
    apart = kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=cum(new), inv_freq=inv, q_weight=w[0], k_weight=w[1])
    assert torch.equal(q, q0)
    assert kernels.paged4_append(q, k, v, cache, tables, ints([0, 0]), cu_seqlens=cum(new), inv_freq=inv, q_weight=w[0],
                                 k_weight=w[1], q_out=q) is q
    assert torch.equal(q, apart) and torch.equal(q[-3:], q0[-3:])
    check_append(q0, k, v, cache, tables, new, [0, 0], before, q, None, inv, w)


@pytest.mark.parametrize("rot,inter", [(0, False), (32, False), (96, True), (128, True)])
def test_append_norms_in_place_with_part_of_the_channels_turned(rot, inter):
    """Every row for float64, in its own memory: some lanes wait for their partners' channels, others do not."""
    from halftone_quantizedkvcache_b200 import kernels
    new = [700, 33]
    q, k, v, cache, tables = append_case(new, [3, 9], 2, 4, torch.bfloat16, 32, 56)
    for x in (q, k):
        x.mul_(2.0 ** 66)
    before = {n: y.clone() for n, y in cache.items()}
    inv = kernels.rope_inv_freq(rot, 1e6)[0] if rot else None
    w = [torch.empty(D, device="cuda").uniform_(0.2, 2.0, generator=gen(57)) for _ in range(2)]
    q0 = q.clone()
    kernels.paged4_append(q, k, v, cache, tables, ints([3, 9]), cu_seqlens=cum(new), inv_freq=inv, interleaved=inter, q_weight=w[0],
                          k_weight=w[1], q_out=q)
    check_append(q0, k, v, cache, tables, new, [3, 9], before, q, None, inv, w, inter)
