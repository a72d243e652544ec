"""The paged 4-bit cache's operators as a server uses them: packed prompts, chunks over a cached past,
captured decode steps, streams and threads, large pools; and the calls they refuse."""
import math
import threading

import pytest
import torch

import paged4_plain as plain

pytestmark = pytest.mark.gpu
D = 128


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cum(v):
    return ints([0] + torch.tensor(v).cumsum(0).tolist())


def close(got, ref, mag, weights):
    """Half a step of the output's type; the weights' rounding against sum p |v|."""
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    assert (err <= 1.01 * half * ref.abs() + weights * mag).all(), float((err - half * ref.abs()).max())


class Server:
    """A few sequences of one layer: norm weights, rotary frequencies, pages."""

    def __init__(self, B, Hkv, rep, dtype, page, per, seed):
        from halftone_quantizedkvcache_b200 import kernels
        self.k = kernels
        self.g = gen(seed)
        self.B, self.Hkv, self.Hq, self.dt, self.page = B, Hkv, Hkv * rep, dtype, page
        self.cache = kernels.paged4_alloc(B * per + 1, Hkv, page_size=page)
        self.tables = plain.random_tables(B, per, B * per + 1, self.g)
        self.w = [torch.empty(D, device="cuda").uniform_(0.5, 1.5, generator=self.g).to(dtype) for _ in range(2)]
        self.inv = kernels.rope_inv_freq(D, 1e6)[0]
        self.lens = torch.zeros(B, dtype=torch.int32, device="cuda")

    def projected(self, T):
        x = torch.randn((T, (self.Hq + 2 * self.Hkv) * D), generator=self.g, device="cuda").to(self.dt)
        return [y.unflatten(1, (-1, D)) for y in x.split([self.Hq * D, self.Hkv * D, self.Hkv * D], 1)]

    def append(self, qkv, cu=None, k_out=None):
        return self.k.paged4_append(*qkv, self.cache, self.tables, self.lens, cu_seqlens=cu, inv_freq=self.inv,
                                    q_weight=self.w[0], k_weight=self.w[1], k_out=k_out)

    def values(self, name, b):
        return plain.values(self.cache, name, self.tables, b, int(self.lens[b])).transpose(0, 1)


@pytest.mark.parametrize("dtype,page", [(torch.bfloat16, 64), (torch.float16, 16)])
def test_prompts_then_chunks_then_steps(dtype, page):
    s = Server(3, 2, 3, dtype, page, 512 // page, 3)
    half = torch.finfo(dtype).eps / 2
    # whole prompts: attention over the 16-bit rows that go into the pages
    new = [70, 1, 129]
    qkv = s.projected(sum(new))
    k_new = torch.empty((sum(new), s.Hkv, D), dtype=dtype, device="cuda")
    q = s.append(qkv, cum(new), k_new)
    s.lens += ints(new)
    out = s.k.packed_prefill_attn(q, k_new, qkv[2], cum(new))
    at = 0
    for n in new:
        i = torch.arange(n, device="cuda")
        kk, vv = (x[at:at + n].transpose(0, 1).repeat_interleave(3, 0) for x in (k_new, qkv[2]))
        ref, mag = plain.attend(q[at:at + n].transpose(0, 1), kk, vv, i <= i[:, None])
        close(out[at:at + n].transpose(0, 1), ref, mag, half + 2.0 ** -13)
        at += n
    # a chunk of every sequence over its past, as the cache holds it
    new = [40, 200, 3]
    qkv = s.projected(sum(new))
    q = s.append(qkv, cum(new))
    s.lens += ints(new)
    held = s.lens.tolist()
    k, v = s.k.paged4_gather(s.cache, s.tables, s.lens, cum(held), sum(held), dtype=dtype)
    out = s.k.packed_prefill_attn(q, k, v, cum(new), cum(held))
    at = 0
    for b, (n, m) in enumerate(zip(new, held)):
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")
        kk, vv = (s.values(x, b).to(dtype).repeat_interleave(3, 0) for x in ("k", "v"))
        ref, mag = plain.attend(q[at:at + n].transpose(0, 1), kk, vv, j <= m - n + i)
        close(out[at:at + n].transpose(0, 1), ref, mag, half + 2.0 ** -13)
        at += n
    # steps of one token each
    for _ in range(3):
        q = s.append(s.projected(3))
        s.lens += 1
        out = s.k.paged4_decode_attn(q, s.cache, s.tables, s.lens)
        for b in range(3):
            n = int(s.lens[b])
            ref, mag = plain.attend(q[b].view(s.Hkv, 3, D), s.values("k", b), s.values("v", b),
                                    torch.ones((1, n), dtype=torch.bool, device="cuda"))
            close(out[b].view(s.Hkv, 3, D), ref, mag, 2.0 ** -10)  # 2^-16 x 64 of a tile's largest weight at most
    assert s.k.ragged_status() == 0


def test_many_sequences_from_a_fused_projection():
    """150 sequences (more than a warp looks up at once), q turned where the projection left it."""
    s = Server(150, 2, 2, torch.bfloat16, 16, 5, 8)
    new = [(7 * i) % 40 for i in range(150)]
    T = sum(new)
    qkv = s.projected(T)
    before = [x.clone() for x in qkv]
    k_new = torch.empty((T, 2, D), dtype=torch.bfloat16, device="cuda")
    q = s.k.paged4_append(*qkv, s.cache, s.tables, s.lens, cu_seqlens=cum(new), inv_freq=s.inv,
                          q_weight=s.w[0], k_weight=s.w[1], q_out=qkv[0], k_out=k_new)
    assert q is qkv[0] and torch.equal(qkv[1], before[1]) and torch.equal(qkv[2], before[2])
    s.lens += ints(new)
    b = torch.repeat_interleave(torch.arange(150, device="cuda"), torch.tensor(new, device="cuda"))
    pos = torch.cat([torch.arange(n, device="cuda") for n in new])
    k64 = plain.turned(before[1], s.w[1], pos, s.inv, False, 1.0, 1e-6)
    held, _ = s.k.paged4_gather(s.cache, s.tables, s.lens, cum(new), T)
    codes, sc = plain.coded(k64)
    assert torch.equal(held, (codes.double() * sc.double().repeat_interleave(32, -1)).float().to(torch.bfloat16))
    out = s.k.packed_prefill_attn(q, k_new, qkv[2], cum(new))
    half = torch.finfo(torch.bfloat16).eps / 2
    for e in range(0, 150, 13):
        rows = (b == e).nonzero()[:, 0]
        if len(rows):
            i = torch.arange(len(rows), device="cuda")
            kk, vv = (x[rows].transpose(0, 1).repeat_interleave(2, 0) for x in (k_new, qkv[2]))
            ref, mag = plain.attend(q[rows].transpose(0, 1), kk, vv, i <= i[:, None])
            close(out[rows].transpose(0, 1), ref, mag, half + 2.0 ** -13)
    assert s.k.ragged_status() == 0


def test_captured_steps_follow_the_lengths():
    s = Server(4, 2, 2, torch.bfloat16, 16, 40, 5)
    new = [3, 100, 0, 250]
    s.append(s.projected(sum(new)), cum(new))
    s.lens += ints(new)
    static = s.projected(4)
    feed = [[y.clone() for y in s.projected(4)] for _ in range(6)]

    def step():
        q = s.append(static)
        s.lens.add_(1)
        return s.k.paged4_decode_attn(q, s.cache, s.tables, s.lens)

    start = s.lens.clone(), {n: x.clone() for n, x in s.cache.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()

    def rewind():
        s.lens.copy_(start[0])
        for n, x in s.cache.items():
            x.copy_(start[1][n])

    got, ref = [], []
    rewind()
    for x in feed:
        for a, b in zip(static, x):
            a.copy_(b)
        graph.replay()
        got.append(out.clone())
    pages = {n: x.clone() for n, x in s.cache.items()}
    rewind()
    for x in feed:
        for a, b in zip(static, x):
            a.copy_(b)
        ref.append(step())
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    for n, x in s.cache.items():
        assert torch.equal(x.view(torch.uint8), pages[n].view(torch.uint8))


def test_captured_prompts_and_gather_follow_their_starts():
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(9)
    q = torch.randn((300, 8, D), generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn((700, 2, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache = plain.random_cache(kernels, 60, 2, 16, g)
    tables = plain.random_tables(2, 30, 60, g)
    cu_q, cu_k, lens, cu = cum([200, 100]), cum([300, 400]), ints([300, 400]), cum([300, 400])

    def run():
        return (kernels.packed_prefill_attn(q, k, v, cu_q, cu_k),
                *kernels.paged4_gather(cache, tables, lens, cu, 700))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for nq, nk in (([200, 100], [300, 400]), ([1, 250], [1, 690]), ([0, 300], [100, 300]), ([30, 0], [470, 0])):
        cu_q.copy_(cum(nq)), cu_k.copy_(cum(nk)), lens.copy_(ints(nk)), cu.copy_(cum(nk))
        graph.replay()
        for a, b in zip(out, run()):
            assert torch.equal(a, b), (nq, nk)


def test_calls_on_two_streams_and_from_two_threads():
    from halftone_quantizedkvcache_b200 import kernels
    jobs = []
    for seed, lens in ((1, [900, 30]), (2, [17, 2000])):
        g = gen(seed)
        cache = plain.random_cache(kernels, 260, 2, 16, g)
        tables = plain.random_tables(2, 128, 260, g)
        q = torch.randn((2, 4, D), generator=g, device="cuda").to(torch.bfloat16)
        qp = torch.randn((500, 4, D), generator=g, device="cuda").to(torch.float16)
        kp = torch.randn((500, 2, D), generator=g, device="cuda").to(torch.float16)
        jobs.append(lambda q=q, c=cache, t=tables, n=ints(lens), qp=qp, kp=kp, s=cum([499, 1]):
                    (kernels.paged4_decode_attn(q, c, t, n), kernels.packed_prefill_attn(qp, kp, kp, s),
                     *kernels.paged4_gather(c, t, n, cum([700, 1400]), 2100)))
    ref = [job() for job in jobs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = jobs[i]()
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, ref[i])):
                    bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_pages_past_32_bits():
    """Pools whose byte offsets pass 2^32: 600 000 pages of 16 tokens and 8 heads hold 4.9 GB of codes."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(4)
    n, Hkv, page = 600_000, 8, 16
    shape = (n, Hkv, page)
    big = {"k": torch.empty(shape + (64,), dtype=torch.uint8, device="cuda"), "v": torch.empty(shape + (64,), dtype=torch.uint8, device="cuda"),
           "k_scale": torch.empty(shape + (4,), dtype=torch.float16, device="cuda"), "v_scale": torch.empty(shape + (4,), dtype=torch.float16, device="cuda")}
    small = plain.random_cache(kernels, 6, Hkv, page, g)
    far = torch.tensor([599_999, 300_001, 524_288, 524_287, 1, 262_144], device="cuda")
    for name in big:
        big[name][far] = small[name]
    tables = plain.random_tables(2, 3, 6, g)
    q = torch.randn((2, 16, D), generator=g, device="cuda").to(torch.bfloat16)
    args = dict(cu_seqlens=cum([20, 7]), inv_freq=kernels.rope_inv_freq(D)[0])
    new = [torch.randn((27, h, D), generator=g, device="cuda").to(torch.bfloat16) for h in (16, 8, 8)]
    lens = ints([15, 33])
    for cache, t in ((small, tables), (big, far[tables.long()].to(torch.int32))):
        kernels.paged4_append(*new, cache, t, lens, **args)
    for name in big:
        assert torch.equal(big[name][far].view(torch.uint8), small[name].view(torch.uint8)), name
    t = far[tables.long()].to(torch.int32)
    assert torch.equal(kernels.paged4_decode_attn(q, big, t, ints([35, 40])), kernels.paged4_decode_attn(q, small, tables, ints([35, 40])))
    for a, b in zip(kernels.paged4_gather(big, t, lens, cum([15, 33]), 48), kernels.paged4_gather(small, tables, lens, cum([15, 33]), 48)):
        assert torch.equal(a, b)
    assert kernels.ragged_status() == 0


def test_rows_past_32_bits():
    """Packed rows at element offsets past 2^31: 1 100 000 rows of 16 heads."""
    from halftone_quantizedkvcache_b200 import kernels
    T, g = 1_100_000, gen(6)
    q = torch.zeros((T, 16, D), dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros((T, 2, D), dtype=torch.bfloat16, device="cuda")
    n = 300
    q[-n:].normal_(generator=g), kv[-n:].normal_(generator=g)
    out = kernels.packed_prefill_attn(q, kv, kv, ints([0, T - n, T]), ints([T - n, T - n, T]))
    assert torch.equal(out[-n:], kernels.packed_prefill_attn(q[-n:].clone(), kv[-n:].clone(), kv[-n:].clone(), ints([0, n])))
    assert (out[:-n:100_000] == 0).all()
    cache = kernels.paged4_alloc(40, 2, page_size=16)
    tables = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
    kernels.paged4_append(q, kv, kv, cache, tables, ints([0, 0]), cu_seqlens=ints([T - n, T - n, T]), q_out=q)
    k, _ = kernels.paged4_gather(cache, tables, ints([0, n]), ints([0, 0, n]), n)
    codes, sc = plain.coded(kv[-n:])
    assert torch.equal(k, (codes.double() * sc.double().repeat_interleave(32, -1)).float().to(torch.bfloat16))
    assert kernels.ragged_status() == 0


def test_refusals():
    from halftone_quantizedkvcache_b200 import kernels
    kernels.reset_ragged_status()
    cache = kernels.paged4_alloc(8, 2, page_size=16)
    other = kernels.paged4_alloc(8, 2, page_size=32)
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, k = bf(4, 4, D), bf(4, 2, D)
    tables, lens, cu = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), ints([0] * 4), ints([0, 1, 2, 3, 4])
    inv = kernels.rope_inv_freq(D)[0]

    def no(kind, call, *args, **kw):
        with pytest.raises(kind):
            call(*args, **kw)
    app, dec, gat, pre = kernels.paged4_append, kernels.paged4_decode_attn, kernels.paged4_gather, kernels.packed_prefill_attn
    # caches and tables
    for call in (lambda c, t: app(q, k, k, c, t, lens), lambda c, t: dec(q, c, t, lens), lambda c, t: gat(c, t, lens, cu, 4)):
        for bad in (dict(cache, k=cache["k"].float()), dict(cache, k_scale=cache["k_scale"].float())):
            no(TypeError, call, bad, tables)
        for bad in (dict(cache, v=other["v"]), dict(cache, v_scale=other["v_scale"]), dict(cache, k=cache["k"][:4]),
                    {n: x.cpu() for n, x in cache.items()}, {n: x.transpose(2, 3) for n, x in cache.items()},
                    {n: x[:, :1].expand(8, 2, *x.shape[2:]) for n, x in cache.items()}, {n: x[:0] for n, x in cache.items()},
                    {n: x[:, :, :8] for n, x in cache.items()}, dict(cache, k=cache["k"].clone().transpose(0, 1).contiguous().transpose(0, 1)),
                    {"k": cache["k"]}):
            no(ValueError, call, bad, tables)
        for bad in (tables.long(), tables[:3], tables[0], tables.t().contiguous().t()[:, ::2], tables.cpu()):
            no((ValueError, TypeError), call, cache, bad) if bad.shape != (4, 1) else None
    # append
    for bad in (dict(cu_seqlens=cu[:4]), dict(cu_seqlens=cu.long()), dict(inv_freq=inv[:4]), dict(inv_freq=inv.double()),
                dict(inv_freq=torch.ones(72, device="cuda")), dict(pos_offset=lens[:2]), dict(q_weight=bf(64)), dict(eps=-1.0),
                dict(q_out=bf(4, 4, 64)), dict(q_out=q[:, :1].expand(4, 4, D)), dict(k_out=bf(4, 4, D)), dict(k_out=k),
                dict(k_out=k.float())):
        no(ValueError, app, q, k, k, cache, tables, lens, **bad)
    no(TypeError, app, q, k, k, cache, tables, lens, q_weight=torch.ones(D, device="cuda", dtype=torch.float16))
    no(TypeError, app, q, k, k, cache, tables, lens, q_weight=bf(D), k_weight=bf(D).float())
    no(TypeError, app, q, k, k.half(), cache, tables, lens)
    no(TypeError, app, q.float(), k.float(), k.float(), cache, tables, lens)
    no(ValueError, app, q, k, bf(4, 1, D), cache, tables, lens)
    no(ValueError, app, q, k[:3], k[:3], cache, tables, lens)
    no(ValueError, app, bf(5, 4, D), bf(5, 2, D), bf(5, 2, D), cache, tables, lens)        # 5 tokens, no starts
    # decode
    no(TypeError, dec, q.float(), cache, tables, lens)
    for bad in (bf(4, 3, D), bf(4, 4, 64), bf(4, 4, 2, D), bf(4, D)):
        no(ValueError, dec, bad, cache, tables, lens)
    no(ValueError, dec, q, cache, tables, lens.long())
    no(ValueError, dec, q, cache, tables, lens, out=bf(4, 2, D))
    no(ValueError, dec, q, cache, tables, lens, out=q[:1].expand(4, 4, D))
    no(ValueError, dec, bf(1025, 4, D), cache, torch.zeros((1025, 2), dtype=torch.int32, device="cuda"), ints([0] * 1025))
    # gather
    no(TypeError, gat, cache, tables, lens, cu, 4, dtype=torch.float32)
    no(ValueError, gat, cache, tables, lens, cu, -1)
    no(TypeError, gat, cache, tables, lens, cu, 1.5)
    no(ValueError, gat, cache, tables, lens, cu[:3], 4)
    no(ValueError, gat, cache, tables, lens, cu, 4, k_out=k)
    no(ValueError, gat, cache, tables, lens, cu, 4, k_out=k, v_out=k)
    no(ValueError, gat, cache, tables, lens, cu, 4, k_out=k, v_out=bf(3, 2, D))
    no(ValueError, gat, cache, tables, lens, cu, 4, first=lens[:2])
    # packed attention
    no(TypeError, pre, q.float(), k.float(), k.float(), cu)
    no(TypeError, pre, q, k.half(), k.half(), cu)
    no(ValueError, pre, bf(4, 3, D), k, k, cu)
    no(ValueError, pre, q, k, k[:3], cu)
    no(ValueError, pre, q, k, k, cu, cu[:4])
    no(ValueError, pre, q, k, k, cu.long())
    for scale in (0.0, -1.0, math.nan, math.inf):
        no(ValueError, pre, q, k, k, cu, sm_scale=scale)
    no(ValueError, pre, q, k, k, cu, out=q[:, :1].expand(4, 4, D))
    # none of it reached the device
    assert kernels.ragged_status() == 0
    # empty batches
    none = lens[:0]
    assert dec(q[:0], cache, tables[:0], none).shape == (0, 4, D)
    assert gat(cache, tables[:0], none, cu[:1], 3)[0].abs().sum() == 0
    assert torch.equal(app(q, k, k, cache, tables[:0], none, cu_seqlens=cu[:1]), q)


def test_outputs_in_one_memory_side_by_side():
    """Rows of q, k and v, of K and V, and of all outputs lie within one another's ranges, but share no byte:
    such calls give what calls on separate memory give, and those that share some are refused."""
    from halftone_quantizedkvcache_b200 import kernels
    T, Hq, H, page, n = 90, 6, 2, 16, 8
    g = gen(61)
    lens, cu, now = ints([0, 0]), ints([0, 50, 90]), ints([50, 40])
    tables = plain.random_tables(2, 4, n, g)
    inv = kernels.rope_inv_freq(D, 1e6)[0]
    qkv = torch.randn((T, Hq + 2 * H, D), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    plainly = kernels.paged4_alloc(n, H, page_size=page)
    k16 = torch.empty((T, H, D), dtype=torch.bfloat16, device="cuda")
    q2 = kernels.paged4_append(q, k, v, plainly, tables, lens, cu_seqlens=cu, inv_freq=inv, k_out=k16)
    # pages of K and V in turn, q in its place, the new k beside other columns
    codes = torch.zeros((n, 2, H, page, 64), dtype=torch.uint8, device="cuda")
    scales = torch.zeros((n, 2, H, page, 4), dtype=torch.float16, device="cuda")
    cache = {"k": codes[:, 0], "v": codes[:, 1], "k_scale": scales[:, 0], "v_scale": scales[:, 1]}
    wide = torch.zeros((T, 3 * H, D), dtype=torch.bfloat16, device="cuda")
    x = qkv.clone()
    xq, xk, xv = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    assert kernels.paged4_append(xq, xk, xv, cache, tables, lens, cu_seqlens=cu, inv_freq=inv, q_out=xq, k_out=wide[:, H:2 * H]) is xq
    assert torch.equal(xq, q2) and torch.equal(wide[:, H:2 * H], k16) and torch.equal(x[:, Hq:], qkv[:, Hq:])
    assert all(torch.equal(cache[c], plainly[c]) for c in cache) and (wide[:, :H] == 0).all()
    kg, vg = kernels.paged4_gather(plainly, tables, now, cu, T)
    kernels.paged4_gather(cache, tables, now, cu, T, k_out=wide[:, :H], v_out=wide[:, 2 * H:])
    assert torch.equal(wide[:, :H], kg) and torch.equal(wide[:, 2 * H:], vg) and torch.equal(wide[:, H:2 * H], k16)
    out = kernels.packed_prefill_attn(q2, k16, v, cu)
    assert kernels.packed_prefill_attn(xq, wide[:, H:2 * H], xv, cu, out=xq) is xq and torch.equal(xq, out)
    step = kernels.paged4_decode_attn(q2[:2], plainly, tables, now)
    y = q2.clone()
    assert torch.equal(kernels.paged4_decode_attn(y[:2], cache, tables, now, out=y[:2]), step) and torch.equal(y[2:], q2[2:])
    assert kernels.ragged_status() == 0
    # shared in part
    big = torch.zeros((T + 1, Hq, D), dtype=torch.bfloat16, device="cuda")
    bad = [
        lambda: kernels.paged4_append(q, k, v, plainly, tables, lens, cu_seqlens=cu, k_out=qkv[:, Hq + 1:Hq + 1 + H]),
        lambda: kernels.paged4_append(q, k, v, plainly, tables, lens, cu_seqlens=cu, q_out=qkv[:, 1:Hq + 1]),
        lambda: kernels.paged4_append(big[:T], k, v, plainly, tables, lens, cu_seqlens=cu, q_out=big[1:]),
        lambda: kernels.paged4_append(q, k, v, plainly, tables, lens, cu_seqlens=cu, q_out=big[1:], k_out=big[:T, :H]),
        lambda: kernels.paged4_append(q, k, v, {**cache, "v": cache["k"]}, tables, lens, cu_seqlens=cu),
        lambda: kernels.paged4_append(q, k, v, {**cache, "v_scale": cache["k_scale"]}, tables, lens, cu_seqlens=cu),
        lambda: kernels.paged4_gather(plainly, tables, now, cu, T, k_out=big[:T, :H], v_out=big[1:, :H]),
        lambda: kernels.paged4_gather(plainly, tables, now, cu, T, k_out=big[:T, :H], v_out=big[:T, 1:H + 1]),
        lambda: kernels.packed_prefill_attn(big[:T], k, v, cu, out=big[1:]),
        lambda: kernels.packed_prefill_attn(q, big[:T, :H], v, cu, out=big[:T]),
        lambda: kernels.packed_prefill_attn(q, k, big[1:, Hq - H:], cu, out=big[:T]),
        lambda: kernels.paged4_decode_attn(big[:2], plainly, tables, now, out=big[1:3]),
        lambda: kernels.paged4_decode_attn(q2[:2], plainly, tables, now, out=torch.as_strided(big, (2, Hq, D), (D, D, 1))),
    ]
    saved = {c: t.clone() for c, t in plainly.items()}
    for call in bad:
        with pytest.raises(ValueError, match="memory of their own"):
            call()
    assert all(torch.equal(plainly[c], saved[c]) for c in saved) and (big == 0).all()


@pytest.mark.parametrize("nq,nk,Hkv,rep", [([512], [512], 8, 2), ([2100, 900], [2100, 900], 2, 2), ([20, 48, 77], [1020, 2600, 4099], 2, 6),
                                           ([64, 65, 63, 1], [64, 65, 63, 1], 2, 4), ([600], [500], 8, 2), ([300, 7], [300, 7], 1, 3)])
def test_attention_over_its_queries(nq, nk, Hkv, rep):
    """out is q: one and two row tiles a block, keys split or not, Q by tensor map or by loads."""
    from halftone_quantizedkvcache_b200 import kernels
    g = gen(62)
    q = torch.randn((sum(nq), Hkv * rep, D), generator=g, device="cuda").to(torch.bfloat16)
    k, v = (torch.randn((sum(nk), Hkv, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ref = kernels.packed_prefill_attn(q, k, v, cum(nq), cum(nk))
    for _ in range(10):
        x = q.clone()
        assert kernels.packed_prefill_attn(x, k, v, cum(nq), cum(nk), out=x) is x
        assert torch.equal(x, ref)
    cache = plain.random_cache(kernels, len(nk) * 65 + 1, Hkv, 64, g)
    tables = plain.random_tables(len(nk), 65, len(nk) * 65 + 1, g)
    y = q[:len(nk)].contiguous()
    step = kernels.paged4_decode_attn(y, cache, tables, ints(nk))
    for _ in range(10):
        x = y.clone()
        kernels.paged4_decode_attn(x, cache, tables, ints(nk), out=x)
        assert torch.equal(x, step)
