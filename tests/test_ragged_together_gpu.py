"""The ragged-batch operators as a server uses them: prompts in ragged chunks, decode steps
captured in a CUDA graph while the sequences grow, a shared prefix, and the calls around that
which no single operator's test makes (other streams, two graphs, long caches, broken values
where no query looks, refusals).  Bounds as in test_ragged_gpu."""
import pytest
import torch

from halftone_quantizedkvcache_b200 import _lib, kernels
from test_ragged_gpu import D, TDT, check, make_cache, ref_rows, window_ref

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def empty_cache(B, Hkv, cap, sdt):
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros((B, Hkv, cap, D), dtype=torch.int8, device="cuda")
    ksc = (torch.rand((B, Hkv, 1, D), generator=g, device="cuda") * 0.02 + 0.02).to(TDT[sdt])
    return k, ksc, torch.zeros_like(k), torch.zeros((B, Hkv, cap, 1), dtype=TDT[sdt], device="cuda")


def projections(g, B, Hq, Hkv, S, dt):
    return [torch.randn((B, h, S, D), generator=g, device="cuda").to(TDT[dt]) for h in (Hq, Hkv, Hkv)]


@pytest.mark.parametrize("dt,sdt,rep", [("bf16", "f16", 2), ("f16", "f32", 2), ("bf16", "f16", 8)])
def test_prompts_in_chunks_then_captured_decode(dt, sdt, rep):
    """Ragged prompts appended and attended chunk by chunk, then decode steps replayed from one
    captured graph across a tile's border; each output against the cache as it then stands."""
    B, Hkv, cap, window, sinks = 3, 2, 700, 200, 4
    Hq = Hkv * rep
    g = torch.Generator(device="cuda").manual_seed(rep)
    cache = empty_cache(B, Hkv, cap, sdt)
    kc, ksc, vc, vsc = cache
    inv, factor = kernels.rope_inv_freq(D, 1e4)
    lens = [0] * B
    n = i32(lens)
    for chunk in ([130, 7, 0], [250, 128, 1], [1, 260, 120]):
        S = max(chunk)
        q, kn, vn = projections(g, B, Hq, Hkv, S, dt)
        m = i32(chunk)
        qr = kernels.rope_append_kv(q, kn, vn, inv, kc, vc, ksc, vsc, n, n_new=m, factor=factor)
        n += m
        lens = [a + b for a, b in zip(lens, chunk)]
        got = kernels.int8_window_prefill_attn(qr, *cache, n, window=window, sinks=sinks, q_lens=m)
        ref, tol = window_ref(qr, cache, lens, chunk, window, sinks, dt)
        check(got, ref, tol, "chunk")

    q, kn, vn = projections(g, B, Hq, Hkv, 1, dt)

    def step():
        qr = kernels.rope_append_kv(q, kn, vn, inv, kc, vc, ksc, vsc, n, factor=factor)
        n.add_(1)
        return qr, kernels.int8_window_decode_attn(qr, *cache, n, window=window, sinks=sinks)

    def verify(qr, out):
        ref, tol = window_ref(qr, cache, lens, [1] * B, window, sinks, dt)
        check(out[:, :, 0], ref[:, 0], tol[:, 0], "step")

    res = step()
    lens = [x + 1 for x in lens]
    verify(*res)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    for _ in range(6):
        for t, h in ((q, Hq), (kn, Hkv), (vn, Hkv)):
            t.copy_(torch.randn((B, h, 1, D), generator=g, device="cuda"))
        graph.replay()
        lens = [x + 1 for x in lens]
        verify(*res)
    assert n.tolist() == lens and kernels.ragged_status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_prefix_then_own_tokens_captured(dt):
    """A prompt quantized once, then samples that go on from it: rotary positions behind the
    prefix, own tokens appended, prefix decode, in one replayed graph."""
    U, Hkv, rep, P, cap = 5, 2, 3, 300, 64
    Hq = Hkv * rep
    g = torch.Generator(device="cuda").manual_seed(3)
    pre, own = empty_cache(1, Hkv, P, "f16"), empty_cache(U, Hkv, cap, "f16")
    own[1].copy_(pre[1].expand_as(own[1]))
    inv, _ = kernels.rope_inv_freq(D, 1e4)
    _, kn, vn = projections(g, 1, Hq, Hkv, P, dt)
    zero = torch.zeros((1, Hq, P, D), dtype=TDT[dt], device="cuda")
    kernels.rope_append_kv(zero, kn, vn, inv, pre[0], pre[2], pre[1], pre[3], i32([0]))
    n, off = i32([0] * U), i32([P] * U)
    q, kn, vn = projections(g, U, Hq, Hkv, 1, dt)

    def step():
        qr = kernels.rope_append_kv(q, kn, vn, inv, own[0], own[2], own[1], own[3], n, pos_offset=off)
        n.add_(1)
        return qr, kernels.int8_prefix_decode_attn(qr, *pre, *own, n)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = step()
    for t in range(2, 5):
        for x, h in ((q, Hq), (kn, Hkv), (vn, Hkv)):
            x.copy_(torch.randn((U, h, 1, D), generator=g, device="cuda"))
        graph.replay()
        # one cache per sequence: the prefix, then its own tokens
        whole = [torch.cat([a.expand(U, *a.shape[1:]), b[:, :, :t]], 2) for a, b in zip(pre, own)]
        whole[1] = own[1]
        ref, tol = window_ref(qr, whole, [P + t] * U, [1] * U, None, 0, dt)
        check(out[:, :, 0], ref[:, 0], tol[:, 0], "prefix step")
        # and the same as decode over the whole, up to both bounds
        flat = kernels.int8_window_decode_attn(qr, *[x.contiguous() for x in whole], i32([P + t] * U))
        assert ((flat.double() - out.double()).abs() <= 2 * tol[:, 0].unsqueeze(2)).all()


def test_two_graphs_and_two_streams_at_once():
    """Two captured graphs and two eager streams run the operators at the same time: none sees
    another's scratch."""
    g = torch.Generator(device="cuda").manual_seed(4)
    sets = []
    for i in range(2):
        cache = make_cache(g, 8, 2, 2000 + 512 * i, "f16")
        n = i32([(251 * (b + 1 + i)) % 2000 for b in range(8)])
        q = torch.randn((8, 4, 1, D), generator=g, device="cuda").to(torch.bfloat16)
        qp = torch.randn((8, 4, 16, D), generator=g, device="cuda").to(torch.bfloat16)
        sets.append((cache, n, q, qp))

    def work(s):
        cache, n, q, qp = s
        return [kernels.int8_window_decode_attn(q, *cache, n, window=700, sinks=4),
                kernels.int8_window_prefill_attn(qp, *cache, n, window=700, sinks=4),
                kernels.int8_prefix_decode_attn(q, *[x[:1] for x in cache], *cache, n)]

    want = [work(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(s))
        graphs.append(gr)
    for _ in range(5):
        eager = [[], []]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
                eager[i] = work(sets[1 - i])
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i] + eager[i], want[i] + want[1 - i]):
                assert torch.equal(a, b)
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("rep", [2, 8])
def test_rows_past_two_to_the_31_bytes(rep):
    """A cache whose last rows lie 2.3 GB behind its base."""
    cap, Hkv = 1_130_000, 16
    g = torch.Generator(device="cuda").manual_seed(5)
    k8 = torch.randint(-127, 128, (1, Hkv, cap, D), generator=g, device="cuda", dtype=torch.int8)
    assert k8.numel() > 1 << 31
    ksc = torch.rand((1, Hkv, 1, D), generator=g, device="cuda") * 0.01 + 0.01
    vsc = torch.rand((1, Hkv, cap, 1), generator=g, device="cuda") * 0.02 + 0.01
    cache, n, window, sinks = (k8, ksc, k8, vsc), i32([cap - 3]), 300, 5
    q = torch.randn((1, Hkv * rep, 3, D), generator=g, device="cuda").to(torch.bfloat16)
    dec = kernels.int8_window_decode_attn(q[:, :, -1:], *cache, n, window=window, sinks=sinks)
    pre = kernels.int8_window_prefill_attn(q, *cache, n, window=window, sinks=sinks)
    # the seen keys as a short cache of their own: sinks, then the run of the last queries
    j = torch.cat([torch.arange(sinks), torch.arange(cap - 3 - window - 2, cap - 3)]).cuda()
    for h in (0, Hkv * rep - 1):
        kh = h // rep
        k, v = k8[0, kh, j].double() * ksc[0, kh].double(), k8[0, kh, j].double() * vsc[0, kh, j].double()
        pos = torch.arange(cap - 6, cap - 3, device="cuda")[:, None]
        seen = (j[None] <= pos) & ((j[None] > pos - window) | (j[None] < sinks))
        ref, tol = ref_rows(q[0, h], k, v, seen, "bf16")
        check(pre[0, :, h], ref, tol, f"prefill head {h}")
        check(dec[0, h], ref[-1:], tol[-1:], f"decode head {h}")


@pytest.mark.parametrize("dt,rep", [("bf16", 2), ("bf16", 8), ("f16", 2), ("f16", 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_broken_scales_where_no_query_looks(dt, rep, bad):
    """V scales that are no numbers between the sinks and the window (decode), and at the newest
    token, which only the last query of a chunk sees (prefill)."""
    g = torch.Generator(device="cuda").manual_seed(6)
    B, Hkv, cap, window, sinks = 2, 2, 600, 70, 3
    cache = make_cache(g, B, Hkv, cap, "f32")
    clean = cache[3].clone()
    lens = [600, 333]
    for b, m in enumerate(lens):
        cache[3][b, :, sinks:m - window] = bad
        cache[3][b, :, m:] = bad
    q = torch.randn((B, Hkv * rep, 9, D), generator=g, device="cuda").to(TDT[dt])
    n = i32(lens)
    got = kernels.int8_window_decode_attn(q[:, :, -1:], *cache, n, window=window, sinks=sinks)
    good = (cache[0], cache[1], cache[2], clean)
    ref, tol = window_ref(q[:, :, -1:], good, lens, [1, 1], window, sinks, dt)
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "decode")
    cache[3].copy_(clean)
    for b, m in enumerate(lens):
        cache[3][b, :, m - 1] = bad
    got = kernels.int8_window_prefill_attn(q, *cache, n, window=window, sinks=sinks)
    ref, tol = window_ref(q, good, lens, [9, 9], window, sinks, dt)
    check(got[:, :-1], ref[:, :-1], tol[:, :-1], "prefill")
    assert not torch.isfinite(got[:, -1]).any()      # the query that does look


def test_nan_query_row_keeps_to_itself():
    g = torch.Generator(device="cuda").manual_seed(7)
    cache = make_cache(g, 1, 1, 300, "f16")
    q = torch.randn((1, 4, 50, D), generator=g, device="cuda").to(torch.bfloat16)
    n = i32([300])
    want = kernels.int8_window_prefill_attn(q, *cache, n)
    q2 = q.clone()
    q2[0, 1, 20, 5] = float("nan")
    got = kernels.int8_window_prefill_attn(q2, *cache, n)
    assert torch.isnan(got[0, 20, 1]).all()
    got[0, 20, 1] = want[0, 20, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rep", [1, 2, 4, 8])
def test_broken_values_that_are_seen(rep, dt):
    """A NaN in one head's query spoils that row alone; a V scale that is no number, in sight,
    spoils its sequence's rows of that kv head alone."""
    g = torch.Generator(device="cuda").manual_seed(13)
    cache = make_cache(g, 2, 2, 400, "f32")
    q = torch.randn((2, 2 * rep, 1, D), generator=g, device="cuda").to(TDT[dt])
    n = i32([400, 150])
    want = kernels.int8_window_decode_attn(q, *cache, n, window=100, sinks=2)
    q2 = q.clone()
    q2[1, rep - 1, 0, 7] = float("nan")
    got = kernels.int8_window_decode_attn(q2, *cache, n, window=100, sinks=2)
    assert torch.isnan(got[1, rep - 1]).all()
    got[1, rep - 1] = want[1, rep - 1]
    assert torch.equal(got, want)
    for bad in (float("nan"), float("inf")):
        cache[3][0, 1, 350] = bad
        got = kernels.int8_window_decode_attn(q, *cache, n, window=100, sinks=2)
        assert not torch.isfinite(got[0, rep:]).any()
        got[0, rep:] = want[0, rep:]
        assert torch.equal(got, want)


@pytest.mark.parametrize("rep", [2, 8])
def test_nan_query_over_many_blocks(rep):
    """The same where a row's keys are cut over many blocks and joined."""
    g = torch.Generator(device="cuda").manual_seed(14)
    cache = make_cache(g, 1, 1, 9000, "f16")
    q = torch.randn((1, rep, 7, D), generator=g, device="cuda").to(torch.bfloat16)
    n = i32([9000])
    for call in (lambda x: kernels.int8_window_decode_attn(x[:, :, -1:], *cache, n)[:, :, 0][None],
                 lambda x: kernels.int8_window_prefill_attn(x, *cache, n),
                 lambda x: kernels.int8_prefix_decode_attn(x[:, :, -1:], *cache, *cache, n)[:, :, 0][None]):
        want = call(q)
        q2 = q.clone()
        q2[0, 1, -1, 100] = float("nan")
        got = call(q2)
        assert torch.isnan(got[0, -1, 1]).all()
        got[0, -1, 1] = want[0, -1, 1]
        assert torch.equal(got, want)


def test_empty_caches():
    q = torch.randn((2, 4, 1, D), device="cuda").to(torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(8)
    none = make_cache(g, 2, 2, 0, "f16")
    assert (kernels.int8_window_decode_attn(q, *none, i32([0, 0])) == 0).all()
    assert (kernels.int8_window_decode_attn(q.repeat(1, 8, 1, 1), *none, i32([3, 0])) == 0).all()
    assert (kernels.int8_window_prefill_attn(q, *none, i32([0, 5])) == 0).all()
    pre = make_cache(g, 1, 2, 100, "f16")
    got = kernels.int8_prefix_decode_attn(q, *pre, *none, i32([0, 0]))
    ref, tol = window_ref(q, [x.expand(2, *x.shape[1:]) for x in pre], [100, 100], [1, 1], None, 0, "bf16")
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "prefix alone")
    own = make_cache(g, 2, 2, 50, "f16")
    nop = make_cache(g, 1, 2, 0, "f16")
    got = kernels.int8_prefix_decode_attn(q, *nop, *own, i32([50, 0]))
    ref, tol = window_ref(q, own, [50, 0], [1, 1], None, 0, "bf16")
    check(got[:, :, 0], ref[:, 0], tol[:, 0], "own alone")
    # no sequences at all
    assert kernels.int8_window_decode_attn(q[:0], *[x[:0] for x in own], i32([])).shape == (0, 4, 1, D)
    assert kernels.ragged_status() == 0


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_query_rows_of_any_alignment(dt):
    """A view whose rows start on odd addresses, after an aligned one of the same strides: the
    rows are copied, whatever an earlier call with these shapes found."""
    g = torch.Generator(device="cuda").manual_seed(9)
    cache = make_cache(g, 2, 2, 333, "f16")
    n = i32([333, 100])
    store = torch.randn((2, 4, 1, 2 * D), generator=g, device="cuda").to(TDT[dt])
    pre = [x[:1] for x in cache]
    for at in (0, 8, 3, 64, 1):
        q = store[..., at:at + D]
        want = kernels.int8_window_decode_attn(q.contiguous(), *cache, n, window=99, sinks=2)
        assert torch.equal(kernels.int8_window_decode_attn(q, *cache, n, window=99, sinks=2), want)
        want = kernels.int8_prefix_decode_attn(q.contiguous(), *pre, *cache, n)
        assert torch.equal(kernels.int8_prefix_decode_attn(q, *pre, *cache, n), want)
        want = kernels.int8_window_prefill_attn(q.contiguous(), *cache, n)
        assert torch.equal(kernels.int8_window_prefill_attn(q, *cache, n), want)
    # one query for all sequences
    q = store[:1, ..., :D].expand(2, 4, 1, D)
    want = kernels.int8_window_decode_attn(q.contiguous(), *cache, n)
    assert torch.equal(kernels.int8_window_decode_attn(q, *cache, n), want)


def test_largest_batch():
    g = torch.Generator(device="cuda").manual_seed(10)
    B, cap = 1024, 40
    cache = make_cache(g, B, 1, cap, "f16")
    lens = [(7 * b) % (cap + 1) for b in range(B)]
    for rep in (1, 8):
        q = torch.randn((B, rep, 1, D), generator=g, device="cuda").to(torch.bfloat16)
        got = kernels.int8_window_decode_attn(q, *cache, i32(lens), window=17, sinks=1)
        some = [0, 1, 5, 511, 1022, 1023]
        ref, tol = window_ref(q[some], [x[some] for x in cache], [lens[b] for b in some], [1] * 6, 17, 1, "bf16")
        check(got[some][:, :, 0], ref[:, 0], tol[:, 0], f"rep {rep}")
        assert (got[[b for b in range(B) if lens[b] == 0]] == 0).all()
    with pytest.raises(ValueError):
        kernels.int8_window_decode_attn(torch.cat([q, q[:1]]), *[torch.cat([x, x[:1]]) for x in cache],
                                        i32(lens + [1]))


def test_refusals():
    g = torch.Generator(device="cuda").manual_seed(11)
    cache = make_cache(g, 2, 2, 64, "f16")
    k, ksc, v, vsc = cache
    q = torch.randn((2, 4, 1, D), generator=g, device="cuda").to(torch.bfloat16)
    n = i32([64, 3])
    dec, pre = kernels.int8_window_decode_attn, kernels.int8_window_prefill_attn
    sh = kernels.int8_prefix_decode_attn
    kn = torch.randn((2, 2, 1, D), generator=g, device="cuda").to(torch.bfloat16)
    inv, _ = kernels.rope_inv_freq(D)
    odd = torch.zeros(k.numel() + 8, dtype=torch.int8, device="cuda")[8:].view_as(k)
    for call in (
            lambda: dec(q, *cache, n, window=0), lambda: dec(q, *cache, n, window=-1),
            lambda: dec(q, *cache, n, sinks=-1), lambda: dec(q, *cache, n, window=2.5),
            lambda: dec(q, *cache, n, sinks="2"), lambda: pre(q, *cache, n, window=1.0), lambda: dec(q, *cache, n, window=1 << 30),
            lambda: dec(q, *cache, n.long()), lambda: dec(q, *cache, n.cpu()),
            lambda: dec(q, *cache, i32([1])), lambda: dec(q.float(), *cache, n),
            lambda: dec(q[..., :64].contiguous(), k[..., :64].contiguous(), ksc[..., :64].contiguous(),
                        v[..., :64].contiguous(), vsc, n),
            lambda: dec(q, k.float(), ksc, v, vsc, n), lambda: dec(q, k, ksc.bfloat16(), v, vsc.bfloat16(), n),
            lambda: dec(q, k, ksc, v, vsc.float(), n), lambda: dec(q, k, ksc, v[:, :, :32], vsc, n),
            lambda: dec(q, k, ksc, v, vsc[:, :, :32], n), lambda: dec(q, k, ksc[:, :1], v, vsc, n),
            lambda: dec(q[:, :3], *cache, n), lambda: dec(q, odd, ksc, v, vsc, n),
            lambda: dec(q, k.cpu(), ksc, v, vsc, n), lambda: dec(q.repeat(1, 1, 2, 1), *cache, n),
            lambda: dec(q, *cache, n, out=torch.empty(2, 4, D, device="cuda")),
            lambda: dec(q, *cache, n, out=torch.empty(2, 4, 2 * D, device="cuda", dtype=q.dtype)[..., ::2]),
            lambda: pre(q[:, :, 0], *cache, n), lambda: pre(q, *cache, n, q_lens=i32([1])),
            lambda: pre(q, *cache, n, q_lens=n.long()),
            lambda: pre(q, *cache, n, out=torch.empty(2, 4, 1, D, device="cuda", dtype=q.dtype)),
            lambda: sh(q, *[x[:0] for x in cache], *cache, n),
            lambda: sh(q[:1].repeat(3, 1, 1, 1), *cache, *[x[:1].repeat(3, 1, 1, 1) for x in cache], i32([1, 1, 1])),
            lambda: sh(q, k[:1], ksc[:1].float(), v[:1], vsc[:1].float(), *cache, n),
            lambda: sh(q, *[x[:1, :1] for x in cache], *cache, n),
            lambda: sh(q, *[x[:1] for x in cache], *cache, n, prefix_lens=i32([1, 2])),
            lambda: kernels.rope_append_kv(q, kn, kn.float(), inv, k, v, ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn[:, :1], inv, k, v, ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn, inv.half(), k, v, ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn, inv.repeat(2), k, v, ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn, inv, k, v.transpose(1, 2), ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn, inv, odd, odd, ksc, vsc, n),
            lambda: kernels.rope_append_kv(q, kn, kn, inv, k, v, ksc, vsc, n, n_new=i32([1])),
            lambda: kernels.rope_append_kv(q, kn, kn, inv, k, v, ksc, vsc, n, q_out=q[:1])):
        with pytest.raises((ValueError, TypeError, _lib.HalftoneError)):
            call()
    torch.cuda.synchronize()
    assert kernels.ragged_status() == 0


def test_no_room_is_reported_and_reset():
    cache = empty_cache(2, 1, 16, "f16")
    g = torch.Generator(device="cuda").manual_seed(12)
    q, kn, vn = projections(g, 2, 2, 1, 4, "bf16")
    inv, _ = kernels.rope_inv_freq(D)
    kernels.rope_append_kv(q, kn, vn, inv, cache[0], cache[2], cache[1], cache[3], i32([13, 12]))
    assert kernels.ragged_status() == _lib.ERR_INVALID_ARGUMENT
    assert (cache[2][0] == 0).all() and (cache[3][1, :, 12:] > 0).all()
    kernels.reset_ragged_status()
    assert kernels.ragged_status() == 0
    # an error found on another stream is seen, too
    side = torch.cuda.Stream()
    full = i32([14, 14])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.rope_append_kv(q, kn, vn, inv, cache[0], cache[2], cache[1], cache[3], full)
    assert kernels.ragged_status() == _lib.ERR_INVALID_ARGUMENT
    kernels.reset_ragged_status()
    assert kernels.ragged_status() == 0
