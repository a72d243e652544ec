"""Calls of the ragged-batch operators at the edges of what their documentation allows, on the
GPU.  Bounds as in test_ragged_gpu."""
import math
import threading

import pytest
import torch

from halftone_quantizedkvcache_b200 import _lib, kernels
from test_ragged_gpu import D, TDT, check, make_cache, ref_rows, window_ref

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


INT_MAX = 2 ** 31 - 1


def c_window(q, cache, lens, window, sinks):
    """The C entries of the windowed attention, whose window and sinks are any int: decode for
    q [B,Hq,D], prefill for q [B,Hq,Sq,D] (output [B,Sq,Hq,D])."""
    k, ksc, v, vsc = cache
    B, Hkv, cap = k.shape[:3]
    Hq, Sq = q.shape[1], q.shape[2] if q.dim() == 4 else 0
    dt, st = kernels._DT[q.dtype], lambda t, n=3: _lib.strides(t.stride()[:n], n)
    nb = _lib.lib().hq_window_workspace_bytes(dt, B, Hq, Hkv, Sq, cap, D, window, sinks)
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kss, vss = _lib.strides((ksc.stride(0), ksc.stride(1), ksc.stride(3)), 3), st(vsc)
    common = (st(k), ksc.data_ptr(), vsc.data_ptr(), kernels._DT[ksc.dtype], kss, vss, lens.data_ptr())
    tail = (D, window, sinks, 1 / math.sqrt(D), 0)
    stream = torch.cuda.current_stream().cuda_stream
    if Sq:
        out = torch.empty((B, Sq, Hq, D), dtype=q.dtype, device="cuda")
        rc = _lib.lib().hq_window_prefill_int8(
            q.data_ptr(), dt, st(q, 4), k.data_ptr(), v.data_ptr(), *common, None, B, Hq, Hkv, Sq, cap,
            *tail, out.data_ptr(), st(out.transpose(1, 2), 4), ws.data_ptr(), nb, status.data_ptr(), stream)
    else:
        out = torch.empty((B, Hq, D), dtype=q.dtype, device="cuda")
        rc = _lib.lib().hq_window_decode_int8(
            q.data_ptr(), dt, st(q), k.data_ptr(), v.data_ptr(), *common, B, Hq, Hkv, cap,
            *tail, out.data_ptr(), st(out), ws.data_ptr(), nb, status.data_ptr(), stream)
    assert rc == 0 and status.item() == 0
    return out


@pytest.mark.parametrize("rep", [2, 8])
@pytest.mark.parametrize("window,sinks", [
    (0, INT_MAX), (100, INT_MAX), (INT_MAX, 0), (INT_MAX, INT_MAX), (100, INT_MAX - 7),
    (1 << 30, 1 << 30), ((1 << 30) + 1, (1 << 30) + 1)])
def test_windows_and_sinks_up_to_the_largest_int(rep, window, sinks):
    """All of these let every query see every key before it."""
    g = torch.Generator(device="cuda").manual_seed(rep)
    lens = [300, 0, 17]
    cache = make_cache(g, 3, 2, 300, "f16")
    q = torch.randn((3, 2 * rep, D), generator=g, device="cuda").to(torch.bfloat16)
    got = c_window(q, cache, i32(lens), window, sinks)
    ref, tol = window_ref(q[:, :, None], cache, lens, [1] * 3, None, 0, "bf16")
    check(got, ref[:, 0], tol[:, 0], "decode")
    # 40 queries each: those of the last two sequences begin before position 0
    q = torch.randn((3, 2 * rep, 40, D), generator=g, device="cuda").to(torch.bfloat16)
    got = c_window(q, cache, i32(lens), window, sinks)
    ref, tol = window_ref(q, cache, lens, [40] * 3, None, 0, "bf16")
    check(got, ref, tol, "prefill")


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("rep", [1, 2, 4, 8])
def test_an_empty_cache_needs_no_pointers(rep, dt):
    """Capacity 0, codes and scales NULL: zeros from every entry, and no read."""
    L, B, Hkv, one = _lib.lib(), 3, 2, _lib.strides((D, D, 1), 3)
    Hq, t = Hkv * rep, kernels._DT[TDT[dt]]
    lens = i32([0, 5, 1])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    rows = _lib.strides((D, D, D), 3)
    none = (None, None, rows, None, None, kernels._DT[torch.float16], one, one)
    q = torch.randn((B, Hq, 9, D), device="cuda").to(TDT[dt])
    end = (ws.data_ptr(), ws.numel(), status.data_ptr(), stream)
    st3, st4 = _lib.strides((Hq * D, D, 1), 3), _lib.strides((Hq * 9 * D, 9 * D, D, 1), 4)
    out = torch.ones((B, Hq, D), dtype=TDT[dt], device="cuda")
    assert L.hq_window_decode_int8(q.data_ptr(), t, st3, *none, lens.data_ptr(), B, Hq, Hkv, 0, D, 7, 1,
                                   0.1, 1, out.data_ptr(), st3, *end) == 0
    assert (out == 0).all()
    wide = torch.ones_like(q)
    assert L.hq_window_prefill_int8(q.data_ptr(), t, st4, *none, lens.data_ptr(), None, B, Hq, Hkv, 9, 0, D,
                                    7, 1, 0.1, 1, wide.data_ptr(), st4, *end) == 0
    assert (wide == 0).all()
    out.fill_(1)
    empty = (None, None, rows, None, None, one, one)
    assert L.hq_prefix_decode_int8(q.data_ptr(), t, st3, *empty, None, 1, 0, *empty, lens.data_ptr(), 0,
                                   kernels._DT[torch.float16], B, Hq, Hkv, D, 0.1, 0, out.data_ptr(), st3,
                                   *end) == 0
    assert (out == 0).all() and status.item() == 0


@pytest.mark.parametrize("dt,sdt,rep", [("bf16", "f16", 8), ("f16", "f32", 8), ("bf16", "f32", 5), ("bf16", "f16", 2)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2500, 9)])
def test_many_tiles_of_one_sequence_to_a_block(rep, dt, sdt, window, sinks):
    """Batches of long caches: a block walks tens of tiles, whole sequences and parts of two."""
    g = torch.Generator(device="cuda").manual_seed(rep)
    B, Hkv, cap = 48, 4, 4000
    cache = make_cache(g, B, Hkv, cap, sdt)
    lens = [(977 * b * b + 13) % (cap + 1) for b in range(B)]
    lens[5], lens[6], lens[40] = cap, 0, cap
    q = torch.randn((B, Hkv * rep, 1, D), generator=g, device="cuda").to(TDT[dt])
    got = kernels.int8_window_decode_attn(q, *cache, i32(lens), window=window, sinks=sinks)
    some = [0, 1, 5, 6, 7, 23, 24, 40, 47]
    ref, tol = window_ref(q[some], [x[some] for x in cache], [lens[b] for b in some], [1] * len(some), window,
                          sinks, dt)
    check(got[some][:, :, 0], ref[:, 0], tol[:, 0], "decode")
    assert kernels.ragged_status() == 0


def test_two_threads_at_once():
    """Two threads on streams of their own make the same calls: each gets its own results."""
    g = torch.Generator(device="cuda").manual_seed(2)
    sets = []
    for i in range(2):
        cache = make_cache(g, 6, 2, 900, "f16")
        n = i32([(331 * (b + 1 + i)) % 900 for b in range(6)])
        q = torch.randn((6, 16, 20, D), generator=g, device="cuda").to(torch.bfloat16)
        sets.append((cache, n, q))

    def calls(cache, n, q):
        few, one = q[:, :4, :1].contiguous(), q[:, :, :1].contiguous()
        return [kernels.int8_window_decode_attn(few, *cache, n, window=500, sinks=4),
                kernels.int8_window_decode_attn(one, *cache, n),
                kernels.int8_window_prefill_attn(q, *cache, n, window=300, sinks=2),
                kernels.int8_prefix_decode_attn(one, *[x[:1] for x in cache], *cache, n)]

    want = [calls(*s) for s in sets]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(2), []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(40):
                    got = calls(*sets[i])
                    torch.cuda.current_stream().synchronize()
                    wrong.extend(k for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
        except Exception as e:  # noqa: BLE001 - reported by the assertion below
            wrong.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and kernels.ragged_status() == 0
