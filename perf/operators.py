"""The operators of ragged serving over the int8 cache, case by case, for timing and comparison.

Four calls of one decode / prefill step whose sequences have lengths of their own:

* ``window_decode``   one new token per sequence, sliding window plus sink tokens;
* ``window_prefill``  a chunk of new tokens per sequence under the same mask;
* ``prefix_decode``   one new token per sequence over a prefix shared by a group and
                      the sequence's own tokens;
* ``rope_append``     rotary positions on q and k, k and v quantized into the cache.

With ``own`` false ``run`` computes them in elementary torch operations (float32; float64
for rotary angles and for codes next to a rounding border); with ``own`` true it calls the
package's public functions.  ``exact`` evaluates the definitions in float64.
"""
import math

import torch

own = False

D = 128          # head_dim of the package's decode attention
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- the cases
def listed():
    """Head counts, lengths and batch sizes are those of the repository's benchmark
    (16 q heads over 8 kv heads, 512 / 8192 / 32768 tokens, 64 sequences) or generic."""
    return [
        # a single chat turn: one sequence, small window; launch latency counts
        dict(name="window_decode 1x1024", op="window_decode", B=1, Hkv=8, rep=2, cap=4096, lo=4096,
             window=1024, sinks=4, dtype="bf16", sdtype="f16"),
        # batched serving at the benchmark's batch: every sequence past its window
        dict(name="window_decode 64x4096", op="window_decode", B=64, Hkv=8, rep=2, cap=8192,
             lo=4500, window=4096, sinks=4, dtype="bf16", sdtype="f16"),
        # ragged small batch, odd window, some sequences shorter than it, wider groups
        dict(name="window_decode 7x777 ragged", op="window_decode", B=7, Hkv=4, rep=4, cap=2501,
             lo=1, window=777, sinks=1, dtype="f16", sdtype="f32"),
        # the benchmark's prompt length in one chunk
        dict(name="window_prefill 512", op="window_prefill", B=1, Hkv=8, rep=2, Sq=512, qlo=512,
             cap=512, lo=512, window=256, sinks=4, dtype="bf16", sdtype="f16"),
        # long prompts, the window much shorter than the prompt
        dict(name="window_prefill 2x8192", op="window_prefill", B=2, Hkv=8, rep=2, Sq=8192,
             qlo=8192, cap=8192, lo=8192, window=2048, sinks=16, dtype="bf16", sdtype="f16"),
        # a padded batch of short chunks appended to long caches
        dict(name="window_prefill 5x77 ragged", op="window_prefill", B=5, Hkv=2, rep=6, Sq=77, qlo=1,
             cap=4099, lo=200, window=1000, sinks=3, dtype="f16", sdtype="f32"),
        # four samples of one short prompt
        dict(name="prefix_decode 4x512", op="prefix_decode", G=1, U=4, Hkv=8, rep=2, P=512, plo=512,
             cap=256, lo=1, dtype="bf16", sdtype="f16"),
        # a long system prompt under a full batch
        dict(name="prefix_decode 64x32768", op="prefix_decode", G=1, U=64, Hkv=8, rep=2, P=32768,
             plo=32768, cap=1024, lo=64, dtype="bf16", sdtype="f16"),
        # three groups with prefixes of their own odd lengths
        dict(name="prefix_decode 3x11 ragged", op="prefix_decode", G=3, U=11, Hkv=4, rep=8, P=5001,
             plo=1300, cap=333, lo=0, dtype="f16", sdtype="f32"),
        # one token of one sequence, and of a full batch
        dict(name="rope_append 1x1", op="rope_append", B=1, Hkv=8, rep=2, S=1, nlo=1, cap=4096,
             lo=4000, rot=128, inter=False, far=0, dtype="bf16", sdtype="f16"),
        # a ragged batch of prompts, part of each head rotated, interleaved pairs, far positions
        dict(name="rope_append 9x501 ragged", op="rope_append", B=9, Hkv=4, rep=3, S=501, nlo=1,
             cap=1003, lo=0, rot=64, inter=True, far=900000, dtype="f16", sdtype="f32"),
        # prompts of a full batch at once
        dict(name="rope_append 8x4096", op="rope_append", B=8, Hkv=8, rep=2, S=4096, nlo=4096,
             cap=8192, lo=0, rot=128, inter=False, far=0, dtype="bf16", sdtype="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window_decode", "window_prefill", "prefix_decode", "rope_append"])
    c = dict(op=op, Hkv=rng.choice([1, 2, 4, 8]), rep=rng.choice([1, 2, 3, 4, 6, 8]),
             dtype=rng.choice(["bf16", "f16"]), sdtype=rng.choice(["f16", "f32"]))
    heads = c["Hkv"] * c["rep"]
    if op == "window_decode":
        c["B"] = _log(rng, 1, 64)
        c["cap"] = _log(rng, 30, min(16384, 2_000_000 // (c["B"] * heads)))
        c["lo"] = rng.randint(0, c["cap"])
        c["window"] = _log(rng, 1, 8192)
        c["sinks"] = rng.choice([0, 1, 4, 37, 130])
    elif op == "window_prefill":
        c["B"] = _log(rng, 1, 8)
        c["Sq"] = _log(rng, 2, max(2, 8192 // c["B"]))
        c["qlo"] = rng.randint(1, c["Sq"])
        c["cap"] = min(16384, c["Sq"] + _log(rng, 1, 4096))
        c["lo"] = rng.randint(c["Sq"], c["cap"])
        c["window"] = _log(rng, 1, 4096)
        c["sinks"] = rng.choice([0, 1, 4, 37, 130])
        while c["B"] * heads * c["Sq"] * c["cap"] > 2 * 16 * 8192 * 8192:
            c["rep"], c["Hkv"] = max(1, c["rep"] // 2), max(1, c["Hkv"] // 2)
            heads = c["Hkv"] * c["rep"]
    elif op == "prefix_decode":
        c["G"] = rng.choice([1, 1, 2, 3])
        c["U"] = _log(rng, 1, max(1, 64 // c["G"]))
        c["P"] = _log(rng, 17, min(32768, 33_000_000 // (c["G"] * c["U"] * heads)))
        c["plo"] = rng.randint(c["P"] // 2, c["P"])
        c["cap"] = _log(rng, 16, 1024)
        c["lo"] = rng.randint(0, c["cap"])
    else:
        c["B"] = _log(rng, 1, 64)
        c["S"] = rng.choice([1, _log(rng, 1, max(1, 65536 // (c["B"] * c["Hkv"])))])
        c["nlo"] = rng.randint(0 if c["S"] > 1 else 1, c["S"])
        c["cap"] = c["S"] + _log(rng, 1, 2048)
        c["lo"] = 0
        c["rot"] = rng.choice([32, 64, 96, 128])
        c["inter"] = rng.random() < 0.5
        c["far"] = rng.choice([0, 0, 131072, 1000003])
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly: a ragged batch whose total does not depend on the seed."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shuffled(values, gen):
    order = torch.randperm(len(values), generator=gen).tolist()
    return [values[i] for i in order]


# ---------------------------------------------------------------- inputs
def _codes(shape, g, sigma):
    x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, sigma, generator=g)
    return x.round_().clamp_(-127, 127).to(torch.int8)


def _k_scale(B, Hkv, g, sdt):
    """Per-channel K scales of N(0,1) keys, four channels of each head twenty times larger."""
    s = torch.full((B, Hkv, 1, D), 4.4 / 127, device="cuda")
    s *= torch.empty_like(s).uniform_(0.8, 1.2, generator=g)
    hot = torch.rand((B, Hkv, 1, D), generator=g, device="cuda").topk(4, dim=-1).indices
    return s.scatter_(3, hot, s.gather(3, hot) * 20).to(sdt)


def _cache(B, Hkv, S, g, sdt):
    k, v = _codes((B, Hkv, S, D), g, 127 / 4.4), _codes((B, Hkv, S, D), g, 127 / 2.7)
    vs = torch.empty((B, Hkv, S, 1), device="cuda").uniform_(2.0 / 127, 3.4 / 127, generator=g)
    return k, _k_scale(B, Hkv, g, sdt), v, vs.to(sdt)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    cpu = torch.Generator().manual_seed(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, sdt = _DT[c["dtype"]], _DT[c["sdtype"]]
    Hkv, Hq = c["Hkv"], c["Hkv"] * c["rep"]
    s = dict(case=c)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    if c["op"] == "window_decode":
        s["q"] = normal(c["B"], Hq, 1, D)
        s["k"], s["ksc"], s["v"], s["vsc"] = _cache(c["B"], Hkv, c["cap"], g, sdt)
        s["lens"] = _ints(_shuffled(_spread(c["lo"], c["cap"], c["B"]), cpu))
    elif c["op"] == "window_prefill":
        s["q"] = normal(c["B"], Hq, c["Sq"], D)
        s["k"], s["ksc"], s["v"], s["vsc"] = _cache(c["B"], Hkv, c["cap"], g, sdt)
        # the shortest chunk continues the longest cache
        s["lens"] = _ints(_spread(c["lo"], c["cap"], c["B"])[::-1])
        s["q_lens"] = _ints(_spread(c["qlo"], c["Sq"], c["B"]))
        s["out"] = torch.zeros((c["B"], c["Sq"], Hq, D), dtype=dt, device="cuda")
    elif c["op"] == "prefix_decode":
        s["q"] = normal(c["G"] * c["U"], Hq, 1, D)
        s["pk"], s["pksc"], s["pv"], s["pvsc"] = _cache(c["G"], Hkv, c["P"], g, sdt)
        s["k"], s["ksc"], s["v"], s["vsc"] = _cache(c["G"] * c["U"], Hkv, c["cap"], g, sdt)
        s["plens"] = _ints(_spread(c["plo"], c["P"], c["G"]))
        s["lens"] = _ints(_shuffled(_spread(c["lo"], c["cap"], c["G"] * c["U"]), cpu))
    else:
        s["q"], s["kn"] = normal(c["B"], Hq, c["S"], D), normal(c["B"], Hkv, c["S"], D)
        s["vn"] = normal(c["B"], Hkv, c["S"], D)
        s["k"], s["v"] = (torch.zeros((c["B"], Hkv, c["cap"], D), dtype=torch.int8, device="cuda")
                          for _ in range(2))
        s["vsc"] = torch.zeros((c["B"], Hkv, c["cap"], 1), dtype=sdt, device="cuda")
        s["ksc"] = torch.empty((c["B"], Hkv, 1, D), device="cuda").uniform_(
            3.0 / 127, 4.8 / 127, generator=g).to(sdt)
        s["n_new"] = _ints(_spread(c["nlo"], c["S"], c["B"]))
        s["lens"] = _ints(_shuffled(_spread(c["lo"], c["cap"] - c["S"], c["B"]), cpu))
        s["pos_offset"] = _ints([c["far"]] * c["B"])
        s["inv_freq"] = (1.0 / 1e6 ** (torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])
                         ).to(device="cuda", dtype=torch.float32)
    return s


# ---------------------------------------------------------------- the pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_window_decode(s):
    from halftone_quantizedkvcache_b200 import kernels
    c = s["case"]
    return kernels.int8_window_decode_attn(s["q"], s["k"], s["ksc"], s["v"], s["vsc"], s["lens"],
                                           window=c["window"], sinks=c["sinks"])


def _own_window_prefill(s):
    from halftone_quantizedkvcache_b200 import kernels
    c = s["case"]
    return kernels.int8_window_prefill_attn(s["q"], s["k"], s["ksc"], s["v"], s["vsc"], s["lens"],
                                            window=c["window"], sinks=c["sinks"],
                                            q_lens=s["q_lens"], out=s["out"])


def _own_prefix_decode(s):
    from halftone_quantizedkvcache_b200 import kernels
    return kernels.int8_prefix_decode_attn(s["q"], s["pk"], s["pksc"], s["pv"], s["pvsc"], s["k"],
                                           s["ksc"], s["v"], s["vsc"], s["lens"],
                                           prefix_lens=s["plens"])


def _own_rope_append(s):
    from halftone_quantizedkvcache_b200 import kernels
    c = s["case"]
    q = kernels.rope_append_kv(s["q"], s["kn"], s["vn"], s["inv_freq"], s["k"], s["v"], s["ksc"],
                               s["vsc"], s["lens"], n_new=s["n_new"], pos_offset=s["pos_offset"],
                               interleaved=c["inter"])
    return {"q": q, "k": s["k"], "v": s["v"], "v_sc": s["vsc"]}


def _grouped_scores(q, k, ksc):
    """q [B,Hkv,rows,D] float32 against int8 keys [B,Hkv,S,D]: scaled scores [B,Hkv,rows,S]."""
    return torch.matmul(q * (ksc.float() / math.sqrt(D)), k.float().transpose(2, 3))


def _masked_softmax(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-1e30)  # a row that sees nothing gives zeros
    p = (scores - top).exp_()
    return p / p.sum(-1, keepdim=True).clamp_min_(1e-30)


def _plain_window_decode(s):
    c, q = s["case"], s["q"]
    B, Hq, cap = q.shape[0], q.shape[1], c["cap"]
    j, n = torch.arange(cap, device="cuda"), s["lens"][:, None].long()
    seen = (j < n) & ((j >= n - c["window"]) | (j < c["sinks"]))
    p = _grouped_scores(q.float().view(B, c["Hkv"], c["rep"], D), s["k"], s["ksc"])
    p = _masked_softmax(p, seen[:, None, None])
    o = torch.matmul(p * s["vsc"].float().transpose(2, 3), s["v"].float())
    return o.view(B, Hq, 1, D).to(q.dtype)


def _plain_window_prefill(s):
    c, q = s["case"], s["q"]
    B, Hq, Sq, cap = c["B"], q.shape[1], c["Sq"], c["cap"]
    i, j = torch.arange(Sq, device="cuda"), torch.arange(cap, device="cuda")
    pos = (s["lens"] - s["q_lens"])[:, None].long() + i          # [B, Sq]
    d = pos[:, :, None] - j                                      # distance to key j
    seen = (d >= 0) & ((d < c["window"]) | (j < c["sinks"]))
    rows = q.float().view(B, c["Hkv"], c["rep"] * Sq, D)
    p = _grouped_scores(rows, s["k"], s["ksc"]).view(B, c["Hkv"], c["rep"], Sq, cap)
    p = _masked_softmax(p, seen[:, None, None]).view(B, c["Hkv"], c["rep"] * Sq, cap)
    o = torch.matmul(p * s["vsc"].float().transpose(2, 3), s["v"].float())
    o = o.view(B, Hq, Sq, D).transpose(1, 2).to(q.dtype)
    live = (i < s["q_lens"][:, None])[:, :, None, None]
    return torch.where(live, o, s["out"])                        # padded rows stay as they were


def _plain_prefix_decode(s):
    c, q = s["case"], s["q"]
    G, U, Hkv, rep, P, cap = c["G"], c["U"], c["Hkv"], c["rep"], c["P"], c["cap"]
    qf = q.float().view(G * U, Hkv, rep, D)
    # the prefix once for all sequences of a group: [G, Hkv, U * rep, P]
    qg = qf.view(G, U, Hkv, rep, D).transpose(1, 2).reshape(G, Hkv, U * rep, D)
    sp = _grouped_scores(qg, s["pk"], s["pksc"])
    sp = sp.reshape(G, Hkv, U, rep, P).transpose(1, 2).reshape(G * U, Hkv, rep, P)
    so = _grouped_scores(qf, s["k"], s["ksc"])
    seen_p = torch.arange(P, device="cuda") < s["plens"][:, None]
    seen_p = seen_p.repeat_interleave(U, 0)
    seen_o = torch.arange(cap, device="cuda") < s["lens"][:, None]
    seen = torch.cat([seen_p, seen_o], 1)[:, None, None]
    p = _masked_softmax(torch.cat([sp, so], 3), seen)
    pp, po = p.split([P, cap], 3)
    pp = pp.reshape(G, U, Hkv, rep, P).transpose(1, 2).reshape(G, Hkv, U * rep, P)
    op = torch.matmul(pp * s["pvsc"].float().transpose(2, 3), s["pv"].float())
    op = op.reshape(G, Hkv, U, rep, D).transpose(1, 2).reshape(G * U, Hkv, rep, D)
    oo = torch.matmul(po * s["vsc"].float().transpose(2, 3), s["v"].float())
    return (op + oo).reshape(G * U, Hkv * rep, 1, D).to(q.dtype)


def _plain_rope_append(s):
    c = s["case"]
    B, S, cap, rot = c["B"], c["S"], c["cap"], c["rot"]
    i = torch.arange(S, device="cuda")
    pos = (s["lens"] + s["pos_offset"])[:, None].long() + i      # [B, S]
    ang = pos[:, None, :, None].double() * s["inv_freq"].double()
    cos, sin = ang.cos(), ang.sin()

    def rotate(x):
        x = x.double()
        y = x.clone()
        if c["inter"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
        return y

    live = (i < s["n_new"][:, None])[:, None, :, None]
    q = torch.where(live, rotate(s["q"]).to(s["q"].dtype), s["q"])
    kc = (rotate(s["kn"]) / s["ksc"].double()).round().clamp(-127, 127).to(torch.int8)
    v = s["vn"].float()
    vs = v.abs().amax(-1, keepdim=True).clamp_min(1e-8) / torch.full((), 127.0, device="cuda")
    vc = (v / vs).round().clamp(-127, 127).to(torch.int8)
    # rows lens[b] .. lens[b] + n_new[b] - 1 of the cache; the others stay as they were
    r = torch.arange(cap, device="cuda") - s["lens"][:, None]    # [B, cap]: which new token
    here = ((r >= 0) & (r < s["n_new"][:, None]))[:, None, :, None]
    at = r.clamp(0, S - 1)[:, None, :, None].expand(B, c["Hkv"], cap, 1)
    for name, new in (("k", kc), ("v", vc), ("vsc", vs.to(s["vsc"].dtype))):
        old = s[name]
        picked = new.gather(2, at.expand(B, c["Hkv"], cap, old.shape[3]))
        s[name].copy_(torch.where(here, picked, old))
    return {"q": q, "k": s["k"], "v": s["v"], "v_sc": s["vsc"]}


_OWN = dict(window_decode=_own_window_decode, window_prefill=_own_window_prefill,
            prefix_decode=_own_prefix_decode, rope_append=_own_rope_append)
_PLAIN = dict(window_decode=_plain_window_decode, window_prefill=_plain_window_prefill,
              prefix_decode=_plain_prefix_decode, rope_append=_plain_rope_append)


# ---------------------------------------------------------------- what a pass cannot do without
def _visible(n, window, sinks):
    """Keys that the query at position n - 1 sees among n."""
    return min(n, window) + max(0, min(sinks, n - window))


def work(case):
    c = case
    Hkv, rep = c["Hkv"], c["rep"]
    eb, sb = 2, 2 if c["sdtype"] == "f16" else 4
    key = Hkv * (2 * D + sb)                                     # a cached token's codes and V scales
    if c["op"] == "window_decode":
        n = sum(_visible(x, c["window"], c["sinks"]) for x in _spread(c["lo"], c["cap"], c["B"]))
        return {"bytes": n * key + c["B"] * Hkv * D * (sb + 2 * rep * eb),
                "flops": 4 * n * Hkv * rep * D}
    if c["op"] == "window_prefill":
        keys = pairs = rows = 0
        for n, m in zip(_spread(c["lo"], c["cap"], c["B"])[::-1], _spread(c["qlo"], c["Sq"], c["B"])):
            first = max(0, n - m - c["window"] + 1)              # the oldest key in any row's window
            keys += n - first + min(first, c["sinks"])
            pairs += sum(_visible(p, c["window"], c["sinks"]) for p in range(n - m + 1, n + 1))
            rows += m
        return {"bytes": keys * key + c["B"] * Hkv * D * sb + 2 * rows * Hkv * rep * D * eb,
                "flops": 4 * pairs * Hkv * rep * D}
    if c["op"] == "prefix_decode":
        p, n = sum(_spread(c["plo"], c["P"], c["G"])), sum(_spread(c["lo"], c["cap"], c["G"] * c["U"]))
        return {"bytes": (p + n) * key + (c["G"] + c["G"] * c["U"]) * Hkv * D * sb
                + 2 * c["G"] * c["U"] * Hkv * rep * D * eb,
                "flops": 4 * (p * c["U"] + n) * Hkv * rep * D}
    n = sum(_spread(c["nlo"], c["S"], c["B"]))
    return {"bytes": n * Hkv * D * (2 * rep * eb + 2 * eb + 2) + n * Hkv * sb + c["B"] * Hkv * D * sb,
            "flops": 6 * n * Hkv * (rep + 1) * c["rot"] // 2 + 4 * n * Hkv * D}


# ---------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "rope_append":
        return _exact_rope(s)
    rep, lens = c["rep"], s["lens"].tolist()
    if c["op"] == "window_prefill":
        q_lens, out = s["q_lens"].tolist(), s["out"].double()
        for b in range(c["B"]):
            n, m = lens[b], q_lens[b]
            pos = torch.arange(n - m, n, device="cuda")
            j = torch.arange(n, device="cuda")
            mask = (j[None] <= pos[:, None]) & ((pos[:, None] - j[None] < c["window"]) | (j[None] < c["sinks"]))
            for h in range(c["Hkv"] * rep):
                kh = h // rep
                k = s["k"][b, kh, :n].double() * s["ksc"][b, kh].double()
                v = s["v"][b, kh, :n].double() * s["vsc"][b, kh, :n].double()
                out[b, :m, h] = _attend64(s["q"][b, h, :m].double(), k, v, mask)
        return out
    B = s["q"].shape[0]
    out = torch.zeros((B, c["Hkv"] * rep, 1, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        for kh in range(c["Hkv"]):
            k = s["k"][b, kh, :n].double() * s["ksc"][b, kh].double()
            v = s["v"][b, kh, :n].double() * s["vsc"][b, kh, :n].double()
            if c["op"] == "prefix_decode":
                g = b // c["U"]
                m = int(s["plens"][g])
                k = torch.cat([s["pk"][g, kh, :m].double() * s["pksc"][g, kh].double(), k])
                v = torch.cat([s["pv"][g, kh, :m].double() * s["pvsc"][g, kh, :m].double(), v])
                mask = torch.ones((1, len(k)), dtype=torch.bool, device="cuda")
            else:
                j = torch.arange(n, device="cuda")
                mask = ((j > n - 1 - c["window"]) | (j < c["sinks"]))[None]
            if len(k):
                q = s["q"][b, kh * rep:(kh + 1) * rep, 0].double()
                out[b, kh * rep:(kh + 1) * rep, 0] = _attend64(q, k, v, mask)
    return out


def _attend64(q, k, v, mask):
    z = (q @ k.T) / math.sqrt(D)
    z = torch.where(mask, z, torch.full_like(z, -math.inf))
    return torch.softmax(z, dim=-1) @ v


def _exact_rope(s):
    """Rotations as complex products; codes are whole numbers and come from the quotient's nearest integer."""
    c = s["case"]
    q, k, v, vsc = s["q"].double(), s["k"], s["v"], s["vsc"].double()
    half = c["rot"] // 2
    for b in range(c["B"]):
        n, row = int(s["n_new"][b]), int(s["lens"][b])
        pos = torch.arange(row, row + n, device="cuda", dtype=torch.float64) + float(s["pos_offset"][b])
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(pos, s["inv_freq"].double()))

        def spin(x):
            x = x.double()
            head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            if c["inter"]:
                z = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * turn
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :half], head[..., half:]) * turn
                head = torch.cat([z.real, z.imag], -1)
            return torch.cat([head, rest], -1)

        q[b, :, :n] = spin(s["q"][b, :, :n])
        k[b, :, row:row + n] = torch.clamp(torch.round(spin(s["kn"][b, :, :n]) / s["ksc"][b].double()),
                                           -127, 127).to(torch.int8)
        x = s["vn"][b, :, :n].float()
        sc = torch.maximum(x.abs().amax(-1, keepdim=True), torch.full((), 1e-8, device="cuda")).div(
            torch.full((), 127.0, device="cuda"))
        v[b, :, row:row + n] = torch.clamp(torch.round(x / sc), -127, 127).to(torch.int8)
        vsc[b, :, row:row + n] = sc.double()
    return {"q": q, "k": k, "v": v, "v_sc": vsc}
