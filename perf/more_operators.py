"""The operators of a paged cache held in 4 bits, and of the packed prompts that fill it, case by
case, for timing and comparison.

* ``append``   q and k normed per head (optional) and rotated (optional), k and v coded in 4 bits
               into the pages of their sequences: prompts, chunks or one token per sequence; and the
               new tokens read back, as every later step sees them;
* ``decode``   one new token per sequence over the pages;
* ``gather``   the pages' tokens as packed 16-bit rows (what a chunk over a cached past attends);
* ``prefill``  causal attention of packed sequences of different lengths, 16-bit K and V.

With ``own`` false ``run`` computes them in elementary torch operations (float32; float64 for
norms, rotary angles and codes next to a rounding border); with ``own`` true it calls the package's
public functions.  ``exact`` evaluates the definitions in float64.

The cache.  Per token and kv head 128 channels in 4 groups of 32: scale ``s = f16(amax / 7.5)``,
codes ``clamp(rint(x / s), -8, 7)``, values ``s * code``.  Code rows have 64 bytes: the 16 bytes at
position p hold chunk ``j = p ^ 2 * ((t >> 1) & 1)`` (t: the token's place in its page), whose four
32-bit words are the groups' channels ``32 g + 8 j + i``, i = 0 .. 7, as ``code + 8`` in bits
``4 i .. 4 i + 3``.
"""
import math

import torch

own = False

D = 128
GROUP = 32
_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- the cases
def listed():
    """Head counts, lengths and batch sizes are those of the repository's benchmark
    (16 q heads over 8 kv heads, 512 / 8192 tokens, 64 sequences) or generic."""
    return [
        # one new token of one chat turn: launch latency counts
        dict(name="append 1x1", op="append", B=1, Hkv=8, rep=2, S=1, nlo=1, past=4000, plo=4000,
             page=64, rot=128, inter=False, norm=True, kout=False, far=0, dtype="bf16"),
        # a packed batch of short prompts, part of each head rotated in interleaved pairs, far
        # positions, no norms, small pages
        dict(name="append 9x501 ragged", op="append", B=9, Hkv=4, rep=3, S=501, nlo=1, past=502,
             plo=0, page=16, rot=64, inter=True, norm=False, kout=True, far=900000, dtype="f16"),
        # prompts of a full batch, their rotated keys kept for the prompt's own attention
        dict(name="append 8x4096", op="append", B=8, Hkv=8, rep=2, S=4096, nlo=4096, past=0, plo=0,
             page=64, rot=128, inter=False, norm=True, kout=True, far=0, dtype="bf16"),
        # one chat turn
        dict(name="decode 1x512", op="decode", B=1, Hkv=8, rep=2, cap=512, lo=512, page=64,
             dtype="bf16"),
        # a small ragged batch, wider groups, small pages, an empty sequence
        dict(name="decode 7x2501 ragged", op="decode", B=7, Hkv=4, rep=4, cap=2501, lo=0, page=16,
             dtype="f16"),
        # the benchmark's batched serving
        dict(name="decode 64x8192", op="decode", B=64, Hkv=8, rep=2, cap=8192, lo=4096, page=64,
             dtype="bf16"),
        # the pasts of a few chunks
        dict(name="gather 5x4099 ragged", op="gather", B=5, Hkv=2, cap=4099, lo=200, page=32,
             dtype="f16"),
        # long pasts of a batch
        dict(name="gather 8x8192", op="gather", B=8, Hkv=8, cap=8192, lo=8192, page=64, dtype="bf16"),
        # the benchmark's prompt length
        dict(name="prefill 512", op="prefill", B=1, Hkv=8, rep=2, S=512, nlo=512, past=0, plo=0,
             dtype="bf16"),
        # a packed batch of short prompts, three q heads to a kv head
        dict(name="prefill 9x501 ragged", op="prefill", B=9, Hkv=4, rep=3, S=501, nlo=1, past=0, plo=0,
             dtype="f16"),
        # chunks of a few dozen tokens over long pasts
        dict(name="prefill 3x77 over 4022", op="prefill", B=3, Hkv=2, rep=6, S=77, nlo=20, past=4022,
             plo=1000, dtype="f16"),
        # two long prompts
        dict(name="prefill 2x8192", op="prefill", B=2, Hkv=8, rep=2, S=8192, nlo=8192, past=0, plo=0,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "gather", "prefill"])
    c = dict(op=op, Hkv=rng.choice([1, 2, 4, 8]), dtype=rng.choice(["bf16", "f16"]))
    if op != "gather":
        c["rep"] = rng.choice([1, 2, 3, 4, 6, 8])
    heads = c["Hkv"] * c.get("rep", 1)
    if op != "prefill":
        c["page"] = rng.choice([16, 32, 64, 128])
    if op == "append":
        c["B"] = _log(rng, 1, 64)
        c["S"] = rng.choice([1, _log(rng, 1, max(1, 1_000_000 // (c["B"] * (heads + 2 * c["Hkv"]))))])
        c["nlo"] = rng.randint(0 if c["S"] > 1 else 1, c["S"])
        c["past"] = _log(rng, 1, 2048)
        c["plo"] = rng.randint(0, c["past"])
        c["rot"] = rng.choice([32, 64, 96, 128])
        c["inter"], c["norm"], c["kout"] = (rng.random() < 0.5 for _ in range(3))
        c["far"] = rng.choice([0, 0, 131072, 1000003])
    elif op == "decode":
        c["B"] = _log(rng, 1, 64)
        c["cap"] = _log(rng, 1, min(131072, 64 * 16 * 8192 // (c["B"] * heads)))
        c["lo"] = rng.randint(0, c["cap"])
    elif op == "gather":
        c["B"] = _log(rng, 1, 64)
        c["cap"] = _log(rng, 1, min(32768, 8 * 8 * 8192 // (c["B"] * c["Hkv"])))
        c["lo"] = rng.randint(0, c["cap"])
    else:
        c["B"] = _log(rng, 1, 16)
        c["S"] = _log(rng, 1, 8192)
        c["nlo"] = rng.randint(0, c["S"])
        c["past"] = rng.choice([0, _log(rng, 1, 8192)])
        c["plo"] = rng.randint(0, c["past"])
        while c["B"] * heads * c["S"] * (c["S"] + c["past"]) > 2 * 16 * 8192 * 8192:
            if c["B"] > 1:
                c["B"] //= 2
            elif c["past"] > c["S"]:
                c["past"] //= 2
                c["plo"] //= 2
            else:
                c["S"] //= 2
                c["nlo"] //= 2
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly: a ragged batch whose total does not depend on the seed."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


# ---------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cum(values):
    return _ints([0] + torch.tensor(values, dtype=torch.int64).cumsum(0).tolist())


def _codes(shape, g):
    """Bytes of two codes of N(0, 3), as groups scaled by their largest value have them."""
    out = torch.empty(shape, dtype=torch.uint8, device="cuda")
    x = torch.empty(shape, dtype=torch.float16, device="cuda")
    out.copy_(x.normal_(0.0, 3.0, generator=g).round_().clamp_(-8, 7).add_(8))
    hi = x.normal_(0.0, 3.0, generator=g).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    return out.bitwise_or_(hi.bitwise_left_shift_(4))


def _pages(n_seq, cap, page):
    """Page counts of n_seq tables for cap tokens each."""
    per = max(1, -(-cap // page))
    return per, n_seq * per


def _cache(B, cap, page, Hkv, g, filled):
    per, n = _pages(B, cap, page)
    n += 3                                                   # a pool is never exactly full
    c = {}
    for name in ("k", "v"):
        if filled:
            c[name] = _codes((n, Hkv, page, D // 2), g)
            sc = torch.empty((n, Hkv, page, D // GROUP), device="cuda").uniform_(0.2, 0.4, generator=g)
            if name == "k":  # channels of large keys: one group of each head is three times larger
                sc[..., 1] *= 3.0
            c[name + "_scale"] = sc.to(torch.float16)
        else:
            c[name] = torch.zeros((n, Hkv, page, D // 2), dtype=torch.uint8, device="cuda")
            c[name + "_scale"] = torch.zeros((n, Hkv, page, D // GROUP), dtype=torch.float16, device="cuda")
    order = torch.randperm(n, generator=g, device="cuda")[:B * per]
    return c, order.view(B, per).to(torch.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, B, Hkv = _DT[c["dtype"]], c["B"], c["Hkv"]
    Hq = Hkv * c.get("rep", 1)
    s = dict(case=c)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    if c["op"] == "append":
        new, past = _spread(c["nlo"], c["S"], B), _spread(c["plo"], c["past"], B)[::-1]
        T = sum(new)
        qkv = normal(T, (Hq + 2 * Hkv) * D)                  # the fused projection's output
        s["q"], s["kn"], s["vn"] = (x.unflatten(1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
        s["cache"], s["tables"] = _cache(B, c["past"] + c["S"], c["page"], Hkv, g, False)
        s["lens"], s["cu"] = _ints(past), _cum(new)
        s["after"] = _ints([a + b for a, b in zip(past, new)])
        s["inv_freq"] = (1.0 / 1e6 ** (torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])
                         ).to(device="cuda", dtype=torch.float32)
        s["pos_offset"] = _ints([c["far"]] * B)
        for name in ("qw", "kw"):
            s[name] = torch.empty(D, device="cuda").uniform_(0.5, 2.0, generator=g).to(dt) if c["norm"] else None
        s["k_out"] = torch.zeros((T, Hkv, D), dtype=dt, device="cuda") if c["kout"] else None
    elif c["op"] == "decode":
        s["q"] = normal(B, Hq, D)
        s["cache"], s["tables"] = _cache(B, c["cap"], c["page"], Hkv, g, True)
        lens = _ints(_spread(c["lo"], c["cap"], B))
        s["lens"] = lens[torch.randperm(B, generator=g, device="cuda")].contiguous()
    elif c["op"] == "gather":
        s["cache"], s["tables"] = _cache(B, c["cap"], c["page"], Hkv, g, True)
        lens = _spread(c["lo"], c["cap"], B)
        s["lens"], s["cu"], s["rows"] = _ints(lens), _cum(lens), sum(lens)
    else:
        new, past = _spread(c["nlo"], c["S"], B), _spread(c["plo"], c["past"], B)[::-1]
        both = [a + b for a, b in zip(new, past)]
        s["q"] = normal(sum(new), Hq, D)
        s["k"], s["v"] = normal(sum(both), Hkv, D), normal(sum(both), Hkv, D)
        s["cu_q"], s["cu_k"] = _cum(new), _cum(both)
    return s


# ---------------------------------------------------------------- the pass
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_append(s):
    from halftone_quantizedkvcache_b200 import kernels
    q = kernels.paged4_append(s["q"], s["kn"], s["vn"], s["cache"], s["tables"], s["lens"],
                              cu_seqlens=s["cu"], inv_freq=s["inv_freq"], interleaved=s["case"]["inter"],
                              pos_offset=s["pos_offset"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                              k_out=s["k_out"])
    k, v = kernels.paged4_gather(s["cache"], s["tables"], s["after"], s["cu"], q.shape[0],
                                 first=s["lens"], dtype=q.dtype)
    return _appended(s, q, k, v)


def _appended(s, q, k, v):
    out = {"q": q, "k": k, "v": v}
    if s["k_out"] is not None:
        out["k_new"] = s["k_out"]
    return out


def _own_decode(s):
    from halftone_quantizedkvcache_b200 import kernels
    return kernels.paged4_decode_attn(s["q"], s["cache"], s["tables"], s["lens"])


def _own_gather(s):
    from halftone_quantizedkvcache_b200 import kernels
    k, v = kernels.paged4_gather(s["cache"], s["tables"], s["lens"], s["cu"], s["rows"],
                                 dtype=_DT[s["case"]["dtype"]])
    return {"k": k, "v": v}


def _own_prefill(s):
    from halftone_quantizedkvcache_b200 import kernels
    return kernels.packed_prefill_attn(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])


def _swap(rows, t):
    """Code rows [.., 4 chunks, ..] at places t of a page: chunks as stored <-> in order."""
    return torch.where(((t >> 1) & 1).bool()[..., None, None, None], rows.roll(2, -3), rows)


def _unpack(codes, t):
    """Code rows uint8 [.., 64] at places t: codes -8 .. 7 as float32 [.., 128]."""
    b = codes.view(*codes.shape[:-1], 4, 4, 4)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)        # [.., position, group, 8]
    return (_swap(n, t).transpose(-3, -2).flatten(-3).float() - 8)


def _pack(codes, t):
    """The other way round: codes [.., 128] to uint8 [.., 64]."""
    n = (codes + 8).to(torch.uint8).unflatten(-1, (4, 4, 8)).transpose(-3, -2)
    n = _swap(n, t).unflatten(-1, (4, 2))
    return (n[..., 0] | n[..., 1] << 4).flatten(-3)


def _quantize(x):
    """x float64 [.., 128]: codes, scales."""
    g = x.unflatten(-1, (4, GROUP))
    sc = (g.abs().amax(-1, keepdim=True) / 7.5).to(torch.float16)
    c = (g / sc.double().clamp_min(1e-30)).round().clamp(-8, 7)
    return c.flatten(-2), sc.squeeze(-1)


def _rows_of(cu, n):
    """Which sequence each of n packed rows belongs to, and its place there."""
    r = torch.arange(n, device="cuda")
    b = torch.searchsorted(cu[1:].long(), r, right=True)
    return b, r - cu.long()[b]


def _plain_append(s):
    c = s["case"]
    rot, T = c["rot"], s["q"].shape[0]
    b, i = _rows_of(s["cu"], T)
    at = s["lens"].long()[b] + i
    ang = (at + s["pos_offset"].long()[b])[:, None, None].double() * s["inv_freq"].double()
    cos, sin = ang.cos(), ang.sin()

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
        y = x.clone()
        if c["inter"]:
            u, v = x[..., 0:rot:2], x[..., 1:rot:2]
            y[..., 0:rot:2], y[..., 1:rot:2] = u * cos - v * sin, v * cos + u * sin
        else:
            u, v = x[..., :rot // 2], x[..., rot // 2:rot]
            y[..., :rot // 2], y[..., rot // 2:rot] = u * cos - v * sin, v * cos + u * sin
        return y

    q, k = turned(s["q"], s["qw"]).to(s["q"].dtype), turned(s["kn"], s["kw"])  # k stays in float64
    page, t = s["tables"].long()[b, at // c["page"]], at % c["page"]
    place = t[:, None].expand(T, c["Hkv"])
    held = {}
    for name, x in (("k", k), ("v", s["vn"].double())):
        codes, sc = _quantize(x)
        s["cache"][name][page, :, t] = _pack(codes, place)
        s["cache"][name + "_scale"][page, :, t] = sc
        codes, sc = _unpack(s["cache"][name][page, :, t], place), s["cache"][name + "_scale"][page, :, t]
        held[name] = (codes.unflatten(-1, (4, GROUP)) * sc.float()[..., None]).flatten(-2).to(q.dtype)
    if s["k_out"] is not None:
        s["k_out"].copy_(k)
    return _appended(s, q, **held)


def _values(s, name):
    """All tokens of the tables' pages: float32 [B, Hkv, tokens, 128]."""
    page = s["cache"][name].shape[2]
    t = torch.arange(page, device="cuda")
    codes, sc = s["cache"][name][s["tables"].long()], s["cache"][name + "_scale"][s["tables"].long()]
    x = _unpack(codes, t.expand(codes.shape[:-1])).unflatten(-1, (4, GROUP)) * sc.float()[..., None]
    return x.flatten(-2).transpose(1, 2).flatten(2, 3)


def _softmax(scores, seen):
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min_(-1e30)    # a row that sees nothing gives zeros
    p = (scores - top).exp_()
    return p / p.sum(-1, keepdim=True).clamp_min_(1e-30)


def _plain_decode(s):
    c, q = s["case"], s["q"]
    k, v = _values(s, "k"), _values(s, "v")
    z = torch.matmul(q.float().view(c["B"], c["Hkv"], c["rep"], D) / math.sqrt(D), k.transpose(2, 3))
    seen = torch.arange(k.shape[2], device="cuda") < s["lens"][:, None]
    return torch.matmul(_softmax(z, seen[:, None, None]), v).view(q.shape).to(q.dtype)


def _plain_gather(s):
    b, i = _rows_of(s["cu"], s["rows"])
    dt = _DT[s["case"]["dtype"]]
    return {name: _values(s, name)[b, :, i].to(dt) for name in ("k", "v")}


def _padded(x, cu, n, most):
    """Packed rows [T, H, D] as float32 [B, H, most, D]."""
    at = (cu[:-1, None].long() + torch.arange(most, device="cuda")).clamp_max_(max(x.shape[0] - 1, 0))
    return x[at].float().transpose(1, 2)


def _plain_prefill(s):
    c, q = s["case"], s["q"]
    if q.shape[0] == 0:
        return torch.empty_like(q)
    cu_q, cu_k, B, Hkv, rep = s["cu_q"], s["cu_k"], c["B"], c["Hkv"], c["rep"]
    nq, nk = cu_q.diff().long(), cu_k.diff().long()
    Sq, Sk = c["S"], c["past"] + c["S"]
    qp = _padded(q, cu_q, nq, Sq) / math.sqrt(D)
    kp, vp = _padded(s["k"], cu_k, nk, Sk), _padded(s["v"], cu_k, nk, Sk)
    i, j = torch.arange(Sq, device="cuda"), torch.arange(Sk, device="cuda")
    seen = (j <= (nk - nq)[:, None, None] + i[:, None]) & (j < nk[:, None, None])
    z = torch.matmul(qp.reshape(B, Hkv, rep * Sq, D), kp.transpose(2, 3)).view(B, Hkv, rep, Sq, Sk)
    p = _softmax(z, seen[:, None, None]).view(B, Hkv, rep * Sq, Sk)
    o = torch.matmul(p, vp).view(B, Hkv * rep, Sq, D)
    b, i = _rows_of(cu_q, q.shape[0])
    return o[b, :, i].to(q.dtype)


_OWN = dict(append=_own_append, decode=_own_decode, gather=_own_gather, prefill=_own_prefill)
_PLAIN = dict(append=_plain_append, decode=_plain_decode, gather=_plain_gather, prefill=_plain_prefill)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    B, Hkv, rep = c["B"], c["Hkv"], c.get("rep", 1)
    held = Hkv * 2 * (D // 2 + 2 * (D // GROUP))             # a cached token
    if c["op"] == "append":
        n = sum(_spread(c["nlo"], c["S"], B))
        row = 2 * D
        # q, k and v read, q and both caches written, their values read back
        return {"bytes": n * (row * Hkv * (2 * rep + 2 + c["kout"] + 2) + held),
                "flops": n * Hkv * (rep + 1) * (3 * c["rot"] + 4 * D * c["norm"]) + 8 * n * Hkv * D}
    if c["op"] == "decode":
        n = sum(_spread(c["lo"], c["cap"], B))
        return {"bytes": n * held + 4 * B * Hkv * rep * D, "flops": 4 * n * Hkv * rep * D}
    if c["op"] == "gather":
        n = sum(_spread(c["lo"], c["cap"], B))
        return {"bytes": n * (held + 4 * Hkv * D), "flops": 2 * n * Hkv * D}
    pairs = rows = keys = 0
    for n, m in zip(_spread(c["nlo"], c["S"], B), _spread(c["plo"], c["past"], B)[::-1]):
        pairs += n * m + n * (n + 1) // 2
        rows += n
        keys += (n + m) if n else 0
    return {"bytes": 4 * D * Hkv * (rows * rep + keys), "flops": 4 * pairs * Hkv * rep * D}


# ---------------------------------------------------------------- the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s)


def _slot(s, b, n):
    """Pages and places of the tokens n of sequence b."""
    page = s["case"]["page"]
    return s["tables"][b].long()[n // page], n % page


def _read64(s, name, b, n):
    """Tokens 0 .. n - 1 of sequence b, channel by channel from the layout's definition: [Hkv, n, 128]."""
    pg, t = _slot(s, b, torch.arange(n, device="cuda"))
    rows, sc = s["cache"][name][pg, :, t], s["cache"][name + "_scale"][pg, :, t].double()
    ch = torch.arange(D, device="cuda")
    g, j, i = ch // 32, ch % 32 // 8, ch % 8
    at = 16 * (j ^ 2 * (t[:, None] >> 1 & 1)) + 4 * g + i // 2
    byte = rows.gather(2, at[:, None].expand(-1, rows.shape[1], -1)).long()
    code = (byte >> 4 * (i % 2) & 15) - 8
    return (code.double() * sc[..., g]).transpose(0, 1)


def _exact_decode(s):
    c = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        if n:
            k, v = _read64(s, "k", b, n), _read64(s, "v", b, n)
            q = s["q"][b].double().view(c["Hkv"], c["rep"], D)
            p = torch.softmax(torch.einsum("hrd,hnd->hrn", q, k) / math.sqrt(D), -1)
            out[b] = torch.einsum("hrn,hnd->hrd", p, v).reshape(-1, D)
    return out


def _exact_gather(s):
    lens = s["lens"].tolist()
    return {name: torch.cat([_read64(s, name, b, n).transpose(0, 1) for b, n in enumerate(lens)])
            for name in ("k", "v")}


def _exact_prefill(s):
    rep = s["case"]["rep"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
    for b in range(len(cq) - 1):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        if n == 0:
            continue
        mask = torch.ones((n, m), dtype=torch.bool, device="cuda").tril(m - n)
        for h in range(s["q"].shape[1]):
            z = s["q"][cq[b]:cq[b + 1], h].double() @ s["k"][ck[b]:ck[b + 1], h // rep].double().T
            p = torch.softmax((z / math.sqrt(D)).masked_fill_(~mask, -math.inf), -1)
            out[cq[b]:cq[b + 1], h] = p @ s["v"][ck[b]:ck[b + 1], h // rep].double()
    return out


def _exact_append(s):
    """Rotations as complex products; what a group holds are whole multiples of its scale."""
    c = s["case"]
    half, lens, cu = c["rot"] // 2, s["lens"].tolist(), s["cu"].tolist()
    q_out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    k_out, held_k, held_v = (torch.zeros(s["kn"].shape, dtype=torch.float64, device="cuda") for _ in range(3))
    g = torch.arange(D, device="cuda") // GROUP
    for b in range(c["B"]):
        rows = slice(cu[b], cu[b + 1])
        at = torch.arange(lens[b], lens[b] + cu[b + 1] - cu[b], device="cuda")
        if not len(at):
            continue
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(at.double() + float(s["pos_offset"][b]), s["inv_freq"].double()))[:, None]

        def spin(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + 1e-6) * w.double()
            head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            if c["inter"]:
                z = torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) * turn
                head = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(head[..., :half], head[..., half:]) * turn
                head = torch.cat([z.real, z.imag], -1)
            return torch.cat([head, rest], -1)

        q_out[rows] = spin(s["q"][rows], s["qw"])
        k_out[rows] = spin(s["kn"][rows], s["kw"])
        for held, x in ((held_k, k_out[rows]), (held_v, s["vn"][rows].double())):
            sc = (x.view(len(at), -1, 4, GROUP).abs().max(-1).values / 7.5).half().double()[..., g]
            held[rows] = torch.clamp(torch.round(x / sc.clamp_min(1e-30)), -8, 7) * sc
    out = {"q": q_out, "k": held_k, "v": held_v}
    if s["k_out"] is not None:
        out["k_new"] = k_out
    return out


_EXACT = dict(append=_exact_append, decode=_exact_decode, gather=_exact_gather, prefill=_exact_prefill)
