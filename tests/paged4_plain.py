"""Plain float64 forms of the paged 4-bit cache's operators, for the tests: the layout read byte by
byte, codes from exact quotients, attention by the formula."""
import math

import torch

D = 128


def slots(tables, page, b, n):
    """Pages and places of tokens 0 .. n - 1 of sequence b."""
    i = torch.arange(n, device=tables.device)
    return tables[b].long()[i // page], i % page


def byte_of(t, device):
    """Byte of channel ch in the row of a token at place t (t [n] -> [n, 128]), and its shift."""
    ch = torch.arange(D, device=device)
    g, j, i = ch // 32, ch % 32 // 8, ch % 8
    return 16 * (j ^ 2 * (t[:, None] >> 1 & 1)) + 4 * g + i // 2, 4 * (i % 2)


def read_codes(cache, name, pg, t):
    """Codes -8 .. 7 and scales (float64) of the tokens (pg, t): [n, Hkv, 128], [n, Hkv, 4]."""
    rows = cache[name][pg, :, t].long()
    at, sh = byte_of(t, rows.device)
    codes = (rows.gather(2, at[:, None].expand(-1, rows.shape[1], -1)) >> sh & 15) - 8
    return codes, cache[name + "_scale"][pg, :, t].double()


def values(cache, name, tables, b, n):
    """Tokens 0 .. n - 1 of sequence b in float64: [n, Hkv, 128]."""
    pg, t = slots(tables, cache[name].shape[2], b, n)
    codes, sc = read_codes(cache, name, pg, t)
    return codes.double() * sc.repeat_interleave(32, -1)


def coded(x):
    """Codes and float16 scales of x [.., 128] float64."""
    g = x.double().unflatten(-1, (4, 32))
    sc = (g.abs().amax(-1) / 7.5).clamp(max=65504.0).half()
    safe = torch.where(sc > 0, sc.double(), torch.ones((), dtype=torch.float64, device=x.device))
    c = torch.round(g / safe[..., None]).clamp(-8, 7)
    return torch.where(sc[..., None] > 0, c, torch.zeros_like(c)).flatten(-2).long(), sc


def turned(x, w, pos, inv_freq, interleaved, factor, eps):
    """Norm and rotation of x [T, H, 128] at positions pos [T], float64."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / D + eps) * w.double()
    if inv_freq is None:
        return y
    rot = 2 * inv_freq.numel()
    ang = pos.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos() * factor, ang.sin() * factor
    out = y.clone()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return out


def attend(q, k, v, seen, scale=None):
    """softmax(q k^T scale) v over the seen keys, zeros where there are none; with the weights' sum of
    |v|.  q [H, n, D], k / v [H, m, D], seen [n, m]."""
    z = (q.double() @ k.double().transpose(1, 2)) * (scale if scale is not None else 1 / math.sqrt(D))
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True).clamp(min=-1e300) if z.shape[-1] else z.new_zeros(z.shape[:2] + (1,))
    p = (z - top).exp().masked_fill(~seen, 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    return p @ v.double(), p @ v.double().abs()


def random_cache(kernels, n_pages, Hkv, page, gen):
    """Pages of random codes and scales, as much as 30 % of a group's range apart."""
    c = kernels.paged4_alloc(n_pages, Hkv, page_size=page)
    for n in ("k", "v"):
        c[n].random_(0, 256, generator=gen)
        c[n + "_scale"].uniform_(0.1, 0.4, generator=gen)
    return c


def random_tables(B, per, n_pages, gen):
    return torch.randperm(n_pages, generator=gen, device="cuda")[:B * per].view(B, per).to(torch.int32)
