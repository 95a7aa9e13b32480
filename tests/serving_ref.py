"""Plain 64-bit forms of the operators that serve several prompts, on the CPU,
with the error bounds that their tests hold the kernels to.

u = 2^-24 is half a step of fp32. A sum of n products in fp32, in any order, is off by at
most n u times the sum of their magnitudes. A result rounded to its type is off
by half a step, `half(dtype)` of its magnitude (at least half the smallest step)."""

import math

import torch

U = 2.0 ** -24
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(ref, dtype):
    """What rounding these values to the type costs at most."""
    f = torch.finfo(dtype)
    return ref.abs() * half(dtype) + f.smallest_normal * half(dtype)


def rope(x, heads, hd, pos, sections, base, w, eps):
    """(out, bound): norms per head and rotation, x [T, heads * hd].

    Bound: the norm's sum of hd squares in at most 8 + 6 + 2 steps per lane and 6 over lanes
    is off by 22 u, its root by half that and 4 u for mean, eps, root and reciprocal; two more
    products make 17 u on y. Sine and cosine: the fraction of a turn rounded to fp32 moves the
    angle by at most pi u, the functions add 2 units in the last place (4 u), together 8 u. Product
    and sum add 2 u: 27 u of |y_i| + |y_(i + half)|."""
    T, h = x.shape[0], hd // 2
    v = x.double().reshape(T, heads, hd)
    if w is not None:
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.double()
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    freq = torch.tensor([float(base) ** (-2.0 * i / hd) for i in range(h)], dtype=torch.float64)
    ang = torch.stack([pos[axis[i]].double() * freq[i] for i in range(h)], 1)[:, None]
    a, b = v[..., :h], v[..., h:]
    out = torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).reshape(T, heads * hd)
    mag = (a.abs() + b.abs()).repeat(1, 1, 2).reshape(T, heads * hd)
    return out, 27 * U * mag + rounding(out, x.dtype)


def softmax_rows(q, k, v, see, scale, p_err, exact_products=False):
    """(out, bound) of one head: q [m, hd], k, v [n, hd] in 64 bits, see [m, n].

    Bound: a score is off by (hd + 3) u times scale * sum |q||k| (the scale, log2 e and their
    products among the 3), which moves a weight relative to another by twice that; exp2, the
    running rescales (one per tile of keys) and the sum over n keys add (n + 24) u, and the
    weights' own rounding p_err, all relative to sum_j w_j |v_j|."""
    m, n = q.shape[0], k.shape[0]
    out = torch.zeros(m, v.shape[1], dtype=torch.float64)
    bound = torch.zeros_like(out)
    for i in range(m):
        j = see[i].nonzero().flatten()
        if j.numel() == 0:
            continue
        s = k[j] @ q[i] * scale
        S = float((k[j].abs() @ q[i].abs()).max()) * abs(scale)
        if math.isfinite(float(s.max())):
            w = torch.exp(s - s.max())
        else:
            w = torch.exp(s - s.max())  # NaN, as the definition gives
        w = w / w.sum()
        out[i] = w @ v[j]
        bound[i] = (w @ v[j].abs()) * (2 * (q.shape[1] + 3) * U * S + (n + 24) * U + p_err)
    return out, bound


def packed(q, k, v, qs, ks, n_q, n_kv, hd, scale, causal, base=None):
    """(out, bound) of packed attention; rows outside the sequences keep `base`'s values."""
    G = n_q // n_kv
    out = torch.zeros(q.shape, dtype=torch.float64) if base is None else base.double().clone()
    bound = torch.zeros_like(out)
    p_err = 0.0 if q.dtype == torch.float32 else half(q.dtype)
    for s in range(len(qs) - 1):
        m, n = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
        i, j = torch.arange(m)[:, None], torch.arange(n)[None]
        see = (j <= i + n - m) if causal else torch.ones(m, n, dtype=torch.bool)
        for h in range(n_q):
            kh = h // G
            o, b = softmax_rows(q[qs[s]:qs[s + 1], h * hd:(h + 1) * hd].double(), k[ks[s]:ks[s + 1], kh * hd:(kh + 1) * hd].double(),
                                v[ks[s]:ks[s + 1], kh * hd:(kh + 1) * hd].double(), see, scale, p_err)
            out[qs[s]:qs[s + 1], h * hd:(h + 1) * hd] = o
            bound[qs[s]:qs[s + 1], h * hd:(h + 1) * hd] = b + rounding(o, q.dtype)
    return out, bound


def quantize(x):
    """[..., hd] -> (codes [..., hd] 0..15, bytes [..., hd / 32]) by the format's definition, value by value."""
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    e = torch.full_like(amax, -100)
    for t in range(-100, 127):  # the smallest exponent with amax <= 7 * 2^e
        e = torch.where(amax > 7 * 2.0 ** t, torch.full_like(e, t + 1), e)
    y = b.abs() / torch.exp2(e)[..., None]
    d = (y[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.double().argmax(-1), near.double().argmax(-1))
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    byte = torch.where(bad, torch.full_like(e, 255), e + 127).long()
    return code.flatten(-2), byte


def values(code, byte):
    sign = torch.where(code >= 8, -1.0, 1.0).double()
    s = torch.exp2(byte.double() - 127)
    s = torch.where(byte == 255, torch.full_like(s, math.nan), s)
    return sign * GRID[code % 8] * s.repeat_interleave(32, -1)


class HostCache:
    """A cache image in host memory, written and read one token at a time through kv4_offset."""

    def __init__(self, vla, n_pages, n_kv, hd, page, fill=0):
        import numpy as np
        self.vla, self.n_pages, self.n_kv, self.hd, self.page = vla, n_pages, n_kv, hd, page
        self.nb = vla.kv4_page_bytes(n_kv, hd, page)
        self.mem = np.full(n_pages * self.nb, fill, np.uint8)

    def at(self, row, tok, part, head, block):
        return self.vla.kv4_offset(row, self.n_kv, self.hd, self.page, self.n_pages, tok, part, head, block)

    def write(self, row, tok, part, x):
        """x [n_kv, hd]"""
        code, byte = quantize(x)
        for h in range(self.n_kv):
            for b in range(self.hd // 32):
                at = self.at(row, tok, part, h, b)
                if at < 0:
                    continue
                c = code[h, 32 * b:32 * b + 32].numpy()
                self.mem[at:at + 16] = c[0::2] | c[1::2] << 4
                self.mem[self.at(row, tok, part + 2, h, b)] = byte[h, b]

    def read(self, row, n, part):
        """[n, n_kv, hd] values; NaN where the row names no page."""
        out = torch.full((n, self.n_kv, self.hd), math.nan, dtype=torch.float64)
        for t in range(n):
            for h in range(self.n_kv):
                for b in range(self.hd // 32):
                    at = self.at(row, t, part, h, b)
                    if at < 0:
                        continue
                    by = torch.from_numpy(self.mem[at:at + 16].astype("int64"))
                    code = torch.stack([by & 15, by >> 4], 1).flatten()
                    byte = torch.tensor([int(self.mem[self.at(row, t, part + 2, h, b)])])
                    out[t, h, 32 * b:32 * b + 32] = values(code, byte)
        return out


def decode(q, ks, vs, new, n_q, n_kv, hd, scale):
    """(out, bound): q [sum(new), n_q * hd]; ks, vs: [len, n_kv, hd] cached values of each sequence."""
    G = n_q // n_kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    p_err = 0.0 if q.dtype == torch.float32 else 2.0 ** -15  # two parts of 8 bits, cut off
    at = 0
    for m, k, v in zip(new, ks, vs):
        n = k.shape[0]
        see = torch.arange(n)[None] <= torch.arange(m)[:, None] + n - m
        for h in range(n_q):
            cols = slice(h * hd, (h + 1) * hd)
            o, b = softmax_rows(q[at:at + m, cols].double(), k[:, h // G], v[:, h // G], see, scale, p_err)
            out[at:at + m, cols] = o
            bound[at:at + m, cols] = b + rounding(o, q.dtype)
        at += m
    return out, bound


def within(got, ref, bound, what=""):
    """Every element within its bound; NaN and infinities where the reference has them."""
    got = got.double().cpu()
    same = (got == ref) | (got.isnan() & ref.isnan())
    bad = ~(same | ((got - ref).abs() <= bound))
    if bool(bad.any()):
        i = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {i}: got {got[tuple(i)].item()}, "
                             f"want {ref[tuple(i)].item()} +- {bound[tuple(i)].item()}")
