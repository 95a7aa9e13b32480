"""Plain 64-bit forms of the operators around drafted tokens, on the CPU, with the
error bounds that their tests hold the kernels to (u = 2^-24 as in serving_ref)."""

import math

import torch

import serving_ref as ref


def parents_of(parent, i):
    """A row's parent number, -1 for none. parent None: the row before."""
    p = i - 1 if parent is None else parent[i]
    return p if 0 <= p < i else -1


def tree(parent, n):
    """(bits, depths) of a sequence's n nodes; bits as whole numbers."""
    bits, depth = [], []
    for i in range(n):
        p = parents_of(parent, i)
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return bits, depth


def words(bits, w):
    """[rows, w] int32 words of whole numbers."""
    out = torch.zeros(len(bits), w, dtype=torch.int64)
    for i, b in enumerate(bits):
        for k in range(w):
            out[i, k] = b >> 32 * k & 0xffffffff
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).to(torch.int32)


def rotated(x, heads, hd, pos, freqs, magnitude, inter, w, eps):
    """[T, heads, hd] normed and turned values in 64 bits, and the magnitude |a| + |b| that their errors go by."""
    T, rot = x.shape[0], 2 * len(freqs)
    v = x.double().reshape(T, heads, hd)
    if w is not None:
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.double()
    ang = (pos.double()[:, None] * freqs.double())[:, None]
    co, si = ang.cos() * magnitude, ang.sin() * magnitude
    out, mag = v.clone(), v.abs()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = v[..., first], v[..., second]
    out[..., first], out[..., second] = a * co - b * si, a * si + b * co
    mag[..., first] = mag[..., second] = (a.abs() + b.abs()) * magnitude
    return out, mag


def attend(q, ks, vs, new, see, n_q, n_kv, hd, scale):
    """(out, bound): q [sum(new), n_q * hd]; ks, vs [len, n_kv, hd] cached values; see: per sequence [n, n] truth values
    among the new tokens. Weights enter the product to 24 bits in fp32, to 16 in fp16 (2^-15 of themselves). In bf16 they
    may be fp16 numbers: rounded by half a step, eps / 2 = 2^-11 of themselves. In both 16-bit types a weight may be a subnormal
    fp16 number: with the largest of its 64 neighbours at least 2^-16 of the row's, which stands at 2^9, that is off by half of
    2^-24, which is 2^-34 of the row's largest and at most 2^-18 of the neighbours' largest, so of the row's."""
    G = n_q // n_kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros_like(out)
    p_err = {torch.float32: 0.0, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -11}[q.dtype]
    at = 0
    for m, k, v, mine in zip(new, ks, vs, see):
        n = k.shape[0]
        full = torch.ones(m, n, dtype=torch.bool)
        for j in range(m):
            if 0 <= n - m + j < n:
                full[:, n - m + j] = mine[:, j]
        for h in range(n_q):
            cols = slice(h * hd, (h + 1) * hd)
            o, b = ref.softmax_rows(q[at:at + m, cols].double(), k[:, h // G], v[:, h // G], full, scale, p_err)
            out[at:at + m, cols] = o
            bound[at:at + m, cols] = b + ref.rounding(o, q.dtype)
            if q.dtype != torch.float32 and n:
                z = torch.where(full, q[at:at + m, cols].double() @ k[:, h // G].T * scale, -math.inf)
                top = torch.softmax(z, 1).nan_to_num(0.0).amax(1, keepdim=True)
                bound[at:at + m, cols] += 2.0 ** -18 * top * v[:, h // G].abs().sum(0)
        at += m
    return out, bound


def verify(p, q, tokens, parent, start, u, u_next):
    """(path, count, token), lists, by the definition: one sequence, one node, one child at a time."""
    path, count, token = [-1] * p.shape[0], [], []
    V = p.shape[1]

    def pos(x):
        return torch.where(x > 0, x, torch.zeros_like(x))

    for s in range(len(start) - 1):
        f, n = start[s], start[s + 1] - start[s]
        if n == 0:
            count.append(0)
            token.append(-1)
            continue
        mine = None if parent is None else parent[f:f + n]
        kept, at = [0], 0
        while True:
            P = p[f + at].double()
            Q = q[f + at].double() if q is not None else None
            a, S, left, refused, nxt = 0.0, 1.0, pos(P), [], None
            for c in range(at + 1, n):
                if parents_of(mine, c) != at:
                    continue
                t, uc = int(tokens[f + c]), float(u[f + c])
                pt = float(P[t]) if 0 <= t < V else 0.0
                if Q is not None:
                    qt = float(Q[t]) if 0 <= t < V else 0.0
                    if uc * S * qt < pt - a * qt:
                        nxt = c
                        break
                    a += S
                    left = pos(P - a * Q)
                    S = float(left.sum())
                    if not S > 0:
                        break
                else:
                    if t in refused:
                        pt = 0.0
                    if uc * S < pt:
                        nxt = c
                        break
                    S -= pt
                    refused.append(t)
                    if 0 <= t < V:
                        left[t] = 0.0
            if nxt is None:
                break
            at = nxt
            kept.append(at)
        if not float(left.sum()) > 0:
            left = pos(P)
        cum, t = 0.0, -1
        want = max(float(u_next[s]), 0.0) * float(left.sum())
        sums = torch.cumsum(left, 0)
        over = (sums > want).nonzero()
        some = (left > 0).nonzero()
        t = int(over[0]) if len(over) else int(some[-1]) if len(some) else -1
        path[f:f + len(kept)] = kept
        count.append(len(kept))
        token.append(t)
    return path, count, token


def freqs(rot, base=10000.0):
    return torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
