"""The operators of a decoder whose next tokens are drafted, as cases that can be timed and checked.

A step drafts a few tokens for every sequence, as a tree behind its last token,
lets the target read all of them at once, accepts a path of the tree and keeps that.

Kinds:
  tree     vla_draft_tree_dev: from the parents of the drafted tokens their
           positions and the words of bits that say which of them each one sees
  append   vla_rope_kv4_append_dev: norms and rotation of queries and keys (half or
           interleaved pairs, all or part of a head, any frequencies), the keys and the
           values into the paged 4-bit cache; its rows are read back (vla_kv4_gather_dev)
  attend   vla_kv4_tree_attention_dev: attention of the drafted tokens over the cache,
           of the newest tokens those that their bits name
  verify   vla_verify_drafts_dev: the accepted path and the token behind it, from the
           target's probabilities, the draft's and given random numbers
  keep     vla_kv4_keep_dev: the path's tokens to the front of the drafted ones in the
           cache, and the new lengths; the rows are read back

`run` computes a pass with elementary torch operations, or with `own` set
through the framework's calls; `exact` is the definition in 64 bits.
"""

from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32  # values of a head that share a scale in the 4-bit cache
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E_MIN = -100
COST = 2 * 131072 * 64 * 32 * 128  # of the largest attention: keys, queries, heads, columns


def _pkg():
    if "vla_simd_amd" not in sys.modules:
        d = os.path.join(ROOT, "vla.simd_amd")
        spec = importlib.util.spec_from_file_location("vla_simd_amd", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["vla_simd_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["vla_simd_amd"]


def listed():
    return [
        # the drafted tokens of one robot's decoder: the smallest call
        dict(name="tree_robot", kind="tree", n=1, nodes=8, spread=0, wide=3, past=200),
        # 256 conversations with a tree of 64 drafted tokens each
        dict(name="tree_batch", kind="tree", n=256, nodes=64, spread=0, wide=16, past=3000),
        # one decoded token of SmolVLA's language tower
        dict(name="append_token", kind="append", n=1, nodes=1, spread=0, wide=0, past=200, n_q=15, n_kv=5, hd=64, rot=64,
             inter=False, scaled=False, norm=False, rows_out=False, page=64, dtype="f32"),
        # the drafted tokens of 48 long conversations, positions scaled beyond the trained length
        dict(name="append_trees", kind="append", n=48, nodes=32, spread=0, wide=8, past=30000, n_q=32, n_kv=8, hd=128, rot=128,
             inter=False, scaled=True, norm=True, rows_out=False, page=64, dtype="bf16"),
        # sixteen prompts of mixed lengths, half of every head rotated in neighbouring pairs, the keys also as rows
        dict(name="append_prompts", kind="append", n=16, nodes=4096, spread=2, wide=0, past=0, n_q=32, n_kv=8, hd=128, rot=64,
             inter=True, scaled=False, norm=False, rows_out=True, page=64, dtype="f16"),
        # a small tree of one robot over its prefix and chunk
        dict(name="attend_robot", kind="attend", n=1, longest=227, spread=0, nodes=8, wide=3, n_q=15, n_kv=5, hd=64, page=64, dtype="f32"),
        # trees of 32 for 48 conversations of mixed lengths
        dict(name="attend_batch", kind="attend", n=48, longest=8192, spread=4, nodes=32, wide=8, n_q=32, n_kv=8, hd=128, page=64, dtype="bf16"),
        # trees of 64 for two very long documents
        dict(name="attend_long", kind="attend", n=2, longest=131072, spread=0, nodes=64, wide=16, n_q=32, n_kv=8, hd=128, page=256, dtype="f16"),
        # a chain of four drafted tokens of one sequence
        dict(name="verify_chain", kind="verify", n=1, nodes=5, spread=0, wide=0, vocab=49280, sampled=True, dtype="f32"),
        # trees of 32 for 48 sequences
        dict(name="verify_trees", kind="verify", n=48, nodes=32, spread=0, wide=8, vocab=49280, sampled=True, dtype="f32"),
        # the accepted ones of one robot's eight
        dict(name="keep_robot", kind="keep", n=1, nodes=8, spread=0, past=219, n_kv=5, hd=64, page=64, dtype="f32"),
        # one layer of 64 conversations with trees of 64
        dict(name="keep_batch", kind="keep", n=64, nodes=64, spread=0, past=2000, n_kv=8, hd=128, page=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "append", "append", "attend", "attend", "verify", "verify", "keep"])
    n_q, n_kv = rng.choice([(15, 5), (32, 8), (16, 2), (12, 12), (8, 1), (16, 8)])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    hd, page = rng.choice([32, 64, 64, 96, 128, 128, 192, 256]), rng.choice([32, 64, 64, 96, 128, 256])
    n, spread, wide = _log(rng, 1, 64), rng.randint(0, 6), rng.choice([0, 1, 2, 5, 8, 30])
    if kind == "tree":
        return dict(kind=kind, n=_log(rng, 1, 256), nodes=_log(rng, 1, 64), spread=spread, wide=wide, past=rng.randint(0, 5000))
    if kind == "append":
        most = 16 * 4096 * 48 * 128 * 2 // (n * (n_q + 2 * n_kv) * hd * SIZE[dtype])
        return dict(kind=kind, n=n, nodes=_log(rng, 1, max(2, min(8192, most))), spread=spread, wide=0 if wide > 5 else wide,
                    past=rng.choice([0, rng.randint(1, 30000 // n)]), n_q=n_q, n_kv=n_kv, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2, 8 * rng.randint(1, hd // 8)]), inter=rng.random() < 0.5, scaled=rng.random() < 0.4,
                    norm=rng.random() < 0.5, rows_out=rng.random() < 0.4, page=page, dtype=dtype)
    if kind == "attend":
        most = COST // ((6 if dtype == "f32" else 1) * n * n_q * hd)
        nodes = _log(rng, 1, 128 if rng.random() < 0.2 else 48)
        return dict(kind=kind, n=n, longest=_log(rng, 1, max(2, min(131072, most // nodes, 2 * 131072 * 8 * 128 // (n * n_kv * hd)))),
                    spread=spread, nodes=nodes, wide=wide, n_q=n_q, n_kv=n_kv, hd=hd, page=page, dtype=dtype)
    if kind == "verify":
        vocab = rng.choice([49280, 32128, _log(rng, 2, 131072)])
        most = 48 * 32 * 49280 // (vocab * n)
        return dict(kind=kind, n=n, nodes=_log(rng, 1, max(2, min(64, most))), spread=spread, wide=wide, vocab=vocab,
                    sampled=rng.random() < 0.6, dtype=dtype)
    return dict(kind=kind, n=n, nodes=_log(rng, 1, 64), spread=spread, past=rng.randint(0, 2000), n_kv=n_kv, hd=hd, page=page, dtype=dtype)


# ---------------------------------------------------------------- sizes --

def _mixed(c, top):
    """All the largest with spread 0, else mixed, the first the largest, none and one among them."""
    n = c["n"]
    if not c["spread"]:
        return [top] * n
    r = random.Random(c["spread"] * 1009 + n * 31 + top)
    out = [top] + [_log(r, max(1, top // 16), top) for _ in range(n - 1)]
    if n >= 4:
        out[n // 2], out[n - 1] = 0, 1
    return out


def _new(c):
    """New tokens of each sequence."""
    if c["kind"] == "attend":
        return [min(c["nodes"], n) for n in _mixed(c, c["longest"])]
    return _mixed(c, c["nodes"])


def _lens(c):
    """Tokens of each sequence, the new ones included."""
    return _mixed(c, c["longest"]) if c["kind"] == "attend" else [c.get("past", 0) + n for n in _new(c)]


def _parents(c):
    """The parent of each new token in its sequence: the one before without `wide`, else one of the last `wide`; -1 for the first."""
    out = []
    for s, n in enumerate(_new(c)):
        r = random.Random(s * 7 + c["wide"])
        out.append([-1] + [i - 1 if not c["wide"] else r.randrange(max(0, i - c["wide"]), i) for i in range(1, n)] if n else [])
    return out


def _seen(parents):
    """For each new token of a sequence those that it sees, as the bits of a whole number, and its depth."""
    bits, depth = [], []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return bits, depth


def _words(c):
    return (max(_new(c)) + 31) // 32


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def work(case):
    c, new = case, _new(case)
    rows = sum(new)
    if c["kind"] == "tree":  # parents, lengths and offsets in, positions and words out
        return {"bytes": 4 * rows * (2 + _words(c)) + 8 * c["n"], "flops": 0}
    sz = SIZE[c["dtype"]]
    if c["kind"] == "verify":  # the rows that the last token is drawn from, and two probabilities of each drafted one
        return {"bytes": c["n"] * c["vocab"] * sz * (2 if c["sampled"] else 1) + rows * (2 * sz + 16), "flops": 4 * c["n"] * c["vocab"]}
    kv = c["n_kv"] * c["hd"]
    cached = 2 * rows * kv * 17 // 32
    if c["kind"] == "append":  # rows in, rotated queries (and keys) and 4-bit values out; the 4-bit values in, rows out
        return {"bytes": rows * sz * (2 * c["n_q"] * c["hd"] + (5 if c["rows_out"] else 4) * kv) + 2 * cached + 4 * rows,
                "flops": 9 * rows * (c["n_q"] + c["n_kv"]) * c["hd"]}
    if c["kind"] == "keep":  # half of them, say, in and out; all in once more, rows out
        return {"bytes": 2 * cached + 2 * rows * kv * sz + 4 * rows, "flops": 2 * rows * kv}
    pairs = sum(m * (n - m) + sum(d + 1 for d in _seen(p)[1]) for m, n, p in zip(new, _lens(c), _parents(c)))
    return {"bytes": sum(_lens(c)) * kv * 17 // 16 + 2 * sz * c["hd"] * c["n_q"] * rows + 4 * rows * _words(c) + 4 * c["n"],
            "flops": 4 * pairs * c["hd"] * c["n_q"]}


# --------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed) * 7919 + 43)


def _n(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _flat(lists):
    return [x for v in lists for x in v]


def _bit_words(c):
    """[rows, words] int32 of the bits that each new token sees."""
    w = _words(c)
    if sum(_new(c)) == 0:
        return torch.zeros(0, max(1, w), dtype=torch.int32, device=DEV)
    raw = b"".join(b.to_bytes(4 * w, "little") for p in _parents(c) for b in _seen(p)[0])
    return torch.from_numpy(np.frombuffer(raw, dtype=np.int32).reshape(-1, w).copy()).to(DEV)


def _quantize(x):
    """[..., hd] values -> (codes [..., hd/2] with the even value in the low half, scale bytes [..., hd/32])."""
    b = x.unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1); amax <= 7 * 2^s where s is e - 3, or e - 2 when m > 7/8
    s = torch.where(m > 0.875, e - 2, e - 3).clamp(min=E_MIN)
    s = torch.where(amax == 0, torch.full_like(s, E_MIN), s)
    y = torch.ldexp(b.abs(), -s)
    # steps of 0.5 below 2, of 1 to 4, of 2 to 6, which takes all up to 7; halves go to the even step
    r = torch.where(y < 2, torch.round(y * 2), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4)).clamp(max=7)
    code = r.to(torch.uint8) | ((b < 0) | ((b == 0) & torch.signbit(b))).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, (s.squeeze(-1) + 127).to(torch.uint8)


def _page_parts(pages, n_kv, page, hd):
    """Views (K codes, V codes, K scales, V scales) of [n, page_bytes] pages."""
    nc, ns = n_kv * page * hd // 2, n_kv * (hd // BLOCK) * page
    return (pages[:, :nc].unflatten(1, (n_kv, page, hd // 2)), pages[:, nc:2 * nc].unflatten(1, (n_kv, page, hd // 2)),
            pages[:, 2 * nc:2 * nc + ns].unflatten(1, (n_kv, hd // BLOCK, page)),
            pages[:, 2 * nc + ns:2 * nc + 2 * ns].unflatten(1, (n_kv, hd // BLOCK, page)))


def _page_bytes(n_kv, page, hd):
    return n_kv * page * (hd + 2 * (hd // BLOCK))


def _table(c, lens, g):
    """A page table of shuffled pages for sequences of these lengths, and the number of pages."""
    need = [(n + c["page"] - 1) // c["page"] for n in lens]
    total = max(1, sum(need))
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, total


def _filled(c, pages, g):
    """A cache whose pages hold normal values."""
    cache = torch.zeros(pages, _page_bytes(c["n_kv"], c["page"], c["hd"]), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 25) // (c["n_kv"] * c["page"] * c["hd"]))
    for p in range(0, pages, step):
        part = cache[p:p + step]
        kc, vc, ks, vs = _page_parts(part, c["n_kv"], c["page"], c["hd"])
        for codes, scales in ((kc, ks), (vc, vs)):
            a, b = _quantize(_n(g, part.shape[0], c["n_kv"], c["page"], c["hd"]))
            codes.copy_(a)
            scales.copy_(b.transpose(2, 3))
    return cache


def _freqs(rot, scaled):
    """Angles a position turns each pair by; scaled: pairs of long waves eight times as slow, of short ones as they
    were, a ramp between them, for positions up to eight times the 4096 trained ones. And the factor on the rotated values."""
    f = [10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)]
    if not scaled:
        return f, 1.0
    turns = [4096 * x / (2 * math.pi) for x in f]  # over the trained length
    keep = [min(1.0, max(0.0, (t - 1) / (32 - 1))) for t in turns]
    return [x * k + x / 8 * (1 - k) for x, k in zip(f, keep)], 0.1 * math.log(8) + 1


def _drawn(g, rows, order):
    """A token of each row's probabilities: drawn from them, or the order[i]-th most probable one."""
    out = []
    step = max(1, (1 << 26) // rows.shape[1])
    for i in range(0, rows.shape[0], step):
        x = rows[i:i + step].double()
        if order is None:
            c = x.cumsum(-1)
            out.append(torch.searchsorted(c, torch.rand(c.shape[0], 1, generator=g, device=DEV, dtype=torch.float64) * c[:, -1:]))
        else:
            out.append(x.topk(min(x.shape[1], 32), -1).indices.gather(1, order[i:i + step, None] % min(x.shape[1], 32)))
    return torch.cat(out)[:, 0].clamp(max=rows.shape[1] - 1)


def _prepare_verify(c, g, dt):
    new, parents = _new(c), _parents(c)
    rows, V = sum(new), c["vocab"]
    first = torch.tensor(_flat([s] * n for s, n in zip(_starts(new), new)), dtype=torch.int64, device=DEV)
    s = {"start": _i32(_starts(new)), "parent": _i32(_flat(parents))}
    above = first + s["parent"].long().clamp(min=0)
    nth = []  # a token's number among those of the same parent
    for p in parents:
        seen = {}
        for x in p:
            nth.append(seen.get(x, 0))
            seen[x] = nth[-1] + 1
    s["p"] = torch.empty(rows, V, dtype=dt, device=DEV)
    s["q"] = torch.empty(rows, V, dtype=dt, device=DEV)
    step = max(1, (1 << 26) // V)
    for i in range(0, rows, step):  # a peaked target and a draft that is not far from it
        z = _n(g, min(step, rows - i), V, std=3.0)
        s["p"][i:i + step] = torch.softmax(z, -1).to(dt)
        s["q"][i:i + step] = torch.softmax(z + _n(g, *z.shape, std=0.7), -1).to(dt)
    tok = torch.empty(0, dtype=torch.int64, device=DEV)
    if rows:
        tok = torch.cat([_drawn(g, s["q"][above[i:i + step]], None if c["sampled"] else torch.tensor(nth[i:i + step], device=DEV))
                         for i in range(0, rows, step)])
    s["tokens"] = tok.to(torch.int32)
    if not c["sampled"]:
        s["q"] = None
    s["u"] = torch.rand(rows, generator=g, device=DEV)
    s["u_next"] = torch.rand(c["n"], generator=g, device=DEV)
    s["path"] = torch.empty(rows, dtype=torch.int32, device=DEV)
    s["count"] = torch.empty(c["n"], dtype=torch.int32, device=DEV)
    s["token"] = torch.empty(c["n"], dtype=torch.int32, device=DEV)
    s["rows"] = (first, torch.tensor(_flat(list(range(n)) for n in new), dtype=torch.int64, device=DEV))
    return s


def _paths(c, seed):
    """Accepted paths: the first few drafted tokens, then ones from behind the room that they move to."""
    r, out, count = random.Random(int(seed) * 31 + 5), [], []
    for n in _new(c):
        k = min(n, r.randint(1, 6))
        j = r.randint(1, k) if k else 0
        path = list(range(j)) + sorted(r.sample(range(k, n), min(k - j, max(0, n - k)))) if k else []
        count.append(len(path))
        out += path + [-1] * (n - len(path))
    return out, count


def prepare(case, seed):
    c, g = case, _gen(seed)
    new, lens = _new(c), _lens(c)
    rows = sum(new)
    s = {"case": c, "vla": _pkg() if own else None, "new_host": new, "lens_host": lens}
    if c["kind"] == "tree":
        shift = random.Random(int(seed)).randint(0, 99)  # another moment of the same conversations
        s["parent"], s["lens"], s["start"] = _i32(_flat(_parents(c))), _i32([n + shift for n in lens]), _i32(_starts(new))
        s["pos"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        s["see"] = torch.empty(rows, max(1, _words(c)), dtype=torch.int32, device=DEV)
        s["row"] = (torch.tensor(_flat([i] * n for i, n in enumerate(new)), device=DEV, dtype=torch.int64),
                    torch.tensor(_flat(list(range(n)) for n in new), device=DEV, dtype=torch.int64))
        return s
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "verify":
        return s | _prepare_verify(c, g, dt)
    kv, hd = c["n_kv"] * c["hd"], c["hd"]
    s["table"], pages = _table(c, lens, g)
    s["lens"], s["start"] = _i32(lens), _i32(_starts(new))
    first = [n - m for n, m in zip(lens, new)]
    s["first"] = _i32(first)
    if c["kind"] != "attend":
        s["slot"] = (torch.tensor(_flat([i] * m for i, m in enumerate(new)), device=DEV, dtype=torch.int64),
                     torch.tensor(_flat(list(range(f, f + m)) for f, m in zip(first, new)), device=DEV, dtype=torch.int64))
        s["k_back"], s["v_back"] = (torch.empty(rows, kv, dtype=dt, device=DEV) for _ in range(2))
    if c["kind"] == "append":
        buf = _n(g, rows, c["n_q"] * hd + 2 * kv, dtype=dt)  # one product's queries, keys and values
        s["q"], s["k"], s["v"] = buf[:, :c["n_q"] * hd], buf[:, c["n_q"] * hd:c["n_q"] * hd + kv], buf[:, c["n_q"] * hd + kv:]
        s["wq"] = 1 + _n(g, hd, std=0.1) if c["norm"] else None
        s["wk"] = 1 + _n(g, hd, std=0.1) if c["norm"] else None
        f, s["magnitude"] = _freqs(c["rot"], c["scaled"])
        s["freqs"] = torch.tensor(f, dtype=torch.float64, device=DEV)
        s["pos"] = _i32(_flat([f0 + d for d in _seen(p)[1]] for f0, p in zip(first, _parents(c)))) if c["wide"] \
            else _i32(_flat(list(range(f0, f0 + m)) for f0, m in zip(first, new)))
        s["eps"] = 1e-6
        s["cache"] = torch.zeros(pages, _page_bytes(c["n_kv"], c["page"], hd), dtype=torch.uint8, device=DEV)
        s["q_out"] = torch.empty(rows, c["n_q"] * hd, dtype=dt, device=DEV)
        s["k_out"] = torch.empty(rows, kv, dtype=dt, device=DEV) if c["rows_out"] else None
        return s
    s["cache"] = _filled(c, pages, g)
    if c["kind"] == "keep":
        path, count = _paths(c, seed)
        s["path"], s["count"], s["new_lens"] = _i32(path), _i32(count), torch.empty(c["n"], dtype=torch.int32, device=DEV)
        return s
    s["see"] = _bit_words(c)
    s["q"] = _n(g, rows, c["n_q"] * hd, dtype=dt)
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(hd)
    s["row"] = (torch.tensor(_flat([i] * m for i, m in enumerate(new)), device=DEV, dtype=torch.int64),
                torch.tensor(_flat(list(range(m)) for m in new), device=DEV, dtype=torch.int64))
    s["work"] = None
    if own:
        n = s["vla"].kv4_tree_attention_work_bytes(rows, c["n"], max(new), c["longest"], c["n_q"], c["n_kv"], hd)
        s["work"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------- the plain forms --

def _plain_tree(s):
    c = s["case"]
    seq, i = s["row"]
    n, m = c["n"], max(s["new_host"])
    # above[s, i, j]: j is i or one above it. The paths of twice the length come from the product with itself
    above = torch.zeros(n, m, m, device=DEV)
    above[seq, i, i] = 1
    has = s["parent"] >= 0
    above[seq, i, s["parent"].long().clamp(min=0)] += has.float()
    above.clamp_(max=1)
    for _ in range(max(1, m - 1).bit_length()):
        above = torch.matmul(above, above).clamp_(max=1)
    mine = above[seq, i].long()
    s["pos"].copy_(s["lens"][seq] - (s["start"][1:] - s["start"][:-1])[seq] + mine.sum(-1) - 1)
    mine = torch.nn.functional.pad(mine, (0, 32 * s["see"].shape[1] - m)).unflatten(1, (-1, 32))
    s["see"].copy_((mine << torch.arange(32, device=DEV)).sum(-1).to(torch.int32))
    return [s["pos"], s["see"]]


def _values(codes, scales, dtype=torch.float32):
    """Values [..., page, hd] of codes [..., page, hd/2] and scale bytes [..., hd/32, page]."""
    lut = torch.tensor(GRID + tuple(-x for x in GRID), device=DEV, dtype=dtype)
    c = codes.int()
    x = torch.stack([lut[c & 15], lut[c >> 4]], -1).flatten(-2)
    e = torch.exp2(scales.to(dtype) - 127)
    e = torch.where(scales == 255, torch.full_like(e, math.nan), e).transpose(-1, -2)
    return (x.unflatten(-1, (-1, BLOCK)) * e[..., None]).flatten(-2)


def _plain_rotate(x, w, s, heads, dtype):
    """Norm and rotation in this type, [rows, heads, hd]."""
    c, rot = s["case"], s["case"]["rot"]
    v = x.to(dtype).unflatten(1, (heads, c["hd"]))
    if w is not None:
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + s["eps"]) * w.to(dtype)
    angle = s["pos"].double()[:, None] * s["freqs"]
    co, si = (angle.cos() * s["magnitude"]).to(dtype)[:, None], (angle.sin() * s["magnitude"]).to(dtype)[:, None]
    out = v.clone()
    a, b = (v[..., 0:rot:2], v[..., 1:rot:2]) if c["inter"] else (v[..., :rot // 2], v[..., rot // 2:rot])
    x0, x1 = a * co - b * si, a * si + b * co
    if c["inter"]:
        out[..., 0:rot:2], out[..., 1:rot:2] = x0, x1
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = x0, x1
    return out


def _plain_read(s):
    """The new tokens' cached values as rows."""
    c = s["case"]
    seq, tok = s["slot"]
    page, slot = s["table"][seq, tok // c["page"]].long(), tok % c["page"]
    kc, vc, ks, vs = _page_parts(s["cache"], c["n_kv"], c["page"], c["hd"])
    for codes, scales, o in ((kc, ks, s["k_back"]), (vc, vs, s["v_back"])):
        back = _values(codes[page, :, slot][:, :, None], scales[page, :, :, slot][..., None])
        o.copy_(back.squeeze(2).flatten(1))
    return [s["k_back"], s["v_back"]]


def _plain_append(s):
    c = s["case"]
    s["q_out"].copy_(_plain_rotate(s["q"], s["wq"], s, c["n_q"], torch.float32).flatten(1))
    k = _plain_rotate(s["k"], s["wk"], s, c["n_kv"], torch.float64)  # its codes lie next to borders
    if s["k_out"] is not None:
        s["k_out"].copy_(k.flatten(1))
    seq, tok = s["slot"]
    page, slot = s["table"][seq, tok // c["page"]].long(), tok % c["page"]
    kc, vc, ks, vs = _page_parts(s["cache"], c["n_kv"], c["page"], c["hd"])
    for x, codes, scales in ((k, kc, ks), (s["v"].float().unflatten(1, (c["n_kv"], c["hd"])), vc, vs)):
        a, b = _quantize(x)
        codes[page, :, slot] = a
        scales[page, :, :, slot] = b
    return [s["q_out"]] + ([s["k_out"]] if s["k_out"] is not None else []) + _plain_read(s)


def _plain_attend(s):
    """All sequences at once, each filled up to the longest."""
    c, hd, G = s["case"], s["case"]["hd"], s["case"]["n_q"] // s["case"]["n_kv"]
    n, m, top = c["n"], max(s["new_host"]), max(s["lens_host"])
    if top == 0:
        return s["out"].zero_()
    seq, i = s["row"]
    pages = s["table"][:, :(top + c["page"] - 1) // c["page"]].long()
    kc, vc, ks, vs = _page_parts(s["cache"][pages.flatten()], c["n_kv"], c["page"], hd)
    k = _values(kc, ks).unflatten(0, (n, -1)).permute(0, 2, 4, 1, 3).flatten(3)  # [n, n_kv, hd, tokens]
    q = torch.zeros(n, m, c["n_q"] * hd, device=DEV)
    q[seq, i] = s["q"].float()
    q = q.view(n, m, c["n_kv"], G, hd).permute(0, 2, 1, 3, 4).reshape(n, c["n_kv"], m * G, hd)
    z = torch.matmul(q, k.contiguous()).mul_(s["scale"]).unflatten(2, (m, G))
    del k
    # keys before the new ones, and of those the ones with a bit
    j = torch.arange(z.shape[-1], device=DEV)[None] - s["first"].long()[:, None]  # [n, tokens]: a key's number among the new
    words = torch.zeros(n, m, s["see"].shape[1], dtype=torch.int64, device=DEV)
    words[seq, i] = s["see"].long() & 0xffffffff
    at = (j // 32).clamp(0, words.shape[2] - 1)[:, None].expand(n, m, -1)
    keep = (words.gather(2, at) >> (j % 32)[:, None] & 1).bool() & (j < 32 * words.shape[2])[:, None] | (j < 0)[:, None]
    keep &= (j < (s["lens"] - s["first"])[:, None])[:, None]
    z.masked_fill_(~keep[:, None, :, None], -math.inf)
    z.sub_(z.amax(-1, keepdim=True).clamp_(min=torch.finfo(z.dtype).min)).exp_()
    z.div_(z.sum(-1, keepdim=True).clamp_(min=torch.finfo(z.dtype).tiny))
    v = _values(vc, vs).unflatten(0, (n, -1)).transpose(1, 2).flatten(2, 3).contiguous()
    o = torch.matmul(z.flatten(2, 3), v).unflatten(2, (m, G)).permute(0, 2, 1, 3, 4).flatten(2)
    return s["out"].copy_(o[seq, i])


def _plain_verify(s):
    """All sequences a drafted token at a time, in 64 bits: tests and draws lie next to borders."""
    c = s["case"]
    n, m, V = c["n"], max(s["new_host"]), c["vocab"]
    first = s["start"][:-1].long()
    size = s["start"][1:].long() - first
    last = max(0, s["path"].shape[0] - 1)
    seqs = torch.arange(n, device=DEV)
    node = torch.zeros(n, dtype=torch.int64, device=DEV)
    a, total = torch.zeros(n, dtype=torch.float64, device=DEV), torch.ones(n, dtype=torch.float64, device=DEV)
    stuck = torch.zeros(n, dtype=torch.bool, device=DEV)
    out = torch.zeros(n, V, dtype=torch.bool, device=DEV)  # tokens refused at the node, without a draft's probabilities
    path, count = torch.full((n, m), -1, dtype=torch.int64, device=DEV), (size > 0).long()
    path[:, 0] = torch.where(size > 0, 0, -1)
    has_rows = s["path"].shape[0] > 0

    def left():
        row = (first + node).clamp(max=last)
        w = s["p"][row].double()
        if s["q"] is not None:
            w = w - a[:, None] * s["q"][row].double()
        else:
            w = w.masked_fill(out, 0.0)
        return w.clamp(min=0)

    for i in range(1, m):
        here = (first + i).clamp(max=last)
        test = (i < size) & (s["parent"][here].long() == node) & ~stuck
        row, tok = (first + node).clamp(max=last), s["tokens"][here].long()
        pr = s["p"][row, tok].double()
        if s["q"] is not None:
            qr = s["q"][row, tok].double()
            yes = s["u"][here].double() * total * qr < pr - a * qr
        else:
            pr = pr.masked_fill(out[seqs, tok], 0.0)
            yes = s["u"][here].double() * total < pr
        yes, no = test & yes, test & ~yes
        if s["q"] is not None:
            a = torch.where(yes, 0.0, torch.where(no, a + total, a))
            total = torch.where(yes, 1.0, torch.where(no, left().sum(-1), total))
            stuck |= no & ~(total > 0)
        else:
            total = torch.where(yes, 1.0, torch.where(no, total - pr, total))
            out[seqs, tok] |= no
            out &= ~yes[:, None]
        node = torch.where(yes, i, node)
        path.scatter_(1, count.clamp(max=m - 1)[:, None], torch.where(yes, i, path.gather(1, count.clamp(max=m - 1)[:, None])[:, 0])[:, None])
        count += yes
    if has_rows:
        w = left()
        none = ~(w.sum(-1, keepdim=True) > 0)
        w = torch.where(none, s["p"][(first + node).clamp(max=last)].double().clamp(min=0), w)
        cum = w.cumsum(-1)
        t = (cum <= s["u_next"].double()[:, None] * cum[:, -1:]).sum(-1)
        rest = V - 1 - (w > 0).flip(-1).long().argmax(-1)
        t = torch.where(t < V, t, rest)
        t = torch.where((size > 0) & (w > 0).any(-1), t, -1)
    else:
        t = torch.full((n,), -1, dtype=torch.int64, device=DEV)
    at = s["rows"]
    seq = torch.searchsorted(s["start"][1:].long(), torch.arange(s["path"].shape[0], device=DEV), right=True)
    s["path"].copy_(path[seq, at[1]])
    s["count"].copy_(count)
    s["token"].copy_(t)
    return [s["path"], s["count"], s["token"]]


def _plain_keep(s):
    c = s["case"]
    seq, tok = s["slot"]
    i = tok - s["first"].long()[seq]
    mine = i < s["count"].long()[seq]
    src = torch.where(mine, s["first"].long()[seq] + s["path"].long(), tok)
    page, slot = s["table"][seq, src // c["page"]].long(), src % c["page"]
    to, at = s["table"][seq, tok // c["page"]].long(), tok % c["page"]
    kc, vc, ks, vs = _page_parts(s["cache"], c["n_kv"], c["page"], c["hd"])
    for codes, scales in ((kc, ks), (vc, vs)):
        codes[to, :, at] = codes[page, :, slot]
        scales[to, :, :, at] = scales[page, :, :, slot]
    s["new_lens"].copy_(s["first"] + s["count"])
    return [s["new_lens"]] + _plain_read(s)


def run(s):
    c, vla = s["case"], s["vla"]
    if not own:
        return {"tree": _plain_tree, "append": _plain_append, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[c["kind"]](s)
    if c["kind"] == "tree":
        vla.draft_tree_dev(s["pos"], s["see"], s["parent"], s["lens"], s["start"])
        return [s["pos"], s["see"]]
    if c["kind"] == "verify":
        vla.verify_drafts_dev(s["path"], s["count"], s["token"], s["p"], s["tokens"], s["start"], s["u"], s["u_next"],
                              parent=s["parent"], q=s["q"])
        return [s["path"], s["count"], s["token"]]
    if c["kind"] == "attend":
        vla.kv4_tree_attention_dev(s["out"], s["q"], s["cache"], c["n_q"], c["n_kv"], c["hd"], c["page"], s["scale"], s["table"],
                                   s["lens"], s["start"], s["see"], max_new=c["nodes"], max_len=c["longest"], work=s["work"])
        return s["out"]
    if c["kind"] == "append":
        vla.rope_kv4_append_dev(s["q_out"], s["cache"], s["q"], s["k"], s["v"], c["n_q"], c["n_kv"], c["hd"], c["page"], s["table"],
                                s["lens"], s["start"], s["freqs"], pos=s["pos"], magnitude=s["magnitude"], interleaved=c["inter"],
                                q_weight=s["wq"], k_weight=s["wk"], eps=s["eps"], k_out=s["k_out"])
        got = [s["q_out"]] + ([s["k_out"]] if s["k_out"] is not None else [])
    else:
        vla.kv4_keep_dev(s["cache"], c["n_kv"], c["hd"], c["page"], s["table"], s["lens"], s["start"], s["path"], s["count"],
                         new_lens=s["new_lens"])
        got = [s["new_lens"]]
    vla.kv4_gather_dev(s["k_back"], s["v_back"], s["cache"], c["n_kv"], c["hd"], c["page"], s["table"], s["start"], s["first"])
    return got + [s["k_back"], s["v_back"]]


# -------------------------------------------------------- the definitions --

def _exact_quantized(x):
    """The nearest values of the 4-bit cache, in 64 bits: every candidate is tried."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.full_like(amax, E_MIN)
    top = torch.ceil(torch.log2(amax.clamp(min=1e-60) / 7))
    for d in (1, 0, -1):  # the smallest exponent that holds the block, whatever the logarithm's last bit
        e = torch.where((amax <= 7 * torch.exp2(top + d)) & (amax > 0), (top + d).clamp(min=E_MIN), e)
    y = b.abs() / torch.exp2(e)
    best, dist = torch.zeros_like(y), y.clone()
    for i, v in enumerate(GRID[1:], 1):
        d = (y - v).abs()
        take = (d < dist) | ((d == dist) & (i % 2 == 0))
        best, dist = torch.where(take, torch.full_like(y, v), best), torch.where(take, d, dist)
    return (torch.copysign(best, b) * torch.exp2(e)).flatten(-2)


def _exact_row(s, seq, toks, head, part):
    """[toks, hd] cached values of one head in 64 bits, byte by byte from the layout."""
    c, hd = s["case"], s["case"]["hd"]
    page, slot = s["table"][seq][toks // c["page"]].long(), toks % c["page"]
    half = c["n_kv"] * c["page"] * hd // 2
    at = part * half + (head * c["page"] + slot) * (hd // 2)
    by = s["cache"][page[:, None], at[:, None] + torch.arange(hd // 2, device=DEV)].long()
    code = torch.stack([by % 16, by // 16], 2).reshape(-1, hd)
    sc = 2 * half + (part * c["n_kv"] + head) * (hd // BLOCK) * c["page"]
    sc = sc + torch.arange(hd // BLOCK, device=DEV)[None] * c["page"] + slot[:, None]
    scale = torch.exp2(s["cache"][page[:, None], sc].double() - 127).repeat_interleave(BLOCK, 1)
    lut = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    return torch.where(code >= 8, -1.0, 1.0) * lut[code % 8] * scale


def _exact_rotated(x, w, s, heads):
    """Pairs as complex numbers, turned by their angle."""
    c, rot = s["case"], s["case"]["rot"]
    v = x.double().reshape(x.shape[0], heads, c["hd"]).clone()
    if w is not None:
        v = v / torch.sqrt((v ** 2).sum(2, keepdim=True) / c["hd"] + s["eps"]) * w.double()
    turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["freqs"][None])
    pairs = v[..., :rot].reshape(*v.shape[:2], rot // 2, 2) if c["inter"] else v[..., :rot].reshape(*v.shape[:2], 2, rot // 2).transpose(2, 3)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    v[..., :rot] = (z if c["inter"] else z.transpose(2, 3)).reshape(*v.shape[:2], rot)
    return v


def _exact_verify(c, s):
    """Sequence by sequence, on the host where whole rows are not needed."""
    parents, path, count, token = _parents(c), [], [], []
    tokens, u, u_next = s["tokens"].tolist(), s["u"].double().tolist(), s["u_next"].double().tolist()
    for k, (p0, ps) in enumerate(zip(_starts(_new(c)), parents)):
        kept = [0] if ps else []
        at, i = 0, 1
        P, Q, a, mass, refused = (s["p"][p0].double() if ps else None), None, 0.0, 1.0, []
        if ps and c["sampled"]:
            Q = s["q"][p0].double()
        dead = False
        while i < len(ps):
            if ps[i] == at and not dead:
                t = tokens[p0 + i]
                pt = float(P[t]) if t not in refused else 0.0
                if c["sampled"]:
                    qt = float(Q[t])
                    ok = u[p0 + i] * mass * qt < pt - a * qt
                else:
                    ok = u[p0 + i] * mass < pt
                if ok:
                    at, a, mass, refused = i, 0.0, 1.0, []
                    kept.append(i)
                    P = s["p"][p0 + i].double()
                    Q = s["q"][p0 + i].double() if c["sampled"] else None
                elif c["sampled"]:
                    a += mass
                    d = P - a * Q
                    mass = float(d[d > 0].sum())
                    dead = not mass > 0
                else:
                    mass -= pt
                    refused.append(t)
            i += 1
        if not ps:
            token.append(-1)
            count.append(0)
            continue
        w = P - a * Q if c["sampled"] else P.clone()
        if refused:
            w[refused] = 0
        w = torch.where(w > 0, w, torch.zeros_like(w))
        if not float(w.sum()) > 0:
            w = torch.where(P > 0, P, torch.zeros_like(P))
        w = w.cpu().numpy()
        run_sum = np.cumsum(w)
        over = np.nonzero(run_sum > u_next[k] * run_sum[-1])[0]
        some = np.nonzero(w > 0)[0]
        token.append(int(over[0]) if len(over) else int(some[-1]) if len(some) else -1)
        count.append(len(kept))
        path += kept + [-1] * (len(ps) - len(kept))
    return [_i32(path), _i32(count), _i32(token)]


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    new, lens = _new(c), _lens(c)
    if c["kind"] == "tree":
        s["see"] = _bit_words(c)
        back = (s["lens"] - _i32(new)).tolist()
        return [_i32(_flat([b + d for d in _seen(p)[1]] for b, p in zip(back, _parents(c)))), s["see"]]
    if c["kind"] == "verify":
        return _exact_verify(c, s)
    hd = c["hd"]
    if c["kind"] == "append":
        q, k = _exact_rotated(s["q"], s["wq"], s, c["n_q"]), _exact_rotated(s["k"], s["wk"], s, c["n_kv"])
        v = s["v"].reshape(s["v"].shape[0], c["n_kv"], hd)
        return [q.flatten(1)] + ([k.flatten(1)] if c["rows_out"] else []) + [_exact_quantized(x).flatten(1) for x in (k, v)]
    if c["kind"] == "keep":
        path, out = s["path"].tolist(), [[], []]
        count, at = s["count"].tolist(), 0
        for i, (m, f) in enumerate(zip(new, s["first"].tolist())):
            src = [f + path[at + j] if j < count[i] else f + j for j in range(m)]
            toks = torch.tensor(src, dtype=torch.int64, device=DEV)
            for part in range(2):
                if m:
                    out[part].append(torch.cat([_exact_row(s, i, toks, h, part) for h in range(c["n_kv"])], 1))
            at += m
        none = torch.zeros(0, c["n_kv"] * hd, dtype=torch.float64, device=DEV)
        return [_i32([f + k for f, k in zip(s["first"].tolist(), count)])] + [torch.cat(o + [none]) for o in out]
    G, out, q0 = c["n_q"] // c["n_kv"], [], 0
    for i, (m, n, ps) in enumerate(zip(new, lens, _parents(c))):
        if not m:
            continue
        see = torch.ones(m, n, dtype=torch.bool)
        for r, bits in enumerate(_seen(ps)[0]):
            see[r, n - m:] = torch.tensor([bits >> j & 1 for j in range(m)], dtype=torch.bool)
        see = see.to(DEV)
        heads = []
        for h in range(c["n_kv"]):
            k, v = (_exact_row(s, i, torch.arange(n, device=DEV), h, part) for part in range(2))
            for j in range(h * G, (h + 1) * G):
                z = torch.mm(s["q"][q0:q0 + m, j * hd:(j + 1) * hd].double(), k.t().contiguous()) * s["scale"]
                z = torch.where(see, z, torch.full_like(z, -1e300))
                w = torch.exp(z - z.max(1, keepdim=True).values) * see
                heads.append(torch.mm(w, v) / w.sum(1, keepdim=True))
        out.append(torch.cat(heads, 1))
        q0 += m
    return torch.cat(out + [torch.zeros(0, c["n_q"] * hd, dtype=torch.float64, device=DEV)])
