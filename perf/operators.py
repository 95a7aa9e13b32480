"""The operators of a decoder that serves several prompts, as cases that can be timed and checked.

Kinds:
  rope     vla_qk_norm_rope_dev: the norms of queries and keys per head and the
           rotation by positions of one or several axes, in one pass
  prompt   vla_packed_attention_dev: attention over packed sequences of
           different lengths, causal or not, with grouped heads
  cache    vla_kv4_append_dev and vla_kv4_gather_dev: rows into a paged cache of
           4-bit values, and the same tokens read back as rows
  decode   vla_kv4_attention_dev: attention of the newest tokens over that cache

`run` computes a pass with elementary torch operations in 32 bits, or with
`own` set through the framework's calls; `exact` is the definition in 64 bits.
"""

from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32  # values of a head that share a scale in the 4-bit cache
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E_MIN = -100


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
        # one decoded token of SmolVLA's language tower: the smallest call
        dict(name="rope_token", kind="rope", T=1, n_q=15, n_kv=5, hd=64, axes=1, norm=True, fused=True, dtype="f32"),
        # the image and text tokens of a few camera views, rows of a fused qkv buffer
        dict(name="rope_views", kind="rope", T=2371, n_q=16, n_kv=8, hd=128, axes=3, norm=True, fused=True, dtype="bf16"),
        # every token of a large batch of prompts
        dict(name="rope_prompts", kind="rope", T=32768, n_q=32, n_kv=8, hd=128, axes=3, norm=True, fused=False, dtype="f16"),
        # the prefixes of eight robots, 177 tokens at most, in the framework's own type
        dict(name="prompt_prefixes", kind="prompt", n=8, longest=177, past=0, spread=5, n_q=15, n_kv=5, hd=64, causal=True, dtype="f32"),
        # prompts of mixed lengths, an empty one and one of a single token among them
        dict(name="prompt_ragged", kind="prompt", n=12, longest=2048, past=0, spread=3, n_q=32, n_kv=8, hd=128, causal=True, dtype="bf16"),
        # one long prompt
        dict(name="prompt_long", kind="prompt", n=1, longest=8192, past=0, spread=0, n_q=32, n_kv=8, hd=128, causal=True, dtype="bf16"),
        # the 1024 patches of three images through SigLIP's heads, without a mask
        dict(name="prompt_images", kind="prompt", n=3, longest=1024, past=0, spread=0, n_q=12, n_kv=12, hd=64, causal=False, dtype="f16"),
        # the prefixes of eight robots into the cache and back
        dict(name="cache_prefixes", kind="cache", n=8, longest=177, past=0, spread=5, n_kv=5, hd=64, page=64, dtype="f32"),
        # a later piece of sixteen prompts, behind what the cache holds already
        dict(name="cache_prompts", kind="cache", n=16, longest=4096, past=333, spread=2, n_kv=8, hd=128, page=64, dtype="bf16"),
        # one token of one robot over its prefix and chunk
        dict(name="decode_robot", kind="decode", n=1, longest=227, spread=0, new=1, n_q=15, n_kv=5, hd=64, page=64, dtype="f32"),
        # one token for each of 48 conversations of mixed lengths
        dict(name="decode_batch", kind="decode", n=48, longest=8192, spread=4, new=1, n_q=32, n_kv=8, hd=128, page=64, dtype="bf16"),
        # one token for two very long documents: few rows, a long axis
        dict(name="decode_long", kind="decode", n=2, longest=131072, spread=0, new=1, n_q=32, n_kv=8, hd=128, page=256, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "prompt", "prompt", "cache", "decode", "decode"])
    n_q, n_kv = rng.choice([(15, 5), (32, 8), (16, 2), (12, 12), (8, 1), (16, 8)])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "rope":
        hd = rng.choice([32, 64, 64, 96, 128, 128, 256])
        most = 32768 * 40 * 128 * 2 // ((n_q + n_kv) * hd * SIZE[dtype])
        return dict(kind=kind, T=_log(rng, 1, min(32768, most)), n_q=n_q, n_kv=n_kv, hd=hd, axes=rng.randint(1, 4),
                    norm=rng.random() < 0.7, fused=rng.random() < 0.5, dtype=dtype)
    if kind == "prompt":
        hd = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
        n = _log(rng, 1, 24)
        # sums of squares of lengths well below those of one prompt of 8192
        most = int(8192 * math.sqrt((0.12 if dtype == "f32" else 0.7) * 32 * 128 / (2 * n * n_q * hd)))
        return dict(kind=kind, n=n, longest=_log(rng, 1, min(8192, most)), past=rng.choice([0, 0, rng.randint(1, 700)]) if most > 1500 else 0,
                    spread=rng.randint(0, 6), n_q=n_q, n_kv=n_kv, hd=hd, causal=rng.random() < 0.75, dtype=dtype)
    hd = rng.choice([32, 64, 64, 96, 128, 128, 256])
    page = rng.choice([32, 64, 64, 96, 128, 256])
    if kind == "cache":
        n = _log(rng, 1, 64)
        most = 16 * 4096 * 8 * 128 // (n * n_kv * hd)
        return dict(kind=kind, n=n, longest=_log(rng, 1, max(2, min(8192, most))), past=rng.choice([0, rng.randint(1, 999)]),
                    spread=rng.randint(0, 6), n_kv=n_kv, hd=hd, page=page, dtype=dtype)
    n = _log(rng, 1, 64)
    most = 2 * 131072 * 8 * 128 // (n * n_kv * hd)
    return dict(kind=kind, n=n, longest=_log(rng, 1, max(2, min(131072, most))), spread=rng.randint(0, 6),
                new=rng.choice([1, 1, 1, rng.randint(2, 50)]), n_q=n_q, n_kv=n_kv, hd=hd, page=page, dtype=dtype)


# ---------------------------------------------------------------- sizes --

def _lens(c):
    """Lengths of the sequences: all the longest with spread 0, else mixed, the first the longest."""
    n, top = c["n"], c["longest"]
    if not c["spread"]:
        return [top] * n
    r = random.Random(c["spread"] * 1009 + n * 31 + top)
    out = [top] + [_log(r, max(1, top // 16), top) for _ in range(n - 1)]
    if n >= 4:
        out[n // 2], out[n - 1] = 0, 1
    return out


def _sections(c):
    """Rotated pairs of each axis: three axes as time, height and width, otherwise nearly equal parts."""
    half, a = c["hd"] // 2, c["axes"]
    if a == 3:
        t = half // 4
        h = (half - t) // 2
        return [t, h, half - t - h]
    return [half // a + (i < half % a) for i in range(a)]


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _new(c):
    """New tokens of each sequence of a decode pass: no more than it has."""
    return [min(c["new"], n) for n in _lens(c)]


def _pairs(n_q, n_k, causal):
    if not causal:
        return n_q * n_k
    return sum(max(0, min(n_k, i + 1 + n_k - n_q)) for i in range(n_q))


def work(case):
    c, sz = case, SIZE[case["dtype"]]
    if c["kind"] == "rope":
        n = c["T"] * (c["n_q"] + c["n_kv"]) * c["hd"]
        return {"bytes": 2 * n * sz + 4 * c["axes"] * c["T"] + (8 * c["hd"] if c["norm"] else 0), "flops": 9 * n}
    lens = _lens(c)
    if c["kind"] == "prompt":
        q, k = sum(lens), sum(n + c["past"] for n in lens)
        pairs = sum(_pairs(n, n + c["past"], c["causal"]) for n in lens)
        return {"bytes": 2 * sz * c["hd"] * (q * c["n_q"] + k * c["n_kv"]) + 8 * (c["n"] + 1),
                "flops": 4 * pairs * c["hd"] * c["n_q"]}
    if c["kind"] == "cache":  # rows in, 4-bit values and scales out; the same in, rows out
        n = 2 * sum(lens) * c["n_kv"] * c["hd"]
        return {"bytes": 2 * (n * sz + n * 17 // 32), "flops": 4 * n}
    new = _new(c)
    pairs = sum(_pairs(m, n, True) for m, n in zip(new, lens))
    return {"bytes": sum(lens) * c["n_kv"] * c["hd"] * 17 // 16 + 2 * sz * c["hd"] * c["n_q"] * sum(new) + 4 * c["n"],
            "flops": 4 * pairs * c["hd"] * c["n_q"]}


# --------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(DEV).manual_seed(int(seed) * 7919 + 29)


def _n(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _positions(c, seed):
    """Positions of a prompt: a run of text counts on every axis, an image keeps its time and counts rows and columns."""
    T, a = c["T"], c["axes"]
    off = random.Random(int(seed)).randint(0, 4000)
    t = torch.arange(T, device=DEV) + off
    if a == 1:
        return t.to(torch.int32).view(1, T)
    side = 32
    img = (torch.arange(T, device=DEV) // (side * side)) % 2 == 0
    within = torch.arange(T, device=DEV) % (side * side)
    axes = [torch.where(img, t - within, t), torch.where(img, off + within // side, t), torch.where(img, off + within % side, t)]
    axes += [t]
    return torch.stack(axes[:a]).to(torch.int32).contiguous()


def _rows(g, T, widths, dtype, fused):
    """Row blocks of these widths: views of one buffer where `fused`, else each its own."""
    if fused:
        buf = _n(g, T, sum(widths), dtype=dtype)
        out, at = [], 0
        for w in widths:
            out.append(buf[:, at:at + w])
            at += w
        return out
    return [_n(g, T, w, dtype=dtype) for w in widths]


def _quantize(x):
    """[..., hd] values -> (codes [..., hd/2] with the even value in the low half, scale bytes [..., hd/32])."""
    b = x.float().unflatten(-1, (-1, BLOCK))
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


def prepare(case, seed):
    c, g, dt = case, _gen(seed), DTYPES[case["dtype"]]
    s = {"case": c, "vla": _pkg() if own else None}
    if c["kind"] == "rope":
        wq, wk = c["n_q"] * c["hd"], c["n_kv"] * c["hd"]
        s["q"], s["k"], _ = _rows(g, c["T"], [wq, wk, wk], dt, c["fused"])
        s["pos"], s["sections"], s["base"], s["eps"] = _positions(c, seed), _sections(c), 10000.0, 1e-6
        s["wq"] = 1 + _n(g, c["hd"], std=0.1) if c["norm"] else None
        s["wk"] = 1 + _n(g, c["hd"], std=0.1) if c["norm"] else None
        s["q_out"] = torch.empty(c["T"], wq, dtype=dt, device=DEV)
        s["k_out"] = torch.empty(c["T"], wk, dtype=dt, device=DEV)
        return s
    lens = _lens(c)
    s["lens_host"] = lens
    if c["kind"] == "prompt":
        klens = [n + c["past"] for n in lens]
        s["klens_host"] = klens
        s["q"] = _n(g, sum(lens), c["n_q"] * c["hd"], dtype=dt)
        s["k"], s["v"] = (_n(g, sum(klens), c["n_kv"] * c["hd"], dtype=dt) for _ in range(2))
        s["out"] = torch.empty_like(s["q"])
        s["q_start"] = _i32(_starts(lens))
        s["k_start"] = _i32(_starts(klens)) if c["past"] else None
        s["scale"] = 1.0 / math.sqrt(c["hd"])
    elif c["kind"] == "cache":
        total = [n + c["past"] for n in lens]
        s["k"], s["v"] = (_n(g, sum(lens), c["n_kv"] * c["hd"], dtype=dt) for _ in range(2))
        s["table"], pages = _table(c, total, g)
        s["cache"] = torch.zeros(pages, _page_bytes(c["n_kv"], c["page"], c["hd"]), dtype=torch.uint8, device=DEV)
        s["start"], s["lens"], s["first"] = _i32(_starts(lens)), _i32(total), _i32([c["past"]] * c["n"])
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    else:
        new = _new(c)
        s["new_host"] = new
        s["table"], pages = _table(c, lens, g)
        s["cache"] = torch.zeros(pages, _page_bytes(c["n_kv"], c["page"], c["hd"]), dtype=torch.uint8, device=DEV)
        step = max(1, (1 << 25) // (c["n_kv"] * c["page"] * c["hd"]))
        for p in range(0, pages, step):
            part = s["cache"][p:p + step]
            kc, vc, ks, vs = _page_parts(part, c["n_kv"], c["page"], c["hd"])
            for codes, scales in ((kc, ks), (vc, vs)):
                a, b = _quantize(_n(g, part.shape[0], c["n_kv"], c["page"], c["hd"]))
                codes.copy_(a)
                scales.copy_(b.transpose(2, 3))
        s["q"] = _n(g, sum(new), c["n_q"] * c["hd"], dtype=dt)
        s["out"] = torch.empty_like(s["q"])
        s["lens"], s["q_start"] = _i32(lens), _i32(_starts(new))
        s["scale"] = 1.0 / math.sqrt(c["hd"])
        s["work"] = None
        if own:
            n = s["vla"].kv4_attention_work_bytes(sum(new), c["n"], max(new), c["longest"], c["n_q"], c["n_kv"], c["hd"])
            s["work"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------- the plain forms --

def _plain_rope(x, w, s, heads):
    c = s["case"]
    half = c["hd"] // 2
    v = x.float().unflatten(1, (heads, c["hd"]))
    if w is not None:
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + s["eps"]) * w
    axis = torch.repeat_interleave(torch.arange(c["axes"], device=DEV), torch.tensor(s["sections"], device=DEV))
    freq = s["base"] ** (-2.0 * torch.arange(half, device=DEV, dtype=torch.float64) / c["hd"])
    angle = s["pos"].double()[axis].t() * freq
    co, si = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = v[..., :half], v[..., half:]
    return torch.cat([a * co - b * si, a * si + b * co], -1).flatten(1).to(x.dtype)


def _plain_softmax(p, keep):
    """Weights of scores [..., n_q, n_k] (overwritten) under the truth values `keep`; zeros where a row keeps nothing."""
    if keep is not None:
        p.masked_fill_(~keep, -math.inf)
    top = p.amax(-1, keepdim=True).clamp_(min=torch.finfo(p.dtype).min)
    p.sub_(top).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp_(min=torch.finfo(p.dtype).tiny))


def _plain_prompt(s):
    c = s["case"]
    G, hd = c["n_q"] // c["n_kv"], c["hd"]
    out, q0, k0 = s["out"], 0, 0
    for m, n in zip(s["lens_host"], s["klens_host"]):
        keep = None
        if c["causal"] and m:
            keep = torch.arange(n, device=DEV)[None] <= torch.arange(m, device=DEV)[:, None] + (n - m)
        for h in range(c["n_kv"] if m else 0):
            q = s["q"][q0:q0 + m, h * G * hd:(h + 1) * G * hd].float().unflatten(1, (G, hd)).transpose(0, 1).contiguous()
            k = s["k"][k0:k0 + n, h * hd:(h + 1) * hd].float()
            v = s["v"][k0:k0 + n, h * hd:(h + 1) * hd].float()
            p = _plain_softmax(torch.matmul(q, k.t().contiguous()).mul_(s["scale"]), keep)
            out[q0:q0 + m, h * G * hd:(h + 1) * G * hd] = torch.matmul(p, v).transpose(0, 1).flatten(1).to(out.dtype)
        q0, k0 = q0 + m, k0 + n
    return out


def _values(codes, scales):
    """fp32 values [..., page, hd] of codes [..., page, hd/2] and scale bytes [..., hd/32, page]."""
    lut = torch.tensor(GRID + tuple(-x for x in GRID), device=DEV)
    c = codes.int()
    x = torch.stack([lut[c & 15], lut[c >> 4]], -1).flatten(-2)
    e = torch.exp2(scales.float() - 127)
    e = torch.where(scales == 255, torch.full_like(e, math.nan), e).transpose(-1, -2)
    return (x.unflatten(-1, (-1, BLOCK)) * e[..., None]).flatten(-2)


def _slots(s, starts, firsts, lens):
    """(page, slot) of each packed row."""
    c = s["case"]
    tok = torch.cat([torch.arange(f, f + n, device=DEV) for f, n in zip(firsts, lens)])
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(lens, device=DEV))
    return s["table"][seq, tok // c["page"]].long(), tok % c["page"]


def _plain_cache(s):
    c = s["case"]
    page, slot = _slots(s, s["start"], [c["past"]] * c["n"], s["lens_host"])
    kc, vc, ks, vs = _page_parts(s["cache"], c["n_kv"], c["page"], c["hd"])
    out = []
    for x, codes, scales, o in ((s["k"], kc, ks, s["k_out"]), (s["v"], vc, vs, s["v_out"])):
        a, b = _quantize(x.unflatten(1, (c["n_kv"], c["hd"])))
        codes[page, :, slot] = a
        scales[page, :, :, slot] = b
        back = _values(codes[page, :, slot][:, :, None], scales[page, :, :, slot][..., None])
        out.append(o.copy_(back.squeeze(2).flatten(1)))
    return out


def _plain_decode(s):
    c = s["case"]
    G, hd = c["n_q"] // c["n_kv"], c["hd"]
    out, q0 = s["out"], 0
    for i, (m, n) in enumerate(zip(s["new_host"], s["lens_host"])):
        if not m:
            continue
        pages = s["table"][i, :(n + c["page"] - 1) // c["page"]].long()
        kc, vc, ks, vs = _page_parts(s["cache"][pages], c["n_kv"], c["page"], hd)
        k = _values(kc, ks).transpose(0, 1).flatten(1, 2)[:, :n]
        v = _values(vc, vs).transpose(0, 1).flatten(1, 2)[:, :n].contiguous()
        q = s["q"][q0:q0 + m].float().view(m, c["n_kv"], G, hd).permute(1, 2, 0, 3).reshape(c["n_kv"], G * m, hd)
        keep = None
        if m > 1:
            keep = torch.arange(n, device=DEV)[None] <= torch.arange(m, device=DEV)[:, None] + (n - m)
            keep = keep.repeat(G, 1)
        p = _plain_softmax(torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s["scale"]), keep)
        o = torch.matmul(p, v).view(c["n_kv"], G, m, hd).permute(2, 0, 1, 3).reshape(m, -1)
        out[q0:q0 + m] = o.to(out.dtype)
        q0 += m
    return out


def run(s):
    c, vla = s["case"], s["vla"]
    if c["kind"] == "rope":
        if own:
            vla.qk_norm_rope_dev(s["q_out"], s["k_out"], s["q"], s["k"], c["n_q"], c["n_kv"], c["hd"], s["pos"], s["sections"],
                                 s["base"], s["wq"], s["wk"], s["eps"])
        else:
            s["q_out"].copy_(_plain_rope(s["q"], s["wq"], s, c["n_q"]))
            s["k_out"].copy_(_plain_rope(s["k"], s["wk"], s, c["n_kv"]))
        return [s["q_out"], s["k_out"]]
    if c["kind"] == "prompt":
        if not own:
            return _plain_prompt(s)
        vla.packed_attention_dev(s["out"], s["q"], s["k"], s["v"], c["n_q"], c["n_kv"], c["hd"], s["scale"], s["q_start"],
                                 s["k_start"], causal=c["causal"])
        return s["out"]
    if c["kind"] == "cache":
        if not own:
            return _plain_cache(s)
        vla.kv4_append_dev(s["cache"], s["k"], s["v"], c["n_kv"], c["hd"], c["page"], s["table"], s["lens"], s["start"])
        vla.kv4_gather_dev(s["k_out"], s["v_out"], s["cache"], c["n_kv"], c["hd"], c["page"], s["table"], s["start"], s["first"])
        return [s["k_out"], s["v_out"]]
    if not own:
        return _plain_decode(s)
    vla.kv4_attention_dev(s["out"], s["q"], s["cache"], c["n_q"], c["n_kv"], c["hd"], c["page"], s["scale"], s["table"], s["lens"],
                          q_start=s["q_start"], max_new=c["new"], max_len=c["longest"], work=s["work"])
    return s["out"]


# -------------------------------------------------------- the definitions --

def _exact_heads(q, k, v, scale, causal):
    """Attention of one head's queries [m, hd] over keys [n, hd] in 64 bits, a strip of queries at a time."""
    m, n = q.shape[0], k.shape[0]
    out = torch.zeros(m, q.shape[1], dtype=torch.float64, device=DEV)
    j = torch.arange(n, device=DEV)
    step = max(1, (1 << 27) // max(1, n))
    for a in range(0, m, step):
        b = min(m, a + step)
        z = torch.mm(q[a:b], k.t().contiguous()) * scale
        see = torch.ones(b - a, n, dtype=torch.bool, device=DEV)
        if causal:
            see = j[None, :] + (m - n) <= torch.arange(a, b, device=DEV)[:, None]
        some = see.any(1)
        z = torch.where(see, z, torch.full_like(z, -1e300))
        w = torch.exp(z - z.max(1, keepdim=True).values) * see
        out[a:b] = torch.where(some[:, None], torch.mm(w, v) / w.sum(1, keepdim=True).clamp(min=1e-300), out[a:b])
    return out


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


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    hd = c["hd"]
    if c["kind"] == "rope":
        out = []
        for x, w, heads in ((s["q"], s["wq"], c["n_q"]), (s["k"], s["wk"], c["n_kv"])):
            v = x.double().reshape(c["T"], heads, 2, hd // 2)
            if w is not None:
                v = v / torch.sqrt((v ** 2).sum((2, 3), keepdim=True) / hd + s["eps"]) * w.double().view(2, hd // 2)
            at = torch.cat([s["pos"][a].double()[:, None].expand(c["T"], n) for a, n in enumerate(s["sections"])], 1)
            z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                            at * torch.exp(torch.arange(hd // 2, device=DEV).double() * (-2.0 / hd * math.log(s["base"]))))
            z = torch.complex(v[:, :, 0].contiguous(), v[:, :, 1].contiguous()) * z[:, None]
            out.append(torch.stack([z.real, z.imag], 2).reshape(c["T"], heads * hd))
        return out
    if c["kind"] == "cache":
        return [_exact_quantized(x.reshape(x.shape[0], c["n_kv"], hd)).reshape(x.shape[0], c["n_kv"] * hd) for x in (s["k"], s["v"])]
    G = c["n_q"] // c["n_kv"]
    if c["kind"] == "prompt":
        qn, kn = _lens(c), [n + c["past"] for n in _lens(c)]
        causal = c["causal"]
    else:
        qn, kn, causal = _new(c), _lens(c), True
        lut = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    out = torch.zeros(sum(qn), c["n_q"] * hd, dtype=torch.float64, device=DEV)
    qs, ks = _starts(qn), _starts(kn)
    for i in range(c["n"]):
        if not qn[i]:
            continue
        for h in range(c["n_kv"]):
            if c["kind"] == "prompt":
                k, v = (s[x][ks[i]:ks[i + 1], h * hd:(h + 1) * hd].double() for x in ("k", "v"))
            else:
                tok = torch.arange(kn[i], device=DEV)
                page, slot = s["table"][i][tok // c["page"]].long(), tok % c["page"]
                kv, half = [], c["n_kv"] * c["page"] * hd // 2
                for part in range(2):
                    at = part * half + (h * c["page"] + slot) * (hd // 2)
                    by = s["cache"][page[:, None], at[:, None] + torch.arange(hd // 2, device=DEV)].long()
                    code = torch.stack([by % 16, by // 16], 2).reshape(-1, hd)
                    sc = 2 * half + (part * c["n_kv"] + h) * (hd // BLOCK) * c["page"]
                    sc = sc + torch.arange(hd // BLOCK, device=DEV)[None] * c["page"] + slot[:, None]
                    scale = torch.exp2(s["cache"][page[:, None], sc].double() - 127).repeat_interleave(BLOCK, 1)
                    kv.append(torch.where(code >= 8, -1.0, 1.0) * lut[code % 8] * scale)
                k, v = kv
            for j in range(h * G, (h + 1) * G):
                cols = slice(j * hd, (j + 1) * hd)
                out[qs[i]:qs[i + 1], cols] = _exact_heads(s["q"][qs[i]:qs[i + 1], cols].double(), k, v, s["scale"], causal)
    return out
