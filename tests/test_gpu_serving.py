"""GPU tests of the operators that serve several prompts, each against its plain
64-bit form (serving_ref.py), whose bounds are derived there."""

import math

import numpy as np
import pytest
import torch

import serving_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
DEV = "cuda"


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(g, n, width, dtype, std=1.0, pad=0):
    """[n, width] host rows; with pad a view of wider rows."""
    return (torch.randn(n, width + pad, generator=g) * std).to(dtype)[:, :width]


def _dev(t, pad=0):
    """The same rows on the GPU, `pad` values between them."""
    if t is None:
        return None
    if not pad:
        return t.contiguous().to(DEV)
    buf = torch.full((t.shape[0], t.shape[1] + pad), 7.0, dtype=t.dtype, device=DEV)
    buf[:, pad // 2 // 8 * 8:][:, :t.shape[1]] = t.to(DEV)
    return buf[:, pad // 2 // 8 * 8:][:, :t.shape[1]]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lens):
    return [0] + list(np.cumsum(lens).tolist())


# ------------------------------------------------------------------ rope --

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,n_q,n_kv,hd,sections,norm,pad", [
    (1, 15, 5, 64, [32], True, 0), (1, 1, 0, 8, [4], False, 0), (3, 0, 2, 24, [5, 7], True, 16), (7, 4, 4, 32, [4, 6, 6], True, 64),
    (33, 8, 1, 96, [48], False, 0), (129, 2, 2, 256, [32, 48, 48], True, 8), (17, 3, 1, 136, [10, 0, 58], True, 0),
    (65, 16, 8, 128, [8] * 8, False, 8), (5, 70, 30, 40, [20], True, 0),
])
def test_rope(vla, dtype, T, n_q, n_kv, hd, sections, norm, pad):
    g = _gen(T * 131 + hd)
    q, k = _rows(g, T, n_q * hd, dtype, 2.0), _rows(g, T, n_kv * hd, dtype, 0.3)
    wq, wk = (1 + 0.2 * torch.randn(hd, generator=g) if norm else None for _ in range(2))
    pos = torch.randint(-5, 5000, (len(sections), T), generator=g, dtype=torch.int32)
    dq, dk = _dev(q, pad), _dev(k, pad)
    qo, ko = _dev(torch.zeros_like(q), pad), _dev(torch.zeros_like(k), pad)
    args = (n_q, n_kv, hd, pos.to(DEV), sections, 10000.0, _dev(wq), _dev(wk), 1e-5)
    vla.qk_norm_rope_dev(qo if n_q else None, ko if n_kv else None, dq if n_q else None, dk if n_kv else None, *args)
    torch.cuda.synchronize()
    for name, x, o, h, w in (("q", q, qo, n_q, wq), ("k", k, ko, n_kv, wk)):
        if h:
            want, bound = ref.rope(x, h, hd, pos, sections, 10000.0, w, 1e-5)
            ref.within(o, want, bound, name)
            if pad:  # what lies between the rows is left alone
                full = torch.as_strided(o, (T, h * hd + pad), (h * hd + pad, 1), o.storage_offset() - pad // 2 // 8 * 8)
                assert float((full.double() == 7.0).sum()) >= T * pad - 1
    # in place: the same bits
    a, b = qo.clone(), ko.clone()
    vla.qk_norm_rope_dev(dq if n_q else None, dk if n_kv else None, dq if n_q else None, dk if n_kv else None, *args)
    assert torch.equal(dq if n_q else a, a) and torch.equal(dk if n_kv else b, b)


def test_rope_far_positions(vla):
    """Positions of 2^31 keep their angle (an fp32 product would be off by whole turns)."""
    g = _gen(3)
    pos = torch.tensor([[0, 1, 2 ** 31 - 1, -(2 ** 31), 10 ** 6, 123456789]], dtype=torch.int32)
    x = _rows(g, 6, 2 * 64, F32)
    o = torch.empty(6, 128, device=DEV)
    vla.qk_norm_rope_dev(o, None, x.to(DEV), None, 2, 0, 64, pos.to(DEV), [32], 500000.0)
    want, bound = ref.rope(x, 2, 64, pos, [32], 500000.0, None, 0.0)
    # 2^31 radians in 64 bits, in the reference and in the kernel: 2^31 * 2^-53 * 4 more
    ref.within(o, want, bound + 2.0 ** -20 * (x.double().abs().max() * 2), "far")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e25, 1e-25, 1e-38, 1e37])
def test_norm_beyond_the_range_of_squares(vla, dtype, size):
    """Values whose squares overflow or vanish in 32 bits are normed all the same."""
    x = (_rows(_gen(6), 5, 2 * 64, F32) * size).to(dtype)
    pos = torch.arange(5, dtype=torch.int32)[None]
    w = torch.ones(64)
    o = torch.empty(5, 128, dtype=dtype, device=DEV)
    vla.qk_norm_rope_dev(o, None, x.to(DEV), None, 2, 0, 64, pos.to(DEV), [32], 1e4, w.to(DEV), None, 0.0)
    want, bound = ref.rope(x, 2, 64, pos, [32], 1e4, w, 0.0)
    ref.within(o, want, bound)


def test_rope_agrees_with_rope_neox(vla, orc):
    x = _rows(_gen(4), 50, 15 * 64, F32)
    pos = np.arange(50, dtype=np.int32) + 3
    a = vla.rope_neox(x.numpy(), pos, 15, 64, 10000.0)
    o = torch.empty(50, 960, device=DEV)
    vla.qk_norm_rope_dev(o, None, x.to(DEV), None, 15, 0, 64, torch.from_numpy(pos)[None].to(DEV), [32], 10000.0)
    assert float((o.cpu() - torch.from_numpy(a)).abs().max()) <= 1e-6 * float(x.abs().max())


def test_rope_nan_stays_in_its_head(vla):
    x = _rows(_gen(5), 4, 3 * 32, F32)
    x[1, 32] = math.nan
    x[2, 70] = math.inf
    o = torch.empty(4, 96, device=DEV)
    vla.qk_norm_rope_dev(o, None, x.to(DEV), None, 3, 0, 32, _i32([[0, 1, 2, 3]]), [16], 1e4, torch.ones(32, device=DEV), None)
    fin = torch.isfinite(o.cpu()).reshape(4, 3, 32).all(-1)
    assert fin.tolist() == [[True] * 3, [True, False, True], [True, True, False], [True] * 3]


# ---------------------------------------------------------------- packed --

def _packed_case(g, qlens, klens, n_q, n_kv, hd, dtype, extra=2):
    """Host q, k, v with `extra` rows behind the last sequence."""
    return (_rows(g, sum(qlens) + extra, n_q * hd, dtype), _rows(g, sum(klens) + extra, n_kv * hd, dtype),
            _rows(g, sum(klens) + extra, n_kv * hd, dtype))


def _run_packed(vla, q, k, v, qlens, klens, n_q, n_kv, hd, scale, causal, pad=0, same=False):
    out = _dev(torch.full_like(q, 5.0), pad)
    vla.packed_attention_dev(out, _dev(q, pad), _dev(k, pad), _dev(v, pad), n_q, n_kv, hd, scale, _i32(_starts(qlens)),
                             None if same else _i32(_starts(klens)), causal=causal)
    torch.cuda.synchronize()
    return out


LENS = [[1], [1, 2, 31, 32, 33], [0, 64, 0, 65, 0], [127, 128, 129], [200, 1, 0, 7]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("n_q,n_kv,hd", [(4, 2, 64), (2, 1, 128)])
def test_packed_lengths(vla, dtype, causal, lens, n_q, n_kv, hd):
    g = _gen(sum(lens) * 7 + hd)
    q, k, v = _packed_case(g, lens, lens, n_q, n_kv, hd, dtype)
    got = _run_packed(vla, q, k, v, lens, lens, n_q, n_kv, hd, hd ** -0.5, causal, same=True)
    s = _starts(lens)
    want, bound = ref.packed(q, k, v, s, s, n_q, n_kv, hd, hd ** -0.5, causal, base=torch.full_like(q, 5.0))
    ref.within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,pad", [(1, 1, 8, 0), (3, 1, 40, 16), (15, 5, 64, 0), (2, 2, 72, 8), (5, 1, 80, 0), (4, 4, 96, 64),
                                             (2, 1, 136, 0), (1, 1, 192, 8), (8, 2, 256, 0), (16, 8, 32, 0)])
def test_packed_heads_and_strides(vla, dtype, n_q, n_kv, hd, pad):
    """k longer than q (a prompt behind cached tokens), shorter (queries that see nothing), and empty."""
    qlens, klens = [5, 40, 70, 3, 0], [133, 40, 11, 0, 9]
    g = _gen(n_q * 1000 + hd)
    q, k, v = _packed_case(g, qlens, klens, n_q, n_kv, hd, dtype)
    got = _run_packed(vla, q, k, v, qlens, klens, n_q, n_kv, hd, hd ** -0.5, True, pad)
    want, bound = ref.packed(q, k, v, _starts(qlens), _starts(klens), n_q, n_kv, hd, hd ** -0.5, True, base=torch.full_like(q, 5.0))
    ref.within(got, want, bound)
    assert bool((got[45:45 + 59] == 0).all()) and bool((got[115:118] == 0).all())  # 70 queries over 11 keys; 3 over none


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,n_q,n_kv,hd", [([700], 2, 1, 64), ([520, 1], 2, 2, 128), ([600], 1, 1, 40), ([300, 259], 28, 7, 64),
                                              ([290, 270], 28, 4, 128)])
def test_packed_keys_shared_by_waves(vla, dtype, causal, lens, n_q, n_kv, hd):
    """Few blocks over some keys: waves that share queries are joined, values taken out of the product
    come back in the queries that see them, whichever waves had their tile."""
    g = _gen(hd + n_q)
    q, k, v = _packed_case(g, lens, lens, n_q, n_kv, hd, dtype)
    args = (_starts(lens), _starts(lens), n_q, n_kv, hd, hd ** -0.5, causal)
    want, bound = ref.packed(q, k, v, *args, base=torch.full_like(q, 5.0))
    ref.within(_run_packed(vla, q, k, v, lens, lens, n_q, n_kv, hd, hd ** -0.5, causal, same=True), want, bound)
    if not causal:
        return
    at = (5, 69, lens[0] - 130, lens[0] - 2)
    for j, bad in zip(at, (math.inf, math.nan, -math.inf, math.nan)):
        v[j, 3] = bad
    got = _run_packed(vla, q, k, v, lens, lens, n_q, n_kv, hd, hd ** -0.5, causal, same=True).cpu()
    cols = [h * hd + 3 for h in range(n_q // n_kv)]  # of the first kv head's queries
    hit = torch.zeros(got.shape, dtype=torch.bool)
    hit[at[0]:lens[0], cols] = True
    ref.within(got[~hit], want[~hit], bound[~hit], "others")
    assert bool((got[at[0]:at[1], cols] == math.inf).all()) and bool(got[at[1]:lens[0], cols].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_many_sequences(vla, dtype):
    """More sequences than lanes in the tile search, and single queries over long keys."""
    for n, long in ((150, 0), (65, 130), (4200, 0)):
        lens = [(i * 7) % 5 if i % 40 else long for i in range(n)]
        g = _gen(9)
        q, k, v = _packed_case(g, lens, lens, 2, 1, 32, dtype)
        got = _run_packed(vla, q, k, v, lens, lens, 2, 1, 32, 0.125, True, same=True)
        s = _starts(lens)
        some = s if n < 1000 else s[:300]  # (the plain form is slow)
        want, bound = ref.packed(q, k, v, some, some, 2, 1, 32, 0.125, True, base=torch.full_like(q, 5.0))
        m = q.shape[0] if n < 1000 else some[-1]
        ref.within(got[:m], want[:m], bound[:m])
        if n > 1000:
            # The others: a query alone in its sequence has weight 1 and gives its own value; in fp32 that
            # value comes as three parts that hold it to u / 2, summed with two roundings of u = 2^-24.
            alone = [s[i] for i in range(300, n) if lens[i] == 1]
            want = v[alone].double().repeat(1, 2)
            ref.within(got[alone], want, want.abs() * (3 * 2.0 ** -24 if dtype is F32 else 0.0))
    qlens, klens = [1, 2], [900, 1025]
    q, k, v = _packed_case(g, qlens, klens, 2, 1, 64, dtype)
    got = _run_packed(vla, q, k, v, qlens, klens, 2, 1, 64, 0.125, True)
    want, bound = ref.packed(q, k, v, _starts(qlens), _starts(klens), 2, 1, 64, 0.125, True, base=torch.full_like(q, 5.0))
    ref.within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [4.0, -0.3, 0.0])
def test_packed_scales(vla, dtype, scale):
    """Sharp rows (one weight takes all), negated and uniform ones."""
    lens = [90, 3]
    q, k, v = _packed_case(_gen(11), lens, lens, 2, 2, 64, dtype)
    got = _run_packed(vla, q, k, v, lens, lens, 2, 2, 64, scale, True, same=True)
    s = _starts(lens)
    want, bound = ref.packed(q, k, v, s, s, 2, 2, 64, scale, True, base=torch.full_like(q, 5.0))
    ref.within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_packed_masked_values_add_nothing(vla, dtype, hd, bad):
    """Keys that no query sees, or only later queries see, may hold anything."""
    qlens, klens = [150, 20, 40], [150, 60, 7]
    g = _gen(13)
    q, k, v = _packed_case(g, qlens, klens, 2, 1, hd, dtype)
    for row in (100, 149, 150 + 45, 150 + 59, 217, 218):  # in and behind the sequences
        k[row, 3] = bad
        v[row, 5] = bad
    got = _run_packed(vla, q, k, v, qlens, klens, 2, 1, hd, hd ** -0.5, True)
    cq, ck, cv = q.clone(), k.clone(), v.clone()
    for row in (100, 149, 150 + 45, 150 + 59, 217, 218):
        ck[row, 3] = 0
        cv[row, 5] = 0
    want, bound = ref.packed(cq, ck, cv, _starts(qlens), _starts(klens), 2, 1, hd, hd ** -0.5, True, base=torch.full_like(q, 5.0))
    clean = torch.zeros(q.shape[0], dtype=torch.bool)
    clean[:100] = True
    clean[150:150 + 5] = True          # 20 queries over 60 keys: query i sees 41 + i
    clean[170:] = True                 # 40 queries over 7 keys, rows behind
    ref.within(got.cpu()[clean], want[clean], bound[clean], "unseen")
    # a value alone (its key finite) reaches every query that sees it, in its own dim and no other
    k2 = ck
    got = _run_packed(vla, q, k2, v, qlens, klens, 2, 1, hd, hd ** -0.5, True)
    g2 = got.cpu().double()
    for h in range(2):
        dim = h * hd + 5
        assert bool((~torch.isfinite(g2[100:150, dim])).all())
        rest = [h * hd + d for d in range(hd) if d != 5]
        ref.within(got.cpu()[:, rest], want[:, rest], bound[:, rest], "other dims")


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_infinite_scores(vla, dtype):
    """A key of -inf against a positive query has weight 0; one of +inf makes its queries NaN."""
    lens = [40]
    g = _gen(17)
    q = torch.rand(40, 64, generator=g).add(0.5).to(dtype)
    k, v = _rows(g, 40, 64, dtype), _rows(g, 40, 64, dtype)
    k[7] = -math.inf
    got = _run_packed(vla, q, k, v, lens, lens, 1, 1, 64, 0.125, True, same=True).cpu()
    keep = torch.tensor([i for i in range(40) if i != 7])
    for i in (6, 7, 8, 39):
        see = keep[keep <= i]
        w, b = ref.softmax_rows(q[i:i + 1].double(), k[see].double(), v[see].double(), torch.ones(1, len(see), dtype=torch.bool), 0.125,
                                0.0 if dtype == F32 else ref.half(dtype))
        ref.within(got[i:i + 1], w, b + ref.rounding(w, dtype))
    k[7] = math.inf
    got = _run_packed(vla, q, k, v, lens, lens, 1, 1, 64, 0.125, True, same=True).cpu()
    assert bool(torch.isfinite(got[:7]).all()) and bool(got[7:].isnan().all())
    k[7] = 1.0
    k[0] = math.nan  # a query that sees nothing else
    got = _run_packed(vla, q, k, v, lens, lens, 1, 1, 64, 0.125, True, same=True).cpu()
    assert bool(got.isnan().all())


def test_packed_offsets_are_clamped(vla):
    """Offsets beyond the buffers, and descending ones, stay inside them."""
    q, k, v = _packed_case(_gen(19), [40], [40], 1, 1, 64, BF16, extra=0)
    out = torch.full((40, 64), 5.0, dtype=BF16, device=DEV)
    vla.packed_attention_dev(out, q.to(DEV), k.to(DEV), v.to(DEV), 1, 1, 64, 0.125, _i32([0, 30, 20, 1000, -5]), causal=False)
    torch.cuda.synchronize()
    want, bound = ref.packed(q, k, v, [0, 30], [0, 30], 1, 1, 64, 0.125, False, base=torch.full_like(q, 5.0))
    ref.within(out[:20], want[:20], bound[:20])
    assert bool(torch.isfinite(out).all())


# ----------------------------------------------------------------- cache --

def _edge_rows(dtype, n_kv, hd, n):
    """Rows whose blocks sit on every edge of the format."""
    g = _gen(23)
    x = _rows(g, n, n_kv * hd, F32, 3.0)
    b = x.reshape(n, -1, 32)
    f = torch.finfo(dtype)
    b[0, 0] = 0.0
    b[0, -1] = -0.0
    if n > 8:
        b[1, 0] = torch.linspace(-7, 7, 32)          # amax = 7 * 2^0 exactly
        b[2, 0] = torch.arange(32) * 0.25            # ties
        b[3, 0] = torch.arange(32) * 0.25 - 7.75
        b[4, 0, :] = 2.0 ** -30
        b[5, 0, 0] = f.max
        b[6, 0] = f.smallest_normal * torch.arange(32) / 16
        b[7, 0, 3], b[7, -1, 4], b[8, 0, 31] = math.nan, math.inf, -math.inf
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,hd,page,pad", [(1, 32, 32, 0), (5, 64, 64, 16), (2, 96, 96, 0), (8, 128, 64, 0), (3, 192, 32, 8), (1, 256, 128, 0)])
def test_append_and_gather(vla, dtype, n_kv, hd, page, pad):
    new, past = [3, 0, 40, 1, 77], [0, 5, 30, 63, 20]
    lens = [a + b for a, b in zip(new, past)]
    need = [max(1, -(-n // page)) for n in lens]
    perm = torch.randperm(sum(need) + 2, generator=_gen(hd))
    table = np.full((5, max(need) + 1), -7, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n].numpy()
        at += n
    pages = sum(need) + 2
    host = ref.HostCache(vla, pages, n_kv, hd, page, fill=0xA5)
    k, v = _edge_rows(dtype, n_kv, hd, sum(new)), _edge_rows(dtype, n_kv, hd, sum(new)).flip(0).contiguous()
    s = _starts(new)
    for i in range(5):
        for j in range(new[i]):
            for part, x in ((0, k), (1, v)):
                host.write(table[i], past[i] + j, part, x[s[i] + j].reshape(n_kv, hd))
    cache = torch.full((pages, host.nb), 0xA5, dtype=torch.uint8, device=DEV)
    extra = torch.full((2, n_kv * hd), 9.0, dtype=dtype)  # rows behind the last sequence
    vla.kv4_append_dev(cache, _dev(torch.cat([k, extra]), pad), _dev(torch.cat([v, extra]), pad), n_kv, hd, page, torch.from_numpy(table).to(DEV),
                       _i32(lens), _i32(s))
    torch.cuda.synchronize()
    assert np.array_equal(cache.cpu().numpy().reshape(-1), host.mem)
    ko, vo = (_dev(torch.full((sum(new) + 2, n_kv * hd), 5.0, dtype=dtype), pad) for _ in range(2))
    vla.kv4_gather_dev(ko, vo, cache, n_kv, hd, page, torch.from_numpy(table).to(DEV), _i32(s), _i32(past))
    for got, x in ((ko, k), (vo, v)):
        want = ref.values(*ref.quantize(x.reshape(-1, n_kv, hd))).reshape(x.shape)
        got = got.cpu()
        assert bool((got[-2:] == 5.0).all())
        w = want.to(dtype)
        assert bool(((got[:-2] == w) | (got[:-2].isnan() & w.isnan())).all())


@pytest.mark.parametrize("n_seqs", [1, 70, 1500])
def test_append_sequence_search(vla, n_seqs):
    """Starts in LDS and, above 1023 sequences, in global memory; empty sequences among them."""
    new = [(i * 5) % 3 for i in range(n_seqs)] if n_seqs > 1 else [4]
    pages = n_seqs
    table = torch.randperm(pages, generator=_gen(1)).to(torch.int32)[:, None].contiguous()
    x = _rows(_gen(2), sum(new), 32, F32)
    cache = torch.zeros(pages, vla.kv4_page_bytes(1, 32, 32), dtype=torch.uint8, device=DEV)
    s = _i32(_starts(new))
    vla.kv4_append_dev(cache, x.to(DEV), -x.to(DEV), 1, 32, 32, table.to(DEV), _i32(new), s)
    ko, vo = torch.empty_like(x, device=DEV), torch.empty_like(x, device=DEV)
    vla.kv4_gather_dev(ko, vo, cache, 1, 32, 32, table.to(DEV), s)
    want = ref.values(*ref.quantize(x[:, None])).reshape(x.shape).float()
    assert torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), -want)


def test_cache_bad_pages(vla):
    """Rows without a page are dropped by append and read as NaN by gather; nothing else changes."""
    page, nb = 32, vla.kv4_page_bytes(2, 64, 32)
    table = torch.tensor([[1, -1, 9], [3, 2, 2 ** 31 - 1]], dtype=torch.int32)
    cache = torch.full((4, nb), 0x11, dtype=torch.uint8, device=DEV)
    new, lens = [100, 10], [100, 70]
    x = _rows(_gen(3), 110, 128, BF16)
    vla.kv4_append_dev(cache, x.to(DEV), x.to(DEV), 2, 64, page, table.to(DEV), _i32(lens), _i32(_starts(new)))
    assert bool((cache[0] == 0x11).all()) and bool((cache[3] == 0x11).all())
    ko, vo = torch.zeros_like(x, device=DEV), torch.zeros_like(x, device=DEV)
    vla.kv4_gather_dev(ko, vo, cache, 2, 64, page, table.to(DEV), _i32(_starts(new)), _i32([0, 60]))
    want = ref.values(*ref.quantize(x.reshape(-1, 2, 64))).reshape(x.shape).to(BF16)
    ok = torch.tensor([i < 32 for i in range(100)] + [60 + i < 64 for i in range(10)])
    assert torch.equal(ko.cpu()[ok], want[ok]) and torch.equal(vo.cpu()[ok], want[ok])
    assert bool(ko.cpu()[~ok].isnan().all())
    # lengths shorter than the new rows: the first rows have no token
    cache.fill_(0)
    vla.kv4_append_dev(cache, x[:10].to(DEV), x[:10].to(DEV), 2, 64, page, table[1:].contiguous().to(DEV), _i32([4]), _i32([0, 10]))
    ko = torch.zeros(4, 128, dtype=BF16, device=DEV)
    vla.kv4_gather_dev(ko, torch.empty_like(ko), cache, 2, 64, page, table[1:].contiguous().to(DEV), _i32([0, 4]))
    assert torch.equal(ko.cpu(), want[6:10])


# ---------------------------------------------------------------- decode --

def _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=1, vstd=1.0):
    """(q, cache, table, host cache): a filled cache; what lies behind each sequence's end is garbage."""
    g = _gen(seed)
    need = [max(1, -(-n // page)) for n in lens]
    pages = sum(need) + 1
    perm = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n].to(torch.int32)
        at += n
    total = sum(lens)
    k, v = _rows(g, total, n_kv * hd, F32), _rows(g, total, n_kv * hd, F32, vstd)
    cache = torch.full((pages, vla.kv4_page_bytes(n_kv, hd, page)), 0xFF, dtype=torch.uint8, device=DEV)
    vla.kv4_append_dev(cache, k.to(DEV), v.to(DEV), n_kv, hd, page, table.to(DEV), _i32(lens), _i32(_starts(lens)))
    kq, vq = (ref.values(*ref.quantize(x.reshape(total, n_kv, hd))) for x in (k, v))
    s = _starts(lens)
    ks, vs = ([x[s[i]:s[i + 1]] for i in range(len(lens))] for x in (kq, vq))
    return _rows(g, sum(new), n_q * hd, dtype), cache, table.to(DEV), ks, vs


def _run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, page, scale, split, max_len=None, pad=0, max_new=None):
    out = _dev(torch.full((q.shape[0] + 2, q.shape[1]), 5.0, dtype=q.dtype), pad)
    qd = _dev(torch.cat([q, torch.full((2, q.shape[1]), math.nan, dtype=q.dtype)]), pad)
    m, mx = max_len or max(lens), max_new or max(new)
    work = None
    if split:
        n = vla.kv4_attention_work_bytes(qd.shape[0], len(lens), mx, m, n_q, n_kv, hd)
        work = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=DEV)
    vla.kv4_attention_dev(out, qd, cache, n_q, n_kv, hd, page, scale, table, _i32(lens), _i32(_starts(new)), mx, m, work)
    torch.cuda.synchronize()
    assert bool((out[-2:] == 5.0).all())
    return out[:-2]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(1, 1, 32, 32), (15, 5, 64, 64), (6, 2, 96, 96), (32, 8, 128, 64), (4, 2, 192, 32), (3, 1, 256, 128),
                                              (20, 1, 64, 32), (16, 1, 128, 64), (34, 2, 64, 64)])
def test_decode_single_tokens(vla, dtype, n_q, n_kv, hd, page):
    lens = [1, 31, 32, 33, 0, 64, 200, 129]
    new = [1] * 8
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=hd + n_q)
    want, bound = ref.decode(q, ks, vs, new, n_q, n_kv, hd, hd ** -0.5)
    got = _run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, page, hd ** -0.5, True)
    ref.within(got, want, bound)
    # without offsets: row s is sequence s's
    out = torch.empty_like(q, device=DEV)
    work = torch.empty(max(16, vla.kv4_attention_work_bytes(8, 8, 1, 200, n_q, n_kv, hd)), dtype=torch.uint8, device=DEV)
    vla.kv4_attention_dev(out, q.to(DEV), cache, n_q, n_kv, hd, page, hd ** -0.5, table, _i32(lens), max_len=200, work=work)
    assert torch.equal(out, got)
    out.fill_(5.0)
    vla.kv4_attention_dev(out, q.to(DEV), cache, n_q, n_kv, hd, page, hd ** -0.5, table, _i32(lens))
    ref.within(out, want, bound, "a block per sequence")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[2, 1, 5], [17, 33, 16], [50, 0, 3]])
@pytest.mark.parametrize("n_q,n_kv,hd", [(15, 5, 64), (8, 1, 128), (4, 4, 96), (40, 2, 32)])
def test_decode_chunks(vla, dtype, new, n_q, n_kv, hd):
    """Several new tokens, causal at the end; one sequence has fewer tokens than queries."""
    lens = [227, 33, 2]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, 64, dtype, seed=hd)
    want, bound = ref.decode(q, ks, vs, new, n_q, n_kv, hd, hd ** -0.5)
    ref.within(_run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, 64, hd ** -0.5, True), want, bound)
    # a max_new that is too small costs time only; rows between others
    ref.within(_run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, 64, hd ** -0.5, False, pad=8, max_new=1), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[3000, 5, 257, 1024], [4097]])
@pytest.mark.parametrize("hd,page", [(64, 96), (128, 256)])
def test_decode_split_keys(vla, dtype, lens, hd, page):
    """The key axis split over blocks: the joined result, the unsplit one and the plain one."""
    new = [1] * len(lens)
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, hd, page, dtype, seed=7)
    assert vla.kv4_attention_work_bytes(len(lens), len(lens), 1, max(lens), 4, 2, hd) > 0
    want, bound = ref.decode(q, ks, vs, new, 4, 2, hd, hd ** -0.5)
    ref.within(_run_decode(vla, q, cache, table, lens, new, 4, 2, hd, page, hd ** -0.5, True), want, bound, "split")
    ref.within(_run_decode(vla, q, cache, table, lens, new, 4, 2, hd, page, hd ** -0.5, False), want, bound, "unsplit")
    # bounds on the length that are too low or high change the launch, not the result
    for m in (64, 100000):
        ref.within(_run_decode(vla, q, cache, table, lens, new, 4, 2, hd, page, hd ** -0.5, True, max_len=m), want, bound, f"max_len {m}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [3.0, -0.2, 0.0])
def test_decode_scales(vla, dtype, scale):
    lens, new = [100, 7], [1, 4]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, 64, 32, dtype, seed=3)
    want, bound = ref.decode(q, ks, vs, new, 2, 1, 64, scale)
    ref.within(_run_decode(vla, q, cache, table, lens, new, 2, 1, 64, 32, scale, True), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_decode_not_finite(vla, dtype, hd):
    """A token with a NaN is seen by the queries that see it and by no others; garbage behind the end by none."""
    lens, new, page = [70, 40], [9, 1], 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, hd, page, dtype, seed=5)
    want, bound = ref.decode(q, ks, vs, new, 4, 2, hd, hd ** -0.5)
    row = table.cpu().numpy()[0]
    flat = cache.view(-1)
    for part in (2, 3):
        c = cache.clone()
        # token 65 of 70 (queries 4..8 of 9 see it), kv head 1, the last block
        c.view(-1)[vla.kv4_offset(row, 2, hd, page, cache.shape[0], 65, part, 1, hd // 32 - 1)] = 255
        got = _run_decode(vla, q, c, table, lens, new, 4, 2, hd, page, hd ** -0.5, True).cpu()
        ref.within(got[:4], want[:4], bound[:4], "before")
        ref.within(got[4:, :2 * hd], want[4:, :2 * hd], bound[4:, :2 * hd], "other kv head")
        ref.within(got[9:], want[9:], bound[9:], "other sequence")
        tail = got[4:9, 2 * hd:].reshape(5, 2, hd)
        assert bool(tail[:, :, hd - 32:].isnan().all())
        if part == 3:
            w, b = (x[4:9, 2 * hd:].reshape(5, 2, hd)[:, :, :hd - 32] for x in (want, bound))
            ref.within(tail[:, :, :hd - 32], w, b, "other blocks")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_new", [33, 4])
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(15, 5, 64, 64), (8, 1, 128, 32), (40, 2, 32, 96), (2, 2, 256, 64), (4, 2, 192, 128)])
def test_decode_chunks_in_runs(vla, dtype, max_new, n_q, n_kv, hd, page):
    """Chunks, empty sequences and queries without a key where runs of tiles cut the sequences anywhere;
    chunks past max_new are not cut."""
    lens, new = [227, 33, 2, 0, 1100, 0, 64], [17, 33, 5, 0, 1, 3, 4]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=hd + 3)
    assert vla.kv4_attention_work_bytes(sum(new) + 2, 7, max_new, 1 << 20, n_q, n_kv, hd) > 0
    want, bound = ref.decode(q, ks, vs, new, n_q, n_kv, hd, hd ** -0.5)
    for m in (1500, 4096, 1 << 20):
        got = _run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, page, hd ** -0.5, True, max_len=m, max_new=max_new)
        ref.within(got, want, bound, f"max_len {m}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [32, 96, 256])
def test_decode_not_finite_in_runs(vla, dtype, hd):
    """The same as without runs: a NaN reaches the queries that see it, whatever block takes its tile."""
    lens, new, page = [70, 40], [9, 1], 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, hd, page, dtype, seed=5)
    want, bound = ref.decode(q, ks, vs, new, 4, 2, hd, hd ** -0.5)
    row = table.cpu().numpy()[0]
    for part in (2, 3):
        c = cache.clone()
        c.view(-1)[vla.kv4_offset(row, 2, hd, page, cache.shape[0], 65, part, 1, hd // 32 - 1)] = 255
        got = _run_decode(vla, q, c, table, lens, new, 4, 2, hd, page, hd ** -0.5, True, max_len=4096).cpu()
        ref.within(got[:4], want[:4], bound[:4], "before")
        ref.within(got[4:, :2 * hd], want[4:, :2 * hd], bound[4:, :2 * hd], "other kv head")
        ref.within(got[9:], want[9:], bound[9:], "other sequence")
        tail = got[4:9, 2 * hd:].reshape(5, 2, hd)
        assert bool(tail[:, :, hd - 32:].isnan().all())
        if part == 3 and hd > 32:
            w, b = (x[4:9, 2 * hd:].reshape(5, 2, hd)[:, :, :hd - 32] for x in (want, bound))
            ref.within(tail[:, :, :hd - 32], w, b, "other blocks")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_packed_without_keys(vla, dtype, hd):
    """No key rows at all, and no sequences: zeros, and nothing written."""
    q = torch.ones(5, 2 * hd, dtype=dtype, device=DEV)
    none = torch.empty(0, hd, dtype=dtype, device=DEV)
    out = torch.full_like(q, 5.0)
    vla.packed_attention_dev(out, q, none, none, 2, 1, hd, 0.1, _i32([0, 3, 4]), _i32([0, 0, 0]))
    assert bool((out[:4] == 0).all()) and bool((out[4] == 5.0).all())
    out.fill_(5.0)
    vla.packed_attention_dev(out, q, none, none, 2, 1, hd, 0.1, _i32([0]))
    vla.packed_attention_dev(none.new_empty(0, 2 * hd), none.new_empty(0, 2 * hd), none, none, 2, 1, hd, 0.1, _i32([0, 0]))
    assert bool((out == 5.0).all())


def test_decode_workspaces_and_rows(vla):
    """A workspace that is too small or not aligned runs unsplit; without offsets, rows behind the sequences stay."""
    lens = [3000, 70, 512]
    q, cache, table, ks, vs = _decode_case(vla, lens, [1] * 3, 4, 2, 64, 64, BF16, seed=19)
    want, bound = ref.decode(q, ks, vs, [1] * 3, 4, 2, 64, 0.125)
    qd = torch.cat([q, q]).to(DEV)
    nb = vla.kv4_attention_work_bytes(6, 3, 1, 3000, 4, 2, 64)
    assert nb > 0
    buf = torch.full((nb + 64,), 0xFF, dtype=torch.uint8, device=DEV)
    for work in (buf, buf[:nb], buf[:nb - 1], buf[8:], buf[:0], None):
        out = torch.full_like(qd, 5.0)
        vla.kv4_attention_dev(out, qd, cache, 4, 2, 64, 64, 0.125, table, _i32(lens), max_len=3000, work=work)
        ref.within(out[:3], want, bound)
        assert bool((out[3:] == 5.0).all())
    assert bool((buf[nb:] == 0xFF).all())


def test_decode_many_sequences(vla):
    """As many sequences as one call takes, all reading the same page."""
    n = 65535
    q, cache, _, ks, vs = _decode_case(vla, [20], [1], 1, 1, 32, 32, BF16, seed=4)
    table = torch.zeros(n, 1, dtype=torch.int32, device=DEV)
    table[:] = int((cache[:, 0] != 0xFF).nonzero()[0])
    lens = torch.arange(n, dtype=torch.int32, device=DEV) % 21
    qd = q.to(DEV).repeat(n, 1)
    out = torch.empty_like(qd)
    for max_len in (32, 2048):
        work = torch.full((max(16, vla.kv4_attention_work_bytes(n, n, 1, max_len, 1, 1, 32)),), 0xFF, dtype=torch.uint8, device=DEV)
        out.fill_(5.0)
        vla.kv4_attention_dev(out, qd, cache, 1, 1, 32, 32, 0.2, table, lens, max_len=max_len, work=work)
        for m in range(21):
            rows = out[m::21].cpu()
            want, bound = ref.decode(q, [ks[0][:m]], [vs[0][:m]], [1], 1, 1, 32, 0.2)
            ref.within(rows, want.expand_as(rows), bound.expand_as(rows), f"{m} keys")


def test_shared_pages(vla):
    """Two sequences with the same first pages: each appends to pages of its own and reads both."""
    n_kv, hd, page, dtype = 2, 64, 32, BF16
    g = _gen(81)
    k, v = _rows(g, 64 + 20, n_kv * hd, dtype), _rows(g, 64 + 20, n_kv * hd, dtype)
    cache = torch.full((5, vla.kv4_page_bytes(n_kv, hd, page)), 0xFF, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[3, 1, 0], [3, 1, 4]], dtype=torch.int32, device=DEV)
    vla.kv4_append_dev(cache, k[:64].to(DEV), v[:64].to(DEV), n_kv, hd, page, table[:1].contiguous(), _i32([64]), _i32([0, 64]))
    vla.kv4_append_dev(cache, k[64:].to(DEV), v[64:].to(DEV), n_kv, hd, page, table, _i32([76, 72]), _i32([0, 12, 20]))
    own = [torch.cat([torch.arange(64), torch.arange(a, b)]) for a, b in ((64, 76), (76, 84))]
    ks, vs = ([ref.values(*ref.quantize(x[i].reshape(-1, n_kv, hd))) for i in own] for x in (k, v))
    q = _rows(g, 5, 4 * hd, dtype)
    want, bound = ref.decode(q, ks, vs, [2, 3], 4, n_kv, hd, 0.125)
    for m in (76, 2048):
        ref.within(_run_decode(vla, q, cache, table, [76, 72], [2, 3], 4, n_kv, hd, page, 0.125, True, max_len=m), want, bound)


def test_two_streams_at_once(vla):
    """The same operators on two streams, each with its own workspace, against one after the other."""
    n_q, n_kv, hd, page = 8, 2, 64, 32
    jobs = []
    for i, lens in enumerate(([3000, 40, 900], [77, 2500, 1])):
        q, cache, table, _, _ = _decode_case(vla, lens, [1] * 3, n_q, n_kv, hd, page, BF16, seed=90 + i)
        x = _rows(_gen(i), 700, n_q * hd, BF16).to(DEV)
        work = torch.empty(vla.kv4_attention_work_bytes(3, 3, 1, 4096, n_q, n_kv, hd), dtype=torch.uint8, device=DEV)
        jobs.append((q.to(DEV), cache, table, _i32(lens), x, x[:, :n_kv * hd].contiguous(), _i32([0, 300 + i, 700]), work))

    def run(job):
        q, cache, table, lens, x, kv, start, work = job
        o, p, r = torch.empty_like(q), torch.empty_like(x), torch.empty_like(x)
        pos = torch.arange(700, dtype=torch.int32, device=DEV)[None]
        for _ in range(5):
            vla.kv4_attention_dev(o, q, cache, n_q, n_kv, hd, page, 0.125, table, lens, max_len=4096, work=work)
            vla.qk_norm_rope_dev(r, None, x, None, n_q, 0, hd, pos, [32], 1e4)
            vla.packed_attention_dev(p, r, kv, kv, n_q, n_kv, hd, 0.125, start)
        return o, p, r

    alone = [run(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    both = []
    for st, j in zip(streams, jobs):
        with torch.cuda.stream(st):
            both.append(run(j))
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_decode_bad_pages(vla):
    """A sequence whose table names no page where it needs one reads NaN, the others are untouched."""
    lens, new = [70, 40, 70], [1, 1, 1]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, 64, 32, BF16, seed=5)
    want, bound = ref.decode(q, ks, vs, new, 4, 2, 64, 0.125)
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0, 1] = bad
        got = _run_decode(vla, q, cache, t, lens, new, 4, 2, 64, 32, 0.125, True).cpu()
        assert bool(got[0].isnan().all())
        ref.within(got[1:], want[1:], bound[1:])
    # a length beyond the table's pages names tokens without a page
    room = table.shape[1] * 32
    for n in (room + 1, room + 32, room + 500, 2 ** 31 - 1):
        for split in (True, False):
            got = _run_decode(vla, q, cache, table, [n, 40, 70], new, 4, 2, 64, 32, 0.125, split).cpu()
            assert bool(got[0].isnan().all()), n
            ref.within(got[1:], want[1:], bound[1:])


def test_decode_chunk_across_the_tables_end(vla):
    """Of a chunk of new tokens, those that the table has room for are right, the others NaN."""
    lens, new = [96], [40]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, 64, 32, BF16, seed=15)
    want, bound = ref.decode(q, ks, vs, new, 4, 2, 64, 0.125)
    q2 = torch.cat([q[10:], q[:10]])  # rows 0..29 stand where rows 10..39 of the whole chunk stood
    got = _run_decode(vla, q2, cache, table, [96 + 10], new, 4, 2, 64, 32, 0.125, True).cpu()
    ref.within(got[:30], want[10:], bound[10:])
    assert bool(got[30:].isnan().all())


def test_decode_long_cache(vla):
    """Pages beyond 4 GiB of the cache are reached."""
    n_kv, hd, page = 8, 128, 256
    nb = vla.kv4_page_bytes(n_kv, hd, page)
    pages = (1 << 32) // nb + 40
    cache = torch.zeros(pages, nb, dtype=torch.uint8, device=DEV)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device=DEV)
    g = _gen(8)
    k, v, q = _rows(g, 700, n_kv * hd, BF16), _rows(g, 700, n_kv * hd, BF16), _rows(g, 1, 16 * hd, BF16)
    vla.kv4_append_dev(cache, k.to(DEV), v.to(DEV), n_kv, hd, page, table, _i32([700]), _i32([0, 700]))
    ks, vs = ([ref.values(*ref.quantize(x.reshape(700, n_kv, hd)))] for x in (k, v))
    want, bound = ref.decode(q, ks, vs, [1], 16, n_kv, hd, hd ** -0.5)
    ref.within(_run_decode(vla, q, cache, table, [700], [1], 16, n_kv, hd, page, hd ** -0.5, True), want, bound)


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 64), (F32, 256)])
def test_rows_far_apart(vla, dtype, hd):
    """Rows of one buffer whose offsets pass 32 bits, through every operator that takes rows."""
    T, ld = 1100, (1 << 22) // (2 if dtype is F32 else 1)
    if dtype is BF16:
        ld //= 2
    buf = torch.empty(T, ld, dtype=dtype, device=DEV)
    assert buf.numel() * buf.element_size() > 1 << 32
    g = _gen(12)
    x = [_rows(g, T, n * hd, dtype) for n in (2, 1, 1)]
    q, k, v, out, kb, vb = (buf[:, at * hd:(at + n) * hd] for at, n in ((0, 2), (2, 1), (3, 1), (4, 2), (6, 1), (7, 1)))
    for d, s in zip((q, k, v), x):
        d.copy_(s)
    lens = [1000, 100]
    s = _starts(lens)
    vla.packed_attention_dev(out, q, k, v, 2, 1, hd, 0.125, _i32(s))
    want, bound = ref.packed(*x, s, s, 2, 1, hd, 0.125, True)
    ref.within(out, want, bound, "attention")
    pos = torch.arange(T, dtype=torch.int32)[None]
    vla.qk_norm_rope_dev(q, k, q, k, 2, 1, hd, pos.to(DEV), [hd // 2], 1e4)
    for got, y, n in ((q, x[0], 2), (k, x[1], 1)):
        want, bound = ref.rope(y, n, hd, pos, [hd // 2], 1e4, None, 0.0)
        ref.within(got, want, bound, "rotation")
    cache = torch.zeros(35, vla.kv4_page_bytes(1, hd, 32), dtype=torch.uint8, device=DEV)
    table = torch.arange(35, dtype=torch.int32, device=DEV)[None].contiguous()
    vla.kv4_append_dev(cache, v, v, 1, hd, 32, table, _i32([T]), _i32([0, T]))
    vla.kv4_gather_dev(kb, vb, cache, 1, hd, 32, table, _i32([0, T]))
    want = ref.values(*ref.quantize(x[2].reshape(T, 1, hd))).reshape(T, hd).to(dtype)
    assert torch.equal(kb.cpu(), want) and torch.equal(vb.cpu(), want)
    vla.kv4_attention_dev(out[:1], q[:1], cache, 2, 1, hd, 32, 0.125, table, _i32([T]))
    vla.kv4_attention_dev(out[-2:-1], q[:1], cache, 2, 1, hd, 32, 0.125, table, _i32([T]))
    assert torch.equal(out[:1], out[-2:-1])


# --------------------------------------------------------- run together --

def _decoder_pass(vla, bufs, steps):
    """A prompt pass and `steps` token passes of one attention layer; returns their outputs."""
    b = bufs
    out = []
    vla.qk_norm_rope_dev(b["q"], b["k"], b["q0"], b["k0"], b["n_q"], b["n_kv"], b["hd"], b["pos"], b["sections"], 1e4, b["wq"], b["wk"])
    o = torch.empty_like(b["q"])
    vla.packed_attention_dev(o, b["q"], b["k"], b["v0"], b["n_q"], b["n_kv"], b["hd"], b["scale"], b["start"])
    vla.kv4_append_dev(b["cache"], b["k"], b["v0"], b["n_kv"], b["hd"], b["page"], b["table"], b["lens"][0], b["start"])
    out.append(o)
    for i in range(steps):
        q, k, v = b["tokens"][i]
        vla.qk_norm_rope_dev(q, k, q, k, b["n_q"], b["n_kv"], b["hd"], b["tpos"][i], b["sections"], 1e4, b["wq"], b["wk"])
        vla.kv4_append_dev(b["cache"], k, v, b["n_kv"], b["hd"], b["page"], b["table"], b["lens"][i + 1], b["one"])
        o = torch.empty_like(q)
        vla.kv4_attention_dev(o, q, b["cache"], b["n_q"], b["n_kv"], b["hd"], b["page"], b["scale"], b["table"], b["lens"][i + 1],
                              max_len=b["max_len"], work=b["work"])
        out.append(o)
    return out


@pytest.mark.parametrize("dtype", TYPES)
def test_decoder_run(vla, dtype):
    """Rotation, prompt attention, cache and decoding as a decoder runs them, each step against the plain
    form of what the step before really left."""
    n_q, n_kv, hd, page, steps = 15, 5, 64, 32, 3
    plens = [30, 1, 65]
    sections = [8, 12, 12]
    g = _gen(31)
    T = sum(plens)
    start = _starts(plens)
    b = dict(n_q=n_q, n_kv=n_kv, hd=hd, page=page, sections=sections, scale=hd ** -0.5, max_len=128)
    host = {n: _rows(g, T, w * hd, dtype) for n, w in (("q0", n_q), ("k0", n_kv), ("v0", n_kv))}
    b.update({n: t.to(DEV) for n, t in host.items()})
    b["q"], b["k"] = torch.empty_like(b["q0"]), torch.empty_like(b["k0"])
    wq, wk = (1 + 0.1 * torch.randn(hd, generator=g) for _ in range(2))
    b["wq"], b["wk"] = wq.to(DEV), wk.to(DEV)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in plens])[None].repeat(3, 1)
    pos[1:] = pos[1:] // 2
    b["pos"], b["start"], b["one"] = pos.to(DEV), _i32(start), _i32([0, 1, 2, 3])
    b["lens"] = [_i32([n + i for n in plens]) for i in range(steps + 1)]
    toks = [tuple(_rows(g, 3, w * hd, dtype) for w in (n_q, n_kv, n_kv)) for _ in range(steps)]
    b["tokens"] = [tuple(t.to(DEV) for t in x) for x in toks]
    tpos = [torch.tensor([[n + i for n in plens]] * 3, dtype=torch.int32) for i in range(steps)]
    b["tpos"] = [t.to(DEV) for t in tpos]
    b["table"] = torch.randperm(12, generator=g).to(torch.int32).reshape(3, 4).to(DEV)
    b["cache"] = torch.full((12, vla.kv4_page_bytes(n_kv, hd, page)), 0xEE, dtype=torch.uint8, device=DEV)
    b["work"] = None
    outs = _decoder_pass(vla, b, steps)
    torch.cuda.synchronize()
    want, bound = ref.rope(host["q0"], n_q, hd, pos, sections, 1e4, wq, 1e-6)
    ref.within(b["q"], want, bound, "q")
    want, bound = ref.rope(host["k0"], n_kv, hd, pos, sections, 1e4, wk, 1e-6)
    ref.within(b["k"], want, bound, "k")
    q, k = b["q"].cpu(), b["k"].cpu()
    want, bound = ref.packed(q, k, host["v0"], start, start, n_q, n_kv, hd, b["scale"], True)
    ref.within(outs[0], want, bound, "prompt")
    quant = lambda x: ref.values(*ref.quantize(x.reshape(-1, n_kv, hd)))
    ks = [quant(k[start[s]:start[s + 1]]) for s in range(3)]
    vs = [quant(host["v0"][start[s]:start[s + 1]]) for s in range(3)]
    for i in range(steps):
        tq, tk = (x.cpu() for x in b["tokens"][i][:2])
        want, bound = ref.rope(toks[i][0], n_q, hd, tpos[i], sections, 1e4, wq, 1e-6)
        ref.within(tq, want, bound, f"q of step {i}")
        for s in range(3):
            ks[s] = torch.cat([ks[s], quant(tk[s:s + 1])])
            vs[s] = torch.cat([vs[s], quant(toks[i][2][s:s + 1])])
        want, bound = ref.decode(tq, ks, vs, [1, 1, 1], n_q, n_kv, hd, b["scale"])
        ref.within(outs[i + 1], want, bound, f"step {i}")


def test_prompt_behind_a_cached_beginning(vla):
    """A prompt's second half attends to its cached first half, read back as rows, through the packed attention."""
    n_q, n_kv, hd, page = 4, 2, 128, 64
    first, second = [70, 0, 33], [40, 20, 1]
    g = _gen(41)
    q, cache, table, ks, vs = _decode_case(vla, [a + b for a, b in zip(first, second)], second, n_q, n_kv, hd, page, BF16, seed=41)
    klens = [a + b for a, b in zip(first, second)]
    K, V = (torch.empty(sum(klens), n_kv * hd, dtype=BF16, device=DEV) for _ in range(2))
    vla.kv4_gather_dev(K, V, cache, n_kv, hd, page, table, _i32(_starts(klens)))
    out = torch.empty_like(q, device=DEV)
    vla.packed_attention_dev(out, q.to(DEV), K, V, n_q, n_kv, hd, hd ** -0.5, _i32(_starts(second)), _i32(_starts(klens)))
    want, bound = ref.packed(q, K.cpu(), V.cpu(), _starts(second), _starts(klens), n_q, n_kv, hd, hd ** -0.5, True)
    ref.within(out, want, bound)
    # the cached values are exact in bf16, so the attention over the cache is held to the same values
    got = _run_decode(vla, q, cache, table, klens, second, n_q, n_kv, hd, page, hd ** -0.5, True)
    want, bound = ref.decode(q, ks, vs, second, n_q, n_kv, hd, hd ** -0.5)
    ref.within(got, want, bound)


def test_streams_and_graphs(vla):
    """A decode step captured on a stream of its own: replays follow new inputs, lengths and pages; a second
    graph that shares the workspace and eager work run between them."""
    n_q, n_kv, hd, page = 8, 2, 64, 32
    lens = [1500, 40]
    q, cache, table, _, _ = _decode_case(vla, lens, [1, 1], n_q, n_kv, hd, page, BF16, seed=51)
    dl, qd = _i32(lens), q.to(DEV)
    kd, vd = (_rows(_gen(i), 2, n_kv * hd, BF16).to(DEV) for i in (1, 2))
    pos, one = _i32([[1499, 39]]), _i32([0, 1, 2])
    nb = vla.kv4_attention_work_bytes(2, 2, 1, 2048, n_q, n_kv, hd)
    assert nb > 0
    work = torch.empty(nb, dtype=torch.uint8, device=DEV)
    qr, kr = torch.empty_like(qd), torch.empty_like(kd)
    outs = [torch.empty_like(qd) for _ in range(2)]
    po = torch.empty_like(qd)

    def step(out):
        vla.qk_norm_rope_dev(qr, kr, qd, kd, n_q, n_kv, hd, pos, [32], 1e4)
        vla.kv4_append_dev(cache, kr, vd, n_kv, hd, page, table, dl, one)
        vla.kv4_attention_dev(out, qr, cache, n_q, n_kv, hd, page, 0.125, table, dl, max_len=2048, work=work)
        vla.packed_attention_dev(po, qr, kr, vd, n_q, n_kv, hd, 0.125, one)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(outs[0])
    st.synchronize()
    graphs = []
    for o in outs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            step(o)
        graphs.append(gr)
    for i in range(4):
        qd.copy_(_rows(_gen(60 + i), 2, n_q * hd, BF16))
        kd.copy_(_rows(_gen(70 + i), 2, n_kv * hd, BF16))
        dl.copy_(torch.tensor([1400 + i, 40 + i], dtype=torch.int32))
        before = cache.clone()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got, pgot, after = outs[i % 2].clone(), po.clone(), cache.clone()
        cache.copy_(before)
        eager = torch.empty_like(qd)
        step(eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(pgot, po) and torch.equal(after, cache), i


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (F32, 128), (F32, 256), (BF16, 128), (F16, 256)])
def test_prompt_graph(vla, dtype, hd):
    """A captured prompt pass: replays follow other lengths in the same buffers."""
    g = _gen(hd)
    q, k, v = (t.to(DEV) for t in _packed_case(g, [150, 40], [150, 40], 2, 1, hd, dtype, extra=0))
    start, out = _i32([0, 150, 190]), torch.zeros_like(q)
    call = lambda o: vla.packed_attention_dev(o, q, k, v, 2, 1, hd, 0.1, start)
    call(out)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        call(out)
    for cut in (1, 100, 190, 0):
        start[1] = cut
        v.copy_(v.flip(0))
        out.zero_()
        gr.replay()
        eager = torch.zeros_like(out)
        call(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager), cut


def test_repeated_calls_give_the_same_bits(vla):
    """No result depends on the order in which blocks run."""
    lens = [700, 3, 129]
    q, k, v = _packed_case(_gen(61), lens, lens, 4, 2, 128, BF16)
    a = _run_packed(vla, q, k, v, lens, lens, 4, 2, 128, 0.1, True, same=True)
    dq, cache, table, _, _ = _decode_case(vla, lens, [1, 1, 1], 4, 2, 64, 64, F32, seed=62)
    b = _run_decode(vla, dq, cache, table, lens, [1, 1, 1], 4, 2, 64, 64, 0.125, True)
    for _ in range(3):
        assert torch.equal(a, _run_packed(vla, q, k, v, lens, lens, 4, 2, 128, 0.1, True, same=True))
        assert torch.equal(b, _run_decode(vla, dq, cache, table, lens, [1, 1, 1], 4, 2, 64, 64, 0.125, True))


@pytest.mark.parametrize("max_len", [64, 4096])
def test_decode_without_a_bound_on_the_new_tokens(vla, max_len):
    """2^31 - 1 where the caller knows no bound."""
    lens, new = [70, 1500, 33], [3, 1, 20]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 32, 8, 64, 64, BF16, seed=33)
    want, bound = ref.decode(q, ks, vs, new, 32, 8, 64, 0.125)
    for split in (True, False):
        got = _run_decode(vla, q, cache, table, lens, new, 32, 8, 64, 64, 0.125, split, max_len=max_len, max_new=2 ** 31 - 1)
        ref.within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,n_q,hd", [(8192, 2, 64), (40000, 1, 128), (2048, 320, 32), (4096, 1, 256), (4096, 1, 192)])
@pytest.mark.parametrize("below,last", [(16, False), (19, False), (22, False), (22, True)])
def test_packed_sink(vla, dtype, n, n_q, hd, below, last):
    """One key takes nearly all and its value is zero: the output is what thousands of weights
    16 to 22 nats below it (2^-23 to 2^-32) add up to."""
    g = _gen(n + below)
    q, k = _rows(g, 3, n_q * hd, dtype), _rows(g, n, hd, dtype)
    v = (1 + 0.1 * torch.randn(n, hd, generator=g)).to(dtype)
    scale = hd ** -0.5  # the other keys' scores: standard normal
    sink = n - 1 if last else 0
    q.view(3, n_q, hd)[:, :, 0] = 8.0
    k[:, 0] = 0.0
    k[sink] = 0.0
    k[sink, 0] = below / (8.0 * scale)
    v[sink] = 0.0
    got = _run_packed(vla, q, k, v, [3], [n], n_q, 1, hd, scale, False)
    want, bound = ref.packed(q, k, v, [0, 3], [0, n], n_q, 1, hd, scale, False)
    if dtype is F16:
        # An fp16 below 2^-14 is off by half of its smallest step, 2^-25. The weights stand 2^9 times as large
        # as relative to a reference that is at most the row's maximum, so their sum is 2^9 at least:
        # 2^-34 of it for every key.
        bound = bound + 2.0 ** -34 * n * v.double().abs().max()
    ref.within(got, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd", [(32, 8, 128), (3, 1, 256), (40, 2, 64)])
def test_decode_a_chunk_among_single_tokens(vla, dtype, n_q, n_kv, hd):
    """Runs of keys where one sequence has many row tiles and the others one."""
    lens, new = [70, 900, 33, 513, 2], [1, 1, 70, 23, 1]  # one chunk is longer than its sequence
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, 64, dtype, seed=hd + 1)
    assert vla.kv4_attention_work_bytes(sum(new) + 2, 5, 70, 20000, n_q, n_kv, hd) > 0
    want, bound = ref.decode(q, ks, vs, new, n_q, n_kv, hd, hd ** -0.5)
    for split in (True, False):
        ref.within(_run_decode(vla, q, cache, table, lens, new, n_q, n_kv, hd, 64, hd ** -0.5, split, max_len=20000), want, bound, f"split {split}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [32, 64, 96, 256])
@pytest.mark.parametrize("byte,codes", [(253, 0x71), (253, 0x6D), (254, 0xC9), (254, 0x53)])
def test_decode_values_past_the_range(vla, dtype, hd, byte, codes):
    """A block with values of 2^128 and more, which 32 bits read as infinities, is nothing to the queries that
    do not see it."""
    lens, new, page = [70, 40], [9, 1], 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, hd, page, dtype, seed=5)
    row = table.cpu().numpy()[0]
    at = lambda part: vla.kv4_offset(row, 2, hd, page, cache.shape[0], 65, part, 1, hd // 32 - 1)
    cache.view(-1)[at(1):at(1) + 16] = codes  # token 65 of 70: queries 4..8 of 9 see it
    cache.view(-1)[at(3)] = byte
    want, bound = ref.decode(q, ks, vs, new, 4, 2, hd, hd ** -0.5)
    other = torch.ones(want.shape, dtype=torch.bool)
    other[4:9].view(5, 4, hd)[:, 2:, hd - 32:] = False
    for split, max_len in ((False, 70), (True, 4096)):
        got = _run_decode(vla, q, cache, table, lens, new, 4, 2, hd, page, hd ** -0.5, split, max_len=max_len).cpu()
        ref.within(got[other], want[other], bound[other], f"split {split}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,n_q,hd", [([40, 1, 2], 2, 64), ([700], 1, 128), ([600, 3], 2, 64), ([200, 90], 40, 96), ([150], 2, 136), ([90, 5], 1, 256)])
def test_packed_large_values(vla, dtype, causal, lens, n_q, hd):
    """Values at the end of fp32's range: their weighted mean is in range, so it comes out."""
    g = _gen(hd + sum(lens))
    q, k, _ = _packed_case(g, lens, lens, n_q, 1, hd, dtype)
    k[:, 0] += 3.0 * torch.arange(k.shape[0]).remainder(7).to(dtype)  # maxima that grow, slowly and at once
    v = (torch.rand(k.shape, generator=g) * 1e38 + 2e38).to(dtype)
    v[:, 1::2] *= -1
    s = _starts(lens)
    want, bound = ref.packed(q, k, v, s, s, n_q, 1, hd, hd ** -0.5, causal, base=torch.full_like(q, 5.0))
    ref.within(_run_packed(vla, q, k, v, lens, lens, n_q, 1, hd, hd ** -0.5, causal, same=True), want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 128, 256])
def test_decode_large_values(vla, dtype, hd):
    lens, new, page = [70, 900, 40], [9, 1, 1], 64
    q, cache, table, ks, _ = _decode_case(vla, lens, new, 4, 2, hd, page, F32, seed=5)
    q = q.to(dtype)
    g = _gen(hd)
    k, v = _rows(g, sum(lens), 2 * hd, F32), torch.rand(sum(lens), 2 * hd, generator=g) * 1.9e38 + 1e38
    v[:, 1::2] *= -1
    vla.kv4_append_dev(cache, k.to(DEV), v.to(DEV), 2, hd, page, table, _i32(lens), _i32(_starts(lens)))
    ks, vs = (ref.values(*ref.quantize(x.reshape(-1, 2, hd))).split(lens) for x in (k, v))
    want, bound = ref.decode(q, ks, vs, new, 4, 2, hd, hd ** -0.5)
    for split, max_len in ((False, 900), (True, 4096)):
        got = _run_decode(vla, q, cache, table, lens, new, 4, 2, hd, page, hd ** -0.5, split, max_len=max_len)
        ref.within(got, want, bound, f"split {split}")


def test_decode_many_sequences_without_a_bound(vla):
    """Not knowing how many new tokens a sequence has costs some time, not a block for every possible one."""
    n = 20000
    q, cache, table, ks, vs = _decode_case(vla, [20], [1], 4, 1, 32, 32, BF16, seed=4)
    table = table.expand(n, 1).contiguous()
    lens, start = torch.full((n,), 20, dtype=torch.int32, device=DEV), torch.arange(n + 1, dtype=torch.int32, device=DEV)
    qd = q.to(DEV).repeat(n, 1)
    out = torch.empty_like(qd)
    took = []
    for max_new in (1, 2 ** 31 - 1):
        for _ in range(2):  # the first call loads the kernel
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ev[0].record()
            vla.kv4_attention_dev(out, qd, cache, 4, 1, 32, 32, 0.2, table, lens, start, max_new, 32)
            ev[1].record()
            torch.cuda.synchronize()
        took.append(ev[0].elapsed_time(ev[1]))
    want, bound = ref.decode(q, ks, vs, [1], 4, 1, 32, 0.2)
    ref.within(out, want.expand(n, -1), bound.expand(n, -1))
    assert took[1] < 20 * took[0], took


def test_rope_small_sines(vla):
    """Sines and cosines next to zero keep their bits: rows of (1, 0) come out as (cos, sin)."""
    T, hd = 5000, 128
    pos = torch.arange(T, dtype=torch.int32)[None]
    x = torch.zeros(T, hd)
    x[:, :hd // 2] = 1.0
    o = torch.empty(T, hd, device=DEV)
    vla.qk_norm_rope_dev(o, None, x.to(DEV), None, 1, 0, hd, pos.to(DEV), [hd // 2], 100.0)
    want, _ = ref.rope(x, 1, hd, pos, [hd // 2], 100.0, None, 0.0)
    small = want.abs() < 0.01
    assert int(small.sum()) > 1000
    # The functions are off by 4 units of 2^-23 at most, the turn by the rest and its rounding add 2. The
    # angle: up to 5000 radians in 64 bits, of a power with some units of error: 2^13 * 2^-53 * 4, in the
    # reference as well.
    bound = 6 * 2.0 ** -23 * want.abs() + 2.0 ** -37
    ref.within(o.cpu()[small], want[small], bound[small])


@pytest.mark.parametrize("dtype,hd", [(BF16, 64), (F32, 128)])
def test_decode_rows_far_apart(vla, dtype, hd):
    """Queries and results whose offsets in their buffer pass 32 bits, through the cache's attention."""
    lens, new = [700, 130, 90], [600, 70, 30]
    T, ld = sum(new), (1 << 22) // (2 if dtype is F32 else 1)
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, hd, 32, dtype, seed=hd)
    buf = torch.empty(T, ld, dtype=dtype, device=DEV)
    assert buf.numel() * buf.element_size() > 1 << 32
    qd, out = buf[:, :2 * hd], buf[:, 2 * hd:4 * hd]
    qd.copy_(q)
    want, bound = ref.decode(q, ks, vs, new, 2, 1, hd, hd ** -0.5)
    for max_len in (700, 16384):
        work = torch.empty(max(16, vla.kv4_attention_work_bytes(T, 3, 600, max_len, 2, 1, hd)), dtype=torch.uint8, device=DEV)
        out.fill_(5.0)
        vla.kv4_attention_dev(out, qd, cache, 2, 1, hd, 32, hd ** -0.5, table, _i32(lens), _i32(_starts(new)), 600, max_len, work)
        ref.within(out, want, bound, f"max_len {max_len}")
    assert work.numel() > 16


@pytest.mark.parametrize("dtype", TYPES)
def test_repeated_joins_give_the_same_bits(vla, dtype):
    """Pieces of sequences are joined in their order, whichever block is done first."""
    lens, new = [3000, 3, 700], [1, 1, 20]
    q, cache, table, _, _ = _decode_case(vla, lens, new, 4, 2, 64, 64, dtype, seed=62)
    assert vla.kv4_attention_work_bytes(sum(new) + 2, 3, 20, 20000, 4, 2, 64) > 0
    run = lambda: _run_decode(vla, q, cache, table, lens, new, 4, 2, 64, 64, 0.125, True, max_len=20000)
    first = run()
    for _ in range(5):
        assert torch.equal(run(), first)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,n_q,hd", [([500], 2, 64), ([200], 2, 64), ([290, 250], 70, 32), ([300], 1, 128), ([260], 1, 200)])
def test_packed_values_that_grow(vla, dtype, causal, lens, n_q, hd):
    """Values that reach the end of the range late, where sums of small ones are under way; tiny values beside them,
    in sequences and queries of their own, keep their bits."""
    g = _gen(hd + sum(lens) + 1)
    q, k, v = _packed_case(g, lens, lens, n_q, 1, hd, dtype)
    v[140:] *= 1e-30
    v[140:lens[0]] *= 1e38
    v[140:lens[0]] = v[140:lens[0]].clamp(-2e8, 2e8)
    v[140:lens[0]] *= 1e30
    assert bool(torch.isfinite(v).all())
    s = _starts(lens)
    want, bound = ref.packed(q, k, v, s, s, n_q, 1, hd, hd ** -0.5, causal, base=torch.full_like(q, 5.0))
    ref.within(_run_packed(vla, q, k, v, lens, lens, n_q, 1, hd, hd ** -0.5, causal, same=True), want, bound)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("hd", [64, 128, 200])
def test_packed_tiny_values_beside_unseen_ones(vla, hd, bad):
    """An infinity or NaN that a query does not see does not cost the small values it does see any bits."""
    q, k, v = _packed_case(_gen(hd), [150], [150], 2, 1, hd, F32)
    v *= 1e-33
    want, bound = ref.packed(q, k, v, [0, 150], [0, 150], 2, 1, hd, hd ** -0.5, True, base=torch.full_like(q, 5.0))
    v[100, 3] = bad
    got = _run_packed(vla, q, k, v, [150], [150], 2, 1, hd, hd ** -0.5, True)
    ref.within(got[:100], want[:100], bound[:100])
