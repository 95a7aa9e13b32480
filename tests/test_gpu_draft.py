"""GPU tests of the operators around drafted tokens, each against its plain 64-bit
form (draft_ref.py), whose bounds are derived there."""

import math
import random

import numpy as np
import pytest
import torch

import draft_ref as dref
import serving_ref as ref
from test_gpu_serving import BF16, DEV, F16, F32, TYPES, _decode_case, _dev, _gen, _i32, _rows, _starts

pytestmark = pytest.mark.gpu


def _tree(r, n, wide):
    """Parents of a sequence's n nodes, each among the `wide` before it; wide 0: a chain."""
    return [-1 if i == 0 else i - 1 if not wide else r.randrange(max(0, i - wide), i) for i in range(n)]


def _truth(bits, n):
    return torch.tensor([[bool(b >> j & 1) for j in range(n)] for b in bits], dtype=torch.bool).reshape(len(bits), n)


# ------------------------------------------------------------------ tree --

@pytest.mark.parametrize("new,wide,extra", [([1], 0, 0), ([8], 3, 0), ([0, 5, 1, 33, 0, 64], 7, 1), ([65, 2], 0, 0), ([300, 31, 32], 0, 2),
                                            ([700], 40, 0), ([3] * 400, 2, 0)])
def test_tree(vla, new, wide, extra):
    r = random.Random(len(new) * 7 + wide)
    parents = [_tree(r, n, wide) for n in new]
    total, w = sum(new), (max(new) + 31) // 32 + extra
    lens = [n + r.randrange(0, 500) for n in new]
    start = _starts(new)
    pos = torch.full((total + 3,), 77, dtype=torch.int32, device=DEV)
    see = torch.full((total + 3, w), 77, dtype=torch.int32, device=DEV)
    for parent in [_i32([x for p in parents for x in p] + [5] * 3)] + ([None] if wide == 0 else []):
        pos.fill_(77)
        see.fill_(77)
        vla.draft_tree_dev(pos, see, parent, _i32(lens), _i32(start))
        at = 0
        for p, n, ln in zip(parents, new, lens):
            bits, depth = dref.tree(p, n)
            assert pos[at:at + n].tolist() == [ln - n + d for d in depth]
            assert torch.equal(see[at:at + n].cpu(), dref.words(bits, w))
            at += n
        assert bool((pos[total:] == 77).all()) and bool((see[total:] == 77).all())  # rows behind the sequences


@pytest.mark.parametrize("wide,words", [(0, 10), (5, 10), (200, 12), (0, 2), (9, 4), (3, 1)])
def test_tree_of_many_rows_among_short_ones(vla, wide, words):
    """Sequences of more than 64 rows where most are short."""
    r = random.Random(wide)
    new = [1, 300, 0, 2] + [1] * 40 + [129, 64, 65]
    parents, lens, start = [_tree(r, n, wide) for n in new], [n + 7 for n in new], _starts(new)
    if wide == 5:
        parents[1][100] = parents[1][200] = -1  # further roots
        parents[1][150] = 150
    pos = torch.empty(sum(new), dtype=torch.int32, device=DEV)
    see = torch.empty(sum(new), words, dtype=torch.int32, device=DEV)
    for _ in range(2):  # whatever the buffers held
        vla.draft_tree_dev(pos, see, _i32([x for p in parents for x in p]), _i32(lens), _i32(start))
        for s, n in enumerate(new):
            bits, depth = dref.tree(parents[s], n)
            assert pos[start[s]:start[s + 1]].tolist() == [7 + d for d in depth]
            assert torch.equal(see[start[s]:start[s + 1]].cpu(), dref.words(bits, words)) if n else True
        pos.fill_(-99), see.fill_(-1)


def test_tree_odd_parents_and_few_words(vla):
    """Parents that are not before their node are none; bits past the words are left out."""
    parent = [7, 0, 2, -5, 1, 4, 2 ** 31 - 1, 3] + [i - 1 for i in range(8, 70)]
    bits, depth = dref.tree(parent, 70)
    for w in (1, 2, 5):
        pos, see = torch.empty(70, dtype=torch.int32, device=DEV), torch.empty(70, w, dtype=torch.int32, device=DEV)
        vla.draft_tree_dev(pos, see, _i32(parent), _i32([100]), _i32([0, 70]))
        assert pos.tolist() == [30 + d for d in depth] and torch.equal(see.cpu(), dref.words(bits, w))


def test_tree_offsets_are_clamped(vla):
    """Offsets past the buffers, out of order or negative write inside the buffers only."""
    for start in ([0, 99, 200], [5, 2, 9], [-4, 3, 6], [0, 0, 2 ** 31 - 1]):
        pos, see = torch.zeros(16, dtype=torch.int32, device=DEV), torch.zeros(16, 2, dtype=torch.int32, device=DEV)
        vla.draft_tree_dev(pos[:8], see[:8], None, _i32([50, 60]), _i32(start))
        torch.cuda.synchronize()
        assert bool((pos[8:] == 0).all()) and bool((see[8:] == 0).all())


# ---------------------------------------------------------------- append --

def _append_case(vla, new, past, n_q, n_kv, hd, page, dtype, seed, pad=0, fill=0xEE):
    g = _gen(seed)
    total, lens = sum(new), [n + past for n in new]
    q, k, v = _rows(g, total, n_q * hd, dtype, 2.0), _rows(g, total, n_kv * hd, dtype, 0.7), _rows(g, total, n_kv * hd, dtype)
    need = [(n + page - 1) // page for n in lens]
    pages = max(1, sum(need))
    perm = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros(len(new), max(1, max(need)), dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = torch.tensor(perm[at:at + m], dtype=torch.int32)
        at += m
    cache = torch.full((pages, vla.kv4_page_bytes(n_kv, hd, page)), fill, dtype=torch.uint8, device=DEV)
    return q, k, v, lens, table, cache


def _cache_image(vla, cache, table, new, past, k, v, n_kv, hd, page, fill=0xEE):
    """The bytes that the cache must hold: 64-bit values [total, n_kv, hd] quantized one token at a time."""
    host = ref.HostCache(vla, cache.shape[0], n_kv, hd, page, fill)
    at = 0
    for s, n in enumerate(new):
        row = table[s].numpy()
        for i in range(n):
            for part, x in enumerate((k, v)):
                host.write(row, past + i, part, x[at + i])
        at += n
    return host.mem


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,rot,page,inter,norm,pad", [
    (15, 5, 64, 64, 64, False, False, 0), (4, 2, 128, 128, 32, False, True, 16), (4, 2, 128, 64, 64, True, False, 0), (3, 3, 96, 24, 96, False, True, 0),
    (2, 1, 256, 256, 32, False, True, 8), (1, 1, 32, 8, 64, True, True, 0), (2, 2, 192, 176, 64, False, False, 0), (6, 1, 192, 192, 64, True, True, 0),
    (0, 2, 64, 40, 64, False, True, 0), (5, 5, 32, 0, 32, False, True, 8),
])
def test_rope_append(vla, dtype, n_q, n_kv, hd, rot, page, inter, norm, pad):
    new, past = [5, 0, 1, 40], 30
    q, k, v, lens, table, cache = _append_case(vla, new, past, n_q, n_kv, hd, page, dtype, hd + rot)
    g, total = _gen(9), sum(new)
    wq, wk = (1 + 0.2 * torch.randn(hd, generator=g) if norm else None for _ in range(2))
    pos = torch.randint(-5, 90000, (total,), generator=g, dtype=torch.int32)
    f, mag = dref.freqs(rot), 1.25
    dq, dk, dv = _dev(q, pad), _dev(k, pad), _dev(v, pad)
    qo, ko = _dev(torch.zeros_like(q), pad), _dev(torch.zeros_like(k), pad)
    start = _i32(_starts(new))
    args = (n_q, n_kv, hd, page, table.to(DEV), _i32(lens), start, f.to(DEV), pos.to(DEV), mag, inter, _dev(wq), _dev(wk), 1e-5)
    vla.rope_kv4_append_dev(qo if n_q else None, cache, dq if n_q else None, dk, dv, *args, k_out=ko)
    torch.cuda.synchronize()
    eps = float(np.float32(1e-5))
    kr, kmag = dref.rotated(k, n_kv, hd, pos, f, mag, inter, wk, eps)
    # 64 bits up to the one rounding: positions below 2^17 leave 2^-35 of the angle, 2^-30 covers all else
    ref.within(ko, kr.flatten(1), (ref.rounding(kr, dtype) + 2.0 ** -30 * kmag).flatten(1), "k")
    if n_q:
        qr, qmag = dref.rotated(q, n_q, hd, pos, f, mag, inter, wq, eps)
        # at most as far as the rotation in 32 bits (27 u, one product more for the magnitude)
        ref.within(qo, qr.flatten(1), (ref.rounding(qr, dtype) + 28 * ref.U * qmag).flatten(1), "q")
    want = _cache_image(vla, cache, table, new, past, kr, v.double().reshape(total, n_kv, hd), n_kv, hd, page)
    assert torch.equal(cache.view(-1).cpu(), torch.from_numpy(want))
    # in place: the same bits
    a, b = qo.clone(), ko.clone()
    again = torch.full_like(cache, 0xEE)
    vla.rope_kv4_append_dev(dq if n_q else None, again, dq if n_q else None, dk, dv, *args, k_out=dk)
    assert torch.equal(dk, b) and torch.equal(again, cache) and (not n_q or torch.equal(dq, a))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rope_append_large(vla, dtype):
    """Many tokens a block, sequences that end anywhere in them, positions of the sequences themselves."""
    r = random.Random(4)
    new = [r.randrange(0, 900) for _ in range(12)] + [0]
    n_q, n_kv, hd, page, past = 3, 2, 64, 64, 7
    q, k, v, lens, table, cache = _append_case(vla, new, past, n_q, n_kv, hd, page, dtype, 5)
    total = sum(new)
    pos = torch.cat([torch.arange(past, past + n) for n in new]).to(torch.int32)
    f = dref.freqs(hd)
    qo = torch.empty_like(q, device=DEV)
    for given in (pos.to(DEV), None):
        cache.fill_(0xEE)
        vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), _i32(_starts(new)),
                                f.to(DEV), pos=given)
        qr, qmag = dref.rotated(q, n_q, hd, pos, f, 1.0, False, None, 0.0)
        ref.within(qo, qr.flatten(1), (ref.rounding(qr, dtype) + 28 * ref.U * qmag).flatten(1), "q")
        kb, vb = (torch.empty(total, n_kv * hd, dtype=F32, device=DEV) for _ in range(2))
        vla.kv4_gather_dev(kb, vb, cache, n_kv, hd, page, table.to(DEV), _i32(_starts(new)), _i32([past] * len(new)))
        kr, _ = dref.rotated(k, n_kv, hd, pos, f, 1.0, False, None, 0.0)
        assert torch.equal(kb.cpu().double(), ref.values(*ref.quantize(kr)).flatten(1))
        assert torch.equal(vb.cpu().double(), ref.values(*ref.quantize(v.reshape(total, n_kv, hd))).flatten(1))


def test_rope_append_agrees_with_its_parts(vla):
    """Rotation and append as calls of their own: the same rows, and in fp32 the same codes but at borders."""
    new, n_q, n_kv, hd, page = [40, 3], 4, 2, 64, 32
    q, k, v, lens, table, cache = _append_case(vla, new, 0, n_q, n_kv, hd, page, F32, 6)
    start, f = _i32(_starts(new)), dref.freqs(hd)
    pos = torch.cat([torch.arange(n) for n in new]).to(torch.int32).to(DEV)
    qo, ko = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), start, f.to(DEV), k_out=ko)
    q2, k2, other = torch.empty_like(qo), torch.empty_like(ko), torch.full_like(cache, 0xEE)
    vla.qk_norm_rope_dev(q2, k2, q.to(DEV), k.to(DEV), n_q, n_kv, hd, pos[None], [32], 10000.0)
    vla.kv4_append_dev(other, k2, v.to(DEV), n_kv, hd, page, table.to(DEV), _i32(lens), start)
    top = float(torch.cat([q, k], 1).abs().max())
    assert float((qo - q2).abs().max()) <= 60 * ref.U * top and float((ko - k2).abs().max()) <= 60 * ref.U * top
    assert float((cache != other).double().mean()) < 1e-3
    # without a cache only the rows are written
    q3, k3 = torch.empty_like(qo), torch.empty_like(ko)
    vla.rope_kv4_append_dev(q3, None, q.to(DEV), k.to(DEV), None, n_q, n_kv, hd, page, None, _i32(lens), start, f.to(DEV), k_out=k3)
    assert torch.equal(q3, qo) and torch.equal(k3, ko)


@pytest.mark.parametrize("dtype", TYPES)
def test_rope_append_codes_at_borders(vla, dtype):
    """Values half way between codes go to the even one; a magnitude just past it does not."""
    hd, page = 32, 32
    x = torch.zeros(4, hd, dtype=dtype)
    x[:, 0] = 7.0  # the block's scale is 1
    x[:, 1:9] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25])
    start, lens, table = _i32([0, 4]), _i32([4]), _i32([[0]])
    for mag in (1.0, 1.0 + 2.0 ** -40, 1.0 - 2.0 ** -40):
        cache = torch.zeros(1, vla.kv4_page_bytes(1, hd, page), dtype=torch.uint8, device=DEV)
        pos = torch.zeros(4, dtype=torch.int32, device=DEV)
        vla.rope_kv4_append_dev(None, cache, None, x.to(DEV), x.to(DEV), 0, 1, hd, page, table, lens, start, dref.freqs(hd).to(DEV), pos=pos, magnitude=mag)
        host = ref.HostCache(vla, 1, 1, hd, page)
        for i in range(4):
            host.write([0], i, 0, x[i:i + 1].double() * mag)
            host.write([0], i, 1, x[i:i + 1])
        assert torch.equal(cache.view(-1).cpu(), torch.from_numpy(host.mem)), mag


def test_rope_append_not_finite(vla):
    """A NaN or an infinity stays in its head; its blocks read as NaN, all others are as without it."""
    new, n_q, n_kv, hd, page = [6], 2, 2, 64, 32
    q, k, v, lens, table, cache = _append_case(vla, new, 0, n_q, n_kv, hd, page, F32, 8)
    clean = torch.full_like(cache, 0xEE)
    qo, qc = torch.empty(6, 128, device=DEV), torch.empty(6, 128, device=DEV)
    a = (n_q, n_kv, hd, page, table.to(DEV), _i32(lens), _i32([0, 6]), dref.freqs(64).to(DEV))
    vla.rope_kv4_append_dev(qc, clean, q.to(DEV), k.to(DEV), v.to(DEV), *a, q_weight=torch.ones(64, device=DEV))
    q[1, 3], k[2, 64 + 5], v[3, 40] = math.nan, math.inf, math.nan
    vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), *a, q_weight=torch.ones(64, device=DEV))
    same = (qo == qc).reshape(6, 2, 64).all(-1)
    assert same.cpu().tolist() == [[True, True], [False, True]] + [[True, True]] * 4
    kb, vb, kc, vc = (torch.empty(6, 128, device=DEV) for _ in range(4))
    vla.kv4_gather_dev(kb, vb, cache, n_kv, hd, page, table.to(DEV), _i32([0, 6]))
    vla.kv4_gather_dev(kc, vc, clean, n_kv, hd, page, table.to(DEV), _i32([0, 6]))
    # pair (5, 37) of head 1: both blocks; value 40 of head 0: its second block
    bad = torch.zeros(6, 128, dtype=torch.bool, device=DEV)
    bad[2, 64:] = True
    assert bool(kb[bad].isnan().all()) and torch.equal(kb[~bad], kc[~bad])
    bad = torch.zeros(6, 128, dtype=torch.bool, device=DEV)
    bad[3, 32:64] = True
    assert bool(vb[bad].isnan().all()) and torch.equal(vb[~bad], vc[~bad])


def test_rope_append_bad_pages_and_rows(vla):
    """Rows whose page is not there are rotated and dropped; rows behind the sequences stay as they are."""
    new, n_q, n_kv, hd, page = [40, 8], 1, 1, 32, 32
    q, k, v, lens, table, cache = _append_case(vla, new, 0, n_q, n_kv, hd, page, F32, 12)
    table = torch.tensor([[0, -1], [7, 1]], dtype=torch.int32)
    cache = torch.full((3, cache.shape[1]), 0xEE, dtype=torch.uint8, device=DEV)
    qo, ko = torch.full((48, 32), 5.0, device=DEV), torch.full((48, 32), 5.0, device=DEV)
    vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), 1, 1, hd, page, table.to(DEV), _i32([40, 6]), _i32([0, 40, 46]),
                            dref.freqs(32).to(DEV), k_out=ko)
    assert bool((qo[46:] == 5.0).all()) and bool((ko[46:] == 5.0).all()) and not bool((ko[:46] == 5.0).all(-1).any())
    assert bool((cache[1:] == 0xEE).all()) and not bool((cache[0] == 0xEE).all())


# ------------------------------------------------------------- attention --

def _attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, scale, split=True, max_len=None, max_new=None, pad=0, behind=2):
    total = sum(new)
    qd = _dev(torch.cat([q, torch.ones(behind, q.shape[1], dtype=q.dtype)]), pad)
    out = _dev(torch.full((total + behind, q.shape[1]), 5.0, dtype=q.dtype), pad)
    see = torch.cat([see, torch.full((behind, see.shape[1]), -1, dtype=torch.int32)]).to(DEV)
    max_new, max_len = max_new or max(1, max(new)), max_len or max(1, max(lens))
    work = None
    if split:
        nb = vla.kv4_tree_attention_work_bytes(total + behind, len(lens), max_new, max_len, n_q, n_kv, hd)
        work = torch.full((max(16, nb),), 0xFF, dtype=torch.uint8, device=DEV)
    vla.kv4_tree_attention_dev(out, qd, cache, n_q, n_kv, hd, page, scale, table, _i32(lens), _i32(_starts(new)), see, max_new, max_len, work)
    torch.cuda.synchronize()
    assert bool((out[total:] == 5.0).all())
    return out[:total]


def _masks(new, wide, seed, keep=1.0, extra=0):
    """([per sequence truth values [n, n]], words) of trees, bits then dropped with probability 1 - keep."""
    r = random.Random(seed)
    w = max(1, (max(new) + 31) // 32 + extra)
    truth, rows = [], []
    for n in new:
        bits = dref.tree(_tree(r, n, wide), n)[0]
        if keep < 1:
            bits = [b & sum((r.random() < keep) << j for j in range(n)) for b in bits]
        truth.append(_truth(bits, n))
        rows.append(dref.words(bits, w))
    return truth, torch.cat(rows) if rows else torch.zeros(0, w, dtype=torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(1, 1, 32, 32), (15, 5, 64, 64), (6, 2, 96, 96), (32, 8, 128, 64), (4, 2, 192, 32), (3, 1, 256, 128),
                                              (40, 2, 64, 64), (35, 1, 128, 32)])
def test_tree_attention(vla, dtype, n_q, n_kv, hd, page):
    lens, new = [100, 8, 0, 33, 64, 70], [9, 8, 0, 33, 1, 17]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=hd + n_q)
    truth, see = _masks(new, 5, 3, extra=1)
    want, bound = dref.attend(q, ks, vs, new, truth, n_q, n_kv, hd, hd ** -0.5)
    for kw in (dict(), dict(split=False), dict(max_len=1 << 20), dict(max_len=4096, max_new=4), dict(pad=16)):
        ref.within(_attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, hd ** -0.5, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd", [(15, 5, 64), (8, 1, 128), (2, 2, 256), (20, 1, 32)])
def test_tree_attention_any_mask(vla, dtype, n_q, n_kv, hd):
    """Bits that are no tree's, rows without a key among them, more new tokens than cached ones, new ones only."""
    lens, new, page = [90, 30, 5, 40], [50, 30, 9, 37], 32
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=hd)
    truth, see = _masks(new, 6, 8, keep=0.5)
    r = random.Random(2)
    for s, at in ((0, 0), (2, 80)):  # any bits, of later nodes too
        for i in range(new[s]):
            for j in range(new[s]):
                b = r.random() < 0.3
                truth[s][i, j] = b
                word = int(see[at + i, j // 32]) & 0xffffffff
                word = word & ~(1 << j % 32) | b << j % 32
                see[at + i, j // 32] = word - 2 ** 32 if word >= 2 ** 31 else word
    truth[1][4] = False
    see[54] = 0
    # of sequence 2 only the newest 5 of 9 rows have a key of their own: token t is key t - 4
    want, bound = dref.attend(q, ks, vs, new, truth, n_q, n_kv, hd, 0.2)
    assert bool((want[54] == 0).all())
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        ref.within(_attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, 0.2, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,new", [([3000, 5, 257, 1024], [6, 5, 40, 1]), ([4097], [64]), ([2000, 2000], [100, 3])])
@pytest.mark.parametrize("n_q,n_kv,hd,page", [(4, 2, 64, 96), (8, 1, 128, 256), (2, 1, 256, 64)])
def test_tree_attention_split_keys(vla, dtype, lens, new, n_q, n_kv, hd, page):
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=7)
    truth, see = _masks(new, 9, 4)
    want, bound = dref.attend(q, ks, vs, new, truth, n_q, n_kv, hd, hd ** -0.5)
    for kw in (dict(), dict(split=False), dict(max_len=64), dict(max_len=100000), dict(max_new=2 ** 31 - 1)):
        ref.within(_attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, hd ** -0.5, **kw), want, bound, str(kw))


def test_tree_attention_of_a_chain_is_causal(vla):
    """A chain's bits give the attention of a causal chunk."""
    lens, new, n_q, n_kv, hd, page = [300, 40], [33, 40], 8, 2, 64, 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, BF16, seed=3)
    truth, see = _masks(new, 0, 1)
    want, _ = ref.decode(q, ks, vs, new, n_q, n_kv, hd, 0.125)
    same, bound = dref.attend(q, ks, vs, new, truth, n_q, n_kv, hd, 0.125)
    assert float((want - same).abs().max()) < 1e-12
    ref.within(_attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, 0.125), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,max_len", [(32, None), (128, None), (256, None), (96, 4096)])
def test_tree_attention_not_finite(vla, dtype, hd, max_len):
    """A drafted token with a NaN is seen by the rows below it and by no others."""
    lens, new, page = [70, 40], [9, 1], 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 4, 2, hd, page, dtype, seed=5)
    parent = [[-1, 0, 0, 1, 1, 2, 4, 4, 5], [-1]]
    truth = [_truth(dref.tree(p, n)[0], n) for p, n in zip(parent, new)]
    see = torch.cat([dref.words(dref.tree(p, n)[0], 1) for p, n in zip(parent, new)])
    want, bound = dref.attend(q, ks, vs, new, truth, 4, 2, hd, hd ** -0.5)
    row = table.cpu().numpy()[0]
    below = truth[0][:, 4]  # token 61 + 4 = 65
    for part in (2, 3):
        c = cache.clone()
        c.view(-1)[vla.kv4_offset(row, 2, hd, page, cache.shape[0], 65, part, 1, hd // 32 - 1)] = 255
        got = _attend(vla, q, c, table, lens, new, see, 4, 2, hd, page, hd ** -0.5, max_len=max_len).cpu()
        keep = torch.cat([~below, torch.tensor([True])])
        ref.within(got[keep], want[keep], bound[keep], "rows that do not see it")
        ref.within(got[:, :2 * hd], want[:, :2 * hd], bound[:, :2 * hd], "other kv head")
        tail = got[~keep][:, 2 * hd:].reshape(-1, 2, hd)
        assert bool(tail[:, :, hd - 32:].isnan().all())
        if part == 3 and hd > 32:
            w, b = (x[~keep][:, 2 * hd:].reshape(-1, 2, hd)[:, :, :hd - 32] for x in (want, bound))
            ref.within(tail[:, :, :hd - 32], w, b, "other blocks")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 128, 256])
def test_tree_attention_bad_pages(vla, dtype, hd):
    """A page that is not there is NaN for the rows that see it; one that only some rows' mask reaches, for those."""
    lens, new, page = [70, 80], [6, 20], 32
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, hd, page, dtype, seed=15)
    truth, see = _masks(new, 4, 5)
    truth[1][3, 4:], see[9, 0] = False, int(see[9, 0]) & 15
    want, bound = dref.attend(q, ks, vs, new, truth, 2, 1, hd, 0.1)
    t = table.clone()
    t[1, 2] = -1  # tokens 64 .. 79, new ones 4 .. 19
    got = _attend(vla, q, cache, t, lens, new, see, 2, 1, hd, page, 0.1).cpu()
    sees = torch.cat([torch.zeros(6, dtype=torch.bool), truth[1][:, 4:].any(1)])
    assert bool(got[sees].isnan().all()) and 0 < int(sees.sum()) < 20
    ref.within(got[~sees], want[~sees], bound[~sees])
    t[0, 0] = 1 << 30
    got = _attend(vla, q, cache, t, lens, new, see, 2, 1, hd, page, 0.1).cpu()
    assert bool(got[:6].isnan().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
def test_tree_attention_past_the_table(vla, dtype, hd):
    """A length beyond the table: tokens behind it read as NaN where a row sees them, never outside the cache."""
    lens, new, page = [64], [4], 32
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, hd, page, dtype, seed=16)
    truth, see = _masks(new, 0, 1)
    got = _attend(vla, q, cache, table, [100], new, see, 2, 1, hd, page, 0.1, max_len=100)
    assert bool(got.isnan().all())
    got = _attend(vla, q, cache, table, [2 ** 31 - 1], new, see, 2, 1, hd, page, 0.1, max_len=100)
    assert bool(got.isnan().all())
    # 66 tokens, of which the newest two have no page: the first two rows do not see them
    got = _attend(vla, q, cache, table, [66], new, see, 2, 1, hd, page, 0.1, max_len=100).cpu()
    assert bool(got[2:].isnan().all()) and bool(torch.isfinite(got[:2].double()).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [3.0, -0.2, 0.0])
def test_tree_attention_scales(vla, dtype, scale):
    lens, new = [100, 7], [20, 4]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, 64, 32, dtype, seed=3)
    truth, see = _masks(new, 3, 6)
    want, bound = dref.attend(q, ks, vs, new, truth, 2, 1, 64, scale)
    ref.within(_attend(vla, q, cache, table, lens, new, see, 2, 1, 64, 32, scale), want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hd", [32, 128, 256])
def test_tree_attention_large_values(vla, dtype, hd):
    """Cached values near the end of fp32's range: no sum on the way overflows."""
    lens, new, page = [600], [12], 64
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, hd, page, dtype, seed=23)
    c, row = cache.clone(), table.cpu().numpy()[0]
    for t in range(600):
        for b in range(hd // 32):
            c.view(-1)[vla.kv4_offset(row, 1, hd, page, c.shape[0], t, 3, 0, b)] += 120
    v = vs[0] * 2.0 ** 120
    truth, see = _masks(new, 4, 7)
    want, bound = dref.attend(q, ks, [v], new, truth, 2, 1, hd, 0.1)
    for kw in (dict(), dict(max_len=1 << 20)):
        ref.within(_attend(vla, q, c, table, lens, new, see, 2, 1, hd, page, 0.1, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("shift,where", [(-40, "early"), (-40, "late"), (25, "late"), (-95, "all"), (90, "all"), (-22, "all"), (8, "all"), (-100, "zero")])
def test_tree_attention_of_any_magnitude(vla, dtype, hd, shift, where):
    """Keys' and values' blocks of other magnitudes than fp16 takes, from the first tile on, from a later one, or in all: the
    results keep their bits whatever form the products take."""
    n_q, n_kv, page, n, m = 8, 1, 32, 500, 40
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=hd)
    c, row = cache.cpu(), table.cpu().numpy()[0]
    v, k, at = vs[0].clone(), ks[0].clone(), lambda t, part: vla.kv4_offset(row, n_kv, hd, page, c.shape[0], t, part, 0, hd // 32 - 1)
    cols = slice(hd - 32, hd)
    for t in {"early": [3], "late": range(300, 310), "all": range(n), "zero": range(0, n, 7)}[where]:
        for part, x in ((2, k), (3, v)):
            if part == 2 and shift > 0:
                continue  # (keys that large would leave one weight)
            byte = int(c.view(-1)[at(t, part)])
            if where == "zero":  # zeros of the smallest exponent count for nothing
                lo = at(t, part - 2)
                c.view(-1)[lo:lo + 16] = 0
                new, x[t, :, cols] = 27, 0.0
            else:
                new = max(27, byte + shift)
                x[t, :, cols] *= 2.0 ** (new - byte)
            c.view(-1)[at(t, part)] = new
    truth, see = _masks([m], 4, 7)
    want, bound = dref.attend(q, [k], [v], [m], truth, n_q, n_kv, hd, hd ** -0.5)
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        got = _attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, hd ** -0.5, **kw).double().cpu()
        # results past the type's range round to infinity, and may from where the bound reaches it
        top = torch.finfo(dtype).max
        over = (want.abs() + bound > top) & got.isinf() & (got.sign() == want.sign())
        assert bool(got[want.abs() - bound > top * (1 + ref.half(dtype))].isinf().all())
        ref.within(torch.where(over, want, got), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("below", [12, 17, 22, 30])
@pytest.mark.parametrize("m", [3, 40])
def test_tree_attention_sink(vla, dtype, hd, below, m):
    """One key takes nearly all of every row's weight and has the value zero: the others' small weights keep their bits."""
    n_q, n_kv, page, n = 4, 1, 64, 2000
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=below)
    c, row = cache.cpu(), table.cpu().numpy()[0]
    q = torch.zeros_like(q)
    q[:, ::hd] = 1.0  # a row's score is its key's first value
    k, v = ks[0].clone(), vs[0].clone()
    k[0, 0, 0], v[0] = 4.0, 0.0
    scale = below / 4.0
    for t in range(n):
        lo = vla.kv4_offset(row, n_kv, hd, page, c.shape[0], t, 0, 0, 0)
        sc = vla.kv4_offset(row, n_kv, hd, page, c.shape[0], t, 2, 0, 0)
        c.view(-1)[lo:lo + 16] = 0
        c.view(-1)[lo] = 6 if t == 0 else 0  # 4 * 2^0, others 0
        c.view(-1)[sc] = 127
        k[t, 0, :32] = 0.0
        k[t, 0, 0] = 4.0 if t == 0 else 0.0
    for b in range(hd // 32):
        lo = vla.kv4_offset(row, n_kv, hd, page, c.shape[0], 0, 1, 0, b)
        c.view(-1)[lo:lo + 16] = 0
    truth, see = _masks([m], 3, 7)
    want, bound = dref.attend(q, [k], [v], [m], truth, n_q, n_kv, hd, scale)
    # keys of the sink's own 64 lose at most 2^-18 of it, as the bound says; all others 2^-18 of their own largest, which is theirs
    w = math.exp(-below) / (1 + (n - 1) * math.exp(-below))
    tight = want.abs() * ref.half(dtype) + torch.finfo(dtype).smallest_normal * ref.half(dtype) \
        + v[:, 0].abs().sum(0).repeat(n_q) * w * (2.0 ** -11 + 64 * ref.U * below) + v[:64, 0].abs().sum(0).repeat(n_q) * 2.0 ** -18 / (1 + n * math.exp(-below)) \
        + v[:, 0].abs().sum(0).repeat(n_q) * w * (n + 24) * ref.U
    for kw in (dict(), dict(max_len=1 << 20)):
        got = _attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, scale, **kw)
        ref.within(got, want, torch.minimum(bound, tight), str(kw))


def test_tree_attention_many_sequences(vla):
    """2000 small trees, a bound on their size or none."""
    r = random.Random(5)
    new = [r.choice([0, 1, 3, 7]) for _ in range(2000)]
    lens = [n + r.randrange(0, 20) for n in new]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, 2, 1, 32, 32, BF16, seed=2)
    truth, see = _masks(new, 2, 6)
    want, bound = dref.attend(q, ks, vs, new, truth, 2, 1, 32, 0.2)
    for m in (7, 2 ** 31 - 1):
        ref.within(_attend(vla, q, cache, table, lens, new, see, 2, 1, 32, 32, 0.2, max_new=m), want, bound)


# ---------------------------------------------------------------- verify --

def _verify(vla, p, q, tokens, parent, start, u, u_next, extra=2, pad=0, shift=0):
    total, n = p.shape[0], len(start) - 1

    def rows(x):
        if x is None:
            return None
        buf = torch.full((total * (x.shape[1] + pad) + shift,), 0.3, dtype=x.dtype, device=DEV)
        v = torch.as_strided(buf, x.shape, (x.shape[1] + pad, 1), shift)
        return v.copy_(x.to(DEV))

    path = torch.full((total,), 77, dtype=torch.int32, device=DEV)
    count, token = (torch.full((n,), 77, dtype=torch.int32, device=DEV) for _ in range(2))
    vla.verify_drafts_dev(path, count, token, rows(p), _i32(tokens), _i32(start), u.to(DEV), u_next.to(DEV), None if parent is None else _i32(parent), rows(q))
    return path.tolist(), count.tolist(), token.tolist()


def _drafts(g, r, new, V, dtype, wide, sampled, peak=2.0, far=0.8):
    """Probabilities of a target and a draft near it, children drawn from the draft or its most probable ones."""
    total, start = sum(new), _starts(new)
    z = torch.randn(total, V, generator=g) * peak
    p = torch.softmax(z, -1).to(dtype)
    q = torch.softmax(z + torch.randn(total, V, generator=g) * far, -1).to(dtype)
    parent, tokens = [], []
    for s, n in enumerate(new):
        ps, seen = _tree(r, n, wide), {}
        for x in ps:
            row = q[start[s] + max(0, x)].double()
            seen[x] = seen.get(x, 0) + 1
            tokens.append(int(torch.multinomial(row, 1, generator=g)) if sampled else int(row.argsort(descending=True)[(seen[x] - 1) % V]))
        parent += ps
    return p, q if sampled else None, tokens, parent, start, torch.rand(total, generator=g), torch.rand(len(new), generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("new,V,wide", [([5], 100, 0), ([1, 0, 30, 7], 37, 4), ([20] * 6, 1000, 3), ([9, 9, 9], 2, 2), ([4] * 5, 4099, 0),
                                        ([12] * 3, 20001, 20), ([2, 3], 1, 1), ([70], 300, 70), ([3], 70001, 2)])
def test_verify(vla, dtype, sampled, new, V, wide):
    g, r = _gen(V + len(new)), random.Random(V)
    case = _drafts(g, r, new, V, dtype, wide, sampled)
    want = dref.verify(*case)
    assert _verify(vla, *case) == want
    # rows that start anywhere, and strides that put p and q at different places of 16 bytes
    assert _verify(vla, *case, pad=3, shift=1) == want
    if wide == 0:
        p, q, tokens, _, start, u, un = case
        assert _verify(vla, p, q, tokens, None, start, u, un) == want


def test_verify_rows_out_of_step(vla):
    """p and q whose rows begin at different places of 16 bytes."""
    g, r = _gen(1), random.Random(1)
    for dtype in TYPES:
        p, q, tokens, parent, start, u, un = _drafts(g, r, [6, 6], 4001, dtype, 3, True)
        want = dref.verify(p, q, tokens, parent, start, u, un)
        wide = torch.zeros(12, 4001 + 5, dtype=dtype, device=DEV)
        wide[:, 3:4004] = q.to(DEV)
        path, count, token = (torch.empty(k, dtype=torch.int32, device=DEV) for k in (12, 2, 2))
        vla.verify_drafts_dev(path, count, token, p.to(DEV), _i32(tokens), _i32(start), u.to(DEV), un.to(DEV), _i32(parent), wide[:, 3:4004])
        assert (path.tolist(), count.tolist(), token.tolist()) == want


@pytest.mark.parametrize("sampled", [True, False])
def test_verify_many_nodes(vla, sampled):
    """More nodes than have room in LDS, most of them children of one node, the same tokens again and again."""
    g, r = _gen(11), random.Random(11)
    for n, wide in ((1500, 1500), (1300, 0), (700, 5)):
        p, q, tokens, parent, start, u, un = _drafts(g, r, [3, n], 50, F32, wide, sampled)
        if wide == n:
            parent = [-1, 0, 0] + [-1] + [0] * (n - 1)
        u = u * 0.001 + 0.999 if wide == n else u * 0.01  # hardly any, or nearly all are accepted
        want = dref.verify(p, q, tokens, parent, start, u, un)
        assert _verify(vla, p, q, tokens, parent, start, u, un) == want


def test_verify_borders(vla):
    """Numbers on a border of exact sums: the strict comparisons of the definition, ties to the lowest token."""
    V = 8
    p = torch.tensor([[0.25, 0, 0.25, 0, 0.125, 0.125, 0.25, 0]] * 4)
    q = torch.tensor([[0.5, 0, 0, 0, 0.25, 0.25, 0, 0]] * 4)
    un = [0.0, 0.25, 0.25 - 2 ** -24, 0.5, 0.75, 0.999999, 1.0, 7.0, math.nan, -1.0, 0.624999]
    for x in un:
        for u, tok in ((0.5, 0), (0.5 - 2 ** -24, 0), (0.0, 1), (0.0, 2), (0.0, 3), (0.0, -1), (0.0, 8), (math.nan, 0)):
            for qq in (q, None):
                case = (p, qq, [0, tok, 2, 4], [-1, 0, 0, 1], [0, 4], torch.tensor([0.0, u, 0.9, 0.0]), torch.tensor([x]))
                if math.isnan(x):  # as 0
                    want = dref.verify(*case[:-1], torch.tensor([0.0]))
                else:
                    want = dref.verify(*case)
                assert _verify(vla, *case) == want, (x, u, tok, qq is None)


def test_verify_without_a_residual(vla):
    """A refusal where p - q leaves nothing draws from p; rows of zeros give no token; NaN counts as 0."""
    p = torch.tensor([[0.5, 0.5, 0.0], [0.0, 0.0, 0.0], [math.nan, 1.0, math.nan]])
    # a token that p does not have, and q above p everywhere else
    q = torch.tensor([[0.5, 0.5, 1.0]] * 3)
    got = _verify(vla, p, q, [0, 2, 0], [-1, 0, -1], [0, 2, 3], torch.tensor([0.1, 0.1, 0.1]), torch.tensor([0.7, 0.0]))
    assert got == ([0, -1, 0], [1, 1], [1, 1])
    got = _verify(vla, p[1:2], None, [0], None, [0, 1], torch.tensor([0.1]), torch.tensor([0.7]))
    assert got == ([0], [1], [-1])
    # one-hot rows: the greedy choice, whatever the random numbers
    hot = torch.eye(3)[[1, 2, 0]]
    for x in (0.0, 0.5, 0.999999):
        got = _verify(vla, hot, None, [0, 1, 1], None, [0, 3], torch.tensor([x] * 3), torch.tensor([x]))
        assert got == ([0, 1, -1], [2], [2])


def test_verify_keeps_the_targets_distribution(vla):
    """Over many random numbers the first token behind the root is distributed as the target's: of 40000 draws each share is
    within 5 standard deviations."""
    V, n = 6, 40000
    g = _gen(3)
    pt = torch.tensor([0.4, 0.05, 0.25, 0.1, 0.2, 0.0], dtype=torch.float64)
    qt = torch.tensor([0.1, 0.3, 0.2, 0.1, 0.1, 0.2], dtype=torch.float64)
    kids = torch.multinomial(qt, 3 * n, replacement=True, generator=g).reshape(n, 3)
    tokens = torch.cat([torch.zeros(n, 1, dtype=torch.int64), kids], 1).flatten().tolist()
    p, q = pt.float().repeat(4 * n, 1), qt.float().repeat(4 * n, 1)
    u, un = torch.rand(4 * n, generator=g), torch.rand(n, generator=g)
    path, count, token = _verify(vla, p, q, tokens, [-1, 0, 0, 0] * n, list(range(0, 4 * n + 1, 4)), u, un)
    first = [tokens[4 * s + path[4 * s + 1]] if count[s] > 1 else token[s] for s in range(n)]
    share = torch.bincount(torch.tensor(first), minlength=V).double() / n
    assert bool(((share - pt).abs() <= 5 * (pt * (1 - pt) / n).sqrt() + 1e-6).all()), share


def test_verify_offsets_are_clamped(vla):
    for start in ([0, 99, 200], [5, 2, 9], [-4, 3, 6], [0, 0, 2 ** 31 - 1], [9, 20, 30]):
        path = torch.full((16,), 77, dtype=torch.int32, device=DEV)
        count, token = (torch.full((4,), 77, dtype=torch.int32, device=DEV) for _ in range(2))
        p = torch.rand(8, 30, device=DEV)
        vla.verify_drafts_dev(path[:8], count[:2], token[:2], p, _i32([3] * 8), _i32(start), torch.rand(8, device=DEV), torch.rand(2, device=DEV))
        torch.cuda.synchronize()
        assert bool((path[8:] == 77).all()) and bool((count[2:] == 77).all())
        assert all(0 <= c <= 8 for c in count[:2].tolist()) and all(-1 <= t < 30 for t in token[:2].tolist())


# ------------------------------------------------------------------ keep --

@pytest.mark.parametrize("n_kv,hd,page", [(5, 64, 64), (2, 32, 32), (3, 96, 96), (8, 128, 64), (1, 192, 32), (2, 256, 32)])
def test_keep(vla, n_kv, hd, page):
    """Every path of rows, those that move onto each other's places among them; everything else keeps its bytes."""
    r = random.Random(hd)
    new = [1, 0, 9, 40, 70, 200, 3, 5]
    past = [0, 5, 60, 31, 500, 64, 33, 2]
    lens = [a + b for a, b in zip(past, new)]
    paths = [[0], [], [0, 1, 3, 4, 8], [0] + list(range(2, 40)), sorted(r.sample(range(70), 30)), list(range(5, 200)), [], [0, 1, 2, 3, 4]]
    need = [(n + page - 1) // page for n in lens]
    g = _gen(hd)
    perm = torch.randperm(sum(need), generator=g).tolist()
    table = torch.zeros(len(new), max(need), dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = torch.tensor(perm[at:at + m], dtype=torch.int32)
        at += m
    cache = torch.randint(0, 256, (sum(need), vla.kv4_page_bytes(n_kv, hd, page)), generator=g, dtype=torch.uint8)
    want = cache.clone().view(-1)
    before = want.clone()
    flat, count = [], [len(p) for p in paths]
    for s, p in enumerate(paths):
        row = table[s].numpy()
        for i, src in enumerate(p):
            for h in range(n_kv):
                for b in range(hd // 32):
                    for part in range(4):
                        x, y = (vla.kv4_offset(row, n_kv, hd, page, sum(need), past[s] + t, part, h, b) for t in (src, i))
                        w = 16 if part < 2 else 1
                        want[y:y + w] = before[x:x + w]
        flat += p + [-1] * (new[s] - len(p))
    out = torch.full((len(new),), 77, dtype=torch.int32, device=DEV)
    c = cache.to(DEV)
    vla.kv4_keep_dev(c, n_kv, hd, page, table.to(DEV), _i32(lens), _i32(_starts(new)), _i32(flat + [3, 3]), _i32(count), out)
    assert torch.equal(c.view(-1).cpu(), want) and out.tolist() == [a + b for a, b in zip(past, count)]
    c = cache.to(DEV)
    vla.kv4_keep_dev(c, n_kv, hd, page, table.to(DEV), _i32(lens), _i32(_starts(new)), _i32(flat), _i32(count))
    assert torch.equal(c.view(-1).cpu(), want)


def test_keep_bad_calls_stay_inside(vla):
    """Paths, counts, pages and lengths that name nothing: no byte outside the pages of the table changes."""
    n_kv, hd, page = 2, 64, 32
    nb = vla.kv4_page_bytes(n_kv, hd, page)
    cache = torch.full((4, nb), 0xAB, dtype=torch.uint8, device=DEV)
    table = _i32([[1, -3], [2, 99]])
    for path, count, lens, start in (([0, -7, 2 ** 31 - 1, 3], [4, 9], [40, 3], [0, 4, 4]), ([5, 6, 7, 8], [-3, 2], [2 ** 31 - 1, 30], [0, 2, 4]),
                                     ([3, 2, 1, 0], [2, 2], [1, -5], [0, 2, 4]), ([1, 1, 1, 1], [2, 2], [33, 64], [-2, 9, 4])):
        vla.kv4_keep_dev(cache, n_kv, hd, page, table, _i32(lens), _i32(start), _i32(path), _i32(count), torch.empty(2, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert bool((cache[0] == 0xAB).all()) and bool((cache[3] == 0xAB).all())


def test_keep_a_token_without_a_page(vla):
    """It moves as NaN where it is kept, and is dropped where it would go."""
    n_kv, hd, page = 1, 32, 32
    cache = torch.zeros(2, vla.kv4_page_bytes(n_kv, hd, page), dtype=torch.uint8, device=DEV)
    vla.kv4_keep_dev(cache, n_kv, hd, page, _i32([[0, -1]]), _i32([34]), _i32([0, 6]), _i32([0, 4, 5, -1, -1, -1]), _i32([3]))
    k, v = torch.empty(6, 32, device=DEV), torch.empty(6, 32, device=DEV)
    vla.kv4_gather_dev(k, v, cache, n_kv, hd, page, _i32([[0, 1]]), _i32([0, 6]), _i32([28]))
    assert k[:, 0].isnan().tolist() == v[:, 0].isnan().tolist() == [False, True, True, False, False, False]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd", [(0, 3, 64), (0, 1, 96), (5, 5, 32), (0, 2, 256)])
def test_rope_append_that_turns_nothing(vla, dtype, n_q, n_kv, hd):
    """Without pairs and norms it is the append, with or without queries; k_out and q_out get the rows as they are."""
    new, page = [40, 1, 0, 7], 32
    q, k, v, lens, table, cache = _append_case(vla, new, 9, max(1, n_q), n_kv, hd, page, dtype, 17)
    other, ko = cache.clone(), torch.empty_like(k, device=DEV)
    start, none = _i32(_starts(new)), torch.empty(0, dtype=torch.float64, device=DEV)
    qd = q.to(DEV) if n_q else None
    qo = torch.empty_like(qd) if n_q else None
    vla.rope_kv4_append_dev(qo, cache, qd, k.to(DEV), v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), start, none, k_out=ko)
    vla.kv4_append_dev(other, k.to(DEV), v.to(DEV), n_kv, hd, page, table.to(DEV), _i32(lens), start)
    assert torch.equal(cache, other) and torch.equal(ko.cpu(), k)
    assert not n_q or torch.equal(qo.cpu(), q)


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (BF16, 64), (F16, 256)])
def test_tree_attention_of_more_than_it_was_told(vla, dtype, hd):
    """max_new and max_len choose the launch only, the workspace of those sizes is all that is used."""
    n_q, n_kv, page, lens, new = 8, 2, 32, [900, 40, 3000, 64], [33, 5, 90, 1]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=19)
    truth, see = _masks(new, 6, 5)
    want, bound = dref.attend(q, ks, vs, new, truth, n_q, n_kv, hd, 0.1)
    for max_new, max_len in ((1, 1), (1, 3000), (40, 1), (90, 100), (2 ** 31 - 1, 2 ** 31 - 1)):
        nb = vla.kv4_tree_attention_work_bytes(sum(new), 4, max_new, max_len, n_q, n_kv, hd)
        room = torch.full((nb + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
        out = torch.empty_like(q, device=DEV)
        vla.kv4_tree_attention_dev(out, q.to(DEV), cache, n_q, n_kv, hd, page, 0.1, table, _i32(lens), _i32(_starts(new)), see.to(DEV), max_new,
                                   max_len, room[:max(16, nb)])
        ref.within(out, want, bound, str((max_new, max_len)))
        assert bool((room[max(16, nb):] == 0xA5).all())


# ------------------------------------------------------ far apart in memory --

def _far_rows(x, ld):
    """The same rows, `ld` elements apart, the last one 2^31 elements or more behind the first."""
    assert (x.shape[0] - 1) * ld >= 2 ** 31
    buf = torch.empty((x.shape[0] - 1) * ld + x.shape[1], dtype=x.dtype, device=DEV)
    return torch.as_strided(buf, x.shape, (ld, 1)).copy_(x)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_append_far_rows(vla, interleaved):
    """Rows, and pages of the cache, behind 2^31 elements and bytes."""
    n_q, n_kv, hd, page, new = 4, 2, 64, 32, [3, 6]
    q, k, v, lens, table, cache = _append_case(vla, new, 20, n_q, n_kv, hd, page, BF16, 71)
    rest = (n_q, n_kv, hd, page)
    args = (_i32(lens), _i32(_starts(new)), dref.freqs(hd).to(DEV))
    qo, ko = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), *rest, table.to(DEV), *args, interleaved=interleaved, k_out=ko)
    nb, ld = cache.shape[1], 2 ** 28 + 64
    far = torch.empty((2 ** 32 + 2 ** 20) // nb, nb, dtype=torch.uint8, device=DEV)
    off = far.shape[0] - cache.shape[0]
    far[off:].fill_(0xEE)
    qf, kf = _far_rows(q, ld), _far_rows(k, ld)
    vla.rope_kv4_append_dev(qf, far, qf, kf, _far_rows(v, ld), *rest, (table + off).to(DEV), *args, interleaved=interleaved, k_out=kf)
    assert torch.equal(qf, qo) and torch.equal(kf, ko) and torch.equal(far[off:], cache)


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (BF16, 128), (F16, 64), (F16, 256)])
@pytest.mark.parametrize("m", [2, 9, 33])
def test_tree_attention_and_keep_far_pages(vla, dtype, hd, m):
    """Rows and pages behind 2^31 elements and 2^32 bytes give the bits that they give near, in each of the forms."""
    n_q, n_kv, page, lens, new = 6, 2, 64, [200, 700], [2, m]
    q, cache, table, _, _ = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=hd + m)
    _, see = _masks(new, 4, 5)
    see, total = see.to(DEV), sum(new)
    need = vla.kv4_tree_attention_work_bytes(total, 2, m, 700, n_q, n_kv, hd)
    work = torch.empty(max(16, need), dtype=torch.uint8, device=DEV)

    def run(out, q, cache, table):
        vla.kv4_tree_attention_dev(out, q, cache, n_q, n_kv, hd, page, hd ** -0.5, table, _i32(lens), _i32(_starts(new)), see, m, 700, work)
        return out

    near = run(torch.empty_like(q, device=DEV), q.to(DEV), cache, table)
    nb = cache.shape[1]
    far = torch.empty((2 ** 32 + 2 ** 20) // nb + cache.shape[0], nb, dtype=torch.uint8, device=DEV)
    off = far.shape[0] - cache.shape[0]
    far[off:].copy_(cache)
    there = torch.where(table >= 0, table + off, table)
    ld = (2 ** 31 // (total - 1) + 64) // 16 * 16
    out = _far_rows(torch.zeros_like(q), ld)
    assert torch.equal(run(out, _far_rows(q, ld), far, there), near)
    path, count = _i32([1, 0] + list(range(m - 1, -1, -1))), _i32([1, 1])
    for c, t in ((cache, table), (far, there)):
        vla.kv4_keep_dev(c, n_kv, hd, page, t, _i32(lens), _i32(_starts(new)), path, count)
    assert torch.equal(far[off:], cache)


@pytest.mark.parametrize("sampled", [True, False])
def test_verify_far_rows(vla, sampled):
    g, r = _gen(81), random.Random(81)
    for dtype in (BF16, F32):
        p, q, tokens, parent, start, u, un = _drafts(g, r, [4, 1, 5], 999, dtype, 2, sampled)
        want = dref.verify(p, q, tokens, parent, start, u, un)
        ld = 2 ** 31 // 9 + 5
        path, count, token = (torch.empty(k, dtype=torch.int32, device=DEV) for k in (10, 3, 3))
        vla.verify_drafts_dev(path, count, token, _far_rows(p, ld), _i32(tokens), _i32(start), u.to(DEV), un.to(DEV), _i32(parent),
                              _far_rows(q, ld) if sampled else None)
        assert (path.tolist(), count.tolist(), token.tolist()) == want


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_verify_many_refused(vla, dtype):
    """A hundred drafted tokens refused at the root, some of them twice, the last values of the vocabulary among them."""
    n, V = 101, 1003
    g = _gen(91)
    p = torch.softmax(torch.randn(n, V, generator=g), -1).to(dtype)
    tokens = [0] + [V - 1 - (i % 80) for i in range(n - 1)]
    parent, u = [-1] + [0] * (n - 1), torch.full((n,), 1.0 - 2.0 ** -20)
    for un in (0.0, 0.5, 1.0 - 2.0 ** -24):
        case = (p, None, tokens, parent, [0, n], u, torch.tensor([un]))
        want = dref.verify(*case)
        assert want[1] == [1] and want[2][0] not in tokens[1:]
        assert _verify(vla, *case) == want
        assert _verify(vla, *case, pad=5, shift=3) == want


# ------------------------------------------------------------ as one step --

def _step(vla, b):
    """A step with drafted tokens: positions and masks, rows into the cache, attention, the choice, what is kept."""
    vla.draft_tree_dev(b["pos"], b["see"], b["parent"], b["lens"], b["start"])
    vla.rope_kv4_append_dev(b["q_rot"], b["cache"], b["q"], b["k"], b["v"], b["n_q"], b["n_kv"], b["hd"], b["page"], b["table"], b["lens"], b["start"],
                            b["freqs"], pos=b["pos"], interleaved=b["inter"], magnitude=b["mag"])
    vla.kv4_tree_attention_dev(b["out"], b["q_rot"], b["cache"], b["n_q"], b["n_kv"], b["hd"], b["page"], b["scale"], b["table"], b["lens"], b["start"],
                               b["see"], b["max_new"], b["max_len"], b["work"])
    vla.verify_drafts_dev(b["path"], b["count"], b["token"], b["p"], b["tokens"], b["start"], b["u"], b["u_next"], b["parent"], b["qp"])
    vla.kv4_keep_dev(b["cache"], b["n_kv"], b["hd"], b["page"], b["table"], b["lens"], b["start"], b["path"], b["count"], b["new_lens"])


def _step_case(vla, dtype, seed, new=(9, 1, 20, 0, 6), past=(40, 0, 1500, 3, 70)):
    n_q, n_kv, hd, page, V = 6, 2, 64, 32, 211
    g, r = _gen(seed), random.Random(seed)
    new, past = list(new), list(past)
    lens = [a + b for a, b in zip(new, past)]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=seed)
    k, v = (_rows(g, sum(new), n_kv * hd, dtype) for _ in range(2))
    p, qp, tokens, parent, start, u, un = _drafts(g, r, new, V, F32, 3, True, far=0.4)
    f, mag = vla.rope_freqs(32, 10000.0, "parts", 4.0, 512.0)
    host = dict(q=q, k=k, v=v, p=p, qp=qp, tokens=tokens, parent=parent, start=start, u=u, un=un, ks=ks, vs=vs, lens=lens, new=new, past=past,
                f=torch.from_numpy(f), mag=mag, table=table.cpu())
    total = sum(new)
    b = dict(n_q=n_q, n_kv=n_kv, hd=hd, page=page, scale=0.125, inter=True, mag=mag, max_new=max(new), max_len=max(lens), cache=cache, table=table,
             freqs=torch.from_numpy(f).to(DEV), q=q.to(DEV), k=k.to(DEV), v=v.to(DEV), p=p.to(DEV), qp=qp.to(DEV), tokens=_i32(tokens), parent=_i32(parent),
             start=_i32(start), u=u.to(DEV), u_next=un.to(DEV), lens=_i32(lens))
    b.update(pos=torch.empty(total, dtype=torch.int32, device=DEV), see=torch.empty(total, 1, dtype=torch.int32, device=DEV),
             path=torch.empty(total, dtype=torch.int32, device=DEV), q_rot=torch.empty_like(b["q"]), out=torch.empty_like(b["q"]),
             **{n: torch.empty(len(new), dtype=torch.int32, device=DEV) for n in ("count", "token", "new_lens")})
    nb = vla.kv4_tree_attention_work_bytes(total, len(new), b["max_new"], b["max_len"], n_q, n_kv, hd)
    b["work"] = torch.empty(max(16, nb), dtype=torch.uint8, device=DEV)
    return host, b


def _check_step(vla, host, b):
    n_q, n_kv, hd, page = b["n_q"], b["n_kv"], b["hd"], b["page"]
    truth, depth = [], []
    for s, n in enumerate(host["new"]):
        bits, d = dref.tree(host["parent"][host["start"][s]:host["start"][s + 1]], n)
        truth.append(_truth(bits, n))
        depth += [host["past"][s] + x for x in d]
    pos = torch.tensor(depth, dtype=torch.int32)
    assert torch.equal(b["pos"].cpu(), pos)
    qr, mag = dref.rotated(host["q"], n_q, hd, pos, host["f"], host["mag"], True, None, 0.0)
    dtype = host["q"].dtype
    ref.within(b["q_rot"], qr.flatten(1), (ref.rounding(qr, dtype) + 28 * ref.U * mag).flatten(1), "q")
    kr, _ = dref.rotated(host["k"], n_kv, hd, pos, host["f"], host["mag"], True, None, 0.0)
    quant = lambda x: ref.values(*ref.quantize(x.reshape(-1, n_kv, hd)))
    kq, vq = quant(kr), quant(host["v"])
    ks, vs = [], []
    for s, n in enumerate(host["new"]):
        sl = slice(host["start"][s], host["start"][s + 1])
        ks.append(torch.cat([host["ks"][s][:host["past"][s]], kq[sl]]))
        vs.append(torch.cat([host["vs"][s][:host["past"][s]], vq[sl]]))
    want, bound = dref.attend(b["q_rot"].cpu(), ks, vs, host["new"], truth, n_q, n_kv, hd, b["scale"])
    ref.within(b["out"], want, bound, "attention")
    path, count, token = dref.verify(host["p"], host["qp"], host["tokens"], host["parent"], host["start"], host["u"], host["un"])
    assert (b["path"].tolist(), b["count"].tolist(), b["token"].tolist()) == (path, count, token)
    new_lens = [a + c for a, c in zip(host["past"], count)]
    assert b["new_lens"].tolist() == new_lens
    kb, vb = (torch.empty(sum(new_lens), n_kv * hd, dtype=F32, device=DEV) for _ in range(2))
    vla.kv4_gather_dev(kb, vb, b["cache"], n_kv, hd, page, b["table"], _i32(_starts(new_lens)))
    at = 0
    for s, c in enumerate(count):
        kept = [host["past"][s] + x for x in path[host["start"][s]:host["start"][s] + c]]
        for x, got in ((ks[s], kb), (vs[s], vb)):
            assert torch.equal(got[at:at + new_lens[s]].cpu().double(), torch.cat([x[:host["past"][s]], x[kept]]).flatten(1))
        at += new_lens[s]


@pytest.mark.parametrize("dtype", TYPES)
def test_draft_step(vla, dtype):
    """A whole step as a decoder runs it, each part against the plain form of what the one before left."""
    host, b = _step_case(vla, dtype, 21)
    _step(vla, b)
    torch.cuda.synchronize()
    _check_step(vla, host, b)


def test_draft_step_graphs_and_streams(vla):
    """Two steps captured on a stream of their own that share a workspace, replayed with eager steps between: each replay
    follows new inputs and gives the eager bits."""
    cases = [_step_case(vla, BF16, 31), _step_case(vla, BF16, 32)]
    room = max(b["work"].numel() for _, b in cases)
    work = torch.empty(room, dtype=torch.uint8, device=DEV)
    clean = [b["cache"].clone() for _, b in cases]
    st = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for _, b in cases:
        b["work"] = work
        with torch.cuda.stream(st):
            _step(vla, b)  # (the first calls load code)
        st.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            _step(vla, b)
        graphs.append(gr)
    for turn in range(3):
        for i, (host, b) in enumerate(cases):
            other = _step_case(vla, BF16, 40 + turn * 2 + i)
            for n in ("q", "k", "v", "p", "qp", "u", "u_next", "tokens", "parent"):
                b[n].copy_(other[1][n])
            for n in ("q", "k", "v", "p", "qp", "tokens", "parent", "u", "un"):
                host[n] = other[0][n]
            b["cache"].copy_(clean[i])
            eager = dict(b, cache=clean[i].clone(), **{n: torch.empty_like(b[n]) for n in ("pos", "see", "path", "q_rot", "out", "count", "token", "new_lens")})
            _step(vla, eager)
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            for n in ("pos", "see", "path", "q_rot", "out", "count", "token", "new_lens", "cache"):
                assert torch.equal(b[n], eager[n]), (turn, i, n)
            _check_step(vla, host, b)


def test_draft_steps_on_two_streams(vla):
    """Two steps at once, each with a workspace of its own."""
    cases = [_step_case(vla, F16, 51), _step_case(vla, F16, 52)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    clean = [b["cache"].clone() for _, b in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        for (_, b), st, c in zip(cases, streams, clean):
            with torch.cuda.stream(st):
                b["cache"].copy_(c)
                _step(vla, b)
    torch.cuda.synchronize()
    for host, b in cases:
        _check_step(vla, host, b)


def test_repeated_steps_give_the_same_bits(vla):
    host, b = _step_case(vla, F32, 61)
    clean = b["cache"].clone()
    first = None
    for _ in range(4):
        b["cache"].copy_(clean)
        b["work"].random_(0, 255)
        _step(vla, b)
        got = [b[n].clone() for n in ("out", "q_rot", "cache", "path", "token")]
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(first, got))
