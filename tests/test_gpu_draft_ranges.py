"""GPU tests of the operators around drafted tokens where values leave the middle of their range: attention's weights
bit by bit, scores past 2^24 and below -1e30, small weights beside a sink, infinities under a norm; and their forms for
many rows."""

import math
import random

import pytest
import torch

import draft_ref as dref
import serving_ref as ref
from test_gpu_draft import _append_case, _attend, _masks
from test_gpu_serving import BF16, DEV, F16, F32, TYPES, _decode_case, _dev, _gen, _i32, _rows, _starts

pytestmark = pytest.mark.gpu


def _put(vla, cache, table, hd, page, t, part, codes=None, byte=None, block=0, head=0, n_kv=1):
    """Codes (32, each of 4 bits) and scale byte of a cached block, in a host copy of the cache."""
    row, flat = table.cpu().numpy()[0], cache.view(-1)
    if codes is not None:
        at = vla.kv4_offset(row, n_kv, hd, page, cache.shape[0], t, part, head, block)
        flat[at:at + 16] = torch.tensor([codes[2 * i] | codes[2 * i + 1] << 4 for i in range(16)], dtype=torch.uint8)
    if byte is not None:
        flat[vla.kv4_offset(row, n_kv, hd, page, cache.shape[0], t, part + 2, head, block)] = byte


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n_q,n_kv,hd,m", [(4, 1, 64, 3), (4, 1, 64, 40), (32, 8, 128, 32), (8, 1, 32, 60), (6, 2, 96, 50), (2, 1, 256, 40)])
def test_tree_attention_weights_keep_16_bits(vla, dtype, n_q, n_kv, hd, m):
    """Rows that see two keys of nearly equal weight and opposite values: what is left shows the weights' bits.

    A weight is off by at most 2^-15 of itself, whatever form takes the call: bf16 in two parts of 8 bits, cut off; fp16 in two
    parts leaves 2^-22, or where the rest is a subnormal number 2^-25 against 2^9 for the row's largest, 2^-34 of that."""
    page = 32
    q, cache, table, ks, vs = _decode_case(vla, [m], [m], n_q, n_kv, hd, page, dtype, seed=m + hd)
    q = (q.float() / 16).to(dtype)  # scores a few hundredths apart
    c, v = cache.cpu(), vs[0].clone()
    for t in range(m):
        for h in range(n_kv):
            for b in range(hd // 32):
                _put(vla, c, table, hd, page, t, 1, [2 if t % 2 else 10] * 32, 127, b, h, n_kv)  # 1 or -1
        v[t] = 1.0 if t % 2 else -1.0
    truth, see = [torch.zeros(m, m, dtype=torch.bool)], torch.zeros(m, (m + 31) // 32, dtype=torch.int32)
    for i in range(m):
        bits = 1 << i | (1 << i - 1 if i else 0)
        truth[0][i, max(0, i - 1):i + 1] = True
        see[i] = dref.words([bits], see.shape[1])[0]
    G, scale = n_q // n_kv, hd ** -0.5
    for kw in (dict(), dict(split=False)):
        got = _attend(vla, q, c.to(DEV), table, [m], [m], see, n_q, n_kv, hd, page, scale, **kw)
        for h in range(n_q):
            cols = slice(h * hd, (h + 1) * hd)
            want, bound = ref.softmax_rows(q[:, cols].double(), ks[0][:, h // G], v[:, h // G], truth[0], scale, 2.0 ** -15 + 2.0 ** -34)
            ref.within(got[:, cols], want, bound + ref.rounding(want, dtype), f"head {h} {kw}")


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_attention_repeats_itself(vla, dtype):
    """The same call gives the same bits, with other work between the calls."""
    n_q, n_kv, hd, page = 32, 8, 128, 64
    r = random.Random(3)
    new = [32] * 10 + [0, 1]
    lens = [n + r.randrange(0, 2500) for n in new]
    q, cache, table, ks, vs = _decode_case(vla, lens, new, n_q, n_kv, hd, page, dtype, seed=4)
    truth, see = _masks(new, 8, 9)
    outs = []
    for i in range(6):
        outs.append(_attend(vla, q, cache, table, lens, new, see, n_q, n_kv, hd, page, hd ** -0.5).clone())
        _attend(vla, q[:sum(new[:3 + i])], cache, table[:3 + i], lens[:3 + i], new[:3 + i], see[:sum(new[:3 + i])], n_q, n_kv, hd, page, 0.3)
    assert all(torch.equal(outs[0], x) for x in outs[1:])


def _large_scores(vla, dtype, hd, m, sign, e, n):
    """Scores past 2^24, where a step of fp32 is 2 and more. They are whole steps s * 2^e + d with the scale's product with log2 e
    exactly 1, so that products, sums and differences are exact and weights depend on d alone: a result has no share of the bound
    for rounded scores."""
    n_q, n_kv, page = 4, 1, 64
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=e)
    scale = float(torch.tensor(math.log(2.0), dtype=torch.float32))  # times log2 e, in fp32: 1
    step = 2.0 ** max(0, e - 23)
    c, k, r = cache.cpu(), torch.zeros(n, 1, hd, dtype=torch.float64), random.Random(e)
    for t in range(n):  # block 0: 32 times the same; block 1: the step in its first column
        step_code = r.choice([0, 2, 4, 5, 6, 7])
        for b in range(hd // 32):
            _put(vla, c, table, hd, page, t, 0, [2] * 32 if b == 0 else [step_code] + [0] * 31 if b == 1 else [0] * 32, 127 + (5 if b == 0 else 0), b)
        k[t, 0, :32], k[t, 0, 32] = 32.0, ref.GRID[step_code]
    q = torch.zeros(m, n_q * hd, dtype=torch.float64)
    for h in range(n_q):
        q[:, h * hd:h * hd + 32] = sign * 2.0 ** (e - 10)  # 32 columns of 2^5: 2^e (fp16 up to 2^15: 2^25 here, more below)
        q[:, h * hd + 32] = step
    if dtype == F16 and e > 25:  # larger keys instead: of blocks that fp16 takes, up to 2^8
        up = min(e - 25, 3)
        q[:, [h * hd + i for h in range(n_q) for i in range(32)]] /= 2.0 ** up
        k[:, :, :32] *= 2.0 ** up
        for t in range(n):
            _put(vla, c, table, hd, page, t, 2 - 2, None, 127 + 5 + up, 0)
        if e > 28:  # and of others
            q[:, [h * hd + i for h in range(n_q) for i in range(32)]] /= 2.0 ** 4
            k[:, :, :32] *= 2.0 ** 4
            for t in range(n):
                _put(vla, c, table, hd, page, t, 0, None, 127 + 5 + up + 4, 0)
    q = q.to(dtype)
    assert bool(torch.isfinite(q.double()).all())
    truth, see = _masks([m], 3, 7)
    full = torch.ones(m, n, dtype=torch.bool)
    full[:, n - m:] = truth[0]
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        got = _attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, scale, **kw).double().cpu()
        z = torch.where(full, (q[:, :hd].double() @ k[:, 0].T) * scale, -math.inf)
        w = torch.softmax(z, 1)
        want = (w @ vs[0][:, 0]).repeat(1, n_q)
        # the exponential's last bits, the sums' order, and the weights' own bits, of fp16 also 2^-18 of the largest of 64
        rel = (n + 24) * ref.U + (0.0 if dtype == F32 else 2.0 ** -15)
        low = 0.0 if dtype == F32 else 2.0 ** -18 * w.amax(1, keepdim=True) * vs[0][:, 0].abs().sum(0)
        bound = (w @ vs[0][:, 0].abs() * rel + low).repeat(1, n_q) + ref.rounding(want, dtype)
        ref.within(got, want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("e", [22, 24, 25, 26, 27, 28, 30])
def test_tree_attention_of_large_scores(vla, dtype, hd, m, sign, e):
    _large_scores(vla, dtype, hd, m, sign, e, 700)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("m", [3, 40])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("e", [24, 25, 27])
def test_tree_attention_of_large_scores_in_a_longer_table(vla, dtype, hd, m, sign, e):
    """The weights' scale is an odd power of two there, which a step of 2 does not take."""
    _large_scores(vla, dtype, hd, m, sign, e, 1300)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [32, 128, 256])
@pytest.mark.parametrize("m", [3, 40])
def test_tree_attention_of_scores_below_all_others(vla, dtype, hd, m):
    """Every score -2^105 (-4e31) or twice that: the mean over the former."""
    n_q, n_kv, page, n = 4, 1, 64, 500
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=11)
    c, r = cache.cpu(), random.Random(2)
    k = torch.zeros(n, 1, hd, dtype=torch.float64)
    up = 15 if dtype == F16 else 60
    for t in range(n):
        code = r.choice([2, 4])
        for b in range(hd // 32):
            _put(vla, c, table, hd, page, t, 0, [code] + [0] * 31 if b == 0 else [0] * 32, 127 + 105 - up if b == 0 else 127, b)
        k[t, 0, 0] = ref.GRID[code] * 2.0 ** (105 - up)
    q = torch.zeros(m, n_q * hd)
    q[:, ::hd] = -2.0 ** up
    q = q.to(dtype)
    truth, see = _masks([m], 3, 7)
    full = torch.ones(m, n, dtype=torch.bool)
    full[:, n - m:] = truth[0]
    w = torch.softmax(torch.where(full, q[:, :hd].double() @ k[:, 0].T, -math.inf), 1)
    want = (w @ vs[0][:, 0]).repeat(1, n_q)
    rel = (n + 24) * ref.U + (0.0 if dtype == F32 else 2.0 ** -15)
    bound = (w @ vs[0][:, 0].abs() * rel).repeat(1, n_q) + ref.rounding(want, dtype)
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        ref.within(_attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, 1.0, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("below", [38, 45, 52, 60])
@pytest.mark.parametrize("m", [3, 40])
def test_tree_attention_far_below_a_sink(vla, dtype, hd, below, m):
    """One key takes the weight of every row and has the value zero; the others' weights, down to e^-60, are what the result is made of."""
    n_q, n_kv, page, n = 4, 1, 64, 2000
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=below)
    c, k, v = cache.cpu(), ks[0].clone(), vs[0].clone()
    q = torch.zeros_like(q)
    q[:, ::hd] = 1.0  # a row's score is its key's first value
    scale = below / 4.0
    for t in range(n):
        _put(vla, c, table, hd, page, t, 0, [6 if t == 0 else 0] + [0] * 31, 127)  # 4, the others 0
        k[t, 0, :32] = 0.0
    k[0, 0, 0], v[0] = 4.0, 0.0
    for b in range(hd // 32):
        _put(vla, c, table, hd, page, 0, 1, [0] * 32, None, b)
    truth, see = _masks([m], 3, 7)
    full = torch.ones(m, n, dtype=torch.bool)
    full[:, n - m:] = truth[0]
    w = torch.softmax(torch.where(full, q[:, :hd].double() @ k[:, 0].T * scale, -math.inf), 1)
    want = (w @ v[:, 0]).repeat(1, n_q)
    # The scores are exact but for the scale's three roundings: 2 * 3 u of `below`. Weights: 2^-15 of themselves, or 2^-18 of the
    # largest among the 64 neighbours, as all of them are. Of those beside the sink that leaves nothing.
    rel = (n + 24) * ref.U + 6 * ref.U * below + (0.0 if dtype == F32 else 2.0 ** -15 + 2.0 ** -18)
    near = w.clone()
    near[:, 64:] = 0.0
    bound = (w @ v[:, 0].abs() * rel + (0.0 if dtype == F32 else near @ v[:, 0].abs())).repeat(1, n_q) + ref.rounding(want, dtype)
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        ref.within(_attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, scale, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("below", [30, 45, 60])
@pytest.mark.parametrize("late", [777, 1470, 1499])
def test_tree_attention_far_below_sinks_of_some_rows(vla, dtype, below, late):
    """Sinks for some rows at the first key, for others at a later one, for the rest none: what one wave of a block leaves to the
    other form the others have done."""
    n_q, n_kv, hd, page, n, m = 4, 1, 64, 64, 1500, 40
    q, cache, table, ks, vs = _decode_case(vla, [n], [m], n_q, n_kv, hd, page, dtype, seed=below)
    c, k, v = cache.cpu(), torch.zeros(n, 1, hd, dtype=torch.float64), vs[0].clone()
    q = torch.zeros_like(q)
    q[:16, ::hd], q[16:32, 1::hd] = 1.0, 1.0
    scale = below / 4.0
    for t in range(n):
        for b in range(2):
            _put(vla, c, table, hd, page, t, 0, [6 if t == 0 and b == 0 else 0, 6 if t == late and b == 0 else 0] + [0] * 30, 127, b)
    k[0, 0, 0] = k[late, 0, 1] = 4.0
    for t in (0, late):
        v[t] = 0.0
        for b in range(2):
            _put(vla, c, table, hd, page, t, 1, [0] * 32, None, b)
    truth, see = torch.ones(m, m, dtype=torch.bool), torch.full((m, 2), -1, dtype=torch.int32)
    truth[5, 3:], see[5] = False, torch.tensor([7, 0])
    full = torch.ones(m, n, dtype=torch.bool)
    full[:, n - m:] = truth
    w = torch.softmax(torch.where(full, q[:, :hd].double() @ k[:, 0].T * scale, -math.inf), 1)
    want = (w @ v[:, 0]).repeat(1, n_q)
    # as above; the largest of 64 neighbours lies in the tile of 32 or one beside it
    tiles = torch.nn.functional.pad(w, (0, -n % 32)).unflatten(1, (-1, 32)).amax(-1)
    near = torch.stack([torch.nn.functional.pad(tiles, (1, 1))[:, i:i + tiles.shape[1]] for i in range(3)]).amax(0).repeat_interleave(32, 1)[:, :n]
    rel = (n + 24) * ref.U + 6 * ref.U * below + (0.0 if dtype == F32 else 2.0 ** -15)
    lost = 0.0 if dtype == F32 else torch.minimum(w, 2.0 ** -18 * near) @ v[:, 0].abs()
    bound = (w @ v[:, 0].abs() * rel + lost).repeat(1, n_q) + ref.rounding(want, dtype)
    for kw in (dict(), dict(max_len=1 << 20), dict(split=False)):
        ref.within(_attend(vla, q, c.to(DEV), table, [n], [m], see, n_q, n_kv, hd, page, scale, **kw), want, bound, str(kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,inter", [(64, False), (128, True), (192, False)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_rope_append_infinities_under_a_norm(vla, dtype, hd, inter, bad):
    """A row with an infinity has an infinite norm: its finite values become zeros, the infinite one and the other of its pair NaN, in
    queries and in keys; a NaN makes the whole head NaN."""
    new, n_q, n_kv, page, rot = [6], 2, 2, 32, 32
    q, k, v, lens, table, cache = _append_case(vla, new, 0, n_q, n_kv, hd, page, dtype, 8)
    w = torch.full((hd,), 1.5)
    q[1, 3], k[2, hd + 5], k[4, 0] = bad, bad, bad
    pos = torch.tensor([3, 7, 11, 0, 2, 900], dtype=torch.int32)
    f = dref.freqs(rot)
    qo, ko = torch.empty_like(q, device=DEV), torch.empty_like(k, device=DEV)
    vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), _i32([0, 6]), f.to(DEV),
                            pos=pos.to(DEV), interleaved=inter, q_weight=w.to(DEV), k_weight=w.to(DEV), k_out=ko)
    for name, x, got, heads in (("q", q, qo, n_q), ("k", k, ko, n_kv)):
        want, mag = dref.rotated(x, heads, hd, pos, f, 1.0, inter, w, 1e-6)
        assert int(want.isnan().sum()) > 0
        mag = torch.where(torch.isfinite(mag), mag, torch.zeros_like(mag))
        bound = ref.rounding(torch.where(want.isnan(), torch.zeros_like(want), want), dtype) + 28 * ref.U * mag
        ref.within(got, want.flatten(1), bound.flatten(1), name)
    kr, _ = dref.rotated(k, n_kv, hd, pos, f, 1.0, inter, w, 1e-6)
    kb, vb = (torch.empty(6, n_kv * hd, dtype=F32, device=DEV) for _ in range(2))
    vla.kv4_gather_dev(kb, vb, cache, n_kv, hd, page, table.to(DEV), _i32([0, 6]))
    ref.within(kb, ref.values(*ref.quantize(kr)).flatten(1), torch.zeros(6, n_kv * hd, dtype=torch.float64), "cached")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,rot,inter,norm,rows", [
    (4, 2, 64, 64, False, True, 5000), (2, 1, 96, 48, True, True, 3000), (3, 1, 192, 176, False, True, 2600), (1, 1, 128, 128, True, False, 7000),
    (2, 2, 32, 24, False, True, 14000), (1, 1, 32, 16, True, True, 14000), (2, 1, 256, 64, False, False, 2000), (6, 2, 96, 96, False, False, 2500),
])
def test_rope_append_forms_of_many_rows(vla, dtype, n_q, n_kv, hd, rot, inter, norm, rows):
    """Two to sixteen tokens a block, in every form: norms, neighbours, part of a head, heads whose lanes a group does not fill,
    keys as rows, in place; positions given and of the sequences themselves."""
    r = random.Random(hd + rot)
    page, past, new = 64, 5, []
    while sum(new) < rows:
        new.append(r.choice([0, 1, 2, 17, 130, 900]))
    q, k, v, lens, table, cache = _append_case(vla, new, past, n_q, n_kv, hd, page, dtype, 5)
    total, g = sum(new), _gen(rot)
    wq, wk = (1 + 0.2 * torch.randn(hd, generator=g) if norm else None for _ in range(2))
    pos = torch.cat([torch.arange(past, past + n) for n in new]).to(torch.int32)
    f, mag = dref.freqs(rot), 1.25
    kr, kmag = dref.rotated(k, n_kv, hd, pos, f, mag, inter, wk, float(torch.tensor(1e-5)))
    qr, qmag = dref.rotated(q, n_q, hd, pos, f, mag, inter, wq, float(torch.tensor(1e-5)))
    start, codes = _starts(new), ref.values(*ref.quantize(kr)).flatten(1)
    vals = ref.values(*ref.quantize(v.reshape(total, n_kv, hd))).flatten(1)
    for given in (pos.to(DEV), None):
        cache.fill_(0xEE)
        dq, dk, qo, ko = q.to(DEV), k.to(DEV), torch.full_like(q, 5.0, device=DEV), torch.full_like(k, 5.0, device=DEV)
        args = (v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), _i32(start), f.to(DEV), given, mag, inter, _dev(wq), _dev(wk), 1e-5)
        vla.rope_kv4_append_dev(qo, cache, dq, dk, *args, k_out=ko)
        ref.within(ko, kr.flatten(1), (ref.rounding(kr, dtype) + 2.0 ** -30 * kmag).flatten(1), "k")
        ref.within(qo, qr.flatten(1), (ref.rounding(qr, dtype) + 28 * ref.U * qmag).flatten(1), "q")
        kb, vb = (torch.empty(total, n_kv * hd, dtype=F32, device=DEV) for _ in range(2))
        vla.kv4_gather_dev(kb, vb, cache, n_kv, hd, page, table.to(DEV), _i32(start), _i32([past] * len(new)))
        assert torch.equal(kb.cpu().double(), codes) and torch.equal(vb.cpu().double(), vals)
        again = torch.full_like(cache, 0xEE)
        vla.rope_kv4_append_dev(dq, again, dq, dk, *args, k_out=dk)
        assert torch.equal(dq, qo) and torch.equal(dk, ko) and torch.equal(again, cache)


@pytest.mark.parametrize("n_seqs", [1023, 1024, 3000])
def test_rope_append_many_sequences(vla, n_seqs):
    """Offsets that LDS has room for, and more, searched where they are."""
    r = random.Random(n_seqs)
    n_q, n_kv, hd, page, past, dtype = 2, 1, 32, 32, 3, BF16
    new = [r.choice([0, 1, 1, 2, 5]) for _ in range(n_seqs)]
    q, k, v, lens, table, cache = _append_case(vla, new, past, n_q, n_kv, hd, page, dtype, 6)
    total, start = sum(new), _starts(new)
    pos = torch.cat([torch.arange(past, past + n) for n in new]).to(torch.int32)
    f = dref.freqs(hd)
    kr, _ = dref.rotated(k, n_kv, hd, pos, f, 1.0, False, None, 0.0)
    qr, qmag = dref.rotated(q, n_q, hd, pos, f, 1.0, False, None, 0.0)
    for given in (pos.to(DEV), None):
        cache.fill_(0xEE)
        qo = torch.empty_like(q, device=DEV)
        vla.rope_kv4_append_dev(qo, cache, q.to(DEV), k.to(DEV), v.to(DEV), n_q, n_kv, hd, page, table.to(DEV), _i32(lens), _i32(start), f.to(DEV), pos=given)
        ref.within(qo, qr.flatten(1), (ref.rounding(qr, dtype) + 28 * ref.U * qmag).flatten(1), "q")
        kb, vb = (torch.empty(total, n_kv * hd, dtype=F32, device=DEV) for _ in range(2))
        vla.kv4_gather_dev(kb, vb, cache, n_kv, hd, page, table.to(DEV), _i32(start), _i32([past] * n_seqs))
        assert torch.equal(kb.cpu().double(), ref.values(*ref.quantize(kr)).flatten(1))
        assert torch.equal(vb.cpu().double(), ref.values(*ref.quantize(v.reshape(total, n_kv, hd))).flatten(1))


@pytest.mark.parametrize("new", [[700, 513], [64, 512, 3, 1469], [512], [513], [1024, 0, 1]])
@pytest.mark.parametrize("words", [1, 16, 17, 46, 50])
def test_tree_of_long_sequences(vla, new, words):
    """Averages on both sides of 512 rows: parents of all kinds, further roots, too few and too many words."""
    r = random.Random(sum(new))
    parents = []
    for n in new:
        p = [-1 if i == 0 else r.choice([i - 1, i - 1, i - 1, max(0, i - 70), r.randrange(i)]) for i in range(n)]
        for i, x in ((n // 3, -1), (n // 2, n // 2), (2 * n // 3, 2 ** 31 - 1), (n - 1, -(2 ** 31))) if n > 9 else ():
            p[i] = x
        parents.append(p)
    lens, start, total = [n + 11 for n in new], _starts(new), sum(new)
    for parent in (parents, None):
        pos = torch.full((total + 2,), 77, dtype=torch.int32, device=DEV)
        see = torch.full((total + 2, words), 77, dtype=torch.int32, device=DEV)
        vla.draft_tree_dev(pos, see, _i32([x for p in parents for x in p] + [0, 0]) if parent else None, _i32(lens), _i32(start))
        for s, n in enumerate(new):
            bits, depth = dref.tree(parents[s] if parent else None, n)
            assert pos[start[s]:start[s + 1]].tolist() == [11 + d for d in depth]
            assert torch.equal(see[start[s]:start[s + 1]].cpu(), dref.words(bits, words)) or n == 0
        assert bool((pos[total:] == 77).all()) and bool((see[total:] == 77).all())


