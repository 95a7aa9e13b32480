"""CPU checks of the operators around drafted tokens: what the C ABI and the Python face
refuse before any device work, and the frequencies of scaled rotations."""

import ctypes
import math

import numpy as np
import pytest
import torch

import draft_ref as dref
from helpers import load_pkg

P = 1 << 20  # an aligned address; refused calls never read it
I32 = torch.int32


@pytest.fixture(scope="module")
def vla():
    return load_pkg()


ORDER = {
    "vla_draft_tree_dev": "pos see ld_see parent lens start n total",
    "vla_rope_kv4_append_dev": "qo ldqo ko ldko cache pages page q ldq k ldk v ldv wq wk eps pos freqs rot mag inter table ld lens start n total n_q "
                               "n_kv hd dtype",
    "vla_kv4_tree_attention_dev": "out ldo q ldq cache pages page table ld lens start see ld_see n total max_new max_len n_q n_kv hd scale dtype work wb",
    "vla_verify_drafts_dev": "path count token p ldp qp ldqp tokens parent start u u_next n total vocab dtype",
    "vla_kv4_keep_dev": "cache pages page table ld lens start path count new_lens n total n_kv hd",
}


def _refused(vla, name, kw):
    a = dict(pos=P, see=P, ld_see=1, parent=None, lens=P, start=P, n=2, total=8, qo=P, ldqo=256, ko=None, ldko=128, cache=P, pages=4, page=64, q=P,
             ldq=256, k=P, ldk=128, v=P, ldv=128, wq=None, wk=None, eps=1e-6, freqs=P, rot=64, mag=1.0, inter=0, table=P, ld=2, n_q=4, n_kv=2, hd=64,
             dtype=1, out=P, ldo=256, max_new=4, max_len=64, scale=0.1, work=None, wb=0, path=P, count=P, token=P, p=P, ldp=100, qp=P, ldqp=100, tokens=P,
             u=P, u_next=P, vocab=100, new_lens=None)
    a.update(kw)
    st = getattr(vla.lib(), name)(*[a[x] for x in ORDER[name].split()], None)
    assert st == vla.VLA_ERR_ARG, st
    return vla.lib().vla_last_error().decode()


@pytest.mark.parametrize("kw,msg", [
    (dict(n=-1), "2^28"), (dict(total=-1), "2^28"), (dict(total=2 ** 28 + 1), "2^28"), (dict(n=2 ** 28 + 1), "2^28"), (dict(ld_see=0), "words"),
    (dict(ld_see=2 ** 20 + 1), "words"), (dict(pos=None), "null"), (dict(see=None), "null"), (dict(lens=None), "null"), (dict(start=None), "null"),
])
def test_tree_refusals(vla, kw, msg):
    assert msg in _refused(vla, "vla_draft_tree_dev", kw)


CACHE = [
    (dict(n=-1), "n_seqs"), (dict(n_kv=0), "kv heads"), (dict(n_kv=1025), "kv heads"), (dict(hd=48), "head_dim"), (dict(page=48), "page_size"),
    (dict(page=4096), "page_size"), (dict(ld=2 ** 30), "2^30"), (dict(pages=0), "hold a page"), (dict(cache=P + 8), "aligned"), (dict(table=None), "table"),
    (dict(ld=0), "table"), (dict(total=2 ** 31 - 1), "2^28"),
]


@pytest.mark.parametrize("kw,msg", CACHE + [
    (dict(dtype=3), "dtype"), (dict(total=1 << 26), "2^26"), (dict(n_q=-1), "query heads"), (dict(n_q=70000), "query heads"), (dict(rot=4), "rot_dim"),
    (dict(rot=72), "rot_dim"), (dict(rot=-8), "rot_dim"), (dict(mag=math.inf), "magnitude"), (dict(mag=math.nan), "magnitude"), (dict(eps=-1.0), "eps"),
    (dict(lens=None), "lens"), (dict(start=None), "start"), (dict(freqs=None), "frequencies"), (dict(k=None), "keys missing"), (dict(ldk=120), "stride"),
    (dict(k=P + 2), "aligned"), (dict(v=None), "values missing"), (dict(ldv=132), "aligned"), (dict(q=None), "queries missing"), (dict(qo=None), "q_out"),
    (dict(ldq=250), "stride"), (dict(ldqo=260), "aligned"), (dict(ko=P + 8), "k_out"), (dict(ko=P, ldko=64), "k_out"), (dict(cache=None, hd=80), "head_dim"),
])
def test_append_refusals(vla, kw, msg):
    assert msg in _refused(vla, "vla_rope_kv4_append_dev", kw)


@pytest.mark.parametrize("kw,msg", CACHE + [
    (dict(dtype=-1), "dtype"), (dict(n_q=5), "multiple"), (dict(n_q=1 << 26), "65536"), (dict(scale=math.nan), "scale"), (dict(max_new=0), "max_new"),
    (dict(max_new=-1), "max_new"), (dict(max_len=-1), "max_len"), (dict(ld_see=0), "words"), (dict(see=None), "null"), (dict(out=None), "null"),
    (dict(start=None), "q_start"), (dict(lens=None), "lens"), (dict(ldq=252), "stride"), (dict(ldo=260), "aligned"), (dict(q=P + 2), "aligned"),
    (dict(n=70000, total=70000), "65535"), (dict(total=2 ** 28, n_q=512, ldq=512 * 64, ldo=512 * 64), "too many"),
])
def test_attention_refusals(vla, kw, msg):
    assert msg in _refused(vla, "vla_kv4_tree_attention_dev", kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(n=-1), "n_seqs"), (dict(total=-1), "2^28"), (dict(total=2 ** 28 + 1), "2^28"), (dict(n=65536), "65535"),
    (dict(vocab=0), "vocabulary"), (dict(vocab=2 ** 30 + 1), "vocabulary"), (dict(count=None), "null"), (dict(token=None), "null"),
    (dict(start=None), "null"), (dict(u_next=None), "null"), (dict(path=None), "null"), (dict(p=None), "null"), (dict(tokens=None), "null"),
    (dict(u=None), "null"), (dict(ldp=99), "stride"), (dict(ldqp=99), "stride"), (dict(p=P + 1), "aligned"), (dict(qp=P + 1), "aligned"),
])
def test_verify_refusals(vla, kw, msg):
    assert msg in _refused(vla, "vla_verify_drafts_dev", kw)


@pytest.mark.parametrize("kw,msg", CACHE + [
    (dict(n=65536), "65535"), (dict(lens=None), "null"), (dict(start=None), "null"), (dict(count=None), "null"), (dict(path=None), "null"),
    (dict(new_lens=P), "new_lens"),
])
def test_keep_refusals(vla, kw, msg):
    if kw == dict(new_lens=P):
        kw = dict(new_lens=P, lens=P)
    assert msg in _refused(vla, "vla_kv4_keep_dev", kw)


def test_results_over_what_other_blocks_read(vla):
    assert "parent" in _refused(vla, "vla_draft_tree_dev", dict(pos=P, parent=P))
    assert "count" in _refused(vla, "vla_kv4_keep_dev", dict(new_lens=P, count=P, lens=P + 64))


def test_work_bytes(vla):
    n = vla.kv4_tree_attention_work_bytes
    assert n(64, 2, 32, 131072, 32, 8, 128) > 0
    for bad in ((0, 2, 32, 4096, 32, 8, 128), (64, 0, 32, 4096, 32, 8, 128), (64, 2, 32, 4096, 31, 8, 128), (64, 2, 32, 4096, 32, 8, 100),
                (64, 70000, 1, 4096, 32, 8, 128), (1 << 28, 2, 1 << 28, 4096, 32, 8, 128), (64, 2, 0, 4096, 32, 8, 128)):
        assert n(*bad) == 0


# ---------------------------------------------------------- frequencies --

@pytest.mark.parametrize("rot", [2, 8, 64, 96, 256])
def test_frequencies(vla, rot):
    i = np.arange(rot // 2)
    plain = 10000.0 ** (-2.0 * i / rot)
    f, m = vla.rope_freqs(rot)
    assert np.allclose(f, plain, rtol=1e-15, atol=0) and m == 1.0
    f, m = vla.rope_freqs(rot, 500000.0, "linear", 4.0)
    assert np.allclose(f, 500000.0 ** (-2.0 * i / rot) / 4, rtol=1e-15, atol=0) and m == 1.0
    if rot > 2:
        f, m = vla.rope_freqs(rot, 10000.0, "base", 8.0)
        # the slowest pair is slowed by the factor, the fastest not at all
        assert f[0] == 1.0 and abs(f[-1] * 8.0 / plain[-1] - 1) < 1e-12 and m == 1.0
    f, m = vla.rope_freqs(rot, 10000.0, "parts", 8.0, 4096, 1.0, 32.0)
    turns = 4096 * plain / (2 * math.pi)
    for a, b, t in zip(f, plain, turns):
        want = b if t >= 32 else b / 8 if t <= 1 else b * (t - 1) / 31 + b / 8 * (1 - (t - 1) / 31)
        assert abs(a / want - 1) < 1e-14
    assert abs(m - (0.1 * math.log(8.0) + 1)) < 1e-15
    assert np.array_equal(vla.rope_freqs(rot, 10000.0, "parts", 1.0, 4096)[0], vla.rope_freqs(rot)[0])


@pytest.mark.parametrize("args,msg", [
    ((0,), "rot_dim"), ((7,), "rot_dim"), ((8, 0.0), "base"), ((8, math.nan), "base"), ((8, 1e4, "linear", 0.5), "factor"), ((2, 1e4, "base", 2.0), "pair"),
    ((8, 1e4, "parts", 2.0), "trained"), ((8, 1e4, "parts", 2.0, 4096, 4.0, 4.0), "low"), ((8, 1e4, "parts", math.inf, 4096), "factor"),
])
def test_frequency_refusals(vla, args, msg):
    with pytest.raises(vla.VlaError, match=msg):
        vla.rope_freqs(*args)


def test_frequency_scalings_by_name(vla):
    with pytest.raises(ValueError, match="scaling"):
        vla.rope_freqs(8, 1e4, "cubic")


# ------------------------------------------------------ the Python face --

def _i(*shape):
    return torch.zeros(*shape, dtype=I32)


def test_tree_shapes(vla):
    good = dict(pos=_i(5), see=_i(5, 2), parent=_i(5), lens=_i(2), start=_i(3))
    for name, bad in (("pos", _i(5, 1)), ("pos", _i(5).long()), ("see", _i(4, 2)), ("see", _i(5, 4)[:, ::2]), ("see", torch.zeros(5, 0, dtype=I32)),
                      ("parent", _i(4)), ("lens", _i(3)), ("start", _i(3, 1)), ("start", torch.zeros(0, dtype=I32))):
        with pytest.raises(ValueError):
            vla.draft_tree_dev(**{**good, name: bad})


def test_append_shapes(vla):
    nb = vla.kv4_page_bytes(2, 64, 64)
    good = dict(q_out=torch.zeros(5, 256), cache=torch.zeros(4, nb, dtype=torch.uint8), q=torch.zeros(5, 256), k=torch.zeros(5, 128), v=torch.zeros(5, 128),
                n_q=4, n_kv=2, head_dim=64, page_size=64, table=_i(2, 2), lens=_i(2), start=_i(3), freqs=torch.zeros(32, dtype=torch.float64))
    for name, bad in (("q", torch.zeros(5, 255)), ("q", torch.zeros(4, 256)), ("q_out", torch.zeros(5, 256, dtype=torch.bfloat16)), ("k", torch.zeros(5, 100)),
                      ("v", torch.zeros(5, 128).half()), ("cache", torch.zeros(4, nb + 1, dtype=torch.uint8)), ("table", _i(3, 2)), ("lens", _i(3)),
                      ("freqs", torch.zeros(32)), ("freqs", torch.zeros(64, dtype=torch.float64)[::2]), ("pos", _i(4)), ("k_out", torch.zeros(5, 64)),
                      ("q_weight", torch.zeros(32)), ("k", torch.zeros(5, 128, dtype=torch.float64))):
        with pytest.raises(ValueError):
            vla.rope_kv4_append_dev(**{**good, name: bad})


def test_attention_shapes(vla):
    nb = vla.kv4_page_bytes(2, 64, 64)
    good = dict(out=torch.zeros(5, 256), Q=torch.zeros(5, 256), cache=torch.zeros(4, nb, dtype=torch.uint8), n_q=4, n_kv=2, head_dim=64, page_size=64,
                scale=0.1, table=_i(2, 2), lens=_i(2), q_start=_i(3), see=_i(5, 1), max_new=3)
    for name, bad in (("out", torch.zeros(4, 256)), ("Q", torch.zeros(5, 256).t()), ("see", _i(4, 1)), ("see", _i(5)), ("see", _i(5, 1).long()),
                      ("lens", _i(1)), ("q_start", _i(2)), ("work", torch.zeros(64)), ("table", _i(2, 2).long())):
        with pytest.raises(ValueError):
            vla.kv4_tree_attention_dev(**{**good, name: bad})


def test_verify_shapes(vla):
    good = dict(path=_i(5), count=_i(2), token=_i(2), p=torch.zeros(5, 30), tokens=_i(5), start=_i(3), u=torch.zeros(5), u_next=torch.zeros(2), q=torch.zeros(5, 30))
    for name, bad in (("path", _i(4)), ("count", _i(3)), ("token", _i(2).long()), ("p", torch.zeros(150)), ("p", torch.zeros(5, 30, dtype=torch.float64)),
                      ("p", torch.zeros(5, 60)[:, ::2]), ("q", torch.zeros(5, 31)), ("q", torch.zeros(5, 30).half()), ("tokens", _i(6)), ("start", _i(4)),
                      ("u", torch.zeros(4)), ("u", torch.zeros(5).double()), ("u_next", torch.zeros(3)), ("parent", _i(4))):
        with pytest.raises(ValueError):
            vla.verify_drafts_dev(**{**good, name: bad})


def test_keep_shapes(vla):
    nb = vla.kv4_page_bytes(2, 64, 64)
    good = dict(cache=torch.zeros(4, nb, dtype=torch.uint8), n_kv=2, head_dim=64, page_size=64, table=_i(2, 2), lens=_i(2), start=_i(3), path=_i(5), count=_i(2))
    for name, bad in (("cache", torch.zeros(4, nb)), ("table", _i(4)), ("lens", _i(1)), ("start", _i(2)), ("path", _i(5, 1)), ("count", _i(1)),
                      ("new_lens", _i(3))):
        with pytest.raises(ValueError):
            vla.kv4_keep_dev(**{**good, name: bad})


# ------------------------------------------- the plain forms on their own --

def test_plain_verification_keeps_the_targets_distribution():
    """Summed over every choice of the random numbers on a fine grid, the token behind the root has the target's share."""
    p, q = torch.tensor([[0.5, 0.25, 0.25]]), torch.tensor([[0.25, 0.75, 0.0]])
    share, steps = torch.zeros(3), 16
    for tok in range(3):
        for i in range(steps):
            for j in range(steps):
                path, count, nxt = dref.verify(p.repeat(2, 1), q.repeat(2, 1), [0, tok], None, [0, 2], torch.tensor([0.0, (i + 0.5) / steps]),
                                               torch.tensor([(j + 0.5) / steps]))
                share[tok if count[0] == 2 else nxt[0]] += float(q[0, tok]) / steps ** 2
    # u moves in steps of 1/16 of a refusal's probability
    assert float((share - p[0]).abs().max()) <= 1 / steps


def test_plain_tree():
    bits, depth = dref.tree([-1, 0, 0, 1, 3], 5)
    assert bits == [1, 3, 5, 11, 27] and depth == [0, 1, 1, 2, 3]
    assert dref.words([1 << 31 | 1, 1 << 32], 2).tolist() == [[-2 ** 31 + 1, 0], [0, 1]]
