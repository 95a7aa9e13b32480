"""CPU checks of the operators that serve several prompts: what the C ABI and the
Python face refuse before any device work, and the cache's layout and page lookup
(the functions the kernels use) over all tokens, bad pages among them."""

import ctypes

import numpy as np
import pytest
import torch

import serving_ref as ref
from helpers import load_pkg

I32 = torch.int32


@pytest.fixture(scope="module")
def vla():
    return load_pkg()


def _arg_error(vla, name, *args):
    st = getattr(vla.lib(), name)(*args)
    assert st == vla.VLA_ERR_ARG, (name, st)
    return vla.lib().vla_last_error().decode()


P = 1 << 20  # an aligned address; refused calls never read it


def _rope(vla, **kw):
    a = dict(qo=P, ldqo=128, ko=P, ldko=64, q=P, ldq=128, k=P, ldk=64, wq=None, wk=None, eps=1e-6, pos=P, ld_pos=4, sections=[32],
             base=1e4, seq=4, n_q=2, n_kv=1, hd=64, dtype=0)
    a.update(kw)
    s = (ctypes.c_int32 * max(1, len(a["sections"])))(*a["sections"])
    return _arg_error(vla, "vla_qk_norm_rope_dev", a["qo"], a["ldqo"], a["ko"], a["ldko"], a["q"], a["ldq"], a["k"], a["ldk"], a["wq"], a["wk"],
                      a["eps"], a["pos"], a["ld_pos"], s, len(a["sections"]), a["base"], a["seq"], a["n_q"], a["n_kv"], a["hd"], a["dtype"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(seq=-1), "seq"), (dict(seq=1 << 26), "2^26"), (dict(n_q=0, n_kv=0), "heads"),
    (dict(hd=0, sections=[0]), "head_dim"), (dict(hd=12, sections=[6]), "head_dim"), (dict(hd=264, sections=[132]), "head_dim"),
    (dict(sections=[31]), "sections"), (dict(sections=[16, 17]), "sections"), (dict(sections=[]), "axes"), (dict(sections=[4] * 9), "axes"),
    (dict(sections=[33, -1]), "section"), (dict(base=0.0), "base"), (dict(base=float("nan")), "base"), (dict(eps=-1.0), "eps"),
    (dict(pos=None), "positions"), (dict(ld_pos=3), "positions"), (dict(q=None), "null"), (dict(ko=None), "null"),
    (dict(ldq=127), "stride"), (dict(ldko=60), "stride"), (dict(q=P + 4), "aligned"), (dict(ldq=130), "aligned"), (dict(k=P + 8), "aligned"),
])
def test_rope_refusals(vla, kw, msg):
    assert msg in _rope(vla, **kw)


def _packed(vla, **kw):
    a = dict(out=P, ldo=128, q=P, ldq=128, k=P, ldk=64, v=P, ldv=64, qs=P, ks=P, n=2, tq=8, tk=8, n_q=2, n_kv=1, hd=64, scale=0.1, causal=1, dtype=1)
    a.update(kw)
    return _arg_error(vla, "vla_packed_attention_dev", a["out"], a["ldo"], a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["qs"], a["ks"],
                      a["n"], a["tq"], a["tk"], a["n_q"], a["n_kv"], a["hd"], a["scale"], a["causal"], a["dtype"], None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=5), "dtype"), (dict(n=-1), "n_seqs"), (dict(tq=-1), "total_q"), (dict(n_q=3, n_kv=2), "multiple"), (dict(n_kv=0), "n_kv"),
    (dict(hd=4), "head_dim"), (dict(hd=264), "head_dim"), (dict(hd=0), "head_dim"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(out=None), "null"), (dict(qs=None, ks=None), "null"), (dict(v=None), "null"),
    (dict(q=P + 2), "aligned"), (dict(ldk=65), "aligned"), (dict(ldo=120), "stride"), (dict(ldv=56), "stride"),
    (dict(tq=2 ** 31 - 1), "2^28"), (dict(tk=2 ** 28 + 1), "2^28"), (dict(n=2 ** 30), "2^28"), (dict(ldk=1 << 22), "2^22"),
    (dict(n_q=1 << 26, tq=1, n=1), "65536"),
    (dict(tq=2 ** 28, n=1, n_q=512, ldq=512 * 64, ldo=512 * 64), "too many"),
])
def test_packed_refusals(vla, kw, msg):
    assert msg in _packed(vla, **kw)


def _kv(vla, name, **kw):
    a = dict(cache=P, pages=4, page=64, k=P, ldk=128, v=P, ldv=128, table=P, ld=2, lens=P, start=P, first=None, n=2, total=8, n_kv=2, hd=64, dtype=1,
             out=P, ldo=256, q=P, ldq=256, max_new=1, max_len=64, n_q=4, scale=0.1, work=None, wb=0)
    a.update(kw)
    g = a.__getitem__
    if name == "append":
        args = map(g, "cache pages page k ldk v ldv table ld lens start n total n_kv hd dtype".split())
    elif name == "gather":
        args = map(g, "k ldk v ldv cache pages page table ld start first n total n_kv hd dtype".split())
    else:
        args = map(g, "out ldo q ldq cache pages page table ld lens start n total max_new max_len n_q n_kv hd scale dtype work wb".split())
    return _arg_error(vla, f"vla_kv4_{name}_dev", *args, None)


@pytest.mark.parametrize("name", ["append", "gather", "attention"])
@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype"), (dict(n=-1), "n_seqs"), (dict(n_kv=0), "kv heads"), (dict(hd=48), "head_dim"), (dict(hd=160), "head_dim"),
    (dict(page=0), "page_size"), (dict(page=48), "page_size"), (dict(page=4096), "page_size"), (dict(ld=2 ** 30), "2^30"),
    (dict(pages=-1), "2^30"), (dict(pages=0), "hold a page"), (dict(cache=None), "hold a page"), (dict(cache=P + 8), "aligned"),
    (dict(table=None), "table"), (dict(ld=0), "table"), (dict(total=2 ** 31 - 1), "2^28"), (dict(n=2 ** 28 + 1), "2^28"),
])
def test_cache_refusals(vla, name, kw, msg):
    assert msg in _kv(vla, name, **kw)


@pytest.mark.parametrize("name,kw,msg", [
    ("append", dict(lens=None), "lens"), ("append", dict(start=None), "null"), ("append", dict(k=None), "null"), ("append", dict(ldk=120), "stride"),
    ("append", dict(v=P + 2), "aligned"), ("gather", dict(v=None), "null"), ("gather", dict(ldv=132), "aligned"),
    ("attention", dict(n_q=5), "multiple"), ("attention", dict(scale=float("nan")), "scale"), ("attention", dict(max_new=0), "max_new"),
    ("attention", dict(max_len=-1), "max_len"), ("attention", dict(start=None, total=1), "one query row"), ("attention", dict(lens=None), "lens"),
    ("attention", dict(out=None), "null"), ("attention", dict(ldq=252), "stride"), ("attention", dict(q=P + 2), "aligned"),
    ("attention", dict(n=70000, total=70000), "65535"), ("attention", dict(n_q=1 << 26), "65536"),
])
def test_cache_call_refusals(vla, name, kw, msg):
    assert msg in _kv(vla, name, **kw)


def test_page_bytes_limits(vla):
    assert vla.kv4_page_bytes(5, 64, 64) == 5 * 64 * (64 + 4)
    for bad in ((0, 64, 64), (5, 48, 64), (5, 64, 48), (5, 64, 4096), (5, 288, 64)):
        with pytest.raises(ValueError):
            vla.kv4_page_bytes(*bad)


@pytest.mark.parametrize("n_kv,hd,page", [(1, 32, 32), (3, 64, 96), (2, 128, 64), (2, 256, 32)])
def test_every_cache_byte_belongs_to_one_token(vla, n_kv, hd, page):
    """All tokens' codes and scales tile the pages exactly, in any page order."""
    pages = 3
    row = [2, 0, 1]
    seen = np.zeros(pages * vla.kv4_page_bytes(n_kv, hd, page), np.int32)
    for tok in range(pages * page):
        for head in range(n_kv):
            for block in range(hd // 32):
                for part in range(4):
                    at = vla.kv4_offset(row, n_kv, hd, page, pages, tok, part, head, block)
                    assert 0 <= at and at // vla.kv4_page_bytes(n_kv, hd, page) == row[tok // page]
                    if part < 2:
                        assert at % 16 == 0
                        seen[at:at + 16] += 1
                    else:
                        seen[at] += 1
    assert np.all(seen == 1)


def test_bad_pages_have_no_address(vla):
    row = [1, -1, 4, 2 ** 31 - 1, -(2 ** 31), 3]
    def at(tok):
        return vla.kv4_offset(row, 2, 64, 32, 4, tok, 0, 0, 0)
    nb = vla.kv4_page_bytes(2, 64, 32)
    for tok in range(-40, 32 * 6 + 80):
        if 0 <= tok < 32:
            assert at(tok) // nb == 1
        elif 160 <= tok < 192:
            assert at(tok) // nb == 3
        else:
            assert at(tok) == -1, tok
    assert vla.kv4_offset(row, 2, 64, 32, 4, 0, 4, 0, 0) == -1
    assert vla.kv4_offset(row, 2, 64, 32, 4, 0, 0, 2, 0) == -1
    assert vla.kv4_offset(row, 2, 64, 32, 4, 0, 0, 0, 2) == -1
    assert vla.kv4_offset(row, 2, 64, 32, 4, 2 ** 40, 0, 0, 0) == -1


def test_offsets_pass_32_bits(vla):
    """A cache of more than 4 GiB: the last page's last scale byte is its last byte."""
    n_kv, hd, page, pages = 8, 128, 64, 70000
    nb = vla.kv4_page_bytes(n_kv, hd, page)
    at = vla.kv4_offset([pages - 1], n_kv, hd, page, pages, page - 1, 3, n_kv - 1, hd // 32 - 1)
    assert at == pages * nb - 1 > 2 ** 32


def test_reference_quantizer():
    """The tests' own quantizer: error at most half a step, exact on its grid."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, 128, generator=g) * torch.exp(torch.randn(64, 1, generator=g) * 4)
    code, byte = ref.quantize(x)
    v = ref.values(code, byte)
    s = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
    y = x.double().abs() / s
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    assert bool(((v - x.double()).abs() <= step / 2 * s).all())
    again = ref.values(*ref.quantize(v.float()))
    assert bool((again == v).all())


def test_wrapper_checks(vla):
    f = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt)
    pos = torch.zeros(1, 4, dtype=I32)
    def rope(**kw):
        a = dict(q_out=f(4, 128), k_out=f(4, 64), q=f(4, 128), k=f(4, 64), n_q=2, n_kv=1, head_dim=64, pos=pos, sections=[32], base=1e4)
        a.update(kw)
        vla.qk_norm_rope_dev(**a)
    for kw, msg in ((dict(q=f(4, 120)), "q:"), (dict(k=f(3, 64)), "k:"), (dict(q_out=f(4, 128, dt=torch.bfloat16)), "q_out"),
                    (dict(q=f(4, 128, dt=torch.int32)), "float32, bfloat16"), (dict(pos=pos.long()), "pos"), (dict(pos=pos[0]), "pos"),
                    (dict(sections=[16, 16]), "pos"), (dict(q_weight=f(32)), "q_weight"), (dict(k_weight=f(64, dt=torch.float16)), "k_weight"),
                    (dict(k=f(64, 4).t()), "contiguous"), (dict(q=f(1, 128).expand(4, 128)), "overlap"), (dict(), "not on the current GPU")):
        with pytest.raises(ValueError, match=msg):
            rope(**kw)
    qs = torch.zeros(3, dtype=I32)
    def packed(**kw):
        a = dict(out=f(4, 128), Q=f(4, 128), K=f(6, 64), V=f(6, 64), n_q=2, n_kv=1, head_dim=64, scale=1.0, q_start=qs, k_start=qs)
        a.update(kw)
        vla.packed_attention_dev(**a)
    for kw, msg in ((dict(out=f(5, 128)), "out"), (dict(V=f(5, 64)), "V"), (dict(K=f(6, 128)), "K"), (dict(q_start=qs.long()), "q_start"),
                    (dict(q_start=qs[:0]), "q_start"), (dict(k_start=qs[:2]), "k_start"), (dict(q_start=torch.zeros(6, dtype=I32)[::2]), "q_start"),
                    (dict(), "not on the current GPU")):
        with pytest.raises(ValueError, match=msg):
            packed(**kw)
    nb = vla.kv4_page_bytes(1, 64, 32)
    cache, table, lens = torch.zeros(4, nb, dtype=torch.uint8), torch.zeros(2, 2, dtype=I32), torch.zeros(2, dtype=I32)
    kv = dict(cache=cache, n_kv=1, head_dim=64, page_size=32, table=table)
    for kw, msg in ((dict(cache=cache[:, 1:]), "cache"), (dict(cache=cache.int()), "cache"), (dict(table=table.long()), "table"),
                    (dict(table=table.t()[:1].t()), "table"), (dict(K=f(4, 32)), "K:"), (dict(V=f(3, 64)), "V:"), (dict(lens=lens[:1]), "lens"),
                    (dict(start=lens), "start"), (dict(page_size=33), "page_size"), (dict(), "not on the current GPU")):
        with pytest.raises(ValueError, match=msg):
            vla.kv4_append_dev(**{**kv, **dict(K=f(4, 64), V=f(4, 64), lens=lens, start=qs), **kw})
    with pytest.raises(ValueError, match="first"):
        vla.kv4_gather_dev(K=f(4, 64), V=f(4, 64), start=qs, first=lens[:1], **kv)
    for kw, msg in ((dict(out=f(2, 64)), "out"), (dict(lens=qs), "lens"), (dict(q_start=lens), "q_start"), (dict(work=f(4)), "work"),
                    (dict(), "not on the current GPU")):
        with pytest.raises(ValueError, match=msg):
            vla.kv4_attention_dev(**{**kv, **dict(out=f(2, 128), Q=f(2, 128), n_q=2, scale=1.0, lens=lens), **kw})


def test_empty_calls_return_without_a_device(vla):
    L = vla.lib()
    assert L.vla_packed_attention_dev(None, 128, None, 128, None, 64, None, 64, None, None, 0, 0, 0, 2, 1, 64, 0.1, 1, 1, None) == 0
    assert L.vla_kv4_append_dev(None, 4, 64, None, 128, None, 128, None, 2, None, None, 0, 0, 2, 64, 1, None) == 0
    s = (ctypes.c_int32 * 1)(32)
    assert L.vla_qk_norm_rope_dev(None, 128, None, 64, None, 128, None, 64, None, None, 0.0, None, 0, s, 1, 1e4, 0, 2, 1, 64, 0, None) == 0


def test_work_bytes(vla):
    w = vla.kv4_attention_work_bytes
    assert w(1, 1, 1, 200, 15, 5, 64) == 0          # one run of keys
    assert w(0, 1, 1, 4096, 15, 5, 64) == 0
    assert w(1, 1, 1, 4096, 15, 4, 64) == 0         # refused shapes need none
    assert 0 < w(2, 2, 1, 131072, 32, 8, 128) < 1 << 22
    assert w(3, 3, 1, 4096, 32, 8, 128) > w(2, 2, 1, 4096, 32, 8, 128) > 0


@pytest.mark.parametrize("total,n,max_len,n_q,n_kv,hd", [(64, 64, 1 << 20, 32, 8, 128), (64, 4, 2 ** 31 - 1, 32, 8, 128), (1, 1, 2 ** 31 - 1, 64, 16, 128),
                                                         (300, 3, 1 << 17, 40, 2, 32), (7, 2, 1 << 17, 3, 1, 256)])
def test_any_bound_on_the_new_tokens(vla, total, n, max_len, n_q, n_kv, hd):
    """No sequence has more new tokens than there are rows: any larger bound plans the same launch."""
    w = lambda m: vla.kv4_attention_work_bytes(total, n, m, max_len, n_q, n_kv, hd)
    assert w(total) > 0
    for m in (total + 1, 1 << 24, 2 ** 31 - 17, 2 ** 31 - 2, 2 ** 31 - 1):
        assert w(m) == w(total), m


def test_work_bytes_of_refused_sizes(vla):
    """Sizes past what a call takes, or splits, need no workspace, and their products do not wrap."""
    w, top = vla.kv4_attention_work_bytes, 2 ** 31 - 1
    for args in ((top, top, top, top, 65536, 1, 256), (1 << 28, 65535, 1 << 28, top, 65536, 1, 256), (8, 70000, 1, 4096, 32, 8, 128), (8, 8, 1, 4096, 32, 8, 160),
                 (8, 8, 1, 4096, 1 << 20, 8, 128), (8, 8, 1, 4096, 4096, 2048, 128), (1 << 20, 8, 1, 1 << 20, 32, 8, 128)):
        assert w(*args) == 0, args


@pytest.mark.parametrize("n,chunk,max_len", [(48, 256, 16384), (48, 128, 16384), (48, 50, 16384), (8, 50, 65536), (64, 1024, 32768), (2, 700, 1 << 20)])
def test_runs_for_a_chunk_among_single_tokens(vla, n, chunk, max_len):
    """The runs of keys are counted by the rows of all sequences: one chunk does not leave the others'
    single tokens, 8 blocks a run here, to a run or two, one sequence behind the other."""
    n_q, n_kv, hd, total = 32, 8, 128, chunk + n - 1
    nb = vla.kv4_attention_work_bytes(total, n, chunk, max_len, n_q, n_kv, hd)
    if nb == 0:  # a block per sequence
        return
    piece = chunk * n_q * (hd + 2) * 4
    runs, rest = divmod(nb - -(-total * 16 // 256) * 256, piece)
    assert rest == 0
    # row tiles of 4 tokens (16 rows of 4 heads); 512 blocks fill the card
    assert (runs - n) * n_kv * (total / 4 + n) / n >= 512


@pytest.mark.parametrize("hd", [160, 224])
def test_pages_of_refused_head_dims(vla, hd):
    """No layout for heads that append and attention refuse."""
    with pytest.raises(ValueError, match="head_dim"):
        vla.kv4_page_bytes(1, hd, 32)
    assert vla.kv4_offset([0], 1, hd, 32, 1, 0, 0, 0, 0) == -1


@pytest.mark.parametrize("n", [1, 2, 3, 4])
def test_work_parts_are_aligned(vla, n):
    """The pieces' values, read 16 bytes at once, lie last in the workspace: a whole number of 16 bytes before them."""
    nb = vla.kv4_attention_work_bytes(n, n, 1, 1 << 17, 1, 1, 32)
    assert nb > 0 and nb % 16 == 0
