"""The 4-bit cache's entry points refuse what the header rules out before
touching a device (CPU only), and the reference of its format agrees with
itself."""
import ctypes

import numpy as np
import pytest

import libpktito_b200 as P
from tests import cache4_ref as R

EINVAL = 1
B = np.zeros(4096, np.float32)  # a host pointer: never dereferenced by a call refused up front
A = (B.ctypes.data + 255) // 256 * 256


def cache(**kw):
    a = dict(pages=A, table=A, lens=A, refs=A, n_layers=2, n_pages=10, max_seqs=4, max_pages=3, page_tokens=16, n_heads=2,
             head_dim=64)
    a.update(kw)
    return P.Cache4(**a)


BAD_CACHES = [dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=512), dict(head_dim=48), dict(head_dim=0),
              dict(head_dim=192), dict(n_heads=0), dict(n_heads=65536), dict(n_layers=0), dict(n_pages=0), dict(max_seqs=0),
              dict(max_pages=0), dict(n_pages=1 << 31), dict(max_pages=1 << 27), dict(pages=None), dict(table=None),
              dict(lens=None), dict(refs=None), dict(pages=A + 8), dict(table=A + 2), dict(refs=A + 1)]


def rows(c=None, append=True, **kw):
    a = dict(layer=1, k=A, ks=128, v=A, vs=128, type=P.F32, seqs=A, starts=A, n=2, rows=4)
    a.update(kw)
    f = P.lib().pkb_cache4_append_dev if append else P.lib().pkb_cache4_read_dev
    return f(0, ctypes.byref(c or cache()), a["layer"], a["k"], a["ks"], a["v"], a["vs"], a["type"], a["seqs"], a["starts"],
             a["n"], a["rows"])


def attend(c=None, **kw):
    a = dict(o=A + 8192, os=256, q=A, qs=256, type=P.F32, H=4, layer=0, seqs=A, starts=A, n=2, rows=4, max_rows=2, scale=0.1,
             causal=1, window=0, work=A, work_bytes=1 << 40)
    a.update(kw)
    return P.lib().pkb_attention_cache4_dev(0, a["o"], a["os"], a["q"], a["qs"], a["type"], a["H"], ctypes.byref(c or cache()),
                                            a["layer"], a["seqs"], a["starts"], a["n"], a["rows"], a["max_rows"], a["scale"],
                                            a["causal"], a["window"], a["work"], a["work_bytes"])


def page_op(name, c=None, **kw):
    a = dict(a=A, b=A, num=A, n=2, status=A, work=A, work_bytes=1 << 20, other=None)
    a.update(kw)
    l, c = P.lib(), ctypes.byref(c or cache())
    tail = (a["status"], a["work"], a["work_bytes"])
    if name == "grow":
        return l.pkb_cache4_grow_dev(0, c, a["a"], a["num"], a["n"], *tail)
    if name == "fork":
        return l.pkb_cache4_fork_dev(0, c, a["a"], a["b"], a["num"], a["n"], *tail)
    if name == "copy":
        return l.pkb_cache4_copy_dev(0, c, ctypes.byref(a["other"]) if a["other"] else c, a["a"], a["b"], a["num"], a["n"], *tail)
    if name == "free":
        return l.pkb_cache4_free_dev(0, c, a["a"], a["n"], *tail)
    return l.pkb_cache4_compact_dev(0, c, a["a"], *tail)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused_by_every_call(kw):
    c = cache(**kw)
    assert rows(c) == rows(c, append=False) == attend(c) == EINVAL
    assert all(page_op(x, c) == EINVAL for x in ("grow", "fork", "copy", "free", "compact"))
    assert P.lib().pkb_cache4_reset_dev(0, ctypes.byref(c)) == EINVAL
    assert P.lib().pkb_last_error()


@pytest.mark.parametrize("kw", [dict(layer=2), dict(k=None), dict(v=None), dict(seqs=None), dict(starts=None), dict(ks=127),
                                dict(vs=127), dict(type=3), dict(type=-1), dict(k=A + 2), dict(v=A + 1), dict(starts=A + 2),
                                dict(type=P.BF16, k=A + 1), dict(rows=1 << 31)])
@pytest.mark.parametrize("append", [True, False])
def test_rows_refused(append, kw):
    assert rows(append=append, **kw) == EINVAL


@pytest.mark.parametrize("kw", [dict(layer=2), dict(H=0), dict(H=3), dict(H=5), dict(type=3), dict(o=None), dict(q=None),
                                dict(seqs=None), dict(starts=None), dict(work=None), dict(work=A + 16), dict(work_bytes=8192),
                                dict(max_rows=0), dict(max_rows=5), dict(qs=255), dict(os=255), dict(q=A + 2),
                                dict(o=A + 4 * 256), dict(o=A), dict(scale=float("nan")), dict(scale=float("inf")),
                                dict(window=1 << 31), dict(rows=1 << 31)])
def test_attention_refused(kw):
    assert attend(**kw) == EINVAL
    assert b"attention_cache4" in P.lib().pkb_last_error()


@pytest.mark.parametrize("name", ["grow", "fork", "copy", "free", "compact"])
def test_page_operations_refused(name):
    for kw in (dict(status=None), dict(work=None), dict(work=A + 4), dict(work_bytes=256), dict(status=A + 1)):
        assert page_op(name, **kw) == EINVAL, kw
    if name != "compact":
        assert page_op(name, n=5) == EINVAL
        assert page_op(name, a=None) == EINVAL
    else:
        assert page_op(name, a=A + 2) == EINVAL
    if name in ("fork", "copy"):
        assert page_op(name, b=None) == EINVAL
    if name not in ("free", "compact"):
        assert page_op(name, num=None) == EINVAL


@pytest.mark.parametrize("kw", [dict(n_layers=1), dict(page_tokens=32), dict(n_heads=1), dict(head_dim=32), dict(n_pages=0)])
def test_copy_between_unlike_caches_is_refused(kw):
    assert page_op("copy", other=cache(**kw)) == EINVAL


def test_nothing_to_do_needs_no_device():
    assert rows(n=0, seqs=None) == rows(rows=0, k=None) == attend(n=0, q=None) == attend(rows=0, max_rows=0) == 0


def test_sizes():
    assert P.cache4_page_bytes(16, 8, 128) == 8 * 18 * 128
    assert P.cache4_page_bytes(64, 1, 96) == 4 * 18 * 96
    assert [P.cache4_page_bytes(*a) for a in ((24, 1, 64), (16, 0, 64), (16, 1, 80))] == [0, 0, 0]
    assert P.cache4_work_bytes(cache()) % 256 == 0
    assert P.attention_cache4_work_bytes(cache(), 3, 4, 2) == 0
    few, many = P.attention_cache4_work_bytes(cache(), 4, 4, 2), P.attention_cache4_work_bytes(cache(max_pages=1 << 20), 4, 4, 2)
    assert 0 < few < many < 200 << 20


def test_descriptor_checks_its_tensors():
    import torch
    pages, table = torch.zeros((2, 5, P.cache4_page_bytes(16, 2, 32)), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.int32)
    lens, refs = torch.zeros(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
    c = P.Cache4.of(pages, table, lens, refs, 16, 2, 32)
    assert (c.n_layers, c.n_pages, c.max_seqs, c.max_pages) == (2, 5, 3, 4)
    for bad in ((pages[:, :4], table, lens, refs), (pages, table[:2], lens, refs), (pages, table.long(), lens, refs),
                (pages, table.t(), lens, refs), (pages, table, lens, refs[:4]), (pages.to("meta"), table, lens, refs)):
        with pytest.raises(P.PkbError):
            P.Cache4.of(*bad, 16, 2, 32)
    with pytest.raises(P.PkbError):
        P.Cache4.of(pages, table, lens, refs, 16, 2, 48)


def test_calls_check_their_tensors():
    import torch
    c = P.Cache4.of(torch.zeros((1, 5, P.cache4_page_bytes(16, 2, 32)), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.int32),
                    torch.zeros(3, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), 16, 2, 32)
    good, work, rows = torch.zeros(4, dtype=torch.int32), torch.zeros(1 << 16, dtype=torch.uint8), torch.zeros((4, 64))
    bad = [good.long(), good[:1], torch.zeros(8, dtype=torch.int32)[::2], good.float(), good.to("meta")]
    for x in bad:
        calls = [lambda: P.cache4_grow_dev(c, x, good, 2, good, work, 0), lambda: P.cache4_grow_dev(c, good, x, 2, good, work, 0),
                 lambda: P.cache4_free_dev(c, x, 2, good, work, 0)]
        calls += [lambda i=i: P.cache4_fork_dev(c, *[x if i == j else good for j in range(3)], 2, good, work, 0) for i in range(3)]
        calls += [lambda i=i: P.cache4_copy_dev(c, c, *[x if i == j else good for j in range(3)], 2, good, work, 0) for i in range(3)]
        calls += [lambda i=i: P.cache4_append_dev(c, 0, rows, 64, rows, 64, *[x if i == j else good for j in range(2)], 2, 4, 0)
                  for i in range(2)]
        calls += [lambda i=i: P.attention_cache4_dev(rows, 64, rows, 64, 2, c, 0, *[x if i == j else good for j in range(2)], 2, 4, 4,
                                                     0.1, True, 0, work, 0) for i in range(2)]
        for call in calls:
            with pytest.raises(P.PkbError):
                call()
    for k, v in ((rows, rows.half()), (rows.int(), rows.int()), (rows.to("meta"), rows), (rows, rows.to("meta"))):
        with pytest.raises(P.PkbError):
            P.cache4_read_dev(c, 0, k, 64, v, 64, good, good, 2, 4, 0)
    for area in (work.to("meta"), work[::2]):
        with pytest.raises(P.PkbError):
            P.cache4_compact_dev(c, None, good, area, 0)
    with pytest.raises(P.PkbError):
        P.cache4_compact_dev(c, None, good.long(), work, 0)


def test_a_scale_that_overflows_is_refused():
    assert attend(scale=3.0e38) == EINVAL  # times log2 e
    assert attend(scale=-3.0e38) == EINVAL


@pytest.mark.parametrize("dk", [32, 64, 96, 128, 256])
def test_every_nibble_is_one_values(dk):
    for at in R.nibble_places(dk):
        assert sorted(at.reshape(-1)) == list(range(16 * dk))


@pytest.mark.parametrize("dk", [32, 96])
def test_reference_reads_what_it_writes(dk):
    rng = np.random.default_rng(dk)
    p = R.Pages(rng.integers(0, 256, 3 * 2 * 2 * 18 * dk).astype(np.uint8), 32, 2, dk)
    x = rng.standard_normal((2, 40, 2, dk)).astype(np.float32)
    for j in range(40):
        for which in (0, 1):
            p.write([2, 0][j // 32], j % 32, which, *R.quantize(x[which, j]))
    for which, got in enumerate(p.read([2, 0], 40)):
        assert np.array_equal(got.transpose(1, 0, 2), R.held(x[which]))


def test_format_of_special_blocks():
    x = np.zeros((7, 32), np.float32)
    x[0, 3], x[1, 4], x[2, 0] = np.nan, -np.inf, 2.0 ** -122
    x[3, 5] = 2.0 ** -121
    x[4] = np.linspace(-1, 1, 32)
    x[5, 31] = np.finfo(np.float32).max
    x[6, :2] = 7, 3.5  # scale 1: a tie, to even
    c, s = R.quantize(x)
    assert (c[:3] == 0).all() and (s[:3, 0] == 0).all()
    assert c[3, 5] == 7 and s[3, 0] > 0 and c[4].min() == -7 and c[4].max() == 7
    assert np.isfinite(R.held(x)).all() and c[5, 31] == 7
    assert s[6, 0] == 1 and list(c[6, :2]) == [7, 4]
