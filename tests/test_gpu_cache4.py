"""The 4-bit cache on a B200 against tests/cache4_ref.py: its bytes and its
books exactly, the attention within what its roundings allow."""
import numpy as np
import pytest
import torch

import libpktito_b200 as P
from tests import cache4_ref as R

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_device")]
KIND = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
PARTS = {"f32": 2.0 ** -24, "f16": 2.0 ** -16, "bf16": 2.0 ** -8}  # what a probability in 3, 2, 1 bf16 parts may be off


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def lay_out(lens, page, extra=3, rng=None, max_pages=None):
    """(table, refs, n_pages) with pages in no order for sequences of these lengths."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + extra
    order = (rng or np.random.default_rng(0)).permutation(n_pages)
    table = np.full((len(lens), max_pages or max(1, *need) + 1), -1, np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    refs = np.zeros(n_pages, np.int32)
    refs[table[table >= 0]] = 1
    return table, refs, n_pages


def make(lens, page, heads, dk, layers=1, seed=0, fill=None, **kw):
    rng = np.random.default_rng(seed)
    table, refs, n_pages = lay_out(lens, page, rng=rng, **kw)
    size = (layers, n_pages, P.cache4_page_bytes(page, heads, dk))
    raw = torch.tensor(rng.integers(0, 256, size).astype(np.uint8) if fill is None else np.full(size, fill, np.uint8), device="cuda")
    return P.Cache4.of(raw, ints(table), ints(lens), ints(refs), page, heads, dk)


def append(c, layer, k, v, seqs, rows, stride=None):
    starts = np.concatenate([[0], np.cumsum(rows)])
    width = k.shape[1]
    if stride:
        k, v = (torch.nn.functional.pad(x, (0, stride - width), value=float("nan")) for x in (k, v))
    P.cache4_append_dev(c, layer, k, stride or width, v, stride or width, ints(seqs), ints(starts), len(seqs), int(starts[-1]))
    torch.cuda.synchronize()


def no_errors():
    torch.cuda.synchronize()
    assert P.device_errors(0) == 0


@pytest.mark.parametrize("dk", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("page,heads,kind", [(16, 1, "f32"), (64, 3, "bf16"), (256, 2, "f16")])
def test_append_writes_the_formats_bytes(dk, page, heads, kind):
    rng = np.random.default_rng(dk + page)
    lens, rows = [1, 47, 16, 300, 5, 33], [1, 20, 16, 290, 0, 1]
    c = make(lens, page, heads, dk, layers=2, seed=dk)
    raw = c.tensors[0].cpu().numpy().copy()
    seqs = [3, 0, 5, 1, 4, 2]
    n = sum(rows)
    x = rng.standard_normal((2, n, heads * dk)).astype(np.float32) * np.exp(rng.standard_normal((2, n, 1)))
    x[0, 3, :5], x[1, 7, 0], x[0, 9, 1], x[1, 11, :32] = 0, np.nan, np.inf, 0
    k, v = (torch.tensor(y, dtype=torch.float32, device="cuda").to(KIND[kind]) for y in x)
    append(c, 1, k, v, seqs, [rows[s] for s in seqs], stride=heads * dk + (16 if dk == 64 else 0) or None)
    want = R.Pages(raw[1].reshape(-1), page, heads, dk)
    table, at = c.tensors[1].cpu().numpy(), 0
    kk, vv = (y.double().cpu().numpy() for y in (k, v))
    for s in seqs:
        for i in range(rows[s]):
            pos = lens[s] - rows[s] + i
            for which, y in enumerate((kk, vv)):
                want.write(table[s, pos // page], pos % page, which, *R.quantize(y[at + i].reshape(heads, dk)))
        at += rows[s]
    got = c.tensors[0].cpu().numpy()
    assert np.array_equal(got[0], raw[0])
    assert np.array_equal(got[1].reshape(-1), want.raw.reshape(-1))  # the tokens, and every byte beside them as it was
    no_errors()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [0, 1])  # values off a 16-byte boundary
def test_read_gives_what_append_took(kind, offset):
    heads, dk, lens, rows = 2, 96, [37, 2, 130, 0], [20, 2, 130, 0]
    n, width = sum(rows), heads * dk
    c = make(lens, 32, heads, dk, seed=3)
    g = torch.Generator("cuda").manual_seed(5)
    buf = torch.randn((2, n * width + 16), generator=g, device="cuda").mul_(3).to(KIND[kind])
    buf[0, 40], buf[1, 77] = float("nan"), float("-inf")
    k, v = (b[offset:offset + n * width].view(n, width) for b in buf)
    seqs, starts = ints([2, 3, 0, 1]), ints([0, 130, 130, 150, 152])
    P.cache4_append_dev(c, 0, k, width, v, width, seqs, starts, 4, n)
    out = torch.full((2, (n + 3) * width + 16), 9.0, device="cuda").to(KIND[kind])
    ko, vo = (b[offset:offset + (n + 3) * width].view(n + 3, width) for b in out)
    P.cache4_read_dev(c, 0, ko, width, vo, width, seqs, starts, 4, n + 3)  # room behind the last sequence
    torch.cuda.synchronize()
    for x, y in ((k, ko), (v, vo)):
        want = torch.tensor(R.held(x.double().cpu().numpy())).to(KIND[kind])
        assert torch.equal(y[:n].cpu(), want)
        assert (y[n:] == 9).all()
    no_errors()


def test_every_f32_magnitude_is_held_as_defined():
    # blocks over all exponents, scales and ties next to their borders
    rng = np.random.default_rng(11)
    n, heads, dk = 640, 4, 128
    x = np.ldexp(rng.uniform(-1, 1, (n, heads * dk // 32, 32)), rng.integers(-130, 129, (n, heads * dk // 32, 1)))
    top = np.ldexp(rng.integers(16, 32, (n // 2, heads * dk // 32, 1)) / 32.0, rng.integers(-100, 120, (n // 2, heads * dk // 32, 1)))
    x[:n // 2] = top * (rng.integers(-14, 15, (n // 2, heads * dk // 32, 32)) / 2.0)  # halves of a 5-bit scale
    x[:n // 2, :, 0] = 7 * top[..., 0]
    x = x.astype(np.float32)
    x[:n // 2, :, 1:5] = np.nextafter(x[:n // 2, :, 1:5], np.float32(0))
    x[: n // 4, :, 0] = np.nextafter(x[: n // 4, :, 0], np.float32(0))
    x = x.reshape(n, heads * dk)
    c = make([n], 64, heads, dk)
    k = torch.tensor(x, device="cuda")
    append(c, 0, k, k.flip(0).contiguous(), [0], [n])
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    P.cache4_read_dev(c, 0, ko, heads * dk, vo, heads * dk, ints([0]), ints([0, n]), 1, n)
    torch.cuda.synchronize()
    want = R.held(x.astype(np.float64))
    assert np.array_equal(ko.double().cpu().numpy(), want)
    assert np.array_equal(vo.double().cpu().numpy(), want[::-1])


def test_rows_out_of_range_set_the_error_word():
    c = make([10, 20], 16, 1, 32, fill=0)
    k = torch.ones((8, 32), device="cuda")
    before = c.tensors[0].clone()
    for seqs, starts in (([2], [0, 4]), ([-1], [0, 4]), ([0], [0, 9]), ([0], [4, 0]), ([0], [-1, 4])):
        P.cache4_append_dev(c, 0, k, 32, k, 32, ints(seqs), ints(starts), 1, 8)
        torch.cuda.synchronize()
        assert P.device_errors(0) == 2, (seqs, starts)
    c.tensors[1][0, 0] = 99
    P.cache4_append_dev(c, 0, k, 32, k, 32, ints([0]), ints([0, 8]), 1, 8)
    torch.cuda.synchronize()
    assert P.device_errors(0) == 2
    P.cache4_append_dev(c, 0, k, 32, k, 32, ints([-1, 7]), ints([0, 0, 0]), 2, 8)  # no rows: a padded batch
    no_errors()
    assert torch.equal(c.tensors[0], before)


# ------------------------------------------------------------------ attention --

def filled(lens, page, heads, dk, seed, layers=1, spread=1.0, **kw):
    """A cache whose tokens hold random rows, its other bytes NaN scales where they can be."""
    c = make(lens, page, heads, dk, layers=layers, seed=seed, fill=0xFF, **kw)
    g = torch.Generator("cuda").manual_seed(seed)
    n = sum(lens)
    for layer in range(layers):
        k, v = torch.randn((2, n, heads * dk), generator=g, device="cuda").mul_(spread)
        if n:
            append(c, layer, k, v, list(range(len(lens))), lens)
    return c


def check_attention(c, lens, rows, seqs, G, kind, causal, window, layer=0, scale=None, seed=1, pad=0, tail=0, q=None, max_rows=None):
    heads, dk, page = c.n_heads, c.head_dim, c.page_tokens
    H, n, starts = heads * G, sum(rows), np.concatenate([[0], np.cumsum(rows)])
    scale = dk ** -0.5 if scale is None else scale
    g = torch.Generator("cuda").manual_seed(seed)
    if q is None:
        q = torch.randn((n + tail, H * dk), generator=g, device="cuda").to(KIND[kind])
    qs, os = H * dk + pad, H * dk + 2 * pad
    qq = torch.nn.functional.pad(q, (0, pad), value=float("nan"))
    o = torch.full((n + tail, os), 5.0, device="cuda").to(KIND[kind])
    work = torch.full((P.attention_cache4_work_bytes(c, H, n + tail, len(seqs)),), 0xFF, dtype=torch.uint8, device="cuda")
    P.attention_cache4_dev(o, os, qq, qs, H, c, layer, ints(seqs), ints(starts), len(seqs), n + tail,
                           max_rows or max(1, *rows), scale, causal, window, work)
    no_errors()
    pages = R.Pages(c.tensors[0][layer].cpu().numpy().reshape(-1), page, heads, dk)
    table = c.tensors[1].cpu().numpy()
    got = o.double().cpu().numpy()
    assert (got[n:] == 5).all() and (got[:, H * dk:] == 5).all()
    worst = 0.0
    for i, s in enumerate(seqs):
        if not rows[i]:
            continue
        mine = slice(starts[i], starts[i + 1])
        L = lens[s]
        k, v = pages.read(table[s], L) if L else (np.zeros((heads, 0, dk)),) * 2
        y, size, score = R.attention(q[mine].double().cpu().numpy().reshape(rows[i], H, dk), k, v, L, scale, causal, window)
        # o's own rounding; the probabilities' parts; a score's error moves a
        # probability by as much, twice over with the sum: sums of dk exact
        # products cut to float at most dk/16 + 8 times, the scaling, the
        # subtraction and 2^x; each further product of 16 keys cuts o once more
        e = (dk / 16 + 12) * 2.0 ** -23 * (1 + score)[..., None]
        tol = HALF[kind] * np.abs(y) + (PARTS[kind] + 2 * e + (L / 16 + 16) * 2.0 ** -23) * size + (2.0 ** -25 if kind == "f16" else 0)
        # a probability below a float's smallest normal number, 2^-126, is
        # zero here and is not in 64 bits: each of L keys may lose that much
        # of its value, against a sum of at least 1 (the largest score's 2^0)
        tol = tol + L * 2.0 ** -126 * np.abs(v).max(initial=0)
        off = np.abs(got[mine, :H * dk].reshape(y.shape) - y)
        bad = ~(off <= tol)
        assert not bad.any(), (s, rows[i], L, np.argwhere(bad)[:3], off[bad][:3], tol[bad][:3])
        worst = max(worst, float((off / np.maximum(tol, 1e-300)).max(initial=0)))
    return worst


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,page,heads,G", [(32, 16, 1, 1), (64, 32, 2, 3), (96, 64, 1, 8), (128, 16, 8, 1), (128, 128, 2, 5),
                                             (256, 32, 2, 2)])
def test_one_token_a_sequence(kind, dk, page, heads, G):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 0, 500]
    c = filled(lens, page, heads, dk, seed=dk + G, layers=2)
    order = [11, 0, 3, 10, 1, 2, 4, 9, 8, 7, 6, 5]
    check_attention(c, lens, [1] * 12, order, G, kind, True, 0, layer=1, pad=8)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 37, 5000])
def test_some_rows_and_windows(kind, causal, window):
    lens, rows = [70, 3, 1, 200, 40, 16], [5, 3, 1, 13, 40, 0]
    c = filled(lens, 16, 2, 64, seed=7)
    check_attention(c, lens, [rows[s] for s in (2, 0, 3, 5, 1, 4)], [2, 0, 3, 5, 1, 4], 3, kind, causal, window, tail=2)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_before_the_first_token_see_nothing(kind):
    # more queries than tokens: the first ones stand before the sequence
    lens, rows = [3, 0, 20], [8, 4, 25]
    c = filled(lens, 16, 2, 32, seed=2)
    check_attention(c, lens, rows, [0, 1, 2], 2, kind, True, 0)
    check_attention(c, lens, rows, [0, 1, 2], 2, kind, True, 2)
    check_attention(c, lens, rows, [0, 1, 2], 2, kind, False, 0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,G,n", [(128, 1, 300), (64, 4, 257), (256, 1, 130), (32, 2, 129), (96, 2, 200)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 100), (False, 0)])
def test_prompts(kind, dk, G, n, causal, window):
    lens, rows = [n, n + 77, 5, 64], [n, 131, 5, 64]
    c = filled(lens, 64, 2, dk, seed=n)
    check_attention(c, lens, rows, [0, 1, 2, 3], G, kind, causal, window, pad=4, tail=1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_long_and_uneven(kind):
    # parts of many shares to one sequence; few heads, so the split runs along the keys
    lens = [20011, 5, 3000]
    c = filled(lens, 64, 1, 128, seed=3)
    check_attention(c, lens, [1, 1, 1], [0, 1, 2], 4, kind, True, 0)
    check_attention(c, lens, [3, 1, 2], [0, 1, 2], 4, kind, True, 1500)


def test_more_sequences_than_a_launch_takes():
    lens = [1 + (7 * i) % 40 for i in range(1500)]
    c = filled(lens, 16, 1, 32, seed=5)
    check_attention(c, lens, [1 + i % 2 for i in range(1500)], list(range(1500))[::-1], 1, "bf16", True, 0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_large_scores_and_a_negative_scale(kind):
    lens = [333, 50]
    c = filled(lens, 32, 2, 64, seed=9, spread=30.0)
    check_attention(c, lens, [1, 2], [0, 1], 2, kind, True, 0, scale=2.0)
    check_attention(c, lens, [1, 2], [0, 1], 2, kind, True, 0, scale=-0.3)
    check_attention(c, lens, [1, 2], [0, 1], 2, kind, True, 0, scale=1e-30)


def test_a_nan_row_stays_its_own():
    lens = [90]
    c = filled(lens, 16, 1, 64, seed=4)
    q = torch.randn((3, 4 * 64), device="cuda")
    q[1, 64:128] = float("nan")
    o, work = torch.empty_like(q), torch.empty(P.attention_cache4_work_bytes(c, 4, 3, 1), dtype=torch.uint8, device="cuda")
    args = (4, c, 0, ints([0]), ints([0, 3]), 1, 3, 3, 0.1, True, 0, work)
    P.attention_cache4_dev(o, 256, q, 256, *args)
    torch.cuda.synchronize()
    assert o[1, 64:128].isnan().all()
    clean = o.clone()
    q[1, 64:128] = 0
    P.attention_cache4_dev(o, 256, q, 256, *args)
    torch.cuda.synchronize()
    o[1, 64:128] = clean[1, 64:128]
    assert torch.equal(torch.nan_to_num(o, 7.0), torch.nan_to_num(clean, 7.0))


def test_bad_tables_and_sequences_do_not_reach_memory():
    lens = [40, 40]
    c = filled(lens, 16, 1, 32, seed=6)
    q = torch.randn((2, 32), device="cuda")
    o, work = torch.empty_like(q), torch.empty(P.attention_cache4_work_bytes(c, 1, 2, 2), dtype=torch.uint8, device="cuda")

    def run(seqs, starts):
        P.attention_cache4_dev(o, 32, q, 32, 1, c, 0, ints(seqs), ints(starts), 2, 2, 1, 0.1, True, 0, work)
        torch.cuda.synchronize()
        return P.device_errors(0)
    assert run([0, 1], [0, 1, 2]) == 0
    for seqs, starts in (([0, 2], [0, 1, 2]), ([-5, 1], [0, 1, 2]), ([0, 1], [0, 1, 3]), ([0, 1], [0, -1, 2]), ([0, 1], [2, 1, 2])):
        assert run(seqs, starts) == 2, (seqs, starts)
    c.tensors[2][1] = 1 << 20
    assert run([0, 1], [0, 1, 2]) == 2
    c.tensors[2][1] = 40
    c.tensors[1][0, 1], c.tensors[1][1, 0] = -7, 1 << 30
    assert run([0, 1], [0, 1, 2]) == 2


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,G,dk", [(17, 1, 32), (20, 3, 64), (33, 2, 32), (40, 1, 128)])
def test_more_heads_than_a_team(kind, heads, G, dk):
    lens = [1, 900, 33, 0, 250]
    c = filled(lens, 16, heads, dk, seed=heads)
    check_attention(c, lens, [1] * 5, [4, 1, 3, 0, 2], G, kind, True, 0)
    check_attention(c, lens, [1, 5, 2, 1, 3], [4, 1, 3, 0, 2], G, kind, True, 70)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_table_with_room_for_a_billion_tokens(kind):
    # places are counted in 32 bits: three entries take two launches, or the way of many rows
    lens = [300, 129, 1000]
    c = filled(lens, 256, 33, 32, seed=21, max_pages=2 ** 22 - 1)
    check_attention(c, lens, [128, 1, 100], [0, 1, 2], 1, kind, True, 0)
    check_attention(c, lens, [1, 1, 1], [2, 0, 1], 2, kind, True, 2 ** 29)
    check_attention(c, lens, [300, 1, 100], [0, 1, 2], 2, kind, False, 2 ** 30 + 500)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,heads,G,dk,rows,page", [(1, 1, 1, 32, 1024, 16), (1, 8, 4, 64, 130, 32), (3, 20, 1, 32, 129, 16), (4, 33, 1, 32, 140, 16),
                                                    (2, 2, 3, 256, 43, 16), (1, 1, 8, 128, 128, 64), (9, 4, 1, 96, 300, 16), (70, 8, 1, 32, 17, 16)])
def test_the_work_area_is_enough(kind, n, heads, G, dk, rows, page):
    """Nothing is written behind the bytes asked for, whichever way the rows are divided; more rows than a wave, and fewer."""
    lens = [rows + 37 * (i % 5) for i in range(n)]
    c = filled(lens, page, heads, dk, seed=rows)
    H, total = heads * G, n * rows
    q = torch.randn((total, H * dk), generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(KIND[kind])
    o = torch.empty_like(q)
    size = P.attention_cache4_work_bytes(c, H, total, n)
    work = torch.full((size + (1 << 20),), 0xA5, dtype=torch.uint8, device="cuda")
    for most in (rows, total):  # max_rows may say more than there are
        P.attention_cache4_dev(o, H * dk, q, H * dk, H, c, 0, ints(range(n)), ints([i * rows for i in range(n + 1)]), n, total, most,
                               dk ** -0.5, True, 0, work[:size])
        no_errors()
        assert (work[size:] == 0xA5).all()
    assert check_attention(c, lens, [rows] * n, list(range(n)), G, kind, True, 0, q=q) <= 1
    assert check_attention(c, lens, [rows] * n, list(range(n)), G, kind, False, 0, q=q, max_rows=total) <= 1


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 150])  # one part, some rows, a prompt
def test_padded_entries_and_a_sequence_listed_twice(kind, rows):
    lens = [160, 400, 151]
    c = filled(lens, 32, 2, 64, seed=13)
    r = [0, rows, 0, 1, rows, 0, rows]
    check_attention(c, lens + [0], r, [-1, 1, 2, 0, 1, 99, 2], 1, kind, True, 0, tail=5)
    check_attention(c, lens, [rows, rows], [2, 0], 2, kind, False, 2 ** 31 - 1)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 200])
def test_a_scale_of_zero_is_the_mean(kind, rows):
    lens = [333, 201]
    c = filled(lens, 32, 2, 64, seed=9)
    check_attention(c, lens, [rows, rows], [0, 1], 1, kind, True, 0, scale=0.0)


@pytest.mark.parametrize("most,rows", [(1, 2), (4, 5), (140, 141)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_rows_than_said_set_the_error_word(kind, most, rows):
    lens = [300, 300]
    c = filled(lens, 16, 1, 32, seed=6)
    n = rows + most
    q = torch.randn((n, 32), device="cuda").to(KIND[kind])
    o, work = torch.empty_like(q), torch.empty(P.attention_cache4_work_bytes(c, 1, n, 2), dtype=torch.uint8, device="cuda")
    P.attention_cache4_dev(o, 32, q, 32, 1, c, 0, ints([0, 1]), ints([0, most, n]), 2, n, most, 0.1, True, 0, work)
    torch.cuda.synchronize()
    assert P.device_errors(0) == 2
    alone = torch.empty_like(q)
    P.attention_cache4_dev(alone, 32, q, 32, 1, c, 0, ints([0]), ints([0, most]), 1, n, most, 0.1, True, 0, work)
    no_errors()
    assert torch.allclose(o[:most].float(), alone[:most].float(), rtol=2 * HALF[kind] + 1e-5, atol=1e-5)  # the other entry's rows


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows", [3, 260])
def test_a_row_that_is_not_finite_stays_its_own(kind, value, rows):
    lens, H, dk = [300], 2, 64
    c = filled(lens, 16, 1, dk, seed=4)
    q = torch.randn((rows, H * dk), generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(KIND[kind])
    o, work = torch.empty_like(q), torch.empty(P.attention_cache4_work_bytes(c, H, rows, 1), dtype=torch.uint8, device="cuda")
    args = (H, c, 0, ints([0]), ints([0, rows]), 1, rows, rows, 0.1, True, 0, work)
    P.attention_cache4_dev(o, H * dk, q, H * dk, *args)
    clean = o.clone()
    q[1, dk:] = value
    P.attention_cache4_dev(o, H * dk, q, H * dk, *args)
    no_errors()
    assert o[1, dk:].isnan().all()
    o[1, dk:] = clean[1, dk:]
    assert torch.equal(o, clean)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_offsets_past_32_bits(kind):
    """The last pages of a layer's 2.2 GB, in the second layer: the same bits as from a small cache, and page copies."""
    heads, dk, page, n_pages = 8, 256, 256, 3700
    lens, rows = [700, 300], [300, 1]
    small = P.Cache4.empty(1, 5, 3, 4, page, heads, dk)
    large = P.Cache4.empty(2, n_pages, 3, 4, page, heads, dk)
    assert large.tensors[0].numel() > 2 ** 32
    k, v = torch.randn((2, 1000, heads * dk), generator=torch.Generator("cuda").manual_seed(2), device="cuda").to(KIND[kind])
    q = torch.randn((301, heads * dk), generator=torch.Generator("cuda").manual_seed(3), device="cuda").to(KIND[kind])
    got = []
    for c, layer, last in ((small, 0, 4), (large, 1, n_pages - 1)):
        c.tensors[1][0, :3], c.tensors[1][1, :2] = ints([last, last - 2, last - 1]), ints([last - 4, last - 3])
        c.tensors[2][:2] = ints(lens)
        c.tensors[3][last - 4:last + 1] = 1
        append(c, layer, k, v, [0, 1], lens)
        out = []
        for r, most in ((rows, 300), ([1, 1], 1)):
            n = sum(r)
            o, work = torch.empty_like(q[:n]), torch.empty(P.attention_cache4_work_bytes(c, heads, n, 2), dtype=torch.uint8, device="cuda")
            P.attention_cache4_dev(o, heads * dk, q, heads * dk, heads, c, layer, ints([0, 1]), ints([0, r[0], n]), 2, n, most, 0.06,
                                   True, 0, work)
            out.append(o)
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        P.cache4_read_dev(c, layer, ko, heads * dk, vo, heads * dk, ints([0, 1]), ints([0, *np.cumsum(lens)]), 2, 1000)
        no_errors()
        got.append(out + [ko, vo])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    status, work = ints([9]), torch.empty(P.cache4_work_bytes(large), dtype=torch.uint8, device="cuda")
    P.cache4_copy_dev(large, large, ints([0]), ints([2]), ints([700]), 1, status, work)  # to the first pages
    P.cache4_read_dev(large, 1, ko, heads * dk, vo, heads * dk, ints([2]), ints([0, 700]), 1, 1000)
    no_errors()
    assert int(status) == 0 and large.tensors[1][2].tolist() == [0, 1, 2, -1]
    assert torch.equal(ko, got[0][2]) and torch.equal(vo, got[0][3])


# ------------------------------------------------------------- page operations --

class Both:
    """A cache on the GPU and its books on the host, changed alike."""

    def __init__(self, n_pages, max_seqs, max_pages, page, heads=1, dk=32, layers=2, seed=0):
        self.c = P.Cache4.empty(layers, n_pages, max_seqs, max_pages, page, heads, dk)
        self.c.tensors[0].copy_(torch.randint(0, 256, self.c.tensors[0].shape, generator=torch.Generator().manual_seed(seed)).byte())
        self.raw = self.c.tensors[0].cpu().numpy().copy()
        self.b = R.Books(n_pages, max_seqs, max_pages, page)
        self.work = torch.full((P.cache4_work_bytes(self.c),), 0xEE, dtype=torch.uint8, device="cuda")
        self.status = torch.full((1,), 77, dtype=torch.int32, device="cuda")

    def same(self, status):
        no_errors()
        assert int(self.status) == status
        for got, want in zip(self.c.tensors[1:], self.b.arrays()):
            assert np.array_equal(got.cpu().numpy(), want)
        assert np.array_equal(self.c.tensors[0].cpu().numpy(), self.raw)
        return status

    def grow(self, seqs, add):
        P.cache4_grow_dev(self.c, ints(seqs), ints(add), len(seqs), self.status, self.work)
        return self.same(self.b.grow(seqs, add))

    def fork(self, src, dst, lens):
        P.cache4_fork_dev(self.c, ints(src), ints(dst), ints(lens), len(src), self.status, self.work)
        status, copies = self.b.take_over(src, dst, lens, True)
        for a, b in copies:
            self.raw[:, b] = self.raw[:, a]
        return self.same(status)

    def copy(self, src, dst, lens, to=None):
        t = to or self
        P.cache4_copy_dev(t.c, self.c, ints(src), ints(dst), ints(lens), len(src), t.status, t.work)
        status, copies = self.b.take_over(src, dst, lens, False, t.b)
        for a, b in copies:
            t.raw[:, b] = self.raw[:, a]
        return t.same(status)

    def free(self, seqs):
        P.cache4_free_dev(self.c, ints(seqs), len(seqs), self.status, self.work)
        return self.same(self.b.free(seqs))

    def compact(self):
        used = torch.zeros(1, dtype=torch.int32, device="cuda")
        P.cache4_compact_dev(self.c, used, self.status, self.work)
        want, moves = self.b.compact()
        for a, b in moves:
            self.raw[:, b] = self.raw[:, a]
        assert self.same(0) == 0 and int(used) == want


def test_page_operations_one_by_one():
    x = Both(12, 6, 4, 16)
    assert x.grow([2, 0], [17, 16]) == 0  # two pages, one page
    assert x.grow([0, 2, 4], [1, 0, 0]) == 0
    assert x.fork([2, 2, 0], [1, 3, 5], [17, 16, 0]) == 0  # a page shared and one copied; a page shared; nothing
    assert x.grow([1, 3], [3, 1]) == 0
    assert x.free([2, 5]) == 0  # its pages stay where the forks hold them
    assert x.copy([1], [2], [18]) == 0
    x.compact()
    assert x.free([1, 3, 2]) == 0
    x.compact()
    x.compact()
    assert x.free([0, 4]) == 0 and int(x.c.tensors[3].sum()) == 0
    x.compact()


def test_page_operations_that_fail_change_nothing():
    x = Both(6, 5, 3, 16)
    assert x.grow([0, 1], [40, 10]) == 0
    assert x.grow([2], [33]) == R.Books.FULL
    assert x.grow([2, 3], [32, 1]) == R.Books.FULL
    assert x.grow([0], [9]) == R.Books.LONG and x.grow([0], [2 ** 31 - 1]) == R.Books.LONG
    assert x.grow([0, 0], [1, 1]) == R.Books.BAD
    assert x.grow([5], [1]) == x.grow([-1], [1]) == x.grow([1], [-1]) == R.Books.BAD
    assert x.fork([0], [1], [5]) == R.Books.BAD  # not empty
    assert x.fork([0], [2], [41]) == x.fork([2], [3], [1]) == x.fork([0], [2], [-1]) == R.Books.BAD
    assert x.fork([0, 0], [2, 2], [5, 5]) == x.fork([9], [2], [0]) == x.fork([0], [9], [5]) == R.Books.BAD
    assert x.fork([0, 0, 0], [2, 3, 4], [39, 39, 40]) == R.Books.FULL
    assert x.copy([0], [2], [40]) == R.Books.FULL and x.copy([0, 1], [2, 2], [1, 1]) == R.Books.BAD
    assert x.free([0, 0]) == x.free([0, 5]) == x.free([-1]) == R.Books.BAD
    small = Both(9, 2, 2, 16)
    assert x.copy([0], [0], [40], small) == R.Books.LONG and x.copy([0], [1], [32], small) == 0
    assert x.grow([], []) == x.free([]) == x.fork([], [], []) == 0


@pytest.mark.parametrize("page,heads,dk,layers", [(16, 1, 32, 1), (64, 3, 96, 2), (256, 1, 256, 1)])
def test_page_operations_at_random(page, heads, dk, layers):
    rng = np.random.default_rng(page)
    x = Both(70, 20, 9, page, heads, dk, layers)
    y = Both(40, 8, 9, page, heads, dk, layers, seed=1)
    seen = set()
    for step in range(120):
        op = rng.choice(["grow", "grow", "grow", "fork", "fork", "free", "copy", "over", "compact"])
        if op == "compact":
            (x if step % 3 else y).compact()
            continue
        n = int(rng.integers(1, 6))
        if op == "grow":
            seen.add((op, x.grow(list(map(int, rng.choice(20, n, replace=False))), list(map(int, rng.integers(0, 2 * page, n))))))
        elif op == "free":
            live = [s for s in range(20) if x.b.lens[s]]
            seen.add((op, x.free(list(map(int, rng.permutation(live)[:n])))))
            y.free([s for s in range(8) if rng.random() < 0.3])
        else:
            t = y if op == "over" else x
            empty = [s for s in range(len(t.b.lens)) if not t.b.lens[s]]
            dst = list(map(int, rng.permutation(empty)[:n]))
            src = list(map(int, rng.choice(20, len(dst))))
            lens = [int(rng.integers(0, x.b.lens[s] + 1)) for s in src]
            if op == "fork":
                seen.add((op, x.fork(src, dst, lens)))
            else:
                seen.add((op, x.copy(src, dst, lens, t)))
    assert {("grow", 0), ("fork", 0), ("free", 0), ("copy", 0), ("over", 0)} <= seen


def test_page_operations_on_a_large_pool():
    # the free pages lie behind many scans' worth of used ones
    x = Both(40003, 3000, 16, 16, 1, 32, 1)
    assert x.grow(list(range(2500)), [16 * 16] * 2500) == R.Books.DONE
    assert x.grow([2999, 2998], [20, 17]) == R.Books.FULL  # three are left, four wanted
    gone = list(range(0, 2500, 7))
    assert x.free(gone) == 0
    assert x.grow([2999, 2600, 2700], [33, 1, 250]) == 0
    assert x.fork(list(range(1, 1001, 1))[:400], list(range(2501, 2501 + 99)) + gone[:301], [100 + i % 9 for i in range(400)]) in (0, R.Books.BAD)
    x.compact()


# ------------------------------------------------------------------ together --

def test_reset():
    x = Both(9, 4, 3, 16)
    x.grow([0, 2], [30, 5])
    P.cache4_reset_dev(x.c)
    x.b = R.Books(9, 4, 3, 16)
    x.status.zero_()
    x.same(0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_beam_decodes(kind):
    """Beam search as a decoder runs it: a prompt, forks of it, then steps of fork, free, grow, append in both layers and
    attend; a compaction on the way. Every step's attention against dense attention over the rows each hypothesis was given."""
    heads, dk, G, page, layers, beams = 2, 64, 2, 16, 2, 4
    x = Both(60, 2 * beams, 6, page, heads, dk, layers)
    g = torch.Generator("cuda").manual_seed(8)
    rng = np.random.default_rng(8)
    history = {s: [] for s in range(2 * beams)}  # a hypothesis' rows: [(k, v) of both layers]

    def rows(n):
        return torch.randn((layers, 2, n, heads * dk), generator=g, device="cuda").to(KIND[kind])

    def give(seqs, each):
        new = rows(len(seqs) * each)
        starts = np.arange(len(seqs) + 1) * each
        for layer in range(layers):
            P.cache4_append_dev(x.c, layer, new[layer, 0], heads * dk, new[layer, 1], heads * dk, ints(seqs), ints(starts),
                                len(seqs), len(seqs) * each)
        for i, s in enumerate(seqs):
            history[s] = history[s] + [new[:, :, i * each + j].double().cpu().numpy() for j in range(each)]
        torch.cuda.synchronize()
        x.raw = x.c.tensors[0].cpu().numpy().copy()
        for layer in range(layers):
            q = check_attention(x.c, x.b.lens, [each] * len(seqs), seqs, G, kind, True, 0, layer=layer, seed=layer)
            assert q <= 1
            for s in seqs:  # the pages hold what the rows are held as
                want = [np.stack([R.held(t[layer, w].reshape(heads, dk)) for t in history[s]], 1) for w in (0, 1)]
                got = R.Pages(x.raw[layer].reshape(-1), page, heads, dk).read(x.c.tensors[1][s].cpu().numpy(), len(history[s]))
                assert np.array_equal(want[0], got[0]) and np.array_equal(want[1], got[1])

    x.grow([0], [21])
    give([0], 21)
    x.fork([0] * (beams - 1), list(range(1, beams)), [21] * (beams - 1))
    for s in range(1, beams):
        history[s] = list(history[0])
    live = list(range(beams))
    for step in range(14):
        x.grow(live, [1] * beams)
        give(live, 1)
        parents = [live[i] for i in rng.integers(0, beams, beams)]
        empty = [s for s in range(2 * beams) if s not in live]
        x.fork(parents, empty[:beams], [x.b.lens[p] for p in parents])
        for p, e in zip(parents, empty):
            history[e] = list(history[p])
        x.free(live)
        live = empty[:beams]
        if step % 5 == 4:
            x.compact()


def test_steps_in_a_graph():
    """grow, append and attention captured once and replayed: lengths and pages move on the device."""
    heads, dk, page = 2, 64, 16
    lens = [5, 40, 15]
    x = Both(30, 3, 6, page, heads, dk, 1)
    x.grow([0, 1, 2], lens)
    g = torch.Generator("cuda").manual_seed(1)
    first = torch.randn((2, sum(lens), heads * dk), generator=g, device="cuda")
    append(x.c, 0, first[0], first[1], [0, 1, 2], lens)
    k, v, q = (torch.randn((3, heads * dk), generator=g, device="cuda") for _ in range(3))
    o = torch.empty_like(q)
    seqs, starts, one = ints([0, 1, 2]), ints([0, 1, 2, 3]), ints([1, 1, 1])
    work = torch.empty(P.attention_cache4_work_bytes(x.c, heads, 3, 3), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.cache4_grow_dev(x.c, seqs, one, 3, x.status, x.work)
        P.cache4_append_dev(x.c, 0, k, heads * dk, v, heads * dk, seqs, starts, 3, 3)
        P.attention_cache4_dev(o, heads * dk, q, heads * dk, heads, x.c, 0, seqs, starts, 3, 3, 1, 0.125, True, 0, work)
    for step in range(20):
        for t in (k, v, q):
            t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        assert x.b.grow([0, 1, 2], [1, 1, 1]) == int(x.status) == 0
        x.raw = x.c.tensors[0].cpu().numpy().copy()
        x.same(0)
        for s in range(3):
            kk, vv = R.Pages(x.raw[0].reshape(-1), page, heads, dk).read(x.c.tensors[1][s].cpu().numpy(), lens[s] + step + 1)
            y, size, score = R.attention(q[s:s + 1].double().cpu().numpy().reshape(1, heads, dk), kk, vv, kk.shape[1], 0.125, True, 0)
            assert np.array_equal(kk[:, -1], R.held(k[s].double().cpu().numpy().reshape(heads, dk)))
            assert np.abs(o[s].double().cpu().numpy().reshape(y.shape) - y).max() <= 1e-5 * (1 + score.max()) * size.max()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_chunked_prompt_in_a_graph(kind):
    """A chunk of 160 rows a replay: pages taken, rows appended and attended, lengths and pages moving on the device."""
    heads, dk, G, page, n = 2, 64, 2, 16, 160
    x = Both(80, 2, 40, page, heads, dk, 1)
    g = torch.Generator("cuda").manual_seed(4)
    k, v = torch.empty((2, n, heads * dk), device="cuda").to(KIND[kind])
    q = torch.empty((n, G * heads * dk), device="cuda").to(KIND[kind])
    o = torch.empty_like(q)
    seqs, starts, add = ints([1]), ints([0, n]), ints([n])
    work = torch.empty(P.attention_cache4_work_bytes(x.c, G * heads, n, 1), dtype=torch.uint8, device="cuda")

    def step(to):
        P.attention_cache4_dev(to, G * heads * dk, q, G * heads * dk, G * heads, x.c, 0, seqs, starts, 1, n, n, 0.125, True, 200, work)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.cache4_grow_dev(x.c, seqs, add, 1, x.status, x.work)
        P.cache4_append_dev(x.c, 0, k, heads * dk, v, heads * dk, seqs, starts, 1, n)
        step(o)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert x.b.grow([1], [n]) == 0
        x.raw = x.c.tensors[0].cpu().numpy().copy()
        x.same(0)
        again = torch.empty_like(o)
        step(again)
        no_errors()
        assert torch.equal(o, again)
        assert check_attention(x.c, x.b.lens, [n], [1], G, kind, True, 200, scale=0.125, q=q) <= 1
    graph.replay()  # 640 tokens are all that a table row has room for
    torch.cuda.synchronize()
    assert int(x.status) == P.CACHE4_LONG and P.device_errors(0) == 0


def test_two_streams_with_work_areas_of_their_own():
    lens = [3000, 700]
    c = filled(lens, 64, 2, 128, seed=12)
    want, got, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = []
    for i in range(2):
        q = torch.randn((2, 4 * 128), generator=torch.Generator("cuda").manual_seed(i), device="cuda").bfloat16()
        calls.append((q, torch.empty_like(q), torch.empty(P.attention_cache4_work_bytes(c, 4, 2, 2), dtype=torch.uint8, device="cuda")))
    seqs, starts = ints([0, 1]), ints([0, 1, 2])

    def call(i):
        q, o, work = calls[i]
        P.attention_cache4_dev(o, 512, q, 512, 4, c, 0, seqs, starts, 2, 2, 1, 0.1, True, 0, work)
    for i in range(2):
        call(i)
        torch.cuda.synchronize()
        want.append(calls[i][1].clone())
    for _ in range(20):
        for i in range(2):
            calls[i][1].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                call(i)
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(calls[i][1], want[i])  # the same bits, whatever runs beside it
