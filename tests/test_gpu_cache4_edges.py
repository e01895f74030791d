"""The 4-bit cache and its attention on a B200 where they go wrong most easily:
precision, ranges, shared and full pages. The helpers, and what each
tolerance is made of, are test_gpu_cache4's."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import libpktito_b200 as P
from tests import cache4_ref as R
from tests import test_gpu_cache4 as T

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_device")]


@pytest.mark.parametrize("dk,G,rows", [(32, 1, 1), (64, 4, 1), (128, 4, 1), (128, 1, 5), (96, 4, 4), (256, 2, 1), (256, 1, 200)])
def test_weights_of_bf16_rows_have_sixteen_bits(dk, G, rows, monkeypatch):
    # two bf16 parts: each leaves at most 2^-8 of what it is taken from
    monkeypatch.setitem(T.PARTS, "bf16", 2.0 ** -16)
    lens = [3000, 700, 260]
    c = T.filled(lens, 32, 2, dk, seed=dk + rows)
    T.check_attention(c, lens, [rows] * 3, [1, 0, 2], G, "bf16", True, 0)
    T.check_attention(c, lens, [rows] * 3, [0, 2, 1], G, "bf16", False, 0, scale=0.05)


def two_layers_of_four(kind="f32", page=16):
    """Books with sequences 0 (40 tokens), 1 (16) and 2 (16, a fork that shares 1's page), rows in both layers, and no page left."""
    x = T.Both(5, 4, 3, page, 2, 64, 2)
    assert x.grow([0, 1], [40, 16]) == 0
    g = torch.Generator("cuda").manual_seed(3)
    for layer in range(2):
        k, v = torch.randn((2, 56, 128), generator=g, device="cuda").to(T.KIND[kind])
        T.append(x.c, layer, k, v, [0, 1], [40, 16])
    x.raw = x.c.tensors[0].cpu().numpy().copy()
    assert x.fork([1], [2], [16]) == 0 and x.grow([3], [5]) == 0
    return x, g


@pytest.mark.parametrize("add,status", [([1, 1, 1], R.Books.FULL), ([9, 0, 0], R.Books.LONG), ([0, -1, 0], R.Books.BAD)])
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("each", [1, 3])
def test_a_step_that_found_no_room_leaves_every_token(add, status, graph, each):
    # grow, append and attention in a row, as a decoder runs them: rows for tokens that were not taken go nowhere
    x, g = two_layers_of_four()
    n, seqs, add = 3 * each, T.ints([0, 1, 2]), T.ints(add)
    k, v, q = torch.randn((3, n, 128), generator=g, device="cuda")
    o, starts = torch.empty_like(q), T.ints([0, each, 2 * each, n])
    work = torch.empty(P.attention_cache4_work_bytes(x.c, 2, n, 3), dtype=torch.uint8, device="cuda")

    def step():
        P.cache4_grow_dev(x.c, seqs, add, 3, x.status, x.work)
        for layer in range(2):
            P.cache4_append_dev(x.c, layer, k, 128, v, 128, seqs, starts, 3, n, status=x.status)
            P.attention_cache4_dev(o, 128, q, 128, 2, x.c, layer, seqs, starts, 3, n, each, 0.125, True, 0, work)
    if graph:
        replay = torch.cuda.CUDAGraph()
        with torch.cuda.graph(replay):
            step()
        step = replay.replay
    step()
    assert x.b.grow([0, 1, 2], add.tolist()) == status
    x.same(status)  # books, and every byte of every page
    x.free([3])
    x.free([2])
    add.copy_(T.ints([1, 1, 0]))
    seqs[2] = 3  # empty: none of its rows is a token
    starts.copy_(T.ints([0, 1, 2, 2]))
    step()
    assert x.b.grow([0, 1, 3], [1, 1, 0]) == 0
    T.no_errors()
    assert int(x.status) == 0
    for layer in range(2):
        pages = R.Pages(x.c.tensors[0][layer].cpu().numpy().reshape(-1), 16, 2, 64)
        for i, s in enumerate((0, 1)):
            kk, vv = pages.read(x.c.tensors[1][s].cpu().numpy(), x.b.lens[s])
            assert np.array_equal(kk[:, -1], R.held(k[i].double().cpu().numpy().reshape(2, 64)))
            assert np.array_equal(vv[:, -1], R.held(v[i].double().cpu().numpy().reshape(2, 64)))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_a_page_that_others_hold_keeps_its_bytes(kind):
    x, g = two_layers_of_four(kind)
    k, v = torch.randn((2, 5, 128), generator=g, device="cuda").to(T.KIND[kind])
    P.cache4_append_dev(x.c, 1, k, 128, v, 128, T.ints([1, 0, 2]), T.ints([0, 2, 3, 5]), 3, 5)
    torch.cuda.synchronize()
    assert P.device_errors(0) == 2
    pages = R.Pages(x.raw[1].reshape(-1), 16, 2, 64)  # sequence 0's row is written, those of 1 and 2 are not
    for which, y in enumerate((k, v)):
        pages.write(x.b.rows[0][2], 39 % 16, which, *R.quantize(y[2].double().cpu().numpy().reshape(2, 64)))
    x.raw[1] = pages.raw.reshape(x.raw[1].shape)
    x.status.zero_()
    x.same(0)
    x.free([2])  # alone again
    P.cache4_append_dev(x.c, 1, k, 128, v, 128, T.ints([1]), T.ints([0, 2]), 1, 5)
    T.no_errors()
    assert not np.array_equal(x.c.tensors[0].cpu().numpy(), x.raw)


SHORT_WAITS = """
import time, torch
import libpktito_b200 as P
from tests import test_gpu_cache4 as T
lens = [40011, 5, 9000, 0, 700]
c = T.filled(lens, 64, 4, 128, seed=3)
P.device_errors(0)
cold, seen = torch.empty(256 << 20, dtype=torch.uint8, device="cuda"), 0
for kind, G, each in (("bf16", 4, 1), ("f32", 1, 3), ("f16", 2, 9)) * 4:
    H, n = 4 * G, 5 * each
    q = torch.randn((n, H * 128), device="cuda").to(T.KIND[kind])
    o = torch.full((n + 3, H * 128 + 8), 5.0, device="cuda").to(T.KIND[kind])
    size = P.attention_cache4_work_bytes(c, H, n, 5)
    work = torch.zeros((size + 4096,), dtype=torch.uint8, device="cuda")
    cold.fill_(1)
    torch.cuda.synchronize()
    t = time.perf_counter()
    P.attention_cache4_dev(o, H * 128 + 8, q, H * 128, H, c, 0, T.ints([0, 1, 2, 3, 4]), T.ints([each * i for i in range(6)]), 5, n, each,
                           0.1, True, 0, work[:size])
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    word = P.device_errors(0)
    assert word in (0, 1), word
    assert not word or t < 0.5, t  # nobody waits for copies that were never asked for, a second each
    assert (work[size:] == 0).all() and (o[n:] == 5).all() and (o[:, H * 128:] == 5).all()
    assert (o[3 * each:4 * each, :H * 128] == 0).all()  # no tokens: zeros, whatever became of the others
    if not word:
        assert T.check_attention(c, lens, [each] * 5, [0, 1, 2, 3, 4], G, kind, True, 0, scale=0.1) <= 1
    seen += word
print("gave up", seen, "of 12")
"""


def test_short_waits_end_in_results_or_in_an_error():
    # a process whose waits may last one cycle: what gives up says so, and nothing is read that the call did not write
    r = subprocess.run([sys.executable, "-c", SHORT_WAITS], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PKB_WAIT_CYCLES="1"), cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,G,rows,at,causal_window", [(64, 2, 5, 268, 0), (128, 1, 40, 250, 17), (32, 1, 200, 150, 0), (128, 4, 150, 200, 0),
                                                        (64, 1, 260, 30, 25), (256, 2, 70, 230, 9), (96, 1, 270, 133, 50)])
def test_a_huge_value_reaches_the_rows_that_see_it_alone(kind, dk, G, rows, at, causal_window):
    # masked weights are 0, so a held value has to be finite in the product: 0 times an infinity is a NaN
    L, heads = 270, 2
    c = T.make([L], 32, heads, dk, seed=5)
    g = torch.Generator("cuda").manual_seed(5)
    k, v = torch.randn((2, L, heads * dk), generator=g, device="cuda")
    q = torch.randn((rows, heads * G * dk), generator=g, device="cuda").to(T.KIND[kind])
    work = torch.empty(P.attention_cache4_work_bytes(c, heads * G, rows, 1), dtype=torch.uint8, device="cuda")

    def run():
        T.append(c, 0, k, v, [0], [L])
        o = torch.empty_like(q)
        P.attention_cache4_dev(o, heads * G * dk, q, heads * G * dk, heads * G, c, 0, T.ints([0]), T.ints([0, rows]), 1, rows, rows,
                               dk ** -0.5, True, causal_window, work)
        T.no_errors()
        return o
    clean = run()
    v[at, 3], v[at, dk] = 3.3e38, -2.0 ** 126
    got = run()
    pos = L - rows + torch.arange(rows, device="cuda")
    sees = (pos >= at) & ((pos < at + causal_window) if causal_window else True)
    assert sees.any() and not sees.all()
    assert torch.equal(got[~sees], clean[~sees])
    assert not torch.equal(got[sees], clean[sees])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,G,rows", [(32, 1, 1), (64, 4, 1), (128, 8, 1), (96, 3, 4), (128, 1, 40), (256, 2, 1), (256, 1, 200), (64, 1, 300)])
def test_sums_are_as_exact_as_what_they_add(kind, dk, G, rows):
    # half of q is large and of one sign, and meets zeros of K: what it does not add may not cost bits of what the rest does
    lens, heads = [700, 320], 2
    c = T.make(lens, 32, heads, dk, seed=dk)
    g = torch.Generator("cuda").manual_seed(dk + rows)
    k, v = torch.randn((2, sum(lens), heads * dk), generator=g, device="cuda")
    k[:, ::2] = 0
    T.append(c, 0, k, v, [0, 1], lens)
    q = torch.randn((2 * rows, heads * G * dk), generator=g, device="cuda") * 2.0 ** -9
    q[:, ::2] = 1
    T.check_attention(c, lens, [rows] * 2, [1, 0], G, kind, True, 0, scale=2.0 ** 9 * 2 / (dk / 2) ** 0.5, q=q.to(T.KIND[kind]))


@pytest.mark.parametrize("kind,big,small,scale", [(k, *x) for x in [(124, -13, -111), (107, 0, -107), (124, -100, -24), (-118, 10, 108)]
                                                  for k in ("f32", "f16", "bf16") if k != "f16" or x[1] > -14])  # where f16 rows end
@pytest.mark.parametrize("dk,G,rows", [(32, 1, 1), (64, 4, 1), (128, 8, 1), (96, 3, 4), (128, 1, 40), (256, 2, 1), (256, 1, 200), (64, 1, 300)])
def test_keys_of_any_size(kind, dk, G, rows, big, small, scale):
    # keys of some 2^big, queries of 2^small and a scale that makes scores of them: what a float holds comes out right
    lens, heads = [300, 303], 1
    c = T.make(lens, 32, heads, dk, seed=dk)
    g = torch.Generator("cuda").manual_seed(dk + rows)
    k, v = torch.randn((2, sum(lens), heads * dk), generator=g, device="cuda").clamp_(-3.5, 3.5)
    T.append(c, 0, k * 2.0 ** big, v, [0, 1], lens)
    q = (torch.randn((2 * rows, heads * G * dk), generator=g, device="cuda") * 2.0 ** small).to(T.KIND[kind])
    T.check_attention(c, lens, [rows] * 2, [1, 0], G, kind, True, 0, scale=2.0 ** scale * dk ** -0.5, q=q)


def test_large_lists_of_page_operations():
    # 1,500 sequences of up to 16 pages in a pool of 40,003: forks of hundreds, and frees of more places than one block takes
    x = T.Both(40003, 3000, 16, 16, 1, 32, 1)
    rng = np.random.default_rng(2)
    lens = rng.integers(1, 257, 1500).tolist()
    assert x.grow(list(range(1500)), lens) == 0
    assert x.free(list(range(0, 1500, 7))) == 0
    live = [s for s in range(1500) if s % 7]
    src = rng.choice(live, 1200).tolist()
    dst = rng.permutation(list(range(1500, 3000)) + list(range(0, 1500, 7)))[:1200].tolist()
    assert x.fork(src, dst, [int(rng.integers(0, lens[s] + 1)) for s in src]) == 0
    held = [d for d in dst if x.b.lens[d]]
    assert x.grow(held, [int(rng.integers(0, 257 - x.b.lens[s])) for s in held]) == 0
    gone = rng.permutation(live)[:1100].tolist()
    assert len(gone) * 16 > 16384
    assert x.free(gone + gone[:1]) == x.free(gone + [3000]) == R.Books.BAD  # nothing of it
    assert x.free(gone) == 0  # pages that forks hold stay
    x.compact()
    assert x.free(rng.permutation(dst).tolist()) == 0
    assert x.copy([s for s in live if s not in set(gone)][:50], gone[:50], [0] * 50) == 0
    x.compact()
    assert x.free([s for s in range(3000)]) == 0 and int(x.c.tensors[3].sum()) == 0


FIRST_CALLS = """
import sys, torch
import libpktito_b200 as P
from tests import test_gpu_cache4 as T
kind, rows = sys.argv[1], int(sys.argv[2])
c = T.filled([300, 270], 32, 2, 64, seed=1)
q = torch.randn((2 * rows, 256), device="cuda").to(T.KIND[kind])
o, again = torch.empty_like(q), torch.empty_like(q)
work = torch.empty(P.attention_cache4_work_bytes(c, 4, 2 * rows, 2), dtype=torch.uint8, device="cuda")
seqs, starts = T.ints([0, 1]), T.ints([0, rows, 2 * rows])
torch.cuda.synchronize()

def call(to):
    P.attention_cache4_dev(to, 256, q, 256, 4, c, 0, seqs, starts, 2, 2 * rows, rows, 0.125, True, 0, work)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call(o)
graph.replay()
call(again)
T.no_errors()
assert torch.equal(o, again)
assert T.check_attention(c, [300, 270], [rows] * 2, [0, 1], 2, kind, True, 0, scale=0.125, q=q) <= 1
"""


@pytest.mark.parametrize("kind,rows", [("f32", 1), ("bf16", 200), ("f16", 200)])
def test_a_process_first_attention_may_be_a_captured_one(kind, rows):
    # the kernels are set up by the first call, here inside a capture
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS, kind, str(rows)], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dk,G", [(128, 1), (96, 3), (32, 8)])
@pytest.mark.parametrize("rows", [8, 9, 16, 17, 24, 25, 32, 33, 40, 41, 48, 64, 65, 127, 128, 129])
def test_every_way_rows_are_put_into_blocks(kind, dk, G, rows):
    # of query heads and tokens; as few sequences as are split along the keys, and as many as may not be
    most = -(-rows // G)
    lens = [most + 40, 333, 1]
    c = T.filled(lens, 32, 2, dk, seed=rows)
    T.check_attention(c, lens, [most, max(1, most - 3), 1], [1, 0, 2], G, kind, True, 0)
    many = [1 + (37 * i) % 150 for i in range(60)]
    c = T.filled(many, 32, 3, dk, seed=rows)
    T.check_attention(c, many, [most if i % 3 == 0 else 1 for i in range(60)], list(range(60)), G, kind, True, 20)
