"""Calls of windows, drafted trees and beams that share things: a buffer that is both input and output, one slot read by
several sequences, graphs of several calls over one workspace, padded trees joined from many parts, bases at an int's end.
What has a plain counterpart is compared bit for bit, the rest with float64."""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8, Kv
from test_gpu_tree import ancestors, attend, close, i32, masks, random_tree

pytestmark = pytest.mark.gpu

TUNE_ATTN_PROMPT = 21


@pytest.fixture(params=[1, 2, 3], ids=["direct", "tiled256", "tiled128"])
def kernel(gpu, request):
    gpu.tune(TUNE_ATTN_PROMPT, request.param)
    yield request.param
    gpu.tune(TUNE_ATTN_PROMPT, 0)


@pytest.mark.parametrize("n,max_seq", [(3, 3000), (40, 500)])
def test_trees_in_place(gpu, kernel, n, max_seq):
    """out is q: in parts and in one."""
    H, KVH, hd, N = 28, 4, 128, 19
    rng = np.random.default_rng(n)
    c = ref.Cache(gpu, KV_Q8, n, max_seq, KVH, hd, rng)
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    seen = np.stack([masks(ancestors(random_tree(rng, int(rng.integers(1, N + 1)), N))) for _ in range(n)])
    base, ds = i32(gpu, rng.integers(0, max_seq - N, n)), gpu.upload(seen)
    dq, out = gpu.upload(q), gpu.alloc(q.nbytes)
    gpu.attn_tree(out, H * hd, dq, H * hd, c.kv, None, base, ds, n, N, H, 0.09)
    gpu.attn_tree(dq, H * hd, dq, H * hd, c.kv, None, base, ds, n, N, H, 0.09)
    assert np.array_equal(gpu.download(out, np.float32, q.shape), gpu.download(dq, np.float32, q.shape))
    for b in (base, ds, dq, out):
        b.free()
    c.free()


def test_windows_in_place(gpu, kernel):
    H, KVH, hd, n = 14, 2, 64, 5
    rng = np.random.default_rng(2)
    c = ref.Cache(gpu, KV_F16, n, 2500, KVH, hd, rng)
    lens, start = np.array([700, 1, 33, 1200, 64], np.int32), np.array([1800, 0, 5, 900, 31], np.int32)
    q = rng.standard_normal((int(lens.sum()), H, hd)).astype(np.float32)
    dq, out = gpu.upload(q), gpu.alloc(q.nbytes)
    for to in (out, dq):
        gpu.attn_prompt_window(to, H * hd, dq, H * hd, c.kv, None, start, lens, n, H, 0.09, 300, 4)
    assert np.array_equal(gpu.download(out, np.float32, q.shape), gpu.download(dq, np.float32, q.shape))
    dl = i32(gpu, start + lens)
    gpu.h2d(dq, q)
    for to in (out, dq):
        gpu.attn_decode_window(to, H * hd, dq, H * hd, c.kv, None, dl, n, H, 0.09, 1500, 4)
    assert np.array_equal(gpu.download(out, np.float32, (n, H, hd)), gpu.download(dq, np.float32, (n, H, hd)))
    for b in (dq, out, dl):
        b.free()
    c.free()


def test_sequences_of_one_slot(gpu, kernel):
    """Two trees and two tokens may read one slot."""
    H, KVH, hd, N, max_seq = 8, 2, 64, 11, 400
    rng = np.random.default_rng(3)
    c = ref.Cache(gpu, KV_Q8, 2, max_seq, KVH, hd, rng)
    K, V = c.values()
    slot, base = [1, 0, 1, 1], [200, 77, 200, 131]
    n = len(slot)
    sets = [ancestors(random_tree(rng, N, N)) for _ in slot]
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    bufs = [gpu.upload(q), gpu.alloc(q.nbytes), i32(gpu, slot), i32(gpu, base), gpu.upload(np.stack([masks(s) for s in sets]))]
    gpu.attn_tree(bufs[1], H * hd, bufs[0], H * hd, c.kv, bufs[2], bufs[3], bufs[4], n, N, H, 0.1)
    got = gpu.download(bufs[1], np.float32, (n, N, H, hd))
    for i in range(n):
        close(got[i], np.array([attend(q[i * N + j], K, V, slot[i], base[i], sets[i][j], max_seq, 0.1) for j in range(N)]))
    gpu.attn_decode_window(bufs[1], H * hd, bufs[0], H * hd, c.kv, bufs[2], bufs[3], n, H, 0.1, 60, 3)
    got = gpu.download(bufs[1], np.float32, (n, H, hd))
    assert np.isfinite(got).all()
    gpu.attn_decode_window(bufs[1], H * hd, gpu_row(gpu, bufs, q[2]), H * hd, c.kv, bufs[2], bufs[3], 1, H, 0.1, 60, 3)
    assert np.array_equal(gpu.download(bufs[1], np.float32, (H, hd)), got[2])   # (both 200 positions of slot 1)
    for b in bufs:
        b.free()
    c.free()


def gpu_row(gpu, bufs, row):
    bufs.append(gpu.upload(np.ascontiguousarray(row)))
    return bufs[-1]


@pytest.mark.parametrize("n,N,nodes,H,KVH", [(1, 40, 3, 28, 4), (2, 64, 17, 16, 2), (3, 64, 33, 28, 4), (5, 7, 2, 28, 4)])
def test_padded_trees_in_parts(gpu, kernel, n, N, nodes, H, KVH):
    """Nodes that are not there are zeros, whatever was in the outputs and in the parts' sums of the call before."""
    hd, max_seq = 128, 4100
    rng = np.random.default_rng(N)
    c = ref.Cache(gpu, KV_Q8, n + 1, max_seq, KVH, hd, rng)
    K, V = c.values()
    base = [int(b) for b in rng.integers(2000, 4000, n)]
    full = gpu.upload(np.stack([masks(ancestors(random_tree(rng, N, N)))] * n))
    sets = [ancestors(random_tree(rng, nodes, N)) for _ in base]
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    q[1] = np.nan                                                                  # (of a node that is there)
    bufs = [gpu.upload(q), gpu.alloc(q.nbytes), i32(gpu, base), gpu.upload(np.stack([masks(s) for s in sets]))]
    gpu.attn_tree(bufs[1], H * hd, bufs[0], H * hd, c.kv, None, bufs[2], full, n, N, H, 0.09)
    gpu.attn_tree(bufs[1], H * hd, bufs[0], H * hd, c.kv, None, bufs[2], bufs[3], n, N, H, 0.09)
    got = gpu.download(bufs[1], np.float32, (n, N, H, hd))
    assert np.isnan(got[0, 1]).all()
    got[0, 1] = 0.0
    for i in range(n):
        for j in range(N):
            if not sets[i][j]:
                assert (got[i, j] == 0.0).all()
            elif (i, j) != (0, 1) and j in (0, nodes // 2, nodes - 1):
                close(got[i, j], attend(q[i * N + j], K, V, i, base[i], sets[i][j], max_seq, 0.09))
    for b in bufs + [full]:
        b.free()
    c.free()


def test_graphs_share_a_workspace(gpu):
    """Graphs of a small tree, a window, a selection; then larger calls, which take the workspaces anew; then each graph
    between other calls, several times: the bits of its eager call."""
    H, KVH, hd, n, N, V = 28, 4, 128, 2, 13, 5003
    rng = np.random.default_rng(8)
    c = ref.Cache(gpu, KV_Q8, 16, 4000, KVH, hd, rng)
    D = H * hd
    q = rng.standard_normal((16 * 64, D)).astype(np.float32)
    logits = rng.standard_normal((64, V)).astype(np.float32)
    dq, out, big = gpu.upload(q), gpu.alloc(4 * n * N * D), gpu.alloc(q.nbytes)
    base, ends = i32(gpu, [3000, 1234] + [3900] * 14), i32(gpu, [3000, 17] + [4000] * 14)
    seen = gpu.upload(np.full((16, 64), 2 ** 64 - 1, np.uint64))
    dx, score = gpu.upload(logits), gpu.upload(np.zeros(64, np.float32))
    par, tok, val = gpu.alloc(4 * 64), gpu.alloc(4 * 64), gpu.alloc(4 * 64)
    calls = {
        "tree": lambda: gpu.attn_tree(out, D, dq, D, c.kv, None, base, seen, n, N, H, 0.09),
        "window": lambda: gpu.attn_decode_window(out, D, dq, D, c.kv, None, ends, n, H, 0.09, 2900, 4),
        "select": lambda: gpu.beam_select(dx, V, V, score, None, -1, 1, 4, 4, False, par, tok, val),
    }

    def larger():
        gpu.attn_tree(big, D, dq, D, c.kv, None, base, seen, 16, 64, H, 0.09)
        gpu.attn_tree(big, D, dq, D, c.kv, None, base, seen, 3, 64, H, 0.09)
        gpu.beam_select(dx, V, V, score, None, -1, 4, 16, 32, False, big, gpu_at(big, 1), gpu_at(big, 2))

    def gpu_at(buf, k):
        return buf.offset(65536 * k)

    def results(name):
        if name == "select":
            return [gpu.download(b, np.int32, 4) for b in (par, tok, val)]
        return [gpu.download(out, np.uint32, (n * N if name == "tree" else n) * D)]

    def spoil():
        gpu.h2d(out, np.full(n * N * D, 5, np.float32))
        for b in (par, tok, val):
            gpu.h2d(b, np.full(64, 77, np.int32))

    want, graphs = {}, {}
    for name, call in calls.items():
        call()
        want[name] = results(name)
        gpu.capture_begin()
        call()
        graphs[name] = gpu.capture_end()
    for step in range(3):
        larger()
        for name in ("select", "tree", "window", "tree"):
            spoil()
            if step == 1:
                larger()
            gpu.graph_launch(graphs[name])
            for a, b in zip(results(name), want[name]):
                assert np.array_equal(a, b), (step, name)
    for g in graphs.values():
        gpu.graph_destroy(g)
    for b in (dq, out, big, base, ends, seen, dx, score, par, tok, val):
        b.free()
    c.free()


@pytest.mark.parametrize("first", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 31 - 64])
def test_bases_at_an_ints_end(gpu, first):
    """A plan's rows and turns past it are none; the attention takes such a base for the cache's end."""
    N, H, KVH, hd, max_seq = 6, 4, 2, 64, 100
    rng = np.random.default_rng(4)
    parents = [-1, 0, 1, 1, 3, 0]
    sets = ancestors(parents)
    base, dp = i32(gpu, [first]), i32(gpu, parents)
    seen, row, turn = gpu.alloc(8 * N), gpu.alloc(4 * N), gpu.alloc(4 * N)
    gpu.tree_plan(None, base, dp, 1, N, seen, None, row, turn)

    def place(k):
        return first + k if first + k < 2 ** 31 else -1

    assert list(gpu.download(row, np.int32, N)) == [place(j) for j in range(N)]
    assert list(gpu.download(turn, np.int32, N)) == [place(len(s) - 1) for s in sets]
    assert np.array_equal(gpu.download(seen, np.uint64, N), masks(sets))
    c = ref.Cache(gpu, KV_Q8, 1, max_seq, KVH, hd, rng)
    K, V = c.values()
    q = rng.standard_normal((N, H, hd)).astype(np.float32)
    dq, out = gpu.upload(q), gpu.alloc(q.nbytes)
    gpu.attn_tree(out, H * hd, dq, H * hd, c.kv, None, base, seen, 1, N, H, 1 / math.sqrt(hd))
    got = gpu.download(out, np.float32, q.shape)
    close(got, np.array([attend(q[j], K, V, 0, max_seq, sets[j], max_seq, 1 / math.sqrt(hd)) for j in range(N)]))
    kv, before = gpu.kv_layers([c.kv]), c.pull()
    path, count = i32(gpu, [2, 0, 1, -1, -1, -1]), i32(gpu, [3])
    gpu.kv_keep(kv, None, base, path, count, 1, N)
    for a, b in zip(c.pull(), before):
        assert np.array_equal(a, b)
    for b in (base, dp, seen, row, turn, dq, out, path, count):
        b.free()
    c.free()


def test_calls_of_nothing(gpu):
    """No sequences, no requests: no work, and the arrays may be null where they hold nothing."""
    c = ref.Cache(gpu, KV_F16, 1, 64, 1, 64, np.random.default_rng(0))
    one, kv = gpu.alloc(4096), gpu.kv_layers([c.kv])
    gpu.attn_tree(one, 64, one, 64, c.kv, None, None, None, 0, 5, 1, 1.0)
    gpu.attn_decode_window(one, 64, one, 64, c.kv, None, None, 0, 1, 1.0, 5, 0)
    gpu.attn_prompt_window(one, 64, one, 64, c.kv, None, None, None, 0, 1, 1.0, 5, 0)
    gpu.tree_plan(None, None, None, 0, 3)
    gpu.tree_accept(None, None, None, None, 0, 3, None, None, None)
    gpu.kv_keep(kv, None, None, None, None, 0, 3)
    gpu.kv_reorder(kv, None, None, 0, 4, None, None)
    gpu.beam_select(one, 8, 8, one, None, -1, 0, 2, 2, False, one, one, one)
    gpu.sync()
    one.free()
    c.free()


def test_offsets_past_32_bits(gpu):
    """A cache of 5 GiB an array: rows of its last slot appended, moved, reordered and attended to."""
    slots, max_seq, KVH, hd, H, n, at = 80, 32768, 8, 128, 16, 24, 32700
    rng = np.random.default_rng(11)
    kv = Kv(KV_F16, slots, max_seq, KVH, hd)
    codes, scales = gpu.kv_bytes(kv)
    assert codes > 2 ** 32
    arrays = [gpu.alloc(b) for b in (codes, codes, scales, scales)]
    kv = Kv(KV_F16, slots, max_seq, KVH, hd, *(b.ptr for b in arrays))
    W = KVH * hd

    def write(slot, pos):
        x = [gpu.upload(rng.standard_normal((n, W)).astype(np.float32)) for _ in range(2)]
        ds, dp = i32(gpu, [slot] * n), i32(gpu, range(pos, pos + n))
        gpu.kv_append(kv, ds, dp, n, *x, W)
        for b in x + [ds, dp]:
            b.free()

    def read(slot, pos):
        out = [gpu.alloc(4 * n * W) for _ in range(2)]
        ds, dp = i32(gpu, [slot] * n), i32(gpu, range(pos, pos + n))
        gpu.kv_read(kv, ds, dp, n, *out, W)
        got = [gpu.download(b, np.float32, (n, KVH, hd)) for b in out]
        for b in out + [ds, dp]:
            b.free()
        return got

    for slot in (79, 78, 3):
        write(slot, at)
    write(79, 0)
    layers = gpu.kv_layers([kv])
    before = {s: read(s, at) for s in (79, 78, 3)}
    # two requests: slots 79 and 3 change places, 78 takes nothing from a beam outside
    ds, par, since, end = i32(gpu, [79, 3]), i32(gpu, [1, 0]), i32(gpu, [at]), i32(gpu, [at + n])
    gpu.kv_reorder(layers, ds, par, 1, 2, since, end)
    for a, b in ((79, 3), (3, 79), (78, 78)):
        for x, y in zip(read(a, at), before[b]):
            assert np.array_equal(x, y)
    base, path, count = i32(gpu, [at]), i32(gpu, [0, 3, 7, 20] + [-1] * (n - 4)), i32(gpu, [4])
    gpu.kv_keep(layers, ds, base, path, count, 1, n)
    kept = read(79, at)
    for x, y in zip(kept, before[3]):
        assert np.array_equal(x[:4], y[[0, 3, 7, 20]]) and np.array_equal(x[4:], y[4:])
    # the last positions under a window, and a tree near the slot's start
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    dq, out, scale = gpu.upload(q), gpu.alloc(q.nbytes), 1 / math.sqrt(hd)
    gpu.attn_decode_window(out, H * hd, dq, H * hd, kv, ds, end, 1, H, scale, 15, 0)
    K, V = (np.moveaxis(x.astype(np.float64), 0, 1)[None] for x in kept)
    close(gpu.download(out, np.float32, (H, hd)), attend(q[0], K[:, :, n - 15:], V[:, :, n - 15:], 0, 15, {1}, 15, scale))
    K, V = (np.moveaxis(x.astype(np.float64), 0, 1)[None] for x in read(79, 0))
    sets = ancestors(random_tree(rng, 9, 9))
    seen, first = gpu.upload(masks(sets)), i32(gpu, [15])
    for knob in (1, 2, 3):
        gpu.tune(TUNE_ATTN_PROMPT, knob)
        gpu.attn_tree(out, H * hd, dq, H * hd, kv, ds, first, seen, 1, 9, H, scale)
        got = gpu.download(out, np.float32, (9, H, hd))
        close(got, np.array([attend(q[j], K, V, 0, 15, sets[j], n, scale) for j in range(9)]))
    gpu.tune(TUNE_ATTN_PROMPT, 0)
    for b in arrays + [ds, par, since, end, base, path, count, dq, out, seen, first]:
        b.free()
