"""Trees of drafted tokens (include/hako_attn.h, include/hako_search.h): attention against float64 on the same cached
values (bound and derivation of test_gpu_attn.py), whole numbers and moved rows exactly."""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8, Rope

pytestmark = pytest.mark.gpu

TUNE_ATTN_PROMPT = 21
TOL = 1e-5
KINDS = [KV_Q8, KV_F16]


@pytest.fixture(params=[1, 2, 3], ids=["direct", "tiled256", "tiled128"])
def kernel(gpu, request):
    """Each kernel of the attention in turn."""
    gpu.tune(TUNE_ATTN_PROMPT, request.param)
    yield request.param
    gpu.tune(TUNE_ATTN_PROMPT, 0)


def close(got, want):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    top = np.nanmax(np.abs(want), initial=0.0)
    err = np.nanmax(np.abs(got - want), initial=0.0)
    assert err <= TOL * top, f"error {err:.3g} of {top:.3g}"


def i32(gpu, v):
    return gpu.upload(np.asarray(v, np.int32))


def random_tree(rng, n, N):
    """Parents of n nodes, the rest of N not there."""
    return [-1] + [int(rng.integers(max(0, j - 12), j)) for j in range(1, n)] + [-2] * (N - n)


def ancestors(parents):
    """Sets of nodes by the definition: none from the first bad parent on."""
    out = []
    for j, p in enumerate(parents):
        if p < -1 or p >= j:
            break
        out.append({j} | (out[p] if p >= 0 else set()))
    return out + [set()] * (len(parents) - len(out))


def masks(sets):
    return np.array([sum(1 << i for i in s) for s in sets], np.uint64)


def attend(q, K, V, slot, base, seen, max_seq, scale, prefix_slot=0, prefix_len=0):
    H, hd = q.shape
    G, out = H // K.shape[1], np.zeros(q.shape)
    if not seen:
        return out
    base = min(base, max_seq)
    p = np.array(list(range(base)) + [base + i for i in sorted(seen) if base + i < max_seq], int)
    if not len(p):
        return out
    sl = np.where(p < prefix_len, prefix_slot, slot)
    for g in range(K.shape[1]):
        s = q[g * G:(g + 1) * G].astype(np.float64) @ K[sl, g, p].T * scale
        w = np.exp(s - s.max(1, keepdims=True))
        out[g * G:(g + 1) * G] = w @ V[sl, g, p] / w.sum(1, keepdims=True)
    return out


def run_tree(gpu, c, q, slot, base, seen, N, scale, prefix=(0, 0), ldo=None):
    n, H, hd = len(base), *q.shape[1:]
    D = H * hd
    ldo = ldo or D
    out = gpu.upload(np.full((n * N + 1, ldo), 7.0, np.float32))
    bufs = [gpu.upload(q), i32(gpu, base), gpu.upload(seen)] + ([] if slot is None else [i32(gpu, slot)])
    gpu.attn_tree(out, ldo, bufs[0], D, c.kv, None if slot is None else bufs[3], bufs[1], bufs[2], n, N, H, scale, *prefix)
    got = gpu.download(out, np.float32, (n * N + 1, ldo))
    for b in bufs + [out]:
        b.free()
    assert (got[:, D:] == 7.0).all() and (got[-1] == 7.0).all()
    return got[:-1, :D].reshape(n, N, H, hd)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,KVH,hd", [(28, 4, 128), (16, 1, 64), (4, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("N", [1, 2, 7, 26, 63, 64])
def test_attention(gpu, kernel, kind, H, KVH, hd, N):
    """Texts of none to several steps, trees whole and padded, drafted rows that cross a step, a slot's last rows, past them."""
    rng = np.random.default_rng(N * H)
    base = [0, 1, 5, 31, 32, 33, 63, 100, 129, 200, 288, 299, 300, 1000]
    n = len(base)
    c = ref.Cache(gpu, kind, n, 300, KVH, hd, rng)
    K, V = c.values()
    sets = [ancestors(random_tree(rng, int(rng.integers(1, N + 1)), N)) for _ in base]
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    slot = rng.permutation(n)
    got = run_tree(gpu, c, q, slot, base, np.stack([masks(s) for s in sets]), N, 1 / math.sqrt(hd), ldo=H * hd + 8)
    for i in range(n):
        close(got[i], np.array([attend(q[i * N + j], K, V, slot[i], base[i], sets[i][j], 300, 1 / math.sqrt(hd)) for j in range(N)]))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefix", [1, 64, 100, 101, 160])
def test_attention_over_a_prefix(gpu, kernel, kind, prefix):
    """Also bases below the prefix, whose drafted rows are then the prefix slot's."""
    H, KVH, hd, N = 28, 4, 128, 9
    rng = np.random.default_rng(prefix)
    base = [100, 101, 164, 300, 161, 350, 97]
    c = ref.Cache(gpu, kind, 8, 400, KVH, hd, rng)
    K, V = c.values()
    sets = [ancestors(random_tree(rng, N, N)) for _ in base]
    q = rng.standard_normal((len(base) * N, H, hd)).astype(np.float32)
    got = run_tree(gpu, c, q, None, base, np.stack([masks(s) for s in sets]), N, 0.1, (7, prefix))
    for i in range(len(base)):
        close(got[i], np.array([attend(q[i * N + j], K, V, i, base[i], sets[i][j], 400, 0.1, 7, prefix) for j in range(N)]))
    c.free()


@pytest.mark.parametrize("n,N,base,H,KVH", [(1, 26, 5000, 16, 2), (2, 64, 5000, 28, 4), (40, 16, 900, 28, 4), (3, 1, 5000, 8, 8)])
def test_attention_in_parts(gpu, kernel, n, N, base, H, KVH):
    hd = 128
    rng = np.random.default_rng(n)
    c = ref.Cache(gpu, KV_Q8, n, base + 100, KVH, hd, rng)
    K, V = c.values()
    bases = [base - 13 * i for i in range(n)]
    sets = [ancestors(random_tree(rng, N, N)) for _ in bases]
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    got = run_tree(gpu, c, q, None, bases, np.stack([masks(s) for s in sets]), N, 0.09)
    for i in range(0, n, max(1, n // 4)):
        for j in {0, N // 2, N - 1}:
            close(got[i, j], attend(q[i * N + j], K, V, i, bases[i], sets[i][j], base + 100, 0.09))
    c.free()


def test_masks_of_any_bits(gpu, kernel):
    """Bits past the tree are nothing; a node may see any others; NaN and huge rows reach those who see them alone."""
    H, KVH, hd, N, base = 8, 2, 128, 20, 70
    rng = np.random.default_rng(4)
    c = ref.Cache(gpu, KV_F16, 2, 128, KVH, hd, rng)
    c.vs[:, :, base + 3] = 1e20
    c.ks[1, :, base + 5] = np.nan
    c.vs[:, :, base + N:] = np.nan
    c.push()
    K, V = c.values()
    seen = rng.integers(0, 1 << 62, (2, N)).astype(np.uint64) << np.uint64(1)
    seen[:, 4] = np.uint64(2 ** 64 - 1) << np.uint64(N)          # nothing of the tree: not there
    sets = [[{i for i in range(N) if int(m) >> i & 1} for m in row] for row in seen]
    q = rng.standard_normal((2 * N, H, hd)).astype(np.float32)
    got = run_tree(gpu, c, q, None, [base, base], seen, N, 0.1)
    assert (got[:, 4] == 0).all()
    for i in range(2):
        for j in range(N):
            if i == 1 and 5 in sets[1][j]:
                assert np.isnan(got[i, j]).all()
            else:
                close(got[i, j], attend(q[i * N + j], K, V, i, base, sets[i][j], 128, 0.1))
    c.free()


def test_sequences_without_a_place(gpu, kernel):
    """A base below 0, a slot outside the cache, an empty mask: zeros, whatever the context holds."""
    H, KVH, hd, N = 8, 2, 64, 3
    rng = np.random.default_rng(6)
    c = ref.Cache(gpu, KV_Q8, 2, 100, KVH, hd, rng)
    c.ks[:] = np.nan
    c.push()
    q = rng.standard_normal((5 * N, H, hd)).astype(np.float32)
    seen = np.tile(masks(ancestors([-1, 0, 1])), (5, 1))
    seen[4] = 0
    got = run_tree(gpu, c, q, [0, 2, -1, 1, 1], [-1, 50, 50, -2 ** 31, 50], seen, N, 0.1)
    assert (got == 0).all()
    c.free()


# ── plans and paths ──

TREES = [[-1], [-1, 0], [-1, 0, 0, 1, 1, 2], [-1] + list(range(63)), [-1] + [0] * 63, [-1, 0, 1, -2, 0], [-2, 0, 0], [-1, 1, 0], [-1, -1, 0, 1],
         [-1, 0, 5, 1], [-1, 0, -5], [-1, 2 ** 31 - 1, 0], [0, 0]]


def test_plan(gpu):
    rng = np.random.default_rng(1)
    N = 64
    trees = [t + [-2] * (N - len(t)) for t in TREES] + [random_tree(rng, int(rng.integers(1, 65)), N) for _ in range(20)]
    n = len(trees)
    base = rng.integers(0, 5000, n).astype(np.int32)
    base[2] = -1
    slot = rng.permutation(n).astype(np.int32)
    for ds in (gpu.upload(slot), None):
        out = [gpu.alloc(8 * n * N)] + [gpu.alloc(4 * n * N) for _ in range(3)]
        dp, db = i32(gpu, trees), gpu.upload(base)
        gpu.tree_plan(ds, db, dp, n, N, *out)
        seen = gpu.download(out[0], np.uint64, (n, N))
        at, row, turn = (gpu.download(o, np.int32, (n, N)) for o in out[1:])
        for i, t in enumerate(trees):
            sets = ancestors(t) if base[i] >= 0 else [set()] * N
            assert np.array_equal(seen[i], masks(sets)), t
            assert (at[i] == (i if ds is None else slot[i])).all()
            assert list(row[i]) == [base[i] + j if s else -1 for j, s in enumerate(sets)]
            assert list(turn[i]) == [base[i] + len(s) - 1 if s else -1 for s in sets]
        gpu.h2d(out[2], np.full((n, N), 9, np.int32))
        gpu.tree_plan(ds, db, dp, n, N, None, None, None, out[3])      # any of the four
        assert (gpu.download(out[2], np.int32, (n, N)) == 9).all()
        for b in out + [dp, db]:
            b.free()


@pytest.mark.parametrize("N", [1, 2, 5, 33, 64])
def test_plan_of_small_trees(gpu, N):
    """Trees next to each other in the arrays do not meet."""
    rng = np.random.default_rng(N)
    trees = [random_tree(rng, N, N) for _ in range(9)]
    seen, dp, db = gpu.upload(np.full(9 * N + 1, 5, np.uint64)), i32(gpu, trees), i32(gpu, [0] * 9)
    gpu.tree_plan(None, db, dp, 9, N, seen)
    got = gpu.download(seen, np.uint64, (9 * N + 1,))
    assert got[-1] == 5 and np.array_equal(got[:-1], np.concatenate([masks(ancestors(t)) for t in trees]))
    for b in (seen, dp, db):
        b.free()


def walk(parent, token, pick):
    there = sum(bool(s) for s in ancestors(parent))
    if not there:
        return [], -1
    path = [0]
    while True:
        child = [j for j in range(1, there) if parent[j] == path[-1] and token[j] == pick[path[-1]]]
        if not child:
            return path, pick[path[-1]]
        path.append(child[0])


@pytest.mark.parametrize("N", [1, 6, 64])
def test_accept(gpu, N):
    """Few tokens, so that several children fit and the first is taken; whole chains; trees that are not there."""
    rng = np.random.default_rng(N)
    trees = [random_tree(rng, int(rng.integers(1, N + 1)), N) for _ in range(40)]
    trees += [([-1] + list(range(N - 1))), [-2] * N, [-1] + [0] * (N - 1), [-1] + [N] * (N - 1)]
    n = len(trees)
    token, pick = rng.integers(0, 3, (n, N)), rng.integers(0, 3, (n, N))
    token[40], pick[40] = 1, 1                     # everything fits: the whole chain
    base = rng.integers(0, 100, n)
    base[0] = -4
    bufs = [i32(gpu, v) for v in (trees, token, pick, base)]
    path, n_path, nxt, new = gpu.alloc(4 * n * N), *(gpu.alloc(4 * n) for _ in range(3))
    for with_base in (True, False):
        gpu.tree_accept(*bufs[:3], bufs[3] if with_base else None, n, N, path, n_path, nxt, new if with_base else None)
        got = gpu.download(path, np.int32, (n, N))
        counts, nexts, bases = (gpu.download(b, np.int32, (n,)) for b in (n_path, nxt, new))
        for i in range(n):
            want, follow = walk(trees[i], token[i], pick[i]) if not (with_base and base[i] < 0) else ([], -1)
            assert list(got[i]) == want + [-1] * (N - len(want))
            assert counts[i] == len(want) and nexts[i] == follow
            if with_base:
                assert bases[i] == base[i] + len(want)
    for b in bufs + [path, n_path, nxt, new]:
        b.free()


# ── rows that move ──

def layers(gpu, kind, n_kv, slots, max_seq, kvh, hd, rng):
    cs = [ref.Cache(gpu, kind, slots, max_seq, kvh, hd, rng) for _ in range(n_kv)]
    return cs, gpu.kv_layers([c.kv for c in cs])


def check_rows(cs, want):
    for c, w in zip(cs, want):
        for a, b in zip(c.pull(), w):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("KVH,hd,n_kv", [(2, 128, 3), (3, 64, 1), (1, 64, 35)])
def test_keep(gpu, kind, KVH, hd, n_kv):
    """Paths whose rows are each other's places (0 2 4, and backwards), all 64, none, ones that end at the cache's end or
    outside it, nodes that are none; all layers, other rows as they were."""
    rng = np.random.default_rng(KVH)
    N, slots, max_seq = 64, 9, 100
    paths = [[0, 2, 4, 8, 16, 32, 63], list(range(64)), list(range(63, -1, -1)), [], [3], [0, 1, 2], [0, 50, 5, 5, -1, 64, 7, 2 ** 31 - 1],
             [1, 0], [9, 8, 7, 6]]
    base = [10, 36, 30, 0, 99, 98, 5, -1, 2 ** 31 - 3]
    counts = [len(p) for p in paths]
    counts[1] = 1000
    slot = [4, 0, 2, 1, 3, 5, 8, 7, 6]
    cs, kv = layers(gpu, kind, n_kv, slots, max_seq, KVH, hd, rng)
    want = []
    for c in cs:
        arrays = [c.k.copy(), c.v.copy(), c.ks.copy(), c.vs.copy()]
        for new, old in zip(arrays, (c.k, c.v, c.ks, c.vs)):
            for i, p in enumerate(paths):
                for d, f in enumerate(p):
                    if base[i] >= 0 and 0 <= f < N and base[i] + max(f, d) < max_seq:
                        new[slot[i], :, base[i] + d] = old[slot[i], :, base[i] + f]
        want.append(arrays)
    bufs = [i32(gpu, v) for v in (slot, base, [p + [-1] * (N - len(p)) for p in paths], counts)]
    gpu.kv_keep(kv, *bufs, 9, N)
    check_rows(cs, want)
    gpu.h2d(bufs[0], np.array([9, -1, 2 ** 31 - 1, 9, 9, 9, 9, 9, -2 ** 31], np.int32))     # slots outside the cache
    gpu.kv_keep(kv, *bufs, 9, N)
    check_rows(cs, want)
    gpu.h2d(bufs[3], np.array([0, -1, -2 ** 31] * 3, np.int32))                              # no paths
    gpu.kv_keep(kv, None, *bufs[1:], 9, N)
    check_rows(cs, want)
    for b in bufs:
        b.free()
    for c in cs:
        c.free()


# ── as they are used ──

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("captured", [False, True])
def test_a_draft_is_the_text_it_guesses(gpu, kind, captured):
    """Several steps of a small attention model: a drafted tree with the text's own next tokens somewhere in it is planned,
    appended, attended, accepted and its rows kept; then the cache holds bit by bit the rows of the text, and the nodes on
    the path answer as the text's tokens one at a time."""
    rng = np.random.default_rng(12)
    H, KVH, hd, N, vocab, n, n_text = 8, 2, 64, 21, 50, 3, 40
    D, KV = H * hd, KVH * hd
    ld = D + 2 * KV
    emb = rng.standard_normal((vocab, ld)).astype(np.float32)            # a token's q, k and v
    text = rng.integers(0, vocab, (n, n_text + N + 1))
    text[:, 0] = 1
    tab = gpu.upload(ref.table(128, hd))
    rope = Rope(tab.ptr, 128, hd, 0)
    c, plain = ref.Cache(gpu, kind, n, 128, KVH, hd, fill=0), ref.Cache(gpu, kind, n, 128, KVH, hd, fill=0)
    kv = gpu.kv_layers([c.kv])
    dx, out, dpar, dtok, dpick = gpu.alloc(4 * n * N * ld), gpu.alloc(4 * n * N * D), *(gpu.alloc(4 * n * N) for _ in range(3))
    seen, at, row, turn, path = gpu.alloc(8 * n * N), *(gpu.alloc(4 * n * N) for _ in range(4))
    base, new, n_path, nxt = (gpu.upload(np.zeros(n, np.int32)) for _ in range(4))

    def step():
        gpu.tree_plan(None, base, dpar, n, N, seen, at, row, turn)
        gpu.kv_append_turned(c.kv, at, row, turn, n * N, dx.ptr + 4 * D, dx.ptr + 4 * (D + KV), ld, rope, dx, dx, H, ld, ld)
        gpu.attn_tree(out, D, dx, ld, c.kv, None, base, seen, n, N, H, 0.125)
        gpu.tree_accept(dpar, dtok, dpick, base, n, N, path, n_path, nxt, new)
        gpu.kv_keep(kv, None, base, path, n_path, n, N)

    # the text's tokens one at a time
    want = np.zeros((n, n_text + N, D), np.float32)
    one, o1, p1, l1 = gpu.alloc(4 * n * ld), gpu.alloc(4 * n * D), *(gpu.alloc(4 * n) for _ in range(2))
    for t in range(n_text + N):
        gpu.h2d(one, emb[text[:, t]])
        gpu.h2d(p1, np.full(n, t, np.int32))
        gpu.h2d(l1, np.full(n, t + 1, np.int32))
        gpu.kv_append(plain.kv, None, p1, n, one.ptr + 4 * D, one.ptr + 4 * (D + KV), ld, rope, one, one, H, ld, ld)
        gpu.attn_decode(o1, D, one, ld, plain.kv, None, l1, n, H, 0.125)
        want[:, t] = gpu.download(o1, np.float32, (n, D))

    graph, done, steps = None, np.zeros(n, int), 0
    while done.min() < n_text and steps < 100:
        parent = np.array([random_tree(rng, N - int(rng.integers(0, 4)), N) for _ in range(n)])
        token = rng.integers(0, vocab, (n, N))
        sets = [ancestors(p) for p in parent]
        for s in range(n):
            done[s] = min(done[s], n_text)
            token[s, 0] = text[s, done[s]]
            deepest = max(sets[s], key=len)                              # a chain of right guesses, cut somewhere
            for d, j in enumerate(sorted(deepest)[:1 + int(rng.integers(0, len(deepest)))]):
                token[s, j] = text[s, done[s] + d]
        pick = np.array([[text[s, done[s] + len(sets[s][j])] if sets[s][j] else 0 for j in range(N)] for s in range(n)])
        for b, v in ((base, done), (dpar, parent), (dtok, token), (dpick, pick)):
            gpu.h2d(b, v.astype(np.int32))
        gpu.h2d(dx, emb[token])
        if captured and graph is None and steps:
            gpu.capture_begin()
            step()
            graph = gpu.capture_end()
        if graph is None:
            step()
        else:
            gpu.graph_launch(graph)
        got, paths = gpu.download(out, np.float32, (n, N, D)), gpu.download(path, np.int32, (n, N))
        counts = gpu.download(n_path, np.int32, (n,))
        for s in range(n):
            for d, j in enumerate(paths[s, :counts[s]]):
                close(got[s, j], want[s, done[s] + d].astype(np.float64))
            assert (got[s, [j for j in range(N) if not sets[s][j]]] == 0).all()
        done = gpu.download(new, np.int32, (n,)).astype(int)
        assert list(gpu.download(nxt, np.int32, (n,))) == [text[s, done[s]] for s in range(n)]
        for a, b in zip(c.pull(), plain.pull()):
            for s in range(n):
                assert np.array_equal(a[s, :, :done[s]], b[s, :, :done[s]])
        steps += 1
    assert done.min() >= n_text and steps < 40
    if graph:
        gpu.graph_destroy(graph)
    for b in (tab, dx, out, dpar, dtok, dpick, seen, at, row, turn, path, base, new, n_path, nxt, one, o1, p1, l1):
        b.free()
    c.free()
    plain.free()
