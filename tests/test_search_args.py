"""Refusals of the window, tree and beam calls: made from the arguments alone, so they need no device."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from hako_amd.gpu import SEARCH_SIGNATURES, KV_F16, Kv, Rope, load_library
from test_attn_args import ATTN_BAD, BAD_KV, EINVAL, ENODEV, ETYPE, P, kv, lib, ref, rope  # noqa: F401


def decode_window(lib, c=None, out=P, ldo=512, q=P, ldq=512, slot=P, length=P, n=2, H=4, scale=1.0, window=8, sinks=4):
    return lib.hako_gpu_attn_decode_window(out, ldo, q, ldq, ref(kv() if c is None else c), slot, length, n, H, scale, window, sinks)


def prompt_window(lib, c=None, out=P, ldo=512, q=P, ldq=512, slot=(0, 1), start=(0, 3), length=(5, 0), n=2, H=4, scale=1.0,
                  window=8, sinks=4):
    a = [None if x is None else np.array(x, np.int32) for x in (slot, start, length)]
    return lib.hako_gpu_attn_prompt_window(out, ldo, q, ldq, ref(kv() if c is None else c),
                                           *(None if x is None else x.ctypes.data for x in a), n, H, scale, window, sinks)


def tree(lib, c=None, out=P, ldo=512, q=P, ldq=512, slot=P, base=P, seen=P, n=2, N=5, H=4, scale=1.0, ps=0, pl=0):
    return lib.hako_gpu_attn_tree(out, ldo, q, ldq, ref(kv() if c is None else c), slot, base, seen, n, N, H, scale, ps, pl)


def turned(lib, c=None, slot=P, pos=P, turn=P, n=2, k=P, v=P, ldk=256, r="rope", q=P, qo=P, H=4, ldq=512, ldo=512):
    return lib.hako_gpu_kv_append_turned(ref(kv() if c is None else c), slot, pos, turn, n, k, v, ldk, ref(rope() if r == "rope" else r),
                                         q, qo, H, ldq, ldo)


def select(lib, logits=P, ld=100, vocab=100, score=P, done=P, eos=3, n=2, K=4, pick=8, arrange=0, parent=P, token=P, out=P, ended=P):
    return lib.hako_gpu_beam_select(logits, ld, vocab, score, done, eos, n, K, pick, arrange, parent, token, out, ended)


def caches(c=None, n=2, **second):
    a = [kv() if c is None else c for _ in range(n)]
    if second:
        a[-1] = kv(**second)
    return (Kv * max(n, 1))(*a)


def reorder(lib, c=None, n_kv=2, slot=P, parent=P, n=2, K=4, since=P, length=P, a=None):
    return lib.hako_gpu_kv_reorder(caches(c) if a is None else a, n_kv, slot, parent, n, K, since, length)


def keep(lib, c=None, n_kv=2, slot=P, base=P, path=P, n_path=P, n=2, N=5, a=None):
    return lib.hako_gpu_kv_keep(caches(c) if a is None else a, n_kv, slot, base, path, n_path, n, N)


def plan(lib, slot=P, base=P, parent=P, n=2, N=5, seen=P, at=P, row=P, turn=P):
    return lib.hako_gpu_tree_plan(slot, base, parent, n, N, seen, at, row, turn)


def accept(lib, parent=P, token=P, pick=P, base=P, n=2, N=5, path=P, n_path=P, nxt=P, new=P):
    return lib.hako_gpu_tree_accept(parent, token, pick, base, n, N, path, n_path, nxt, new)


@pytest.mark.parametrize("bad", BAD_KV, ids=str)
@pytest.mark.parametrize("call", [decode_window, prompt_window, tree, turned, reorder, keep])
def test_bad_cache(lib, call, bad):
    assert call(lib, kv(**bad)) == (ETYPE if bad in (dict(type=0), dict(type=3)) else EINVAL)
    assert lib.hako_gpu_last_error()


NO_PREFIX = [b for b in ATTN_BAD if "pl" not in b]
WINDOW_BAD = NO_PREFIX + [dict(window=0), dict(window=-1), dict(sinks=-1)]


@pytest.mark.parametrize("bad", WINDOW_BAD + [dict(length=None), dict(slot=None, n=3), dict(n=65536)], ids=str)
def test_decode_window_refuses(lib, bad):
    assert decode_window(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", WINDOW_BAD + [
    dict(length=None), dict(start=None), dict(slot=(0, 2)), dict(slot=(-1, 0)), dict(start=(-1, 0)), dict(length=(-1, 2)),
    dict(start=(252, 0)), dict(start=(2 ** 31 - 1, 0), length=(2 ** 31 - 1, 0)),
    dict(slot=None, start=(0, 0, 0), length=(1, 1, 1), n=3)], ids=str)
def test_prompt_window_refuses(lib, bad):
    assert prompt_window(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", ATTN_BAD + [dict(base=None), dict(seen=None), dict(seen=P + 4), dict(N=0), dict(N=65), dict(N=-1),
                                            dict(n=2 ** 31 - 1), dict(slot=None, n=3)], ids=str)
def test_tree_refuses(lib, bad):
    assert tree(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [
    dict(turn=None), dict(pos=None), dict(n=-1), dict(slot=None, n=3), dict(k=None), dict(v=P + 8), dict(ldk=252), dict(q=None),
    dict(H=0), dict(ldq=508), dict(r=None), dict(r=None, q=None, qo=None), dict(r=rope(rot_dim=12)), dict(ldo=516)], ids=str)
def test_append_turned_refuses(lib, bad):
    assert turned(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(score=None), dict(parent=None), dict(token=None), dict(out=None), dict(n=-1), dict(K=0), dict(K=17),
    dict(n=65536, K=1), dict(n=8192, K=8), dict(n=2 ** 31 - 1), dict(vocab=0), dict(vocab=-5), dict(ld=99), dict(vocab=2 ** 24 + 1, ld=2 ** 25),
    dict(pick=0), dict(pick=33), dict(arrange=1), dict(arrange=1, pick=3)], ids=str)
def test_select_refuses(lib, bad):
    assert select(lib, **bad) == EINVAL


OTHER = [dict(n_slots=3), dict(max_seq=257), dict(n_kv_heads=1), dict(head_dim=64), dict(type=KV_F16), dict(k=None)]


@pytest.mark.parametrize("bad", [dict(n_kv=0), dict(n_kv=-1), dict(n=-1), dict(n=65536), dict(K=0), dict(K=17), dict(parent=None),
                                 dict(length=None), dict(slot=None, n=1, K=3)] + [dict(a=caches(**o)) for o in OTHER], ids=str)
def test_reorder_refuses(lib, bad):
    assert reorder(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(n_kv=0), dict(n=-1), dict(n=65536), dict(N=0), dict(N=65), dict(base=None), dict(path=None),
                                 dict(n_path=None), dict(slot=None, n=3)] + [dict(a=caches(**o)) for o in OTHER], ids=str)
def test_keep_refuses(lib, bad):
    assert keep(lib, **bad) == EINVAL


def test_null_caches(lib):
    assert lib.hako_gpu_kv_reorder(None, 1, P, P, 2, 4, P, P) == EINVAL
    assert lib.hako_gpu_kv_keep(None, 1, P, P, P, P, 2, 5) == EINVAL


@pytest.mark.parametrize("bad", [dict(base=None), dict(parent=None), dict(n=-1), dict(N=0), dict(N=65), dict(seen=P + 4)], ids=str)
def test_plan_refuses(lib, bad):
    assert plan(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(parent=None), dict(token=None), dict(pick=None), dict(path=None), dict(n_path=None), dict(nxt=None),
                                 dict(base=None), dict(new=None), dict(n=-1), dict(N=0), dict(N=65)], ids=str)
def test_accept_refuses(lib, bad):
    assert accept(lib, **bad) == EINVAL


def test_binding_covers_the_header():
    path = os.path.join(os.path.dirname(__file__), "..", "include", "hako_search.h")
    src = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    assert sorted(re.findall(r"^int (hako_gpu_\w+)\(", src, flags=re.M)) == sorted(SEARCH_SIGNATURES)


@pytest.mark.parametrize("call,args", [
    (decode_window, {}), (decode_window, dict(window=2 ** 31 - 1, sinks=2 ** 31 - 1)), (prompt_window, {}),
    (prompt_window, dict(window=2 ** 31 - 1, sinks=2 ** 31 - 1)), (tree, {}), (tree, dict(N=64)), (turned, {}),
    (turned, dict(q=None, qo=None)), (select, {}), (select, dict(done=None, ended=None)), (select, dict(pick=4, arrange=1)),
    (select, dict(pick=32, K=16, n=4095, ld=2 ** 40)), (reorder, {}), (reorder, dict(since=None)), (keep, {}), (keep, dict(N=64)),
    (plan, {}), (plan, dict(slot=None, seen=None, at=None, row=None, turn=None)), (accept, {}), (accept, dict(base=None, new=None))],
    ids=lambda x: getattr(x, "__name__", str(x)))
def test_without_a_device(lib, call, args):
    """What is accepted goes on to the device, and says so where none was initialised."""
    assert call(lib, **args) == ENODEV


@pytest.mark.parametrize("call,args", [("hako_gpu_decoder_window", (None, 8, 4)), ("hako_gpu_decoder_beam", (None, 2, P, 3, -1, P, P)),
                                       ("hako_gpu_decoder_verify", (None, 0, P, P, 3, P, P))])
def test_decoder_calls_refuse(lib, call, args):
    assert getattr(lib, call)(*args) == EINVAL
