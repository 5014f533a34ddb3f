"""Refusals of the cache and attention calls: made from the arguments alone, so they need no device."""
import ctypes as C
import os
import re

import numpy as np
import pytest

from hako_amd.gpu import ATTN_SIGNATURES, KV_F16, KV_Q8, Kv, Rope, load_library

EINVAL, ENODEV, ETYPE = -1, -2, -6
P = 0x10000   # an aligned address that no accepted call here reaches a device with


@pytest.fixture(scope="module")
def lib():
    lb = load_library()
    if lb.hako_gpu_stream():
        pytest.skip("a device is initialised: made-up addresses must not reach it")
    return lb


def kv(**kw):
    f = dict(type=KV_Q8, n_slots=2, max_seq=256, n_kv_heads=2, head_dim=128, k=P, v=P, k_scale=P, v_scale=P)
    f.update(kw)
    return Kv(*f.values())


def rope(**kw):
    f = dict(table=P, n_pos=256, rot_dim=128, interleaved=0)
    f.update(kw)
    return Rope(*f.values())


def ref(s):
    return None if s is None else C.byref(s)


def append(lib, c=None, slot=P, pos=P, n=2, k=P, v=P, ldk=256, r="rope", q=P, qo=P, H=4, ldq=512, ldo=512):
    c = kv() if c is None else c
    r = rope() if r == "rope" else r
    return lib.hako_gpu_kv_append(ref(c), slot, pos, n, k, v, ldk, ref(r), q, qo, H, ldq, ldo)


def read(lib, c=None, slot=P, pos=P, n=2, k=P, v=P, ldk=256):
    return lib.hako_gpu_kv_read(ref(kv() if c is None else c), slot, pos, n, k, v, ldk)


def decode(lib, c=None, out=P, ldo=512, q=P, ldq=512, slot=P, length=P, n=2, H=4, scale=1.0, ps=0, pl=0):
    return lib.hako_gpu_attn_decode(out, ldo, q, ldq, ref(kv() if c is None else c), slot, length, n, H, scale, ps, pl)


def prompt(lib, c=None, out=P, ldo=512, q=P, ldq=512, slot=(0, 1), start=(0, 3), length=(5, 0), n=2, H=4, scale=1.0,
           ps=0, pl=0):
    a = [None if x is None else np.array(x, np.int32) for x in (slot, start, length)]
    return lib.hako_gpu_attn_prompt(out, ldo, q, ldq, ref(kv() if c is None else c),
                                    *(None if x is None else x.ctypes.data for x in a), n, H, scale, ps, pl)


BAD_KV = [dict(n_slots=2 ** 31 - 1, n_kv_heads=65535, max_seq=2 ** 20), dict(type=0), dict(type=3), dict(n_slots=0), dict(max_seq=0), dict(n_kv_heads=0), dict(n_kv_heads=65536),
          dict(head_dim=96), dict(head_dim=0), dict(max_seq=1 << 24), dict(type=KV_F16, max_seq=1 << 23), dict(k=None),
          dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 4), dict(k_scale=P + 2),
          dict(v_scale=P + 1)]


@pytest.mark.parametrize("bad", BAD_KV, ids=str)
@pytest.mark.parametrize("call", [append, read, decode, prompt])
def test_bad_cache(lib, call, bad):
    assert call(lib, kv(**bad)) == (ETYPE if bad in (dict(type=0), dict(type=3)) else EINVAL)
    assert lib.hako_gpu_last_error()


@pytest.mark.parametrize("bad", [
    dict(pos=None), dict(n=-1), dict(slot=None, n=3), dict(k=None), dict(v=None), dict(k=P + 4), dict(v=P + 8),
    dict(ldk=255), dict(ldk=252), dict(ldk=258), dict(q=None), dict(qo=None), dict(q=P + 4), dict(qo=P + 12), dict(H=0),
    dict(H=65536), dict(ldq=508), dict(ldo=510), dict(r=None), dict(ldo=516),
    dict(r=rope(table=None)), dict(r=rope(table=P + 8)), dict(r=rope(n_pos=0)), dict(r=rope(rot_dim=0)),
    dict(r=rope(rot_dim=12)), dict(r=rope(rot_dim=136)), dict(r=rope(interleaved=2))], ids=str)
def test_append_refuses(lib, bad):
    assert append(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(pos=None), dict(n=-1), dict(slot=None, n=3), dict(k=None, v=None), dict(k=P + 4),
                                 dict(v=P + 8), dict(ldk=252), dict(ldk=257)], ids=str)
def test_read_refuses(lib, bad):
    assert read(lib, **bad) == EINVAL


ATTN_BAD = [dict(out=None), dict(q=None), dict(out=P + 4), dict(q=P + 8), dict(ldo=508), dict(ldq=511), dict(ldq=516),
            dict(n=-1), dict(H=0), dict(H=3), dict(H=34), dict(ps=-1, pl=1), dict(ps=2, pl=1), dict(pl=-1), dict(pl=257)]


@pytest.mark.parametrize("bad", ATTN_BAD + [dict(length=None), dict(slot=None, n=3)], ids=str)
def test_decode_refuses(lib, bad):
    assert decode(lib, **bad) == EINVAL


@pytest.mark.parametrize("bad", ATTN_BAD + [
    dict(length=None), dict(start=None), dict(slot=(0, 2)), dict(slot=(-1, 0)), dict(start=(-1, 0)), dict(length=(-1, 2)),
    dict(start=(252, 0)), dict(length=(257, 0)), dict(start=(257, 0), length=(0, 0)),
    dict(start=(2 ** 31 - 1, 0), length=(2 ** 31 - 1, 0)),
    dict(slot=None, start=(0, 0, 0), length=(1, 1, 1), n=3)], ids=str)
def test_prompt_refuses(lib, bad):
    assert prompt(lib, **bad) == EINVAL


def test_binding_covers_the_header():
    path = os.path.join(os.path.dirname(__file__), "..", "include", "hako_attn.h")
    src = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    assert sorted(re.findall(r"^int (hako_gpu_\w+)\(", src, flags=re.M)) == sorted(ATTN_SIGNATURES)


@pytest.mark.parametrize("call,args", [
    ("hako_gpu_decoder_create_kv", (None, 1, 64, 3, None)), ("hako_gpu_decoder_create_kv", (None, 1, 64, -1, None)),
    ("hako_gpu_decoder_cache", (None, 0, None)), ("hako_gpu_decoder_share_prefix", (None, 0, 0))])
def test_decoder_calls_refuse(lib, call, args):
    args = [C.byref(C.c_void_p()) if a is None and i == 4 else a for i, a in enumerate(args)]
    assert getattr(lib, call)(*args) in (EINVAL, ETYPE)


def test_kv_bytes(lib):
    codes, scales = C.c_size_t(), C.c_size_t()
    c = kv(k=None, v=None, k_scale=None, v_scale=None, n_slots=70, max_seq=65536, n_kv_heads=8)
    assert lib.hako_gpu_kv_bytes(C.byref(c), C.byref(codes), C.byref(scales)) == 0
    assert codes.value == 70 * 65536 * 8 * 128 and scales.value == 70 * 65536 * 8 * 4
    c.type = KV_F16
    assert lib.hako_gpu_kv_bytes(C.byref(c), C.byref(codes), C.byref(scales)) == 0
    assert codes.value == 2 * 70 * 65536 * 8 * 128
    for name, value in (("type", 7), ("head_dim", 32), ("n_slots", 0)):
        d = kv(**{name: value})
        assert lib.hako_gpu_kv_bytes(C.byref(d), C.byref(codes), C.byref(scales)) < 0
    assert lib.hako_gpu_kv_bytes(None, C.byref(codes), C.byref(scales)) == EINVAL


@pytest.mark.parametrize("call", [append, read, decode, prompt])
def test_without_a_device(lib, call):
    """What is accepted goes on to the device, and says so where none was initialised."""
    assert call(lib) == ENODEV


# Shapes whose number of rows is a multiple of 2^64, or wraps to a small one: no cache of theirs can be addressed.
WRAPS = [dict(type=KV_Q8, head_dim=64, max_seq=1 << 24, n_kv_heads=1 << 15, n_slots=1 << 25),
         dict(type=KV_F16, head_dim=64, max_seq=1 << 23, n_kv_heads=1 << 15, n_slots=1 << 26),
         dict(type=KV_Q8, head_dim=64, max_seq=(1 << 24) + 1, n_kv_heads=1 << 15, n_slots=1 << 25)]


@pytest.mark.parametrize("shape", WRAPS, ids=str)
def test_shapes_that_wrap_are_refused(lib, shape):
    assert (shape["max_seq"] * shape["n_kv_heads"] * shape["n_slots"]) % 2 ** 64 < 2 ** 48
    codes, scales = C.c_size_t(7), C.c_size_t(7)
    c = kv(k=None, v=None, k_scale=None, v_scale=None, **shape)
    assert lib.hako_gpu_kv_bytes(C.byref(c), C.byref(codes), C.byref(scales)) == EINVAL
    assert (codes.value, scales.value) == (7, 7)
    c = kv(**shape)
    assert append(lib, c, ldk=shape["n_kv_heads"] * 64) == EINVAL and read(lib, c, ldk=shape["n_kv_heads"] * 64) == EINVAL


def test_the_largest_shapes_are_taken(lib):
    """2^48 - 2^24 rows, and one slot more."""
    codes, scales = C.c_size_t(), C.c_size_t()
    c = kv(k=None, v=None, k_scale=None, v_scale=None, head_dim=64, max_seq=1 << 24, n_kv_heads=1, n_slots=(1 << 24) - 1)
    assert lib.hako_gpu_kv_bytes(C.byref(c), C.byref(codes), C.byref(scales)) == 0
    assert codes.value == ((1 << 48) - (1 << 24)) * 64 and scales.value == ((1 << 48) - (1 << 24)) * 4
    c.n_slots += 1
    assert lib.hako_gpu_kv_bytes(C.byref(c), C.byref(codes), C.byref(scales)) == EINVAL
