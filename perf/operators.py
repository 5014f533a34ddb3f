"""The cache and attention operators of include/hako_attn.h, case by case.

A case is a plain dict. Its "kind" says which calls a user's program makes:

* "append": hako_gpu_kv_append of n new tokens (their queries and keys
  rotated, their keys and values written to the cache in 8 or 16 bits) and
  hako_gpu_kv_read of the rows just written.
* "read": hako_gpu_kv_read of cached rows, as a program does that moves a
  sequence out of the cache.
* "decode": hako_gpu_attn_decode, one query token per sequence over its cached
  positions; with "prefix" > 0 the positions below it are one slot's, which
  all sequences share.
* "prompt": hako_gpu_attn_prompt, whole prompts of several lengths packed one
  after the other, each causal over its own positions and over those that its
  slot held before ("starts").

A cache row (one position of one key/value head) is head_dim codes and a scale:
int8 codes ("q8"; scale max|x| / 127) or halves ("f16"; scale a power of two).
The caches are [slot][kv head][position][head_dim], the scales the same without
the last axis. Everything else is float32.
"""
import math

import numpy as np
import torch

own = False

FLT_MIN = 1.17549435e-38


def listed():
    b3 = {"heads": 16, "kv_heads": 2, "head_dim": 128}   # the attention of a 3B model of the benchmark
    b7 = {"heads": 28, "kv_heads": 4, "head_dim": 128}   # and of a 7B model
    return [
        # one token of one conversation: the smallest call, all latency
        dict(b3, name="append_1", kind="append", type="q8", lens="1", starts="1024", rot=128, interleaved=False, stretch=1.0),
        # a full prompt pass
        dict(b7, name="append_512", kind="append", type="q8", lens="512", starts="0", rot=128, interleaved=False, stretch=1.0),
        # a serving batch of ragged prompts; positions stretched fourfold for a long context, neighbouring dims as pairs,
        # a part of the head rotated
        dict(b7, name="append_packed_f16", kind="append", type="f16", lens="1200,77,4096,1,1523,640,333,322",
             starts="0,2000,0,511,64,0,7,30000", rot=96, interleaved=True, stretch=4.0),
        # a short conversation of a small-headed model leaves the cache
        {"name": "read_100", "kind": "read", "heads": 14, "kv_heads": 2, "head_dim": 64, "type": "f16", "lens": "100"},
        # four long conversations leave it
        dict(b7, name="read_32k", kind="read", type="q8", lens="8192,16384,1000,7111"),
        # one conversation in its middle: latency
        dict(b3, name="decode_1", kind="decode", type="q8", lens="1025", prefix=0),
        # serving: 16 sequences of 4096 positions
        dict(b7, name="decode_16", kind="decode", type="q8", lens=",".join(["4096"] * 16), prefix=0),
        # 48 sequences with a long system prompt in common and turns of their own
        dict(b7, name="decode_prefix_48", kind="decode", type="q8",
             lens=",".join(str(6000 + 1 + (i * 167) % 700) for i in range(48)), prefix=6000),
        # two book-length contexts in 16 bits
        dict(b3, name="decode_long_f16", kind="decode", type="f16", lens="32768,20011", prefix=0),
        # a chat turn
        dict(b3, name="prompt_77", kind="prompt", type="q8", lens="77", starts="0", prefix=0),
        # ragged prompts of a serving batch, two of them further turns
        dict(b7, name="prompt_packed", kind="prompt", type="f16", lens="700,77,1500,1,333,1024,61,400",
             starts="0,2000,0,511,64,0,7,0", prefix=0),
        # one long document
        dict(b7, name="prompt_8192", kind="prompt", type="q8", lens="8192", starts="0", prefix=0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(v):
    return ",".join(map(str, v))


def draw(rng):
    """One more case: any kind, head layout and type; ragged lengths up to what the largest listed cases take."""
    kind = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt"])
    head_dim = rng.choice([64, 128, 128])
    group, kv_heads = rng.choice([1, 2, 4, 6, 7, 8, 16]), rng.choice([1, 2, 4, 8])
    while group * kv_heads > 32:
        kv_heads //= 2
    c = {"kind": kind, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "type": rng.choice(["q8", "q8", "f16"])}
    n_seq = _log_int(rng, 1, 12)
    if kind == "append":
        lens = [_log_int(rng, 1, 8000 // n_seq + 1) for _ in range(n_seq)]
        c.update(lens=_text(lens), starts=_text(rng.choice([0, _log_int(rng, 1, 20000)]) for _ in lens),
                 rot=rng.choice([head_dim, head_dim, head_dim // 2, head_dim - 16]), interleaved=rng.random() < 0.4,
                 stretch=rng.choice([1.0, 1.0, 2.5, 8.0]))
    elif kind == "read":
        c["lens"] = _text(_log_int(rng, 1, 32000 // n_seq + 1) for _ in range(n_seq))
    elif kind == "decode":
        n_seq = _log_int(rng, 1, 40)
        most = max(2, min(32768, 16 * 4096 // (n_seq * kv_heads) * 4))
        lens = [_log_int(rng, 1, most) for _ in range(n_seq)]
        prefix = rng.choice([0, _log_int(rng, 1, 6000)]) if n_seq > 1 else 0
        if prefix:
            lens = [prefix + _log_int(rng, 1, 700) for _ in lens]
        c.update(lens=_text(lens), prefix=prefix)
    else:
        lens = [_log_int(rng, 1, 6000 // n_seq + 1) for _ in range(n_seq)]
        starts = [rng.choice([0, _log_int(rng, 1, 3000)]) for _ in lens]
        prefix = rng.choice([0, 0, _log_int(rng, 1, 2000)]) if n_seq > 1 else 0
        c.update(lens=_text(lens), starts=_text(s + prefix for s in starts), prefix=prefix)
    return c


# ── inputs ──

def _ints(text):
    return [int(x) for x in text.split(",")]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _max_seq(case):
    ends = [a + b for a, b in zip(_ints(case["lens"]), _ints(case.get("starts", _text([0] * len(_ints(case["lens"]))))))]
    return (max(ends) + 63) // 64 * 64


def _codes(x, kind):
    """Cache rows of x [..., head_dim]: codes and scales."""
    a = x.abs()
    amax = torch.where(a < FLT_MIN, torch.zeros_like(a), a).amax(-1)
    if kind == "q8":
        scale = amax * np.float32(1 / 127)
        scale = torch.where(scale < FLT_MIN, torch.zeros_like(scale), scale)
        inv = torch.where(scale > 0, torch.div(torch.full_like(amax, 127.0), amax), torch.zeros_like(amax))
        return torch.round(torch.where(a < FLT_MIN, torch.zeros_like(x), x) * inv.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), scale
    exp = torch.where(amax > 0, torch.frexp(amax).exponent - 1, torch.zeros_like(amax, dtype=torch.int32))
    return torch.ldexp(x, -exp.unsqueeze(-1)).to(torch.float16), torch.ldexp(torch.ones_like(amax), exp)


def _cache(case, g, slots, max_seq):
    """Filled caches: keys with a few large channels, as trained models have, and values, both N(0, 1) elsewhere."""
    shape = (slots, case["kv_heads"], max_seq, case["head_dim"])
    k = _randn(g, *shape)
    k[..., 5::32] *= 3.0
    ck, ks = _codes(k, case["type"])
    del k
    cv, vs = _codes(_randn(g, *shape), case["type"])
    return {"k": ck, "v": cv, "ks": ks, "vs": vs}


def _table(case, positions):
    """cos and sin of every position below `positions`: [positions][rot / 2][2]."""
    f = 1e6 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"]) / case["stretch"]
    a = torch.arange(positions, device="cuda", dtype=torch.float64).unsqueeze(1) * f
    return torch.stack([a.cos(), a.sin()], 2).float().contiguous()


def prepare(case, seed):
    if own:
        _lib()
    g, lens = _gen(seed), _ints(case["lens"])
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    n_seq, max_seq = len(lens), _max_seq(case)
    s = {"case": case, "lens": lens, "max_seq": max_seq}
    if case["kind"] in ("append", "read"):
        starts = _ints(case["starts"]) if "starts" in case else [0] * n_seq
        n = sum(lens)
        s["slot"] = _i32([i for i, m in enumerate(lens) for _ in range(m)])
        s["pos"] = _i32([p for a, m in zip(starts, lens) for p in range(a, a + m)])
        s["k_out"], s["v_out"] = (torch.zeros(n, KVH * hd, device="cuda") for _ in range(2))
        if case["kind"] == "read":
            s["cache"] = _cache(case, g, n_seq, max_seq)
            return s
        code = torch.int8 if case["type"] == "q8" else torch.float16
        shape = (n_seq, KVH, max_seq)
        s["cache"] = {c: torch.zeros(*shape, hd, dtype=code, device="cuda") for c in ("k", "v")}
        s["cache"].update({c: torch.zeros(*shape, device="cuda") for c in ("ks", "vs")})
        s["qkv"] = _randn(g, n, (H + 2 * KVH) * hd)   # one row a token: its queries, keys and values
        s["q_out"] = torch.zeros(n, H * hd, device="cuda")
        s["table"] = _table(case, max_seq)
        return s
    s["slots"] = list(range(n_seq))
    slots = n_seq
    if case["prefix"]:
        slots, s["prefix_slot"] = n_seq + 1, n_seq
    s["cache"] = _cache(case, g, slots, max_seq)
    n = n_seq if case["kind"] == "decode" else sum(lens)
    s["q"], s["out"] = _randn(g, n, H * hd), torch.zeros(n, H * hd, device="cuda")
    if case["kind"] == "decode":
        s["slot_d"], s["len_d"] = _i32(s["slots"]), _i32(lens)
    else:
        s["starts"] = _ints(case["starts"])
        s["host"] = [np.array(v, dtype=np.int32) for v in (s["slots"], s["starts"], lens)]
    return s


# ── the framework's calls ──

_gpu = _stream = None


def _lib():
    """The library; torch's work goes to its stream from here on, as in a program that uses both."""
    global _gpu, _stream
    if _gpu is None:
        from hako_amd.gpu import Gpu
        gpu = Gpu(0)
        _stream = torch.cuda.ExternalStream(gpu.lib.hako_gpu_stream())
        torch.cuda.current_stream().synchronize()
        torch.cuda.set_stream(_stream)
        _gpu = gpu
    return _gpu


def _view(s):
    """The call's description of the caches."""
    from hako_amd.gpu import KV_F16, KV_Q8, Kv
    case, c = s["case"], s["cache"]
    return Kv(KV_Q8 if case["type"] == "q8" else KV_F16, c["k"].shape[0], s["max_seq"], case["kv_heads"], case["head_dim"],
              c["k"].data_ptr(), c["v"].data_ptr(), c["ks"].data_ptr(), c["vs"].data_ptr())


def _own_run(s):
    """The calls, on the library's stream: in order with torch's work there, and made to be so for a caller on another."""
    _lib()
    if torch._C._cuda_getCurrentRawStream(0) == _stream.cuda_stream:   # (2.5 us less than torch.cuda.current_stream())
        return _own_calls(s)
    caller = torch.cuda.current_stream()
    _stream.wait_stream(caller)
    out = _own_calls(s)
    caller.wait_stream(_stream)
    return out


def _own_calls(s):
    gpu, case = _gpu, s["case"]
    H, KV, hd, kv = case["heads"], case["kv_heads"] * case["head_dim"], case["head_dim"], _view(s)
    D, scale = H * hd, 1.0 / math.sqrt(hd)
    if case["kind"] in ("append", "read"):
        n, slot, pos = len(s["slot"]), s["slot"].data_ptr(), s["pos"].data_ptr()
        if case["kind"] == "append":
            from hako_amd.gpu import Rope
            x, ld = s["qkv"].data_ptr(), D + 2 * KV
            rope = Rope(s["table"].data_ptr(), s["max_seq"], case["rot"], case["interleaved"])
            gpu.kv_append(kv, slot, pos, n, x + 4 * D, x + 4 * (D + KV), ld, rope, x, s["q_out"].data_ptr(), H, ld, D)
        gpu.kv_read(kv, slot, pos, n, s["k_out"].data_ptr(), s["v_out"].data_ptr(), KV)
        out = {"k": s["k_out"], "v": s["v_out"]}
        return dict(out, q=s["q_out"]) if case["kind"] == "append" else out
    prefix = (s.get("prefix_slot", 0), case["prefix"])
    if case["kind"] == "decode":
        gpu.attn_decode(s["out"].data_ptr(), D, s["q"].data_ptr(), D, kv, s["slot_d"].data_ptr(), s["len_d"].data_ptr(),
                        len(s["lens"]), H, scale, *prefix)
    else:
        slots, starts, lens = s["host"]
        gpu.attn_prompt(s["out"].data_ptr(), D, s["q"].data_ptr(), D, kv, slots, starts, lens, len(lens), H, scale, *prefix)
    return s["out"]


# ── the same with plain torch ──

def _rotate(x, t, rot, interleaved):
    """x [tokens][heads][head_dim], the first `rot` dims of a head rotated by t [tokens][rot / 2][2]."""
    c, sn = t[:, None, :, 0], t[:, None, :, 1]
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    u, v = a * c - b * sn, a * sn + b * c
    y = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _rows(s, name, slot, pos):
    """Cached rows [tokens][kv heads][head_dim] as values."""
    c = s["cache"]
    return c[name][slot, :, pos].float() * c[name + "s"][slot, :, pos].unsqueeze(-1)


def _plain_append(s):
    case, c = s["case"], s["cache"]
    H, KVH, hd = case["heads"], case["kv_heads"], case["head_dim"]
    slot, pos = s["slot"].long(), s["pos"].long()
    x = s["qkv"].reshape(len(slot), H + 2 * KVH, hd)
    x, v = x[:, :H + KVH], x[:, H + KVH:]
    x = _rotate(x, s["table"][pos], case["rot"], case["interleaved"])
    c["k"][slot, :, pos], c["ks"][slot, :, pos] = _codes(x[:, H:], case["type"])
    c["v"][slot, :, pos], c["vs"][slot, :, pos] = _codes(v, case["type"])
    return x[:, :H].reshape(len(slot), H * hd)


def _softmax(sc, seen):
    """Weights over the last axis where `seen`, 0 elsewhere."""
    sc = sc.masked_fill(~seen, -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_decode(s):
    case, L = s["case"], max(s["lens"])
    KVH, hd, n = case["kv_heads"], case["head_dim"], len(s["lens"])
    p = torch.arange(L, device="cuda").expand(n, L)
    slot = s["slot_d"].long().unsqueeze(1).expand(n, L)
    slot = torch.where(p < case["prefix"], s.get("prefix_slot", 0), slot)
    k, v = (_rows(s, name, slot, p).transpose(1, 2).contiguous() for name in "kv")   # [sequence][kv head][position][dim]
    q = s["q"].reshape(n, KVH, -1, hd)
    w = _softmax(q @ k.transpose(2, 3) / math.sqrt(hd), (p < s["len_d"].unsqueeze(1))[:, None, None, :])
    return (w @ v).reshape(n, -1)


def _plain_prompt_one(s, q, slot, start):
    """One sequence's prompt: q [tokens][heads * head_dim] at positions from start."""
    case, n = s["case"], len(q)
    KVH, hd = case["kv_heads"], case["head_dim"]
    p = torch.arange(start + n, device="cuda")
    at = torch.where(p < case["prefix"], s.get("prefix_slot", 0), slot)
    k, v = (_rows(s, name, at, p).transpose(0, 1).contiguous() for name in "kv")   # [kv head][position][dim]
    q = q.reshape(n, KVH, -1, hd).permute(1, 2, 0, 3).reshape(KVH, -1, hd)         # rows: query heads of a group x tokens
    sc = (q @ k.transpose(1, 2) / math.sqrt(hd)).reshape(KVH, -1, n, start + n)
    w = _softmax(sc, p <= p[start:].unsqueeze(1))
    return (w.reshape(KVH, -1, start + n) @ v).reshape(KVH, -1, n, hd).permute(2, 0, 1, 3).reshape(n, -1)


def run(state):
    s = state
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "decode":
        return _plain_decode(s)
    if kind == "prompt":
        q = torch.split(s["q"], s["lens"])
        return torch.cat([_plain_prompt_one(s, *one) for one in zip(q, s["slots"], s["starts"])])
    out = {"q": _plain_append(s)} if kind == "append" else {}
    slot, pos = s["slot"].long(), s["pos"].long()
    return dict(out, k=_rows(s, "k", slot, pos).flatten(1), v=_rows(s, "v", slot, pos).flatten(1))


# ── what a pass cannot do without ──

def work(case):
    lens, H, KVH, hd = _ints(case["lens"]), case["heads"], case["kv_heads"], case["head_dim"]
    row = 2 * KVH * (hd * (1 if case["type"] == "q8" else 2) + 4)   # a position's keys and values in the cache
    n = sum(lens)
    if case["kind"] == "read":
        return {"bytes": n * (row + 8 * KVH * hd + 8), "flops": 2 * n * KVH * hd}
    if case["kind"] == "append":
        # q, k, v in and the rotated q out; the rows written, read again and handed out; the angles
        return {"bytes": n * (4 * (2 * H + 2 * KVH) * hd + 2 * row + 8 * KVH * hd + 4 * case["rot"] + 16),
                "flops": n * (3 * (H + KVH) * case["rot"] + 6 * KVH * hd)}
    prefix = case["prefix"]
    if case["kind"] == "decode":
        held = min(prefix, max(lens)) + sum(max(0, m - prefix) for m in lens)
        return {"bytes": held * row + 8 * len(lens) * H * hd, "flops": 4 * H * hd * sum(lens)}
    starts = _ints(case["starts"])
    held = min(prefix, max(a + m for a, m in zip(starts, lens))) + sum(max(0, a + m - prefix) for a, m in zip(starts, lens))
    seen = sum(m * a + m * (m + 1) // 2 for a, m in zip(starts, lens))
    return {"bytes": held * row + 8 * n * H * hd, "flops": 4 * H * hd * seen}


# ── the same in 64 bits, from the definition ──

def _f32(v):
    """Rounded to 32 bits, in 64."""
    return v.float().double()


def _held(x, kind):
    """What a cache row of x (float64 values of 32 bits) stands for. The 8-bit rule's roundings to 32 bits (of 127 / max,
    of the product that is rounded to a code, of the scale) are part of its definition."""
    top = x.abs().amax(-1, keepdim=True)
    if kind == "q8":
        return torch.round(_f32(x * _f32(127.0 / top))) * _f32(top * float(np.float32(1 / 127)))
    step = torch.exp2(torch.floor(torch.log2(top)))
    return (x / step).half().double() * step


def _exact_append(s):
    case = s["case"]
    H, KVH, hd, rot = case["heads"], case["kv_heads"], case["head_dim"], case["rot"]
    x = s["qkv"].double().reshape(-1, H + 2 * KVH, hd)
    t = s["table"].double()[s["pos"].long()].unsqueeze(1)
    i = torch.arange(rot // 2, device="cuda")
    lo, hi = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
    a, b, c, sn = x[..., lo], x[..., hi], t[..., 0], t[..., 1]
    q, k = x[:, :H].clone(), x[:, H:H + KVH].clone()
    q[..., lo], q[..., hi] = (a * c - b * sn)[:, :H], (a * sn + b * c)[:, :H]
    # a key that is written is the rotated one in 32 bits, every product and sum rounded
    a, b = a[:, H:H + KVH], b[:, H:H + KVH]
    k[..., lo], k[..., hi] = _f32(_f32(a * c) - _f32(b * sn)), _f32(_f32(a * sn) + _f32(b * c))
    return {"q": q.flatten(1), "k": _held(k, case["type"]).flatten(1), "v": _held(x[:, H + KVH:], case["type"]).flatten(1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    c, hd = s["cache"], case["head_dim"]
    K, V = (c[n].double() * c[n + "s"].double().unsqueeze(-1) for n in "kv")
    if case["kind"] == "read":
        slot, pos = s["slot"].long(), s["pos"].long()
        return {"k": K[slot, :, pos].flatten(1), "v": V[slot, :, pos].flatten(1)}
    G, P, out, row = case["heads"] // case["kv_heads"], case["prefix"], [], 0
    for i, m in enumerate(s["lens"]):
        n, end = (1, m) if case["kind"] == "decode" else (m, s["starts"][i] + m)
        q = s["q"][row:row + n].double().reshape(n, case["heads"], hd)
        row += n
        heads = []
        for h in range(case["heads"]):
            k, v = (torch.cat([x[s.get("prefix_slot", 0), h // G, :min(P, end)], x[i, h // G, min(P, end):end]]) for x in (K, V))
            parts = []
            for a in range(0, n, 2048):
                b = min(n, a + 2048)
                sc = q[a:b, h] @ k.t() / math.sqrt(hd)
                later = torch.arange(end, device="cuda")[None, :] > torch.arange(end - n + a, end - n + b, device="cuda")[:, None]
                parts.append(torch.softmax(sc.masked_fill(later, -math.inf), 1) @ v)
            heads.append(torch.cat(parts))
        out.append(torch.stack(heads, 1).reshape(n, -1))
    return torch.cat(out)
