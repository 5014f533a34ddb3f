"""Windows, drafted trees and beams over the quantised cache (include/hako_attn.h, include/hako_search.h), case by case.

A case is a plain dict. Its "kind" says which calls a user's program makes:

* "window": hako_gpu_attn_decode_window, one query token per sequence over the
  last "window" of its cached positions and its first "sinks".
* "window_prompt": hako_gpu_attn_prompt_window, packed prompts whose every
  token sees the "window" positions that end with its own, and the sinks.
* "tree": hako_gpu_attn_tree, the drafted tokens of every sequence over its
  cached positions and over those of the draft that lead to them.
* "select": hako_gpu_beam_select, the best continuations of all beams, best
  first, twice as many as there are beams (so that ended ones can be set aside).
* "step": hako_gpu_beam_select as many as there are beams, each survivor's best
  in its own place, and hako_gpu_kv_reorder, which brings the caches of all
  layers after it.
* "accept": hako_gpu_tree_plan, hako_gpu_tree_accept and hako_gpu_kv_keep, what
  a step with a drafted tree does around its model: the positions and masks of
  the tree, the path that the model's own picks follow, and that path's rows
  moved together in the caches of all layers.

A cache row (one position of one key/value head) is head_dim codes and a scale:
int8 codes ("q8"; scale max|x| / 127) or halves ("f16"; scale a power of two).
The caches are [slot][kv head][position][head_dim], the scales the same without
the last axis. Queries, outputs, logits and scores are float32.
"""
import math
import random

import numpy as np
import torch

own = False

FLT_MIN = 1.17549435e-38


def listed():
    b3 = {"heads": 16, "kv_heads": 2, "head_dim": 128}   # the attention of a 3B model of the benchmark
    b7 = {"heads": 28, "kv_heads": 4, "head_dim": 128}   # and of a 7B model
    return [
        # one long conversation under a short window: the smallest call, all latency
        dict(b3, name="window_1", kind="window", type="q8", lens="9001", window=1024, sinks=4),
        # serving: 64 sequences of every length, some shorter than the window
        dict(b7, name="window_64", kind="window", type="q8", lens=",".join(str(300 + (i * 1777) % 12000) for i in range(64)),
             window=4096, sinks=4),
        # ragged prompts of a serving batch, some of them further turns, more first tokens kept
        dict(b7, name="window_packed_f16", kind="window_prompt", type="f16", lens="700,77,1500,1,333,1024,61,400",
             starts="0,2000,0,511,64,0,7,5000", window=512, sinks=20),
        # one long document
        dict(b7, name="window_16384", kind="window_prompt", type="q8", lens="16384", starts="0", window=4096, sinks=4),
        # one conversation with a small tree of guesses: latency
        dict(b3, name="tree_1", kind="tree", type="q8", lens="1025", nodes="26", tree=26, prefix=0),
        # serving: large trees over long contexts
        dict(b7, name="tree_16", kind="tree", type="q8", lens=",".join(["4096"] * 16), nodes=",".join(["64"] * 16), tree=64, prefix=0),
        # many sequences with a system prompt in common and small trees, not all of one size
        dict(b7, name="tree_prefix_f16", kind="tree", type="f16", lens=",".join(str(3001 + (i * 167) % 500) for i in range(32)),
             nodes=",".join(str(1 + (i * 5) % 16) for i in range(32)), tree=16, prefix=3001),
        # 32 requests of 8 beams over the benchmark's vocabulary
        {"name": "select_32x8", "kind": "select", "requests": 32, "beams": 8, "vocab": 152064, "ended": 0.1},
        # one request of 4 beams with the caches of a small model's layers: latency
        dict(b3, name="step_1x4", kind="step", type="f16", requests=1, beams=4, vocab=152064, layers=4, since="300", lens="345"),
        # four requests of 8 beams, the answers some hundred tokens long
        dict(b7, name="step_4x8", kind="step", type="f16", requests=4, beams=8, vocab=152064, layers=12, since="512,40,0,1000",
             lens="900,541,777,1300"),
        # one conversation's small tree: latency
        dict(b3, name="accept_1", kind="accept", type="f16", layers=12, lens="1025", tree=26, kept="4"),
        # a serving batch's large trees, all layers of a 7B model
        dict(b7, name="accept_32", kind="accept", type="f16", layers=28, lens=",".join(str(200 + (i * 331) % 700) for i in range(32)),
             tree=64, kept=",".join(str(1 + (i * 3) % 9) for i in range(32))),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(v):
    return ",".join(map(str, v))


def draw(rng):
    """One more case: any kind, head layout and type; sizes up to what the largest listed cases take."""
    kind = rng.choice(["window", "window", "window_prompt", "window_prompt", "tree", "tree", "select", "step", "accept"])
    head_dim = rng.choice([64, 128, 128])
    group, kv_heads = rng.choice([1, 2, 4, 6, 7, 8, 16]), rng.choice([1, 2, 4, 8])
    while group * kv_heads > 32:
        kv_heads //= 2
    c = {"kind": kind, "heads": group * kv_heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "type": rng.choice(["q8", "q8", "f16"])}
    if kind == "window":
        n = _log_int(rng, 1, 64)
        c.update(window=_log_int(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 37, 64]))
        c["lens"] = _text(_log_int(rng, 1, 12000) for _ in range(n))
    elif kind == "window_prompt":
        n = _log_int(rng, 1, 12)
        c.update(window=_log_int(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 37, 64]))
        c["lens"] = _text(_log_int(rng, 1, 12000 // n + 1) for _ in range(n))
        c["starts"] = _text(rng.choice([0, _log_int(rng, 1, 6000)]) for _ in range(n))
    elif kind == "tree":
        n, tree = _log_int(rng, 1, 32), rng.randint(1, 64)
        prefix = rng.choice([0, 0, _log_int(rng, 1, 3000)]) if n > 1 else 0
        most = max(2, 16 * 4096 * 64 // (n * tree * 2))
        c.update(tree=tree, prefix=prefix, lens=_text(prefix + _log_int(rng, 1, min(most, 8000)) for _ in range(n)))
        c["nodes"] = _text(rng.choice([tree, rng.randint(1, tree)]) for _ in range(n))
    elif kind == "select":
        c = {"kind": kind, "requests": _log_int(rng, 1, 32), "beams": rng.choice([1, 2, 3, 4, 5, 8]),
             "vocab": rng.choice([152064, _log_int(rng, 100, 152064)]), "ended": rng.choice([0.0, 0.0, 0.2])}
    elif kind == "step":
        n, beams = _log_int(rng, 1, 4), rng.choice([2, 4, 6, 8])
        since = [rng.choice([0, _log_int(rng, 1, 600)]) for _ in range(n)]
        c.update(type="f16", requests=n, beams=beams, vocab=rng.choice([152064, _log_int(rng, 200, 152064)]),
                 layers=_log_int(rng, 1, 12), since=_text(since), lens=_text(s + _log_int(rng, 1, 400) for s in since))
    else:
        n, tree = _log_int(rng, 1, 32), rng.randint(2, 64)
        c.update(type="f16", layers=_log_int(rng, 1, 28), tree=tree, lens=_text(_log_int(rng, 1, 900) for _ in range(n)),
                 kept=_text(rng.randint(1, max(1, tree // 4)) for _ in range(n)))
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


def _codes(x, kind):
    """Cache rows of x [..., head_dim]: codes and scales."""
    a = x.abs()
    amax = torch.where(a < FLT_MIN, torch.zeros_like(a), a).amax(-1)
    if kind == "q8":
        scale = amax * np.float32(1 / 127)
        inv = torch.where(scale > 0, torch.div(torch.full_like(amax, 127.0), amax), torch.zeros_like(amax))
        return torch.round(x * inv.unsqueeze(-1)).clamp(-127, 127).to(torch.int8), scale
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


def _layers(case, g, slots, max_seq):
    """The caches of all layers, one after the other in each array."""
    one = _cache(case, g, slots, max_seq)
    out = {n: torch.empty(case["layers"], *x.shape, dtype=x.dtype, device="cuda") for n, x in one.items()}
    for i in range(case["layers"]):
        for n, x in (one if i == 0 else _cache(case, g, slots, max_seq)).items():
            out[n][i] = x
    return out


def _round_up(n):
    return (n + 63) // 64 * 64


def _parents(rng, n):
    """A tree of n nodes, each after its parent; node 0 the root."""
    return [-1] + [rng.randrange(max(0, j // 3 - 2), (j + 1) // 2 + 1) if j > 2 else 0 for j in range(1, n)]


def _seen(parents):
    """Bit i of node j's mask: the node itself or one that leads to it."""
    seen = []
    for j, p in enumerate(parents):
        seen.append(1 << j | (seen[p] if p >= 0 else 0))
    return seen


def _signed(v):
    return v - (1 << 64) if v >> 63 else v


def _logits(case, g, rng):
    """A step's logits and the beams' scores. For "step" half of the beams hold two likely tokens each, so that these
    survive and the others do not; "select" takes what comes."""
    n, K, V = case["requests"], case["beams"], case["vocab"]
    logits = _randn(g, n * K, V) * 2.0
    score = -30.0 + 2.0 * torch.rand(n * K, generator=g, device="cuda")
    if case["kind"] == "step":
        at = [(r * K + b, t) for r in range(n) for b in rng.sample(range(K), K // 2) for t in rng.sample(range(V), 2)]
        rows, toks = (torch.tensor(x, device="cuda") for x in zip(*at))
        logits[rows, toks] = 25.0 + torch.rand(len(at), generator=g, device="cuda")
        score -= 10.0
        score[rows.unique()] += 10.0
    else:
        rows = torch.arange(n * K, device="cuda").repeat_interleave(3)
        toks = torch.randint(0, V, (3 * n * K,), generator=g, device="cuda")
        logits[rows, toks] += 8.0
    done = _i32([int(rng.random() < case.get("ended", 0.0)) for _ in range(n * K)])
    return {"logits": logits, "score": score, "done": done, "eos": V // 2}


def _tree_inputs(case, rng):
    """Trees with their tokens and the model's picks: `kept` nodes of each are followed, the root first. What is followed
    stands past the places that it moves to."""
    N, out = case["tree"], {"parent": [], "token": [], "pick": []}
    for kept in _ints(case["kept"]):
        parents = _parents(rng, N)
        kept = max(1, min(kept, (N + 1) // 2))
        path = [0] + sorted(rng.sample(range(kept, N), kept - 1))
        for a, b in zip(path, path[1:]):
            parents[b] = a
        token = [rng.randrange(50000) for _ in range(N)]
        pick = [50000 + rng.randrange(50000) for _ in range(N)]   # (elsewhere no pick is a child's token)
        for a, b in zip(path, path[1:]):
            pick[a] = token[b] = 100000 + rng.randrange(50000)
        for name, v in (("parent", parents), ("token", token), ("pick", pick)):
            out[name].append(v)
    return {n: _i32(v) for n, v in out.items()}


def prepare(case, seed):
    if own:
        _lib()
    g, rng, kind = _gen(seed), random.Random(seed * 7919 + 13), case["kind"]
    s = {"case": case}
    if kind in ("select", "step"):
        n, K = case["requests"], case["beams"]
        s.update(_logits(case, g, rng), pick=2 * K if kind == "select" else K)
        s["parent"], s["token"], s["ended"] = (torch.zeros(n, s["pick"], dtype=torch.int32, device="cuda") for _ in range(3))
        s["best"] = torch.zeros(n, s["pick"], device="cuda")
        if kind == "step":
            s["since"], s["len"] = _i32(_ints(case["since"])), _i32(_ints(case["lens"]))
            s["max_seq"] = _round_up(max(_ints(case["lens"])))
            s["cache"] = _layers(case, g, n * K, s["max_seq"])
        return s
    lens, H, hd = _ints(case["lens"]), case["heads"], case["head_dim"]
    n_seq = len(lens)
    s.update(lens=lens, len_d=_i32(lens), slot_d=_i32(list(range(n_seq))))
    if kind == "accept":
        N = case["tree"]
        s.update(_tree_inputs(case, rng), max_seq=_round_up(max(lens) + N))
        s["cache"] = _layers(case, g, n_seq, s["max_seq"])
        s["seen"] = torch.zeros(n_seq, N, dtype=torch.int64, device="cuda")
        s["at"], s["row"], s["turn"], s["path"] = (torch.zeros(n_seq, N, dtype=torch.int32, device="cuda") for _ in range(4))
        s["n_path"], s["next"], s["ends"] = (torch.zeros(n_seq, dtype=torch.int32, device="cuda") for _ in range(3))
        return s
    if kind == "tree":
        N = case["tree"]
        s["seen"] = torch.tensor([[_signed(v) for v in _seen(_parents(rng, m))] + [0] * (N - m) for m in _ints(case["nodes"])],
                                 dtype=torch.int64, device="cuda")
        s["max_seq"], rows = _round_up(max(lens) + N), n_seq * N
    elif kind == "window":
        s["max_seq"], rows = _round_up(max(lens)), n_seq
    else:
        s["starts"] = _ints(case["starts"])
        s["max_seq"], rows = _round_up(max(a + b for a, b in zip(s["starts"], lens))), sum(lens)
        s["host"] = [np.array(v, dtype=np.int32) for v in (list(range(n_seq)), s["starts"], lens)]
    s["cache"] = _cache(case, g, n_seq + (1 if case.get("prefix") else 0), s["max_seq"])   # (the last slot: the prefix)
    s["q"], s["out"] = _randn(g, rows, H * hd), torch.zeros(rows, H * hd, device="cuda")
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


def _views(s):
    """The calls' descriptions of the caches, one a layer."""
    from hako_amd.gpu import KV_F16, KV_Q8, Kv
    case, c = s["case"], s["cache"]
    n = case.get("layers", 1)
    slots = c["k"].shape[-4]
    step = [c[name].numel() * c[name].element_size() // n for name in ("k", "v", "ks", "vs")]
    at = [c[name].data_ptr() for name in ("k", "v", "ks", "vs")]
    return [Kv(KV_Q8 if case["type"] == "q8" else KV_F16, slots, s["max_seq"], case["kv_heads"], case["head_dim"],
               *(a + i * b for a, b in zip(at, step))) for i in range(n)]


def _kv(s):
    """The same, made once: as one description, or as the list of all layers' that the calls over layers take."""
    if "kv" not in s:
        s["kv"] = _gpu.kv_layers(_views(s)) if "layers" in s["case"] else _views(s)[0]
    return s["kv"]


def _own_run(s):
    """The calls, on the library's stream: in order with torch's work there, and made to be so for a caller on another."""
    _lib()
    if torch._C._cuda_getCurrentRawStream(0) == _stream.cuda_stream:
        return _own_calls(s)
    caller = torch.cuda.current_stream()
    _stream.wait_stream(caller)
    out = _own_calls(s)
    caller.wait_stream(_stream)
    return out


def _own_calls(s):
    gpu, case = _gpu, s["case"]
    kind = case["kind"]
    if kind in ("select", "step"):
        n, K, V = case["requests"], case["beams"], case["vocab"]
        gpu.beam_select(s["logits"].data_ptr(), V, V, s["score"].data_ptr(), s["done"].data_ptr(), s["eos"], n, K, s["pick"],
                        kind == "step", s["parent"].data_ptr(), s["token"].data_ptr(), s["best"].data_ptr(), s["ended"].data_ptr())
        out = {"parent": s["parent"], "token": s["token"], "score": s["best"], "done": s["ended"]}
        if kind == "select":
            return out
        gpu.kv_reorder(_kv(s), None, s["parent"].data_ptr(), n, K, s["since"].data_ptr(), s["len"].data_ptr())
        return dict(out, **s["cache"])
    if kind == "accept":
        n, N = len(s["lens"]), case["tree"]
        slot, base, parent = s["slot_d"].data_ptr(), s["len_d"].data_ptr(), s["parent"].data_ptr()
        gpu.tree_plan(slot, base, parent, n, N, s["seen"].data_ptr(), s["at"].data_ptr(), s["row"].data_ptr(), s["turn"].data_ptr())
        gpu.tree_accept(parent, s["token"].data_ptr(), s["pick"].data_ptr(), base, n, N, s["path"].data_ptr(),
                        s["n_path"].data_ptr(), s["next"].data_ptr(), s["ends"].data_ptr())
        gpu.kv_keep(_kv(s), slot, base, s["path"].data_ptr(), s["n_path"].data_ptr(), n, N)
        return dict(s["cache"], **{name: s[name] for name in ("seen", "at", "row", "turn", "path", "n_path", "next", "ends")})
    H, D, scale = case["heads"], case["heads"] * case["head_dim"], 1.0 / math.sqrt(case["head_dim"])
    kv, n, q, out = _kv(s), len(s["lens"]), s["q"].data_ptr(), s["out"].data_ptr()
    if kind == "window":
        gpu.attn_decode_window(out, D, q, D, kv, s["slot_d"].data_ptr(), s["len_d"].data_ptr(), n, H, scale, case["window"],
                               case["sinks"])
    elif kind == "window_prompt":
        gpu.attn_prompt_window(out, D, q, D, kv, *s["host"], n, H, scale, case["window"], case["sinks"])
    else:
        gpu.attn_tree(out, D, q, D, kv, s["slot_d"].data_ptr(), s["len_d"].data_ptr(), s["seen"].data_ptr(), n, case["tree"], H,
                      scale, n, case["prefix"])
    return s["out"]


# ── the same with plain torch ──

def _rows(s, name, slot, pos):
    """Cached rows as values, the axes of slot and pos, then kv heads and head_dim."""
    c = s["cache"]
    return c[name][slot, :, pos].float() * c[name + "s"][slot, :, pos].unsqueeze(-1)


def _softmax(sc, seen):
    """Weights over the last axis where `seen`, 0 elsewhere and throughout where nothing is."""
    sc = sc.masked_fill(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return e / e.sum(-1, keepdim=True).clamp_min(FLT_MIN)


def _plain_window(s):
    case, W, S = s["case"], s["case"]["window"], s["case"]["sinks"]
    KVH, hd, n = case["kv_heads"], case["head_dim"], len(s["lens"])
    ends = s["len_d"].long().unsqueeze(1)
    own_ = torch.arange(min(W, max(s["lens"])), device="cuda").expand(n, -1) + (ends - W).clamp_min(0)   # the window's positions
    first = torch.arange(min(S, max(s["lens"])), device="cuda").expand(n, -1)
    p = torch.cat([first, own_], 1)
    seen = torch.cat([first < (ends - W).clamp_min(0), own_ < ends], 1)
    slot = s["slot_d"].long().unsqueeze(1)
    p = p.clamp_max(s["max_seq"] - 1)
    k, v = (_rows(s, name, slot, p).transpose(1, 2).contiguous() for name in "kv")   # [sequence][kv head][key][dim]
    q = s["q"].reshape(n, KVH, -1, hd)
    w = _softmax(q @ k.transpose(2, 3).contiguous() / math.sqrt(hd), seen[:, None, None, :])
    return (w @ v).reshape(n, -1)


def _plain_window_prompt_one(s, q, slot, start):
    """One sequence's prompt, some tokens at a time over the positions that one of them sees."""
    case, n, W, S = s["case"], len(q), s["case"]["window"], s["case"]["sinks"]
    KVH, hd, out = case["kv_heads"], case["head_dim"], []
    for a in range(0, n, 1024):
        b = min(n, a + 1024)
        lo = max(0, start + a - W + 1)
        p = torch.cat([torch.arange(min(S, lo), device="cuda"), torch.arange(lo, start + b, device="cuda")])
        t = torch.arange(start + a, start + b, device="cuda").unsqueeze(1)
        seen = (p <= t) & ((p > t - W) | (p < S))
        k, v = (_rows(s, name, torch.full_like(p, slot), p).transpose(0, 1).contiguous() for name in "kv")   # [kv head][key][dim]
        x = q[a:b].reshape(b - a, KVH, -1, hd).permute(1, 2, 0, 3).reshape(KVH, -1, hd)   # rows: query heads of a group x tokens
        w = _softmax((x @ k.transpose(1, 2).contiguous() / math.sqrt(hd)).reshape(KVH, -1, b - a, len(p)), seen)
        out.append((w.reshape(KVH, -1, len(p)) @ v).reshape(KVH, -1, b - a, hd).permute(2, 0, 1, 3).reshape(b - a, -1))
    return torch.cat(out)


def _plain_tree(s):
    case, N, n = s["case"], s["case"]["tree"], len(s["lens"])
    KVH, hd, L = case["kv_heads"], case["head_dim"], max(s["lens"]) + s["case"]["tree"]
    p = torch.arange(L, device="cuda").expand(n, L)
    slot = torch.where(p < case["prefix"], n, s["slot_d"].long().unsqueeze(1))
    base = s["len_d"].long()[:, None, None]
    node = p[:, None, :] - base                                                         # [sequence][1][position]
    bit = (s["seen"][:, :, None] >> node.clamp(0, 63)) & 1                              # [sequence][node][position]
    seen = (s["seen"] != 0)[:, :, None] & ((node < 0) | ((bit != 0) & (node < N)))
    k, v = (_rows(s, name, slot, p).transpose(1, 2).contiguous() for name in "kv")      # [sequence][kv head][position][dim]
    q = s["q"].reshape(n, N, KVH, -1, hd).permute(0, 2, 3, 1, 4).reshape(n, KVH, -1, hd)
    sc = (q @ k.transpose(2, 3).contiguous() / math.sqrt(hd)).reshape(n, KVH, -1, N, L)
    w = _softmax(sc, seen[:, None, None])
    return (w.reshape(n, KVH, -1, L) @ v).reshape(n, KVH, -1, N, hd).permute(0, 3, 1, 2, 4).reshape(n * N, -1)


def _plain_select(s):
    """In 64 bits: continuations of two beams may lie next to each other."""
    case = s["case"]
    n, K, V, P = case["requests"], case["beams"], case["vocab"], s["pick"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    value = s["score"].double().unsqueeze(1) + (x - (top + torch.log(torch.exp(x - top).sum(1, keepdim=True))))
    ended = (s["done"] != 0).unsqueeze(1)
    at_eos = torch.arange(V, device="cuda") == s["eos"]
    value = torch.where(ended, torch.where(at_eos, s["score"].double().unsqueeze(1), -math.inf), value)
    value, flat = torch.sort(value.reshape(n, K * V), dim=1, descending=True, stable=True)
    value, flat = value[:, :P], flat[:, :P]
    found = value > -math.inf
    parent = torch.where(found, flat // V, -1)
    token = torch.where(found, flat % V, -1)
    done = (found & ((token == s["eos"]) | (s["done"].reshape(n, K).gather(1, parent.clamp_min(0)) != 0))).int()
    out = {"parent": parent.int(), "token": token.int(), "score": value.float(), "done": done}
    if case["kind"] == "select":
        return out
    # a parent's best pick goes to the parent's own place, the others best first to the places that are left
    same = parent[:, :, None] == parent[:, None, :]
    first = found & ~(same & torch.ones(P, P, dtype=torch.bool, device="cuda").tril(-1)).any(2)
    taken = torch.zeros(n, P + 1, dtype=torch.bool, device="cuda").scatter(1, torch.where(first, parent, P), True)[:, :P]
    free = torch.argsort(taken.int(), dim=1, stable=True)          # the free places first, in order
    rest = (~first).long().cumsum(1) - 1
    place = torch.where(first, parent, free.gather(1, rest.clamp_min(0)))
    return {name: torch.empty_like(v).scatter(1, place, v) for name, v in out.items()}


def _plain_step(s):
    out, K, c = _plain_select(s), s["case"]["beams"], s["cache"]
    parent = out["parent"].long()
    rows = torch.arange(parent.numel(), device="cuda").reshape(parent.shape)
    src = torch.where(parent >= 0, rows[:, :1] + parent, rows)
    moved = (src != rows).nonzero()
    for r, b in moved.tolist():     # (survivors stay where they are, so none of these is another's source)
        lo, hi = _ints(s["case"]["since"])[r], _ints(s["case"]["lens"])[r]
        for x in c.values():
            x[:, r * K + b, :, lo:hi] = x[:, int(src[r, b]), :, lo:hi]
    return dict(out, **c)


def _plain_accept(s):
    n, N = s["parent"].shape
    parent, base, c = s["parent"].long(), s["len_d"].long(), s["cache"]
    node = torch.arange(N, device="cuda")
    seen, depth, rows = torch.zeros(n, N, dtype=torch.int64, device="cuda"), torch.zeros(n, N, dtype=torch.int64, device="cuda"), torch.arange(n, device="cuda")
    for j in range(N):
        p, root = parent[:, j].clamp_min(0), parent[:, j] < 0
        seen[:, j] = torch.where(root, 0, seen[rows, p]) | (1 << j if j < 63 else -(1 << 63))
        depth[:, j] = torch.where(root, 0, depth[rows, p] + 1)
    path, count, here = torch.full((n, N), -1, device="cuda"), torch.ones(n, dtype=torch.int64, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    on = torch.ones(n, dtype=torch.bool, device="cuda")
    for _ in range(1, N):
        fits = (parent == here[:, None]) & (s["token"] == s["pick"][rows, here][:, None])
        on = on & fits.any(1)
        here = torch.where(on, torch.where(fits, node, N).amin(1).clamp_max(N - 1), here)
        path[rows, count.clamp_max(N - 1)] = torch.where(on, here, path[rows, count.clamp_max(N - 1)])
        count = count + on.long()
    q = torch.arange(N, device="cuda").expand(n, N)
    kept = q < count[:, None]
    sq, d = kept.nonzero(as_tuple=True)
    to, frm = base[sq] + d, base[sq] + path[sq, d]
    for x in c.values():
        x[:, sq, :, to] = x[:, sq, :, frm]
    return dict(c, seen=seen, at=rows[:, None].expand(n, N).int(), row=(base[:, None] + node).int(), turn=(base[:, None] + depth).int(),
                path=path.int(), n_path=count.int(), next=s["pick"][rows, here], ends=(base + count).int())


def run(state):
    s = state
    if own:
        return _own_run(s)
    kind = s["case"]["kind"]
    if kind == "window_prompt":
        q = torch.split(s["q"], s["lens"])
        return torch.cat([_plain_window_prompt_one(s, x, i, s["starts"][i]) for i, x in enumerate(q)])
    return {"window": _plain_window, "tree": _plain_tree, "select": _plain_select, "step": _plain_step, "accept": _plain_accept}[kind](s)


# ── what a pass cannot do without ──

def work(case):
    kind = case["kind"]
    if kind in ("select", "step"):
        n, K, V = case["requests"], case["beams"], case["vocab"]
        w = {"bytes": 4 * n * K * V, "flops": 5 * n * K * V}
        if kind == "step":
            row = 2 * case["kv_heads"] * (2 * case["head_dim"] + 4) * case["layers"]
            moved = sum(b - a for a, b in zip(_ints(case["since"]), _ints(case["lens"])))
            w["bytes"] += 2 * (K // 2) * moved * row     # half of the beams are read, the other half written
        return w
    lens, H, KVH, hd = _ints(case["lens"]), case["heads"], case["kv_heads"], case["head_dim"]
    row = 2 * KVH * (hd * (1 if case["type"] == "q8" else 2) + 4)   # a position's keys and values in the cache
    if kind == "accept":
        N = case["tree"]
        moved = sum(max(0, min(k, (N + 1) // 2) - 1) for k in _ints(case["kept"]))
        return {"bytes": 2 * moved * row * case["layers"] + len(lens) * N * 36, "flops": 0}
    if kind == "tree":
        prefix, N, nodes = case["prefix"], case["tree"], _ints(case["nodes"])
        held = min(prefix, max(lens)) + sum(max(0, m - prefix) + k for m, k in zip(lens, nodes))
        # (of its own tree a node sees about its depth: a handful)
        return {"bytes": held * row + len(lens) * N * (8 * H * hd + 8), "flops": 4 * H * hd * sum(m * k for m, k in zip(lens, nodes))}
    W, S = case["window"], case["sinks"]
    if kind == "window":
        held = sum(min(m, W + S) for m in lens)
        return {"bytes": held * row + 8 * len(lens) * H * hd, "flops": 4 * H * hd * held}
    held = seen = 0
    for a, m in zip(_ints(case["starts"]), lens):
        lo = max(0, a - W + 1)
        held += a + m - lo + min(S, lo)
        full = max(0, min(m, a + m - (W + S)))                  # tokens that see W + S positions
        seen += full * (W + S) + (m - full) * a + (m - full) * (m - full + 1) // 2
    return {"bytes": held * row + 8 * sum(lens) * H * hd, "flops": 4 * H * hd * seen}


# ── the same in 64 bits, from the definition ──

def _exact_attention(q, K, V, positions, sees):
    """Rows of q [rows][heads][dim] over some positions of one slot's values K, V [kv head][position][dim]; sees [rows][positions]."""
    H, hd = q.shape[1:]
    out = torch.zeros_like(q)
    for h in range(H):
        k, v = (x[h * K.shape[0] // H, positions] for x in (K, V))
        sc = (q[:, h] @ k.t() / math.sqrt(hd)).masked_fill(~sees, -math.inf)
        out[:, h] = torch.nan_to_num(torch.softmax(sc, 1)) @ v
    return out.flatten(1)


def _exact_select(s):
    case = s["case"]
    n, K, V, P = case["requests"], case["beams"], case["vocab"], s["pick"]
    names, got = ("parent", "token", "score", "done"), []
    for r in range(n):
        all_ = []
        for b in range(K):
            row, old = r * K + b, float(s["score"][r * K + b])
            if int(s["done"][row]):
                all_.append((-old, b, s["eos"], 1))
                continue
            logp = torch.log_softmax(s["logits"][row].double(), 0) + old
            v, t = torch.topk(logp, min(P + 4, V))
            all_ += [(-x, b, y, int(y == s["eos"])) for x, y in zip(v.tolist(), t.tolist()) if x > -math.inf]
        best = [(b, t, -x, e) for x, b, t, e in sorted(all_)[:P]]
        best += [(-1, -1, -math.inf, 0)] * (P - len(best))
        if case["kind"] == "step":
            place = [None] * P
            rest = []
            for c in best:
                if c[0] >= 0 and place[c[0]] is None:
                    place[c[0]] = c
                else:
                    rest.append(c)
            best = [c if c is not None else rest.pop(0) for c in place]
        got.append(best)
    return {name: torch.tensor([[c[i] for c in row] for row in got], dtype=torch.float64 if name == "score" else torch.int32, device="cuda")
            for i, name in enumerate(names)}


def _exact_step(s):
    out, K = _exact_select(s), s["case"]["beams"]
    new = {name: x.clone() for name, x in s["cache"].items()}
    for r, row in enumerate(out["parent"].tolist()):
        lo, hi = _ints(s["case"]["since"])[r], _ints(s["case"]["lens"])[r]
        for b, p in enumerate(row):
            if p >= 0:
                for name, x in s["cache"].items():
                    new[name][:, r * K + b, :, lo:hi] = x[:, r * K + p, :, lo:hi]
    return dict(out, **new)


def _exact_accept(s):
    N = s["parent"].shape[1]
    new = {name: x.clone() for name, x in s["cache"].items()}
    out = {name: [] for name in ("seen", "at", "row", "turn", "path", "n_path", "next", "ends")}
    for i, (parent, token, pick, base) in enumerate(zip(s["parent"].tolist(), s["token"].tolist(), s["pick"].tolist(), s["lens"])):
        chains = []
        for j in range(N):
            chain = [j]
            while parent[chain[-1]] >= 0:
                chain.append(parent[chain[-1]])
            chains.append(chain)
        path = [0]
        while True:
            child = [j for j in range(N) if parent[j] == path[-1] and token[j] == pick[path[-1]]]
            if not child:
                break
            path.append(child[0])
        for d, j in enumerate(path):
            for name, x in s["cache"].items():
                new[name][:, i, :, base + d] = x[:, i, :, base + j]
        for name, v in (("seen", [_signed(sum(1 << a for a in c)) for c in chains]), ("at", [i] * N),
                        ("row", [base + j for j in range(N)]), ("turn", [base + len(c) - 1 for c in chains]),
                        ("path", path + [-1] * (N - len(path))), ("n_path", len(path)), ("next", pick[path[-1]]), ("ends", base + len(path))):
            out[name].append(v)
    return dict(new, **{name: torch.tensor(v, dtype=torch.int64 if name == "seen" else torch.int32, device="cuda") for name, v in out.items()})


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("select", "step", "accept"):
        return {"select": _exact_select, "step": _exact_step, "accept": _exact_accept}[case["kind"]](s)
    H, hd, c, kind, n = case["heads"], case["head_dim"], s["cache"], case["kind"], len(s["lens"])
    out, row = [], 0
    for i, m in enumerate(s["lens"]):
        K, V = (c[x][i].double() * c[x + "s"][i].double().unsqueeze(-1) for x in "kv")
        if kind == "tree":
            N, P = case["tree"], case["prefix"]
            if P:
                for x, name in ((K, "k"), (V, "v")):
                    x[:, :P] = c[name][n, :, :P].double() * c[name + "s"][n, :, :P].double().unsqueeze(-1)
            pos = torch.arange(m + N, device="cuda")
            bits = [[v >> j & 1 for j in range(N)] for v in s["seen"][i].tolist()]
            sees = torch.tensor([[1 if any(b) else 0] * m + b for b in bits], dtype=torch.bool, device="cuda")
            out.append(_exact_attention(s["q"][i * N:i * N + N].double().reshape(N, H, hd), K, V, pos, sees))
            continue
        W, S = case["window"], case["sinks"]
        tokens, start = (1, m - 1) if kind == "window" else (m, s["starts"][i])
        for a in range(0, tokens, 2048):
            b = min(tokens, a + 2048)
            lo = max(S, start + a - W + 1)
            pos = torch.cat([torch.arange(min(S, start + b), device="cuda"), torch.arange(lo, max(lo, start + b), device="cuda")])
            t = torch.arange(start + a, start + b, device="cuda").unsqueeze(1)
            sees = (pos <= t) & ((t - pos < W) | (pos < S))
            out.append(_exact_attention(s["q"][row + a:row + b].double().reshape(b - a, H, hd), K, V, pos, sees))
        row += tokens
    return torch.cat(out)
