"""The decoder on 8- and 16-bit caches (hako_gpu_decoder_create_kv).

A step is held against a forward in numpy (the oracle's matmuls, float64
attention) over the values that the caches stand for, the new row rounded as
the cache rounds it. What separates the two: the q8 rounding of the
activations, where a value next to an edge falls on the other side (up to
5e-4 of the logits' range a layer, as in the batched step's tests), and with
it the new key's codes: a drift of 5e-4 of a row's maximum moves 6% of the
8-bit codes (127 of them to the maximum) by a step of 1/127, 0.2% of the row
in the root mean square, and a half's by 2^-11. Three layers: 4e-3 (8 bits)
and 2e-3 (halves) of the largest logit.

Against the fp32 decoder's prompt every key and value differs by its
rounding, up to 1/254 of a row's maximum (8 bits; three times its root mean
square: 0.7% of that) or 2^-11; through up to three layers 5% and 1% of the
largest logit are the bars there.
"""
import ctypes as C

import numpy as np
import pytest

import attn_ref as ref
from hako_amd import mlf2
from hako_amd.decoder import Decoder
from hako_amd.gpu import KV_F16, KV_Q8, HakoGpuError
from helpers import maxabs_rel, within
from test_gpu_decode_batched import DENSE, KQM, SMALL_128, TINY, UNTIED_Q4_OUT

pytestmark = pytest.mark.gpu

STEP_BAR = {KV_Q8: 4e-3, KV_F16: 2e-3}


def rows_of(gpu, dec, kv, seq, upto):
    """Values of positions [0, upto) of a sequence in one layer's cache, through the cache calls."""
    kvd = dec.kv_dim
    bufs = [gpu.upload(np.full(upto, seq, np.int32)), gpu.upload(np.arange(upto, dtype=np.int32)),
            gpu.alloc(4 * upto * kvd), gpu.alloc(4 * upto * kvd)]
    gpu.kv_read(kv, bufs[0], bufs[1], upto, bufs[2], bufs[3], kvd)
    out = [gpu.download(b, np.float32, (upto, kvd)) for b in bufs[2:]]
    for b in bufs:
        b.free()
    return out


class Forward:
    """The model's forward for one token in numpy, on given cached values."""

    def __init__(self, oracle, path):
        self.f = mlf2.Mlf2File(path)
        self.h, self.oracle = self.f.header, oracle

    def mul(self, name, x, n_out, bias=None):
        b = self.f.data(bias).view(np.float32) if bias in self.f.tensors else None
        return self.oracle.matmul(int(self.f.tensors[name]["type"]), self.f.data(name), x, n_out, x.size, b)

    def norm(self, x, name):
        w = self.f.data(name).view(np.float32).astype(np.float64)
        x = x.astype(np.float64)
        return (x / np.sqrt((x * x).mean() + self.h["rms_eps"]) * w).astype(np.float32)

    def step(self, token, caches, pos, kind):
        """Logits, and the new rows' values per layer; caches: per layer (k, v) values [pos][kv_dim]."""
        h = self.h
        D, H, KVH, hd = h["d_model"], h["n_heads"], h["n_kv_heads"], h["head_dim"]
        F, V = h["ffn_dim"], h["vocab"]
        emb = "token_embd.weight"
        t = int(self.f.tensors[emb]["type"])
        row = self.f.data(emb).view(np.uint8).reshape(V, -1)[token].copy()
        x = self.oracle.dequant(t, row, D).astype(np.float32)
        tab = ref.table(pos + 1, hd, float(h["rope_theta"]))[pos:]
        new = []
        for l in range(h["n_layers"]):
            p = f"blk.{l}."
            xn = self.norm(x, p + "attn_norm.weight")
            q, k, v = (self.mul(f"{p}attn_{c}.weight", xn, n, f"{p}attn_{c}.bias") for c, n in (("q", D), ("k", KVH * hd), ("v", KVH * hd)))
            q = ref.rotate(q.reshape(1, H, hd), tab, hd, 0)[0]
            k = ref.rotate(k.reshape(1, KVH, hd), tab, hd, 0)[0]
            ck, cv = (c.astype(np.float64) * s.astype(np.float64)[:, None] for c, s in (ref.rows(k, kind), ref.rows(v.reshape(KVH, hd), kind)))
            new.append((ck.ravel(), cv.ravel()))
            K, V2 = (np.concatenate([old.reshape(pos, KVH, hd), n[None]]).transpose(1, 0, 2)[None] for old, n in zip(caches[l], (ck, cv)))
            att = ref.attend(q, K, V2, 0, pos + 1, 1 / np.sqrt(hd)).ravel().astype(np.float32)
            x = x + self.mul(p + "attn_output.weight", att, D)
            xn = self.norm(x, p + "ffn_norm.weight")
            g, u = (self.mul(f"{p}ffn_{c}.weight", xn, F).astype(np.float64) for c in ("gate", "up"))
            x = x + self.mul(p + "ffn_down.weight", (g / (1 + np.exp(-g)) * u).astype(np.float32), D)
        out = "output.weight" if "output.weight" in self.f.tensors else emb
        return self.mul(out, self.norm(x, "output_norm.weight"), V), new


@pytest.mark.parametrize("kind", [KV_Q8, KV_F16])
@pytest.mark.parametrize("cfg,n_seq", [(TINY, 1), (SMALL_128, 1), (DENSE, 1), (SMALL_128, 3), (UNTIED_Q4_OUT, 2), (KQM, 16),
                                       (DENSE, 4)])
def test_step(gpu, oracle, tmp_path, kind, cfg, n_seq):
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, cfg, 21)
    rng = np.random.default_rng(n_seq)
    n = [int(x) for x in rng.integers(32, 120, n_seq)]
    dec = Decoder(gpu, path, n_seq, 160, kind)
    try:
        for s, m in enumerate(n):
            dec.prefill(rng.integers(0, cfg.vocab, m), s)
        tok = rng.integers(0, cfg.vocab, n_seq).astype(np.int32)
        layers = [dec.cache(l) for l in range(cfg.n_layers)]
        before = [[rows_of(gpu, dec, kv, s, n[s]) for kv in layers] for s in range(n_seq)]
        nxt, lg = dec.step(tok, logits=True)
        after = [[rows_of(gpu, dec, kv, s, n[s] + 1) for kv in layers] for s in range(n_seq)]
    finally:
        dec.close()
    assert (nxt == np.argmax(lg, 1)).all()
    fwd = Forward(oracle, path)
    for s in range(n_seq):
        want, new = fwd.step(int(tok[s]), before[s], n[s], kind)
        for l in range(cfg.n_layers):
            for i in range(2):   # a step leaves the rows before it alone
                np.testing.assert_array_equal(after[s][l][i][:-1], before[s][l][i])
        for i in range(2):       # layer 0's new row: its inputs differ by fp32 rounding alone, so by a code at most
            got, w = (a.reshape(-1, cfg.head_dim) for a in (after[s][0][i][-1], new[0][i]))
            step = 1 / 127 if kind == KV_Q8 else 2.0 ** -10
            assert (np.abs(got - w) <= (step + 1e-5) * np.abs(w).max(1, keepdims=True)).all()
            assert (np.abs(got - w) > 1e-5 * np.abs(w).max(1, keepdims=True)).mean() < 0.05
        within(f"sequence {s}", lg[s], want, STEP_BAR[kind])


@pytest.mark.parametrize("kind,bar", [(KV_Q8, 0.05), (KV_F16, 0.01)])
@pytest.mark.parametrize("cfg", [TINY, SMALL_128])
def test_prompt_and_greedy_tokens(gpu, tmp_path, kind, bar, cfg):
    """A prompt over two passes, then captured greedy steps: near the fp32 decoder's, and repeatable."""
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, cfg, 5)
    prompt = np.random.default_rng(1).integers(0, cfg.vocab, 700)
    runs = []
    for t in (0, kind, kind):
        dec = Decoder(gpu, path, 1, 760, t)
        try:
            nxt, lg = dec.prefill(prompt, logits=True)
            runs.append((lg, dec.generate(nxt, 12).ravel()))
        finally:
            dec.close()
    (want, _), (a, ta), (b, tb) = runs
    print(f"[bar] prompt: {maxabs_rel(a, want):.3e}")
    assert maxabs_rel(a, want) < bar
    np.testing.assert_array_equal(a, b)
    np.testing.assert_array_equal(ta, tb)


@pytest.mark.parametrize("kind", [KV_Q8, KV_F16])
def test_generate_equals_steps(gpu, tmp_path, kind):
    """The captured step, the eager step and a replay give the same tokens."""
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, SMALL_128, 6)
    dec = Decoder(gpu, path, 3, 200, kind)
    try:
        rng = np.random.default_rng(2)
        for s in range(3):
            dec.prefill(rng.integers(0, SMALL_128.vocab, 40 + 30 * s), s)
        start = [40, 70, 100]
        tok = np.array([1, 2, 3], np.int32)
        out = dec.generate(tok, 6)
        dec.set_pos(start)
        cur, got = tok, []
        for _ in range(6):
            cur = dec.step(cur)
            got.append(cur)
        np.testing.assert_array_equal(np.stack(got), out)
        dec.set_pos(start)
        np.testing.assert_array_equal(dec.generate(tok, 6), out)
    finally:
        dec.close()


@pytest.mark.parametrize("kind", [KV_Q8, KV_F16])
def test_shared_prefix(gpu, tmp_path, kind):
    """A prefix stored once answers as the same prefix fed to every sequence; sharing can be ended and begun again."""
    cfg = SMALL_128
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, cfg, 7)
    rng = np.random.default_rng(3)
    prefix = rng.integers(0, cfg.vocab, 150)
    turns = [rng.integers(0, cfg.vocab, m) for m in (5, 20, 33, 1)]
    tok = np.array([4, 5, 6, 7], np.int32)
    dec = Decoder(gpu, path, 4, 260, kind)
    try:
        for s in range(4):
            dec.prefill(prefix, s)
            dec.prefill(turns[s], s)
        nxt, want = dec.step(tok, logits=True)
        want_gen = dec.generate(nxt, 5)
    finally:
        dec.close()
    dec = Decoder(gpu, path, 4, 260, kind)
    try:
        dec.prefill(prefix, 2)
        dec.generate(tok, 2)   # a step captured without the prefix: not the one replayed below
        dec.share_prefix(2, len(prefix))
        dec.set_pos(len(prefix))
        for s in range(4):
            dec.prefill(turns[s], s)
        nxt, got = dec.step(tok, logits=True)
        # the prefix's weights meet in another order: fp32 sums, and the q8 edges after them
        within("shared prefix", got, want, 1e-3)
        np.testing.assert_array_equal(nxt, np.argmax(got, 1))
        gen = dec.generate(nxt, 5)
        assert gen.shape == want_gen.shape
        with pytest.raises(HakoGpuError, match="prefix"):
            dec.set_pos(len(prefix) - 1)
            dec.step(tok)
        with pytest.raises(HakoGpuError, match="prefix"):
            dec.prefill([1, 2], 0)
        dec.share_prefix(0, 0)
        dec.set_pos(3)
        dec.step(tok)
    finally:
        dec.close()


def test_refusals(gpu, tmp_path):
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, TINY, 1)
    with pytest.raises(HakoGpuError, match="cache type"):
        Decoder(gpu, path, 1, 64, 9)
    plain, typed = Decoder(gpu, path, 1, 64), None
    try:
        with pytest.raises(HakoGpuError, match="8 or 16 bits"):
            plain.share_prefix(0, 5)
        with pytest.raises(HakoGpuError, match="fp32"):
            plain.cache(0)
    finally:
        plain.close()
    typed = Decoder(gpu, path, 2, 64, KV_Q8)
    try:
        with pytest.raises(HakoGpuError, match="not fp32"):
            typed.kv()
        for bad in ((-1, 0), (2, 0), (0, -1), (0, 65)):
            with pytest.raises(HakoGpuError, match="prefix of"):
                typed.share_prefix(*bad)
        with pytest.raises(HakoGpuError, match="layer"):
            typed.cache(2)
        k = typed.cache(1)
        assert (k.type, k.n_slots, k.max_seq, k.head_dim) == (KV_Q8, 2, 64, 64) and C.sizeof(k) > 0
    finally:
        typed.close()


@pytest.mark.parametrize("kind", [KV_Q8, KV_F16])
@pytest.mark.parametrize("cfg", [SMALL_128, TINY])
def test_captured_steps_follow_the_prefix(gpu, tmp_path, kind, cfg):
    """Captured steps against eager ones on the same decoder, bit for bit: without a prefix, under one (the step captured
    before is not replayed), after its end (as a decoder that never shared one), and under one again. Besides the tokens
    (a random model soon repeats one, whatever it sees) the rows that the steps write in the last layer's cache count:
    they follow from the attention of the layers before it."""
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, cfg, 9)
    rng = np.random.default_rng(11)
    prefix = rng.integers(0, cfg.vocab, 130)
    turns = [rng.integers(0, cfg.vocab, m) for m in (5, 40, 17)]
    plain = [rng.integers(0, cfg.vocab, m) for m in (60, 9, 33)]
    tok, n = np.array([4, 5, 6], np.int32), 6
    assert cfg.n_layers > 1

    def written(dec, pos):
        """Keys and values of the n positions from pos on."""
        return np.stack([[x[p:] for x in rows_of(gpu, dec, dec.cache(cfg.n_layers - 1), s, p + n)] for s, p in enumerate(pos)])

    def fed(dec, at, prompts):
        """Prompts from position `at`, then n captured steps; the same steps eagerly, and captured again, write the same."""
        dec.set_pos(at)
        for s, p in enumerate(prompts):
            dec.prefill(p, s)
        pos = [at + len(p) for p in prompts]
        gen = dec.generate(tok, n)
        rows = written(dec, pos)
        assert np.isfinite(rows).all()
        dec.set_pos(pos)
        cur, eager = tok, []
        for _ in range(n):
            cur = dec.step(cur)
            eager.append(cur)
        np.testing.assert_array_equal(gen, np.stack(eager))
        np.testing.assert_array_equal(rows, written(dec, pos))
        dec.set_pos(pos)
        np.testing.assert_array_equal(dec.generate(tok, n), gen)
        np.testing.assert_array_equal(rows, written(dec, pos))
        return rows

    other = Decoder(gpu, path, 3, 260, kind)
    try:
        want = fed(other, 0, plain)
    finally:
        other.close()
    dec = Decoder(gpu, path, 3, 260, kind)
    try:
        np.testing.assert_array_equal(fed(dec, 0, plain), want)
        shared = []
        for owner in (1, 2):
            dec.set_pos(0)
            dec.prefill(prefix, owner)
            dec.share_prefix(owner, len(prefix))
            shared.append(fed(dec, len(prefix), turns))
            dec.share_prefix(0, 0)
            np.testing.assert_array_equal(fed(dec, 0, plain), want)
        np.testing.assert_array_equal(shared[0], shared[1])
        # and the prefix counts: without it every sequence's rows come out otherwise
        assert (fed(dec, len(prefix), turns) != shared[0]).any((1, 2, 3)).all()
    finally:
        dec.close()


class Model(C.Structure):
    """hakm_model (include/hako_mlf2.h)."""
    _fields_ = [("h", C.c_char * 128), ("tensors", C.c_void_p), ("data", C.c_void_p), ("tok", C.c_void_p), ("map", C.c_void_p),
                ("map_size", C.c_size_t)]


@pytest.mark.parametrize("kind", [0, KV_Q8, KV_F16])
def test_decoder_from_a_mapped_model(gpu, tmp_path, kind):
    """hako_decoder_from_model_kv over a model in host memory: the decoder of the same file and cache type, bit for bit."""
    from dropin import host_lib
    path = str(tmp_path / "m.mlf2")
    mlf2.write_qwen2(path, SMALL_128, 13)
    prompt, tok = np.random.default_rng(1).integers(0, SMALL_128.vocab, 40).astype(np.int32), np.array([5], np.int32)
    dec = Decoder(gpu, path, 1, 64, kind)
    try:
        dec.prefill(prompt, 0)
        want = dec.step(tok, logits=True)[1]
    finally:
        dec.close()
    image = np.fromfile(path, np.uint8)
    at = {n: int(np.frombuffer(image[o:o + 8].tobytes(), np.uint64)[0]) for n, o in (("tensors", 60), ("tok", 68), ("data", 76))}
    m = Model(image[:128].tobytes(), *(image.ctypes.data + at[n] for n in ("tensors", "data", "tok")), image.ctypes.data, image.nbytes)
    C.memmove(C.byref(m), image.ctypes.data, 128)   # (a char array field stops at a 0)
    host, lib, d = host_lib(), gpu.lib, C.c_void_p()
    host.hako_decoder_from_model_kv.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_int, C.POINTER(C.c_void_p)]
    assert host.hako_decoder_from_model_kv(C.byref(m), 1, 64, 9, C.byref(d)) == -6 and not d.value
    assert host.hako_decoder_from_model_kv(C.byref(m), 1, 64, kind, C.byref(d)) == 0
    try:
        assert host.hako_model_release(C.byref(m)) != 0   # its weights are in use
        lg = np.empty((1, SMALL_128.vocab), np.float32)
        assert lib.hako_gpu_decoder_prefill(d, 0, prompt.ctypes.data, len(prompt), None, None) == 0
        assert lib.hako_gpu_decoder_step(d, tok.ctypes.data, lg.ctypes.data, None) == 0
        np.testing.assert_array_equal(lg, want)
    finally:
        assert lib.hako_gpu_decoder_destroy(d) == 0
        assert host.hako_model_release(C.byref(m)) == 0
