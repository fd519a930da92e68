"""The decode runtime on the 8-bit K/V cache (tf_model_use_kv8)."""
import ctypes as C

import numpy as np
import pytest
import torch

import _op_ref as ref
import oracle
from _model_ref import RefModel, prefill64
from taraference_amd import capi, synth
from test_gpu_model import TINY
from test_gpu_prefill_model import calm

pytestmark = pytest.mark.gpu


class Kv8Ref(RefModel):
    """RefModel.step on rows held in 8 bits: RoPE and attention in 64 bits, over the rows
    that the model under test wrote.  Its rows come from activations that agree to about
    1e-6, so a few in 10^4 values fall a step apart, and one such value moves a 128-wide
    row by 1 / 50 / sqrt(128) = 2e-3 of it, 6e-3 of the RMS in the largest of 1000
    logits: taken over, the logits are held as closely as those of the f16 cache."""

    def __init__(self, cfg, layers, emb, max_seq):
        super().__init__(cfg, layers, emb, 8)
        self.apart = self.values = 0
        n = cfg["n_kv"] * cfg["head_dim"]
        self.rows = [[np.zeros((max_seq, n)) for _ in range(2)] for _ in layers]

    def step(self, token, pos):
        c = self.c
        e, hd, h, kv = c["n_embd"], c["head_dim"], c["n_head"], c["n_kv"]
        x = oracle.embed_row(self.E, 210, token, e, self.ecb)
        for li, L in enumerate(self.L):
            xb = oracle.rms_norm(x, L["attn_norm"], c["rms_eps"])
            q8, d8 = self._q8(xb)
            wq, cb = L["wq"]
            q, k = oracle.gemv_q4k_pair(wq, L["wk"][0], q8, d8, e, h * hd, kv * hd, cb, L["bq"],
                                        L["bk"])
            v = oracle.gemv_q6k_f32(L["wv"][0], xb, e, kv * hd, L["wv"][1], bias=L["bv"])
            q, k = (ref.norm_rope(a.reshape(1, -1, hd), None, 0, [pos], c["rope_theta"])[0]
                    .astype(np.float32).reshape(1, -1) for a in (q, k))
            k8, kd, v8, vd = (a[pos:pos + 1] for a in self.model.kv8_cache(li, pos + 1))
            for store, row, c8, cd in zip(self.rows[li], (k, v.reshape(1, -1)), (k8, v8), (kd, vd)):
                mine, d = ref.q8_rows(row)
                assert (np.abs(cd - d) <= 1e-4 * d).all()
                diff = np.abs(c8.astype(int) - mine.astype(int))
                assert diff.max() <= 1
                self.apart += int(diff.sum())
                self.values += diff.size
                store[pos] = ref.q8_values(c8, cd)[0]
            K, V = (r[:pos + 1] for r in self.rows[li])
            att = ref.attention(q.reshape(h, hd), K, V, kv, 1 / np.sqrt(hd))[0]
            x = self._global_q8(L["wo"], h * hd, att.reshape(-1).astype(np.float32), False, out=x)
            xb = oracle.rms_norm(x, L["ffn_norm"], c["rms_eps"])
            q8, d8 = self._q8(xb)
            g, gcb = L["gate"]
            hid = oracle.gemv_q4k_ffn(g, L["up"][0], q8, d8, e, c["n_ff"], gcb, 1)
            x = self._global_q8(L["down"], c["n_ff"], hid, L["down_q6k"], out=x)
        xb = oracle.rms_norm(x, np.ones(e, np.float32), c["rms_eps"])
        return self._global_q8((self.E, self.ecb), e, xb, True)


def build(ci, seed, max_seq):
    from taraference_amd.model import DecodeModel

    cfg = TINY[ci]
    rng = np.random.default_rng(seed)
    layers = calm([synth.qwen_layer(rng, cfg, li) for li in range(cfg["n_layer"])])
    emb = synth.qwen_embedding(rng, cfg)
    return cfg, layers, emb, lambda: DecodeModel(dict(cfg, max_seq=max_seq), layers, emb)


@pytest.mark.parametrize("ci", [0, 1])
def test_steps(gpu, ci):
    """Logits to 2e-3 of their RMS, as test_gpu_model has them over f16 rows."""
    cfg, layers, emb, make = build(ci, 40 + ci, 48)
    gm, rm = make(), Kv8Ref(cfg, layers, emb, 48)
    gm.use_kv8()
    rm.model = gm
    assert gm.path() == 0
    rng = np.random.default_rng(ci)
    toks = rng.integers(0, cfg["n_vocab"], 24).tolist()
    for pos, tok in enumerate(toks):
        gm.forward(tok, pos)
        got, want = gm.logits().astype(np.float64), rm.step(tok, pos).astype(np.float64)
        assert np.abs(got - want).max() <= 2e-3 * np.sqrt(np.mean(want**2)), pos
    assert rm.apart <= 2e-3 * rm.values  # rows agree to 1e-5 RMS: one value in 10^3
    gm.close()


def test_graph_replays(gpu):
    cfg, layers, emb, make = build(1, 5, 64)
    gm = make()
    gm.use_kv8()
    gm.use_kv8()  # again: nothing to do
    prompt = list(range(5, 21))
    eager = gm.generate(prompt, 20, use_graph=False)
    for _ in range(3):
        assert np.array_equal(gm.generate(prompt, 20, use_graph=True), eager)
    gm.close()


def put_rows(f16, gm, cfg, rows):
    """gm's 8-bit rows 0 .. rows - 1, read back as f16, into the f16 model's cache."""
    hip = C.CDLL("libamdhip64.so.7")
    torch.cuda.synchronize()
    for li in range(cfg["n_layer"]):
        k8, kd, v8, vd = gm.kv8_cache(li, rows)
        for q, d, dst in ((k8, kd, f16.lib.tf_model_k_cache), (v8, vd, f16.lib.tf_model_v_cache)):
            x = (q.reshape(-1, 32).astype(np.float32) * d.reshape(-1, 1)).astype(np.float16)
            assert hip.hipMemcpy(C.c_void_p(dst(f16.h, li)), x.ctypes.data_as(C.c_void_p),
                                 C.c_size_t(x.nbytes), 1) == 0


@pytest.mark.parametrize("n,more", [(40, 0), (33, 21), (1024 + 37, 11)])
def test_prompts(gpu, n, more):
    """A chunk of a prompt attends over its own rows as they are and over earlier ones
    as the 8-bit cache has them: bit for bit what the f16 model gives once its earlier
    rows are those."""
    cfg, layers, emb, make = build(0, n, n + more + 8)
    toks = np.random.default_rng(n).integers(0, cfg["n_vocab"], n + more).tolist()
    f16, gm = make(), make()
    gm.use_kv8()
    done = 0
    for part in (n, more):
        if not part:
            continue
        tok = gm.prefill(toks[done:done + part], done)
        for at in range(done, done + part, 1024):  # the chunks of a call
            if at:
                put_rows(f16, gm, cfg, at)
            want = f16.prefill(toks[at:min(at + 1024, done + part)], at)
        done += part
        assert tok == want and np.array_equal(f16.logits(), gm.logits())
    # layer 0's rows: half a step from the exact ones, which f16 and the GEMM's 2e-4 of
    # the row's RMS (and the f32 angle, 2^-22 of a turned value a position) precede
    K, V, _ = prefill64(cfg, layers, emb, toks)
    k8, kd, v8, vd = gm.kv8_cache(0, n + more)
    for q, d, want, turn in ((k8, kd, K[0], 2.0**-22), (v8, vd, V[0], 0.0)):
        step = np.repeat(d.astype(np.float64), 32, axis=1)
        rms = np.sqrt(np.mean(want**2, axis=1, keepdims=True))
        near = 2e-4 * rms + np.abs(want) * 2.0**-10
        near = near + turn * np.arange(n + more)[:, None] * np.abs(want).max(1, keepdims=True)
        # the scale itself is as near, and so is every multiple of it up to 127
        assert (np.abs(ref.q8_values(q, d) - want) <= 0.5 * step + 2 * near + 2.0**-20 * rms).all()
    # and on with the decode path
    gm.generate([1], 3, pos0=n + more)
    f16.close()
    gm.close()


def test_refusals(gpu):
    _, _, _, make = build(0, 1, 16)
    gm = make()
    lib, h = gm.lib, gm.h
    assert not lib.tf_model_kv8_cache(h, 0, 0)
    assert lib.tf_model_use_kv8(None) == 1
    gm.use_kv8()
    for path in (1, 2, 3, 4):
        with pytest.raises(capi.HipError):
            gm.set_path(path)
    gm.set_path(0)
    assert not lib.tf_model_k_cache(h, 0) and not lib.tf_model_v_cache(h, 0)
    assert lib.tf_model_kv8_cache(h, 1, 3) and not lib.tf_model_kv8_cache(h, 1, 4)
    assert not lib.tf_model_kv8_cache(h, 2, 0) and not lib.tf_model_kv8_cache(h, -1, 0)
    with pytest.raises(capi.HipError):
        gm.kv_cache(0, 1)
    gm.close()


@pytest.mark.parametrize("pos", [0, 32000, 130000])
def test_steps_and_prompts_turn_rows_alike(gpu, pos):
    """A token's K row is turned by one angle whether a step or a prompt stores it, in 8 bits
    or in f16.  Layer 0's input is the embedding's row, so a step's rows are the same numbers
    in both caches: apart by half a step of each, and the rotation's roundings."""
    cfg, layers, emb, make = build(0, 11, pos + 24)
    f16, gm = make(), make()
    gm.use_kv8()
    f16.set_path(0)
    toks = np.random.default_rng(pos).integers(0, cfg["n_vocab"], 24).tolist()
    f16.generate(toks, 1, pos0=pos)
    gm.generate(toks, 1, pos0=pos)
    rows16 = [a[pos:].view(np.float16).astype(np.float64) for a in f16.kv_cache(0, pos + 24)]
    k8, kd, v8, vd = (a[pos:] for a in gm.kv8_cache(0, pos + 24))
    for q, d, want in ((k8, kd, rows16[0]), (v8, vd, rows16[1])):
        step, got = np.repeat(d.astype(np.float64), 32, axis=1), ref.q8_values(q, d)
        near = 2.0**-11 * np.abs(want) * (1 + 2.0**-10) + 2.0**-25
        near = near + 2.0**-21 * np.abs(want).max(1, keepdims=True)
        assert (np.abs(got - want) <= (0.5 + 2.0**-15) * step + near).all()
    # the same tokens as a prompt (whose GEMMs take x unquantised, the steps' GEMVs its Q8):
    # the f16 rows' Q8, exactly
    f16.prefill(toks, pos)
    gm.prefill(toks, pos)
    rows16 = [a[pos:].view(np.float16).astype(np.float32) for a in f16.kv_cache(0, pos + 24)]
    k8, kd, v8, vd = (a[pos:] for a in gm.kv8_cache(0, pos + 24))
    for q, d, rows in ((k8, kd, rows16[0]), (v8, vd, rows16[1])):
        want = ref.q8_rows(rows)
        assert np.array_equal(q, want[0]) and np.array_equal(d, want[1])
    f16.close()
    gm.close()


def test_the_8_bit_cache_takes_the_place_of_the_f16_one(gpu):
    """A model made with it never holds the f16 cache, one that is switched gives it back;
    both go on alike."""
    from taraference_amd.model import DecodeModel
    rows = 400_000
    cfg, layers, emb, _ = build(0, 9, rows)

    def make(**how):
        return DecodeModel(dict(cfg, max_seq=rows), layers, emb, **how)

    n = cfg["n_layer"] * rows * cfg["n_kv"] * cfg["head_dim"]
    other = 64 << 20  # weights and workspaces

    def used():
        torch.cuda.synchronize()
        return torch.cuda.mem_get_info()[1] - torch.cuda.mem_get_info()[0]

    warm = build(0, 9, 64)[3]()
    warm.prefill([1, 2, 3], 0)
    warm.generate([4], 2, pos0=3)
    warm.close()
    base = used()
    early = make(kv8=True)
    assert early.path() == 0 and early.kv8
    assert 2.25 * n <= used() - base < 2.25 * n + other
    early.generate([3, 4, 5], 3)
    assert used() - base < 2.25 * n + other
    want, tok = early.logits(), early.generate([3, 4, 5], 3)
    early.close()
    base = used()
    late = make()
    late.forward(7, 0)
    assert used() - base >= 4 * n
    late.use_kv8()
    assert used() - base < 2.25 * n + other
    assert np.array_equal(late.generate([3, 4, 5], 3), tok) and np.array_equal(late.logits(), want)
    late.prefill(list(range(20)), 0)
    assert used() - base < 2.25 * n + 4 * n / cfg["n_layer"] + 2 * other  # and a layer in f16
    late.close()


@pytest.mark.parametrize("kv8", [False, True])
def test_a_cache_that_does_not_fit(gpu, kv8):
    """Refused with hipErrorOutOfMemory, which the next launch does not report again."""
    from taraference_amd.model import DecodeModel
    cfg, layers, emb, make = build(1, 2, 16)
    gm = make()
    want = gm.generate([1, 2], 3, use_graph=False)
    with pytest.raises(capi.HipError, match="returned 2$"):
        DecodeModel(dict(cfg, max_seq=2**31 - 1), layers, emb, kv8=kv8)
    assert np.array_equal(gm.generate([1, 2], 3, use_graph=False), want)
    gm.close()


@pytest.mark.parametrize("start", [1, 31, 257, 600])
def test_steps_after_a_prompt_over_several_splits(gpu, start, monkeypatch):
    """Steps over rows that a prompt stored, in a cache that the attention splits (16 parts
    of 704 rows), eager, and captured bit for bit.  Rows are held as step() holds them; the
    logits by their norm, as a quotient that lies on a half may round either way in the Q8 of
    an activation: in the head's (512 values, none above 8 of their RMS) it moves the logits
    by 8 / 127 of that RMS times a column of the head, 8 / 127 / sqrt(512) = 2.8e-3 of their
    norm.  Four of them are allowed for: 1.2e-2."""
    cfg, layers, emb, make = build(1, 60, 704)
    gm, rm = make(), Kv8Ref(cfg, layers, emb, 704)
    gm.use_kv8()
    rm.model = gm
    assert gm.lib.tf_flash_decode_kv8_n_split(cfg["n_kv"], cfg["head_dim"], 704) == 16

    def turned(x, w, eps, at, theta):  # the reference's angle, as steps have it
        assert w is None and len(at) == 1
        y = oracle.rope_neox(np.asarray(x).reshape(-1), x.shape[1], x.shape[2], int(at[0]), theta)
        return y.reshape(x.shape), None

    monkeypatch.setattr(ref, "norm_rope", turned)
    toks = np.random.default_rng(start).integers(0, cfg["n_vocab"], start + 3).tolist()
    gm.prefill(toks[:start], 0)
    for li in range(cfg["n_layer"]):
        k8, kd, v8, vd = gm.kv8_cache(li, start)
        rm.rows[li][0][:start], rm.rows[li][1][:start] = ref.q8_values(k8, kd), ref.q8_values(v8, vd)
    for pos in range(start, start + 3):
        gm.forward(toks[pos], pos)
        got, want = gm.logits().astype(np.float64), rm.step(toks[pos], pos).astype(np.float64)
        assert np.linalg.norm(got - want) <= 1.2e-2 * np.linalg.norm(want), pos
    last = gm.logits()
    for graph in (False, True, True):
        gm.prefill(toks[:start], 0)
        nxt = gm.generate(toks[start:], 1, pos0=start, use_graph=graph)
        assert np.array_equal(gm.logits(), last) and nxt[0] == int(np.argmax(last))
    gm.close()


@pytest.mark.parametrize("max_seq", [40, 700])
def test_steps_of_a_q5_0_model(gpu, monkeypatch, max_seq):
    """Layers whose norm, q, k and v (and over an f16 cache wo) are fused launches of their
    own.  Attention in 64 bits over the rows that the model wrote; logits as
    test_gpu_q05_model has them."""
    from _model_ref import RefModelMixed
    from _util import q8_0_dequant
    from taraference_amd.model import DecodeModel
    from test_gpu_q05_model import CFG as cfg
    rng = np.random.default_rng(71)
    layers = [synth.qwen05_layer(rng, cfg, li) for li in range(cfg["n_layer"])]
    emb = synth.qwen05_embedding(rng, cfg)
    gm = DecodeModel(dict(cfg, max_seq=max_seq), layers, emb, kv8=True)
    rm = RefModelMixed(cfg, layers, emb, 16)

    def attend(q, K, V, h, kv, hd, pos, split, scale):
        li = next(i for i, k in enumerate(rm.K) if k is K)
        k8, kd, v8, vd = gm.kv8_cache(li, pos + 1)
        return ref.attention(np.asarray(q).reshape(h, hd), ref.q8_values(k8, kd),
                             ref.q8_values(v8, vd), kv, scale)[0].astype(np.float32).reshape(-1)

    monkeypatch.setattr(oracle, "flash_partial", attend)
    monkeypatch.setattr(oracle, "flash_reduce", lambda out, h, hd, split: out)
    nb = cfg["n_embd"] // 32
    wmax = float(np.abs(q8_0_dequant(emb[0][:, : nb * 34].reshape(-1, 34))).max())
    toks = rng.integers(0, cfg["n_vocab"], 12).tolist()
    for pos, tok in enumerate(toks):
        gm.forward(tok, pos)
        got, want = gm.logits().astype(np.float64), rm.step(tok, pos)[0].astype(np.float64)
        _, d8 = oracle.quantize_q8(rm.head_x)
        tol = 2e-3 * np.sqrt(np.mean(want**2)) + 4 * float(d8.max()) * wmax
        assert np.abs(got - want).max() <= tol, pos
        k8, kd, v8, vd = (a[pos:] for a in gm.kv8_cache(0, pos + 1))
        for q, d, bits in ((k8, kd, rm.K[0][pos]), (v8, vd, rm.V[0][pos])):
            r = bits.view(np.float16).astype(np.float64)
            step = np.repeat(d.astype(np.float64), 32, axis=1)[0]
            near = 2.0**-11 * np.abs(r) + 2.1e-4 * np.sqrt(np.mean(r * r))
            assert (np.abs(ref.q8_values(q, d)[0] - r) <= (0.5 + 2.0**-15) * step + near).all(), pos
    last = gm.logits()
    for graph in (False, True, True):
        gm.generate(toks, 1, use_graph=graph)
        assert np.array_equal(gm.logits(), last)
    u = np.linspace(0.05, 0.95, 6).astype(np.float32)
    eager = gm.generate_sampled(toks[:3], u, temperature=0.8, top_k=9, use_graph=False)
    assert np.array_equal(gm.generate_sampled(toks[:3], u, temperature=0.8, top_k=9), eager)
    gm.close()
