"""Sampled continuations of the decode runtime: every token is the one that the
64-bit definition draws from the step's logits."""
import numpy as np
import pytest

import _op_ref as ref
from taraference_amd import capi
from test_gpu_model import TINY, build

pytestmark = pytest.mark.gpu

HOW = [dict(temperature=0.9), dict(temperature=1.3, top_k=20),
       dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.02), dict(temperature=1.0, top_p=0.8)]


def pick(logits, how, u):
    return ref.sample(logits, how["temperature"], how.get("top_k", 0), np.float32(how.get("top_p", 1)),
                      np.float32(how.get("min_p", 0)), u)


@pytest.mark.parametrize("path,kv8", [(0, False), (3, False), (4, False), (0, True)])
def test_generate_sampled(gpu, path, kv8):
    cfg = TINY[1]
    gm, _ = build(cfg, 17, 64)
    if kv8:
        gm.use_kv8()
    gm.set_path(path)
    rng = np.random.default_rng(path)
    prompt, u = list(range(3, 15)), rng.random(18).astype(np.float32)
    for how in HOW:
        eager = gm.generate_sampled(prompt, u, use_graph=False, **how)
        for _ in range(2):
            assert np.array_equal(gm.generate_sampled(prompt, u, use_graph=True, **how), eager)
        toks = list(prompt)
        for pos in range(len(prompt) + len(u) - 1):
            gm.forward(toks[pos], pos)
            if pos >= len(prompt) - 1:
                want = pick(gm.logits(), how, u[pos - len(prompt) + 1])
                assert gm.sample_logits(float(u[pos - len(prompt) + 1]), **how) == want
                toks.append(want)
        assert toks[len(prompt):] == eager.tolist(), how
    # greedy generation still is what it was, sampling at temperature 0 the same
    greedy = gm.generate(prompt, len(u))
    assert np.array_equal(gm.generate_sampled(prompt, u, temperature=0.0), greedy)
    gm.close()


def test_sample_after_prefill(gpu):
    cfg = TINY[0]
    gm, _ = build(cfg, 3, 96)
    prompt = list(range(40))
    how = HOW[2]
    got = gm.sample(prompt, 10, seed=5, **how)
    assert np.array_equal(got, gm.sample(prompt, 10, seed=5, use_graph=False, **how))
    u = np.random.default_rng(5).random(10, dtype=np.float32)
    gm.prefill(prompt)
    assert got[0] == pick(gm.logits(), how, u[0])
    assert np.array_equal(gm.generate_sampled([int(got[0])], u[1:], pos0=40, **how), got[1:])
    assert gm.sample(prompt, 0).size == 0 and gm.sample(prompt, 1, seed=5, **how)[0] == got[0]
    gm.close()


def test_refusals(gpu):
    cfg = TINY[0]
    gm, _ = build(cfg, 3, 32)
    for call in (lambda: gm.generate_sampled([1], np.zeros(0)),
                 lambda: gm.generate_sampled([1], np.zeros(33)),
                 lambda: gm.generate_sampled([cfg["n_vocab"]], np.zeros(2)),
                 lambda: gm.generate_sampled([1, 2], np.zeros(4), pos0=28)):
        with pytest.raises(capi.HipError):
            call()
    import ctypes as C
    assert gm.lib.tf_model_sample(gm.h, None, 0.5, C.byref(C.c_int()), None) == 1
    gm.close()


def test_ranges_past_32_bits(gpu):
    """Positions and counts whose sum passes 2^31 are outside of the cache too."""
    import ctypes as C
    cfg = TINY[0]
    gm, _ = build(cfg, 3, 32)
    lib, h, last = gm.lib, gm.h, 2**31 - 1
    from taraference_amd.model import TfSampling
    how, out, u = TfSampling(1.0, 0, 1.0, 0.0), (C.c_int * 4)(), (C.c_float * 4)()
    one = (C.c_int * 1)(5)
    for pos0, n_gen in ((last, 1), (last, 2), (1, last), (last, last), (32, 1), (0, 33)):
        assert lib.tf_model_generate_sampled(h, one, 1, pos0, n_gen, C.byref(how), u, out, 0, None) == 1
        assert lib.tf_model_generate(h, one, 1, pos0, n_gen, out, 0, None) == 1
    for pos0 in (last, 32):
        with pytest.raises(capi.HipError):
            gm.prefill([1, 2], pos0)
    gm.close()
