"""What the per-head norm + RoPE, 8-bit cache and sampling entry points refuse,
before they touch the device."""
import ctypes as C

import pytest

INVALID = 1  # hipErrorInvalidValue
A = 4096     # an aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    from taraference_amd import capi
    return capi.load()


ROPE = dict(q=A, q_stride=2048, k=A * 2, k_stride=256, q_norm=A, k_norm=A, eps=1e-6, q_out=A * 3,
            k_out=A * 4, n_head=16, n_kv=2, head_dim=128, n_tok=4, pos0=0, pos0_dev=None, theta=1e6)


@pytest.mark.parametrize("bad", [
    {"q": None}, {"k": None}, {"q_out": None}, {"k_out": None}, {"q_stride": 2047},
    {"k_stride": 255}, {"n_head": 0}, {"n_kv": 0}, {"head_dim": 0}, {"head_dim": 127},
    {"head_dim": 258, "q_stride": 1 << 20, "k_stride": 1 << 20}, {"n_tok": 0}, {"n_tok": -1},
    {"pos0": -1}, {"pos0": 2**31 - 2}, {"theta": 0.0}, {"theta": -1.0}, {"theta": float("nan")},
    {"theta": float("inf")}, {"eps": -1.0}, {"eps": float("nan")},
    {"q": A * 3, "q_stride": 2052}, {"k": A * 4, "k_stride": 260}, {"q_stride": -2048},
])
def test_rope_rows(lib, bad):
    a = {**ROPE, **bad}
    assert lib.tf_qk_norm_rope(*a.values(), None) == INVALID


def append_args(kv8, bad):
    a = dict(q=A, q_stride=2048, k=A, k_stride=256, v=A, v_stride=256, q_norm=None, k_norm=None,
             eps=1e-6, q_out=A * 3, kc=A, vc=A, n_head=16, n_kv=2, head_dim=128, n_tok=4, pos0=0,
             pos0_dev=None, theta=1e6)
    if kv8:
        a = {**{n: a[n] for n in list(a)[:10]}, "kc": A, "kd": A, "vc": A, "vd": A,
             **{n: a[n] for n in list(a)[12:]}}
    assert not set(bad) - set(a)
    return [*{**a, **bad}.values(), None]


@pytest.mark.parametrize("bad", [{"q": None}, {"k": None}, {"v": None}, {"v_stride": 255},
                                 {"kc": None}, {"vc": None}, {"q_out": None}, {"head_dim": 129},
                                 {"n_tok": 0}, {"pos0": -2}, {"theta": 0.0}])
def test_rope_append(lib, bad):
    assert lib.tf_qk_norm_rope_append(*append_args(False, bad)) == INVALID
    assert lib.tf_qk_norm_rope_append_kv8(*append_args(True, bad)) == INVALID


@pytest.mark.parametrize("bad", [{"kd": None}, {"vd": None}, {"head_dim": 80}])
def test_rope_append_kv8(lib, bad):
    assert lib.tf_qk_norm_rope_append_kv8(*append_args(True, bad)) == INVALID


WRITE = dict(k=A, v=A, src_type=0, src_stride=256, k8=A, kd=A, v8=A, vd=A, n=256, pos0=0,
             pos0_dev=None, n_tok=1)


@pytest.mark.parametrize("bad", [{"k": None}, {"v": None}, {"k8": None}, {"kd": None}, {"v8": None},
                                 {"vd": None}, {"src_type": 2}, {"src_type": -1},
                                 {"src_stride": 255}, {"n": 0}, {"n": 48}, {"n": -32}, {"pos0": -1},
                                 {"n_tok": 0}, {"pos0": 2**31 - 1},
                                 {"n_tok": 2**30, "n": 1 << 12, "src_stride": 1 << 12}])
def test_kv8_write(lib, bad):
    assert lib.tf_kv8_write(*{**WRITE, **bad}.values(), None) == INVALID


READ = dict(k8=A, kd=A, v8=A, vd=A, k=A, v=A, dst_type=1, n=256, row0=0, n_rows=1)


@pytest.mark.parametrize("bad", [{"k": None}, {"v": None}, {"k8": None}, {"kd": None}, {"v8": None},
                                 {"vd": None}, {"dst_type": 2}, {"n": 0}, {"n": 33}, {"row0": -1},
                                 {"n_rows": 0}, {"n_rows": 2**31 - 1, "n": 1 << 20}])
def test_kv8_read(lib, bad):
    assert lib.tf_kv8_read(*{**READ, **bad}.values(), None) == INVALID


FLASH = dict(q=A, k8=A, kd=A, v8=A, vd=A, partial=A, out=A, q8=None, d8=None, n_head=16, n_kv=2,
             head_dim=128, pos0=5, pos0_dev=None, n_split=8, scale=0.1)


@pytest.mark.parametrize("bad", [{"q": None}, {"k8": None}, {"kd": None}, {"v8": None}, {"vd": None},
                                 {"partial": None}, {"out": None}, {"q8": A}, {"d8": A},
                                 {"n_head": 0}, {"n_kv": 0}, {"n_head": 15}, {"n_kv": -2},
                                 {"n_head": 34}, {"head_dim": 96}, {"head_dim": 0}, {"pos0": -1},
                                 {"n_split": 0}, {"n_split": 1025}])
def test_flash_kv8(lib, bad):
    assert lib.tf_flash_decode_kv8(*{**FLASH, **bad}.values(), None) == INVALID


@pytest.mark.parametrize("bad", [{"q": A + 4}, {"k8": A + 8}, {"v8": A + 1}, {"kd": A + 4},
                                 {"vd": A + 8}, {"kd": A + 2, "head_dim": 64},
                                 {"v8": A + 8, "head_dim": 64}, {"pos0": 2**31 - 1024}])
def test_flash_kv8_alignment(lib, bad):
    assert lib.tf_flash_decode_kv8(*{**FLASH, **bad}.values(), None) == INVALID


SAMPLE = dict(logits=A, n_rows=2, n_vocab=1000, row_stride=1000, temperature=None, top_k=None,
              top_p=None, min_p=None, u=A, out=A, ws=A, ws_bytes=1 << 30)


@pytest.mark.parametrize("bad", [{"logits": None}, {"u": None}, {"out": None}, {"ws": None},
                                 {"n_rows": 0}, {"n_vocab": 0}, {"n_vocab": 1 << 19},
                                 {"row_stride": 999}, {"ws": A + 8}, {"ws_bytes": 0},
                                 {"ws_bytes": -1}])
def test_sample(lib, bad):
    assert lib.tf_sample(*{**SAMPLE, **bad}.values(), None) == INVALID


def test_sample_ws_bytes(lib):
    f = lib.tf_sample_ws_bytes
    assert f.restype is C.c_longlong
    for bad in ((0, 10), (1, 0), (-1, 10), (1, -5), (1, 1 << 19)):
        assert f(*bad) == -1
    assert 0 < f(1, 10) <= f(1, 151936) <= f(64, 151936)
    need = f(3, 1000)
    assert lib.tf_sample(*{**SAMPLE, "n_rows": 3, "ws_bytes": need - 1}.values(), None) == INVALID


def test_oracles_agree_with_themselves():
    """The 64-bit forms the GPU tests use, on cases that can be told by hand."""
    import numpy as np

    import _op_ref as ref
    x = np.array([1.0, 3.0, 2.0, 3.0, -np.inf], np.float32)
    e = np.exp([-2.0, 0, -1, 0])
    assert ref.sample(x, 0.0, 0, 1, 0, 0.5) == 1                 # greedy, lowest index
    assert ref.sample(x, 1.0, 1, 1, 0, 0.99) == 1                # one of the tied two
    assert ref.sample(x, 1.0, 2, 1, 0, 0.6) == 3
    assert ref.sample(x, 1.0, 0, 1, 0, np.float32(e[0] / e.sum() * 0.99)) == 0
    assert ref.sample(x, 1.0, 0, 1, 0.9, 0.0) == 1               # the two largest
    assert ref.sample(x, 1.0, 0, 0.5, 0, 0.9) == 3               # 2 of e.sum() is over a half
    assert ref.sample(x, 1.0, 0, 0.0, 0, 0.9) == 1
    assert ref.sample(np.full(3, -np.inf, np.float32), 1, 0, 1, 0, 0.5) == 0
    out, tol = ref.attention(np.ones((2, 32)), np.zeros((4, 32)), np.arange(128.).reshape(4, 32), 1, 1)
    assert np.allclose(out, np.arange(32) + 48) and (tol > 0).all()
    y, _ = ref.norm_rope(np.full((1, 1, 2), 3.0), np.ones(2), 0.0, [0], 10.0)
    assert np.allclose(y, 1.0)
    q, d = ref.q8_rows(np.arange(-16, 16, dtype=np.float32)[None])
    assert q[0, 0] == -127 and d.shape == (1, 1)


@pytest.mark.parametrize("shape", [dict(n_embd=512, n_head=16, n_kv=16, head_dim=32),
                                   dict(n_embd=2176, n_head=34, n_kv=2, head_dim=64)])
def test_models_without_an_8_bit_cache(lib, shape):
    """Heads that its attention does not take: refused before anything is allocated."""
    from taraference_amd import model as M
    M._bind(lib)
    cfg = M.TfModelConfig(n_layer=1, n_ff=512, n_vocab=100, max_seq=8, rope_theta=1e4, rms_eps=1e-6,
                          **shape)
    out, mat = C.c_void_p(), M.TfMat()
    args = (C.byref(cfg), (M.TfLayer * 1)(), C.byref(mat), C.byref(mat), A, C.byref(out))
    assert lib.tf_model_create_kv8(*args) == 801  # hipErrorNotSupported
    assert lib.tf_model_create_kv8(None, *args[1:]) == INVALID
    assert not out.value and lib.tf_model_use_kv8(None) == INVALID


@pytest.mark.parametrize("n_vocab,most", [(10, 4194303), (8192, 4194303), (8193, 2097151),
                                          (151936, 220752), (524287, 65535)])
def test_sample_rows(lib, n_vocab, most):
    """Rows past a launch's 2^32 threads have no workspace, as tf_sample refuses them."""
    f = lib.tf_sample_ws_bytes
    assert f(most, n_vocab) == most * f(1, n_vocab) > 0
    assert f(most + 1, n_vocab) == -1 and f(2**31 - 1, n_vocab) == -1
    big = {**SAMPLE, "n_rows": most + 1, "n_vocab": n_vocab, "row_stride": n_vocab,
           "ws_bytes": 2**62}
    assert lib.tf_sample(*big.values(), None) == INVALID
