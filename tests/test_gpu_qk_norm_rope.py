"""Per-head norms with RoPE in one pass, to f32 rows, the f16 and the 8-bit cache."""
import numpy as np
import pytest

import _op_ref as ref
import oracle
from _gpu import P, S, call, dev, empty, host

pytestmark = pytest.mark.gpu

EPS, THETA = 1e-6, 1e6


def tolerance(size):
    """Of a rotated value: the norm's factor rounds at most 11 times (a sum of
    squares in a tree, a square root, a quotient, two products), the rotation 3,
    sine and cosine 2, and the angle's fraction of a turn (at most 1/2, so within
    2^-26) is worth 2 pi 2^-26 < 2 * 2^-24: 18 halves of 2^-23, taken as 24."""
    return 24 * 2.0**-24 * size + 1e-30


def inputs(rng, t, h, kv, hd, spare=0):
    row = (h + 2 * kv) * hd + spare
    x = (2 * rng.standard_normal((t, row))).astype(np.float32)
    wq = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    wk = (1 + 0.3 * rng.standard_normal(hd)).astype(np.float32)
    return x, row, wq, wk


def parts(x, h, kv, hd):
    t = x.shape[0]
    return (x[:, :h * hd].reshape(t, h, hd), x[:, h * hd:(h + kv) * hd].reshape(t, kv, hd),
            x[:, (h + kv) * hd:(h + 2 * kv) * hd])


SHAPES = [  # heads, kv heads, head_dim, tokens, first position
    (16, 2, 128, 1, 0), (28, 4, 128, 1, 32767), (14, 2, 64, 1, 5), (16, 4, 256, 1, 1000001),
    (14, 2, 64, 37, 0), (16, 2, 128, 130, 130000), (28, 4, 128, 65, 777), (3, 3, 256, 9, 8000),
    (5, 1, 128, 700, 11), (1, 1, 64, 1, 123456789),
    (6, 2, 96, 5, 40), (4, 2, 80, 3, 9), (2, 1, 2, 4, 3), (3, 1, 250, 2, 100), (2, 2, 32, 33, 1),
]


@pytest.mark.parametrize("h,kv,hd,t,pos", SHAPES)
@pytest.mark.parametrize("norms", ["both", "none", "k"])
def test_rows(gpu, h, kv, hd, t, pos, norms):
    rng = np.random.default_rng(hd + t)
    x, row, wq, wk = inputs(rng, t, h, kv, hd, spare=4 if t % 2 else 3)
    wq, wk = wq if norms == "both" else None, wk if norms != "none" else None
    d = dev(x)
    qo, ko = empty(t * h * hd), empty(t * kv * hd)
    call("tf_qk_norm_rope", P(d), row, P(d) + 4 * h * hd, row, None if wq is None else P(dev(wq)),
         None if wk is None else P(dev(wk)), EPS, P(qo), P(ko), h, kv, hd, t, pos, None, THETA, S())
    q, k, _ = parts(x, h, kv, hd)
    at = pos + np.arange(t)
    for got, src, w in ((qo, q, wq), (ko, k, wk)):
        want, size = ref.norm_rope(src, w, EPS, at, THETA)
        err = np.abs(host(got).reshape(want.shape).astype(np.float64) - want)
        assert (err <= tolerance(size)).all(), (err / tolerance(size)).max()


def test_rows_in_place_and_device_position(gpu):
    h, kv, hd, t = 16, 2, 128, 3
    rng = np.random.default_rng(1)
    q, k = (rng.standard_normal((t, n * hd)).astype(np.float32) for n in (h, kv))
    dq, dk, pos = dev(q), dev(k), dev(np.array([70001], np.int32))
    call("tf_qk_norm_rope", P(dq), h * hd, P(dk), kv * hd, None, None, EPS, P(dq), P(dk), h, kv, hd,
         t, -5, P(pos), THETA, S())
    for got, src, n in ((dq, q, h), (dk, k, kv)):
        want, size = ref.norm_rope(src.reshape(t, n, hd), None, EPS, 70001 + np.arange(t), THETA)
        assert (np.abs(host(got).reshape(want.shape) - want) <= tolerance(size)).all()


@pytest.mark.parametrize("h,kv,hd,t,pos", [s for s in SHAPES if s[4] < 10000])
def test_append_f16(gpu, h, kv, hd, t, pos):
    rng = np.random.default_rng(hd + t)
    x, row, wq, wk = inputs(rng, t, h, kv, hd)
    d, n = dev(x), kv * hd
    kc, vc = (dev(np.full((pos + t + 2, n), 0x1234, np.uint16)) for _ in range(2))
    qo = empty(t * h * hd)
    call("tf_qk_norm_rope_append", P(d), row, P(d) + 4 * h * hd, row, P(d) + 4 * (h + kv) * hd, row,
         P(dev(wq)), P(dev(wk)), EPS, P(qo), P(kc), P(vc), h, kv, hd, t, pos, None, THETA, S())
    q, k, v = parts(x, h, kv, hd)
    at = pos + np.arange(t)
    want, size = ref.norm_rope(q, wq, EPS, at, THETA)
    assert (np.abs(host(qo).reshape(want.shape) - want) <= tolerance(size)).all()
    want, size = ref.norm_rope(k, wk, EPS, at, THETA)
    got = host(kc)
    err = np.abs(got[pos:pos + t].view(np.float16).astype(np.float64) - want.reshape(t, n))
    tol = tolerance(size).reshape(t, n)  # half a step of f16, or of its subnormals
    assert (err <= tol + 2.0**-11 * (np.abs(want.reshape(t, n)) + tol) + 2.0**-25).all()
    gv = host(vc)
    assert np.array_equal(gv[pos:pos + t], oracle.f32_to_f16(v.reshape(-1)).reshape(t, n))
    for c in (got, gv):  # rows before and behind stay as they were
        assert (c[:pos] == 0x1234).all() and (c[pos + t:] == 0x1234).all()


@pytest.mark.parametrize("h,kv,hd,t,pos", [s for s in SHAPES if s[4] < 10000 and s[2] % 32 == 0])
def test_append_kv8(gpu, h, kv, hd, t, pos):
    rng = np.random.default_rng(hd + t)
    x, row, wq, wk = inputs(rng, t, h, kv, hd)
    d, n = dev(x), kv * hd
    k8, v8 = (dev(np.full((pos + t + 2, n), 77, np.int8)) for _ in range(2))
    kd, vd = (dev(np.full((pos + t + 2, n // 32), -3, np.float32)) for _ in range(2))
    qo = empty(t * h * hd)
    call("tf_qk_norm_rope_append_kv8", P(d), row, P(d) + 4 * h * hd, row, P(d) + 4 * (h + kv) * hd,
         row, P(dev(wq)), P(dev(wk)), EPS, P(qo), P(k8), P(kd), P(v8), P(vd), h, kv, hd, t, pos,
         None, THETA, S())
    q, k, v = parts(x, h, kv, hd)
    at = pos + np.arange(t)
    want, size = ref.norm_rope(q, wq, EPS, at, THETA)
    assert (np.abs(host(qo).reshape(want.shape) - want) <= tolerance(size)).all()
    want, size = ref.norm_rope(k, wk, EPS, at, THETA)
    want, tol = want.reshape(t, n), tolerance(size).reshape(t, n)
    k8, kd, v8, vd = host(k8), host(kd), host(v8), host(vd)
    g, gd = k8[pos:pos + t], kd[pos:pos + t]
    # the scale is the largest of 32 over 127, each within its tolerance, and
    # rounds twice; a value is then off by half a step and its own tolerance
    groups = np.abs(want).reshape(t, -1, 32)
    top, ttol = groups.max(-1), tol.reshape(t, -1, 32).max(-1)
    assert (np.abs(gd - top / 127) <= ttol / 127 + 2 * 2.0**-24 * top / 127).all()
    step = np.repeat(gd.astype(np.float64), 32, axis=1)
    assert (np.abs(ref.q8_values(g, gd) - want) <= step * (0.5 + 127 * 2.0**-23) + tol).all()
    q8, d8 = ref.q8_rows(v)
    assert np.array_equal(v8[pos:pos + t], q8) and np.array_equal(vd[pos:pos + t], d8)
    for c, mark in ((k8, 77), (v8, 77), (kd, -3), (vd, -3)):
        assert (c[:pos] == mark).all() and (c[pos + t:] == mark).all()


def test_angle_is_exact_far_out(gpu):
    """A unit vector at position 2^24 - 1 with theta 1e4: the rotated pair is
    (cos, sin) of the 64-bit angle; the f32 angle would be off by 0.5 rad."""
    hd, pos = 128, 2**24 - 1
    x = np.zeros((1, hd), np.float32)
    x[0, :hd // 2] = 1
    d, qo, ko = dev(x), empty(hd), empty(hd)
    call("tf_qk_norm_rope", P(d), hd, P(d), hd, None, None, EPS, P(qo), P(ko), 1, 1, hd, 1, pos,
         None, 1e4, S())
    want, size = ref.norm_rope(x.reshape(1, 1, hd), None, EPS, [pos], 1e4)
    assert (np.abs(host(qo) - want.ravel()) <= tolerance(size.ravel())).all()
    assert np.array_equal(host(qo), host(ko))


@pytest.mark.parametrize("h,kv,hd", [(14, 2, 64), (6, 1, 128), (3, 2, 256)])
@pytest.mark.parametrize("t", [127, 128, 1023, 1025, 1026, 1027])
def test_many_tokens_and_in_place(gpu, h, kv, hd, t):
    """Token counts around those at which a workgroup takes all heads, or four tokens."""
    rng = np.random.default_rng(t)
    q, k = (rng.standard_normal((t, n * hd)).astype(np.float32) for n in (h, kv))
    wq, wk = (rng.standard_normal(hd).astype(np.float32) for _ in range(2))
    dq, dk = (dev(np.concatenate([a, np.full((2, a.shape[1]), 7, np.float32)])) for a in (q, k))
    call("tf_qk_norm_rope", P(dq), h * hd, P(dk), kv * hd, P(dev(wq)), P(dev(wk)), EPS, P(dq), P(dk),
         h, kv, hd, t, 3, None, THETA, S())
    for got, src, n, w in ((dq, q, h, wq), (dk, k, kv, wk)):
        want, size = ref.norm_rope(src.reshape(t, n, hd), w, EPS, 3 + np.arange(t), THETA)
        assert (np.abs(host(got)[:t].reshape(want.shape) - want) <= tolerance(size)).all()
        assert (host(got)[t:] == 7).all()


@pytest.mark.parametrize("t", [3, 1030])
def test_caches_off_alignment(gpu, t):
    """f16 and 8-bit rows that start one element past an aligned address equal the others."""
    h, kv, hd = 4, 2, 128
    n = kv * hd
    x, row, wq, wk = inputs(np.random.default_rng(t), t, h, kv, hd)
    d, dwq, dwk, qo = dev(x), dev(wq), dev(wk), empty(t * h * hd)
    head = (P(d), row, P(d) + 4 * h * hd, row, P(d) + 4 * (h + kv) * hd, row, P(dwq), P(dwk), EPS,
            P(qo))
    tail = (h, kv, hd, t, 0, None, THETA, S())
    v = x[:, (h + kv) * hd:(h + 2 * kv) * hd]
    q8, d8 = ref.q8_rows(v)
    for off in (0, 1):
        kc, vc = (dev(np.zeros(t * n + 1, np.uint16)) for _ in range(2))
        call("tf_qk_norm_rope_append", *head, P(kc) + 2 * off, P(vc) + 2 * off, *tail)
        k8, v8 = (dev(np.zeros(t * n + 1, np.int8)) for _ in range(2))
        kd, vd = (dev(np.zeros(t * n // 32, np.float32)) for _ in range(2))
        call("tf_qk_norm_rope_append_kv8", *head, P(k8) + off, P(kd), P(v8) + off, P(vd), *tail)
        end = off + t * n
        assert np.array_equal(host(vc)[off:end], oracle.f32_to_f16(np.ascontiguousarray(v).ravel()))
        assert np.array_equal(host(v8)[off:end], q8.ravel()) and np.array_equal(host(vd), d8.ravel())
        want, size = ref.norm_rope(parts(x, h, kv, hd)[1], wk, EPS, np.arange(t), THETA)
        want, tol = want.reshape(t, n), tolerance(size).reshape(t, n)
        got = host(kc)[off:end].view(np.float16).astype(np.float64).reshape(t, n)
        assert (np.abs(got - want) <= tol + 2.0**-11 * (np.abs(want) + tol) + 2.0**-25).all()
        gd = host(kd).reshape(t, -1)
        step = np.repeat(gd.astype(np.float64), 32, axis=1)
        val = ref.q8_values(host(k8)[off:end].reshape(t, n), gd)
        assert (np.abs(val - want) <= step * (0.5 + 127 * 2.0**-23) + tol).all()
