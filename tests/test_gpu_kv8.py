"""The 8-bit K/V cache: rows written and read back, one token's attention over it."""
import numpy as np
import pytest
import torch

import _op_ref as ref
import oracle
from _gpu import KEEP, P, S, call, dev, empty, host

pytestmark = pytest.mark.gpu


def rows(rng, t, n):
    x = rng.standard_normal((t, n)).astype(np.float32)
    x *= np.float32(10.0) ** rng.integers(-6, 5, (t, n // 32)).astype(np.float32).repeat(32, 1)
    x[:, :32] = 0  # a group without any value
    if t > 1:
        x[1, 32:64] = 1e-42 * np.arange(32)  # subnormal
    return x


@pytest.mark.parametrize("src", ["f32", "f16"])
@pytest.mark.parametrize("n,t,pos,spare", [(128, 1, 0, 0), (256, 1, 17, 0), (512, 300, 1000, 64),
                                           (64, 5, 3, 5), (1024, 33, 0, 0), (2048, 7, 9, 32),
                                           (32, 70001, 2, 0), (96, 11, 1, 1)])
def test_write_and_read(gpu, n, t, pos, spare, src):
    rng = np.random.default_rng(n + t)
    # f16 rows lie in f16's range
    k, v = (rows(rng, t, n + 32)[:, :n] if src == "f32" else
            rng.standard_normal((t, n)).astype(np.float16).astype(np.float32) for _ in range(2))
    stride = n + spare
    ty = np.float32 if src == "f32" else np.float16
    dk, dv = (dev(np.concatenate([a.astype(ty), np.full((t, spare), 9e9 if src == "f32" else 6e4,
                                                        ty)], 1)) for a in (k, v))
    k8, v8 = (dev(np.full((pos + t + 1, n), 77, np.int8)) for _ in range(2))
    kd, vd = (dev(np.full((pos + t + 1, n // 32), -3, np.float32)) for _ in range(2))
    call("tf_kv8_write", P(dk), P(dv), gpu.KV_F32 if src == "f32" else gpu.KV_F16, stride, P(k8),
         P(kd), P(v8), P(vd), n, pos, None, t, S())
    for x, c8, cd in ((k, k8, kd), (v, v8, vd)):
        q, d = oracle.quantize_q8(np.ascontiguousarray(x).reshape(-1))
        g8, gd = host(c8), host(cd)
        assert np.array_equal(g8[pos:pos + t].ravel(), q)
        assert np.array_equal(gd[pos:pos + t].ravel(), d)
        assert (g8[:pos] == 77).all() and (g8[pos + t:] == 77).all()
        assert (gd[:pos] == -3).all() and (gd[pos + t:] == -3).all()
        f32 = (g8[pos:pos + t].reshape(-1, 32).astype(np.float32) *
               gd[pos:pos + t].reshape(-1, 1)).reshape(t, n)
        for dst in ("f32", "f16"):
            ty = torch.float32 if dst == "f32" else torch.float16
            a, b = empty((t + 1, n), ty).fill_(5), empty((t + 1, n), ty).fill_(5)
            call("tf_kv8_read", P(k8), P(kd), P(v8), P(vd), P(a), P(b),
                 gpu.KV_F32 if dst == "f32" else gpu.KV_F16, n, pos, t, S())
            got = host(a if c8 is k8 else b)
            with np.errstate(over="ignore"):
                assert np.array_equal(got[:t], f32.astype(got.dtype))
            assert (got[t] == 5).all()


def test_write_at_a_device_position(gpu):
    n, t = 128, 3
    x = np.random.default_rng(3).standard_normal((t, n)).astype(np.float32)
    d, pos = dev(x), dev(np.array([4], np.int32))
    k8, v8 = (dev(np.zeros((9, n), np.int8)) for _ in range(2))
    kd, vd = (dev(np.zeros((9, n // 32), np.float32)) for _ in range(2))
    call("tf_kv8_write", P(d), P(d), gpu.KV_F32, n, P(k8), P(kd), P(v8), P(vd), n, 0, P(pos), t, S())
    q, s = ref.q8_rows(x)
    for c8, cd in ((k8, kd), (v8, vd)):
        assert np.array_equal(host(c8)[4:7], q) and np.array_equal(host(cd)[4:7], s)
        assert not host(c8)[:4].any() and not host(c8)[7:].any()


def cache(rng, seq, n, spread=1.0):
    x = (spread * rng.standard_normal((seq, n))).astype(np.float32)
    x[:, ::17] *= 5  # a few channels larger than the rest
    return ref.q8_rows(x)


def attend(q, k8, kd, v8, vd, n_kv, pos, n_split, scale, pos_dev=None, want_q8=False):
    h, hd = q.shape
    part, out = empty(h * n_split * (2 + hd)).fill_(float("nan")), empty(h * hd)
    q8, d8 = (empty(h * hd, torch.int8), empty(h * hd // 32)) if want_q8 else (None, None)
    call("tf_flash_decode_kv8", P(dev(q)), P(k8), P(kd), P(v8), P(vd), P(part), P(out), P(q8),
         P(d8), h, n_kv, hd, pos, P(pos_dev), n_split, scale, S())
    return (host(out).reshape(h, hd),) + ((host(q8), host(d8)) if want_q8 else ())


def check(got, q, k, v, n_kv, scale):
    want, tol = ref.attention(q, k, v, n_kv, scale)
    err = np.abs(got - want)
    assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()


GROUPS = [(16, 2, 128), (28, 4, 128), (14, 2, 64), (16, 4, 256), (5, 5, 64), (16, 1, 128),
          (3, 1, 256), (16, 1, 64), (15, 1, 256), (8, 8, 128)]


@pytest.mark.parametrize("h,kv,hd", GROUPS)
@pytest.mark.parametrize("seq,n_split", [(1, 1), (1, 8), (2, 1), (31, 1), (33, 2), (130, 8), (257, 1),
                                         (1000, 3), (1025, 16), (4099, 64)])
def test_attention(gpu, h, kv, hd, seq, n_split):
    rng = np.random.default_rng(seq + hd)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k8, kd = cache(rng, seq, kv * hd)
    v8, vd = cache(rng, seq, kv * hd)
    scale = 1 / np.sqrt(hd)
    # rows behind the position hold what must not be read into anything
    def behind(a, fill):
        return dev(np.concatenate([a, np.full((40, a.shape[1]), fill, a.dtype)]))
    got = attend(q, behind(k8, 127), behind(kd, np.nan), behind(v8, -127), behind(vd, np.inf), kv,
                 seq - 1, n_split, scale)[0]
    check(got, q, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, scale)


@pytest.mark.parametrize("h,kv,hd", [(16, 2, 128), (14, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("case", ["sink", "tiny", "huge", "flat", "zero_q", "mixed_scales"])
def test_attention_values(gpu, h, kv, hd, case):
    rng = np.random.default_rng(hd)
    seq, n = 700, kv * hd
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k = rng.standard_normal((seq, n)).astype(np.float32)
    v = rng.standard_normal((seq, n)).astype(np.float32)
    scale = 1 / np.sqrt(hd)
    if case == "sink":  # one key far above the rest, late and early
        k[[0, 650]] *= 12
    elif case == "tiny":
        v *= 1e-20
        k *= 1e-12
    elif case == "huge":
        v *= 1e25
        k *= 1e9
        scale = scale * 1e-9
    elif case == "flat":
        k[:] = 0
    elif case == "zero_q":
        q[:] = 0
    else:  # scales of neighbouring groups and rows 10^12 apart
        v *= (10.0 ** rng.integers(-6, 7, (seq, n // 32))).repeat(32, 1).astype(np.float32)
        v[::3] = 0
    k8, kd = ref.q8_rows(k)
    v8, vd = ref.q8_rows(v)
    got = attend(q, dev(k8), dev(kd), dev(v8), dev(vd), kv, seq - 1, 4, scale)[0]
    check(got, q, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, scale)


def test_attention_q8_device_position_and_empty(gpu):
    h, kv, hd, seq = 28, 4, 128, 600
    rng = np.random.default_rng(5)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k8, kd = cache(rng, seq, kv * hd)
    v8, vd = cache(rng, seq, kv * hd)
    c = [dev(a) for a in (k8, kd, v8, vd)]
    scale = 1 / np.sqrt(hd)
    k, v = ref.q8_values(k8, kd), ref.q8_values(v8, vd)
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    KEEP.append(pos)
    for n_split in (1, 8):
        for at in (599, 0, 64, -1):
            pos.fill_(at)
            out, q8, d8 = attend(q, *c, kv, 0, n_split, scale, pos_dev=pos, want_q8=True)
            check(out, q, k[:at + 1], v[:at + 1], kv, scale)
            wq, wd = oracle.quantize_q8(out.reshape(-1))
            assert np.array_equal(q8, wq) and np.array_equal(d8, wd)


def test_attention_long(gpu):
    """A cache whose element offsets pass 2^31: only its last rows and first rows
    hold anything, and the query finds them."""
    h, kv, hd = 8, 8, 256
    seq, n = 1_100_000, 8 * 256
    k8 = torch.zeros(seq, n, dtype=torch.int8, device="cuda")
    v8 = torch.zeros(seq, n, dtype=torch.int8, device="cuda")
    kd = torch.ones(seq, n // 32, device="cuda")
    vd = torch.ones(seq, n // 32, device="cuda")
    KEEP.extend([k8, v8, kd, vd])
    rng = np.random.default_rng(2)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    scale = 1 / np.sqrt(hd)
    for r in (3, seq - 2):
        k8[r] = torch.from_numpy(np.clip(np.rint(q.reshape(-1) * 20), -127, 127).astype(np.int8))
        v8[r] = (r % 100) + 1
    n_split = gpu.load().tf_flash_decode_kv8_n_split(kv, hd, seq)
    got = attend(q, k8, kd, v8, vd, kv, seq - 1, n_split, scale)[0]
    kk = np.clip(np.rint(q * 20), -127, 127)
    x = (kk * q).sum(1) * scale  # both rows' score; the others score 0
    e = np.exp(-x)
    want = ((3 % 100 + 1) + ((seq - 2) % 100 + 1)) / (2 + (seq - 2) * e)
    assert np.abs(got - want[:, None]).max() <= 2e-4 * want.max()


def test_split_counts(gpu):
    f = gpu.load().tf_flash_decode_kv8_n_split
    for kv in (1, 2, 4, 8, 32, 300):
        for hd in (64, 128, 256):
            for seq in (1, 100, 5000, 131072, 10**7):
                assert 1 <= f(kv, hd, seq) <= 256


@pytest.mark.parametrize("ty", ["f32", "f16"])
@pytest.mark.parametrize("off", ["rows", "cache", "read"])
def test_rows_off_alignment(gpu, ty, off):
    """Sources, caches and destinations at one element past an aligned address."""
    n, t = 96, 37
    np_t, kv_t = (np.float32, gpu.KV_F32) if ty == "f32" else (np.float16, gpu.KV_F16)
    x = np.random.default_rng(5).standard_normal((t, n)).astype(np_t)
    d = dev(np.concatenate([[0], x.ravel()]).astype(np_t)) if off == "rows" else dev(x)
    src = P(d) + (d.element_size() if off == "rows" else 0)
    at = 1 if off == "cache" else 0
    k8, v8 = (dev(np.full(t * n + 2, 77, np.int8)) for _ in range(2))
    kd, vd = (dev(np.zeros(t * n // 32, np.float32)) for _ in range(2))
    call("tf_kv8_write", src, src, kv_t, n, P(k8) + at, P(kd), P(v8) + at, P(vd), n, 0, None, t, S())
    q, s = ref.q8_rows(x.astype(np.float32))
    f32 = (q.reshape(-1, 32).astype(np.float32) * s.reshape(-1, 1)).ravel()
    out = [empty(t * n + 2, torch.float32 if ty == "f32" else torch.float16).fill_(5)
           for _ in range(2)]
    skip = 1 if off == "read" else 0
    call("tf_kv8_read", P(k8) + at, P(kd), P(v8) + at, P(vd), *(P(o) + skip * o.element_size()
         for o in out), kv_t, n, 0, t, S())
    for c8, cd, o in ((k8, kd, out[0]), (v8, vd, out[1])):
        assert np.array_equal(host(c8)[at:at + t * n], q.ravel()) and np.array_equal(host(cd), s.ravel())
        assert (host(c8)[:at] == 77).all() and (host(c8)[at + t * n:] == 77).all()
        assert np.array_equal(host(o)[skip:skip + t * n], f32.astype(np_t))
        assert (host(o)[:skip] == 5).all() and (host(o)[skip + t * n:] == 5).all()


def test_attention_of_scales_at_any_word(gpu):
    """Head_dim 64: the scales' arrays may start at any float."""
    h, kv, hd, seq = 14, 2, 64, 333
    rng = np.random.default_rng(21)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k8, kd = cache(rng, seq, kv * hd)
    v8, vd = cache(rng, seq, kv * hd)
    pad = lambda a: dev(np.concatenate([[9.0], a.ravel()]).astype(np.float32))  # noqa: E731
    dkd, dvd = pad(kd), pad(vd)
    for n_split in (1, 8):
        part, out = empty(h * n_split * (2 + hd)), empty(h * hd)
        call("tf_flash_decode_kv8", P(dev(q)), P(dev(k8)), P(dkd) + 4, P(dev(v8)), P(dvd) + 4,
             P(part), P(out), None, None, h, kv, hd, seq - 1, None, n_split, 0.125, S())
        check(host(out).reshape(h, hd), q, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, 0.125)


@pytest.mark.parametrize("h,kv,hd", [(16, 2, 128), (14, 2, 64), (16, 1, 256), (3, 3, 128)])
@pytest.mark.parametrize("seq,n_split", [(2000, 1), (20000, 1), (20000, 3)])
def test_attention_whose_maximum_keeps_rising(gpu, h, kv, hd, seq, n_split):
    """Scores that grow along the sequence: every tile of a long split renews the maximum.
    (h == kv: one query head beside fifteen columns without one.)"""
    rng = np.random.default_rng(seq + hd)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    scale = 1 / np.sqrt(hd)
    x = 0.2 * rng.standard_normal((seq, kv, hd))
    for j in range(kv):  # along the group's mean query, up to a score of 8
        m = q[j * (h // kv):(j + 1) * (h // kv)].mean(0)
        x[:, j] += np.linspace(0, 8, seq)[:, None] * m / (m @ m) / scale
    k8, kd = ref.q8_rows(x.reshape(seq, -1).astype(np.float32))
    v8, vd = cache(rng, seq, kv * hd)
    got = attend(q, dev(k8), dev(kd), dev(v8), dev(vd), kv, seq - 1, n_split, scale)[0]
    check(got, q, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, scale)


@pytest.mark.parametrize("h,kv,hd", [(16, 2, 128), (14, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 3e38])
def test_a_query_that_is_not_finite_stays_in_its_head(gpu, h, kv, hd, bad):
    rng = np.random.default_rng(hd)
    seq, scale = 500, 1 / np.sqrt(hd)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k8, kd = cache(rng, seq, kv * hd)
    v8, vd = cache(rng, seq, kv * hd)
    at = h // kv - 1
    q[at, 7] = bad
    rest = q.copy()
    rest[at] = 0
    want, tol = ref.attention(rest, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, scale)
    others = np.arange(h) != at
    for n_split in (1, 8):
        got = attend(q, dev(k8), dev(kd), dev(v8), dev(vd), kv, seq - 1, n_split, scale)[0]
        assert (np.abs(got - want)[others] <= tol[others]).all()
        if not np.isfinite(bad):
            assert np.isnan(got[at]).all()


@pytest.mark.parametrize("h,kv,hd", [(16, 2, 128), (14, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("big", [1e6, 1e15, 1e30])
@pytest.mark.parametrize("case", ["unseen", "by_one_head", "seen_before_a_rise"])
def test_attention_of_values_far_apart(gpu, h, kv, hd, big, case):
    """Tokens, alone and by whole tiles of 32, whose values are larger than the others' by
    more than f16 products hold: of no weight; of all the weight in one head and none in the
    others; and of weight until later keys outweigh them."""
    rng = np.random.default_rng(hd)
    seq, n, scale = 900, kv * hd, 1 / np.sqrt(hd)
    q = rng.standard_normal((h, hd)).astype(np.float32)
    k = 0.1 * rng.standard_normal((seq, kv, hd))
    v = rng.standard_normal((seq, n)).astype(np.float32)
    at = [5, *range(288, 352), 899]
    if case == "seen_before_a_rise":
        at = [1]
        k[600:] += 150 * (q.reshape(kv, -1, hd).mean(1) / (q.reshape(kv, -1, hd).mean(1)**2).sum(
            -1, keepdims=True) / scale)
    for r in at:
        if case == "unseen":  # 150 below for all heads, by a channel that they share
            q[:, 0] = 3
            k[r] = 0
            k[r, :, 0] = -50 / scale
        elif case == "by_one_head":
            q[:, 0] = 3
            q[::h // kv, 0] = -3
            k[r] = 0
            k[r, :, 0] = -50 / scale
    v[at] *= np.float32(big)
    k8, kd = ref.q8_rows(k.reshape(seq, n).astype(np.float32))
    v8, vd = ref.q8_rows(v)
    for n_split in (1, 4):
        got = attend(q, dev(k8), dev(kd), dev(v8), dev(vd), kv, seq - 1, n_split, scale)[0]
        check(got, q, ref.q8_values(k8, kd), ref.q8_values(v8, vd), kv, scale)


@pytest.mark.parametrize("dest", ["f16", "kv8", "write", "write_off_alignment"])
def test_rows_at_negative_positions_are_left(gpu, dest):
    """*pos0_dev = -2: the first two of the rows have no place, the others go to 0, 1, .."""
    h, kv, hd, t, spare = 4, 2, 64, 5, 4
    n, w = kv * hd, (h + 2 * kv) * hd
    x = np.random.default_rng(8).standard_normal((t, w)).astype(np.float32)
    d, pos, qo = dev(x), dev(np.array([-2], np.int32)), empty(t * h * hd)
    off = 1 if dest == "write_off_alignment" else 0
    k8, v8 = (dev(np.full((spare + t) * n + off, 77, np.int8)) for _ in range(2))
    kd, vd = (dev(np.full((spare + t) * n // 32, -3, np.float32)) for _ in range(2))
    kc, vc = (dev(np.full((spare + t) * n, 0x1234, np.uint16)) for _ in range(2))
    c8 = (P(k8) + spare * n + off, P(kd) + spare * n // 8, P(v8) + spare * n + off,
          P(vd) + spare * n // 8)
    pk, pv = P(d) + 4 * h * hd, P(d) + 4 * (h + kv) * hd
    rows = (P(d), w, pk, w, pv, w, None, None, 1e-6, P(qo))
    tail = (h, kv, hd, t, 0, P(pos), 1e4, S())
    if dest == "f16":
        call("tf_qk_norm_rope_append", *rows, P(kc) + 2 * spare * n, P(vc) + 2 * spare * n, *tail)
    elif dest == "kv8":
        call("tf_qk_norm_rope_append_kv8", *rows, *c8, *tail)
    else:
        call("tf_kv8_write", pk, pv, gpu.KV_F32, w, *c8, n, 0, P(pos), t, S())
    v = np.ascontiguousarray(x[2:, (h + kv) * hd:])
    if dest == "f16":
        for c in (kc, vc):
            assert (host(c)[:spare * n] == 0x1234).all() and (host(c)[(spare + t - 2) * n:] == 0x1234).all()
        assert np.array_equal(host(vc)[spare * n:(spare + t - 2) * n], oracle.f32_to_f16(v.ravel()))
        return
    q8, d8 = ref.q8_rows(v)
    for c, s, want, mark in ((k8, 1, None, 77), (v8, 1, q8, 77), (kd, 32, None, -3), (vd, 32, d8, -3)):
        a, b = spare * n // s + (off if s == 1 else 0), (spare + t - 2) * n // s + (off if s == 1 else 0)
        assert (host(c)[:a] == mark).all() and (host(c)[b:] == mark).all()
        if want is not None:
            assert np.array_equal(host(c)[a:b], want.ravel())
