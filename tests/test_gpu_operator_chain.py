"""The operators around a decode step as a program uses them, one after the other:
norm + RoPE into the 8-bit cache, attention over it, logits, a drawn token; eager,
on streams of their own, and captured."""
import numpy as np
import pytest
import torch

import _op_ref as ref
from _gpu import KEEP, P

pytestmark = pytest.mark.gpu

H, KV, HD, VOCAB, SEQ = 14, 2, 64, 5000, 640
EPS, THETA = 1e-6, 1e4


class Chain:
    """One attention layer and a head; its buffers, and a step enqueued on the current
    stream."""

    def __init__(self, gpu, seed):
        self.gpu, rng = gpu, np.random.default_rng(seed)
        n = KV * HD
        self.qkv_w = (rng.standard_normal(((H + 2 * KV) * HD, 96)) / 8).astype(np.float32)
        self.head_w = (rng.standard_normal((VOCAB, H * HD)) / 6).astype(np.float32)
        self.norms = (1 + 0.2 * rng.standard_normal((2, HD))).astype(np.float32)
        self.x = rng.standard_normal((SEQ, 96)).astype(np.float32)
        self.u = rng.random(SEQ).astype(np.float32)
        up = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        self.d = {k: up(getattr(self, k)) for k in ("qkv_w", "head_w", "norms", "x", "u")}
        z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        self.k8, self.v8 = z(SEQ, n, dtype=torch.int8), z(SEQ, n, dtype=torch.int8)
        self.kd, self.vd = z(SEQ, n // 32), z(SEQ, n // 32)
        self.split = gpu.load().tf_flash_decode_kv8_n_split(KV, HD, SEQ)
        self.part, self.q, self.att = z(H * self.split * (2 + HD)), z(H * HD), z(H * HD)
        self.pos = z(1, dtype=torch.int32)
        self.set = dict(t=torch.full((1,), 0.8).cuda(), k=torch.full((1,), 50).int().cuda(),
                        p=torch.full((1,), 0.9).cuda(), m=torch.full((1,), 0.01).cuda())
        size = gpu.load().tf_sample_ws_bytes(1, VOCAB)
        self.ws, self.tok = z(size, dtype=torch.uint8), z(1, dtype=torch.int32)
        KEEP.append(self.__dict__)

    def step(self):
        """At *pos; pos moves on."""
        s, call = self.gpu.stream_ptr(), self.gpu.call
        at = self.pos.long()
        qkv = self.d["qkv_w"] @ self.d["x"][at].reshape(-1)
        w = (H + 2 * KV) * HD
        call("tf_qk_norm_rope_append_kv8", P(qkv), w, P(qkv) + 4 * H * HD, w,
             P(qkv) + 4 * (H + KV) * HD, w, P(self.d["norms"]), P(self.d["norms"]) + 4 * HD, EPS,
             P(self.q), P(self.k8), P(self.kd), P(self.v8), P(self.vd), H, KV, HD, 1, 0,
             P(self.pos), THETA, s)
        call("tf_flash_decode_kv8", P(self.q), P(self.k8), P(self.kd), P(self.v8), P(self.vd),
             P(self.part), P(self.att), None, None, H, KV, HD, 0, P(self.pos), self.split,
             HD**-0.5, s)
        self.logits = self.d["head_w"] @ self.att
        self.un = self.d["u"][at]
        call("tf_sample", P(self.logits), 1, VOCAB, VOCAB, P(self.set["t"]), P(self.set["k"]),
             P(self.set["p"]), P(self.set["m"]), P(self.un), P(self.tok), P(self.ws),
             self.ws.numel(), s)
        self.keep = qkv
        self.pos += 1

    def seen(self):
        return (self.att.cpu().numpy().copy(), self.logits.cpu().numpy().copy(), int(self.tok[0]))

    def reset(self):
        for t in (self.pos, self.k8, self.v8, self.kd, self.vd):
            t.zero_()


def test_eager_against_64_bits(gpu):
    c = Chain(gpu, 1)
    K, V = np.zeros((SEQ, KV * HD)), np.zeros((SEQ, KV * HD))
    for pos in range(40):
        c.step()
        att, logits, tok = c.seen()
        qkv = c.keep.cpu().numpy()
        q, k, v = np.split(qkv, [H * HD, (H + KV) * HD])
        q = ref.norm_rope(q.reshape(1, H, HD), c.norms[0], EPS, [pos], THETA)[0][0]
        # the cache's own rows: a value between two steps may fall to either
        K[pos] = ref.q8_values(c.k8[pos:pos + 1].cpu().numpy(), c.kd[pos:pos + 1].cpu().numpy())[0]
        V[pos] = ref.q8_values(c.v8[pos:pos + 1].cpu().numpy(), c.vd[pos:pos + 1].cpu().numpy())[0]
        k = ref.norm_rope(k.reshape(1, KV, HD), c.norms[1], EPS, [pos], THETA)[0].reshape(1, -1)
        for row, want in ((K[pos], k[0]), (V[pos], v)):
            top = np.repeat(np.abs(want).reshape(-1, 32).max(1), 32)
            assert (np.abs(row - want) <= top / 127 * 0.501 + 1e-6 * top).all()
        want, tol = ref.attention(q, K[:pos + 1], V[:pos + 1], KV, HD**-0.5)
        # q itself is off by up to 24 roundings, which its scores share
        assert (np.abs(att.reshape(H, HD) - want) <= 3 * tol).all()
        assert tok == ref.sample(logits, 0.8, 50, np.float32(0.9), np.float32(0.01), c.u[pos])


def test_captured_and_replayed(gpu):
    c = Chain(gpu, 2)
    want = []
    for _ in range(300):
        c.step()
        want.append(c.seen())
    c.reset()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.step()
    c.reset()
    for i in range(300):  # eager work and a synchronization between the replays
        g.replay()
        torch.cuda.synchronize()
        got = c.seen()
        assert np.array_equal(got[0], want[i][0]) and np.array_equal(got[1], want[i][1]), i
        assert got[2] == want[i][2], i


def test_two_streams_and_two_graphs(gpu):
    """Two chains side by side, each with its own buffers, give what each gives alone."""
    chains = [Chain(gpu, s) for s in (3, 4)]
    alone = []
    for c in chains:
        got = []
        for _ in range(60):
            c.step()
            got.append(c.seen()[2])
        alone.append(got)
        c.reset()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in chains]
    toks = [torch.zeros(60, dtype=torch.int32, device="cuda") for _ in chains]
    for i in range(30):
        for c, s, t in zip(chains, streams, toks):
            with torch.cuda.stream(s):
                c.step()
                t[i:i + 1] = c.tok
    torch.cuda.synchronize()
    graphs = []
    for c in chains:
        g = torch.cuda.CUDAGraph()
        at = c.pos.clone()
        with torch.cuda.graph(g):
            c.step()
        c.pos.copy_(at)
        graphs.append(g)
    torch.cuda.synchronize()
    for i in range(30, 60):
        for c, g, s, t in zip(chains, graphs, streams, toks):
            with torch.cuda.stream(s):
                g.replay()
                t[i:i + 1] = c.tok
    torch.cuda.synchronize()
    for t, a in zip(toks, alone):
        assert t.cpu().tolist() == a


def test_an_8_bit_cache_against_the_f16_one(gpu):
    """The same rows in both caches: outputs apart by what 8 bits leave out.  A row is
    within half a step of each group's largest / 127; the exact attention over the two
    sets of rows says how far apart the outputs may be, both kernels stay at theirs."""
    h, kv, hd, t = 16, 2, 128, 300
    rng = np.random.default_rng(9)
    x = rng.standard_normal((t, (h + 2 * kv) * hd)).astype(np.float32)
    d, n, w = torch.from_numpy(x).cuda(), kv * hd, (h + 2 * kv) * hd
    qo = [torch.zeros(t, h * hd, device="cuda") for _ in range(2)]
    kc, vc = (torch.zeros(t, n, dtype=torch.float16, device="cuda") for _ in range(2))
    k8, v8 = (torch.zeros(t, n, dtype=torch.int8, device="cuda") for _ in range(2))
    kd, vd = (torch.zeros(t, n // 32, device="cuda") for _ in range(2))
    part, out = torch.zeros(h * 8 * (2 + hd), device="cuda"), torch.zeros(2, h * hd, device="cuda")
    KEEP.extend([d, *qo, kc, vc, k8, v8, kd, vd, part, out])
    s = gpu.stream_ptr()
    rows = (P(d), w, P(d) + 4 * h * hd, w, P(d) + 4 * (h + kv) * hd, w, None, None, EPS)
    gpu.call("tf_qk_norm_rope_append", *rows, P(qo[0]), P(kc), P(vc), h, kv, hd, t, 0, None, THETA, s)
    gpu.call("tf_qk_norm_rope_append_kv8", *rows, P(qo[1]), P(k8), P(kd), P(v8), P(vd), h, kv, hd, t,
             0, None, THETA, s)
    assert torch.equal(qo[0], qo[1])
    q = P(qo[0]) + 4 * (t - 1) * h * hd
    gpu.call("tf_flash_decode", q, P(kc), P(vc), P(part), None, P(out), None, None, h, kv, hd, t - 1,
             None, 8, hd**-0.5, s)
    gpu.call("tf_flash_decode_kv8", q, P(k8), P(kd), P(v8), P(vd), P(part), P(out[1]), None, None, h,
             kv, hd, t - 1, None, 8, hd**-0.5, s)
    got = out.cpu().numpy().reshape(2, h, hd)
    qh = qo[0][t - 1].cpu().numpy().reshape(h, hd)
    want16, tol16 = ref.attention(qh, kc.cpu().numpy(), vc.cpu().numpy(), kv, hd**-0.5)
    K, V = (ref.q8_values(a.cpu().numpy(), b.cpu().numpy()) for a, b in ((k8, kd), (v8, vd)))
    want8, tol8 = ref.attention(qh, K, V, kv, hd**-0.5)
    assert (np.abs(got[0] - want16) <= tol16).all() and (np.abs(got[1] - want8) <= tol8).all()
    # 300 near-uniform weights average half steps of 1 / 40 of a unit: under 1 %
    assert np.abs(got[0] - got[1]).max() < 0.02
    # read back, the 8-bit rows serve a prompt's attention: the last row of it
    rk, rv = (torch.zeros(t, n, dtype=torch.float16, device="cuda") for _ in range(2))
    pre = torch.zeros(t, h * hd, device="cuda")
    KEEP.extend([rk, rv, pre])
    gpu.call("tf_kv8_read", P(k8), P(kd), P(v8), P(vd), P(rk), P(rv), gpu.KV_F16, n, 0, t, s)
    gpu.call("tf_attn_prefill", P(qo[0]), P(rk), P(rv), P(pre), h, kv, hd, 0, t, hd**-0.5, s)
    want, tol = ref.attention(qh, rk.cpu().numpy(), rv.cpu().numpy(), kv, hd**-0.5)
    assert (np.abs(pre[t - 1].cpu().numpy().reshape(h, hd) - want) <= tol).all()
