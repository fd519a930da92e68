"""The operators around a decode step's attention and at its end, as measurable cases.

  rope    per-head RMS norms of q and k with the NeoX rotation in the same
          pass (tf_qk_norm_rope), q and k as f32 rows, or K/V appended to the
          f16 cache (tf_qk_norm_rope_append) or to the 8-bit cache
          (tf_qk_norm_rope_append_kv8, its rows then read back as f16);
  store   K/V rows quantised into the 8-bit cache as they are written
          (tf_kv8_write) and rows of it read back (tf_kv8_read);
  flash   one token's attention over the 8-bit cache (tf_flash_decode_kv8);
  sample  a token a row from its logits: temperature, top-k, top-p, min-p and
          a given random number (tf_sample).

An 8-bit cache row is int8 values with one f32 scale per 32 of them:
d = amax * f32(1/127), q = rint(x / d), in f32.  Heads and widths are those of
the Qwen2.5 0.5B, 3B and 7B shapes, and a generic one of head_dim 256.
"""
import math

import numpy as np
import torch

own = False

# query heads, kv heads, head_dim
HEADS = {"0.5b": (14, 2, 64), "3b": (16, 2, 128), "7b": (28, 4, 128), "hd256": (16, 4, 256)}
VOCAB = 151936
EPS, THETA = 1e-6, 1e6
INV127 = float(np.float32(1.0) / np.float32(127.0))


def listed():
    return [
        # one decoded token of the smallest model, K/V to the f16 cache: launch latency
        {"name": "rope_one", "kind": "rope", "size": "0.5b", "to": "f16", "pos": 611, "t": 1},
        # a prompt chunk far into a long document, rows for a caller with a cache of its own
        {"name": "rope_far_777", "kind": "rope", "size": "3b", "to": "f32", "pos": 130000, "t": 777},
        # a long prompt of a 7B model straight into the 8-bit cache
        {"name": "rope_kv8_4096", "kind": "rope", "size": "7b", "to": "kv8", "pos": 0, "t": 4096},
        # one decoded token into the 8-bit cache, its row read back
        {"name": "store_one", "kind": "store", "size": "3b", "src": "f32", "dst": "f32",
         "pos": 1000, "t": 1, "back": 1},
        # the last 509 rows of a prompt stored from f32, the whole cache read back as the f16
        # rows that prompt attention takes
        {"name": "store_prompt_8k", "kind": "store", "size": "7b", "src": "f32", "dst": "f16",
         "pos": 7683, "t": 509, "back": 8192},
        # an f16 cache of 32K tokens converted to 8 bits, and read back to compare
        {"name": "store_f16_32k", "kind": "store", "size": "7b", "src": "f16", "dst": "f32",
         "pos": 0, "t": 32768, "back": 32768},
        # a token early in a chat
        {"name": "flash_3b_512", "kind": "flash", "size": "3b", "ctx": 512},
        # an odd length at head_dim 64
        {"name": "flash_05b_5001", "kind": "flash", "size": "0.5b", "ctx": 5001},
        # one token of a 7B model at the end of a 128K context
        {"name": "flash_7b_128k", "kind": "flash", "size": "7b", "ctx": 131072},
        # one token of a chat with the usual filters
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": VOCAB, "temp": 0.8,
         "top_k": 40, "top_p": 0.95, "min_p": 0.05},
        # one token by temperature alone, nothing filtered
        {"name": "sample_one_pure", "kind": "sample", "rows": 1, "vocab": VOCAB, "temp": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # many continuations at once, each by its nucleus
        {"name": "sample_64_nucleus", "kind": "sample", "rows": 64, "vocab": VOCAB, "temp": 1.0,
         "top_k": 0, "top_p": 0.95, "min_p": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "store", "flash", "flash", "sample", "sample"])
    size = rng.choice(["0.5b", "3b", "7b", "hd256"])
    if kind == "rope":
        return {"kind": kind, "size": size, "to": rng.choice(["f32", "f16", "kv8"]),
                "pos": rng.choice([0, _log(rng, 10, 130000)]),
                "t": _log(rng, 1, 2048 if size == "hd256" else 4096)}
    if kind == "store":
        t = _log(rng, 1, 8192)
        pos = _log(rng, 1, 8192)
        return {"kind": kind, "size": size, "src": rng.choice(["f32", "f16"]),
                "dst": rng.choice(["f32", "f16"]), "pos": pos, "t": t,
                "back": rng.choice([t, pos + t])}
    if kind == "flash":
        return {"kind": kind, "size": size, "ctx": _log(rng, 1, 65536 if size == "hd256" else 131072)}
    return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, VOCAB),
            "temp": round(rng.uniform(0.4, 1.6), 2),
            "top_k": rng.choice([0, 0, 1, rng.randint(2, 100), _log(rng, 100, 5000)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
            "min_p": rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)])}


# ------------------------------------------------------------------ inputs

def _gen(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * (seed % 2000003) + 31 * len(case["kind"]))
    return g


def _quantise(x):
    """int8 values and f32 scales of rows of f32 values, 32 at a time."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    amax = y.abs().amax(-1, keepdim=True)
    d = amax * torch.tensor(INV127, device=x.device)
    q = torch.round(y / torch.where(d > 0, d, torch.ones_like(d)))
    return q.to(torch.int8).reshape(x.shape), d.squeeze(-1)


def _values(q, d):
    y = q.reshape(*q.shape[:-1], -1, 32).float() * d.unsqueeze(-1)
    return y.reshape(q.shape)


def _kv_rows(g, n, n_kv, hd):
    """Cache rows: a few channels of each head larger than the rest, as keys have them."""
    x = torch.randn(n, n_kv, hd, generator=g, device="cuda")
    gain = 0.6 + 3.0 * torch.rand(n_kv, hd, generator=g, device="cuda").pow(8)
    return (x * gain).reshape(n, n_kv * hd)


def prepare(case, seed):
    g = _gen(case, seed)
    s = {"case": case}

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["kind"] == "rope":
        h, kv, hd = HEADS[case["size"]]
        t, end = case["t"], case["pos"] + case["t"]
        # q, k and v side by side, as one projection leaves them
        s["qkv"] = 2.0 * rand(t, (h + 2 * kv) * hd)
        s["q_norm"] = 1.0 + 0.3 * rand(hd)
        s["k_norm"] = 1.0 + 0.3 * rand(hd)
        s["q_out"] = torch.zeros(t, h * hd, device="cuda")
        if case["to"] == "f32":
            s["k_out"] = torch.zeros(t, kv * hd, device="cuda")
        elif case["to"] == "f16":
            s["kc"] = torch.zeros(end, kv * hd, dtype=torch.float16, device="cuda")
            s["vc"] = torch.zeros_like(s["kc"])
        else:
            _cache8(s, end, kv * hd)
            s["k_back"] = torch.zeros(t, kv * hd, dtype=torch.float16, device="cuda")
            s["v_back"] = torch.zeros_like(s["k_back"])
    elif case["kind"] == "store":
        h, kv, hd = HEADS[case["size"]]
        n, end = kv * hd, case["pos"] + case["t"]
        ty = torch.float16 if case["src"] == "f16" else torch.float32
        s["k"], s["v"] = (_kv_rows(g, case["t"], kv, hd).to(ty) for _ in range(2))
        _cache8(s, end, n)
        if case["back"] > case["t"]:  # rows that an earlier prompt stored
            old = case["pos"]
            s["k8"][:old], s["kd"][:old] = _quantise(_kv_rows(g, old, kv, hd))
            s["v8"][:old], s["vd"][:old] = _quantise(_kv_rows(g, old, kv, hd))
        ty = torch.float16 if case["dst"] == "f16" else torch.float32
        s["k_back"] = torch.zeros(case["back"], n, dtype=ty, device="cuda")
        s["v_back"] = torch.zeros_like(s["k_back"])
    elif case["kind"] == "flash":
        h, kv, hd = HEADS[case["size"]]
        s["q"] = rand(h, hd)
        s["k8"], s["kd"] = _quantise(_kv_rows(g, case["ctx"], kv, hd))
        s["v8"], s["vd"] = _quantise(_kv_rows(g, case["ctx"], kv, hd))
        # room for the partials of any split count that the library recommends
        s["partial"] = torch.zeros(h * (128 * 1024 // (kv * hd) + 256) * (2 + hd), device="cuda")
        s["out"] = torch.zeros(h, hd, device="cuda")
    else:
        r, n = case["rows"], case["vocab"]
        # a broad body and a few dozen tokens that the context makes likely
        x = 2.2 * rand(r, n)
        likely = torch.randint(0, n, (r, 40), generator=g, device="cuda")
        lift = 4.0 + 9.0 * torch.rand(r, 40, generator=g, device="cuda")
        s["logits"] = x.scatter_add_(1, likely, lift)

        def vary(v):  # settings of a row of their own, near the case's
            f = 0.9 + 0.2 * torch.rand(r, generator=g, device="cuda")
            return (f * v).float()

        s["temp"] = vary(case["temp"])
        s["top_k"] = torch.ceil(vary(case["top_k"])).int()
        s["top_p"] = (1.0 - vary(1.0 - case["top_p"])).float()
        s["min_p"] = vary(case["min_p"])
        s["u"] = torch.rand(r, generator=g, device="cuda")
        s["out"] = torch.zeros(r, dtype=torch.int32, device="cuda")
        # a workspace of four times the logits, and room for the smallest call
        s["ws"] = torch.zeros(4 * r * n + (1 << 18) * r, dtype=torch.int32, device="cuda")
    return s


def _cache8(s, rows, n):
    s["k8"], s["v8"] = (torch.zeros(rows, n, dtype=torch.int8, device="cuda") for _ in range(2))
    s["kd"], s["vd"] = (torch.zeros(rows, n // 32, device="cuda") for _ in range(2))


# ------------------------------------------------------------------ one pass

def run(s):
    return _RUN[s["case"]["kind"]](s)


def _rotate(x, pos, inv_freq):
    """x [t, heads, hd] rotated by the positions' angles (formed in 64 bits)."""
    ang = pos.double().unsqueeze(-1) * inv_freq
    c, n = ang.cos().float().unsqueeze(1), ang.sin().float().unsqueeze(1)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def _norm(x, w):
    return x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w


def _run_rope(s):
    c = s["case"]
    h, kv, hd = HEADS[c["size"]]
    t, pos, x = c["t"], c["pos"], s["qkv"]
    if own:
        from taraference_amd import capi
        row, st = x.shape[1], capi.stream_ptr()
        q = x.data_ptr()
        k, v = q + 4 * h * hd, q + 4 * (h + kv) * hd
        norms = (s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS)
        shape = (h, kv, hd, t, pos, None, THETA, st)
        if c["to"] == "f32":
            capi.call("tf_qk_norm_rope", q, row, k, row, *norms, s["q_out"].data_ptr(),
                      s["k_out"].data_ptr(), *shape)
            return s["q_out"], s["k_out"]
        if c["to"] == "f16":
            capi.call("tf_qk_norm_rope_append", q, row, k, row, v, row, *norms,
                      s["q_out"].data_ptr(), s["kc"].data_ptr(), s["vc"].data_ptr(), *shape)
            return s["q_out"], s["kc"][pos:], s["vc"][pos:]
        cache = [s[n].data_ptr() for n in ("k8", "kd", "v8", "vd")]
        capi.call("tf_qk_norm_rope_append_kv8", q, row, k, row, v, row, *norms,
                  s["q_out"].data_ptr(), *cache, *shape)
        capi.call("tf_kv8_read", *cache, s["k_back"].data_ptr(), s["v_back"].data_ptr(),
                  capi.KV_F16, kv * hd, pos, t, st)
        return s["q_out"], s["k_back"], s["v_back"]
    q, k, v = x.split([h * hd, kv * hd, kv * hd], 1)
    inv = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=x.device) / hd)
    p = torch.arange(pos, pos + t, device=x.device)
    q = _rotate(_norm(q.reshape(t, h, hd), s["q_norm"]), p, inv).reshape(t, -1)
    k = _rotate(_norm(k.reshape(t, kv, hd), s["k_norm"]), p, inv).reshape(t, -1)
    if c["to"] == "f32":
        return q, k
    if c["to"] == "f16":
        s["kc"][pos:], s["vc"][pos:] = k.half(), v.half()
        return q, s["kc"][pos:], s["vc"][pos:]
    s["k8"][pos:], s["kd"][pos:] = _quantise(k)
    s["v8"][pos:], s["vd"][pos:] = _quantise(v)
    return (q, _values(s["k8"][pos:], s["kd"][pos:]).half(),
            _values(s["v8"][pos:], s["vd"][pos:]).half())


def _run_store(s):
    c = s["case"]
    h, kv, hd = HEADS[c["size"]]
    n, pos, t, first = kv * hd, c["pos"], c["t"], c["pos"] + c["t"] - c["back"]
    if own:
        from taraference_amd import capi
        st = capi.stream_ptr()
        cache = [s[m].data_ptr() for m in ("k8", "kd", "v8", "vd")]
        ty = {"f32": capi.KV_F32, "f16": capi.KV_F16}
        capi.call("tf_kv8_write", s["k"].data_ptr(), s["v"].data_ptr(), ty[c["src"]], n, *cache,
                  n, pos, None, t, st)
        capi.call("tf_kv8_read", *cache, s["k_back"].data_ptr(), s["v_back"].data_ptr(),
                  ty[c["dst"]], n, first, c["back"], st)
        return s["k_back"], s["v_back"]
    s["k8"][pos:], s["kd"][pos:] = _quantise(s["k"].float())
    s["v8"][pos:], s["vd"][pos:] = _quantise(s["v"].float())
    ty = s["k_back"].dtype
    return (_values(s["k8"][first:], s["kd"][first:]).to(ty),
            _values(s["v8"][first:], s["vd"][first:]).to(ty))


def _run_flash(s):
    c = s["case"]
    h, kv, hd = HEADS[c["size"]]
    ctx, scale = c["ctx"], 1.0 / math.sqrt(hd)
    if own:
        from taraference_amd import capi
        n_split = capi.load().tf_flash_decode_kv8_n_split(kv, hd, ctx)
        capi.call("tf_flash_decode_kv8", s["q"].data_ptr(), s["k8"].data_ptr(), s["kd"].data_ptr(),
                  s["v8"].data_ptr(), s["vd"].data_ptr(), s["partial"].data_ptr(),
                  s["out"].data_ptr(), None, None, h, kv, hd, ctx - 1, None, n_split, scale,
                  capi.stream_ptr())
        return s["out"]
    k = _values(s["k8"], s["kd"]).reshape(ctx, kv, hd).transpose(0, 1)
    v = _values(s["v8"], s["vd"]).reshape(ctx, kv, hd).transpose(0, 1)
    q = s["q"].reshape(kv, h // kv, hd)
    x = torch.matmul(k, q.transpose(1, 2).contiguous()) * scale  # [kv, ctx, group]
    e = torch.exp(x - x.amax(1, keepdim=True))
    o = torch.matmul(e.transpose(1, 2).contiguous(), v)  # [kv, group, hd]
    return (o / e.sum(1).unsqueeze(-1)).reshape(h, hd)


def _run_sample(s):
    c = s["case"]
    r, n = c["rows"], c["vocab"]
    if own:
        from taraference_amd import capi
        on = {"top_k": c["top_k"] > 0, "top_p": c["top_p"] < 1, "min_p": c["min_p"] > 0}
        filters = [s[m].data_ptr() if on[m] else None for m in ("top_k", "top_p", "min_p")]
        capi.call("tf_sample", s["logits"].data_ptr(), r, n, n, s["temp"].data_ptr(), *filters,
                  s["u"].data_ptr(), s["out"].data_ptr(), s["ws"].data_ptr(),
                  4 * s["ws"].numel(), capi.stream_ptr())
        return s["out"]
    z = s["logits"].double() / s["temp"].double().unsqueeze(1)
    e = torch.exp(z - z.amax(1, keepdim=True))
    if c["top_k"] or c["top_p"] < 1 or c["min_p"]:
        _, order = torch.sort(s["logits"], dim=1, descending=True, stable=True)
        w = torch.gather(e, 1, order)
        at = torch.arange(n, device=w.device).unsqueeze(0)
        if c["top_k"]:
            w = torch.where(at < s["top_k"].unsqueeze(1), w, 0.0)
        before = torch.cumsum(w, 1) - w
        keep = w > 0
        if c["top_p"] < 1:
            keep &= before < s["top_p"].double().unsqueeze(1) * w.sum(1, keepdim=True)
        if c["min_p"]:
            keep &= w >= s["min_p"].double().unsqueeze(1)
        keep[:, 0] = True
        e = torch.zeros_like(e).scatter_(1, order, torch.where(keep, w, 0.0))
    run_sum = torch.cumsum(e, 1)
    return (run_sum <= s["u"].double().unsqueeze(1) * run_sum[:, -1:]).sum(1).int()


_RUN = {"rope": _run_rope, "store": _run_store, "flash": _run_flash, "sample": _run_sample}


# ------------------------------------------------------------------ the work

def work(case):
    if case["kind"] == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": 4 * values + 24 * case["rows"], "flops": 4 * values}
    h, kv, hd = HEADS[case["size"]]
    n = kv * hd
    if case["kind"] == "rope":
        t = case["t"]
        out = {"f32": 4 * n, "f16": 2 * 2 * n, "kv8": 2 * (n + n // 8) * 2 + 2 * 2 * n}[case["to"]]
        read = 4 * (h * hd + (n if case["to"] == "f32" else 2 * n))
        return {"bytes": t * (read + 4 * h * hd + out) + 8 * hd, "flops": 10 * t * (h + kv) * hd}
    if case["kind"] == "store":
        src, dst = (4 if case[m] == "f32" else 2 for m in ("src", "dst"))
        row8 = n + n // 8
        return {"bytes": 2 * (case["t"] * (src * n + row8) + case["back"] * (dst * n + row8)),
                "flops": 2 * n * (4 * case["t"] + case["back"])}
    return {"bytes": 2 * case["ctx"] * (n + n // 8) + 8 * h * hd,
            "flops": 4 * case["ctx"] * h * hd}


# ------------------------------------------------------------------ in 64 bits

def _quantised64(x):
    """The values that 8-bit rows of x stand for: the scale and the quotient are
    f32 numbers by the format's definition."""
    y = x.reshape(x.shape[0], -1, 32)
    d = (np.abs(y).max(-1, keepdims=True).astype(np.float32) * np.float32(INV127))
    d64 = d.astype(np.float64)
    q = np.rint((y / np.where(d64 > 0, d64, 1.0)).astype(np.float32)).astype(np.float64)
    return (q * d64).reshape(x.shape)


def _exact_rope(case, s):
    h, kv, hd = HEADS[case["size"]]
    t = case["t"]
    x = s["qkv"].double().cpu().numpy()
    half = hd // 2
    ang = (case["pos"] + np.arange(t, dtype=np.float64))[:, None] * np.power(
        float(THETA), np.arange(half) / -float(half))[None, :]
    rot = np.exp(1j * ang)[:, None, :]

    def heads(y, w):
        y = y.reshape(t, -1, hd)
        y = y / np.sqrt(np.mean(np.square(y), axis=-1, keepdims=True) + EPS)
        y = y * w.double().cpu().numpy()
        z = (y[..., :half] + 1j * y[..., half:]) * rot
        return np.concatenate([z.real, z.imag], axis=-1).reshape(t, -1)

    q = heads(x[:, :h * hd], s["q_norm"])
    k = heads(x[:, h * hd:(h + kv) * hd], s["k_norm"])
    v = x[:, (h + kv) * hd:]
    if case["to"] == "f32":
        return q, k
    if case["to"] == "f16":
        return q, k, v
    return q, _quantised64(k), _quantised64(v)


def _exact_store(case, s):
    first = case["pos"] + case["t"] - case["back"]
    got = []
    for name in ("k", "v"):
        new = _quantised64(s[name].double().cpu().numpy())
        q8 = s[name + "8"][first:case["pos"]].double().cpu().numpy()
        d = s[name + "d"][first:case["pos"]].double().cpu().numpy()
        got.append(np.concatenate([q8 * np.repeat(d, 32, axis=1), new]))
    return tuple(got)


def _exact_flash(case, s):
    h, kv, hd = HEADS[case["size"]]
    out = []
    for head in range(h):
        j = head // (h // kv)
        cols, groups = slice(j * hd, (j + 1) * hd), slice(j * hd // 32, (j + 1) * hd // 32)
        k, v = (s[m + "8"][:, cols].double() *
                s[m + "d"][:, groups].double().repeat_interleave(32, 1) for m in ("k", "v"))
        x = (k * s["q"][head].double()).sum(1) / math.sqrt(hd)
        p = torch.exp(x - torch.logsumexp(x, 0))
        out.append((p.unsqueeze(1) * v).sum(0))
    return torch.stack(out)


def _exact_sample(case, s):
    x = s["logits"].double().cpu().numpy()
    par = {m: s[m].double().cpu().numpy() for m in ("temp", "top_k", "top_p", "min_p", "u")}
    n, got = case["vocab"], []
    for r in range(case["rows"]):
        z = x[r] / par["temp"][r]
        order = np.argsort(-z, kind="stable")
        w = np.exp(z[order] - z[order[0]])
        m = min(int(par["top_k"][r]), n) if case["top_k"] else n
        w = w[:m]
        if case["top_p"] < 1:
            m = int(np.searchsorted(np.cumsum(w), par["top_p"][r] * w.sum(), side="left")) + 1
        if case["min_p"]:
            m = min(m, max(1, int((w >= par["min_p"][r]).sum())))
        kept = np.sort(order[:m])
        c = np.cumsum(np.exp(z[kept] - z[order[0]]))
        at = int(np.searchsorted(c, par["u"][r] * c[-1], side="right"))
        got.append(int(kept[min(at, len(kept) - 1)]))
    return np.array(got, np.int32)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "flash": _exact_flash,
            "sample": _exact_sample}[case["kind"]](case, s)
