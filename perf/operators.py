"""The block operators of a quantised, text-conditioned transformer, as cases to measure.

Four operators: ``rms_norm_quant`` (residual addition, root-mean-square norm and an 8-bit output
with one scale a row), ``linear_fp8`` (the product that reads that output), ``rope_axes`` (rotary
positions with several axes) and ``cross_attention`` (queries of one length, an encoder's states of
another, padded and masked).  Where ``own`` is false, ``run`` computes them from elementary torch
operations in 32 bits; where it is true it calls this package.
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the norm in front of one row's projection (a timestep's or a pooled embedding): latency
        dict(name="norm one row", op="norm", rows=1, dim=1536, dtype="bf16", residual=True),
        # a text encoder's layer at the full prompt length
        dict(name="norm text 512x4096", op="norm", rows=512, dim=4096, dtype="bf16", residual=True),
        # the hidden states of an 81-frame 480p video: 21 x 30 x 52 tokens
        dict(name="norm video 32760x1536", op="norm", rows=32760, dim=1536, dtype="bf16", residual=True),
        # the six modulation vectors of a block from two timestep embeddings: a weight-bound product
        dict(name="linear two rows", op="linear", rows=2, k=1536, n=9216, out="bf16", epi="bias"),
        # the up-projection of a text encoder over a prompt
        dict(name="linear text up", op="linear", rows=512, k=4096, n=10240, out="bf16", epi="gelu"),
        # the feed-forward up-projection of a video model
        dict(name="linear video up", op="linear", rows=32760, k=1536, n=8960, out="bf16", epi="gelu"),
        # queries and keys of a 512 x 512 image's 32 x 32 patches, two axes, halves rotated
        dict(name="rope image 1024", op="rope", t=1, h=32, w=32, heads=24, heads_k=24, head_dim=64, dims="32,32",
             layout="half", dtype="fp16"),
        # queries and keys of a 480p video, three axes, neighbouring pairs rotated
        dict(name="rope video 32760", op="rope", t=21, h=30, w=52, heads=12, heads_k=12, head_dim=128,
             dims="44,42,42", layout="interleaved", dtype="bf16"),
        # one pooled query for each of two prompts over 512 text slots
        dict(name="cross one query", op="cross", batch=2, sq=1, sk=512, heads=12, heads_kv=12, head_dim=128,
             mask="lens", lse=False, dtype="bf16"),
        # image patches over the joint text context, prompts of several lengths
        dict(name="cross image 4x1024x333", op="cross", batch=4, sq=1024, sk=333, heads=24, heads_kv=24,
             head_dim=64, mask="lens", lse=False, dtype="fp16"),
        # shared key heads, holes in the mask, and one prompt of which nothing is left
        dict(name="cross grouped 3x777x257", op="cross", batch=3, sq=777, sk=257, heads=16, heads_kv=4,
             head_dim=128, mask="holes", lse=True, dtype="bf16"),
        # the two guidance branches of a 480p video over 512 text tokens
        dict(name="cross video 2x32760x512", op="cross", batch=2, sq=32760, sk=512, heads=12, heads_kv=12,
             head_dim=128, mask="none", lse=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "rope", "cross"])
    if op == "norm":
        rows, dim = _log(rng, 1, 32760), _log(rng, 64, 8192)
        if rng.random() < 0.5:
            dim = max(64, dim // 64 * 64)
        rows = min(rows, 32760 * 1536 // dim)
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    residual=rng.random() < 0.7)
    if op == "linear":
        rows, k, n = _log(rng, 1, 32760), _log(rng, 64, 10240), _log(rng, 64, 10240)
        if rng.random() < 0.6:
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        rows = min(rows, max(1, 32760 * 1536 * 8960 // (k * n)))
        return dict(op=op, rows=rows, k=k, n=n, out=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    epi=rng.choice(["none", "bias", "gelu", "residual", "gated"]))
    if op == "rope":
        head_dim, dims = rng.choice([(128, "44,42,42"), (64, "32,32"), (64, "16,24,24"), (96, "32,32,32"), (128, "32,48"),
                                     (80, "20,30,30"), (128, "128")])
        axes = dims.count(",") + 1
        heads = rng.choice([4, 8, 12, 24])
        t = _log(rng, 1, 21) if axes == 3 else 1
        h = _log(rng, 1, 40) if axes > 1 else 1
        w = _log(rng, 1, 60)
        heads_k, dtype = rng.choice([heads, heads // 4, 1]), rng.choice(["bf16", "fp16", "fp32"])
        t = min(t, max(1, 400_000_000 // (2 * h * w * (heads + heads_k) * head_dim * BYTES[dtype])))
        return dict(op=op, t=t, h=h, w=w, heads=heads, heads_k=heads_k, head_dim=head_dim, dims=dims,
                    layout=rng.choice(["interleaved", "half"]), dtype=dtype)
    head_dim = rng.choice([64, 128])
    heads = rng.choice([4, 12, 16, 24])
    batch, sk = rng.randint(1, 5), _log(rng, 1, 4096)
    sq = min(_log(rng, 1, 32760), max(1, 2 * 32760 * 512 * 12 * 128 // (batch * sk * heads * head_dim)))
    return dict(op=op, batch=batch, sq=sq, sk=sk, heads=heads, heads_kv=rng.choice([heads, heads // 4]),
                head_dim=head_dim, mask=rng.choice(["none", "lens", "holes"]), lse=rng.random() < 0.5,
                dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _lens(case):
    """Valid keys of each batch entry: a fixed spread from all of them downwards."""
    b, sk = case["batch"], case["sk"]
    return [max(1, sk - (i * sk * 7) // (8 * b)) for i in range(b)]


def _holes(case):
    """Keys that may be attended to: two in three, none in the last entry of a batch of three or more."""
    b, sk = case["batch"], case["sk"]
    m = (torch.arange(sk)[None, :] + torch.arange(b)[:, None]) % 3 != 2
    if b >= 3:
        m[-1] = False
    return m


def _pitched(rows, cols, device):
    """fp8 [rows, cols] whose rows start 16 bytes apart or a multiple of it, as weights are laid out once."""
    return torch.zeros(rows, -(-cols // 16) * 16, device=device, dtype=torch.uint8).view(FP8)[:, :cols]


def _quantised(x):
    scale = (x.abs().amax(dim=1) / FP8_MAX).clamp_min(1e-30)
    q = _pitched(x.shape[0], x.shape[1], x.device)
    q.copy_((x / scale[:, None]).to(FP8))
    return q, scale


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        dt = DTYPES[case["dtype"]]
        s["x"] = randn(case["rows"], case["dim"], dtype=dt)
        s["res"] = randn(case["rows"], case["dim"], dtype=dt, std=3.0) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * randn(case["dim"])).to(dt)
    elif case["op"] == "linear":
        dt = DTYPES[case["out"]]
        m, k, n, epi = case["rows"], case["k"], case["n"], case["epi"]
        s["xq"], s["xs"] = _quantised(randn(m, k))
        s["wq"], s["ws"] = _quantised(randn(n, k, std=1.0 / math.sqrt(k)))
        s["b"] = randn(n, dtype=dt, std=0.5) if epi != "none" else None
        s["act"] = "gelu" if epi == "gelu" else None
        s["res"] = randn(m, n, dtype=dt) if epi in ("residual", "gated") else None
        s["gate"] = randn(2, n) if epi == "gated" else None
        s["rpb"] = (m + 1) // 2
    elif case["op"] == "rope":
        dt = DTYPES[case["dtype"]]
        t, h, w = case["t"], case["h"], case["w"]
        s["dims"] = tuple(int(v) for v in case["dims"].split(","))
        grid = torch.stack(torch.meshgrid(torch.arange(t), torch.arange(h), torch.arange(w), indexing="ij"), -1)
        s["pos"] = grid.reshape(-1, 3)[:, 3 - len(s["dims"]):].contiguous().to(dev)
        s["q"] = randn(t * h * w, case["heads"] * case["head_dim"], dtype=dt)
        s["k"] = randn(t * h * w, case["heads_k"] * case["head_dim"], dtype=dt)
    else:
        dt = DTYPES[case["dtype"]]
        b, sq, sk, d = case["batch"], case["sq"], case["sk"], case["head_dim"]
        s["q"] = randn(b, sq, case["heads"] * d, dtype=dt)
        s["k"] = randn(b, sk, case["heads_kv"] * d, dtype=dt)
        s["v"] = randn(b, sk, case["heads_kv"] * d, dtype=dt)
        s["lens"] = torch.tensor(_lens(case), device=dev, dtype=torch.int32) if case["mask"] == "lens" else None
        s["allowed"] = _holes(case).to(dev) if case["mask"] == "holes" else None
    return s


def _plain_norm(s):
    if s["res"] is None:
        h = s["x"]
    else:
        h = (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    scale = (y.abs().amax(-1) / FP8_MAX).clamp_min(1e-30)
    return (y / scale[:, None]).to(FP8), scale, None if s["res"] is None else h


def _plain_linear(s):
    y = (s["xq"].float() @ s["wq"].float().t()) * s["xs"][:, None] * s["ws"]
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["gate"] is not None:
        y = y * s["gate"][torch.arange(y.shape[0], device=y.device) // s["rpb"]]
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(DTYPES[s["out"]])


def _frequencies(s, device):
    """The axis and the frequency of every rotated pair, in 64 bits."""
    axis = torch.cat([torch.full((d // 2,), i) for i, d in enumerate(s["dims"])])
    freq = torch.cat([10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d) for d in s["dims"]])
    return axis.to(device), freq.to(device)


def _plain_rotate(x, cos, sin, head_dim, layout):
    f = x.float().reshape(x.shape[0], -1, head_dim)
    n = cos.shape[1]
    if layout == "half":
        a, b = f[..., :n], f[..., n:2 * n]
    else:
        a, b = f[..., 0:2 * n:2], f[..., 1:2 * n:2]
    c, d = a * cos[:, None] - b * sin[:, None], a * sin[:, None] + b * cos[:, None]
    r = torch.cat([c, d], -1) if layout == "half" else torch.stack([c, d], -1).flatten(-2)
    return torch.cat([r, f[..., 2 * n:]], -1).reshape(x.shape).to(x.dtype)


def _plain_rope(s):
    axis, freq = _frequencies(s, s["q"].device)
    angle = s["pos"].double()[:, axis] * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    return tuple(_plain_rotate(s[n], cos, sin, s["head_dim"], s["layout"]) for n in ("q", "k"))


def _plain_cross(s):
    b, sq, sk, h, hk, d = (s[n] for n in ("batch", "sq", "sk", "heads", "heads_kv", "head_dim"))
    q = s["q"].float().reshape(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, h // hk * sq, d)
    k = s["k"].float().reshape(b, sk, hk, d).permute(0, 2, 3, 1)
    v = s["v"].float().reshape(b, sk, hk, d).transpose(1, 2)
    p = (q @ k).mul_(1.0 / math.sqrt(d))
    allowed = s["allowed"]
    if s["lens"] is not None:
        allowed = torch.arange(sk, device=q.device) < s["lens"][:, None]
    if allowed is not None:
        p = p.masked_fill_(~allowed[:, None, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, torch.zeros_like(total))
    o = o.reshape(b, h, sq, d).transpose(1, 2).reshape(b, sq, h * d).to(s["q"].dtype)
    return (o, (top + total.log()).reshape(b, h, sq)) if s["lse"] else o


def _own_norm(s):
    from ditserve_b200 import ops
    return ops.rms_norm_quant(s["x"], s["weight"], residual=s["res"], eps=1e-6)


def _own_linear(s):
    from ditserve_b200 import ops
    return ops.linear_fp8(s["xq"], s["xs"], s["wq"], s["ws"], s["b"], act=s["act"], residual=s["res"], gate=s["gate"],
                          rows_per_batch=s["rpb"], out_dtype=DTYPES[s["out"]])


def _own_rope(s):
    from ditserve_b200 import ops
    return ops.rope_axes(s["q"], s["pos"], s["dims"], k=s["k"], head_dim=s["head_dim"], theta=10000.0, layout=s["layout"])


def _own_cross(s):
    from ditserve_b200 import ops
    return ops.cross_attention(s["q"], s["k"], s["v"], s["heads"], heads_kv=s["heads_kv"], kv_lens=s["lens"],
                               key_mask=s["allowed"], return_lse=s["lse"])


def run(state):
    if own:
        return {"norm": _own_norm, "linear": _own_linear, "rope": _own_rope, "cross": _own_cross}[state["op"]](state)
    return {"norm": _plain_norm, "linear": _plain_linear, "rope": _plain_rope, "cross": _plain_cross}[state["op"]](state)


def work(case):
    if case["op"] == "norm":
        n, e = case["rows"] * case["dim"], BYTES[case["dtype"]]
        return {"bytes": n * (e * (3 if case["residual"] else 1) + 1) + 4 * case["rows"] + e * case["dim"], "flops": 6 * n}
    if case["op"] == "linear":
        m, k, n, e = case["rows"], case["k"], case["n"], BYTES[case["out"]]
        extra = (m * n * e if case["epi"] in ("residual", "gated") else 0) + (8 * n if case["epi"] == "gated" else 0)
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e + (n * e if case["epi"] != "none" else 0) + extra,
                "flops": 2 * m * n * k}
    if case["op"] == "rope":
        rows = case["t"] * case["h"] * case["w"]
        n = rows * (case["heads"] + case["heads_k"]) * case["head_dim"]
        return {"bytes": 2 * n * BYTES[case["dtype"]] + 8 * rows * (case["dims"].count(",") + 1), "flops": 3 * n}
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "sq", "sk", "heads", "heads_kv", "head_dim"))
    keys = b * sk
    if case["mask"] == "lens":
        keys = sum(_lens(case))
    elif case["mask"] == "holes":
        keys = int(_holes(case).sum())
    e = BYTES[case["dtype"]]
    return {"bytes": e * (2 * b * sq * h * d + 2 * keys * hk * d) + (4 * b * h * sq if case["lse"] else 0)
            + (b * sk if case["mask"] == "holes" else 0) + 4 * b, "flops": 4 * sq * h * d * keys}


def exact(case, seed):
    s = prepare(case, seed)
    dev = torch.device("cuda")
    f64 = torch.float64
    if case["op"] == "norm":
        h, stored = s["x"], None
        if s["res"] is not None:
            stored = s["x"].to(f64) + s["res"].to(f64)
            h = stored.to(s["x"].dtype)  # the norm reads the residual as it is stored
        f = h.to(f64)
        y = s["weight"].to(f64) * f / torch.sqrt(torch.sum(f * f, 1, keepdim=True) / case["dim"] + 1e-6)
        scale = torch.max(y.abs(), dim=1).values / FP8_MAX
        return y / scale.unsqueeze(1), scale, stored
    if case["op"] == "linear":
        y = torch.mm(s["xq"].to(f64), s["wq"].to(f64).T)
        y.mul_(s["xs"].to(f64).unsqueeze(1)).mul_(s["ws"].to(f64))
        if s["b"] is not None:
            y.add_(s["b"].to(f64))
        if case["epi"] == "gelu":
            y = y / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3)))
        if case["epi"] == "gated":
            y[: s["rpb"]] *= s["gate"][0].to(f64)
            y[s["rpb"]:] *= s["gate"][1].to(f64)
        return y if s["res"] is None else y.add_(s["res"].to(f64))
    if case["op"] == "rope":
        got = []
        for name in ("q", "k"):
            x = s[name].to(f64).reshape(s[name].shape[0], -1, case["head_dim"])
            y, pair, rotated = x.clone(), 0, sum(s["dims"])
            for a, d in enumerate(s["dims"]):
                for j in range(d // 2):
                    angle = s["pos"][:, a].to(f64) * math.pow(10000.0, -2.0 * j / d)
                    c, n = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
                    i0, i1 = (pair, pair + rotated // 2) if case["layout"] == "half" else (2 * pair, 2 * pair + 1)
                    y[..., i0] = c * x[..., i0] - n * x[..., i1]
                    y[..., i1] = n * x[..., i0] + c * x[..., i1]
                    pair += 1
            got.append(y.reshape(s[name].shape))
        return tuple(got)
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "sq", "sk", "heads", "heads_kv", "head_dim"))
    out = torch.zeros(b, sq, h * d, dtype=f64, device=dev)
    lse = torch.full((b, h, sq), -math.inf, dtype=f64, device=dev)
    for i in range(b):
        keep = torch.arange(sk, device=dev)
        if case["mask"] == "lens":
            keep = keep[: _lens(case)[i]]
        elif case["mask"] == "holes":
            keep = keep[_holes(case)[i].to(dev)]
        if keep.numel() == 0:
            continue
        for j in range(h):
            at, kv = slice(j * d, (j + 1) * d), slice(j // (h // hk) * d, (j // (h // hk) + 1) * d)
            z = torch.mm(s["q"][i, :, at].to(f64), s["k"][i, keep, kv].to(f64).T) / math.sqrt(d)
            out[i, :, at] = torch.mm(torch.softmax(z, 1), s["v"][i, keep, kv].to(f64))
            lse[i, j] = torch.logsumexp(z, 1)
    return (out, lse) if case["lse"] else out
