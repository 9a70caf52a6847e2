"""Workloads of the clip-token operators: rotary positions with several axes, attention with its gradient, and the dense layer with
bias, activation and residual in one call.

Every case is one call (or one forward + backward pair) as a program over clips of video makes it: tokens of T frames, slots of a frame,
single slots of a stream over the memory of earlier frames, the channel widths of the slot head (256, feed-forward 2048) and of the Swin-L
backbone (192 .. 1536, factor 4). `own` chooses between plain elementary torch (False) and the framework's operators (True).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # ---- rotary positions -------------------------------------------------------------------------------------------------
        # a stream's newest slot: one token, queries and shared keys in one call; the angle of a far frame index
        dict(name="rotary_one_token", op="rotary", B=1, N=1, H=16, Hk=4, D=128, split="32,48,48", pairing="half", ladder="axis",
             dtype="fp16", pos="int64", t0=90000, packed=True, train=False),
        # queries and keys of a clip of 5 frames at 32 x 64 (the 1/32 level of 1024 x 2048), 8 heads of 32, views of the packed projection
        dict(name="rotary_clip", op="rotary", B=2, N=10240, H=8, Hk=8, D=32, split="8,12,12", pairing="adjacent", ladder="axis",
             dtype="bf16", pos="int64", t0=0, packed=True, train=False),
        # a training step of the same at 64 x 128 with wide heads: forward and gradient, part of each head left as it is
        dict(name="rotary_train", op="rotary", B=1, N=40960, H=16, Hk=4, D=128, split="32,32,32", pairing="half", ladder="shared",
             dtype="bf16", pos="int32", t0=17, packed=True, train=True),
        # ---- attention --------------------------------------------------------------------------------------------------------
        # slot self-attention of 8 clips x 5 frames in training: 100 slots, 8 heads of 32
        dict(name="attn_slots_train", op="attention", B=40, N=100, M=100, H=8, Hk=8, D=32, dtype="bf16", frame=0, window=0,
             qlens=False, klens=False, packed=True, train=True),
        # serving: one query per stream over its own memory of earlier frames, shared key heads, every stream at another length
        dict(name="attn_one_query", op="attention", B=5, N=1, M=16383, H=16, Hk=4, D=128, dtype="fp16", frame=0, window=0,
             qlens=False, klens=True, packed=False, train=False),
        # a clip of 5 frames x 2048 pixels: a pixel sees its own and earlier frames, at most three of them
        dict(name="attn_clip_frames", op="attention", B=1, N=10240, M=10240, H=8, Hk=8, D=64, dtype="bf16", frame=2048, window=3,
             qlens=False, klens=False, packed=True, train=False),
        # a training step over long ragged token sequences in causal order, four query heads to a key head
        dict(name="attn_long_train", op="attention", B=2, N=4097, M=4097, H=16, Hk=4, D=128, dtype="bf16", frame=1, window=0,
             qlens=True, klens=True, packed=False, train=True),
        # ---- dense layer ------------------------------------------------------------------------------------------------------
        # one token through a projection of the last Swin-L stage, residual added
        dict(name="dense_one_token", op="dense", M=1, K=1536, N=1536, act="none", bias=True, residual=True, dtype="fp16",
             train=False),
        # the slot feed-forward's first layer in training: 5 frames x 100 slots, 256 -> 2048, GELU
        dict(name="dense_slots_train", op="dense", M=500, K=256, N=2048, act="gelu", bias=True, residual=False, dtype="bf16",
             train=True),
        # fc1 of Swin-L's second stage over one 1024 x 2048 frame
        dict(name="dense_fc1", op="dense", M=32768, K=384, N=1536, act="gelu", bias=True, residual=False, dtype="bf16",
             train=False),
        # fc2 of the last stage over a clip of 5 frames in training, residual added
        dict(name="dense_fc2_train", op="dense", M=10240, K=6144, N=1536, act="none", bias=True, residual=True, dtype="bf16",
             train=True),
        # sizes that fill no tile: an odd number of tokens, odd widths
        dict(name="dense_odd", op="dense", M=7777, K=253, N=331, act="relu", bias=True, residual=True, dtype="fp16", train=False),
    ]


# ---- sizes drawn from the ranges of the listed cases --------------------------------------------------------------------------

def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "dense"])
    if op == "rotary":
        while True:
            D = rng.choice([32, 64, 80, 96, 128])
            axes = rng.randint(1, 4)
            split = [2 * rng.randint(1, max(1, D // (2 * axes))) for _ in range(axes)]
            Hk = rng.choice([1, 2, 3, 4, 8])
            c = dict(op=op, B=rng.randint(1, 3), N=_log(rng, 1, 40960), H=Hk * rng.choice([1, 2, 4]), Hk=Hk, D=D,
                     split=",".join(map(str, split)), pairing=rng.choice(["half", "adjacent"]), ladder=rng.choice(["axis", "shared"]),
                     dtype=rng.choice(["bf16", "fp16", "fp32"]), pos=rng.choice(["int64", "int32", "fp32"]),
                     t0=rng.choice([0, 17, 5000, 90000]), packed=rng.random() < 0.5, train=rng.random() < 0.5)
            if work(c)["bytes"] <= 700e6:
                return c
    if op == "attention":
        while True:
            Hk = rng.choice([1, 2, 3, 4, 8])
            N, M = _log(rng, 1, 10240), _log(rng, 1, 16383)
            if rng.random() < 0.5:
                M = N
            c = dict(op=op, B=_log(rng, 1, 40), N=N, M=M, H=Hk * rng.choice([1, 2, 4]), Hk=Hk, D=rng.choice([16, 32, 40, 64, 72, 96, 128]),
                     dtype=rng.choice(["bf16", "fp16"]), frame=rng.choice([0, 0, 1, 1, 100, 2048]), window=0, qlens=rng.random() < 0.3,
                     klens=rng.random() < 0.5, packed=M == N and rng.random() < 0.5, train=rng.random() < 0.5)
            if c["frame"] > 1:
                c["window"] = rng.choice([0, 1, 3])
            pairs = c["B"] * c["H"] * N * M
            if pairs * (2.5 if c["train"] else 1) <= 1.2e9:
                return c
    while True:
        c = dict(op="dense", M=_log(rng, 1, 32768), K=_log(rng, 16, 6144), N=_log(rng, 16, 6144), act=rng.choice(["none", "relu", "gelu"]),
                 bias=rng.random() < 0.8, residual=rng.random() < 0.5, dtype=rng.choice(["bf16", "fp16"]), train=rng.random() < 0.5)
        if rng.random() < 0.5:                                   # widths of networks are mostly multiples of 64, some are odd
            c["K"], c["N"] = max(64, c["K"] // 64 * 64), max(64, c["N"] // 64 * 64)
        if c["train"] and c["act"] == "relu":                    # relu's gradient jumps at zero: which side a sum next to it falls on is chance
            c["act"] = "gelu"
        if c["M"] * c["K"] * c["N"] * (3 if c["train"] else 1) <= 2.9e11:
            return c


# ---- what a program has in hand before the call -------------------------------------------------------------------------------

def _lens(case, which, n, top):
    """Lengths of a ragged batch: between a third of the longest and the longest, which is there once."""
    r = random.Random(f"{which}-{case['B']}-{top}")
    out = [r.randint(max(1, top // 3), top) for _ in range(n)]
    out[r.randrange(n)] = top
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=dev) * scale).to(dt)

    s = dict(case=case)
    if case["op"] == "rotary":
        B, N, H, Hk, D = (case[k] for k in ("B", "N", "H", "Hk", "D"))
        split = tuple(map(int, case["split"].split(",")))
        if case["packed"]:                                       # views of one projection's output [B, N, (H + 2 Hk) D]
            qkv = randn(B, N, H + 2 * Hk, D)
            s["q"], s["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        else:
            s["q"], s["k"] = randn(B, N, H, D), randn(B, N, Hk, D)
        s["pos"] = _positions(case, N, len(split), dev, seed)
        s["split"] = split
        if case["train"]:
            s["dq"], s["dk"] = randn(B, N, H, D), randn(B, N, Hk, D)
    elif case["op"] == "attention":
        B, N, M, H, Hk, D = (case[k] for k in ("B", "N", "M", "H", "Hk", "D"))
        if case["packed"]:
            qkv = randn(B, N, H + 2 * Hk, D)
            s["q"], s["k"], s["v"] = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
        else:
            s["q"], s["k"], s["v"] = randn(B, N, H, D), randn(B, M, Hk, D), randn(B, M, Hk, D)
        s["qlens"] = torch.tensor(_lens(case, "q", B, N), dtype=torch.int32, device=dev) if case["qlens"] else None
        s["klens"] = torch.tensor(_lens(case, "k", B, M), dtype=torch.int32, device=dev) if case["klens"] else None
        if case["train"]:
            s["dout"] = randn(B, N, H, D)
    else:
        M, K, N = case["M"], case["K"], case["N"]
        s["x"] = randn(M, K)
        s["w"] = ((torch.rand((N, K), generator=g, device=dev) * 2 - 1) * (3.0 / K) ** 0.5).to(dt)
        s["b"] = randn(N, scale=0.1) if case["bias"] else None
        s["r"] = randn(M, N) if case["residual"] else None
        if case["train"]:
            s["dy"] = randn(M, N)
    return s


def _positions(case, N, axes, dev, seed):
    """(frame, row, column, ...) of every token: columns fastest, frames from t0 on; times of a stream are fractions when float."""
    side = max(1, int(N ** (1.0 / (axes + 1))) + seed % 3)
    n = torch.arange(N, device=dev)
    cols = []
    for a in range(axes - 1):
        cols.append(n % side)
        n = n // side
    cols.append(n + case["t0"])
    pos = torch.stack(cols[::-1], dim=1)
    if case["pos"] == "fp32":
        return pos.float() * 0.5
    return pos.to(torch.int32) if case["pos"] == "int32" else pos


# ---- one pass -----------------------------------------------------------------------------------------------------------------

def run(state):
    return {"rotary": _rotary, "attention": _attention, "dense": _dense}[state["case"]["op"]](state)


def _rotary(s):
    c = s["case"]
    if own:
        from slotvps_amd import ops
        kw = dict(pairing=c["pairing"], ladder=c["ladder"])
        out = list(ops.rotary_axes(s["q"], s["pos"], s["split"], also=s["k"], **kw))
        if c["train"]:
            out += ops.rotary_axes_bwd(s["dq"], s["pos"], s["split"], also=s["dk"], **kw)
        return out
    R = sum(s["split"])
    half = R // 2
    axis, expo = [], []
    for a, d in enumerate(s["split"]):
        for i in range(d // 2):
            axis.append(a)
            expo.append(2.0 * i / d if c["ladder"] == "axis" else 2.0 * len(expo) / R)
    dev = s["q"].device
    freq = 10000.0 ** -torch.tensor(expo, dtype=torch.float64, device=dev)
    ang = s["pos"].double()[:, axis] * freq                      # [N, R/2]; far positions lose the angle in 32 bits
    cos, sin = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]

    def turn(x, sn):
        x32 = x.float()
        y = x32.clone()
        if c["pairing"] == "half":
            a, b = x32[..., :half], x32[..., half:R]
            y[..., :half], y[..., half:R] = a * cos - b * sn, b * cos + a * sn
        else:
            a, b = x32[..., 0:R:2], x32[..., 1:R:2]
            y[..., 0:R:2], y[..., 1:R:2] = a * cos - b * sn, b * cos + a * sn
        return y.to(x.dtype)

    out = [turn(s["q"], sin), turn(s["k"], sin)]
    if c["train"]:
        out += [turn(s["dq"], -sin), turn(s["dk"], -sin)]
    return out


def _attention(s):
    c = s["case"]
    if own:
        from slotvps_amd import ops
        kw = dict(q_lens=s["qlens"], k_lens=s["klens"], frame=c["frame"], window=c["window"])
        if not c["train"]:
            return ops.attention(s["q"], s["k"], s["v"], **kw)
        out, lse = ops.attention(s["q"], s["k"], s["v"], return_lse=True, **kw)
        return [out, *ops.attention_bwd(s["dout"], s["q"], s["k"], s["v"], out, lse, **kw)]
    q, k, v = s["q"], s["k"], s["v"]
    B, N, H, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = D ** -0.5
    i, j = torch.arange(N, device=q.device)[None], torch.arange(M, device=q.device)
    ql = (s["qlens"].long() if s["qlens"] is not None else torch.full((B,), N, device=q.device))[:, None]
    kl = (s["klens"].long() if s["klens"] is not None else torch.full((B,), M, device=q.device))[:, None]
    # the last query stands at the last key; a row sees [lo, hi)
    hi, lo = kl.expand(B, N), torch.zeros((B, N), dtype=torch.long, device=q.device)
    if c["frame"]:
        f = torch.div(i + kl - ql, c["frame"], rounding_mode="floor")
        hi = torch.minimum(hi, (f + 1) * c["frame"])
        if c["window"]:
            lo = (f - c["window"] + 1) * c["frame"]
    hi = torch.where(i < ql, hi, torch.zeros_like(hi))
    hide = ~((j >= lo[..., None]) & (j < hi[..., None]))                                               # [B, N, M]

    def heads(x, n):                                                                                   # -> [B Hk, rows, D]
        return x.float().transpose(1, 2).reshape(B * Hk, n, D)

    qh, kh, vh = heads(q, G * N), heads(k, M), heads(v, M)
    p = torch.bmm(qh, kh.transpose(1, 2).contiguous()).view(B, H, N, M).mul_(scale)
    p.masked_fill_(hide[:, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
    den = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(den > 0, den, torch.ones_like(den))).view(B * Hk, G * N, M)
    o = torch.bmm(p, vh)

    def back(x, n):                                                                                    # -> [B, n, heads, D]
        return x.view(B, -1, n, D).transpose(1, 2).to(q.dtype)

    if not c["train"]:
        return back(o, N)
    do = heads(torch.where((i < ql)[..., None, None], s["dout"].float(), 0.0), G * N)
    delta = (do * o).sum(-1, keepdim=True)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
    ds = torch.bmm(do, vh.transpose(1, 2).contiguous()).sub_(delta).mul_(p).mul_(scale)
    return [back(o, N), back(torch.bmm(ds, kh), N), back(torch.bmm(ds.transpose(1, 2).contiguous(), qh), M), back(dv, M)]


def _dense(s):
    c = s["case"]
    if own:
        from slotvps_amd import ops
        act = {"none": ops.ACT_NONE, "relu": ops.ACT_RELU, "gelu": ops.ACT_GELU}[c["act"]]
        if not c["train"]:
            return ops.linear_act(s["x"], s["w"], s["b"], act=act, residual=s["r"])
        y, gate = ops.linear_act(s["x"], s["w"], s["b"], act=act, residual=s["r"], return_gate=True)
        dx, dw, db = ops.linear_act_bwd(s["dy"], s["x"], s["w"], gate=gate, bias=s["b"])     # the residual's gradient is dy itself
        return [y, dx, dw] + ([db] if s["b"] is not None else [])
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    if c["act"] == "relu":
        y = z.clamp_min(0.0)
    elif c["act"] == "gelu":
        half = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        y = z * half
    else:
        y = z
    if s["r"] is not None:
        y = y + s["r"].float()
    y = y.to(s["x"].dtype)
    if not c["train"]:
        return y
    dz = s["dy"].float()
    if c["act"] == "relu":
        dz = dz * (z > 0)
    elif c["act"] == "gelu":
        dz = dz * (half + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5)
    out = [y, (dz @ w).to(y.dtype), (dz.t() @ x).to(y.dtype)]
    return out + ([dz.sum(0).to(y.dtype)] if s["b"] is not None else [])


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_attention(case, s) if case["op"] == "attention" else _exact_dense(case, s)


def _exact_rotary(case, s):
    """Every pair of channels as a complex number, times exp(+- i angle)."""
    R = sum(s["split"])
    first = [0]
    for d in s["split"]:
        first.append(first[-1] + d // 2)
    ang = torch.empty((s["pos"].shape[0], R // 2), dtype=torch.float64, device=s["q"].device)
    for a, d in enumerate(s["split"]):
        for i in range(d // 2):
            j = first[a] + i
            e = i / (d / 2) if case["ladder"] == "axis" else j / (R / 2)
            ang[:, j] = s["pos"][:, a].double() / 10000.0 ** e

    def turn(x, sign):
        x = x.double()
        body = x[..., :R]
        pair = body.unflatten(-1, (2, R // 2)).transpose(-1, -2) if case["pairing"] == "half" else body.unflatten(-1, (R // 2, 2))
        z = torch.view_as_complex(pair.contiguous()) * torch.polar(torch.ones_like(ang), sign * ang)[None, :, None]
        z = torch.view_as_real(z)
        z = z.transpose(-1, -2) if case["pairing"] == "half" else z
        return torch.cat([z.reshape(body.shape), x[..., R:]], -1)

    out = [turn(s["q"], 1.0), turn(s["k"], 1.0)]
    if case["train"]:
        out += [turn(s["dq"], -1.0), turn(s["dk"], -1.0)]
    return out


def _exact_attention(case, s):
    """One batch entry and query head at a time over its valid rows and keys only."""
    B, N, M, H, Hk, D = (case[k] for k in ("B", "N", "M", "H", "Hk", "D"))
    dev = s["q"].device
    z = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)
    out, dq, dk, dv = z(B, N, H, D), z(B, N, H, D), z(B, M, Hk, D), z(B, M, Hk, D)
    ql = s["qlens"].tolist() if s["qlens"] is not None else [N] * B
    kl = s["klens"].tolist() if s["klens"] is not None else [M] * B
    for b in range(B):
        n, m = ql[b], kl[b]
        place = torch.arange(n, device=dev) + (m - n)             # where a query stands among the keys
        key = torch.arange(m, device=dev)
        seen = torch.ones((n, m), dtype=torch.bool, device=dev)
        if case["frame"]:
            fq, fk = torch.floor(place.double() / case["frame"])[:, None], torch.floor(key.double() / case["frame"])[None]
            seen = fk <= fq
            if case["window"]:
                seen &= fq - fk < case["window"]
        some = seen.any(1, keepdim=True)
        for h in range(H):
            q, k, v = s["q"][b, :n, h].double(), s["k"][b, :m, h // (H // Hk)].double(), s["v"][b, :m, h // (H // Hk)].double()
            a = (q @ k.t()) / math.sqrt(D)
            a = torch.where(seen, a, torch.full_like(a, -math.inf))
            p = torch.where(some, torch.softmax(torch.where(some, a, torch.zeros_like(a)), -1), torch.zeros_like(a))
            o = p @ v
            out[b, :n, h] = o
            if case["train"]:
                do = s["dout"][b, :n, h].double()
                dv[b, :m, h // (H // Hk)] += p.t() @ do
                dp = do @ v.t()
                da = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, :n, h] = da @ k
                dk[b, :m, h // (H // Hk)] += da.t() @ q
    return [out, dq, dk, dv] if case["train"] else out


def _exact_dense(case, s):
    x, w = s["x"].double(), s["w"].double()
    z = torch.nn.functional.linear(x, w, None if s["b"] is None else s["b"].double())
    if case["act"] == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        y, slope = z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    elif case["act"] == "relu":
        y, slope = torch.relu(z), (z > 0).double()
    else:
        y, slope = z, torch.ones_like(z)
    if s["r"] is not None:
        y = y + s["r"].double()
    if not case["train"]:
        return y
    dz = s["dy"].double() * slope
    return [y, dz @ w, dz.t() @ x] + ([dz.sum(0)] if s["b"] is not None else [])


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        tok = case["B"] * case["N"]
        axes = case["split"].count(",") + 1
        heads = case["H"] + case["Hk"]
        once = 2 * tok * heads * case["D"] * size + case["N"] * axes * (8 if case["pos"] == "int64" else 4)
        rot = sum(map(int, case["split"].split(",")))
        times = 2 if case["train"] else 1
        return dict(bytes=times * once, flops=times * 3 * tok * heads * rot)
    if case["op"] == "attention":
        B, N, M, H, Hk, D = (case[k] for k in ("B", "N", "M", "H", "Hk", "D"))
        ql = _lens(case, "q", B, N) if case["qlens"] else [N] * B
        kl = _lens(case, "k", B, M) if case["klens"] else [M] * B
        pairs = 0
        for n, m in zip(ql, kl):
            if not case["frame"]:
                pairs += n * m
                continue
            f = case["frame"]
            for i in range(n):
                fr = (i + m - n) // f
                lo = max(0, (fr - case["window"] + 1) * f) if case["window"] else 0
                pairs += max(0, min(m, (fr + 1) * f) - lo)
        rows_q, rows_k = sum(ql) * H * D * size, sum(kl) * Hk * D * size
        if case["train"]:                                        # forward, then the backward pass with the scores computed again
            return dict(bytes=(2 * rows_q + 2 * rows_k) + (4 * rows_q + 4 * rows_k), flops=14 * pairs * H * D)
        return dict(bytes=2 * rows_q + 2 * rows_k, flops=4 * pairs * H * D)
    M, K, N = case["M"], case["K"], case["N"]
    x, w, y = M * K * size, N * K * size, M * N * size
    fwd = x + w + y + (y if case["residual"] else 0) + (N * size if case["bias"] else 0)
    if not case["train"]:
        return dict(bytes=fwd, flops=2 * M * N * K)
    gate = 2 * y if case["act"] != "none" else 0                 # the activation's slope, written and read back
    return dict(bytes=fwd + gate + y + 2 * x + 2 * w, flops=6 * M * N * K)
