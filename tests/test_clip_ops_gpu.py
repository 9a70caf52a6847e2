"""Clip-token operators (rotary_axes, attention, linear_act and their gradients) against plain 64-bit forms on the same inputs.

Tolerances, derived before the first run; u = eps / 2 of the type (half a step of its rounding), sums over the terms a rounding touches:
  rotary      u |y| + 2^-21 (|x1| + |x2|): sine and cosine to 2^-23 each, three fp32 roundings
  attention   out: the rounding of o, and every probability rounded once (u) after an fp32 exponent (2e-4 covers D 2^-24 sum |q k| scale
              for the inputs here): u |o| + (u + 2e-4) sum_j p |v|; fp16 adds 2^-25 sum |v| (probabilities below its normal range)
              dv:  u |dv| + (u + 2e-4) sum_i p |dO|, fp16 + 2^-25 sum |dO|
              dq, dk: every ds rounded once and p relative 2e-4, delta from the rounded output: e_i = sum_d |dO| (2 u + 2e-4) (p |v|)_d;
              u |dq| + scale sum_j ((u + 4e-4) |ds| + p (e_i + 1e-5 sum |dO v|)) |k|, fp16 + 2^-25 scale sum |k|; dk the same over i
  dense       z: 2 K 2^-24 sum |x w|; y: u |y| + 1.2 z-error + 2^-20 (|z| + |r|); gate in steps of 2^-14, dz rounded once:
              dx: u |dx| + u sum |dz w| + sum |dy| (2^-15 + 2^-20 + z-error) |w|, fp16 + 2^-25 sum |w|; dW alike; db: the gate's step
"""
import math

import pytest
import torch

from slotvps_amd import _lib, ops

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _u(dt):
    return torch.finfo(dt).eps / 2


def _sub(dt):
    return 2.0 ** -25 if dt == HF else 0.0


def _close(got, ref, tol, what):
    got = got.double()
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    bad = (got - ref).abs() - tol
    assert (bad <= 0).all(), f"{what}: off by {float((got - ref).abs().max()):.3e}, over the tolerance by {float(bad.max()):.3e} at {int(bad.argmax())}"


def _rand(shape, dt, seed, dev, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dt)


# ---- rotary -------------------------------------------------------------------------------------------------------------------

def _rotary_ref(x, pos, split, base, pairing, ladder, sign):
    R = sum(split)
    f, ax = [], []
    for a, d in enumerate(split):
        for i in range(d // 2):
            f.append(base ** -(2.0 * i / d if ladder == "axis" else 2.0 * len(f) / R))
            ax.append(a)
    pos = pos.double() if pos.dim() == 3 else pos.double()[None]
    ang = pos[:, :, ax] * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = ang.cos()[:, :, None], sign * ang.sin()[:, :, None]
    x = x.double()
    y, mag = x.clone(), torch.zeros_like(x)
    ia = torch.arange(R // 2, device=x.device) if pairing == "half" else torch.arange(0, R, 2, device=x.device)
    ib = ia + (R // 2 if pairing == "half" else 1)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    return y, mag


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("B,N,H,H2,D,split,pairing,ladder,ptype", [
    (1, 1, 16, 4, 128, (32, 48, 48), "half", "axis", torch.int64),
    (2, 37, 8, 8, 32, (8, 12, 12), "adjacent", "axis", torch.int32),
    (1, 515, 3, 1, 80, (16, 16, 16, 32), "half", "shared", F32),
    (3, 5, 2, 0, 24, (6, 10), "half", "axis", torch.int64),        # sections that fill no 16-byte access
    (1, 9, 1, 2, 33, (2,), "adjacent", "shared", torch.int32),     # odd head size
    (1, 4100, 2, 1, 64, (64,), "adjacent", "axis", torch.int64),
])
def test_rotary_axes(cuda, dt, B, N, H, H2, D, split, pairing, ladder, ptype):
    x, k = _rand((B, N, H, D), dt, 1, cuda), (_rand((B, N, H2, D), dt, 2, cuda) if H2 else None)
    g = torch.Generator(device=cuda).manual_seed(3)
    pos = torch.randint(-3000, 1_000_000, (N, len(split)), generator=g, device=cuda).to(ptype)
    if B > 1:
        pos = torch.stack([pos + 7 * b for b in range(B)])
    for sign, fn in ((1.0, ops.rotary_axes), (-1.0, ops.rotary_axes_bwd)):
        got = fn(x, pos, split, pairing=pairing, ladder=ladder, also=k)
        got = got if k is not None else (got,)
        for t, y in zip((x, k), got):
            ref, mag = _rotary_ref(t, pos, split, 10000.0, pairing, ladder, sign)
            _close(y, ref, _u(dt) * ref.abs() + 2.0 ** -21 * mag + 1e-12 + _sub(dt) , f"rotary sign {sign}")
            assert y.is_contiguous()
            R = sum(split)
            assert torch.equal(y[..., R:], t[..., R:])


def test_rotary_far_positions_strides_and_turning_back(cuda):
    qkv = _rand((2, 50, 12, 64), F32, 5, cuda)
    q, k = qkv[:, :, :8], qkv[:, ::1, 8:10]
    pos = torch.stack([torch.arange(50, device=cuda) + 2 ** 31 + 11, torch.arange(50, device=cuda) * -40000], 1)
    a, b = ops.rotary_axes(q, pos, (32, 16), base=500.0, also=k)
    for t, y in ((q, a), (k, b)):
        ref, mag = _rotary_ref(t, pos, (32, 16), 500.0, "half", "axis", 1.0)
        # p f at 2^31 holds 2^-53 2^31 / 2 pi turns: 2.4e-7 radians on top
        _close(y, ref, _u(F32) * ref.abs() + (2.0 ** -21 + 1e-6) * mag, "far positions")
    back = ops.rotary_axes_bwd(a, pos, (32, 16), base=500.0)
    assert (back - q).abs().max() < 1e-5 * q.abs().max()
    # a transposed head axis, a row taken from every second token, broadcast tokens
    xt = _rand((2, 8, 50, 64), F32, 6, cuda).transpose(1, 2)
    assert torch.equal(ops.rotary_axes(xt, pos, (32, 16)), ops.rotary_axes(xt.contiguous(), pos, (32, 16)))
    xe = q[:, :1].expand(2, 50, 8, 64)
    assert torch.equal(ops.rotary_axes(xe, pos, (32, 16)), ops.rotary_axes(xe.contiguous(), pos, (32, 16)))
    un = torch.empty(2 * 50 * 8 * 64 + 1, device=cuda)[1:].view(2, 50, 8, 64).copy_(q)      # 4-byte aligned only
    assert torch.equal(ops.rotary_axes(un, pos, (32, 16)), ops.rotary_axes(q, pos, (32, 16)))
    assert ops.rotary_axes(q[:, :0], pos[:0], (32, 16)).shape == (2, 0, 8, 64)


def test_rotary_autograd(cuda):
    x, k = _rand((1, 7, 3, 16), F32, 1, cuda).requires_grad_(), _rand((1, 7, 1, 16), F32, 2, cuda).requires_grad_()
    pos = torch.arange(14, device=cuda).view(7, 2)
    w, w2 = _rand((1, 7, 3, 16), F32, 3, cuda), _rand((1, 7, 1, 16), F32, 4, cuda)

    def loss():
        a, b = ops.rotary_axes(x, pos, (8, 8), also=k, pairing="adjacent")
        return (a * a * w).sum() + (b * w2).sum()
    gx, gk = torch.autograd.grad(loss(), (x, k))
    for t, gr in ((x, gx), (k, gk)):
        for idx in (0, 5, t.numel() - 1):
            with torch.no_grad():
                f = []
                for e in (1e-2, -1e-2):
                    t.view(-1)[idx] += e
                    f.append(float(loss().double()))
                    t.view(-1)[idx] -= e
            # central difference of a quadratic is exact up to fp32 sums of ~70 values of size ~3: 70 * 3 * 2^-22 / 2e-2 < 3e-3
            assert abs((f[0] - f[1]) / 2e-2 - float(gr.reshape(-1)[idx])) < 5e-3


# ---- attention ----------------------------------------------------------------------------------------------------------------

def _visible(N, M, ql, kl, frame, window, dev):
    i, j = torch.arange(N, device=dev)[:, None], torch.arange(M, device=dev)[None]
    ok = (i < ql) & (j < kl)
    if frame:
        fq, fk = torch.div(i + kl - ql, frame, rounding_mode="floor"), torch.div(j, frame, rounding_mode="floor")
        ok = ok & (fk <= fq)
        if window:
            ok = ok & (fk > fq - window)
    return ok


def _attention_ref(q, k, v, do, ql, kl, frame, window, scale, dt):
    """values and tolerances in float64; garbage behind the lengths is cut off first"""
    B, N, H, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    dev, u, sb = q.device, _u(dt), _sub(dt)
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device=dev)
    out, lse = z(B, N, H, D), torch.full((B, H, N), -math.inf, dtype=torch.float64, device=dev)
    dq, dk, dv = z(B, N, H, D), z(B, M, Hk, D), z(B, M, Hk, D)
    to, tq, tk, tv = z(B, N, H, D), z(B, N, H, D), z(B, M, Hk, D), z(B, M, Hk, D)
    for b in range(B):
        ok = _visible(N, M, ql[b], kl[b], frame, window, dev)
        row, col = (torch.arange(N, device=dev) < ql[b])[:, None], (torch.arange(M, device=dev) < kl[b])[:, None]
        for h in range(H):
            g = h // (H // Hk)
            cut = lambda t, m: torch.where(m, t.double(), torch.zeros((), dtype=torch.float64, device=dev))
            qq, kk, vv = cut(q[b, :, h], row), cut(k[b, :, g], col), cut(v[b, :, g], col)
            s = (qq @ kk.t() * scale).masked_fill(~ok, -math.inf)
            some = ok.any(1)
            l = torch.logsumexp(s, 1)
            p = torch.where(some[:, None], torch.exp(s - torch.where(some, l, 0.0)[:, None]), 0.0)
            lse[b, h] = torch.where(some, l, -math.inf)
            o = p @ vv
            pv = p @ vv.abs()
            out[b, :, h] = o
            to[b, :, h] = u * o.abs() + (u + 2e-4) * pv + sb * (ok.double() @ vv.abs()) + 1e-30
            if do is None:
                continue
            d = cut(do[b, :, h], row)
            dp = d @ vv.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            e = (d.abs() * (2 * u + 2e-4) * pv).sum(1, keepdim=True) + 1e-5 * (d.abs() @ vv.abs().t())
            es = (u + 4e-4) * ds.abs() + p * e + sb * ok
            dq[b, :, h] = scale * ds @ kk
            tq[b, :, h] = u * dq[b, :, h].abs() + scale * es @ kk.abs() + 1e-30
            dk[b, :, g] += scale * ds.t() @ qq
            tk[b, :, g] += scale * es.t() @ qq.abs() + 1e-30
            dv[b, :, g] += p.t() @ d
            tv[b, :, g] += (u + 2e-4) * (p.t() @ d.abs()) + sb * (ok.double().t() @ d.abs()) + 1e-30
    tk += u * dk.abs()
    tv += u * dv.abs()
    return (out, lse, dq, dk, dv), (to, tq, tk, tv)


def _lens(x, n, top, dev):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)


ATT = [  # B, N, M, H, Hk, D, frame, window, qlens, klens
    (2, 100, 100, 8, 8, 32, 0, 0, None, None),
    (1, 1, 1, 1, 1, 8, 0, 0, None, None),
    (3, 1, 2000, 4, 1, 128, 0, 0, None, [2000, 1, 0]),              # single queries, one memory empty; split over the keys
    (2, 5, 777, 6, 2, 64, 1, 0, None, [700, 3]),                    # new tokens of a stream, fewer keys than queries once
    (1, 300, 300, 4, 2, 128, 1, 0, None, None),
    (1, 257, 257, 2, 1, 64, 50, 2, None, None),                     # frames of 50, two visible
    (2, 130, 260, 3, 3, 40, 7, 0, [130, 13], [260, 64]),
    (2, 64, 65, 2, 2, 16, 0, 0, [0, 64], [65, 65]),                 # an entry without queries
    (1, 200, 90, 2, 2, 72, 1, 0, None, None),                       # more queries than keys: the first rows see nothing
    (1, 33, 129, 5, 5, 96, 1, 3, None, None),                       # a window of three keys
    (1, 700, 31, 8, 1, 128, 0, 0, None, None),                      # eight heads on one key head, few keys: rows split in the backward
]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("case", ATT)
def test_attention_forward_and_gradients(cuda, dt, case):
    B, N, M, H, Hk, D, frame, window, ql, kl = case
    q, k, v, do = _rand((B, N, H, D), dt, 1, cuda), _rand((B, M, Hk, D), dt, 2, cuda), _rand((B, M, Hk, D), dt, 3, cuda), _rand((B, N, H, D), dt, 4, cuda)
    qt, kt = _lens(ql, B, N, cuda), _lens(kl, B, M, cuda)
    qv, kv = ql or [N] * B, kl or [M] * B
    for b in range(B):                                               # what stands behind a length takes no part, whatever it is
        q[b, qv[b]:], do[b, qv[b]:], k[b, kv[b]:], v[b, kv[b]:] = math.nan, math.inf, math.nan, -math.inf
    kw = dict(q_lens=qt, k_lens=kt, frame=frame, window=window)
    out, lse = ops.attention(q, k, v, return_lse=True, **kw)
    ref, tol = _attention_ref(q, k, v, do, qv, kv, frame, window, D ** -0.5, dt)
    _close(out, ref[0], tol[0], "out")
    none = torch.isinf(ref[1])
    assert torch.equal(torch.isinf(lse), none)
    assert (lse.double() - ref[1])[~none].abs().max() < 1e-3 if (~none).any() else True
    assert torch.equal(out, ops.attention(q, k, v, **kw))
    got = ops.attention_bwd(do, q, k, v, out, lse, **kw)
    for name, a, r, t in zip(("dq", "dk", "dv"), got, ref[2:], tol[1:]):
        _close(a, r, t, name)
    again = ops.attention_bwd(do, q, k, v, out, lse, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_attention_long_and_split(cuda):
    """Lengths past several tiles and splits on either side, large scores included (a row that puts all its weight on one key)."""
    B, N, M, H, Hk, D, dt = 1, 1000, 3001, 2, 1, 64, BF
    q, k, v, do = _rand((B, N, H, D), dt, 1, cuda, 6.0), _rand((B, M, Hk, D), dt, 2, cuda, 6.0), _rand((B, M, Hk, D), dt, 3, cuda), _rand((B, N, H, D), dt, 4, cuda)
    q[:, 5] = 0                                                      # equal weights
    out, lse = ops.attention(q, k, v, return_lse=True)
    # scores of ~36 sqrt(64): sum |q k| scale up to ~ 64 * 25 / 8 = 200, times D 2^-24 = 7.6e-4 relative in p; the products' 2e-4 times 4
    ref, tol = _attention_ref(q, k, v, do, [N], [M], 0, 0, D ** -0.5, dt)
    _close(out, ref[0], 4 * tol[0], "out")
    for name, a, r, t in zip(("dq", "dk", "dv"), ops.attention_bwd(do, q, k, v, out, lse), ref[2:], tol[1:]):
        _close(a, r, 4 * t, name)


@pytest.mark.parametrize("frame,window", [(0, 0), (1, 0), (50, 2)])
@pytest.mark.parametrize("D", [64, 40])
def test_attention_of_many_full_workgroups(cuda, D, frame, window):
    """Batches whose rows fill workgroups of 256 rows on every compute unit, with rows and keys behind the lengths."""
    B, N, M, H, Hk = 32, 250, 203, 16, 8
    ql, kl = [N - 3 * b for b in range(B)], [M - 5 * b for b in range(B)]
    q, k, v, do = _rand((B, N, H, D), BF, 1, cuda), _rand((B, M, Hk, D), BF, 2, cuda), _rand((B, M, Hk, D), BF, 3, cuda), _rand((B, N, H, D), BF, 4, cuda)
    for b in range(B):
        q[b, ql[b]:], do[b, ql[b]:], k[b, kl[b]:], v[b, kl[b]:] = math.nan, math.inf, math.nan, -math.inf
    kw = dict(q_lens=_lens(ql, B, N, cuda), k_lens=_lens(kl, B, M, cuda), frame=frame, window=window)
    out, lse = ops.attention(q, k, v, return_lse=True, **kw)
    ref, tol = _attention_ref(q, k, v, do, ql, kl, frame, window, D ** -0.5, BF)
    _close(out, ref[0], tol[0], "out")
    none = torch.isinf(ref[1])
    assert torch.equal(torch.isinf(lse), none) and (lse.double() - ref[1])[~none].abs().max() < 1e-3
    for name, a, r, t in zip(("dq", "dk", "dv"), ops.attention_bwd(do, q, k, v, out, lse, **kw), ref[2:], tol[1:]):
        _close(a, r, t, name)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("N,M,H,Hk,D,frame,window", [(5, 5, 4, 2, 64, 1, 0), (70, 1, 2, 2, 32, 0, 0), (200, 200, 4, 1, 128, 1, 1), (33, 90, 3, 3, 40, 1, 1)])
def test_attention_gradient_of_one_visible_key(cuda, N, M, H, Hk, D, frame, window, dt):
    """A row that sees a single key has p = 1 whatever q and k are: its dS, and so its dQ, is zero but for fp32 rounding.
    |dS| <= p |dP - delta|: dP and delta are D fp32 additions of the same products, 2 D 2^-24 S with S = sum_d |dO_d v_d|, and p is off by
    2^-19 at |s| < 8 (three roundings of a number below 16 in front of exp2): together below (2 D + 32) 2^-24 S, times 1 + 2^-6 for the
    roundings of dS and dQ to 16 bits. fp16 cannot hold less than 2^-25 of either."""
    B = 2
    q, k, v, do = _rand((B, N, H, D), dt, 41, cuda), _rand((B, M, Hk, D), dt, 42, cuda), _rand((B, M, Hk, D), dt, 43, cuda), _rand((B, N, H, D), dt, 44, cuda)
    out, lse = ops.attention(q, k, v, frame=frame, window=window, return_lse=True)
    dq = ops.attention_bwd(do, q, k, v, out, lse, frame=frame, window=window)[0]
    for n in range(N):
        one = n + M - N if frame else 0                                    # the only key that row n sees, if it does see only one
        if (window != 1 and M > 1 and one != 0) or one < 0:
            continue
        kk, vv = k[:, one].repeat_interleave(H // Hk, 1).double(), v[:, one].repeat_interleave(H // Hk, 1).double()
        assert (q[:, n].double() * kk).sum(-1).abs().max() * D ** -0.5 < 8
        S = (do[:, n].double() * vv).abs().sum(-1, keepdim=True)
        tol = (2 * D + 32) * 2.0 ** -24 * S * D ** -0.5 * kk.abs() * (1 + 2.0 ** -6) + 2.0 ** -25 * (1 + kk.abs())
        assert (dq[:, n].double().abs() <= tol).all(), f"token {n}: {float((dq[:, n].double().abs() - tol).max()):.3e} over"


def test_attention_views_strides_and_broadcast(cuda):
    B, N, H, Hk, D = 2, 70, 4, 2, 64
    qkv = _rand((B, N, H + 2 * Hk, D), BF, 1, cuda)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), frame=1)
    assert torch.equal(ops.attention(q, k, v, frame=1), want)
    qt, kt = q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.attention(qt, kt, v, frame=1), want)
    odd = _rand((B, N, H + 2 * Hk, D + 3), BF, 1, cuda)              # rows that do not start on 16 bytes
    qo, ko, vo = odd[:, :, :H, 3:], odd[:, :, H:H + Hk, 1:D + 1], odd[:, :, H + Hk:, :D]
    ref = ops.attention(qo.contiguous(), ko.contiguous(), vo.contiguous())
    assert torch.equal(ops.attention(qo, ko, vo), ref)
    # one memory for the whole batch, by stride 0; its gradient sums over the batch
    k1, v1 = k[:1].detach().contiguous().requires_grad_(), v[:1].detach().contiguous().requires_grad_()
    ke, ve = k1.expand(B, N, Hk, D), v1.expand(B, N, Hk, D)
    out = ops.attention(q, ke, ve)
    do = _rand(out.shape, BF, 9, cuda)
    gk, gv = torch.autograd.grad(out, (k1, v1), do)
    o2, lse = ops.attention(q, ke.detach().contiguous(), ve.detach().contiguous(), return_lse=True)
    assert torch.equal(out, o2)
    _, dk, dv = ops.attention_bwd(do, q, ke.detach(), ve.detach(), o2, lse)
    assert (gk - dk.float().sum(0, keepdim=True)).abs().max() <= 2 ** -7 * dk.float().abs().sum(0).max()
    assert (gv - dv.float().sum(0, keepdim=True)).abs().max() <= 2 ** -7 * dv.float().abs().sum(0).max()


def test_attention_empty(cuda):
    q, k = torch.ones((2, 3, 2, 16), dtype=BF, device=cuda), torch.ones((2, 0, 2, 16), dtype=BF, device=cuda)
    out, lse = ops.attention(q, k, k, return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    dq, dk, dv = ops.attention_bwd(q, q, k, k, out, lse)
    assert not dq.any() and dk.shape == dv.shape == k.shape
    assert ops.attention(q[:, :0], q, q).shape == (2, 0, 2, 16)
    assert ops.attention(q[:0], q[:0], q[:0]).shape == (0, 3, 2, 16)


def test_attention_autograd_matches_differences(cuda):
    """The gradient against differences of the 64-bit formula it belongs to (16-bit inputs cannot be stepped finely enough themselves)."""
    q, k, v = (_rand((1, 6, 2, 16), HF, s, cuda) for s in (1, 2, 3))
    w = _rand((1, 6, 2, 16), HF, 4, cuda)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*leaves, frame=1), leaves, w)

    def loss(q, k, v):
        return float((_attention_ref(q, k, v, None, [6], [6], 1, 0, 0.25, HF)[0][0] * w.double()).sum())
    x = [t.double() for t in (q, k, v)]
    for n in range(3):
        for idx in (0, 37, 100, 191):
            f = []
            for e in (1e-5, -1e-5):
                y = [t.clone() for t in x]
                y[n].view(-1)[idx] += e
                f.append(loss(*y))
            diff = (f[0] - f[1]) / 2e-5
            # half steps: output, ds, p, delta: each at most 2^-11 of sums of six terms of size <= |w| |v| ~ 10
            assert abs(diff - float(grads[n].reshape(-1)[idx])) < 4 * 2 ** -11 * 10 + 1e-4


# ---- dense layer --------------------------------------------------------------------------------------------------------------

def _act64(z, act):
    if act == ops.ACT_RELU:
        return z.clamp_min(0), (z > 0).double()
    if act == ops.ACT_GELU:
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


DENSE = [  # M, K, N, act, bias, residual
    (1, 256, 256, ops.ACT_NONE, True, True),
    (1, 1, 1, ops.ACT_GELU, True, False),
    (500, 256, 2048, ops.ACT_GELU, True, False),
    (130, 2048, 256, ops.ACT_NONE, True, True),
    (77, 253, 331, ops.ACT_GELU, True, True),
    (300, 40, 72, ops.ACT_RELU, False, True),
    (129, 129, 130, ops.ACT_NONE, False, False),
    (5, 1536, 1000, ops.ACT_GELU, True, True),
    (3000, 64, 33, ops.ACT_GELU, True, False),
    (513, 700, 515, ops.ACT_RELU, True, False),
]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("case", DENSE)
def test_linear_act_forward_and_gradients(cuda, dt, case):
    M, K, N, act, has_b, has_r = case
    u, sb = _u(dt), _sub(dt)
    x, w = _rand((M, K), dt, 1, cuda), _rand((N, K), dt, 2, cuda, K ** -0.5)
    b = _rand((N,), dt if M % 2 else F32, 3, cuda) if has_b else None
    r = _rand((M, N), dt, 4, cuda) if has_r else None
    dy = _rand((M, N), dt, 5, cuda)
    if act == ops.ACT_RELU:                                          # sums of small integers are exact: no value can fall on the wrong side of zero
        x, w = x.mul(2).round(), (w * K ** 0.5 * 2).round() / 8
        b = None if b is None else b.mul(4).round() / 8 + 1 / 16
    y, gate = ops.linear_act(x, w, b, act=act, residual=r, return_gate=True)
    xd, wd = x.double(), w.double()
    z = xd @ wd.t() + (0 if b is None else b.double())
    ez = 2 * (K + 1) * 2.0 ** -24 * (xd.abs() @ wd.abs().t() + (0 if b is None else b.double().abs()))
    a, slope = _act64(z, act)
    ref = a + (0 if r is None else r.double())
    _close(y, ref, u * ref.abs() + 1.2 * ez + 2.0 ** -20 * (z.abs() + (0 if r is None else r.double().abs())) + sb, "y")
    assert torch.equal(y, ops.linear_act(x, w, b, act=act, residual=r))
    if act == ops.ACT_NONE:
        assert gate is None
    else:
        ezg = ez * (act == ops.ACT_GELU) + (2.0 ** -20 if act == ops.ACT_GELU else 0.0)
        assert gate.dtype == torch.int16
        _close(gate.double() / 2 ** 14, slope, 2.0 ** -15 + ezg, "gate")
    dx, dw, db = ops.linear_act_bwd(dy, x, w, gate=gate, bias=b)
    dyd = dy.double()
    dz = dyd * slope
    # the gate's step and one rounding of dz (none of either without an activation: dz is dy)
    eg = dyd.abs() * ((ez if act == ops.ACT_GELU else 0) + 2.0 ** -20 + 2.0 ** -15)
    edz = (dz.abs() + eg) * u + eg + sb if act != ops.ACT_NONE else torch.zeros_like(dz)
    rx, rw = dz @ wd, dz.t() @ xd
    _close(dx, rx, u * rx.abs() + edz @ wd.abs() + 2 * N * 2.0 ** -24 * (dz.abs() @ wd.abs()) + sb, "dx")
    _close(dw, rw, u * rw.abs() + edz.t() @ xd.abs() + 2 * M * 2.0 ** -24 * (dz.t().abs() @ xd.abs()) + sb, "dw")
    if has_b:
        rb = dz.sum(0)
        assert db.dtype == b.dtype
        _close(db, rb, _u(b.dtype) * rb.abs() + (eg.sum(0) if act != ops.ACT_NONE else 0) + 2 * M * 2.0 ** -24 * dz.abs().sum(0) + sb, "db")
    else:
        assert db is None
    again = ops.linear_act_bwd(dy, x, w, gate=gate, bias=b)
    assert all(p is None or torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_linear_act_views_autograd_and_parts(cuda):
    big = _rand((4, 30, 96), BF, 1, cuda)
    x = big[:, :, 16:80]                                             # rows of 64 inside rows of 96
    w, b = _rand((48, 64), BF, 2, cuda, 0.1), _rand((48,), BF, 3, cuda)
    r = _rand((4, 30, 48), BF, 4, cuda)
    want = ops.linear_act(x.contiguous(), w, b, act=ops.ACT_GELU, residual=r)
    assert want.shape == (4, 30, 48) and torch.equal(ops.linear_act(x, w, b, act=ops.ACT_GELU, residual=r), want)
    wt = w.t().contiguous().t()                                      # column-major weight
    assert torch.equal(ops.linear_act(x, wt, b, act=ops.ACT_GELU, residual=r), want)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b, r)]
    y = ops.linear_act(leaves[0], leaves[1], leaves[2], act=ops.ACT_GELU, residual=leaves[3])
    dy = _rand(y.shape, BF, 5, cuda)
    grads = torch.autograd.grad(y, leaves, dy)
    _, gate = ops.linear_act(x, w, b, act=ops.ACT_GELU, residual=r, return_gate=True)
    dx, dw, db = ops.linear_act_bwd(dy, x, w, gate=gate, bias=b)
    for g, e in zip(grads, (dx, dw, db, dy)):
        assert torch.equal(g, e)
    only = ops.linear_act_bwd(dy, x, w, gate=gate, want_dw=False)
    assert only[1] is None and only[2] is None and torch.equal(only[0], dx)
    only = ops.linear_act_bwd(dy, x, w, gate=gate, bias=b, want_dx=False, want_dw=False)
    assert only[:2] == (None, None) and torch.equal(only[2], db)
    (g,) = torch.autograd.grad(ops.linear_act(leaves[0], w).sum(), leaves[0])       # an expanded gradient, only one input asks
    assert torch.equal(g, ops.linear_act_bwd(torch.ones_like(y), x, w)[0])
    assert ops.linear_act(x[:0], w, b).shape == (0, 30, 48)
    e = ops.linear_act_bwd(dy[:0], x[:0], w, bias=b)
    assert e[0].shape == (0, 30, 64) and not e[1].any() and not e[2].any()


# ---- together -----------------------------------------------------------------------------------------------------------------

def _layer(p, x, pos, klens, H, Hk, D):
    """one transformer layer over clip tokens: projection, rotation, attention, projection + residual, feed-forward + residual"""
    B, N, C = x.shape
    qkv = ops.linear_act(x, p["wqkv"], p["bqkv"]).view(B, N, H + 2 * Hk, D)
    q, k = ops.rotary_axes(qkv[:, :, :H], pos, (8, 12, 12), also=qkv[:, :, H:H + Hk])
    o = ops.attention(q, k, qkv[:, :, H + Hk:], q_lens=klens, k_lens=klens, frame=20, window=2)
    x = ops.linear_act(o.reshape(B, N, H * D), p["wo"], p["bo"], residual=x)
    h = ops.linear_act(x, p["w1"], p["b1"], act=ops.ACT_GELU)
    return ops.linear_act(h, p["w2"], p["b2"], residual=x)


def _layer64(p, x, pos, klens, H, Hk, D):
    lin = torch.nn.functional.linear
    B, N, C = x.shape
    qkv = lin(x, p["wqkv"], p["bqkv"]).view(B, N, H + 2 * Hk, D)
    rot = lambda t: _rotary_diff(t, pos)
    q, k, v = rot(qkv[:, :, :H]), rot(qkv[:, :, H:H + Hk]), qkv[:, :, H + Hk:]
    k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    s = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * D ** -0.5
    ok = torch.stack([_visible(N, N, n, n, 20, 2, x.device) for n in klens])[:, None]
    p_ = torch.where(ok, torch.softmax(torch.where(ok, s, -1e30), -1), 0.0)
    o = torch.matmul(p_, v.transpose(1, 2)).transpose(1, 2).reshape(B, N, H * D)
    x = lin(o, p["wo"], p["bo"]) + x
    return lin(torch.nn.functional.gelu(lin(x, p["w1"], p["b1"])), p["w2"], p["b2"]) + x


def _rotary_diff(x, pos):
    f, ax = [], []
    for a, d in enumerate((8, 12, 12)):
        for i in range(d // 2):
            f.append(10000.0 ** -(2.0 * i / d))
            ax.append(a)
    ang = pos.double()[:, ax] * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
    a, b = x[..., :16], x[..., 16:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _layer_inputs(dev, dt=BF):
    H, Hk, D, C, B, N = 8, 4, 32, 256, 2, 100
    shapes = dict(wqkv=((H + 2 * Hk) * D, C), bqkv=((H + 2 * Hk) * D,), wo=(C, H * D), bo=(C,), w1=(2048, C), b1=(2048,), w2=(C, 2048), b2=(C,))
    p = {n: _rand(s, dt, 10 + i, dev, s[1] ** -0.5 if len(s) == 2 else 0.1) for i, (n, s) in enumerate(shapes.items())}
    x, dy = _rand((B, N, C), dt, 1, dev), _rand((B, N, C), dt, 2, dev)
    n = torch.arange(N, device=dev)
    pos = torch.stack([n // 20 + 5000, n % 20 // 5, n % 5], 1)
    return p, x, dy, pos, torch.tensor([100, 57], dtype=torch.int32, device=dev), (H, Hk, D)


def test_a_layer_of_them_together(cuda):
    p, x, dy, pos, lens, dims = _layer_inputs(cuda)
    leaves = {n: t.clone().requires_grad_() for n, t in p.items()}
    xl = x.clone().requires_grad_()
    names = list(leaves)
    y = _layer(leaves, xl, pos, lens, *dims)
    grads = torch.autograd.grad(y, [xl] + [leaves[n] for n in names], dy)
    ld = {n: t.double().requires_grad_() for n, t in p.items()}
    xd = x.double().requires_grad_()
    yd = _layer64(ld, xd, pos, lens.tolist(), *dims)
    gd = torch.autograd.grad(yd, [xd] + [ld[n] for n in names], dy.double())
    # six roundings to bf16 follow one another on the way up, about twice that on the way down; each is off by u / sqrt(3) of the value in
    # the mean, so relative to the tensor's rms the error stays below sqrt(12) u ~ 1.4e-2; 2e-2 leaves the products' mixing room
    for name, a, r in zip(["y", "x"] + names, (y, *grads), (yd, *gd)):
        err = (a.double() - r).pow(2).mean().sqrt() / r.pow(2).mean().sqrt()
        assert err < 2e-2, f"{name}: {float(err):.3e}"


def test_captured_step_replays(cuda):
    """forward and plain gradients in one HIP graph, replayed with other inputs and eager work between; a second graph beside it."""
    p, x, dy, pos, lens, (H, Hk, D) = _layer_inputs(cuda)
    mem = _rand((2, 4000, Hk, D), BF, 30, cuda)
    mlens = torch.tensor([4000, 2900], dtype=torch.int32, device=cuda)

    def step(x, mlens):
        B, N, C = x.shape
        qkv, _ = ops.linear_act(x, p["wqkv"], p["bqkv"], return_gate=True)
        qkv = qkv.view(B, N, H + 2 * Hk, D)
        q, k = ops.rotary_axes(qkv[:, :, :H], pos, (8, 12, 12), also=qkv[:, :, H:H + Hk])
        v = qkv[:, :, H + Hk:]
        o, lse = ops.attention(q, k, v, frame=20, return_lse=True)
        one = ops.attention(q[:, -1:], mem, mem, k_lens=mlens)                       # split over the keys: workspace inside the graph
        h, gate = ops.linear_act(o.reshape(B, N, H * D), p["w1"], p["b1"], act=ops.ACT_GELU, return_gate=True)
        dh, dw1, db1 = ops.linear_act_bwd(h, o.reshape(B, N, H * D), p["w1"], gate=gate, bias=p["b1"])
        dq, dk, dv = ops.attention_bwd(dh.view(B, N, H, D), q, k, v, o, lse, frame=20)
        dq, dk = ops.rotary_axes_bwd(dq, pos, (8, 12, 12), also=dk)
        dx, dw, _ = ops.linear_act_bwd(torch.cat([dq, dk, dv], 2).view(B, N, -1), x, p["wqkv"])
        return [one, h, dw1, db1, dx, dw]

    graphs = []
    for s in range(2):
        xs, ls = x.clone(), mlens.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(xs, ls)
        torch.cuda.current_stream().wait_stream(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(xs, ls)
        graphs.append((g, xs, ls, res))
    for it in range(4):
        for s, (g, xs, ls, res) in enumerate(graphs):
            xs.copy_(_rand(x.shape, BF, 100 + 10 * it + s, cuda))
            ls.copy_(torch.tensor([4000 - 700 * it, 1 + 900 * s + it], dtype=torch.int32, device=cuda))
            g.replay()
        torch.cuda.synchronize()
        for g, xs, ls, res in graphs:
            for a, b in zip(res, step(xs, ls)):
                assert torch.equal(a, b)


def test_autograd_in_a_capture_is_refused(cuda):
    x = _rand((4, 64), BF, 1, cuda).requires_grad_()
    w = _rand((64, 64), BF, 2, cuda)
    alive = ops.linear_act(x, w).sum()                               # an eager graph of the same leaf
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(g):
            y = ops.linear_act(x, w)
            torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.synchronize()
    alive.backward()
    assert x.grad is not None


def test_other_stream(cuda):
    s = torch.cuda.Stream()
    x, w = _rand((600, 256), BF, 1, cuda), _rand((512, 256), BF, 2, cuda)
    q = _rand((2, 130, 4, 64), BF, 3, cuda)
    want = ops.linear_act(x, w), ops.attention(q, q, q, frame=1)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_act(x, w), ops.attention(q, q, q, frame=1)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda):
    q = torch.zeros((1, 4, 2, 16), dtype=BF, device=cuda)
    pos = torch.zeros((4, 1), dtype=torch.int32, device=cuda)
    for err, fn in [
        (ValueError, lambda: ops.rotary_axes(q, pos, (3,))), (ValueError, lambda: ops.rotary_axes(q, pos, (18,))),
        (ValueError, lambda: ops.rotary_axes(q, pos, (4, 4))), (ValueError, lambda: ops.rotary_axes(q[0], pos, (4,))),
        (ValueError, lambda: ops.rotary_axes(q, pos, (4,), pairing="x")), (ValueError, lambda: ops.rotary_axes(q, pos, (4,), base=-1.0)),
        (TypeError, lambda: ops.rotary_axes(q, pos.double(), (4,))), (TypeError, lambda: ops.rotary_axes(q.double(), pos, (4,))),
        (TypeError, lambda: ops.rotary_axes(q, pos, (4,), also=q.half())), (RuntimeError, lambda: ops.rotary_axes(q, pos.cpu(), (4,))),
        (TypeError, lambda: ops.attention(q.float(), q.float(), q.float())), (TypeError, lambda: ops.attention(q, q.half(), q)),
        (ValueError, lambda: ops.attention(q, q[:, :, :1].expand(1, 4, 3, 16), q)), (ValueError, lambda: ops.attention(q[..., :12], q[..., :12], q[..., :12])),
        (ValueError, lambda: ops.attention(q, q, q, window=2)), (ValueError, lambda: ops.attention(q, q, q, frame=-1)),
        (ValueError, lambda: ops.attention(q, q, q, scale=0.0)), (TypeError, lambda: ops.attention(q, q, q, k_lens=torch.ones(1, device=cuda))),
        (ValueError, lambda: ops.attention(q, q, q, k_lens=torch.ones(2, dtype=torch.int32, device=cuda))),
        (RuntimeError, lambda: ops.attention(q, q.cpu(), q)), (ValueError, lambda: ops.attention(torch.zeros((1, 2, 1, 136), dtype=BF, device=cuda), *[torch.zeros((1, 2, 1, 136), dtype=BF, device=cuda)] * 2)),
        (ValueError, lambda: ops.linear_act(q, q[0, 0, :, :8])), (TypeError, lambda: ops.linear_act(q.float(), q[0, 0].float())),
        (TypeError, lambda: ops.linear_act(q, q[0, 0].half())), (ValueError, lambda: ops.linear_act(q, q[0, 0], act=3)),
        (ValueError, lambda: ops.linear_act(q, q[0, 0], bias=q[0, 0, 0])), (TypeError, lambda: ops.linear_act(q, q[0, 0], bias=torch.zeros(2, device=cuda, dtype=torch.float64))),
        (ValueError, lambda: ops.linear_act(q, q[0, 0], residual=q)), (ValueError, lambda: ops.linear_act_bwd(q, q, q[0, 0])),
    ]:
        with pytest.raises(err):
            fn()


def test_views_whose_offsets_pass_32_bits(cuda):
    """Tokens that lie 40 MB apart (a slice of a memory of many layers) and rows of almost 2^22 channels: the bits are those of packed copies."""
    n = 130
    far = torch.empty(n, 20 << 20, dtype=BF, device=cuda)
    def view(i, heads, d):
        x = far[:, 8192 * i:8192 * i + heads * d]
        x.copy_(_rand((n, heads * d), BF, 51 + i, cuda))
        return x.unflatten(1, (heads, d))[None]
    q, k, v, do = view(0, 4, 64), view(1, 2, 64), view(2, 2, 64), view(3, 4, 64)
    assert k.stride(1) * (n - 1) * 2 > 1 << 32
    near = [t.contiguous() for t in (q, k, v, do)]
    for kw in (dict(), dict(frame=1)):
        out, lse = ops.attention(q, k, v, return_lse=True, **kw)
        ref, rlse = ops.attention(*near[:3], return_lse=True, **kw)
        assert torch.equal(out, ref) and torch.equal(lse, rlse)
        got, want = ops.attention_bwd(do, q, k, v, out, lse, **kw), ops.attention_bwd(near[3], *near[:3], ref, rlse, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos = torch.arange(n, device=cuda)[:, None]
    assert all(torch.equal(a, b) for a, b in zip(ops.rotary_axes(q, pos, (64,), also=k), ops.rotary_axes(near[0], pos, (64,), also=near[1])))
    del far, q, k, v, do
    wide = torch.empty(600, (1 << 22) - 8, dtype=BF, device=cuda)
    x, w = wide[:, :136], wide[:200, 4096:4096 + 136]
    x.copy_(_rand((600, 136), BF, 61, cuda))
    w.copy_(_rand((200, 136), BF, 62, cuda))
    dy = wide[:, 8192:8192 + 200]
    dy.copy_(_rand((600, 200), BF, 63, cuda))
    assert torch.equal(ops.linear_act(x, w), ops.linear_act(x.contiguous(), w.contiguous()))
    got, want = ops.linear_act_bwd(dy, x, w)[:2], ops.linear_act_bwd(dy.contiguous(), x.contiguous(), w.contiguous())[:2]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("c", [8, 64, 72, 136, 192, 264])
def test_linear_act_short_sums_over_wide_results(cuda, c):
    """One to five steps of the contraction over results of 4100 x 4088, in each of the three products. Tolerance: c fp32 additions (c 2^-24 of
    the absolute sum, twice that for the products' own order) and half a step of bf16."""
    big, wide = 4100, 4088
    def check(got, a, b):                                            # got = a b^T over c columns
        a, b = a.double(), b.double()
        ref, mass = a @ b.t(), a.abs() @ b.abs().t()
        _close(got, ref, 2 * c * 2.0 ** -24 * mass + 2.0 ** -8 * ref.abs(), f"{tuple(got.shape)} over {c}")
    x, w = _rand((big, c), BF, 71, cuda), _rand((wide, c), BF, 72, cuda)
    check(ops.linear_act(x, w), x, w)
    dy, w = _rand((big, c), BF, 73, cuda), _rand((c, wide), BF, 74, cuda)
    check(ops.linear_act_bwd(dy, _rand((big, wide), BF, 75, cuda), w, want_dw=False)[0], dy, w.t())
    dy, x = _rand((c, big), BF, 76, cuda), _rand((c, wide), BF, 77, cuda)
    check(ops.linear_act_bwd(dy, x, _rand((big, wide), BF, 78, cuda), want_dx=False)[1], dy.t(), x.t())


# ---- values that are not finite -----------------------------------------------------------------------------------------------

NONFINITE = [  # B, N, M, H, Hk, D, frame
    (2, 70, 90, 4, 2, 64, 0),                                       # few keys: the statistics' own products
    (2, 150, 200, 4, 2, 128, 0),
    (2, 200, 200, 2, 1, 40, 1),
    (2, 1, 3000, 4, 2, 128, 0),                                     # the keys are split
    (2, 9, 2500, 6, 2, 32, 1),
]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("case", NONFINITE)
@pytest.mark.parametrize("kind", ["nan key", "infinite key", "infinite query", "nan value"])
def test_attention_of_visible_values_that_are_not_finite(cuda, dt, case, kind):
    """A row that sees a score (or a value) that is not finite is NaN, as its softmax is; rows of other entries and key heads do not change."""
    B, N, M, H, Hk, D, frame = case
    G = H // Hk
    q, k, v, do = _rand((B, N, H, D), dt, 1, cuda), _rand((B, M, Hk, D), dt, 2, cuda), _rand((B, M, Hk, D), dt, 3, cuda), _rand((B, N, H, D), dt, 4, cuda)
    ref, tol = _attention_ref(q, k, v, do, [N] * B, [M] * B, frame, 0, D ** -0.5, dt)
    at = max(M - max(N // 2, 1), 0)                                  # seen by about half of the rows in order, by all without
    hit = torch.zeros((B, N, H), dtype=torch.bool, device=cuda)
    if kind == "infinite query":
        q[1, N - 1, 1, 3] = math.inf                                 # products of either sign: inf - inf, or a maximum of inf
        hit[1, N - 1, 1] = True
    else:
        (v if kind == "nan value" else k)[1, at, 0, 5] = math.inf if kind == "infinite key" else math.nan
        hit[1, :, :G] = _visible(N, M, N, M, frame, 0, cuda)[:, at, None]
    if kind == "infinite key":                                       # a score of -inf has no weight, one of +inf is the row's maximum
        hit &= (q[..., 5] > 0)
    out, lse = ops.attention(q, k, v, frame=frame, return_lse=True)
    got = torch.isnan(out.float()).any(-1)
    if kind == "nan value":                                          # in order it may reach rows that do not see it: 0 times NaN
        assert torch.isfinite(lse).all() and (got.equal(hit) if not frame else got[hit].all())
    else:
        assert got.equal(hit) and torch.isnan(out.float()).all(-1).equal(hit), "out"
        assert torch.isnan(lse.transpose(1, 2)).equal(hit), "lse"
    away = torch.ones((B, H), dtype=torch.bool, device=cuda)         # (entry, head) pairs that have nothing to do with it
    away[1, :G] = False
    pick = lambda t: t.transpose(1, 2)[away]
    _close(pick(out), pick(ref[0]), pick(tol[0]), "out elsewhere")
    dq, dk, dv = ops.attention_bwd(do, q, k, v, out, lse, frame=frame)
    _close(pick(dq), pick(ref[2]), pick(tol[1]), "dq elsewhere")
    for t, r, e, name in ((dk, ref[3], tol[2], "dk elsewhere"), (dv, ref[4], tol[3], "dv elsewhere")):
        # fp16: e's share of the result's own rounding vanishes with |dk|, the rounding itself stays half of 2^-24 below 2^-14
        _close(torch.cat([t[0], t[1, :, 1:]], 1), torch.cat([r[0], r[1, :, 1:]], 1), torch.cat([e[0], e[1, :, 1:]], 1) + _sub(dt), name)
    assert torch.isnan(dq.float()).any(-1)[hit].all(), "dq"
    if kind != "nan value":                                          # their weights are NaN, and so is what these weights carry to the keys they see
        seen = (_visible(N, M, N, M, frame, 0, cuda) & hit[1, :, :G].any(1)[:, None]).any(0)
        assert torch.isnan(dv[1, :, 0].float()).all(-1)[seen].all(), "dv"


@pytest.mark.parametrize("N,M", [(70, 90), (1, 3000)])
def test_attention_of_rows_whose_scores_are_all_minus_infinity_or_very_low(cuda, N, M):
    """A row whose visible scores are all -inf has no softmax (0 / 0), which is not a row that sees nothing. Scores of -2^29 (far below any
    16-bit mask value) are a softmax like any other: equal ones give the mean of the values."""
    q, k, v = (torch.zeros((1, n, 1, 16), dtype=BF, device=cuda) for n in (N, M, M))
    v.copy_(_rand(v.shape, BF, 3, cuda))
    k[..., 0], q[..., 0] = 2.0 ** 16, -2.0 ** 13
    out, lse = ops.attention(q, k, v, return_lse=True, scale=1.0)
    mean = v.double().mean(1, keepdim=True).expand_as(out)
    _close(out, mean, 2.0 ** -8 * mean.abs() + 2.0 ** -7 * v.double().abs().mean(1, keepdim=True), "mean")
    # base 2 and back: two roundings of a number of 2^30
    assert (lse.double() / -2.0 ** 29 - 1).abs().max() < 2.0 ** -22
    k[..., 0] = 1
    q.zero_()
    q[:, 0, :, 0] = -math.inf
    out, lse = ops.attention(q, k, v, return_lse=True)
    assert torch.isnan(out[:, 0].float()).all() and torch.isfinite(out[:, 1:].float()).all()
    assert not torch.isfinite(lse[:, :, 0]).any()
    dq, dk, dv = ops.attention_bwd(torch.ones_like(out), q, k, v, out, lse)
    assert torch.isnan(dq[:, 0].float()).any() and torch.isnan(dv.float()).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("N,M,H,Hk,D,frame,window", [(70, 90, 4, 2, 64, 0, 0), (150, 200, 4, 2, 128, 0, 0), (200, 200, 2, 1, 40, 1, 0), (1, 3000, 4, 2, 128, 0, 0),
                                                     (2000, 40, 4, 1, 32, 0, 0), (70, 300, 2, 2, 64, 10, 2)])
def test_attention_gradients_behind_the_lengths_are_zero_beside_values_that_are_not_finite(cuda, dt, N, M, H, Hk, D, frame, window):
    """Rows and keys behind the lengths, rows that see nothing and keys that no row sees have zero outputs and gradients, also where others are NaN."""
    B = 3
    ql, kl = [N, max(N - 37, 0), max(N - 5, 1)], [M - 33, M, M // 2]
    base = [_rand((B, N, H, D), dt, 1, cuda), _rand((B, M, Hk, D), dt, 2, cuda), _rand((B, M, Hk, D), dt, 3, cuda), _rand((B, N, H, D), dt, 4, cuda)]
    kw = dict(q_lens=_lens(ql, B, N, cuda), k_lens=_lens(kl, B, M, cuda), frame=frame, window=window)
    for which in range(4):                                           # a NaN in q, k, v, dO
        x = [t.clone() for t in base]
        x[which][:, 0] = math.nan
        out, lse = ops.attention(*x[:3], return_lse=True, **kw)
        dq, dk, dv = ops.attention_bwd(x[3], *x[:3], out, lse, **kw)
        for b in range(B):
            none = ~_visible(N, M, ql[b], kl[b], frame, window, cuda)
            row, key = none.all(1), none.all(0)
            assert not out[b, row].any() and torch.isneginf(lse[b][:, row]).all(), (which, b)
            assert not dq[b, row].any(), (which, b)
            assert not dk[b, key].any() and not dv[b, key].any(), (which, b)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("act", [ops.ACT_RELU, ops.ACT_GELU])
@pytest.mark.parametrize("M,K,N", [(4, 64, 64), (130, 64, 33), (300, 64, 72), (66, 712, 16), (1234, 16, 3304)])
def test_linear_act_slope_of_a_value_that_is_not_finite(cuda, dt, act, M, K, N):
    """A NaN in front of the activation comes back as a NaN gradient of its row; infinities have the slopes 1 and 0."""
    x, w, dy = _rand((M, K), dt, 1, cuda), _rand((N, K), dt, 2, cuda, 0.1), _rand((M, N), dt, 3, cuda)
    b = torch.zeros(N, dtype=F32, device=cuda)
    x[1], b[1], b[2] = math.nan, math.inf, -math.inf
    y, gate = ops.linear_act(x, w, b, act=act, return_gate=True)
    rows = torch.zeros(M, dtype=torch.bool, device=cuda)
    rows[1] = True
    assert torch.isnan(y.float()).all(1).equal(rows) and torch.isposinf(y[~rows, 1].float()).all() and not y[~rows, 2].any()
    assert (gate[~rows, 1] == 1 << 14).all() and (gate[~rows, 2] == 0).all()
    x[1] = 0                                                         # the slope alone carries it on
    dx, dw, db = ops.linear_act_bwd(dy, x, w, gate=gate, bias=b)
    assert torch.isnan(dx.float()).all(1).equal(rows) and torch.isnan(db).all()


@pytest.mark.parametrize("dt", [BF, HF])
def test_linear_act_gelu_far_below_zero(cuda, dt):
    """z cdf(z) is tiny there but in bf16 an ordinary number: right relative to itself. Tolerance: half a step of the type, and 2^-13 for
    the 5e-5 of the fit, 1e-5 of the exponent's fp32 roundings at z = -12 (two of a number of 104) and the products of fp32 behind them."""
    x = torch.linspace(-12.0, -3.0, 4097, device=cuda).to(dt)[:, None]
    w = torch.ones((1, 1), dtype=dt, device=cuda)
    for rows in (slice(None), slice(0, 4096, 83)):                   # tiles, and few rows
        z = x[rows].contiguous()
        y = ops.linear_act(z, w, act=ops.ACT_GELU)
        ref = _act64(z.double(), ops.ACT_GELU)[0]
        _close(y, ref, (_u(dt) + 2.0 ** -13) * ref.abs() + _sub(dt), "gelu")


def test_forward_mode_tangents_are_refused(cuda):
    """The operators have no forward-mode derivative: a dual tensor is refused, not answered without its tangent."""
    import torch.autograd.forward_ad as fw
    x, w = _rand((4, 64), BF, 1, cuda), _rand((64, 64), BF, 2, cuda)
    q, b = x.view(1, 4, 2, 32), torch.zeros(64, dtype=F32, device=cuda)
    pos = torch.zeros((4, 1), device=cuda)
    out, lse = ops.attention(q, q, q, return_lse=True)
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.linear_act(d(x), w), lambda: ops.linear_act(x, d(w)), lambda: ops.linear_act(x, w, d(b)),
                     lambda: ops.linear_act(x, w, residual=d(x)), lambda: ops.linear_act_bwd(d(x), x, w), lambda: ops.linear_act_bwd(x, x, w, bias=d(b)),
                     lambda: ops.attention(d(q), q, q), lambda: ops.attention(q, d(q), q), lambda: ops.attention(q, q, d(q)),
                     lambda: ops.attention_bwd(d(q), q, q, q, out, lse), lambda: ops.attention_bwd(q, q, q, q, out, d(lse)),
                     lambda: ops.rotary_axes(d(q), pos, (4,)), lambda: ops.rotary_axes(q, pos, (4,), also=d(q)),
                     lambda: ops.rotary_axes(q, d(pos), (4,)), lambda: ops.rotary_axes_bwd(d(q), pos, (4,))):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with pytest.raises(RuntimeError, match="tangent"), torch.no_grad():
                call()
        assert torch.equal(ops.linear_act(x, w), ops.linear_act(x.clone(), w))      # plain tensors inside a level


# ---- every tile, split and row-block variant ----------------------------------------------------------------------------------

def _linear_plan(M, N, K, cus):
    """The library's choice of tile and split, restated: a case below that no longer reaches its variant fails instead of testing another."""
    best, steps = None, (K + 63) // 64
    for tile, fit, full, alone, fixed in ((256, 1, 1.5, 1.5, 6.0), (128, 2, 0.68, 0.9, 4.0), (64, 4, 0.36, 0.6, 3.0)):
        tiles = -(-M // tile) * -(-N // tile)
        for s in range(1, 33):
            if s > 1 and steps // s < 4:
                break
            rest, depth = tiles * s % (cus * fit), float((steps + s - 1) // s)
            one = lambda on: depth * max(on * full, alone) + fixed
            t = tiles * s // (cus * fit) * one(fit) + (one((rest + cus - 1) // cus) if rest else 0.0) + (4.0 + s * M * N * 8.0 / 4e6 if s > 1 else 0.0)
            if best is None or t < best[0]:
                best = (t, tile, s)
    return best[1:]


VARIANTS = [  # M, K, N, act, bias, residual, (tile, split) of y, dx, dW; 0: any
    (17, 1096, 331, ops.ACT_GELU, True, True, 0, 0, 0),             # few rows: two and four blocks of 16, more than one pass over k
    (32, 2056, 72, ops.ACT_RELU, True, False, 0, 0, 0),
    (33, 40, 130, ops.ACT_GELU, True, True, 0, 0, 0),
    (64, 1100, 128, ops.ACT_GELU, False, True, 0, 0, 0),
    (1234, 136, 3304, ops.ACT_GELU, True, True, (128, False), 0, 0),
    (1233, 136, 3301, ops.ACT_GELU, True, True, (128, False), 0, 0),
    (1746, 69, 4104, ops.ACT_GELU, True, True, (128, False), 0, (128, True)),
    (73, 1744, 4264, ops.ACT_GELU, True, True, (128, True), 0, (128, False)),
    (1155, 3424, 16, ops.ACT_GELU, True, False, 0, (128, False), 0),
    (2389, 65, 3967, ops.ACT_GELU, True, True, (256, False), (128, True), 0),
    (6332, 136, 4488, ops.ACT_GELU, True, True, (256, False), (128, True), (256, True)),
    (4096, 2048, 4096, ops.ACT_RELU, True, True, (256, False), (128, False), (128, False)),
    (66, 2728, 2960, ops.ACT_GELU, True, True, 0, 0, (256, False)),
    (6697, 4238, 129, ops.ACT_GELU, True, True, (256, True), (256, False), (128, True)),
    (5631, 140, 4971, ops.ACT_GELU, True, False, 0, (256, True), (128, True)),
]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("case", VARIANTS)
def test_linear_act_variants(cuda, dt, case):
    M, K, N = case[:3]
    cus = torch.cuda.get_device_properties(cuda).multi_processor_count
    for want, size in zip(case[6:], ((M, N, K), (M, K, N), (N, K, M))):
        if want:
            tile, s = _linear_plan(*size, cus)
            assert (tile, s > 1) == want
    tile, s = _linear_plan(M, N, K, cus)
    packed = 2 * (M + N) * (K + 7 & ~7) if K % 8 else 0
    parts = 4 * s * M * (N + 7 & ~7) if s > 1 and M > 64 else 0
    assert 0 <= _lib.load().svps_linear_act_workspace_bytes(M, K, N, K, K, 0) - packed - parts < 3 * 256
    test_linear_act_forward_and_gradients(cuda, dt, case[:6])


@pytest.mark.parametrize("dt,G,D,N,M,frame,window", [
    (BF, 2, 128, 250, 203, 0, 0), (HF, 2, 128, 250, 203, 1, 0), (BF, 3, 72, 171, 190, 1, 0), (HF, 3, 96, 171, 90, 0, 0), (BF, 3, 128, 171, 203, 50, 2),
    (HF, 5, 128, 103, 120, 1, 7)])
def test_attention_of_two_row_blocks_per_wave(cuda, dt, G, D, N, M, frame, window):
    """Heads above 64 with workgroups of 256 rows for four rounds of the compute units, lengths that end inside them, group sizes that divide no tile."""
    B, Hk = 32, 16
    H = G * Hk
    assert B * Hk * -(-N * G // 256) >= 4 * torch.cuda.get_device_properties(cuda).multi_processor_count
    ql, kl = [N - 3 * b for b in range(B)], [M - 2 * b for b in range(B)]
    q, k, v, do = _rand((B, N, H, D), dt, 1, cuda), _rand((B, M, Hk, D), dt, 2, cuda), _rand((B, M, Hk, D), dt, 3, cuda), _rand((B, N, H, D), dt, 4, cuda)
    for b in range(B):
        q[b, ql[b]:], do[b, ql[b]:], k[b, kl[b]:], v[b, kl[b]:] = math.nan, math.inf, math.nan, -math.inf
    kw = dict(q_lens=_lens(ql, B, N, cuda), k_lens=_lens(kl, B, M, cuda), frame=frame, window=window)
    out, lse = ops.attention(q, k, v, return_lse=True, **kw)
    some = [0, 1, 7, B - 1]                                          # entries that are compared
    part = lambda t: t[some]
    ref, tol = _attention_ref(part(q), part(k), part(v), part(do), [ql[b] for b in some], [kl[b] for b in some], frame, window, D ** -0.5, dt)
    _close(part(out), ref[0], tol[0], "out")
    none = torch.isinf(ref[1])
    assert torch.equal(torch.isinf(part(lse)), none) and (part(lse).double() - ref[1])[~none].abs().max() < 1e-3
    for name, a, r, t in zip(("dq", "dk", "dv"), ops.attention_bwd(do, q, k, v, out, lse, **kw), ref[2:], tol[1:]):
        _close(part(a), r, t, name)
    for b in some:                                                   # alone, an entry runs in another variant: equal but for the order of its fp32 sums
        one = ops.attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], q_lens=kw["q_lens"][b:b + 1], k_lens=kw["k_lens"][b:b + 1], frame=frame, window=window)
        _close(one, ref[0][some.index(b)][None], tol[0][some.index(b)][None], "alone")


def test_attention_of_eight_waves_in_fp16(cuda):
    B, N, M, H, Hk, D = 32, 250, 203, 16, 8, 64
    q, k, v = _rand((B, N, H, D), HF, 1, cuda), _rand((B, M, Hk, D), HF, 2, cuda), _rand((B, M, Hk, D), HF, 3, cuda)
    out = ops.attention(q, k, v, frame=1)
    ref, tol = _attention_ref(q[:2], k[:2], v[:2], None, [N] * 2, [M] * 2, 1, 0, D ** -0.5, HF)
    _close(out[:2], ref[0], tol[0], "out")
