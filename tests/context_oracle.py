"""Plain 64-bit forms of the context operators and how far the kernels may be from them.

The bounds are first-order sums of the roundings a kernel makes: u = half a step of the operand type (P, dS, outputs),
e = 2^-24 (every fp32 operation), d = 2^-25 (fp16: half of the smallest subnormal, absolute: the outputs, and the
forward pass's P, which is at least 1 somewhere in its row; the backward pass scales its P and dS by powers of two).
"""
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows(x, C, Hk):
    """[B, L, H, D] -> fp64 [C, Hk, rows, D]"""
    B, L, H, D = x.shape
    return x.double().reshape(C, B // C, L, Hk, H // Hk, D).permute(0, 3, 1, 2, 4, 5).reshape(C, Hk, -1, D)


def unrows(y, shape, C, Hk):
    B, L, H, D = shape
    return y.reshape(C, Hk, B // C, L, H // Hk, D).permute(0, 2, 3, 1, 4, 5).reshape(B, L, H, D)


def attention(q, k, v, query_lengths=None, context_lengths=None, context_mask=None, scale=None, out_grad=None):
    """{name: (value, bound)} of out, lse and, with out_grad, dq, dk, dv."""
    B, Lq, Hq, D = q.shape
    C, Lk, Hk = k.shape[:3]
    scale = D ** -0.5 if scale is None else scale
    u = half_step(q.dtype)
    up = 0.0 if q.dtype == torch.float32 else u
    d = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    dev = q.device
    keep = torch.ones((C, Lk), dtype=torch.bool, device=dev)
    if context_lengths is not None:
        keep &= torch.arange(Lk, device=dev)[None] < context_lengths[:, None]
    if context_mask is not None:
        keep &= context_mask.bool()
    live = torch.ones((B, Lq), dtype=torch.bool, device=dev)
    if query_lengths is not None:
        live &= torch.arange(Lq, device=dev)[None] < query_lengths[:, None]
    zero = torch.zeros((), dtype=torch.float64, device=dev)
    lv = rows(live[:, :, None, None].expand(B, Lq, Hq, 1), C, Hk).bool()
    K = torch.where(keep[:, None, :, None], k.double().permute(0, 2, 1, 3), zero)
    V = torch.where(keep[:, None, :, None], v.double().permute(0, 2, 1, 3), zero)
    Q = torch.where(lv, rows(q, C, Hk), zero)
    S = scale * Q @ K.transpose(2, 3)
    S = S.masked_fill(~keep[:, None, None, :], -math.inf)
    m = S.amax(-1, keepdim=True) if Lk else S.new_full((C, Hk, Q.shape[2], 1), -math.inf)
    m = m.masked_fill(m == -math.inf, 0.0)
    p = torch.exp(S - m)
    z = p.sum(-1, keepdim=True)
    lse = torch.where(lv, m + torch.log(z), zero - math.inf)
    P = torch.where(lv & (z > 0), p / z.clamp_min(1e-300), zero)
    O = P @ V
    # score error: D products and sums, the scale; P's relative error: twice that (its row's sum has it too), the
    # exponential and its argument (some steps of a number of the score's size)
    sa = (abs(scale) * Q.abs() @ K.abs().transpose(2, 3)).amax(-1, keepdim=True) if Lk else torch.zeros_like(z)
    eS = (D + 6) * E * sa
    eP = 2 * eS + (Lk + 16) * E + 4 * E * S.masked_fill(S == -math.inf, 0.0).abs().amax(-1, keepdim=True) if Lk else eS
    tO = (up + eP) * (P @ V.abs()) + u * O.abs() + d * V.abs().sum(2, keepdim=True) + d
    back = lambda x: unrows(x, (B, Lq, Hq, x.shape[-1]), C, Hk)                                        # noqa: E731
    t_lse = eS + 4 * E * (1 + lse.masked_fill(lse == -math.inf, 0.0).abs()) + (Lk + 8) * E
    res = {"out": (back(O), back(tO.expand_as(O))),
           "lse": (back(lse)[..., 0].transpose(1, 2), back(t_lse)[..., 0].transpose(1, 2))}
    if out_grad is None:
        return res
    G = torch.where(lv, rows(out_grad, C, Hk), zero)
    dP = G @ V.transpose(2, 3)
    delta = (G * O).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    # P is recomputed from lse (rounded to fp32); delta from the rounded output
    eP = eP + 2 * t_lse
    t_delta = (G.abs() * (tO + D * E * O.abs())).sum(-1, keepdim=True)
    t_dP = (D + 2) * E * (G.abs() @ V.abs().transpose(2, 3))
    # fp16: what a column's scale cuts off is 2^-25 of its largest dS, and of 2^14 P 2^-25
    cut = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    tS = (up + eP + 4 * E) * dS.abs() + P * (t_dP + t_delta) + cut * (dS.abs().amax((2, 3), keepdim=True) if Lk else 0.0)
    n = Q.shape[2]
    tQ = abs(scale) * (tS + (Lk + 2) * E * dS.abs()) @ K.abs()
    tK = abs(scale) * (tS + (n + 2) * E * dS.abs()).transpose(2, 3) @ Q.abs()
    tV = ((up + eP + (n + 2) * E) * P + cut * 2.0 ** -14 * (P > 0)).transpose(2, 3) @ G.abs()
    dQ, dK, dV = scale * dS @ K, scale * dS.transpose(2, 3) @ Q, P.transpose(2, 3) @ G
    res["dq"] = (back(dQ), back(tQ + u * dQ.abs() + d))
    res["dk"] = tuple(x.permute(0, 2, 1, 3) for x in (dK, tK + u * dK.abs() + d))
    res["dv"] = tuple(x.permute(0, 2, 1, 3) for x in (dV, tV + u * dV.abs() + d))
    return res


def _pairs(axes, D, interleaved, theta):
    lo, hi, ax, fr, at = [], [], [], [], 0
    for a, n in enumerate(list(axes) + [D - sum(axes)]):
        for j in range(n // 2):
            lo.append(at + 2 * j if interleaved else at + j)
            hi.append(at + 2 * j + 1 if interleaved else at + j + n // 2)
            ax.append(min(a, len(axes) - 1))
            fr.append(theta ** (-2.0 * j / n) if a < len(axes) else 0.0)
        at += n
    return lo, hi, ax, fr


def norm_rotary(x, w, positions, axes, theta=10000.0, eps=1e-6, interleaved=False, grad=None):
    """{name: (value, bound)} of y or, with the output's gradient, dx and dw."""
    D = x.shape[-1]
    u = half_step(x.dtype)
    d = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    lo, hi, ax, fr = _pairs(axes, D, interleaved, theta)
    lo, hi, ax = (torch.tensor(t, device=x.device) for t in (lo, hi, ax))
    fr = torch.tensor(fr, dtype=torch.float64, device=x.device)
    pos = positions.double()
    angle = (pos if pos.dim() == 3 else pos[None])[..., ax] * fr
    c, s = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    X = x.double()
    W = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    r = 1 / torch.sqrt((X * X).mean(-1, keepdim=True) + eps)
    # r: D products and sums in fp32, halved by the square root; then a few products, and the angle (an fp32 sine)
    n = (D / 2 + 16) * E

    def turn(z, sign):
        a, b = z[..., lo], z[..., hi]
        out, size = torch.empty_like(z), torch.empty_like(z)
        out[..., lo], out[..., hi] = a * c - sign * b * s, b * c + sign * a * s
        size[..., lo] = size[..., hi] = a.abs() + b.abs()
        return out, size
    if grad is None:
        y, size = turn(X * r * W, 1.0)
        return {"y": (y, u * y.abs() + n * size + d)}
    g, size = turn(grad.double(), -1.0)
    g, size = g.expand_as(X), size.expand_as(X)
    U = g * W
    m = (U * X).mean(-1, keepdim=True) * r * r
    dx = r * (U - X * m)
    t_m = (1.5 * D + 16) * E * (size * W.abs() * X.abs()).mean(-1, keepdim=True) * r * r
    tx = u * dx.abs() + r * (n * size * W.abs() + X.abs() * (t_m + n * m.abs())) + d
    dw = (g * X * r).sum((0, 1, 2))
    count = x.shape[0] * x.shape[1] * x.shape[2]
    tw = ((n + count * E) * size * (X * r).abs()).sum((0, 1, 2))
    uw = 0.0 if w is None or w.dtype == torch.float32 else half_step(w.dtype)
    return {"dx": (dx, tx), "dw": (dw, tw + uw * dw.abs())}


def check(name, got, value, bound):
    """Every element of `got` within its bound of `value` (equal where not finite)."""
    g = got.double()
    assert g.shape == value.shape, (name, tuple(g.shape), tuple(value.shape))
    fin = torch.isfinite(value)
    same = torch.where(fin, torch.zeros_like(g), g) == torch.where(fin, torch.zeros_like(value), value)
    assert bool((same | fin).all()), f"{name}: not finite where it should be (or the reverse)"
    off = torch.where(fin, (g - value).abs() / bound.clamp_min(1e-38), torch.zeros_like(g))
    off = torch.where(fin & (g == value), torch.zeros_like(off), off)
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: an element is {worst:.3g} times its bound off"   # NaN fails too
    return worst
