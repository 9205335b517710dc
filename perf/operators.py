"""Measured cases of the context operators: per-head norm + rotation of queries and keys, and cross attention.

``run`` makes one pass: with ``own`` the framework's calls (``ecnf_amd.context``), otherwise the same operators in
elementary torch operations in 32 bits (the rotation's angles in 64), rounded once at the end.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_THETA = 10000.0
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------------ the cases
def _qkn(name, grad, dtype, B, Lq, Hq, Bk, Lk, Hk, D, axes, interleaved=False, real=False):
    """Norm + rotation of q [B, Lq, Hq, D] and, where Lk > 0, k [Bk, Lk, Hk, D]; `axes` is written "32" or "32+48+48".
    real: positions are real numbers (coordinates, times), else whole ones (indices)."""
    return dict(name=name, op="qk_norm_rotary_grad" if grad else "qk_norm_rotary", dtype=dtype, B=B, Lq=Lq, Hq=Hq,
                Bk=Bk, Lk=Lk, Hk=Hk, D=D, axes=axes, interleaved=interleaved, real=real)


def _att(name, grad, dtype, B, Lq, Hq, Bk, Lk, Hk, D, ragged=False, masked=False):
    """Cross attention of q [B, Lq, Hq, D] to k, v [Bk, Lk, Hk, D] (Bk = 1: one context for the whole batch).
    ragged: contexts of different lengths, some empty; masked: a tenth of the keys is masked besides."""
    return dict(name=name, op="cross_attention_grad" if grad else "cross_attention", dtype=dtype, B=B, Lq=Lq, Hq=Hq,
                Bk=Bk, Lk=Lk, Hk=Hk, D=D, ragged=ragged, masked=masked)


def listed():
    return [
        # a batch of LJ13 clusters (13 atoms, 64 hidden features as 2 heads) and one context of 64 states, all in fp32:
        # what every conditional solve of the framework's headline batch does first
        _qkn("norm_lj13_fp32", False, "fp32", 1024, 13, 2, 1, 64, 2, 32, "32"),
        # one new token a sequence, its keys already there: the smallest call, where latency counts
        _qkn("norm_one_token_bf16", False, "bf16", 64, 1, 32, 1, 0, 0, 128, "128"),
        # long queries and a longer context with grid coordinates on three axes, shared key heads
        _qkn("norm_axes_long_bf16", False, "bf16", 4, 4096, 32, 4, 8192, 8, 128, "32+48+48", real=True),
        # the gradient of the same in a training step of odd length, adjacent pairs, some dims unrotated
        _qkn("norm_grad_long_bf16", True, "bf16", 4, 4095, 32, 4, 2047, 8, 128, "32+32+32", interleaved=True),
        # the gradient at alanine dipeptide's 22 atoms and small heads, all in fp32
        _qkn("norm_grad_aldp_fp32", True, "fp32", 512, 22, 4, 512, 37, 4, 16, "8+8"),
        # LJ13 clusters of the headline batch against one shared context
        _att("attn_lj13_shared_fp32", False, "fp32", 1024, 13, 2, 1, 64, 2, 32),
        # one query token a sequence over long contexts: reading keys and values is all
        _att("attn_one_token_bf16", False, "bf16", 64, 1, 32, 64, 8192, 8, 128),
        # a padded batch of alanine dipeptide with a context of its own for each molecule
        _att("attn_aldp_ragged_bf16", False, "bf16", 512, 22, 8, 512, 333, 4, 64, ragged=True, masked=True),
        # long queries over a longer context: the largest product
        _att("attn_long_bf16", False, "bf16", 2, 4096, 32, 2, 8192, 8, 128),
        # training passes (forward, then gradients): molecules with their own padded contexts in fp32,
        _att("attn_train_aldp_fp32", True, "fp32", 512, 22, 4, 512, 129, 4, 16, ragged=True),
        # a large batch of molecules that share one context, in fp16,
        _att("attn_train_shared_fp16", True, "fp16", 1024, 22, 8, 1, 512, 8, 64),
        # and long sequences
        _att("attn_train_long_bf16", True, "bf16", 1, 4096, 32, 1, 8192, 8, 128),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, its logarithm uniform; odd ones as likely as even ones."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw_qkn(rng, grad):
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    D = rng.choice([16, 32, 64, 96, 128])
    n_axes = rng.choice([1, 1, 2, 3])
    rest = rng.choice([0, 0, 8]) if D > 16 else 0
    cut = sorted(rng.sample(range(1, (D - rest) // 4), n_axes - 1)) if n_axes > 1 else []
    ends = [0] + [4 * c for c in cut] + [D - rest]
    axes = "+".join(str(b - a) for a, b in zip(ends, ends[1:]))
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 1, 2, 4])
    B = _spread(rng, 1, 1024)
    room = max(1, (4 << 20) * 48 // (B * D * (Hq + Hk)))          # a third of the largest listed call at most
    Lq, Lk = _spread(rng, 1, min(8192, room)), _spread(rng, 1, min(8192, room))
    Bk = rng.choice([1, B])
    if not grad and rng.random() < 0.2:
        Bk, Lk, Hk = 1, 0, 0
    return _qkn(None, grad, dtype, B, Lq, Hq, Bk, Lk, Hk, D, axes, rng.random() < 0.5, rng.random() < 0.5)


def _draw_att(rng, grad):
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    D = rng.choice([16, 32, 64, 96, 128])
    Hk = rng.choice([1, 2, 4, 8])
    Hq = Hk * rng.choice([1, 1, 2, 4])
    kind = rng.choice(["molecules", "token", "long"])
    if kind == "molecules":
        B, Lq, Lk = _spread(rng, 1, 1024), rng.randint(2, 64), _spread(rng, 1, 1024)
    elif kind == "token":
        B, Lq, Lk = _spread(rng, 1, 64), 1, _spread(rng, 1, 16384)
    else:
        B, Lq, Lk = rng.randint(1, 4), _spread(rng, 64, 4096), _spread(rng, 64, 8192)
    Bk = rng.choice([1, B, B])
    most = (3e9 if dtype == "fp32" else 3e10) / (3 if grad else 1)  # multiply-adds; the largest listed has 2.7e11
    while B * Lq * Hq * Lk * D > most:
        Lk = max(1, Lk * 3 // 4)
        B = max(1, B * 7 // 8) if Bk == 1 else B
        Lq = max(1, Lq * 7 // 8)
    return _att(None, grad, dtype, B, Lq, Hq, Bk, Lk, Hk, D, rng.random() < 0.4, rng.random() < 0.3)


def draw(rng):
    op = rng.choice([(_draw_qkn, False), (_draw_qkn, True), (_draw_att, False), (_draw_att, False),
                     (_draw_att, True), (_draw_att, True)])
    case = op[0](rng, op[1])
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------------ the inputs
def _lengths(case):
    """Lengths of the contexts (whole numbers spread from none to all of Lk), in their unshuffled order."""
    n, L = case["Bk"], case["Lk"]
    if not case["ragged"]:
        return [L] * n
    return [L] if n == 1 else [(L * i) // (n - 1) for i in range(n)]


def prepare(case, seed):
    dt = _DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s = {"case": case}
    B, Lq, Hq, Bk, Lk, Hk, D = (case[n] for n in ("B", "Lq", "Hq", "Bk", "Lk", "Hk", "D"))
    s["q"] = normal(B, Lq, Hq, D)
    if case["op"].startswith("qk_norm"):
        A = len(case["axes"].split("+"))

        def positions(n, L):
            if case["real"]:
                return torch.rand((n, L, A), generator=g, device="cuda", dtype=torch.float32) * 200 - 100
            return torch.randint(0, 32768, (n, L, A), generator=g, device="cuda", dtype=torch.int32)

        def weight():
            return 1 + 0.1 * torch.randn(D, generator=g, device="cuda", dtype=torch.float32)
        s["q_positions"], s["q_weight"] = positions(B, Lq), weight()
        s["k"] = s["k_positions"] = s["k_weight"] = None
        if Lk:
            s["k"], s["k_positions"], s["k_weight"] = normal(Bk, Lk, Hk, D), positions(Bk, Lk), weight()
        if case["op"].endswith("grad"):
            s["q_grad"], s["k_grad"] = normal(B, Lq, Hq, D), normal(Bk, Lk, Hk, D)
    else:
        s["k"], s["v"] = normal(Bk, Lk, Hk, D), normal(Bk, Lk, Hk, D)
        s["lengths"] = s["mask"] = None
        if case["ragged"]:
            order = torch.randperm(Bk, generator=g, device="cuda")
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).to("cuda")[order].contiguous()
        if case["masked"]:
            s["mask"] = torch.rand((Bk, Lk), generator=g, device="cuda") > 0.1
        if case["op"].endswith("grad"):
            s["out_grad"] = normal(B, Lq, Hq, D)
    if own:
        package = os.path.join(os.getcwd(), "ecnf-baseline-neurips-2023_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        from ecnf_amd import context
        s["context"] = context
        s["axes"] = tuple(int(a) for a in case["axes"].split("+")) if "axes" in case else None
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    C, case = s["context"], s["case"]
    if case["op"].startswith("qk_norm"):
        kw = dict(q_weight=s["q_weight"], k_weight=s["k_weight"], q_positions=s["q_positions"],
                  k_positions=s["k_positions"], axes=s["axes"], theta=_THETA, eps=_EPS,
                  interleaved=case["interleaved"])
        if case["op"] == "qk_norm_rotary":
            q, k = C.qk_norm_rotary(s["q"], s["k"], **kw)
            return [q] if k is None else [q, k]
        return list(C.qk_norm_rotary_grad(s["q_grad"], s["k_grad"], s["q"], s["k"], **kw))
    kw = dict(context_lengths=s["lengths"], context_mask=s["mask"])
    if case["op"] == "cross_attention":
        return [C.cross_attention(s["q"], s["k"], s["v"], **kw)]
    out, lse = C.cross_attention(s["q"], s["k"], s["v"], return_lse=True, **kw)
    return [out, *C.cross_attention_grad(s["out_grad"], s["q"], s["k"], s["v"], out, lse, **kw)]


def _pairs(axes, interleaved):
    """(index of each rotated pair's first and second element, axis of the pair, its frequency) from the axes' dims."""
    lo, hi, ax, fr, at = [], [], [], [], 0
    for a, d in enumerate(axes):
        for j in range(d // 2):
            lo.append(at + 2 * j if interleaved else at + j)
            hi.append(at + 2 * j + 1 if interleaved else at + j + d // 2)
            ax.append(a)
            fr.append(_THETA ** (-2.0 * j / d))
        at += d
    return lo, hi, ax, fr


def _plain_angles(case, positions):
    lo, hi, ax, fr = _pairs([int(a) for a in case["axes"].split("+")], case["interleaved"])
    ax = torch.tensor(ax).to("cuda")
    angle = positions.double()[..., ax] * torch.tensor(fr, dtype=torch.float64).to("cuda")
    turn = angle - 2 * math.pi * torch.round(angle / (2 * math.pi))
    c, s = torch.cos(turn).float(), torch.sin(turn).float()
    return torch.tensor(lo).to("cuda"), torch.tensor(hi).to("cuda"), c[:, :, None], s[:, :, None]


def _plain_norm(case, x, w, positions):
    lo, hi, c, s = _plain_angles(case, positions)
    xf = x.float()
    y = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + _EPS) * w
    a, b = y[..., lo], y[..., hi]
    y[..., lo] = a * c - b * s
    y[..., hi] = a * s + b * c
    return y.to(x.dtype)


def _plain_norm_grad(case, dy, x, w, positions):
    lo, hi, c, s = _plain_angles(case, positions)
    g, xf = dy.float(), x.float()
    a, b = g[..., lo], g[..., hi]
    if dy.dtype == torch.float32:
        g = g.clone()
    g[..., lo] = a * c + b * s
    g[..., hi] = b * c - a * s
    r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + _EPS)
    xh = xf * r
    u = g * w
    dx = r * (u - xh * (u * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * xh).sum((0, 1, 2))


def _rows(x, Bk, Hk):
    """[B, L, H, D] -> [Bk, Hk, rows, D]: the rows that read one key head of one context."""
    B, L, H, D = x.shape
    return x.float().reshape(Bk, B // Bk, L, Hk, H // Hk, D).permute(0, 3, 1, 2, 4, 5).reshape(Bk, Hk, -1, D)


def _unrows(y, like, Bk, Hk):
    B, L, H, D = like.shape
    y = y.reshape(Bk, Hk, B // Bk, L, H // Hk, D).permute(0, 2, 3, 1, 4, 5)
    return y.reshape(B, L, H, D).to(like.dtype).contiguous()


def _run_plain(s):
    case = s["case"]
    if case["op"] == "qk_norm_rotary":
        out = [_plain_norm(case, s["q"], s["q_weight"], s["q_positions"])]
        return out if s["k"] is None else out + [_plain_norm(case, s["k"], s["k_weight"], s["k_positions"])]
    if case["op"] == "qk_norm_rotary_grad":
        dq, dqw = _plain_norm_grad(case, s["q_grad"], s["q"], s["q_weight"], s["q_positions"])
        dk, dkw = _plain_norm_grad(case, s["k_grad"], s["k"], s["k_weight"], s["k_positions"])
        return [dq, dk, dqw, dkw]
    Bk, Hk, scale = case["Bk"], case["Hk"], case["D"] ** -0.5
    q = _rows(s["q"], Bk, Hk)
    k = s["k"].float().permute(0, 2, 1, 3).contiguous()
    v = s["v"].float().permute(0, 2, 1, 3).contiguous()
    allowed = None
    if s["lengths"] is not None:
        allowed = torch.arange(case["Lk"], device="cuda")[None, :] < s["lengths"][:, None]
    if s["mask"] is not None:
        allowed = s["mask"] if allowed is None else allowed & s["mask"]
    p = torch.matmul(q, k.transpose(2, 3)) * scale
    if allowed is not None:
        p = p.masked_fill(~allowed[:, None, None, :], -math.inf)
        m = p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    else:
        m = p.amax(-1, keepdim=True)
    p = torch.exp(p - m)
    p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    o = torch.matmul(p, v)
    out = [_unrows(o, s["q"], Bk, Hk)]
    if case["op"] == "cross_attention":
        return out
    do = _rows(s["out_grad"], Bk, Hk)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    keys = [x.permute(0, 2, 1, 3).to(s["k"].dtype).contiguous() for x in (dk, dv)]
    return out + [_unrows(dq, s["q"], Bk, Hk)] + keys


# ------------------------------------------------------------------------------------------------------ what it takes
def work(case):
    e = _DTYPES[case["dtype"]].itemsize
    B, Lq, Hq, Bk, Lk, Hk, D = (case[n] for n in ("B", "Lq", "Hq", "Bk", "Lk", "Hk", "D"))
    nq, nk = B * Lq * Hq * D, Bk * Lk * Hk * D
    if case["op"].startswith("qk_norm"):
        grad = case["op"].endswith("grad")
        position_bytes = 4 * len(case["axes"].split("+")) * (B * Lq + Bk * Lk)
        return {"bytes": (3 if grad else 2) * e * (nq + nk) + position_bytes + 4 * D * (4 if grad else 2),
                "flops": (18 if grad else 8) * (nq + nk)}
    keys = sum(_lengths(case))                       # of all contexts
    kv = keys * Hk * D
    products = (B // Bk) * Lq * Hq * keys * D        # multiply-adds of one of the products
    if case["op"] == "cross_attention":
        return {"bytes": e * (2 * nq + 2 * kv), "flops": 4 * products}
    return {"bytes": e * (4 * nq + 2 * kv + 2 * nk), "flops": 14 * products}


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("qk_norm"):
        names = ["q"] + (["k"] if case["Lk"] else [])
        if case["op"] == "qk_norm_rotary":
            return [_exact_norm(case, s[n], s[n + "_weight"], s[n + "_positions"]) for n in names]
        both = [_exact_norm_grad(case, s[n + "_grad"], s[n], s[n + "_weight"], s[n + "_positions"]) for n in names]
        return [b[0] for b in both] + [b[1] for b in both]
    return _exact_attention(case, s)


def _turns(case, positions):
    """exp(i angle) of every rotated pair and the two index lists, from the definition, axis by axis."""
    first, second, turns, at = [], [], [], 0
    for a, d in enumerate(int(n) for n in case["axes"].split("+")):
        j = torch.arange(d // 2, dtype=torch.float64, device="cuda")
        angle = positions[..., a].double().unsqueeze(-1) * torch.exp(-2.0 * j / d * math.log(_THETA))
        turns.append(torch.polar(torch.ones_like(angle), angle))
        n = j.long()
        first.append(at + (2 * n if case["interleaved"] else n))
        second.append(at + (2 * n + 1 if case["interleaved"] else n + d // 2))
        at += d
    return torch.cat(first), torch.cat(second), torch.cat(turns, -1).unsqueeze(-2)


def _exact_norm(case, x, w, positions):
    first, second, turn = _turns(case, positions)
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.double()
    z = torch.complex(y[..., first], y[..., second]) * turn
    return y.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)


def _exact_norm_grad(case, dy, x, w, positions):
    first, second, turn = _turns(case, positions)
    x, dy = x.double(), dy.double()
    z = torch.complex(dy[..., first], dy[..., second]) * turn.conj()
    g = dy.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)
    n = x.shape[-1]
    size = torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS)
    along = (g * w.double() * x).sum(-1, keepdim=True)
    dx = g * w.double() / size - x * along / (n * size ** 3)
    return dx, (g * x / size).reshape(-1, n).sum(0)


def _exact_attention(case, s):
    grad = case["op"].endswith("grad")
    B, Lq, Hq, Bk, Lk, Hk, D = (case[n] for n in ("B", "Lq", "Hq", "Bk", "Lk", "Hk", "D"))
    G, per = Hq // Hk, B // Bk
    out = torch.zeros((B, Lq, Hq, D), dtype=torch.float64, device="cuda")
    dq, dk, dv = (torch.zeros_like(out), *(torch.zeros((Bk, Lk, Hk, D), dtype=torch.float64, device="cuda")
                                           for _ in range(2))) if grad else (None, None, None)
    keep = torch.ones((Bk, Lk), dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        keep &= torch.arange(Lk, device="cuda") < s["lengths"].reshape(-1, 1)
    if s["mask"] is not None:
        keep &= s["mask"]
    step = max(1, int(1.5e8) // max(1, per * Lq * Lk))               # contexts at a time, one query head after another
    for b in range(0, Bk, step):
        c = slice(b, min(b + step, Bk))
        n = c.stop - c.start
        rows = slice(c.start * per, c.stop * per)
        hidden = ~keep[c][:, None, :]
        for h in range(Hq):
            q = s["q"][rows, :, h].double().reshape(n, per * Lq, D)
            k, v = s["k"][c, :, h // G].double(), s["v"][c, :, h // G].double()
            score = torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(D)
            score = score.masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1).nan_to_num(0.0)
            o = torch.bmm(p, v)
            out[rows, :, h] = o.reshape(n * per, Lq, D)
            if grad:
                do = s["out_grad"][rows, :, h].double().reshape(n, per * Lq, D)
                dp = torch.bmm(do, v.transpose(1, 2).contiguous())
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[rows, :, h] = torch.bmm(ds, k).reshape(n * per, Lq, D)
                dk[c, :, h // G] += torch.bmm(ds.transpose(1, 2).contiguous(), q)
                dv[c, :, h // G] += torch.bmm(p.transpose(1, 2).contiguous(), do)
    return [out, dq, dk, dv] if grad else [out]
