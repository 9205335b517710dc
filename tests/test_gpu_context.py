"""Context operators on the GPU against plain 64-bit forms (tests/context_oracle.py: values and derived bounds)."""
import math

import pytest
import torch

import context_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda x: str(x).replace("torch.", "") if isinstance(x, torch.dtype) else None   # noqa: E731


@pytest.fixture(scope="module")
def C():
    from ecnf_amd import context
    return context


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def say(*a):
    print(*a, flush=True)


# ------------------------------------------------------------------------------------------------- norm + rotation
NORM = [  # B, Lq, Hq, C, Lk, Hk, D, axes, interleaved
    (1, 1, 1, 0, 0, 0, 2, (2,), False),
    (2, 13, 2, 1, 64, 2, 32, (32,), False),
    (3, 22, 4, 3, 37, 4, 16, (8, 8), False),
    (2, 5, 3, 2, 7, 1, 128, (32, 48, 48), False),
    (2, 5, 3, 2, 7, 1, 128, (32, 48, 48), True),
    (1, 9, 2, 1, 3, 5, 96, (2, 6, 10), False),          # odd halves, a tail of dims that do not turn
    (1, 9, 2, 1, 3, 5, 96, (2, 6, 10, 20), True),
    (2, 3, 33, 1, 1, 1, 64, (60,), False),              # a rest of 4 dims
    (7, 401, 2, 1, 0, 0, 24, (12, 12), False),          # head_dim that fills no power of two lanes
    (1, 3000, 5, 1, 2049, 1, 128, (128,), False),       # several tiles a block in the backward pass
]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("B,Lq,Hq,Ck,Lk,Hk,D,axes,inter", NORM)
def test_norm_rotary(C, dtype, B, Lq, Hq, Ck, Lk, Hk, D, axes, inter):
    say("norm", dtype, B, Lq, Hq, Ck, Lk, Hk, D, axes, inter)
    g = gen(D + Lq)
    q, dq = normal(g, B, Lq, Hq, D, dtype=dtype), normal(g, B, Lq, Hq, D, dtype=dtype)
    A = len(axes)
    qp = torch.randint(-40, 60000, (B, Lq, A), generator=g, device="cuda", dtype=torch.int32)
    qw = 1 + 0.1 * normal(g, D)
    k = dk = kp = kw = None
    if Lk:
        k, dk = normal(g, Ck, Lk, Hk, D, dtype=dtype), normal(g, Ck, Lk, Hk, D, dtype=dtype)
        kp, kw = 100 * normal(g, Lk, A), 1 + 0.1 * normal(g, D, dtype=dtype)   # real, the same for every context
    opt = dict(axes=axes, theta=500.0, eps=1e-5, interleaved=inter)
    kwargs = dict(q_positions=qp, k_positions=kp, q_weight=qw, k_weight=kw, **opt)
    y, z = C.qk_norm_rotary(q, k, **kwargs)
    O.check("q", y, *O.norm_rotary(q, qw, qp, **opt)["y"])
    dx, dz, dw, dv = C.qk_norm_rotary_grad(dq, dk, q, k, **kwargs)
    want = O.norm_rotary(q, qw, qp, grad=dq, **opt)
    O.check("dq", dx, *want["dx"])
    O.check("dq_weight", dw, *want["dw"])
    if k is None:
        assert z is None and dz is None and dv is None
    else:
        O.check("k", z, *O.norm_rotary(k, kw, kp, **opt)["y"])
        want = O.norm_rotary(k, kw, kp, grad=dk, **opt)
        O.check("dk", dz, *want["dx"])
        O.check("dk_weight", dv, *want["dw"])
        assert dv.dtype == kw.dtype and dz.dtype == dtype


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_norm_rotary_strides_no_weight_far_positions(C, dtype):
    """q and k as slices of one projection, of odd alignment; no weights; int64 and huge positions."""
    g = gen(3)
    big = normal(g, 2, 11, 3, 2, 67, dtype=dtype)
    q, k = big[:, :, :, 0, 1:65], big[:, ::2, :, 1, 3:67]
    qp = torch.randint(0, 2 ** 40, (11, 1), generator=g, device="cuda", dtype=torch.int64)
    kp = torch.tensor([[0.0], [1e7], [-1e7], [3.5], [1e-3], [2.0 ** 24]], device="cuda")
    opt = dict(axes=(64,), theta=10000.0)
    # the oracle's angle p theta^(-2j/d) in 64 bits is itself off by 2^-53 of it, up to 2^40: as a part of a turn
    for x, p, y in zip((q, k), (qp, kp), C.qk_norm_rotary(q, k, q_positions=qp, k_positions=kp, **opt)):
        value, bound = O.norm_rotary(x, None, p, **opt)["y"]
        O.check("y", y, value, bound + 4 * 2.0 ** -13 * value.abs().amax(-1, keepdim=True) * (p.abs().max() > 2 ** 30))
    dq, dk, dw, dv = C.qk_norm_rotary_grad(big[:, :, :, 1, 2:66], big[:, ::2, :, 0, :64], q, k, q_positions=qp % 1000,
                                           k_positions=kp, **opt)
    assert dw is None and dv is None
    O.check("dq", dq, *O.norm_rotary(q, None, qp % 1000, grad=big[:, :, :, 1, 2:66], **opt)["dx"])
    O.check("dk", dk, *O.norm_rotary(k, None, kp, grad=big[:, ::2, :, 0, :64], **opt)["dx"])


def test_norm_rotary_differences(C):
    """The gradient against central differences of the forward pass (fp32, along random directions)."""
    g = gen(4)
    q, w = normal(g, 1, 3, 2, 16), 1 + 0.1 * normal(g, 16)
    dy, pos = normal(g, 1, 3, 2, 16), 10 * normal(g, 1, 3, 2)
    opt = dict(q_positions=pos, axes=(8, 6))
    dx, _, dw, _ = C.qk_norm_rotary_grad(dy, None, q, q_weight=w, **opt)
    f = lambda x, ww: (C.qk_norm_rotary(x, q_weight=ww, **opt)[0].double() * dy.double()).sum()   # noqa: E731
    h = 2.0 ** -7
    for _ in range(4):
        a, b = normal(g, 1, 3, 2, 16), normal(g, 16)
        # third derivatives of x / rms are O(1) for rows of O(1): h^2 |a|^3; fp32 values of sum |dy y|: 2^-22 / h of it
        num = (f(q + h * a, w + h * b) - f(q - h * a, w - h * b)) / (2 * h)
        ana = (dx.double() * a.double()).sum() + (dw.double() * b.double()).sum()
        tol = 4 * h * h * float(a.abs().max()) ** 3 * float(dy.abs().sum()) + 2.0 ** -22 / h * float(dy.abs().sum())
        assert abs(float(num - ana)) < tol


def test_norm_rotary_zero_rows(C):
    """A zero row has no direction: the output is 0 and the gradient is w g / sqrt(eps), finite."""
    q = torch.zeros((1, 2, 1, 8), device="cuda")
    q[0, 1] = 1.0
    pos = torch.ones((2, 1), device="cuda", dtype=torch.int32)
    y, _ = C.qk_norm_rotary(q, q_positions=pos, axes=(8,))
    assert float(y[0, 0].abs().max()) == 0.0
    g = torch.ones_like(q)
    dx, *_ = C.qk_norm_rotary_grad(g, None, q, q_positions=pos, axes=(8,))
    O.check("dx", dx, *O.norm_rotary(q, None, pos, (8,), grad=g)["dx"])


# ------------------------------------------------------------------------------------------------- cross attention
ATT = [  # B, Lq, Hq, C, Lk, Hk, D
    (1, 1, 1, 1, 1, 1, 8),
    (2, 13, 2, 1, 64, 2, 32),
    (3, 22, 4, 3, 37, 4, 16),
    (2, 1, 8, 2, 333, 2, 128),
    (1, 70, 4, 1, 130, 1, 64),
    (2, 33, 6, 2, 65, 3, 96),
    (1, 128, 2, 1, 129, 2, 128),
    (2, 300, 1, 1, 700, 1, 40),
    (1, 5, 32, 1, 4097, 4, 128),         # few rows, many keys: split over the keys
    (130, 31, 2, 1, 21, 1, 72),          # many rows, few keys: the gradients split over the rows
    (1, 257, 8, 1, 2050, 8, 64),
    (4, 4, 4, 4, 0, 2, 32),              # contexts without keys
]


def attention_case(C, dtype, shape, lengths, mask, queries, seed=0, scale=None, grads=1.0):
    B, Lq, Hq, Ck, Lk, Hk, D = shape
    g = gen(seed)
    q, do = normal(g, B, Lq, Hq, D, dtype=dtype), (grads * normal(g, B, Lq, Hq, D)).to(dtype)
    k, v = normal(g, Ck, Lk, Hk, D, dtype=dtype), normal(g, Ck, Lk, Hk, D, dtype=dtype)
    kw = dict(scale=scale)
    if lengths:
        n = torch.randint(0, Lk + 1, (Ck,), generator=g, device="cuda", dtype=torch.int32)
        if Ck > 1:
            n[0], n[1] = 0, Lk
        kw["context_lengths"] = n
    if mask:
        kw["context_mask"] = torch.rand((Ck, Lk), generator=g, device="cuda") > 0.4
        if Ck > 2:
            kw["context_mask"][2] = False
    if queries:
        kw["query_lengths"] = torch.randint(0, Lq + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    clean = (q.clone(), k.clone(), v.clone(), do.clone())
    # what lies behind a mask or a length holds anything: NaN, infinities, the type's lowest value
    low = torch.finfo(dtype).min
    if lengths or mask:
        keep = torch.ones((Ck, Lk), dtype=torch.bool, device="cuda")
        if lengths:
            keep &= torch.arange(Lk, device="cuda")[None] < kw["context_lengths"][:, None]
        if mask:
            keep &= kw["context_mask"]
        bad = torch.tensor([math.nan, math.inf, -math.inf, low], device="cuda").to(dtype)
        fill = bad[torch.arange(Lk, device="cuda") % 4][None, :, None, None].expand_as(k)
        k, v = torch.where(keep[:, :, None, None], k, fill), torch.where(keep[:, :, None, None], v, fill)
    if queries:
        live = torch.arange(Lq, device="cuda")[None] < kw["query_lengths"][:, None]
        q = torch.where(live[:, :, None, None], q, torch.full_like(q, math.nan))
        do = torch.where(live[:, :, None, None], do, torch.full_like(do, math.nan))
    want = O.attention(*clean[:3], out_grad=clean[3], **kw)
    out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
    dq, dk, dv = C.cross_attention_grad(do, q, k, v, out, lse, **kw)
    for name, got in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
        O.check(name, got, *want[name])
        if name != "lse":
            assert got.dtype == dtype
    return out, lse, dq, dk, dv


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", ATT, ids=str)
def test_attention(C, dtype, shape):
    say("attention", dtype, shape)
    attention_case(C, dtype, shape, False, False, False)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("lengths,mask,queries", [(True, False, False), (False, True, False), (True, True, True)])
@pytest.mark.parametrize("shape", [(5, 13, 2, 5, 64, 2, 32), (4, 22, 4, 4, 333, 2, 64), (3, 1, 8, 3, 700, 2, 128),
                                   (6, 33, 2, 1, 130, 1, 48), (3, 200, 2, 3, 129, 2, 128)], ids=str)
def test_attention_masks(C, dtype, shape, lengths, mask, queries):
    say("masks", dtype, shape, lengths, mask, queries)
    attention_case(C, dtype, shape, lengths, mask, queries, seed=1)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("grads", [1e-3, 300.0])
@pytest.mark.parametrize("shape", [(1, 40, 2, 1, 6000, 2, 64), (1, 4, 2, 1, 6000, 1, 32), (1, 3000, 2, 1, 20, 2, 128)], ids=str)
def test_attention_small_and_large_gradients(C, dtype, grads, shape):
    """dS far below and far above 1 (in fp16 below its subnormals): long contexts make P small, the loss scales dO."""
    attention_case(C, dtype, shape, False, False, False, seed=2, grads=grads)


def test_attention_gradients_of_very_different_rows(C):
    """fp16: rows whose gradients differ by 2^20 share a key's sums, and keys far apart a row's."""
    g = gen(14)
    q, k, v = (normal(g, 1, n, 2, 64, dtype=torch.float16) for n in (200, 700, 700))
    do = (normal(g, 1, 200, 2, 64) * 2.0 ** torch.linspace(-14, 6, 200, device="cuda").round()[None, :, None, None]).half()
    v = (v.float() * 2.0 ** torch.linspace(5, -5, 700, device="cuda").round()[None, :, None, None]).half()
    want = O.attention(q, k, v, out_grad=do)
    out, lse = C.cross_attention(q, k, v, return_lse=True)
    for name, got in zip(("dq", "dk", "dv"), C.cross_attention_grad(do, q, k, v, out, lse)):
        O.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows", [20, 200])
def test_attention_few_keys(C, dtype, rows):
    """Two or three keys: dP - delta cancels, but dQ and dK stay as exact as their own rounding and that of dS."""
    g = gen(15)
    q, do = normal(g, 64, rows, 2, 64, dtype=dtype), normal(g, 64, rows, 2, 64, dtype=dtype)
    k, v = normal(g, 64, 3, 2, 64, dtype=dtype), normal(g, 64, 3, 2, 64, dtype=dtype)
    n = torch.arange(64, device="cuda", dtype=torch.int32) % 2 + 2
    want = O.attention(q, k, v, context_lengths=n, out_grad=do)
    out, lse = C.cross_attention(q, k, v, return_lse=True, context_lengths=n)
    u = O.half_step(dtype)
    for name, got in zip(("dq", "dk", "dv"), C.cross_attention_grad(do, q, k, v, out, lse, context_lengths=n)):
        O.check(name, got, *want[name])
        # two roundings of at most u (uniform in a binade: their rms is at most u / sqrt(3) each), none amplified
        off = float((got.double() - want[name][0]).norm() / want[name][0].norm())
        assert off <= 1.5 * math.sqrt(2.0 / 3.0) * u, (name, off)


def test_attention_one_key(C):
    """One key takes all: out is v up to the rounding of exp2(s - m) = 1 (s sc - m sc, one of them rounded) and its division,
    dV the sum of dO, and dS is 0 up to the roundings of equal products."""
    g = gen(16)
    for dtype in TYPES:
        q, do = normal(g, 2, 40, 2, 32, dtype=dtype), normal(g, 2, 40, 2, 32, dtype=dtype)
        k, v = normal(g, 2, 1, 2, 32, dtype=dtype), normal(g, 2, 1, 2, 32, dtype=dtype)
        want = O.attention(q, k, v, out_grad=do)
        out, lse = C.cross_attention(q, k, v, return_lse=True)
        grads = C.cross_attention_grad(do, q, k, v, out, lse)
        for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            O.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,Lk", [(3, 1), (200, 1), (200, 70), (3, 600)])
def test_attention_one_key_has_no_score_gradient(C, dtype, rows, Lk):
    """A context of one key: P is 1 whatever q and k are, so dq and dk are 0 exactly, and dv is the sum of out_grad."""
    g = gen(25)
    q, do = normal(g, 3, rows, 4, 64, dtype=dtype), normal(g, 3, rows, 4, 64, dtype=dtype)
    k, v = 3 * normal(g, 3, Lk, 4, 64, dtype=dtype), normal(g, 3, Lk, 4, 64, dtype=dtype)
    n = torch.ones(3, dtype=torch.int32, device="cuda")
    out, lse = C.cross_attention(q, k, v, context_lengths=n, return_lse=True)
    dq, dk, dv = C.cross_attention_grad(do, q, k, v, out, lse, context_lengths=n)
    assert float(dq.abs().max()) == 0.0 and float(dk.abs().max()) == 0.0
    # P = 2^(s - lse) and lse, natural log, round at |s|: |P - 1| <= 2^-21 |s|; rows * 2^-23 for the sums
    want, size = do.double().sum(1), do.double().abs().sum(1)
    s = float(lse.abs().max())
    tol = (2.0 ** -21 * s + rows * 2.0 ** -23 + torch.finfo(dtype).eps) * size
    assert bool(((dv[:, 0].double() - want).abs() <= tol).all()) and float(dv[:, 1:].abs().sum()) == 0.0


def test_attention_sharp_scores(C):
    """Scores far apart: one key takes everything, in a tile that comes late (the running maximum moves every tile)."""
    q = torch.full((1, 2, 1, 32), 2.0, device="cuda")
    k = torch.arange(1000, device="cuda", dtype=torch.float32)[None, :, None, None].expand(1, 1000, 1, 32) * 0.05
    v = normal(gen(5), 1, 1000, 1, 32)
    out, lse = C.cross_attention(q, k.contiguous(), v, return_lse=True, scale=1.0)
    want = O.attention(q, k, v, scale=1.0)
    O.check("out", out, *want["out"])
    O.check("lse", lse, *want["lse"])


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_attention_scales(C, scale):
    """No scale (an average over the allowed keys), a negative one and a large one."""
    for dtype in TYPES:
        attention_case(C, dtype, (3, 20, 2, 3, 150, 2, 32), True, True, False, seed=3, scale=scale)
        attention_case(C, dtype, (1, 70, 2, 1, 150, 2, 32), False, False, False, seed=3, scale=scale)


def test_attention_differences(C):
    """The gradients against central differences of the forward pass (fp32, along random directions)."""
    g = gen(6)
    q, k, v, do = normal(g, 2, 5, 4, 16), normal(g, 1, 9, 2, 16), normal(g, 1, 9, 2, 16), normal(g, 2, 5, 4, 16)
    f = lambda *x: (C.cross_attention(*x).double() * do.double()).sum()   # noqa: E731
    out, lse = C.cross_attention(q, k, v, return_lse=True)
    grads = C.cross_attention_grad(do, q, k, v, out, lse)
    h = 2.0 ** -8
    for n, x in enumerate((q, k, v)):
        a = normal(g, *x.shape)
        args = [q, k, v]
        args[n] = x + h * a
        up = f(*args)
        args[n] = x - h * a
        num = float(up - f(*args)) / (2 * h)
        ana = float((grads[n].double() * a.double()).sum())
        # third derivative of a softmax average along unit-size directions: a few |v| |s'|^3 with |s'| <= |a| |k| / 4
        tol = 30 * h * h * float(do.abs().sum()) + 2.0 ** -22 / h * float(do.abs().sum())
        assert abs(num - ana) < tol, (n, num, ana, tol)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_attention_strides_and_alignment(C, dtype):
    """q, k and v as slices of fused projections (other orders of dimensions, rows off 16-byte boundaries) and expanded
    over heads and batch equal their contiguous copies, bit by bit."""
    g = gen(7)
    kv = normal(g, 2, 3, 50, 2, 72, dtype=dtype)                      # [batch, heads, length, k | v, 72]
    k, v = kv[:, :, :, 0, 3:67].transpose(1, 2), kv[:, :, :, 1, :64].transpose(1, 2)
    q = normal(g, 20, 2, 3, 64, dtype=dtype).transpose(0, 1)
    do = normal(g, 2, 20, 3, 65, dtype=dtype)[..., 1:]
    a = C.cross_attention(q, k, v, return_lse=True)
    b = C.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), return_lse=True)
    ga = C.cross_attention_grad(do, q, k, v, *a)
    gb = C.cross_attention_grad(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), *b)
    for x, y in zip((*a, *ga), (*b, *gb)):
        assert torch.equal(x, y)
    e = normal(g, 1, 50, 1, 64, dtype=dtype).expand(2, 50, 3, 64)
    assert torch.equal(C.cross_attention(q, e, e), C.cross_attention(q, e.contiguous(), e.contiguous()))
    d = normal(g, 2, 20, 64, 3, dtype=dtype).transpose(2, 3)          # last dimension strided: copied
    assert torch.equal(C.cross_attention(d, k, v), C.cross_attention(d.contiguous(), k, v))


def test_attention_same_bits_and_streams(C):
    """Repeated calls, calls on another stream, and two at once give the same bits."""
    g = gen(8)
    q, k, v = (normal(g, *s, dtype=torch.bfloat16) for s in ((2, 40, 8, 64), (2, 3000, 2, 64), (2, 3000, 2, 64)))
    first = C.cross_attention(q, k, v, return_lse=True)
    grads = C.cross_attention_grad(q, q, k, v, *first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            o = C.cross_attention(q, k, v, return_lse=True)
            got.append((*o, *C.cross_attention_grad(q, q, k, v, *o)))
    torch.cuda.synchronize()
    for r in got:
        for x, y in zip(r, (*first, *grads)):
            assert torch.equal(x, y)


def test_captured_and_replayed(C):
    """Norm, attention and their gradients in one graph, replayed on new inputs with eager work between."""
    g = gen(9)
    shape = dict(q=(3, 22, 4, 32), k=(1, 600, 2, 32), v=(1, 600, 2, 32))
    buf = {n: normal(g, *s) for n, s in shape.items()}
    w = 1 + 0.1 * normal(g, 32)
    qp, kp = torch.arange(22, device="cuda", dtype=torch.int32)[:, None], torch.arange(600, device="cuda", dtype=torch.int32)[:, None]
    opt = dict(q_positions=qp, k_positions=kp, q_weight=w, k_weight=w, axes=(32,))

    def work():
        q, k = C.qk_norm_rotary(buf["q"], buf["k"], **opt)
        out, lse = C.cross_attention(q, k, buf["v"], return_lse=True)
        dq, dk, dv = C.cross_attention_grad(out, q, k, buf["v"], out, lse)
        return [out, dv, *C.qk_norm_rotary_grad(dq, dk, buf["q"], buf["k"], **opt)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    with torch.cuda.graph(other):
        outs2 = work()
    for n in range(3):
        for name in buf:
            buf[name].copy_(normal(g, *shape[name]))
        want = [x.clone() for x in work()]
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(want, outs, outs2):
            assert torch.equal(x, y) and torch.equal(x, z)
        work()


def test_lengths_outside_the_range_are_clamped(C):
    q, k = normal(gen(10), 2, 3, 1, 16), normal(gen(11), 2, 40, 1, 16)
    full = C.cross_attention(q, k, k)[1]
    for n in ([-5, 10 ** 9], [-2 ** 40, 2 ** 40]):
        n = torch.tensor(n, device="cuda")
        for x in (n, n.clamp(-2 ** 31, 2 ** 31 - 1).int()):
            out = C.cross_attention(q, k, k, context_lengths=x)
            assert float(out[0].abs().max()) == 0.0 and torch.equal(out[1], full)


def test_nothing_to_do(C):
    """Empty batches, queries and contexts: shapes, zeros, no launch on empty grids."""
    for B, Lq, Ck, Lk in ((0, 3, 0, 5), (2, 0, 2, 5), (2, 0, 1, 5), (2, 3, 2, 0), (2, 0, 2, 0)):
        q, k = normal(gen(0), B, Lq, 2, 16), normal(gen(0), Ck, Lk, 1, 16)
        if not Ck and B:
            continue
        out, lse = C.cross_attention(q, k, k, return_lse=True)
        dq, dk, dv = C.cross_attention_grad(out, q, k, k, out, lse)
        assert out.shape == q.shape and dk.shape == dv.shape == k.shape
        for x in (out, dq, dk, dv):
            assert not x.numel() or float(x.abs().max()) == 0.0
        w = torch.ones(16, device="cuda")
        p = torch.zeros((Lq, 1), device="cuda")
        dx, _, dw, _ = C.qk_norm_rotary_grad(q, None, q, q_positions=p, q_weight=w, axes=(16,))
        assert dx.shape == q.shape and float(dw.abs().max()) >= 0.0
        if not q.numel():
            assert float(dw.abs().max()) == 0.0


def test_nan_in_a_row_stays_in_the_row(C):
    """A NaN query gives a NaN row and leaves the other rows as they were."""
    g = gen(12)
    q, k, v = normal(g, 1, 40, 2, 32), normal(g, 1, 90, 2, 32), normal(g, 1, 90, 2, 32)
    want = C.cross_attention(q, k, v)
    q[0, 7, 1, 3] = math.nan
    out = C.cross_attention(q, k, v)
    assert bool(torch.isnan(out[0, 7, 1]).all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, 7, 1] = False
    assert torch.equal(out[keep], want[keep])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,keys", [(5, 40), (200, 40), (5, 700), (200, 300)])
def test_nan_gradients_stay_with_their_row(C, dtype, rows, keys):
    """NaN in out_grad: 0 for a row without keys and for keys that no row may read, and the rows beside it as they were."""
    g = gen(13)
    q, do = normal(g, 2, rows, 2, 32, dtype=dtype), normal(g, 2, rows, 2, 32, dtype=dtype)
    k, v = normal(g, 2, keys, 1, 32, dtype=dtype), normal(g, 2, keys, 1, 32, dtype=dtype)
    mask = torch.ones((2, keys), dtype=torch.bool, device="cuda")
    mask[0] = False                                    # no row of molecule 0 has a key
    mask[1, ::3] = False
    out, lse = C.cross_attention(q, k, v, context_mask=mask, return_lse=True)
    want = C.cross_attention_grad(do, q, k, v, out, lse, context_mask=mask)[0]
    do[:, 3, 1] = math.nan
    dq, dk, dv = C.cross_attention_grad(do, q, k, v, out, lse, context_mask=mask)
    assert float(dq[0].abs().max()) == 0.0
    for x in (dk, dv):
        assert float(x[~mask].abs().max()) == 0.0
        assert bool(torch.isnan(x[mask]).all())
    assert bool(torch.isnan(dq[1, 3, 1]).all())
    dq[1, 3, 1] = want[1, 3, 1]
    assert torch.equal(dq, want)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_offsets_past_32_bits(C, dtype):
    """Rows of k, v and q far apart (more than 2^32 bytes from the first to the last): as their contiguous copies."""
    g, e = gen(14), torch.finfo(dtype).bits // 8
    step = (8 << 20) // e - 64                         # elements from one key to the next (the largest is below 8 MiB)
    far = torch.empty(620 * step, dtype=dtype, device="cuda")
    k = far.as_strided((1, 620, 1, 32), (step, step, 32, 1))
    v = far.as_strided((1, 620, 1, 32), (step, step, 32, 1), 32)
    q = far.as_strided((2, 40, 1, 32), (300 * step, 7 * step, 32, 1), 64)
    do = far.as_strided((2, 40, 1, 32), (300 * step, 7 * step, 32, 1), 96)
    for x in (k, v, q, do):
        x.copy_(normal(g, *x.shape, dtype=dtype))
    near = [x.contiguous() for x in (q, k, v, do)]
    pq, pk = torch.arange(40, device="cuda")[:, None], torch.arange(620, device="cuda")[:, None]
    turn = dict(q_positions=pq, k_positions=pk, axes=(32,))

    def run(q, k, v, do):
        o = C.cross_attention(q, k, v, return_lse=True)
        return (*o, *C.cross_attention_grad(do, q, k, v, *o), *C.qk_norm_rotary(q, k, **turn),
                *C.qk_norm_rotary_grad(do, v, q, k, **turn)[:2])
    for a, b in zip(run(q, k, v, do), run(*near)):
        assert torch.equal(a, b)


def test_sizes_out_of_their_range(C):
    x, p = normal(gen(0), 1, 4, 1, 16), torch.zeros((4, 1), device="cuda")
    with pytest.raises(ValueError, match="32-bit"):
        C.qk_norm_rotary(x, q_positions=p, axes=(2 ** 40,))


def test_rows_behind_the_outputs_are_left_alone():
    """The C entry writes its outputs and nothing behind them."""
    import ctypes

    from ecnf_amd import _lib, context as X
    g = gen(13)
    q, k, v = normal(g, 2, 5, 2, 24), normal(g, 2, 77, 2, 24), normal(g, 2, 77, 2, 24)
    pad = 512
    out = torch.full((q.numel() + pad,), 7.0, device="cuda")
    lse = torch.full((20 + pad,), 7.0, device="cuda")
    args = X._attention_args(q, k, v, out[:q.numel()].view(q.shape), None, lse, None, None, None, None, None, None, 0.2)
    n = ctypes.c_size_t()
    _lib.check(_lib.load().ecnf_cross_attention_workspace_size(args, 0, ctypes.byref(n)))
    ws = torch.full((n.value // 4 + pad,), 7.0, device="cuda")
    _lib.check(_lib.load().ecnf_cross_attention(args, ws.data_ptr(), n.value, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert bool((out[q.numel():] == 7.0).all()) and bool((lse[20:] == 7.0).all()) and bool((ws[n.value // 4:] == 7.0).all())
    O.check("out", out[:q.numel()].view(q.shape), *O.attention(q, k, v, scale=0.2)["out"])
