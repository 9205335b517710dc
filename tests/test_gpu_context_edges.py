"""Edges of the context operators on the GPU: few keys left by a mask, scales, strides, what one rounding more would show,
and graphs of the widest heads (plain 64-bit forms and derived bounds: tests/context_oracle.py)."""
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


def chosen(g, contexts, keys, n):
    """A mask [contexts, keys] of n[c] keys at random places."""
    m = torch.zeros((contexts, keys), dtype=torch.bool, device="cuda")
    for c in range(contexts):
        m[c, torch.randperm(keys, generator=g, device="cuda")[:n[c]]] = True
    return m


# ------------------------------------------------------------------------------------------------- few keys
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows,Lk", [(3, 2), (200, 2), (3, 70), (200, 70), (3, 1100), (200, 1100), (40, 5000)])
def test_one_key_left_by_a_mask(C, dtype, rows, Lk, D):
    """P is 1 whatever q and k are, so dq and dk are 0 exactly, also where the one key is what a mask leaves of many (and,
    in the same batch, where it leaves none or two: those contexts' gradients are as ever)."""
    g = gen(31)
    q, do = normal(g, 4, rows, 4, D, dtype=dtype), normal(g, 4, rows, 4, D, dtype=dtype)
    k, v = 3 * normal(g, 4, Lk, 2, D, dtype=dtype), normal(g, 4, Lk, 2, D, dtype=dtype)
    m = chosen(g, 4, Lk, [1, 0, 2, 1])
    m[3] = False
    m[3, -1] = True                                    # the last key of all
    kw = dict(context_mask=m)
    out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
    dq, dk, dv = C.cross_attention_grad(do, q, k, v, out, lse, **kw)
    one = [0, 3]
    assert float(dq[one].abs().max()) == 0.0 and float(dk[one].abs().max()) == 0.0
    want = O.attention(q, k, v, out_grad=do, **kw)
    for name, got in dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv).items():
        O.check(name, got, *want[name])
    assert float(dq[2].abs().max()) > 0.0 and float(dv[one].abs().max()) > 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows", [20, 200])
def test_few_keys_left_by_a_mask(C, dtype, rows):
    """Two or three keys of a context of one tile: dP - delta cancels, but dQ and dK stay as exact as their own rounding
    and that of dS: two roundings of at most u, in norm u / sqrt(3) each, none amplified (1.5 for their spread)."""
    g = gen(32)
    q, do = normal(g, 64, rows, 2, 64, dtype=dtype), normal(g, 64, rows, 2, 64, dtype=dtype)
    k, v = normal(g, 64, 60, 2, 64, dtype=dtype), normal(g, 64, 60, 2, 64, dtype=dtype)
    kw = dict(context_mask=chosen(g, 64, 60, [2 + c % 2 for c in range(64)]))
    want = O.attention(q, k, v, out_grad=do, **kw)
    out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
    u = O.half_step(dtype)
    for name, got in zip(("dq", "dk", "dv"), C.cross_attention_grad(do, q, k, v, out, lse, **kw)):
        O.check(name, got, *want[name])
        off = float((got.double() - want[name][0]).norm() / want[name][0].norm())
        assert off <= 1.5 * math.sqrt(2.0 / 3.0) * u, (name, off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows", [20, 200])
def test_few_keys_left_of_a_long_context(C, dtype, rows):
    """Two or three keys of a context of many tiles: delta comes from the rounded output, so dS = P (dP - delta) carries
    that rounding too.  Per element it is u |dO O| summed over D, against |dS|: the derived bounds hold, and in norm the
    sum of three roundings where the terms that cancel are at most four times dS."""
    g = gen(33)
    q, do = normal(g, 16, rows, 2, 64, dtype=dtype), normal(g, 16, rows, 2, 64, dtype=dtype)
    k, v = normal(g, 16, 900, 2, 64, dtype=dtype), normal(g, 16, 900, 2, 64, dtype=dtype)
    kw = dict(context_mask=chosen(g, 16, 900, [2 + c % 2 for c in range(16)]))
    want = O.attention(q, k, v, out_grad=do, **kw)
    out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
    u = O.half_step(dtype)
    for name, got in zip(("dq", "dk", "dv"), C.cross_attention_grad(do, q, k, v, out, lse, **kw)):
        O.check(name, got, *want[name])
        off = float((got.double() - want[name][0]).norm() / want[name][0].norm())
        assert off <= math.sqrt((2.0 + 16.0) / 3.0) * u, (name, off)


# ------------------------------------------------------------------------------------------------- scales
@pytest.mark.parametrize("rows,keys", [(5, 40), (200, 300)])
def test_scales_far_from_one(C, rows, keys):
    """A scale of 0 is an average whatever the scores are, and a tiny one meets scores that make up for it."""
    g = gen(34)
    for size, scale in ((1e14, 0.0), (2.0 ** 52, 2.0 ** -104), (2.0 ** 52, -2.0 ** -104), (2.0 ** 60, 2.0 ** -121)):
        q, k = size * normal(g, 2, rows, 2, 32), size * normal(g, 2, keys, 2, 32)
        v, do = normal(g, 2, keys, 2, 32), normal(g, 2, rows, 2, 32)
        kw = dict(scale=scale, context_lengths=torch.tensor([keys, keys // 2], device="cuda"))
        want = O.attention(q, k, v, out_grad=do, **kw)
        out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
        O.check("out", out, *want["out"])
        O.check("lse", lse, *want["lse"])
        for name, got in zip(("dq", "dk", "dv"), C.cross_attention_grad(do, q, k, v, out, lse, **kw)):
            O.check(name, got, *want[name])


# ------------------------------------------------------------------------------------------------- strides
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_rows_of_keys_far_apart(C, dtype):
    """Rows of k and v 8 MiB and more apart (a slice of a very wide buffer): as their contiguous copies."""
    g, e = gen(35), torch.finfo(dtype).bits // 8
    for step in ((8 << 20) // e, (9 << 20) // e):
        far = torch.empty(7 * step, dtype=dtype, device="cuda")
        k, v = far.as_strided((1, 6, 2, 32), (step, step, 32, 1)), far.as_strided((1, 6, 2, 32), (step, step, 32, 1), 64)
        for x in (k, v):
            x.copy_(normal(g, 1, 6, 2, 32, dtype=dtype))
        q = normal(g, 3, 5, 4, 32, dtype=dtype)
        a = C.cross_attention(q, k, v, return_lse=True)
        b = C.cross_attention(q, k.contiguous(), v.contiguous(), return_lse=True)
        for x, y in zip((*a, *C.cross_attention_grad(q, q, k, v, *a)),
                        (*b, *C.cross_attention_grad(q, q, k.contiguous(), v.contiguous(), *b))):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [5, 200])
def test_rows_of_keys_that_overlap(C, dtype, rows):
    """Keys that repeat one row in memory (expanded), or slide over it: as their contiguous copies, infinities included."""
    g = gen(36)
    q = normal(g, 2, rows, 2, 32, dtype=dtype)
    one = normal(g, 2, 1, 2, 32, dtype=dtype)
    one[0, 0, 0, 3] = math.inf
    slide = normal(g, 400, dtype=dtype).as_strided((1, 41, 1, 32), (400, 8, 32, 1))
    for x in (one.expand(2, 70, 2, 32), one, slide):
        k = torch.nan_to_num(x, posinf=1.0)
        a = C.cross_attention(q, k, x, return_lse=True)
        assert torch.equal(torch.isinf(a[0]), torch.isinf(x[:, :1].expand(2, 1, 2, 32)).expand_as(a[0]))
        b = C.cross_attention(q, k.contiguous(), x.contiguous(), return_lse=True)
        c = C.cross_attention(q, x.new_zeros(()).expand(x.shape) + k, x.contiguous(), return_lse=True)
        for y, z, w in zip(a, b, c):
            assert torch.equal(y, z) and torch.equal(y, w)


# ------------------------------------------------------------------------------------------------- groups and widths
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(3, 17, 6, 3, 70, 2, 32), (4, 9, 15, 1, 300, 3, 64), (2, 40, 36, 2, 33, 3, 16),
                                   (3, 1, 14, 3, 500, 2, 128), (5, 50, 5, 1, 130, 1, 8), (2, 3, 300, 1, 90, 1, 16),
                                   (2, 65, 2, 2, 200, 2, 56), (2, 64, 2, 2, 200, 2, 104)], ids=str)
@pytest.mark.parametrize("masked", [False, True])
def test_groups_that_do_not_divide_a_tile(C, dtype, shape, masked):
    """Query heads a key head of 3, 5, 7, 12 and 300, and widths between the compiled ones: rows of a token cross tiles."""
    B, Lq, Hq, Ck, Lk, Hk, D = shape
    g = gen(39)
    q, do = normal(g, B, Lq, Hq, D, dtype=dtype), normal(g, B, Lq, Hq, D, dtype=dtype)
    k, v = normal(g, Ck, Lk, Hk, D, dtype=dtype), normal(g, Ck, Lk, Hk, D, dtype=dtype)
    kw = {}
    if masked:
        kw = dict(context_mask=torch.rand((Ck, Lk), generator=g, device="cuda") > 0.5,
                  query_lengths=torch.randint(0, Lq + 1, (B,), generator=g, device="cuda"),
                  context_lengths=torch.randint(1, Lk + 1, (Ck,), generator=g, device="cuda"))
    want = O.attention(q, k, v, out_grad=do, **kw)
    out, lse = C.cross_attention(q, k, v, return_lse=True, **kw)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *C.cross_attention_grad(do, q, k, v, out, lse, **kw))):
        O.check(name, got, *want[name])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_queries_expanded_over_batch_length_and_heads(C, dtype):
    """q and out_grad that repeat in memory: the bits of their contiguous copies."""
    g = gen(40)
    k, v = normal(g, 1, 90, 2, 32, dtype=dtype), normal(g, 1, 90, 2, 32, dtype=dtype)
    for shape in ((1, 20, 4, 32), (5, 1, 4, 32), (5, 20, 1, 32), (1, 1, 4, 32), (1, 1, 1, 32)):
        for full in ((5, 20, 4, 32), (5, 1, 4, 32)):
            if any(a not in (1, b) for a, b in zip(shape, full)):
                continue
            q, do = normal(g, *shape, dtype=dtype).expand(full), normal(g, *shape, dtype=dtype).expand(full)
            a = C.cross_attention(q, k, v, return_lse=True)
            b = C.cross_attention(q.contiguous(), k, v, return_lse=True)
            for x, y in zip((*a, *C.cross_attention_grad(do, q, k, v, *a)),
                            (*b, *C.cross_attention_grad(do.contiguous(), q.contiguous(), k, v, *b))):
                assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------- roundings
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("shape", [(4, 22, 8, 4, 333, 4, 64), (2, 300, 4, 2, 700, 2, 128), (64, 13, 2, 1, 64, 2, 32),
                                   (16, 1, 8, 16, 600, 2, 128)], ids=str)
def test_errors_are_those_of_two_roundings(C, dtype, shape):
    """Every output is rounded once, and P (out, dv) or dS (dq, dk) before its product.  A rounding to a type of half step u
    is uniform in a binade: u / sqrt(3) in norm, times the lower end of the value's binade over the value.  That ratio is
    0.737 for normal values (the root of E[4^floor(log2 |x|)]), so a rounding is 0.425 u, two are 0.602 u and three 0.737 u.
    0.67 u is half way to a third."""
    B, Lq, Hq, Ck, Lk, Hk, D = shape
    g = gen(37)
    q, do = normal(g, B, Lq, Hq, D, dtype=dtype), normal(g, B, Lq, Hq, D, dtype=dtype)
    k, v = normal(g, Ck, Lk, Hk, D, dtype=dtype), normal(g, Ck, Lk, Hk, D, dtype=dtype)
    want = O.attention(q, k, v, out_grad=do)
    out, lse = C.cross_attention(q, k, v, return_lse=True)
    u = O.half_step(dtype)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *C.cross_attention_grad(do, q, k, v, out, lse))):
        off = float((got.double() - want[name][0]).norm() / want[name][0].norm())
        print(shape, name, f"{off / u:.3f} u", flush=True)
        assert off <= 0.67 * u, (name, off / u)


# ------------------------------------------------------------------------------------------------- graphs
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [2, 100])
def test_wide_heads_captured_and_replayed(C, dtype, rows):
    """Heads of 128 take more than 64 KiB of LDS, which a launch asks for beforehand: in a capture too, and replays on new
    inputs with eager work between them equal the eager results."""
    g = gen(38)
    shape = dict(q=(2, rows, 4, 128), k=(2, 1500, 2, 128), v=(2, 1500, 2, 128))
    buf = {n: normal(g, *s, dtype=dtype) for n, s in shape.items()}
    mask = torch.rand((2, 1500), generator=g, device="cuda") > 0.2

    def work():
        out, lse = C.cross_attention(buf["q"], buf["k"], buf["v"], return_lse=True, context_mask=mask)
        return [out, *C.cross_attention_grad(out, buf["q"], buf["k"], buf["v"], out, lse, context_mask=mask)]
    graph = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        outs = work()
    for n in range(3):
        for name in buf:
            buf[name].copy_(normal(g, *shape[name], dtype=dtype))
        mask.copy_(torch.rand((2, 1500), generator=g, device="cuda") > 0.2 + 0.2 * n)
        want = [x.clone() for x in work()]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, outs):
            assert torch.equal(x, y)
        work()
