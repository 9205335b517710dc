"""The conditional flow's edges: states in 16 bits, what lies behind lengths and masks, empty batches and contexts, feature
shapes and ids, and the embedding's table across streams."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

from ecnf_amd import CONFIGS, init_params  # noqa: E402
from ecnf_amd import cnf as F  # noqa: E402
from ecnf_amd import context as C  # noqa: E402
from ecnf_amd import train as TR  # noqa: E402
from ecnf_amd.engine import EcnfHandle, SolveOptions  # noqa: E402
from ecnf_amd.params import CNFConfig  # noqa: E402

from test_gpu_context_flow import CTX, build, features, make_context, plain  # noqa: E402

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rel(a, b):
    """|a - b| / |b|, Euclidean, in 64 bits"""
    return float((a.double() - b.double()).norm() / b.double().norm())


def reference(emb, f, ctx, dn):
    """The embeddings and every gradient of sum(dn * node_embedding), by autograd through the plain 64-bit form."""
    leaf = lambda t: t.detach().double().requires_grad_(True)   # noqa: E731
    p, e, s = {n: leaf(t) for n, t in ctx.params.items()}, leaf(emb), leaf(ctx.states)
    out = plain(e, f, ctx._replace(params=p, states=s))
    (out * dn.double()).sum().backward()
    return out.detach(), dict({n: t.grad for n, t in p.items()}, embedding=e.grad, states=s.grad)


def case(contexts, length, dtype, B=6, seed=4):
    cfg = CONFIGS["aldp"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    emb = torch.randn((cfg.n_features, cfg.hidden), generator=g, device="cuda")
    f = torch.randint(0, cfg.n_features, (B, cfg.n_nodes), generator=g, device="cuda", dtype=torch.int32)
    ctx = make_context(cfg, contexts, length, seed=seed, dtype=dtype)
    n = torch.linspace(length / 2, length, contexts, device="cuda").to(torch.int32)
    return cfg, g, emb, f, ctx._replace(lengths=n)


# ------------------------------------------------------------------------------------------------ states in 16 bits
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("size", [1.0, 1e-6, 5e-9])
@pytest.mark.parametrize("contexts,length", [(1, 40), (6, 33)])
def test_gradients_of_16_bit_states(contexts, length, size, dtype):
    """The gradient of a mean loss over a batch is 1e-6 and less, below fp16's smallest number at the end: the gradients
    keep their size whatever that of the nodes' is.  At most 16 roundings lie between the inputs and a gradient (x, its
    weights, q, k, v, their turned forms, P, o, do, dP's P, dS, dq, dk, dv and the turned-back ones), each at most u of what
    it rounds, in norm u / sqrt(3) and independent, and dS is a difference of two terms that are at most twice its size:
    2 sqrt(16 / 3) u = 4.6 u, so 8 u."""
    cfg, g, emb, f, ctx = case(contexts, length, dtype)
    nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
    dn = size * torch.randn(nodes.shape, generator=g, device="cuda")
    ref, want = reference(emb, f, ctx, dn)
    e = emb[f.long()].double()
    assert rel(nodes - e, ref - e) <= 8 * HALF[dtype]
    got = C.node_embedding_grad(dn, saved)
    assert got["states"].dtype == (torch.float32 if dtype == torch.float16 else dtype)
    off = {n: rel(got[n], w) for n, w in want.items()}
    print(dtype, size, {n: f"{v / HALF[dtype]:.2f} u" for n, v in off.items()}, flush=True)
    assert max(off.values()) <= 8 * HALF[dtype], off


def test_gradients_of_fp16_parameters():
    """Parameters in fp16 themselves: their gradients come in fp32, a loss's size of 5e-9 included."""
    cfg, g, emb, f, ctx = case(1, 40, torch.float32)
    ctx = ctx._replace(params={n: p.half() for n, p in ctx.params.items()})
    nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
    dn = 5e-9 * torch.randn(nodes.shape, generator=g, device="cuda")
    got = C.node_embedding_grad(dn, saved)
    for n, w in reference(emb, f, ctx, dn)[1].items():
        assert got[n].dtype == torch.float32 and rel(got[n], w) <= 1e-5, n   # fp32 throughout


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_training_gradients_of_16_bit_states(dtype):
    """A training step of 1024 clusters on one shared context: the loss's own node gradients (1e-8) reach every parameter."""
    cnf = build("lj13")
    cfg = cnf.cfg
    params = torch.as_tensor(F.flatten_params(init_params(cfg, 6), cfg), device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    B = 1024
    x1, x0 = cnf.sample_base(g, B) * 1.5, cnf.sample_base(g, B)
    t = torch.rand(B, generator=g, device="cuda")
    f = features(cfg)[None].expand(B, -1).contiguous()
    ctx = make_context(cfg, 1, 64, dtype=dtype)._replace(lengths=None)
    grads = []
    for c in (ctx, ctx._replace(states=ctx.states.float())):
        _, info, grad = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True, context=c)
        grads.append(dict(info["context_grad"], embedding=grad[-cfg.n_features * cfg.hidden:]))
    # 13 atoms of one feature: their rows differ by their positions only, so the scores' gradients (query, key) are sums that
    # cancel; the values' and outputs' do not.  As above, 8 u
    for n in ("value", "out", "embedding"):
        assert rel(grads[0][n], grads[1][n]) <= 8 * HALF[dtype], n
    for n in ("query", "key", "states", "query_norm", "key_norm"):
        assert rel(grads[0][n], grads[1][n]) <= 0.5, n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_fp32_parameters_get_fp32_gradients(dtype):
    """The sums over batch and atoms that give a parameter's gradient are not rounded to the states' type: the gradient of
    the output projection is o^T d_nodes of the o that was saved up to fp32 sums, and no product is a 16-bit number."""
    cfg, g, emb, f, ctx = case(6, 33, dtype)
    nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
    dn = torch.randn(nodes.shape, generator=g, device="cuda")
    got = C.node_embedding_grad(dn, saved)
    o = saved[8].double().reshape(-1, CTX.n_heads * CTX.head_dim)
    d = dn.double().reshape(o.shape[0], -1)
    want, size = o.t() @ d, o.abs().t() @ d.abs()
    # rows + 1 products and sums in fp32
    assert bool(((got["out"].double() - want).abs() <= (o.shape[0] + 1) * 2.0 ** -24 * size).all())
    for n in ("query", "key", "value", "out"):
        assert got[n].dtype == torch.float32
        assert float((got[n] == got[n].to(dtype).float()).float().mean()) < 0.05, n


# ------------------------------------------------------------------------------------------------ lengths and masks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("contexts", [1, 6])
def test_what_lies_behind_lengths_and_masks_is_not_read(contexts, dtype):
    """States and their positions behind a length or a mask hold NaN and infinities: embeddings and gradients have the bits
    that they have with zeros there."""
    cfg, g, emb, f, ctx = case(contexts, 33, dtype)
    mask = torch.rand((contexts, 33), generator=g, device="cuda") > 0.3
    keep = mask & (torch.arange(33, device="cuda")[None] < ctx.lengths[:, None])
    pos = 50 * torch.rand((contexts, 33, 3), generator=g, device="cuda")
    dn = torch.randn((6, cfg.n_nodes, cfg.hidden), generator=g, device="cuda")
    res = []
    for fill in (0.0, math.nan, math.inf):
        s = torch.where(keep[..., None], ctx.states, torch.full_like(ctx.states, fill))
        p = torch.where(keep[..., None], pos, torch.full_like(pos, fill))
        nodes, saved = C.node_embedding(emb, f, ctx._replace(states=s, positions=p, mask=mask), cfg, return_saved=True)
        res.append(dict(C.node_embedding_grad(dn, saved), nodes=nodes))
    # one row of positions for all contexts, NaN where none reads it: as with zeros there
    p = torch.where(keep.any(0)[:, None], pos[0], torch.full_like(pos[0], math.nan))
    s = torch.where(keep[..., None], ctx.states, torch.full_like(ctx.states, math.nan))
    shared = [dict(C.node_embedding_grad(dn, C.node_embedding(emb, f, ctx._replace(states=s, positions=x, mask=mask), cfg,
                                                              return_saved=True)[1])) for x in (p, torch.nan_to_num(p))]
    assert all(torch.equal(shared[0][n], t) for n, t in shared[1].items())
    for r in res + shared:
        assert all(bool(torch.isfinite(t).all()) for t in r.values())
        assert float(r["states"][~keep].abs().max()) == 0.0
    for r in res:
        assert all(torch.equal(r[n], res[0][n]) for n in r)


def test_masks_of_the_context_are_checked():
    cfg, g, emb, f, ctx = case(6, 33, torch.float32)
    for bad in (dict(lengths=torch.ones(5, dtype=torch.int32, device="cuda")), dict(lengths=torch.ones(6, device="cuda")),
                dict(mask=torch.ones((6, 32), dtype=torch.bool, device="cuda")),
                dict(mask=torch.ones((6, 33), device="cuda")), dict(mask=torch.ones((1, 33), dtype=torch.bool, device="cuda"))):
        with pytest.raises(ValueError, match="context_"):
            C.node_embedding(emb, f, ctx._replace(**bad), cfg)


# ------------------------------------------------------------------------------------------------ shapes
@pytest.mark.parametrize("B,contexts,length", [(0, 1, 9), (0, 0, 9), (3, 1, 0), (3, 3, 0), (0, 1, 0)])
def test_empty_batches_and_contexts(B, contexts, length):
    """No molecules, or contexts without states: embeddings of that shape (the table's own rows), gradients of 0."""
    cfg, g, emb, f, ctx = case(max(contexts, 1), 9, torch.float32, B=B)
    ctx = ctx._replace(states=ctx.states[:contexts, :length], positions=ctx.positions[:length], lengths=None)
    nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
    assert torch.equal(nodes, emb[f.long()])
    grads = C.node_embedding_grad(torch.ones_like(nodes), saved)
    for n, t in ctx.params.items():
        assert grads[n].shape == t.shape and float(grads[n].abs().max()) == 0.0
    assert grads["states"].shape == ctx.states.shape
    count = torch.bincount(f.reshape(-1), minlength=cfg.n_features).float()
    assert torch.equal(grads["embedding"], count[:, None].expand_as(emb).contiguous())


def test_feature_shapes():
    """The shapes of feature ids that the flow takes without a context give the same with one."""
    cnf = build("aldp")
    cfg = cnf.cfg
    params = init_params(cfg, 5)
    x, t = cnf.sample_base(7, 4), torch.full((4,), 0.5, device="cuda")
    f = features(cfg)
    each = f[None].expand(4, -1)
    ctx = make_context(cfg, 1, 30)._replace(lengths=None)
    want = cnf.apply(params, x, t, f, context=ctx)
    for shape in (each, each[..., None], each[..., None].cpu(), each.reshape(4, -1, 2)):
        assert torch.equal(cnf.apply(params, x, t, shape), cnf.apply(params, x, t, f))
        assert torch.equal(cnf.apply(params, x, t, shape, context=ctx), want)
    assert torch.equal(cnf.apply(params, x[:1], t[:1], f[:, None], context=ctx), cnf.apply(params, x[:1], t[:1], f, context=ctx))
    with pytest.raises(ValueError, match="features"):
        cnf.apply(params, x, t, each[:, :-1], context=ctx)


def test_device_ids_outside_the_table_are_reported():
    """A solve with a context names bad ids as one without does; the field itself gives NaN for that molecule alone."""
    cnf = build("aldp")
    cfg = cnf.cfg
    params = init_params(cfg, 5)
    x0 = cnf.sample_base(7, 3)
    f = features(cfg)[None].repeat(3, 1)
    f[1, 4] = cfg.n_features
    kw = dict(use_fixed_step_size=True, step_size=0.25)
    for ctx in (None, make_context(cfg, 1, 30)._replace(lengths=None), make_context(cfg, 3, 30)):
        with pytest.raises(ValueError, match="ids must lie in"):
            F.sample_cnf(cnf, params, None, features=f, x0=x0, context=ctx, **kw)
        for call in (F.get_log_prob, lambda cnf, params, x, key, **k: F.sample_and_log_prob_cnf(cnf, params, key, **k)):
            with pytest.raises(ValueError, match="ids must lie in"):
                call(cnf, params, x0, 1, features=f, approx=True, context=ctx, **kw)
        v = cnf.apply(params, x0, torch.full((3,), 0.5, device="cuda"), f, context=ctx)
        assert bool(torch.isnan(v[1]).all()) and bool(torch.isfinite(v[[0, 2]]).all())


# ------------------------------------------------------------------------------------------------ streams
class _Queued:
    """A library whose update_params leaves 50 ms of work on the current stream behind it."""

    def __init__(self, lib):
        self._lib = lib

    def __getattr__(self, name):
        fn = getattr(self._lib, name)
        if name != "ecnf_update_params":
            return fn

        def update(*a):
            rc = fn(*a)
            torch.cuda._sleep(100_000_000)
            return rc
        return update


def test_the_table_is_there_on_every_stream():
    """Weights are in place when a handle's construction or update returns, on whatever stream; so is the table."""
    cfg = CONFIGS["aldp"]
    blobs = [torch.as_tensor(F.flatten_params(init_params(cfg, i), cfg), device="cuda") for i in range(3)]
    tables = [b[-cfg.n_features * cfg.hidden:].reshape(cfg.n_features, cfg.hidden) for b in blobs]
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        h = EcnfHandle(cfg, blobs[0].cpu().numpy(), 0)
        assert a.query()
    lib = h.lib
    h.lib = _Queued(lib)
    try:
        for i in (1, 2, 0):
            with torch.cuda.stream(a):
                h.update_params(blobs[i])
                assert a.query()
            with torch.cuda.stream(b):
                got = h.embedding.clone()
            b.synchronize()
            assert torch.equal(got, tables[i])
    finally:
        h.lib = lib


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_embeddings_captured_and_replayed(dtype):
    """The embeddings and their gradients in one graph, replayed on new inputs with eager work between, equal the eager ones."""
    cfg, g, emb, f, ctx = case(6, 33, dtype)
    ctx = ctx._replace(positions=50 * torch.rand((33, 3), generator=g, device="cuda"))
    dn = torch.randn((6, cfg.n_nodes, cfg.hidden), generator=g, device="cuda")

    def work():
        nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
        return [nodes, *C.node_embedding_grad(dn, saved).values()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    for n in range(3):
        for t in (emb, dn, ctx.states, ctx.params["query"]):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
        ctx.lengths.copy_(torch.randint(0, 34, (6,), generator=g, device="cuda", dtype=torch.int32))
        want = [x.clone() for x in work()]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, outs):
            assert torch.equal(x, y)
        work()


# ------------------------------------------------------------------------------------------------ a call's own table
@pytest.mark.parametrize("B", [1, 2, 12])
def test_own_table_in_team_solves(B):
    """QM9's solves of few molecules run as teams; with a call's own table too, in every team size, bit by bit."""
    cfg = CONFIGS["qm9"]
    h = EcnfHandle(cfg, init_params(cfg, 1), 0)
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    x = torch.randn((B, cfg.event_dim), generator=g, device="cuda")
    f = features(cfg)
    e = h.embedding[f.long()][None]
    opts = SolveOptions("euler", 0.25)
    want = h.integrate(x, f, 0.0, 1.0, opts)[0]
    for mode in (0, 1, 4):
        h.set_team(mode)
        assert torch.equal(h.integrate(x, None, 0.0, 1.0, opts, node_embedding=e)[0], want)
        assert torch.equal(h.integrate(x, f, 0.0, 1.0, opts, node_embedding=e.expand(B, -1, -1))[0], want)
    h.set_team(0)
    moved = e + 0.1 * torch.randn(e.shape, generator=g, device="cuda")
    res = []
    for mode in (0, 1):
        h.set_team(mode)
        res.append(h.integrate(x, None, 0.0, 1.0, opts, node_embedding=moved)[0])
    h.set_team(0)
    assert torch.equal(*res) and not torch.equal(res[0], want)


def test_own_table_of_large_molecules_and_in_fp32():
    """Molecules of more than 33 atoms (receiver-tiled edges) and the strict fp32 kernels read the table as well."""
    big = CNFConfig(n_nodes=48, dim=3, n_features=3, hidden=64, mlp_width=128, mlp_depth=3, n_blocks=2, base_scale=1.0,
                    sigma_min=0.01)
    for cfg, precision in ((big, "split_f16"), (big, "fp32"), (CONFIGS["aldp"], "fp32")):
        h = EcnfHandle(cfg, init_params(cfg, 1), 0, precision=precision)
        g = torch.Generator(device="cuda")
        g.manual_seed(9)
        x = torch.randn((5, cfg.event_dim), generator=g, device="cuda")
        f = features(cfg)
        e = h.embedding[f.long()][None]
        opts = SolveOptions("euler", 0.25)
        assert torch.equal(h.integrate(x, None, 0.0, 1.0, opts, node_embedding=e)[0], h.integrate(x, f, 0.0, 1.0, opts)[0])
        t = torch.full((5,), 0.5, device="cuda")
        assert torch.equal(h.vector_field(x, t, node_embedding=e.expand(5, -1, -1)), h.vector_field(x, t, f))
