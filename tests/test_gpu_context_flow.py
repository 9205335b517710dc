"""The conditional flow: node embeddings that read a context, through the solver, the log-densities and the training step.

The field's own arithmetic is pinned elsewhere (tests/test_gpu_parity.py, test_gpu_train.py); here: a call's own table
with the embedding's rows gives the results of the embedding ids, the embeddings and their gradients are those of a plain
64-bit form (autograd), and the whole loss's gradient is that of central differences.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs a ROCm GPU", allow_module_level=True)

from ecnf_amd import CONFIGS, init_params  # noqa: E402
from ecnf_amd import cnf as F  # noqa: E402
from ecnf_amd import context as C  # noqa: E402
from ecnf_amd import train as TR  # noqa: E402
from ecnf_amd import _lib  # noqa: E402
from ecnf_amd.engine import EcnfHandle, SolveOptions  # noqa: E402

CTX = C.ContextConfig(state_dim=24, n_heads=4, n_kv_heads=2, head_dim=16, axes=(8, 4, 4))


def build(name):
    c = CONFIGS[name]
    return F.build_cnf(n_frames=c.n_nodes, dim=c.dim, sigma_min=c.sigma_min, base_scale=c.base_scale,
                       n_blocks_egnn=c.n_blocks, mlp_units=c.mlp_units, n_invariant_feat_hidden=c.hidden,
                       time_embedding_dim=c.time_embedding_dim, n_features=c.n_features, device=0)


def features(cfg):
    return torch.arange(cfg.n_nodes, device="cuda", dtype=torch.int32) % cfg.n_features


def make_context(cfg, contexts, length, seed=0, out=0.3, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    p = C.init_context_params(CTX, cfg, seed)
    p["out"] = out * torch.randn(p["out"].shape, generator=g, device="cuda") * p["out"].shape[0] ** -0.5
    states = torch.randn((contexts, length, CTX.state_dim), generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 50, (length, 3), generator=g, device="cuda", dtype=torch.int32)
    node = torch.randint(0, 50, (cfg.n_nodes, 3), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.randint(0, length + 1, (contexts,), generator=g, device="cuda", dtype=torch.int32)
    return C.Context(CTX, p, states, node, pos, lengths=lengths)


# ------------------------------------------------------------------------------------------------ a call's own table
@pytest.mark.parametrize("name", ["dw4", "lj13", "aldp"])
def test_own_table_gives_the_embedding_ids_results(name):
    cfg = CONFIGS[name]
    h = EcnfHandle(cfg, init_params(cfg, 1), 0)
    B = 9
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn((B, cfg.event_dim), generator=g, device="cuda")
    t = torch.rand(B, generator=g, device="cuda")
    f = features(cfg)
    shared = h.embedding[f.long()][None]
    each = shared.expand(B, -1, -1).contiguous()
    # one-feature 13-atom molecules: block 1 in pair tiles without a table, edge by edge with one (fp32 rounding of the
    # same sums); every other shape runs the same instructions
    exact = name != "lj13"

    def same(a, b, scale):
        assert torch.equal(a, b) if exact else float((a - b).abs().max()) <= 2e-5 * max(1.0, scale)
    v = h.vector_field(x, t, f)
    for e in (shared, each):
        same(v, h.vector_field(x, t, node_embedding=e), float(v.abs().max()))
    eps = torch.randn(x.shape, generator=g, device="cuda")
    for opts, div in ((SolveOptions("euler", 0.1), _lib.DIV_NONE), (SolveOptions("dopri5", 0.1), _lib.DIV_HUTCHINSON),
                      (SolveOptions("dopri5", 0.25), _lib.DIV_EXACT)):
        y, dl, nfe, _ = h.integrate(x, f, 0.0, 1.0, opts, divergence=div, eps=eps)
        for e in (shared, each):
            z, dm, nfe2, _ = h.integrate(x, None, 0.0, 1.0, opts, divergence=div, eps=eps, node_embedding=e)
            assert torch.equal(nfe, nfe2)
            assert torch.equal(y, z) if exact else float((y - z).abs().max()) <= 1e-4
            if dl is not None:
                assert torch.equal(dl, dm) if exact else float((dl - dm).abs().max()) <= 1e-4 * max(1.0, float(dl.abs().max()))


def test_own_table_in_a_redealt_adaptive_solve():
    """More molecules than CUs, adaptive: the chunked, re-dealt launches and the tail teams read the table too."""
    cfg = CONFIGS["aldp"]
    h = EcnfHandle(cfg, init_params(cfg, 1), 0)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    B = 320
    x = 0.2 * torch.randn((B, cfg.event_dim), generator=g, device="cuda")
    eps = torch.randn(x.shape, generator=g, device="cuda")
    f = features(cfg)
    opts = SolveOptions("dopri5", None, rtol=1e-3, atol=1e-3)
    a = h.integrate(x, f, 1.0, 0.0, opts, divergence=_lib.DIV_HUTCHINSON, eps=eps)
    e = h.embedding[f.long()][None].expand(B, -1, -1)
    b = h.integrate(x, None, 1.0, 0.0, opts, divergence=_lib.DIV_HUTCHINSON, eps=eps, node_embedding=e)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_rows_outside_the_table_are_reported():
    cfg = CONFIGS["dw4"]
    h = EcnfHandle(cfg, init_params(cfg, 1), 0)
    x, t = torch.randn((2, cfg.event_dim), device="cuda"), torch.zeros(2, device="cuda")
    row = torch.tensor([[0, 1, 2, 3], [0, 1, 2, 4]], device="cuda", dtype=torch.int32)
    nodes = torch.randn((4, cfg.hidden), device="cuda")
    v = torch.empty_like(x)
    lib = _lib.load()
    s = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.ecnf_vector_field_nodes(h._h, x.data_ptr(), t.data_ptr(), nodes.data_ptr(), 4, row.data_ptr(),
                                           v.data_ptr(), 2, s))
    assert bool(torch.isfinite(v[0]).all()) and bool(torch.isnan(v[1]).all())
    for n in (0, -1, 1 << 30):
        assert lib.ecnf_vector_field_nodes(h._h, x.data_ptr(), t.data_ptr(), nodes.data_ptr(), n, row.data_ptr(),
                                           v.data_ptr(), 2, s) in (_lib.ECNF_E_INVALID, _lib.ECNF_E_UNSUPPORTED)


# ------------------------------------------------------------------------------------------------ the embeddings
def plain(embedding, f, ctx):
    """node_embedding in elementary fp64 operations; f [B, N]"""
    c, p = ctx.cfg, ctx.params
    B, N = f.shape
    s = ctx.states.expand(B, -1, -1)
    e = embedding[f.long()]

    def turned(x, w, pos):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + c.eps) * w
        out, at = [], 0
        for a, d in enumerate(c.axes):
            j = torch.arange(d // 2, device=x.device, dtype=torch.float64)
            ang = (pos[..., a].double()[..., None] * c.theta ** (-2 * j / d))[..., None, :]
            lo, hi = x[..., at:at + d // 2], x[..., at + d // 2:at + d]
            out += [lo * ang.cos() - hi * ang.sin(), lo * ang.sin() + hi * ang.cos()]
            at += d
        return torch.cat(out + [x[..., at:]], -1)
    q = turned((e @ p["query"]).reshape(B, N, c.n_heads, -1), p["query_norm"], ctx.node_positions)
    k = turned((s @ p["key"]).reshape(B, s.shape[1], c.n_kv_heads, -1), p["key_norm"], ctx.positions)
    v = (s @ p["value"]).reshape(B, s.shape[1], c.n_kv_heads, -1)
    G = c.n_heads // c.n_kv_heads
    k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    S = torch.einsum("bihd,bjhd->bhij", q, k) * c.head_dim ** -0.5
    keep = torch.arange(s.shape[1], device=s.device)[None] < ctx.lengths.expand(B)[:, None]
    S = S.masked_fill(~keep[:, None, None], -1e300)
    P = torch.softmax(S, -1) * keep[:, None, None]
    o = torch.einsum("bhij,bjhd->bihd", P, v).reshape(B, N, -1)
    return e + o @ p["out"]


@pytest.mark.parametrize("contexts,length", [(1, 40), (6, 33), (6, 1)])
def test_node_embedding_and_its_gradients(contexts, length):
    cfg, c = CONFIGS["aldp"], CTX
    B = 6
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    emb = torch.randn((cfg.n_features, cfg.hidden), generator=g, device="cuda")
    f = torch.randint(0, cfg.n_features, (B, cfg.n_nodes), generator=g, device="cuda", dtype=torch.int32)
    ctx = make_context(cfg, contexts, length, seed=4)
    nodes, saved = C.node_embedding(emb, f, ctx, cfg, return_saved=True)
    dn = torch.randn(nodes.shape, generator=g, device="cuda")
    got = C.node_embedding_grad(dn, saved)
    leaf = lambda t: t.double().requires_grad_(True)   # noqa: E731
    p64, e64, s64 = {n: leaf(t) for n, t in ctx.params.items()}, leaf(emb), leaf(ctx.states)
    ref = plain(e64, f, ctx._replace(params=p64, states=s64))
    (ref * dn.double()).sum().backward()
    # fp32 throughout: sums of at most B N + Lk rows; a few hundred steps of the largest magnitude of each result
    tol = 512 * 2.0 ** -24
    ref = ref.detach()
    assert float((nodes - ref).abs().max()) <= tol * float(ref.abs().max())
    want = dict({n: t.grad for n, t in p64.items()}, embedding=e64.grad, states=s64.grad)
    assert set(got) == set(want)
    for n, w in want.items():
        w = torch.zeros_like(got[n]) if w is None else w
        assert got[n].shape == w.shape
        # dS = P (dP - delta) cancels (to 0 with one key), but its two terms are sums of D products do v, each off by
        # D 2^-24 of their size: what they make of the gradients behind them (times scale k, times x) stays as error
        term = c.head_dim * float((dn @ ctx.params["out"].t()).abs().max() * saved[5].abs().max())
        behind = c.head_dim ** -0.5 * float(saved[7].abs().max() * max(emb.abs().max(), ctx.states.abs().max(), 1.0))
        uncancelled = term * behind if n in ("query", "key", "query_norm", "key_norm", "states", "embedding") else 0.0
        assert float((got[n] - w).abs().max()) <= tol * max(float(w.abs().max()), uncancelled), n


def test_results_carry_no_autograd_history():
    """Leaves that require gradients: the results have none of their own (a part of the chain would be worse than none)."""
    cfg = CONFIGS["aldp"]
    ctx = make_context(cfg, 1, 20)
    table = torch.randn((cfg.n_features, cfg.hidden), device="cuda", requires_grad=True)
    ctx = ctx._replace(params={n: p.requires_grad_() for n, p in ctx.params.items()})
    nodes, saved = C.node_embedding(table, features(cfg), ctx, cfg, return_saved=True)
    grads = C.node_embedding_grad(torch.ones_like(nodes), saved)
    assert not nodes.requires_grad and not any(x.requires_grad for x in grads.values())


def test_shared_features_and_context_are_computed_once():
    cfg = CONFIGS["aldp"]
    ctx = make_context(cfg, 1, 20)
    emb = torch.randn((cfg.n_features, cfg.hidden), device="cuda")
    one = C.node_embedding(emb, features(cfg), ctx, cfg)
    assert one.shape == (1, cfg.n_nodes, cfg.hidden)
    many = C.node_embedding(emb, features(cfg)[None].expand(5, -1), ctx, cfg)
    assert torch.equal(many, one.expand(5, -1, -1))


def test_low_precision_states():
    """bf16 states: the projections and the attention in bf16, the embedding itself in fp32."""
    cfg = CONFIGS["aldp"]
    ctx = make_context(cfg, 1, 40, dtype=torch.bfloat16)
    emb = torch.randn((cfg.n_features, cfg.hidden), device="cuda")
    f = features(cfg)[None]
    a = C.node_embedding(emb, f, ctx, cfg)
    b = plain(emb.double(), f, ctx._replace(params={n: t.double() for n, t in ctx.params.items()}, states=ctx.states.double()))
    # five roundings in a row (x, q and k, their turned forms, out, the result), each 2^-8 of what the row adds up
    size = (b - emb[f.long()].double()).abs().max()
    assert a.dtype == torch.float32 and float((a - b).abs().max()) <= 8 * 2.0 ** -8 * max(1.0, float(size)) * 4


# ------------------------------------------------------------------------------------------------ the flow
def test_untrained_context_changes_nothing_and_a_trained_one_stays_equivariant():
    cnf = build("aldp")
    cfg = cnf.cfg
    params = init_params(cfg, 5)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x0 = cnf.sample_base(g, 7)
    f = features(cfg)
    kw = dict(use_fixed_step_size=True, step_size=0.1, x0=x0)
    base = F.sample_cnf(cnf, params, None, features=f, **kw)
    zero = make_context(cfg, 1, 30, out=0.0)
    assert torch.equal(F.sample_cnf(cnf, params, None, features=f, context=zero, **kw), base)
    ctx = make_context(cfg, 7, 30)
    y = F.sample_cnf(cnf, params, None, features=f, context=ctx, **kw)
    has = ctx.lengths > 0
    assert float((y - base)[has].abs().max()) > 1e-4 and torch.equal(y[~has], base[~has])
    R = torch.linalg.qr(torch.randn((3, 3), generator=g, device="cuda"))[0]
    turn = lambda x: (x.reshape(-1, cfg.n_nodes, 3) @ R).reshape(-1, cfg.event_dim)   # noqa: E731
    y2 = F.sample_cnf(cnf, params, None, features=f, context=ctx, **dict(kw, x0=turn(x0)))
    assert float((turn(y) - y2).abs().max()) <= 1e-4
    # one molecule, the field itself, and the densities take it too
    one = F.sample_cnf(cnf, params, None, features=f, context=zero._replace(params=ctx.params), **dict(kw, x0=x0[0]))
    assert one.shape == (cfg.event_dim,)
    v = cnf.apply(params, x0, torch.full((7,), 0.5, device="cuda"), f, context=ctx)
    assert v.shape == x0.shape
    opts = dict(use_fixed_step_size=True, step_size=0.25, approx=True)
    lp, _, _ = F.get_log_prob(cnf, params, y, 1, features=f, context=ctx, **opts)
    x1, lq = F.sample_and_log_prob_cnf(cnf, params, 1, features=f[None].expand(7, -1), context=ctx, **opts)
    assert lp.shape == lq.shape == (7,) and bool(torch.isfinite(lp).all()) and bool(torch.isfinite(lq).all())


@pytest.mark.parametrize("name,contexts", [("aldp", 6), ("lj13", 1)])
def test_loss_gradient(name, contexts):
    cnf = build(name)
    cfg = cnf.cfg
    params = torch.as_tensor(F.flatten_params(init_params(cfg, 6), cfg), device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    B = 6
    x1, x0 = cnf.sample_base(g, B) * 1.5, cnf.sample_base(g, B)
    t = torch.rand(B, generator=g, device="cuda")
    f = features(cfg)[None].expand(B, -1).contiguous()
    zero = make_context(cfg, contexts, 25, out=0.0)
    loss, _, grad = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True)
    loss0, info, grad0 = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True, context=zero)
    assert abs(float(loss - loss0)) <= 1e-6 * float(loss)
    assert float((grad - grad0).abs().max()) <= 1e-5 * float(grad.abs().max())
    assert float(info["context_grad"]["query"].abs().max()) == 0.0 and float(info["context_grad"]["out"].abs().max()) > 0.0

    ctx = make_context(cfg, contexts, 25)
    _, info, grad = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True, context=ctx)
    cg = info["context_grad"]
    h = 2.0 ** -6

    def value(p, c):
        return float(TR.flow_matching_loss_fn(cnf, p, x1, None, f, x0=x0, t=t, context=c)[0].double())
    # along each gradient itself: (L(+h) - L(-h)) / 2h = |grad| + O(h^2) + 2^-22 L / h (fp32 loss)
    n = cfg.n_features * cfg.hidden
    for key in ("embedding", "query", "key", "value", "out", "query_norm", "key_norm", "states"):
        d = grad[-n:] if key == "embedding" else cg[key]
        size = float(d.double().norm())
        assert size > 0.0, key
        step = d / size
        if key == "embedding":
            up, down = params.clone(), params.clone()
            up[-n:] += h * step
            down[-n:] -= h * step
            num = (value(up, ctx) - value(down, ctx)) / (2 * h)
        elif key == "states":
            num = (value(params, ctx._replace(states=ctx.states + h * step))
                   - value(params, ctx._replace(states=ctx.states - h * step))) / (2 * h)
        else:
            at = lambda s: ctx._replace(params=dict(ctx.params, **{key: ctx.params[key] + s * step}))   # noqa: E731
            num = (value(params, at(h)) - value(params, at(-h))) / (2 * h)
        assert abs(num - size) <= 0.02 * size + 2.0 ** -22 * float(loss) / h, (key, num, size)
    # the same bits again
    _, info2, grad2 = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True, context=ctx)
    assert torch.equal(grad, grad2) and all(torch.equal(cg[k], info2["context_grad"][k]) for k in cg)


def test_update_step():
    """flow_matching_update_fn with a context: the loss and gradients of flow_matching_loss_fn, Adam on the field's."""
    cnf = build("lj13")
    cfg = cnf.cfg
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    B = 5
    x1, x0 = cnf.sample_base(g, B) * 1.5, cnf.sample_base(g, B)
    t = torch.rand(B, generator=g, device="cuda")
    f = features(cfg)[None].expand(B, -1).contiguous()
    ctx = make_context(cfg, 1, 25)
    params = torch.as_tensor(F.flatten_params(init_params(cfg, 6), cfg), device="cuda")
    loss, want, grad = TR.flow_matching_loss_fn(cnf, params, x1, None, f, x0=x0, t=t, with_grad=True, context=ctx)
    opt = TR.adam(1e-3)
    state = TR.init_training_state(cnf, params, opt, key=0)
    new, info = TR.flow_matching_update_fn(cnf, opt, state, x1, f, x0=x0, t=t, context=ctx)
    assert torch.equal(info["loss"], loss)
    assert all(torch.equal(info["context_grad"][n], want["context_grad"][n]) for n in want["context_grad"])
    moved = params - new.params                        # Adam's first step: lr * grad / (|grad| + eps)
    at = grad.abs() > 1e-4 * grad.abs().max()
    assert torch.equal(moved[at].sign(), grad[at].sign())


def test_padded_widths():
    """A reference network zero-padded onto a compiled shape: embeddings of the reference's width, same results as ids."""
    cnf = F.build_cnf(n_frames=5, dim=3, sigma_min=0.01, base_scale=1.0, n_blocks_egnn=2, mlp_units=(48, 40),
                      n_invariant_feat_hidden=20, time_embedding_dim=8, n_features=3, device=0)
    params = cnf.init(3)
    f = torch.tensor([0, 1, 2, 1, 0], device="cuda", dtype=torch.int32)
    x, t = torch.randn((4, 15), device="cuda"), torch.rand(4, device="cuda")
    ctx = make_context(cnf.cfg, 1, 9, out=0.0)
    assert ctx.params["query"].shape[0] == 20
    assert torch.equal(cnf.apply(params, x, t, f), cnf.apply(params, x, t, f, context=ctx))
    ctx = make_context(cnf.cfg, 4, 9)
    tr_params = torch.as_tensor(F.flatten_params(params, cnf.cfg), device="cuda")
    loss, info, grad = TR.flow_matching_loss_fn(cnf, tr_params, x, None, f[None].expand(4, -1), x0=x.flip(0), t=t,
                                                with_grad=True, context=ctx)
    assert bool(torch.isfinite(grad).all()) and info["context_grad"]["out"].shape == (64, 20)


def test_refusals():
    cfg = CONFIGS["aldp"]
    h = EcnfHandle(cfg, init_params(cfg, 1), 0)
    ctx = make_context(cfg, 3, 9)
    f = features(cfg)
    x, t = torch.randn((2, cfg.event_dim), device="cuda"), torch.zeros(2, device="cuda")
    with pytest.raises(ValueError, match="molecules"):        # 3 contexts, 2 molecules
        h.vector_field(x, t, node_embedding=C.node_embedding(h.embedding, f, ctx, cfg))
    for bad in (torch.zeros(2, cfg.n_nodes + 1, cfg.hidden), torch.zeros(2, cfg.n_nodes, cfg.hidden - 1), torch.zeros(7)):
        with pytest.raises(ValueError, match="node_embedding"):
            h.vector_field(x, t, node_embedding=bad)
    with pytest.raises(ValueError, match="batch"):
        C.node_embedding(h.embedding, f[None].expand(2, -1), ctx, cfg)
    with pytest.raises(ValueError, match="features"):
        C.node_embedding(h.embedding, None, ctx, cfg)
    with pytest.raises(ValueError, match="ids"):
        C.node_embedding(h.embedding, f.float(), ctx, cfg)
    with pytest.raises(ValueError, match="lie in"):
        C.node_embedding(h.embedding, f.cpu() + 1, ctx, cfg)
    with pytest.raises(ValueError, match="states"):
        C.node_embedding(h.embedding, f, ctx._replace(states=ctx.states[..., :5]), cfg)
    # device ids are not read back: the atom's row is NaN
    n = C.node_embedding(h.embedding, f + 1, ctx._replace(states=ctx.states[:1], lengths=ctx.lengths[:1]), cfg)
    assert bool(torch.isnan(n[0, -1]).all()) and bool(torch.isfinite(n[0, :-1]).all())


def test_handle_embedding_follows_the_weights():
    cfg = CONFIGS["aldp"]
    a, b = init_params(cfg, 1), init_params(cfg, 2)
    h = EcnfHandle(cfg, a, 0)
    np.testing.assert_array_equal(h.embedding.cpu().numpy(), a["Embed_0/embedding"])
    h.update_params(b)
    np.testing.assert_array_equal(h.embedding.cpu().numpy(), b["Embed_0/embedding"])
    h.update_params(torch.as_tensor(F.flatten_params(a, cfg), device="cuda"))
    np.testing.assert_array_equal(h.embedding.cpu().numpy(), a["Embed_0/embedding"])
