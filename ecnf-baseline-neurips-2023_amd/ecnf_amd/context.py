"""Context operators: attention from a molecule's atoms to an encoder's states of another length, with gradients.

  * :func:`qk_norm_rotary` / :func:`qk_norm_rotary_grad`     per-head norm of queries and keys and the rotation by
    their positions (one to four axes, e.g. chain / residue / atom) in one pass        (ecnf_qk_norm_rotary)
  * :func:`cross_attention` / :func:`cross_attention_grad`   softmax(scale q k^T) v     (ecnf_cross_attention)
  * :class:`Context`, :func:`node_embedding` / :func:`node_embedding_grad`: a conditional flow.  The embedding row of an
    atom's feature also attends to the states; the result takes the row's place in the vector field
    (``context=`` of ``cnf.apply``, ``sample_cnf``, ``get_log_prob``, ``sample_and_log_prob_cnf`` and
    ``flow_matching_loss_fn``).  It reads no coordinates, so the field stays equivariant, and it is constant along the
    ODE, so a solve computes it once.

Tensors are [batch, length, heads, head_dim] in float32, bfloat16 or float16, on one device, with any strides (the last
dimension contiguous, else it is copied first).  The calls run on the tensors' device and torch's current stream of
it, allocate outputs and workspace from torch's stream-ordered allocator and never synchronise, so they can be captured
into a graph.  As everywhere in this package gradients are explicit calls: results carry no autograd history.
Nothing here falls back to the CPU.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass
from typing import Dict, Mapping, NamedTuple, Optional, Sequence, Tuple

import torch

from . import _lib
from .params import CNFConfig

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_POSITIONS = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32}
# the layouts of _lib.EcnfQkNorm (its two sides first) and _lib.EcnfAttention: packed at once, which costs a tenth of
# filling a ctypes structure field by field (tests/test_context.py holds them to the compiled library's layout)
_QK_NORM = struct.Struct("@" + 2 * "6P8q4i" + "9ifd")
_ATTENTION = struct.Struct("@12P12q9if")
_CONTIGUOUS = torch.contiguous_format
_NO_SIDE, _NO_STRIDES, _NO_AXES = (0,) * 18, (0,) * 3, (0,) * 4


def _tensor(x, name: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [batch, length, heads, head_dim] on a device, its last dimension contiguous; dtype and device of `like`."""
    if not (torch.is_tensor(x) and x.is_cuda):
        raise ValueError(f"{name} must be a device (cuda) tensor")
    if x.dim() != 4:
        raise ValueError(f"{name} must be [batch, length, heads, head_dim], got {tuple(x.shape)}")
    if like is None:
        if x.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    elif x.dtype != like.dtype or x.device != like.device:
        raise ValueError(f"{name} must have the dtype and device of q ({like.dtype}, {like.device}), got {x.dtype}, "
                         f"{x.device}")
    return x if x.stride(3) == 1 else x.contiguous()


def _strides(x: torch.Tensor) -> Tuple[int, int, int]:
    """Strides of the first three dimensions; 0 where there is one element (torch's may be anything there)."""
    (a, b, c, d), (sa, sb, sc, _) = x.shape, x.stride()
    return (sa if a > 1 else 0, sb if b > 1 else 0, sc if c > 1 else 0)


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """x with its rows on 16-byte boundaries (a copy if they are not)."""
    e = x.element_size()
    a, b, c = _strides(x)
    return x if (x.data_ptr() | a * e | b * e | c * e) % 16 == 0 else x.contiguous() if not x.is_contiguous() else x.clone()


def _key_rows(x: torch.Tensor) -> torch.Tensor:
    """k or v as the library takes them: aligned, and its keys neither on top of each other nor 8 MiB or more apart (a copy
    if they are)."""
    s = x.stride(1)
    if x.shape[1] > 1 and not x.shape[3] <= s < (8 << 20) // x.element_size():
        return x.contiguous()
    return _aligned(x)


def _stream(device: torch.device) -> int:
    """torch's current stream of the device (torch.cuda.current_stream(device).cuda_stream, without building the stream
    object: 2 us of a 10 us call)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _pack(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:
        raise ValueError(f"a size or axis is out of its 32-bit range ({e})") from None


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=_CONTIGUOUS)


def _same_shape(x: torch.Tensor, like: torch.Tensor, name: str) -> None:
    if x.shape != like.shape:
        raise ValueError(f"{name} must have shape {tuple(like.shape)}, got {tuple(x.shape)}")


# ------------------------------------------------------------------------------------------------------ norm + rotation
def _weight(w, x: torch.Tensor, name: str) -> torch.Tensor:
    if not (torch.is_tensor(w) and w.device == x.device and w.dim() == 1 and w.shape[0] == x.shape[3]
            and w.dtype in _DTYPES):
        raise ValueError(f"{name} must be a floating [head_dim = {x.shape[3]}] tensor on {x.device}")
    return w if w.dtype == torch.float32 and w.is_contiguous() else w.float().contiguous()


def _positions(p, x: torch.Tensor, n_axes: int, name: str) -> Tuple[torch.Tensor, int, int]:
    """(positions, batch stride, token stride)"""
    if not (torch.is_tensor(p) and p.device == x.device and p.dtype in _POSITIONS):
        raise ValueError(f"{name} must be an int32, int64 or float32 tensor on {x.device}")
    n, shape = p.dim(), p.shape
    if not (2 <= n <= 3 and shape[-1] == n_axes and shape[-2] == x.shape[1] and (n == 2 or shape[0] == x.shape[0])):
        raise ValueError(f"{name} must be [{x.shape[1]}, {n_axes}] or [{x.shape[0]}, {x.shape[1]}, {n_axes}], got "
                         f"{tuple(shape)}")
    st = p.stride()
    if st[-1] != 1 and n_axes > 1:
        p = p.contiguous()
        st = p.stride()
    return p, (st[0] if n == 3 else 0), st[-2]


def _norm_call(q, k, axes, theta, eps, interleaved, grad: bool):
    """q, k: (x, weight, positions, output gradient or None, name), k None for none; returns (outputs, weight gradients)."""
    axes = tuple(int(a) for a in axes)
    n_axes = len(axes)
    if not 1 <= n_axes <= 4:
        raise ValueError("axes must name one to four axes")
    packed, outs, dws, keep = (), [], [], []
    for side in (q, k):
        if side is None:
            packed += _NO_SIDE
            outs.append(None)
            dws.append(None)
            continue
        x, w, pos, g, name = side
        w32 = None if w is None else _weight(w, x, name + "_weight")
        p, pb, pl = _positions(pos, x, n_axes, name + "_positions")
        out = _new(x)
        dw = torch.empty(x.shape[3], dtype=torch.float32, device=x.device) if grad and w is not None else None
        packed += (x.data_ptr(), 0 if g is None else g.data_ptr(), out.data_ptr(), 0 if w is None else w32.data_ptr(),
                   0 if dw is None else dw.data_ptr(), p.data_ptr(), *_strides(x), *(_NO_STRIDES if g is None else _strides(g)),
                   pb, pl, *x.shape[:3], _POSITIONS[p.dtype])
        outs.append(out)
        dws.append(dw)
        keep.append((w32, p))   # alive until the launch
    x = q[0]
    device = x.device
    args = _pack(_QK_NORM, *packed, _DTYPES[x.dtype], x.shape[3], n_axes, *(axes + _NO_AXES)[:4], bool(interleaved),
                 device.index, eps, theta)
    lib = _lib.load()
    if not grad:
        _lib.check(lib.ecnf_qk_norm_rotary(args, _stream(device)))
        return outs, dws
    n = ctypes.c_size_t()
    _lib.check(lib.ecnf_qk_norm_workspace_size(args, ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device=device)
    _lib.check(lib.ecnf_qk_norm_rotary_grad(args, ws.data_ptr(), n.value, _stream(device)))
    for i, side in enumerate((q, k)):
        if dws[i] is not None and side[1].dtype != torch.float32:
            dws[i] = dws[i].to(side[1].dtype)
    return outs, dws


def qk_norm_rotary(q, k=None, *, q_positions, k_positions=None, axes: Sequence[int], q_weight=None, k_weight=None,
                   theta: float = 10000.0, eps: float = 1e-6, interleaved: bool = False):
    """(q', k') for q [B, Lq, Hq, D] and k [C, Lk, Hk, D] (or None): each head y = weight * x / sqrt(mean(x^2) + eps),
    then axis a, ``axes[a]`` dims wide (in order from dim 0), turns its pair j by position[a] * theta^(-2j / axes[a]).
    Pairs are (j, j + axes[a] / 2) inside the axis, or neighbours with ``interleaved``; dims behind the axes are not
    turned.  Positions [L, n_axes] or [batch, L, n_axes], whole (int32, int64) or real (float32); their angles are
    reduced in fp64, so far positions keep their accuracy.  Weights [D], shared by the heads (None: 1).  D is even and
    at most 128."""
    q = _tensor(q, "q")
    if k is not None:
        k = _tensor(k, "k", q)
        if k.shape[3] != q.shape[3]:
            raise ValueError(f"k must have q's head_dim {q.shape[3]}, got {k.shape[3]}")
    outs, _ = _norm_call((q, q_weight, q_positions, None, "q"),
                         None if k is None else (k, k_weight, k_positions, None, "k"), axes, float(theta), float(eps),
                         interleaved, False)
    return outs[0], outs[1]


def qk_norm_rotary_grad(q_grad, k_grad, q, k=None, *, q_positions, k_positions=None, axes: Sequence[int],
                        q_weight=None, k_weight=None, theta: float = 10000.0, eps: float = 1e-6,
                        interleaved: bool = False):
    """(dq, dk, dq_weight, dk_weight) of :func:`qk_norm_rotary` for the gradients of its outputs (None where the
    operand is).  Weight gradients are summed in fp32 over all rows in a fixed order."""
    q = _tensor(q, "q")
    q_grad = _tensor(q_grad, "q_grad", q)
    _same_shape(q_grad, q, "q_grad")
    if k is not None:
        k = _tensor(k, "k", q)
        if k.shape[3] != q.shape[3]:
            raise ValueError(f"k must have q's head_dim {q.shape[3]}, got {k.shape[3]}")
        k_grad = _tensor(k_grad, "k_grad", q)
        _same_shape(k_grad, k, "k_grad")
    outs, dws = _norm_call((q, q_weight, q_positions, q_grad, "q"),
                           None if k is None else (k, k_weight, k_positions, k_grad, "k"), axes, float(theta),
                           float(eps), interleaved, True)
    return outs[0], outs[1], dws[0], dws[1]


# ------------------------------------------------------------------------------------------------------ cross attention
def _lengths(x, n: int, most: int, like: torch.Tensor, name: str) -> Optional[torch.Tensor]:
    if x is None:
        return None
    if not (torch.is_tensor(x) and x.device == like.device and x.dtype in (torch.int32, torch.int64)
            and tuple(x.shape) == (n,)):
        raise ValueError(f"{name} must be an int32 or int64 [{n}] tensor on {like.device}")
    return x.contiguous() if x.dtype == torch.int32 else x.clamp(0, most).to(torch.int32).contiguous()


def _mask(m, shape: Tuple[int, int], like: torch.Tensor) -> Optional[torch.Tensor]:
    if m is None:
        return None
    if not (torch.is_tensor(m) and m.device == like.device and m.dtype in (torch.bool, torch.uint8)
            and tuple(m.shape) == shape):
        raise ValueError(f"context_mask must be a bool [{shape[0]}, {shape[1]}] tensor on {like.device}")
    return m.contiguous()


def _attention_operands(q, k, v, query_lengths, context_lengths, context_mask, scale):
    q = _tensor(q, "q")
    k, v = _tensor(k, "k", q), _tensor(v, "v", q)
    _same_shape(v, k, "v")
    B, _, Hq, D = q.shape
    C, Lk, Hk = k.shape[:3]
    if C != B and C != 1:
        raise ValueError(f"k must have q's batch {B} or 1, got {C}")
    if k.shape[3] != D:
        raise ValueError(f"k must have q's head_dim {D}, got {k.shape[3]}")
    if Hk < 1 or Hq < 1 or Hq % Hk:
        raise ValueError(f"q's heads ({Hq}) must be a multiple of k's ({Hk})")
    q, k, v = _aligned(q), _key_rows(k), _key_rows(v)
    ql = _lengths(query_lengths, B, q.shape[1], q, "query_lengths")
    cl = _lengths(context_lengths, C, Lk, q, "context_lengths")
    m = _mask(context_mask, (C, Lk), q)
    return q, k, v, ql, cl, m, float(D ** -0.5 if scale is None else scale)


def _attention_args(q, k, v, out, dout, lse, dq, dk, dv, ql, cl, m, scale) -> bytes:
    B, Lq, Hq, D = q.shape
    C, Lk, Hk = k.shape[:3]

    def ptr(t):
        return 0 if t is None else t.data_ptr()
    return _pack(_ATTENTION, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(dout), ptr(lse), ptr(dq), ptr(dk),
                 ptr(dv), ptr(ql), ptr(cl), ptr(m), *_strides(q), *_strides(k), *_strides(v),
                 *(_NO_STRIDES if dout is None else _strides(dout)), _DTYPES[q.dtype], B, C, Lq, Lk, Hq, Hk, D,
                 q.device.index, scale)


def _run_attention(args: bytes, grad: int, device) -> None:
    lib = _lib.load()
    n = ctypes.c_size_t()
    _lib.check(lib.ecnf_cross_attention_workspace_size(args, grad, ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None
    fn = lib.ecnf_cross_attention_grad if grad else lib.ecnf_cross_attention
    _lib.check(fn(args, None if ws is None else ws.data_ptr(), n.value, _stream(device)))


def cross_attention(q, k, v, *, query_lengths=None, context_lengths=None, context_mask=None,
                    scale: Optional[float] = None, return_lse: bool = False):
    """softmax(scale q k^T) v for q [B, Lq, Hq, D] and k, v [C, Lk, Hk, D]: out [B, Lq, Hq, D], and with ``return_lse``
    the rows' log sum exp [B, Hq, Lq] (fp32), which :func:`cross_attention_grad` takes.

    C is B, or 1: one context for the whole batch.  Hq is a multiple of Hk: query head h reads key head
    h // (Hq // Hk).  D is a multiple of 8, at most 128; scale defaults to D^-0.5.  A row reads the keys below
    ``context_lengths`` [C] (clamped to [0, Lk]) where ``context_mask`` [C, Lk] is true; what lies behind is never used,
    NaN included.  A row without keys, and a query at or behind ``query_lengths`` [B], gives 0 and lse -inf."""
    q, k, v, ql, cl, m, scale = _attention_operands(q, k, v, query_lengths, context_lengths, context_mask, scale)
    out = _new(q)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device) if return_lse else None
    if q.shape[0]:
        _run_attention(_attention_args(q, k, v, out, None, lse, None, None, None, ql, cl, m, scale), 0, q.device)
    return (out, lse) if return_lse else out


def cross_attention_grad(out_grad, q, k, v, out, lse, *, query_lengths=None, context_lengths=None, context_mask=None,
                         scale: Optional[float] = None):
    """(dq, dk, dv) of :func:`cross_attention` for ``out_grad``, from its results ``out`` and ``lse``.  The gradients of
    key heads that several query heads share, and of a context that the whole batch shares, are summed (fp32, in a
    fixed order); those of keys that no row may read are 0."""
    q, k, v, ql, cl, m, scale = _attention_operands(q, k, v, query_lengths, context_lengths, context_mask, scale)
    out_grad, out = _tensor(out_grad, "out_grad", q), _tensor(out, "out", q)
    _same_shape(out_grad, q, "out_grad")
    _same_shape(out, q, "out")
    want = (q.shape[0], q.shape[2], q.shape[1])
    if not (torch.is_tensor(lse) and lse.device == q.device and lse.dtype == torch.float32 and tuple(lse.shape) == want):
        raise ValueError(f"lse must be the float32 {want} tensor of cross_attention(return_lse=True)")
    out_grad, out, lse = _aligned(out_grad), _aligned(out.contiguous()), lse.contiguous()
    dq, dk, dv = _new(q), _new(k), _new(k)
    if q.shape[0]:
        _run_attention(_attention_args(q, k, v, out, out_grad, lse, dq, dk, dv, ql, cl, m, scale), 1, q.device)
    else:
        dk.zero_()
        dv.zero_()
    return dq, dk, dv


# ------------------------------------------------------------------------------------------------------ the conditional flow
@dataclass(frozen=True)
class ContextConfig:
    """Attention from the atoms to states [.., state_dim]: n_heads query heads on n_kv_heads key heads of head_dim, turned
    by positions on ``axes`` (:func:`qk_norm_rotary`)."""
    state_dim: int
    n_heads: int = 2
    n_kv_heads: int = 2
    head_dim: int = 32
    axes: Tuple[int, ...] = (32,)
    theta: float = 10000.0
    eps: float = 1e-6
    interleaved: bool = False


class Context(NamedTuple):
    """What a batch of molecules is conditioned on.  params: :func:`init_context_params`; states [C, Lk, state_dim] in
    the dtype to compute in (C: the batch, or 1 for all of it); node_positions [N, n_axes] or [batch, N, n_axes] of the
    atoms and positions [Lk, n_axes] or [C, Lk, n_axes] of the states (the same axes); lengths [C] and mask [C, Lk] as
    in :func:`cross_attention`: the states and positions behind them are not used, NaN included."""
    cfg: ContextConfig
    params: Mapping[str, torch.Tensor]
    states: torch.Tensor
    node_positions: torch.Tensor
    positions: torch.Tensor
    lengths: Optional[torch.Tensor] = None
    mask: Optional[torch.Tensor] = None


def _hidden(cnf_cfg: CNFConfig) -> int:
    return cnf_cfg.ref_hidden or cnf_cfg.hidden


def init_context_params(cfg: ContextConfig, cnf_cfg: CNFConfig, seed: int = 0, device=0) -> Dict[str, torch.Tensor]:
    """Projections (fan-in scaled normal) and norm weights (1), fp32; the output projection is 0, so an untrained
    context leaves the field as it is."""
    dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
    g = torch.Generator()
    g.manual_seed(seed)
    H, q, kv = _hidden(cnf_cfg), cfg.n_heads * cfg.head_dim, cfg.n_kv_heads * cfg.head_dim

    def normal(rows, cols):
        return (torch.randn((rows, cols), generator=g) * rows ** -0.5).to(dev)
    return {"query": normal(H, q), "key": normal(cfg.state_dim, kv), "value": normal(cfg.state_dim, kv),
            "out": torch.zeros((q, H), device=dev), "query_norm": torch.ones(cfg.head_dim, device=dev),
            "key_norm": torch.ones(cfg.head_dim, device=dev)}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[batch, length, ..] -> [batch * length, features] (explicit sizes: any of them may be 0)"""
    return t.reshape(t.shape[0] * t.shape[1], math.prod(t.shape[2:]))


def _mm(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a @ b in fp32.  Two 16-bit operands of a kind go to the matrix units as they are (512 x 333 states of 256: a parameter's
    gradient 399 us of 589), their sums and the result in fp32 all the same."""
    if a.dtype == b.dtype and a.dtype != torch.float32:
        return torch.mm(a, b, out_dtype=torch.float32)
    return a.float() @ b.float()


def _project(x: torch.Tensor, w: torch.Tensor, heads: int) -> torch.Tensor:
    """[B, L, F] @ [F, heads * D] -> [B, L, heads, D] in x's dtype"""
    return (_rows(x) @ w.to(x.dtype)).reshape(x.shape[0], x.shape[1], heads, w.shape[1] // heads)


def _without_padding(context: Context, s: torch.Tensor):
    """(states, positions) with zeros behind the lengths and masks.  The attention does not read there, but the projections
    and the norm do, and in the backward pass NaN times a gradient of 0 would be NaN in every parameter."""
    pos, (n, L) = context.positions, s.shape[:2]
    lengths, mask = _lengths(context.lengths, n, L, s, "context_lengths"), _mask(context.mask, (n, L), s)
    if lengths is None and mask is None:
        return s, pos
    keep = torch.ones((n, L), dtype=torch.bool, device=s.device) if mask is None else mask.bool()
    if lengths is not None:
        keep = keep & (torch.arange(L, device=s.device) < lengths[:, None])
    if torch.is_tensor(pos) and pos.is_floating_point() and pos.device == s.device:
        if pos.dim() == 2 and pos.shape[0] == L:
            pos = pos.expand(n, L, pos.shape[1])   # (a row may lie behind one context's length and not another's)
        if pos.dim() == 3 and pos.shape[:2] == keep.shape:
            pos = pos.masked_fill(~keep[..., None], 0.0)
    return s.masked_fill(~keep[..., None], 0.0), pos


@torch.no_grad()
def node_embedding(embedding: torch.Tensor, features, context: Context, cnf_cfg: CNFConfig,
                   return_saved: bool = False):
    """h_i = E[f_i] + W_out attention(norm_rotary(W_q E[f_i]), norm_rotary(W_k s), W_v s) for every atom i:
    [batch, N, H] in fp32 (batch 1 where features are [N] and the context is shared: the same for every molecule).
    embedding: the field's nn.Embed table [n_features, H] (``EcnfHandle.embedding``).  return_saved: also what
    :func:`node_embedding_grad` takes."""
    c, p = context.cfg, context.params
    H, N = _hidden(cnf_cfg), cnf_cfg.n_nodes
    s = context.states
    if not (torch.is_tensor(s) and s.device == embedding.device and s.dim() == 3 and s.shape[2] == c.state_dim
            and s.dtype in _DTYPES):
        raise ValueError(f"states must be a floating [contexts, length, {c.state_dim}] tensor on {embedding.device}")
    if features is None:
        raise ValueError("features must be given for the EGNN vector field (build_cnf.py:73-75)")
    f = torch.as_tensor(features)
    if f.dtype.is_floating_point:
        raise ValueError("features are integer embedding ids")
    if not f.is_cuda and f.numel() and (int(f.min()) < 0 or int(f.max()) >= cnf_cfg.n_features):
        raise ValueError(f"feature ids must lie in [0, {cnf_cfg.n_features})")
    f = f.to(embedding.device).long()
    if f.dim() == 1:
        f = f[None].expand(s.shape[0], -1)
    elif f.dim() > 1 and f.numel() % N == 0:
        f = f.reshape(f.numel() // N, N)   # [batch, N, 1], as a call without a context takes it
    if f.dim() != 2 or f.shape[1] != N or s.shape[0] not in (1, f.shape[0]):
        raise ValueError(f"features must be [{N}] or [batch, {N}] and states of the same batch or 1, got "
                         f"{tuple(f.shape)} and {tuple(s.shape)}")
    # device-resident ids are not read back: an id outside the table gives NaN rows, as elsewhere on the call path (and a
    # solve, which gets the ids too, reports the molecule)
    known = ((f >= 0) & (f < cnf_cfg.n_features))[..., None]
    e = embedding[:, :H][f.clamp(0, cnf_cfg.n_features - 1)]
    e = torch.where(known, e, torch.full_like(e, float("nan")))
    x = e.to(s.dtype)
    positions = context.positions
    if return_saved:   # (the forward pass reads nothing behind lengths and masks)
        s, positions = _without_padding(context, s)
    q, k, v = (_project(x, p["query"], c.n_heads), _project(s, p["key"], c.n_kv_heads),
               _project(s, p["value"], c.n_kv_heads))
    turn = dict(q_positions=context.node_positions, k_positions=positions, q_weight=p["query_norm"],
                k_weight=p["key_norm"], axes=c.axes, theta=c.theta, eps=c.eps, interleaved=c.interleaved)
    qr, kr = qk_norm_rotary(q, k, **turn)
    keep = dict(context_lengths=context.lengths, context_mask=context.mask)
    o, lse = cross_attention(qr, kr, v, return_lse=True, **keep)
    nodes = e + (_rows(o) @ p["out"].to(o.dtype)).float().reshape(e.shape)
    if not return_saved:
        return nodes
    return nodes, (f, x, s, q, k, v, qr, kr, o, lse, turn, keep, p, embedding.shape)


@torch.no_grad()
def node_embedding_grad(d_nodes: torch.Tensor, saved) -> Dict[str, torch.Tensor]:
    """Gradients of :func:`node_embedding` for the gradient of its result: {"embedding" (the table's), "states", and one
    per context parameter}: the table's in fp32, the others' in their operand's dtype, but in fp32 where that is float16
    (a mean loss's gradients are 1e-8 and less, nothing in float16)."""
    f, x, s, q, k, v, qr, kr, o, lse, turn, keep, p, table = saved
    d_nodes = d_nodes.float().reshape(x.shape)
    weight = lambda n: p[n].to(s.dtype).t()   # what the forward pass multiplied by                   # noqa: E731
    do = _mm(_rows(d_nodes), weight("out")).reshape(o.shape)
    if s.dtype == torch.float16:
        # fp16 ends at 2^-24, and the loss's mean over the batch puts these gradients below (LJ13, 1024 molecules: rms
        # 6e-9).  No power of two is safe for all of the chain, since dK and dV are sums over the batch and the norm divides
        # dK by the keys' size: so the operators' gradients of fp16 values are taken in fp32
        q, k, v, qr, kr, o = (t.float() for t in (q, k, v, qr, kr, o))
    turn = dict(turn, q_weight=turn["q_weight"].float(), k_weight=turn["k_weight"].float())   # their gradients in fp32
    dqr, dkr, dv = cross_attention_grad(do.to(o.dtype), qr, kr, v, o, lse, **keep)
    dq, dk, dqn, dkn = qk_norm_rotary_grad(dqr, dkr, q, k, **turn)
    # the sums over the batch in fp32; the states' two products as one, rounded once
    xt, st, ot, dq, dk, dv = _rows(x).t(), _rows(s).t(), _rows(o).t(), _rows(dq), _rows(dk), _rows(dv)
    g = {"query": _mm(xt, dq), "key": _mm(st, dk), "value": _mm(st, dv), "out": _mm(ot, _rows(d_nodes)), "query_norm": dqn,
         "key_norm": dkn,
         "states": (torch.cat((dk, dv), 1) @ torch.cat((weight("key"), weight("value"))).to(dk.dtype)).reshape(s.shape)}
    like = dict(p, states=s)
    g = {n: t.to(torch.float32 if like[n].dtype == torch.float16 else like[n].dtype) for n, t in g.items()}
    de = d_nodes + _mm(dq, weight("query")).reshape(x.shape)
    # the table's rows: one product with the features' indicator (a fixed order of sums, unlike a scatter)
    hot = (_rows(f[..., None]) == torch.arange(table[0], device=f.device)).to(torch.float32)
    emb = torch.zeros(table, device=f.device, dtype=torch.float32)
    emb[:, :x.shape[-1]] = hot.t() @ _rows(de)
    g["embedding"] = emb
    return g
