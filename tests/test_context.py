"""CPU checks of the context operators' boundary: argument layouts and refusals (nothing is launched)."""
import ctypes

import pytest
import torch

from ecnf_amd import _lib, context


def test_packed_layouts_match_the_library():
    for packed, cls in ((context._QK_NORM, _lib.EcnfQkNorm), (context._ATTENTION, _lib.EcnfAttention)):
        assert packed.size == ctypes.sizeof(cls)
    # field by field: numbers packed in declaration order come out of the structure's fields
    a = _lib.EcnfAttention.from_buffer_copy(context._ATTENTION.pack(*range(1, 34), 0.5))
    assert (a.q, a.context_mask, list(a.q_stride), list(a.out_grad_stride), a.dtype, a.device, a.scale) == (
        1, 12, [13, 14, 15], [22, 23, 24], 25, 33, 0.5)
    n = _lib.EcnfQkNorm.from_buffer_copy(context._QK_NORM.pack(*range(1, 37), *range(1, 10), 0.25, 2.0))
    assert (n.q.x, list(n.q.x_stride), list(n.q.position_stride), n.q.position_type, n.k.x, n.k.position_type) == (
        1, [7, 8, 9], [13, 14], 18, 19, 36)
    assert (n.dtype, n.head_dim, n.n_axes, list(n.axes), n.interleaved, n.device, n.eps, n.theta) == (
        1, 2, 3, [4, 5, 6, 7], 8, 9, 0.25, 2.0)


def _attention(**over):
    d = dict(q=16, k=16, v=16, out=16, out_grad=16, lse=16, q_grad=16, k_grad=16, v_grad=16, dtype=1, batch=2,
             context_batch=2, n_queries=3, context_length=5, heads=4, kv_heads=2, head_dim=64, device=0, scale=0.125)
    d.update(over)
    a = _lib.EcnfAttention(**{k: v for k, v in d.items() if not k.endswith("stride")})
    for n in ("q_stride", "k_stride", "v_stride", "out_grad_stride"):
        setattr(a, n, (ctypes.c_int64 * 3)(*d.get(n, (1024, 64, 64))))
    return bytes(a)


@pytest.mark.parametrize("over,code", [
    (dict(dtype=3), _lib.ECNF_E_INVALID), (dict(dtype=-1), _lib.ECNF_E_INVALID),
    (dict(batch=-1), _lib.ECNF_E_INVALID), (dict(n_queries=-1), _lib.ECNF_E_INVALID),
    (dict(context_length=-1), _lib.ECNF_E_INVALID), (dict(context_batch=3), _lib.ECNF_E_INVALID),
    (dict(context_batch=0), _lib.ECNF_E_INVALID), (dict(heads=3), _lib.ECNF_E_INVALID),
    (dict(kv_heads=0), _lib.ECNF_E_INVALID), (dict(heads=0), _lib.ECNF_E_INVALID),
    (dict(head_dim=0), _lib.ECNF_E_UNSUPPORTED), (dict(head_dim=20), _lib.ECNF_E_UNSUPPORTED),
    (dict(head_dim=136), _lib.ECNF_E_UNSUPPORTED), (dict(scale=float("nan")), _lib.ECNF_E_INVALID),
    (dict(scale=float("inf")), _lib.ECNF_E_INVALID),
    (dict(context_batch=1, batch=2 ** 30, n_queries=4), _lib.ECNF_E_UNSUPPORTED),
    (dict(q_stride=(1024, -64, 64)), _lib.ECNF_E_INVALID), (dict(k_stride=(-1024, 64, 64)), _lib.ECNF_E_INVALID),
    (dict(v_stride=(1024, 2 ** 23, 64)), _lib.ECNF_E_UNSUPPORTED),
])
def test_attention_refusals_of_both_calls(over, code):
    lib, n = _lib.load(), ctypes.c_size_t()
    args = _attention(**over)
    for grad in (0, 1):
        assert lib.ecnf_cross_attention_workspace_size(args, grad, ctypes.byref(n)) == code
    assert lib.ecnf_cross_attention(args, None, 0, None) == code
    assert lib.ecnf_cross_attention_grad(args, None, 0, None) == code
    assert lib.ecnf_last_error()


@pytest.mark.parametrize("over", [dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(q=8), dict(k=2), dict(v=4),
                                  dict(out=24), dict(q_stride=(1024, 64, 4)), dict(k_stride=(1023, 64, 64)),
                                  dict(v_stride=(1024, 36, 64))])
def test_attention_refuses_missing_and_unaligned_operands(over):
    assert _lib.load().ecnf_cross_attention(_attention(**over), None, 0, None) == _lib.ECNF_E_INVALID


@pytest.mark.parametrize("over", [dict(out_grad=None), dict(lse=None), dict(q_grad=None), dict(k_grad=None),
                                  dict(v_grad=None), dict(out_grad=8), dict(out_grad_stride=(1024, 4, 64))])
def test_attention_grad_refuses_missing_operands(over):
    assert _lib.load().ecnf_cross_attention_grad(_attention(**over), 16, 1 << 30, None) == _lib.ECNF_E_INVALID


def test_attention_refuses_a_small_workspace():
    lib, n = _lib.load(), ctypes.c_size_t()
    args = _attention(n_queries=1, context_length=65536)
    for grad, call in ((0, lib.ecnf_cross_attention), (1, lib.ecnf_cross_attention_grad)):
        assert lib.ecnf_cross_attention_workspace_size(args, grad, ctypes.byref(n)) == _lib.ECNF_OK and n.value > 0
        assert call(args, 16, n.value - 1, None) == _lib.ECNF_E_INVALID
        assert call(args, None, n.value, None) == _lib.ECNF_E_INVALID
        assert call(args, 8, n.value, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_cross_attention_workspace_size(None, 0, ctypes.byref(n)) == _lib.ECNF_E_INVALID
    assert lib.ecnf_cross_attention_workspace_size(args, 0, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_cross_attention(None, None, 0, None) == _lib.ECNF_E_INVALID


def _norm(**over):
    d = dict(dtype=1, head_dim=64, axes=(64,), theta=1e4, eps=1e-6, batch=2, length=3, heads=4, position_type=0, x=16,
             grad=16, out=16, positions=16, weight=16, weight_grad=16)
    d.update(over)
    side = (d["x"], d["grad"], d["out"], d["weight"], d["weight_grad"], d["positions"], 768, 256, 64, 768, 256, 64, 3, 1,
            d["batch"], d["length"], d["heads"], d["position_type"])
    axes = tuple(d["axes"])
    return context._QK_NORM.pack(*side, *context._NO_SIDE, d["dtype"], d["head_dim"], d.get("n_axes", len(axes)),
                                 *(axes + (0,) * 4)[:4], 0, 0, d["eps"], d["theta"])


@pytest.mark.parametrize("over,code", [
    (dict(dtype=5), _lib.ECNF_E_INVALID), (dict(head_dim=63), _lib.ECNF_E_UNSUPPORTED),
    (dict(head_dim=0), _lib.ECNF_E_UNSUPPORTED), (dict(head_dim=130), _lib.ECNF_E_UNSUPPORTED),
    (dict(n_axes=0), _lib.ECNF_E_INVALID), (dict(n_axes=5), _lib.ECNF_E_INVALID),
    (dict(axes=(63,)), _lib.ECNF_E_INVALID), (dict(axes=(66,)), _lib.ECNF_E_INVALID),
    (dict(axes=(32, 34)), _lib.ECNF_E_INVALID), (dict(axes=(32, 0)), _lib.ECNF_E_INVALID),
    (dict(axes=(32, -2)), _lib.ECNF_E_INVALID), (dict(axes=(2 ** 30, 2 ** 30)), _lib.ECNF_E_INVALID),
    (dict(theta=0.0), _lib.ECNF_E_INVALID), (dict(theta=float("nan")), _lib.ECNF_E_INVALID),
    (dict(eps=-1.0), _lib.ECNF_E_INVALID), (dict(eps=float("inf")), _lib.ECNF_E_INVALID),
    (dict(batch=-1), _lib.ECNF_E_INVALID), (dict(position_type=3), _lib.ECNF_E_INVALID),
    (dict(x=None), _lib.ECNF_E_INVALID), (dict(out=None), _lib.ECNF_E_INVALID),
    (dict(positions=None), _lib.ECNF_E_INVALID), (dict(batch=2 ** 16, length=2 ** 16), _lib.ECNF_E_UNSUPPORTED),
])
def test_norm_refusals_of_both_calls(over, code):
    lib = _lib.load()
    args = _norm(**{k: 0 if v is None else v for k, v in over.items()})
    assert lib.ecnf_qk_norm_rotary(args, None) == code
    assert lib.ecnf_qk_norm_rotary_grad(args, 16, 1 << 30, None) == code
    assert lib.ecnf_last_error()


def test_norm_grad_refuses_missing_operands_and_a_small_workspace():
    lib, n = _lib.load(), ctypes.c_size_t()
    for over in (dict(grad=0), dict(weight_grad=0)):
        assert lib.ecnf_qk_norm_rotary_grad(_norm(**over), 16, 1 << 30, None) == _lib.ECNF_E_INVALID
    args = _norm()
    assert lib.ecnf_qk_norm_workspace_size(args, ctypes.byref(n)) == _lib.ECNF_OK and n.value > 0
    assert lib.ecnf_qk_norm_rotary_grad(args, None, n.value, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_qk_norm_rotary_grad(args, 16, 3, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_qk_norm_workspace_size(None, ctypes.byref(n)) == _lib.ECNF_E_INVALID
    assert lib.ecnf_qk_norm_rotary(None, None) == _lib.ECNF_E_INVALID


def test_host_tensors_are_refused():
    q = torch.zeros(1, 2, 1, 16)
    with pytest.raises(ValueError, match="device"):
        context.cross_attention(q, q, q)
    with pytest.raises(ValueError, match="device"):
        context.qk_norm_rotary(q, q_positions=torch.zeros(2, 1), axes=(16,))


def test_node_entries_refuse_missing_handles():
    lib = _lib.load()
    assert lib.ecnf_vector_field_nodes(None, None, None, None, 1, None, None, 1, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_integrate_nodes(None, None, None, None, 1, None, None, None, None, None, None, 1, None, 0,
                                    None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_fm_loss_grad_nodes(None, None, None, None, None, None, 0.0, 1, None, None, None,
                                       None) == _lib.ECNF_E_INVALID
