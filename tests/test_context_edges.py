"""CPU checks of the context operators' edges: refusals that no launch follows, and how the Python side hands calls over."""
import pytest
import torch

from ecnf_amd import _lib, context
from test_context import _attention, _norm


@pytest.mark.parametrize("over", [dict(k_stride=(1024, 0, 64)), dict(v_stride=(1024, 0, 64)), dict(k_stride=(1024, 56, 64)),
                                  dict(v_stride=(1024, 8, 64))])
def test_rows_of_keys_that_overlap_are_refused(over):
    lib = _lib.load()
    assert lib.ecnf_cross_attention(_attention(**over), None, 0, None) == _lib.ECNF_E_INVALID
    assert lib.ecnf_cross_attention_grad(_attention(**over), None, 0, None) == _lib.ECNF_E_INVALID
    assert b"overlap" in lib.ecnf_last_error()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_keys_are_copied_where_the_library_refuses_them(dtype):
    e = torch.finfo(dtype).bits // 8
    x = torch.zeros((2, 3, 2, 16), dtype=dtype)
    same = [x, x[:, :1].expand(2, 1, 2, 16), x.transpose(0, 1), torch.zeros(4 << 20, dtype=dtype).as_strided((1, 2, 1, 16), (0, (8 << 20) // e - 16, 16, 1))]
    copied = [x[:, :1].expand(2, 3, 2, 16), torch.zeros(100, dtype=dtype).as_strided((1, 3, 1, 16), (48, 8, 16, 1)),
              torch.zeros(5 << 20, dtype=dtype).as_strided((1, 2, 1, 16), (0, (8 << 20) // e, 16, 1))]
    for t in same:
        assert context._key_rows(t).data_ptr() == t.data_ptr()
    for t in copied:
        y = context._key_rows(t)
        assert y.is_contiguous() and y.shape == t.shape and y.data_ptr() != t.data_ptr()


@pytest.mark.parametrize("over", [
    dict(batch=2 ** 22, context_batch=2 ** 22, n_queries=1, context_length=1, heads=4, kv_heads=4),
    dict(batch=2 ** 13, context_batch=2 ** 13, n_queries=128 * 2 ** 9, context_length=3, heads=4, kv_heads=4)])
def test_more_workgroups_than_a_launch_takes_are_refused(over):
    """A launch has fewer than 2^32 threads, so 2^24 workgroups of 256: refused before the first of a call's launches."""
    lib = _lib.load()
    args = _attention(**over)
    assert lib.ecnf_cross_attention(args, 16, 1 << 40, None) == _lib.ECNF_E_UNSUPPORTED
    assert lib.ecnf_cross_attention_grad(args, 16, 1 << 40, None) == _lib.ECNF_E_UNSUPPORTED
    assert b"too many rows" in lib.ecnf_last_error()


def test_more_workgroups_of_the_norm_than_a_launch_takes_are_refused():
    lib = _lib.load()
    args = _norm(batch=2 ** 12, length=2 ** 12, heads=2 ** 15)
    assert lib.ecnf_qk_norm_rotary(args, None) == _lib.ECNF_E_UNSUPPORTED
    assert b"too many tokens" in lib.ecnf_last_error()
