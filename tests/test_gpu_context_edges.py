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


