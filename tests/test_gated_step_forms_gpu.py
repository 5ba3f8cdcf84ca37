"""What the tests of linear_int4 and gate_add_norm leave between them: the table of kernel instances has every one, rows that are not finite under each activation,
and a block in which every step is held to its bound."""
import pytest
import torch

import brodiffusion_amd as bd
import test_gate_norm_gpu as step
import test_linear_int4_gpu as linear
from helpers import TORCH_DT

pytestmark = pytest.mark.gpu

MORE = {(32, linear.TILE64x192, 0): (386, 136, 14000)}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group,form,shared", list(MORE))
def test_more_forms(dtype, zeros, group, form, shared):
    m, k, n = MORE[group, form, shared]
    got, shares = linear._launch(m, k, n, group)
    assert got == form and (shares > 1) == bool(shared)
    linear._case(dtype, m, k, n, group, zeros, bias=True, act="silu", residual=True)


def test_the_table_of_forms_is_whole():
    """Every form of each kind of groups, with the contraction whole and in shares"""
    table = {(g, *f) for g in linear.PROBLEMS for f in linear.PROBLEMS[g]} | set(MORE)
    never = {(32, linear.FEW64), (32, linear.TILE64x256), (64, linear.TILE64x256)}
    assert table == {(g, f, s) for g in (32, 64, 128) for f in range(9) for s in (0, 1) if (g, f) not in never}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,k,n,group", [(4, 520, 264, 128), (50, 520, 264, 64), (90, 520, 264, 32), (300, 520, 264, 128), (2049, 264, 1160, 64), (4, 8200, 264, 128), (300, 8200, 264, 32)])
def test_rows_that_are_not_finite_under_an_activation(dtype, act, m, k, n, group):
    """... with zero points of 0 and a residual: such rows are NaN throughout, the others keep their bits"""
    g = torch.Generator().manual_seed(m + k)
    t = TORCH_DT[dtype]
    q, scales, z = linear._checkpoint(g, n, k, group, True, t)
    z[:, ::2] = 0
    w = bd.pack_int4(q, scales, z, group=group)
    x, r = torch.randn(m, k, generator=g).to(t).cuda(), torch.randn(m, n, generator=g).to(t).cuda()
    want = bd.linear_int4(x, w, activation=act, residual=r)
    x[1, k - 1], x[3, 0], x[2, 130] = float("inf"), float("nan"), float("-inf")
    y = bd.linear_int4(x, w, activation=act, residual=r)
    keep = [i for i in range(m) if i not in (1, 2, 3)]
    assert torch.equal(y[keep], want[keep]) and torch.isfinite(want).all() and torch.isnan(y[1:4]).all()


def test_every_step_of_a_block():
    """Gated residual with a norm behind the block, two 4-bit products, the gated residual of their result with the next block's norm: each on what the step before stored"""
    g = torch.Generator().manual_seed(12)
    t, d, hidden, items, tokens = torch.bfloat16, 1152, 4608, 2, 37
    q1, s1, _ = linear._checkpoint(g, hidden, d, 128, False, t)
    q2, s2, z2 = linear._checkpoint(g, d, hidden, 64, True, t)
    w1, w2 = bd.pack_int4(q1, s1), bd.pack_int4(q2, s2, z2, group=64)
    x, att = (torch.randn(items, tokens, d, generator=g).to(t).cuda() for _ in range(2))
    mod = (0.3 * torch.randn(items, 6 * d, generator=g)).to(t).cuda()
    part = lambda i: mod[:, i * d:(i + 1) * d]
    first = dict(gate=part(2), scale=part(4), shift=part(3), norm="layer")
    next_ = dict(gate=part(5), post="rms", norm="layer", scale=part(1), shift=part(0))
    wide = lambda kw: {k: v if isinstance(v, str) else v[:, None] for k, v in kw.items()}
    h, y = bd.gate_add_norm(x, att, **first)
    step._check(x, att, t, h, y, **wide(first))
    u = bd.linear_int4(y, w1, activation="gelu_tanh")
    linear._check(u.view(-1, hidden), *linear._reference(y.view(-1, d), q1, s1, None, 128, None, "gelu_tanh", None))
    v = bd.linear_int4(u, w2)
    linear._check(v.view(-1, d), *linear._reference(u.view(-1, hidden), q2, s2, z2, 64, None, "none", None))
    h2, y2 = bd.gate_add_norm(h, v, **next_)
    step._check(h, v, t, h2, y2, **wide(next_))
