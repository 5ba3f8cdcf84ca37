"""linear_act for few rows on every form of that kernel, the form asserted for each call (tests/test_linear_few_rule.py has the rule): rows at both ends of a form's
class, features that fill the last work group and that leave it a rest, whole and partial steps, rows on 128-byte lines and off them where the rule lets
both. Operands with poisoned borders; tests/test_linear_act_gpu.py derives the bounds. And rows by themselves and among others."""
import pytest
import torch

import brodiffusion_amd as bd
from test_linear_act_forms_gpu import _poisoned
from test_linear_act_gpu import call, check, make
from test_linear_few_rule import KINDS, few_form, table

pytestmark = pytest.mark.gpu

ACTS = ("none", "gelu", "gelu_tanh", "silu")


def _row(K, kind, on_lines):
    """The stride of rows of K elements that begin on 128-byte lines (INT8: of both operands), or the next one that is allowed and is off them"""
    line, least = (128, 16) if kind == "w8a8" else (64, 8)
    if kind == "w8":
        line = 128
    row = -(-(K + least) // line) * line
    return row if on_lines else row + least * (2 if kind == "w8" and K % 16 == 0 else 1)


def _problems(kind, form, compute_units):
    """(M, N, K, on lines): of every pair of a width and a contraction that get the form the first and the last number of rows, up to 12 spread over all"""
    found = []
    per_cu = compute_units
    for N in (24, 1160, 8 * per_cu - 8, 8 * per_cu + 8, 12 * per_cu - 8, 13 * per_cu, 16 * per_cu, 16 * per_cu + 8, 5128, 24 * per_cu - 8, 24 * per_cu + 8, 28 * per_cu, 32 * per_cu - 8, 32 * per_cu,
              32 * per_cu + 8, 64 * per_cu - 8, 64 * per_cu, 64 * per_cu + 8):
        for K in (80, 1168, 2032, 4880, 5184):
            for on_lines in (True, False):
                rows = [M for M in range(1, 33) if few_form(M, N, K, kind, _row(K, kind, on_lines), compute_units) == form]
                found += [(M, N, K, on_lines) for M in sorted({*rows[:1], *rows[-1:]})]
    step = -(-len(found) // 12) | 1       # (odd: first and last rows in turn)
    return found[::step] + found[-1:]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind,form", [(k, f) for k in KINDS for f in table(k)])
def test_every_form(kind, form, dtype):
    compute_units = bd.device_info()["compute_units"]
    problems = _problems(kind, form, compute_units)
    assert problems
    for i, (M, N, K, on_lines) in enumerate(problems):
        k = K - 8 if kind == "w8" and i % 2 else K       # (INT8 weights of rows on 8-byte addresses)
        row = _row(k, kind, on_lines)
        if few_form(M, N, k, kind, row, compute_units) != form:
            k, row = K, _row(K, kind, on_lines)
        assert few_form(M, N, k, kind, row, compute_units) == form
        c = make(M + N + k + i, kind, M, N, k, dtype, bias=i % 3 != 1, residual=i % 3 != 2)
        c["x"], c["w"] = _poisoned(c["x"], row - k), _poisoned(c["w"], row - k)
        wide = torch.full((M + 1, N + 8), 7.0, dtype=c["dt"], device="cuda")
        call(c, ACTS[i % 4], out=wide[:M, :N])
        check(c, ACTS[i % 4], wide[:M, :N], f"{M} x {N} x {k}, {'on' if on_lines else 'off'} lines")
        assert bool((wide[M:] == 7).all()) and bool((wide[:, N:] == 7).all())


def _rows_of(c, rows):
    d = {**c, "x": c["x"][rows].contiguous(), "residual": c["residual"][rows].contiguous()}
    if c["x_scales"] is not None:
        d["x_scales"] = c["x_scales"][rows].contiguous()
    return d


@pytest.mark.parametrize("kind,K", [("w16", 5184), ("w8", 5184), ("w8a8", 10368)])
def test_any_number_of_rows_of_a_class_gives_the_same_bits(kind, K):
    """9 to 16 rows, in any order: one form of the kernel for few rows."""
    N = 6136
    c = make(5, kind, 16, N, K, "bf16")
    whole = call(c, "silu")
    check(c, "silu", whole)
    for M in range(9, 17):
        assert few_form(M, N, K, kind, 0, bd.device_info()["compute_units"]) == (2, 3, 2, 2, 4)
        rows = torch.randperm(16, generator=torch.Generator().manual_seed(M))[:M].cuda()
        assert torch.equal(call(_rows_of(c, rows), "silu"), whole[rows]), M


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,K", [(12, 6136, 5184), (40, 328, 640), (46, 368, 16000), (300, 1160, 1168), (2188, 5392, 1152)])
def test_other_rows_do_not_change_a_row(kind, M, N, K):
    """Every third row kept, the others replaced (some by what is not finite): the kept rows' bits."""
    c, other = make(7, kind, M, N, K, "fp16"), make(8, kind, M, N, K, "fp16")
    whole = call(c, "gelu")
    kept = torch.arange(M, device="cuda") % 3 == 0
    d = {**c, "x": torch.where(kept[:, None], c["x"], other["x"])}
    if kind == "w8a8":
        d["x_scales"] = torch.where(kept, c["x_scales"], other["x_scales"])
        d["x_scales"][1] = float("nan")
    else:
        d["x"][1, 3], d["x"][M - 1 if (M - 1) % 3 else M - 2, K - 1] = float("inf"), float("nan")
    again = call(d, "gelu")
    assert torch.equal(again[kept], whole[kept]) and not torch.isfinite(again[1]).any()
