"""The C entries of the linear layer with 4-bit weights without a GPU: struct layouts, sizes, and refusals ahead of any launch (what is passed as a tensor is never read)."""
import ctypes as C
import os
import re
import subprocess

import pytest

from brodiffusion_amd import _capi as capi
from brodiffusion_amd import build
from test_kernel_resources import kernels  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAR = 1 << 40


def test_struct_layouts_match_c(tmp_path):
    pairs = [("mi_pack_int4_args", capi.MiPackInt4Args), ("mi_linear_int4_args", capi.MiLinearInt4Args)]
    lines, want = [], []
    for name, cls in pairs:
        lines += [f'printf("%zu\\n", sizeof({name}));'] + [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
        want += [C.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mi_attention.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    assert [int(v) for v in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()] == want


@pytest.mark.parametrize("n,k,size", [(8, 8, 1024), (16, 128, 1024), (24, 136, 4096), (16384, 6144, 16384 * 6144 // 2), (0, 128, 0), (16, -8, 0), (1 << 30, 1 << 30, 1 << 59)])
def test_packed_bytes(n, k, size):
    assert capi.lib().mi_int4_packed_bytes(n, k) == size


# (4 rows, 264 in, 40 out, groups of 64: x 2112 bytes, w 9216, scales 400, zeros 200, bias 80, residual and y 320)
def _linear(**kw):
    a = capi.MiLinearInt4Args()
    a.struct_size, a.dtype, a.rows, a.in_features, a.out_features, a.group = C.sizeof(a), capi.MI_DTYPE_BF16, 4, 264, 40, 64
    a.x, a.w, a.scales, a.zeros, a.bias, a.residual, a.y = (0x10000 * i for i in range(1, 8))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _pack(**kw):
    a = capi.MiPackInt4Args()
    a.struct_size, a.out_features, a.in_features = C.sizeof(a), 40, 264
    a.q, a.packed = 0x10000, 0x20000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fields,said", [
    (dict(struct_size=8), "struct_size"), (dict(dtype=7), "dtype"), (dict(rows=-1), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(in_features=0), "features"), (dict(out_features=-8), "features"),
    (dict(in_features=260), "multiples of 8"), (dict(out_features=36), "multiples of 8"), (dict(in_features=(1 << 30) + 8), "2^30"), (dict(activation=4), "activation"), (dict(activation=-1), "activation"),
    (dict(group=0), "group"), (dict(group=-64), "group"), (dict(group=16), "group"), (dict(group=96), "group"), (dict(group=192), "group"), (dict(x=None), "null"), (dict(w=None), "null"),
    (dict(scales=None), "null"), (dict(y=None), "null"), (dict(x_row_stride=268), "multiples"), (dict(x_row_stride=256), "smaller"), (dict(y_row_stride=32), "smaller"), (dict(residual_row_stride=8), "smaller"),
    (dict(y_row_stride=FAR + 8), "2^40"), (dict(rows=1 << 30, x_row_stride=FAR), "2^56"), (dict(x=0x10008), "16-byte"), (dict(scales=0x30008), "16-byte"), (dict(bias=0x50002), "16-byte"), (dict(zeros=0x40004), "8-byte"),
    (dict(y=0x60010), "overlaps the residual"), (dict(y=0x60000, y_row_stride=48), "overlaps the residual"), (dict(y=0x10100, residual=None), "overlaps x"), (dict(y=0x223f0), "overlaps w"),
    (dict(y=0x30180), "overlaps scales"), (dict(y=0x3fed0), "overlaps zeros"), (dict(y=0x4fed0), "overlaps the bias")])
def test_refusals(fields, said):
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(**fields))) == -1
    assert "mi_linear_int4_forward" in capi.last_error() and said in capi.last_error(), capi.last_error()


@pytest.mark.parametrize("fields,said", [
    (dict(struct_size=8), "struct_size"), (dict(in_features=260), "multiples of 8"), (dict(out_features=0), "features"), (dict(q=None), "null"), (dict(packed=None), "null"), (dict(q_row_stride=128), "stride"),
    (dict(q_row_stride=134), "stride"), (dict(q_row_stride=FAR + 4), "2^56"), (dict(out_features=1 << 30, q_row_stride=1 << 34), "2^56"), (dict(q=0x10002), "4-byte"), (dict(packed=0x20008), "16-byte"),
    (dict(packed=0x11490), "overlaps"), (dict(q=0x223fc), "overlaps")])
def test_pack_refusals(fields, said):
    assert capi.lib().mi_pack_int4(C.byref(_pack(**fields))) == -1
    assert "mi_pack_int4" in capi.last_error() and said in capi.last_error(), capi.last_error()


def test_no_rows_is_no_error():
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(rows=0, x=None))) == 0


def _launch(m, n, k, group, row=0, lent=(1 << 64) - 1):
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    shares = C.c_int()
    return C.CDLL(build.FORMS_LIB).int4_form_test(m, n, k, C.c_long(row or k), group, 256, C.c_ulong(lent), C.byref(shares)), shares.value


def test_instances_are_those_that_calls_reach(kernels):  # noqa: F811
    """Work groups by the rule (csrc/linear_int4_forms.h), over sizes and kinds of groups, against what is in the library"""
    sizes = [(m, n, k) for m in (1, 16, 40, 200, 333, 777, 2049, 3000) for n in (8, 264, 1160, 2056, 4104, 8200, 16392) for k in (8, 264, 1160, 2056, 3088, 8200, 16392)]
    reached = {(p, _launch(m, n, k, 128 // p)[0]) for p in (1, 2, 4) for m, n, k in sizes}
    assert reached == {(p, f) for p in (1, 2, 4) for f in range(9)} - {(4, 2), (2, 8), (4, 8)}
    few = {(p, 1 << f) for p, f in reached if f < 3}
    tiles = {(p, z, *((2, 1), (2, 2), (4, 2), (4, 3), (6, 3), (4, 4))[f - 3]) for p, f in reached if f >= 3 for z in (0, 1)}
    for t in ("DF16_", "DF16b"):
        assert {tuple(map(int, m.groups())) for name in kernels if (m := re.search(rf"linear_int4_few_kernelI{t}Li(\d+)ELi(\d+)E", name))} == few
        assert {tuple(map(int, m.groups())) for name in kernels if (m := re.search(rf"linear_int4_tile_kernelI{t}Li(\d+)ELb(\d)ELi(\d+)ELi(\d+)E", name))} == tiles


def test_more_rows_than_a_c_int(monkeypatch):
    import torch
    from brodiffusion_amd import ops
    monkeypatch.setattr(ops, "_dev", lambda *a: None)
    rows = lambda n: torch.empty(n, 8, dtype=torch.float16, device="meta")
    assert ops._rows_of("op", rows(2 ** 31 - 1), "X", torch.float16) == (2 ** 31 - 1, 8)
    with pytest.raises(RuntimeError, match="more than 2\\^31 - 1 rows"):
        ops._rows_of("op", rows(2 ** 32 + 5), "X", torch.float16)


def test_rows_far_apart_and_many_features_get_64_bit_offsets():
    for m in (70, 5000):
        assert _launch(m, 1160, 136, 64, 11184816)[0] < 3 and _launch(m, (1 << 24) + 8, 136, 64)[0] < 3
        assert _launch(5000, 1160, 136, 64, 11184808)[0] >= 3


def test_shares_of_the_contraction():
    """No more than are lent, none of less than four blocks, none where nothing is lent; sizes whose sums pass 64 bits"""
    for m, n, k in [(1, 264, 16392), (17, 8200, 8200), (200, 1160, 16384), (333, 2056, 4616), (1, 8, 8)]:
        shares = _launch(m, n, k, 128)[1]
        assert 1 <= shares <= 16 and -(-k // 128) >= 4 * shares or shares == 1
        for lent in (0, 1, 4 * m * n, 8 * m * n - 1, 8 * m * n, 4 * shares * m * n - 1, 4 * shares * m * n):
            got = _launch(m, n, k, 128, lent=lent)[1]
            assert got == 1 or 4 * got * m * n <= lent
        assert _launch(m, n, k, 128, lent=4 * shares * m * n)[1] == shares
    for m, n, k in [(1 << 30, 1 << 30, 1 << 30), (1 << 30, 8, 1 << 30), (1, 1 << 30, 8)]:
        assert _launch(m, n, k, 128)[1] == 1


def test_scratch_bytes():
    a = _linear(rows=1, in_features=16392, out_features=264, group=128, x=0x1000000, w=0x2000000, scales=0x3000000, zeros=None, residual=None, y=0x5000000)
    need = capi.lib().mi_linear_int4_scratch_bytes(C.byref(a))
    assert need > 0 and need % (4 * 264) == 0
    a.scratch, a.scratch_bytes = 0x2000000, 1 << 20
    assert capi.lib().mi_linear_int4_scratch_bytes(C.byref(a)) == need
    assert capi.lib().mi_linear_int4_scratch_bytes(C.byref(_linear())) == 0 and capi.lib().mi_linear_int4_scratch_bytes(None) == 0
    a.group = 100
    assert capi.lib().mi_linear_int4_scratch_bytes(C.byref(a)) == 0


@pytest.mark.parametrize("name,at", [("x", 0x10000), ("x", 0x10830), ("w", 0x20000), ("w", 0x223f0), ("scales", 0x30180), ("zeros", 0x400c0), ("bias", 0x50040), ("residual", 0x60130), ("y", 0x70000)])
def test_scratch_that_is_part_of_an_operand(name, at):
    for scratch, size in ((at, 64), (at - 0x400, 0x410)):
        assert capi.lib().mi_linear_int4_forward(C.byref(_linear(scratch=scratch, scratch_bytes=size))) == -1
        assert f"scratch overlaps {name}" in capi.last_error(), capi.last_error()
    assert capi.lib().mi_linear_int4_forward(C.byref(_linear(scratch=0x80008, scratch_bytes=64))) == -1 and "scratch must be 16-byte" in capi.last_error()


def test_no_scratch_memory(kernels):  # noqa: F811
    found = {name: (k[".private_segment_fixed_size"], k[".vgpr_spill_count"]) for name, k in kernels.items() if "linear_int4_" in name or "pack_int4" in name}
    assert len(found) > 60 and not {name: use for name, use in found.items() if use != (0, 0)}
