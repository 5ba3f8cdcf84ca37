"""Which problems the linear layer's kernel for few rows takes and with which work groups (csrc/linear_few_forms.h), asked of the rule on the host: every
form of its tables is one that calls reach, and every form that they reach is in the tables and in the library."""
import ctypes as C
import os
import re

import pytest

from brodiffusion_amd import build
from test_kernel_resources import kernels  # noqa: F401

KINDS = {"w16": 0, "w8": 1, "w8a8": 2}


def few_form(M, N, K, kind, row=0, compute_units=256):
    """The form of a problem, None if the kernel does not take it"""
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    form = (C.c_int * 5)()
    return tuple(form) if C.CDLL(build.FORMS_LIB).linear_few(M, N, K, row or K, KINDS[kind], compute_units, form) else None


def table(kind):
    if not os.path.exists(build.FORMS_LIB):
        build.build_host()
    forms = (C.c_int * 160)()
    n = C.CDLL(build.FORMS_LIB).linear_few_table(KINDS[kind], forms)
    return [tuple(forms[5 * i:5 * i + 5]) for i in range(n)]


@pytest.mark.parametrize("kind", KINDS)
def test_every_form_is_reached_and_built(kernels, kind):
    reached = set()
    for N in list(range(1024, 20000, 504)) + [8, 2048, 2056, 4096, 4104, 6144, 6152, 8192, 8200, 12288, 12296, 16384, 16392]:
        for K in (64, 1024, 1152, 2112, 4096, 5120, 16384):
            reached |= {few_form(M, N, K, kind) for M in range(1, 34)}
    reached.discard(None)
    assert len(table(kind)) == len(set(table(kind))) and reached == set(table(kind))
    for t in ("DF16_", "DF16b"):
        built = {tuple(map(int, m.groups())) for name in kernels
                 if (m := re.search(rf"linear_few_kernelI{t}Li{KINDS[kind]}ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)E", name))}
        assert built == reached


@pytest.mark.parametrize("kind", KINDS)
def test_a_form_holds_the_rows_and_fills_the_features(kind):
    for M in range(1, 33):
        for N in (8, 1152, 2056, 4104, 6144, 6152, 8200, 16384, 16392):
            for K in (64, 1168, 4880, 16384):
                if (f := few_form(M, N, K, kind)) is not None:
                    groups, features, rows, steps, wavefronts = f
                    assert 16 // groups * rows >= M and wavefronts in (4, 8) and steps in (1, 2)
    assert few_form(33, 1152, 64, kind) is None


def test_the_widest_layers_take_the_form_that_the_busiest_compute_unit_has_less_of():
    for kind in KINDS:
        assert few_form(8, 6144, 16384, kind)[1] == 3 and few_form(8, 8192, 16384, kind)[1] == 4 and few_form(8, 7168, 16384, kind)[1] == 4
        assert few_form(16, 6144, 16384, kind) == (2, 3, 2, 2, 4) and few_form(16, 7168, 16384, kind) == (2, 4, 2, 2, 4)
    for kind in ("w16", "w8"):
        assert few_form(20, 6144, 16384, kind) == (2, 3, 3, 2, 4) and few_form(20, 7168, 16384, kind) == (2, 4, 3, 2, 4)
    assert few_form(32, 6144, 16384, "w8") == (2, 3, 4, 2, 4) and few_form(32, 8192, 16384, "w8") == (2, 4, 4, 2, 4)


def test_wide_layers_off_lines():
    assert few_form(24, 16384, 6144, "w16") == (2, 4, 3, 2, 4) and few_form(24, 16384, 6144, "w16", 6152) is None and few_form(4, 16384, 6144, "w16", 6152) is not None
