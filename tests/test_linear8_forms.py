"""The choice among the forms of nb_linear8's product (csrc/nb_linear8_forms.h, host
arithmetic), compiled for the CPU: every form is reached by the shapes that the GPU
tests run, and every launch within the documented sizes is one that the runtime takes."""
import ctypes
import os
import shutil
import subprocess

import pytest

from tests.conftest import ROOT
from tests.test_gpu_linear8 import FORMS

CXX = shutil.which("g++") or shutil.which("c++")
SHIM = """
#include "nb_linear8_forms.h"
using namespace nb::linear8;
extern "C" int count() { return kFormCount; }
extern "C" int chosen(int M, int N, int K, int cus) { return form_of(M, N, K, cus); }
extern "C" int tiles(int i) { return kForms[i].tiles; }
extern "C" long groups(int i, int M, int N, long* rows) {
    *rows = (long)row_groups(kForms[i], M);
    return (long)output_groups(kForms[i], N);
}
"""


@pytest.fixture(scope="module")
def forms(tmp_path_factory):
    if CXX is None:
        pytest.skip("no host compiler")
    where = tmp_path_factory.mktemp("forms")
    (where / "shim.cpp").write_text(SHIM)
    so = where / "shim.so"
    subprocess.run([CXX, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "nativebit_amd", "csrc"), str(where / "shim.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    lib.groups.restype = ctypes.c_long
    lib.groups.argtypes = [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_long)]
    return lib


def test_every_form_is_reached(forms):
    assert forms.count() == 9
    assert {forms.chosen(M, N, K, 256) for M, N, K in FORMS} == set(range(9))


@pytest.mark.parametrize("cus", [32, 228, 256, 304])
def test_launches_fit(forms, cus):
    """Grids: a form for few rows has its row tiles in the second dimension (at most
    65535), all are under 2^22 workgroups of up to 512 threads."""
    rows = [1, 7, 33, 1 << 12, 65535 * 16 - 1, 65535 * 16, 65535 * 16 + 1, (1 << 20) - 1, 1 << 20]
    outputs = [1, 16, 17, 32, 33, 100, 1000, 4096, 65535, 1 << 20, 1 << 24]
    for M in rows:
        for N in outputs:
            if M * N >= 1 << 36:
                continue
            for K in (128, 384, 2560, 6912, 1 << 17):
                i = forms.chosen(M, N, K, cus)
                y = ctypes.c_long()
                x = forms.groups(i, M, N, ctypes.byref(y))
                assert x * y.value < 1 << 22, (M, N, K, i)
                assert forms.tiles(i) or y.value <= 65535, (M, N, K, i)
