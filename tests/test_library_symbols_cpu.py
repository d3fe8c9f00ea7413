"""libnabla_g1.so shows its C entries and nothing else: two copies of it in one process (the profile build beside the
product, a program that compiles the same sources in) share neither kernels nor what a copy remembers of its own."""
import shutil
import subprocess

import pytest

from nablaengine_b200 import build, capi


def test_the_library_exports_its_c_entries_alone():
    nm = shutil.which("nm")
    if not nm:
        pytest.skip("no nm")
    capi.load()
    out = subprocess.run([nm, "-D", "--defined-only", str(build.LIB)], capture_output=True, text=True, check=True).stdout
    names = {line.split()[-1] for line in out.splitlines()}
    assert names == set(capi.declared_symbols())
