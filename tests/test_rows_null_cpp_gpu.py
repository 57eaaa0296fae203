"""Runs the C++ client that passes null pointers to HashTable::find_layer_norm
(tests/cpp/rows_null_test.cu)."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BINARY = os.path.join(ROOT, "tests", "cpp", "build", "rows_null_test")


def build():
    r = subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp"), "build/rows_null_test"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_null_parameters_compile(product_lib):
    build()
    assert os.path.exists(BINARY)


@pytest.mark.gpu
def test_null_parameters_are_ones_and_zeros(product_lib):
    if not os.path.exists(BINARY):
        build()
    r = subprocess.run([BINARY], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "PASS" in r.stdout
