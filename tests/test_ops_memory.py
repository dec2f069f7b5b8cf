"""The C entries of the paged-cache operators while memory runs out."""
import subprocess

import pytest


def run(binary, *arguments):
    result = subprocess.run([str(binary), *arguments], capture_output=True, text=True, timeout=120)
    assert result.returncode == 0, result.stderr
    assert "ops without memory: ok" in result.stdout


def test_no_exception_leaves_a_c_entry(built):
    run(built["test:ops_memory_test"])


@pytest.mark.gpu
def test_no_exception_leaves_a_c_entry_with_a_device(gpu, built):
    run(built["test:ops_memory_test"], "gpu")
