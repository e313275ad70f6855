"""The operators of expert layers and orthogonalize on their second host path: Python + ctypes in place of the C++ registration (GNK_NO_TORCH_SHIM=1, or where
it is not built).  Their checks run once more in a child process on that path; every registered operator is in this selection or in that of
tests/test_gpu_host_paths.py."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

from gn_kernels import _cabi

ROOT = Path(__file__).resolve().parent.parent

SELECTION = {
    "grouped_scaled_mm": ["tests/test_gpu_grouped.py::test_rows_feature_sizes", "tests/test_gpu_grouped.py::test_fp8_formats_mix", "tests/test_gpu_grouped.py::test_refusals_on_device"],
    "grouped_scaled_mm_depth": ["tests/test_gpu_grouped.py::test_depth_feature_sizes", "tests/test_gpu_grouped.py::test_depth_in_parts_output_types",
                                "tests/test_gpu_grouped_long_sums.py::test_weight_gradient_of_constant_columns"],
    "quantize_int8_grouped": ["tests/test_gpu_grouped.py::test_quantize_grouped_long", "tests/test_gpu_grouped.py::test_quantize_grouped_strides",
                              "tests/test_gpu_grouped.py::test_quantize_grouped_stochastic"],
    "grouped_linear_int8": ["tests/test_gpu_grouped_linear.py::test_against_the_formula"],
    "grouped_linear_int8_backward": ["tests/test_gpu_grouped_linear.py::test_many_rows_of_small_experts", "tests/test_gpu_grouped_linear.py::test_forward_and_backward_in_a_graph"],
    "orthogonalize": ["tests/test_gpu_ortho.py::test_types", "tests/test_gpu_ortho.py::test_strides", "tests/test_gpu_ortho.py::test_refusals"],
}
DENSE = {"int8_mm", "scaled_mm", "scaled_mm_t", "tile_scaled_mm", "quantize_int8", "quantize_int8_rowwise_colmax", "quantize_int8_colwise_given"}


def test_every_registered_operator_is_selected():
    assert set(_cabi._SHIM_OPS) == DENSE | set(SELECTION)


@pytest.mark.gpu
def test_python_ctypes_host_path():
    env = dict(os.environ, GNK_NO_TORCH_SHIM="1", GNK_EXPECT_NO_SHIM="1")
    chosen = [t for tests in SELECTION.values() for t in tests]
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "gpu", "-p", "no:cacheprovider", "--timeout", "60", "--timeout-method", "thread",
                        *chosen, "tests/test_gpu_host_paths.py::test_child_sees_no_shim"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=100)
    tail = (r.stdout + r.stderr)[-3000:]
    assert r.returncode == 0, tail
    assert " passed" in r.stdout and "skipped" not in r.stdout, tail
