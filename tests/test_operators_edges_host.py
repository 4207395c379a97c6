"""The training-side operators at the edge of what their entry points allow, without a GPU: the kernels' own source on the CPU (tests/hipemu/run_kernels14.cpp)."""
import os
import shutil

import pytest

import test_hip_emulation as emulation

needs_clang = pytest.mark.skipif(not (os.path.isfile(emulation.CLANG) or shutil.which(emulation.CLANG)),
                                 reason="needs a clang++ with ext_vector_type / _Float16 / __bf16 (ROCm's)")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    return emulation._compile(str(tmp_path_factory.mktemp("edges")), "run_kernels14")


@needs_clang
def test_layer_norm_without_an_eps(kernels):
    """A thread without a position holds zeros; with eps = 0 its 1 / sqrt(0) stays out of the weight gradient."""
    emulation._run(kernels, ["eps 0 f32 (2, 8, 65)", "eps 0 f32 (1, 3, 65)", "eps 0 bf16"], "eps0")
