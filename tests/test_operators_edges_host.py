"""The training-side operators at the edge of what their entry points allow, without a GPU: the host's side, and the kernels'
own source on the CPU (tests/hipemu/run_kernels14.cpp)."""
import os
import shutil
import subprocess
import threading

import pytest
import torch

import casmvsnet_pl_amd as M
from casmvsnet_pl_amd import _lib, training

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


def test_a_forward_without_a_graph_leaves_the_plan_of_another_thread_alone():
    """A layer-norm model's eval forward packs on its own; the training step of another thread keeps its plan meanwhile, and what it releases stays released."""
    def elsewhere(call):
        out = []
        thread = threading.Thread(target=lambda: out.append(call()))
        thread.start()
        thread.join()
        return out[0]
    plan = training.PackPlan()
    seen = []

    def forward(m, x):
        seen.append(training._active_plan())
        seen.append(training.without_graph(lambda m, x: training._active_plan(), m, x))   # one inside another
        seen.append(training._active_plan())
        seen.append(elsewhere(training._active_plan))
        elsewhere(training.release_plan)
        assert not torch.is_grad_enabled()
        return x
    try:
        training.set_active_plan(plan)
        assert training.without_graph(forward, None, 3) == 3
        assert seen == [None, None, None, plan] and training._active_plan() is None
        training.set_active_plan(plan)
        with pytest.raises(ZeroDivisionError):
            training.without_graph(lambda m, x: 1 // 0, None, None)
        assert training._active_plan() is plan
    finally:
        training.release_plan()


@pytest.mark.parametrize("first", [0, 1])
def test_a_model_with_both_kinds_of_norm_is_refused_in_eval_mode(first):
    """Layer by layer an ABN would take batch statistics (and change its running ones); folded, a layer norm has nothing to fold."""
    kinds = (M.LayerNormAct, M.ABN) if first == 0 else (M.ABN, M.LayerNormAct)
    for net in (M.FeatureNet(lambda c: kinds[c != 8](c)), M.CostRegNet(8, lambda c: kinds[c != 8](c))):
        with pytest.raises(RuntimeError, match="both|no running statistics"):
            assert net.foldable
            net.packed_layers("cpu")
    for norm in (M.ABN, M.InPlaceABN, M.LayerNormAct):
        assert M.FeatureNet(norm).foldable == M.CostRegNet(8, norm).foldable == (norm is not M.LayerNormAct)


@needs_clang
def test_abn8_far_from_zero(kernels):
    """Channels whose mean is many times their spread, whose first element is far from the others, constant ones."""
    emulation._run(kernels, ["abn8 shifted (2, 3, 70) at -3e+06", "abn8 first apart", "abn8 constant"], "far")


@needs_clang
def test_depth_cross_entropy_reads_nothing_of_masked_pixels(kernels):
    """Whatever the number of pieces that a pixel's axis is cut into; and a piece without a hypothesis (or a finite distance) changes no class."""
    emulation._run(kernels, ["depth_ce masked (1, 192, 20)", "depth_ce pieces (65, 40) to 3e+38"], "masked")


def test_a_library_of_older_sources_is_named_as_such(tmp_path, monkeypatch):
    """Same ABI version, but without an entry point that was added since."""
    source, path = tmp_path / "old.c", tmp_path / "libold.so"
    source.write_text("int casmvs_abi_version(void) { return %d; }\n" % _lib.ABI_VERSION)
    subprocess.run(["gcc", "-shared", "-fPIC", str(source), "-o", str(path)], check=True)
    monkeypatch.setattr(_lib, "LIB_PATH", str(path))
    monkeypatch.setattr(_lib, "_lib", None)
    with pytest.raises(_lib.CasMVSLibraryError, match="older sources"):
        _lib.load()
