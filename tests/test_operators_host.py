"""The training-side operators (layer norm, 8-bit checkpoints, depth cross entropy) without a GPU: what their Python entry points and the C ABI refuse, the module's
contract, and the kernels' own source on the CPU (tests/hipemu/run_kernels13.cpp against float64)."""
import ctypes
import os
import shutil

import pytest
import torch

import casmvsnet_pl_amd as M
from casmvsnet_pl_amd import _lib, autograd, ops, training
from casmvsnet_pl_amd.build import build_library

import test_hip_emulation as emulation


@pytest.fixture(scope="module", autouse=True)
def built():
    build_library()


def _p(i=8):
    return ctypes.c_void_p(i)


def test_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 8, 4)
    for call in (lambda: ops.layer_norm(x), lambda: autograd.layer_norm(x), lambda: ops.pack8(x), lambda: M.LayerNormAct(8)(x),
                 lambda: autograd.depth_cross_entropy(torch.zeros(1, 2, 3, 3), torch.zeros(1, 2), torch.zeros(1, 3, 3))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError, match="Packed8"):
        ops.unpack8(x)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.unpack8(ops.Packed8(torch.zeros(2, 1, 32, dtype=torch.uint8), torch.zeros(2, 1, dtype=torch.uint8), (2, 4), torch.float32))


def test_checkpoint_and_loss_names_are_checked():
    with pytest.raises(ValueError, match="checkpoint='4bit'"):
        training.abn_train(M.ABN(8), torch.zeros(1, 8, 4), checkpoint="4bit")
    with pytest.raises(ValueError, match="loss='l2'"):
        training.train_steps(None, [], None, loss="l2")
    with pytest.raises(ValueError, match="return_cost"):
        training.cross_entropy_loss({}, {}, {f"level_{l}": None for l in range(3)})


@pytest.mark.parametrize("shape,rows_n", [((), (1, 1)), ((7,), (1, 7)), ((3, 5), (3, 5)), ((2, 3, 4), (6, 4)), ((2, 3, 4, 5, 6), (6, 120)), ((2, 0, 4), (0, 4))])
def test_planes_of_the_8_bit_format(shape, rows_n):
    assert ops._planes(shape) == rows_n


def test_c_abi_refuses_bad_arguments():
    lib = _lib.load()

    def refused(rc, text):
        assert rc == -1 and text in lib.casmvs_last_error(), (rc, lib.casmvs_last_error())

    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 3, 1, 8, 4, 1e-5, 1.0, None), b"dtype 3")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1, 0, 4, 1e-5, 1.0, None), b"C=0")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1, 65536, 4, 1e-5, 1.0, None), b"C=65536")
    refused(lib.casmvs_layer_norm_forward(None, None, None, _p(), 0, 1, 8, 4, 1e-5, 1.0, None), b"null pointer")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1 << 31, 8, 1, 1e-5, 1.0, None), b"positions of 8 channels")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1 << 24, 9000, 1, 1e-5, 1.0, None), b"positions of 9000 channels")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1 << 15, 600, 1 << 15, 1e-5, 1.0, None), b"positions of 600 channels")
    refused(lib.casmvs_layer_norm_forward(_p(), None, None, _p(), 0, 1 << 62, 8, 16, 1e-5, 1.0, None), b"positions")
    refused(lib.casmvs_layer_norm_backward(_p(), _p(), None, None, _p(), _p(), None, _p(), 0, 1, 8, 4, 1e-5, 1.0, None), b"go together")
    refused(lib.casmvs_layer_norm_backward(_p(), _p(), None, None, _p(), None, None, None, 0, 1, 8, 4, 1e-5, 1.0, None), b"workspace")
    assert lib.casmvs_layer_norm_forward(None, None, None, None, 0, 0, 8, 4, 1e-5, 1.0, None) == 0   # nothing to do
    assert lib.casmvs_layer_norm_backward_workspace_bytes(9, 1, 8, 4) == 0
    refused(lib.casmvs_pack8(_p(), 7, 1, 32, _p(), _p(), None), b"dtype 7")
    refused(lib.casmvs_pack8(None, 0, 1, 32, _p(), _p(), None), b"null pointer")
    refused(lib.casmvs_pack8(_p(), 0, 1, 32, _p(6), _p(), None), b"alignment")
    refused(lib.casmvs_pack8(_p(), 0, 1 << 40, 1 << 40, _p(), _p(), None), b"rows")
    refused(lib.casmvs_unpack8(_p(), _p(), _p(), None, 8, 1.0, _p(), 0, 8, 32, None), b"go together")
    refused(lib.casmvs_unpack8(_p(), _p(), _p(), _p(), 0, 1.0, _p(), 0, 8, 32, None), b"go together")
    assert lib.casmvs_pack8(None, 0, 0, 32, None, None, None) == 0
    args = [_p(), _p(), _p(), -1.0, 1e-5, 0.1, None, None] + [_p()] * 6
    refused(lib.casmvs_abn8_forward_f32(*args, 0, 8, 32, 0.01, None), b"N=0")
    refused(lib.casmvs_abn8_forward_f32(*args, 1 << 20, 8, 32, 0.01, None), b"planes")
    refused(lib.casmvs_abn8_forward_f32(*args, 1, 8, 1 << 35, 0.01, None), b"planes")
    refused(lib.casmvs_abn8_forward_f32(*args, 1, 8, 1 << 50, 0.01, None), b"planes")
    refused(lib.casmvs_abn8_forward_f32(*(args[:6] + [_p()] + args[7:]), 1, 8, 32, 0.01, None), b"go together")
    refused(lib.casmvs_abn8_forward_f32(*(args[:13] + [_p(12)]), 1, 8, 32, 0.01, None), b"words")
    refused(lib.casmvs_abn8_backward_f32(_p(), _p(6), _p(), _p(), _p(), -1.0, _p(), _p(), _p(), _p(), _p(), 1, 8, 32, 0.01, None), b"words")
    refused(lib.casmvs_abn8_backward_f32(_p(), _p(), _p(), _p(), _p(), -1.0, _p(), None, _p(), _p(), _p(), 1, 8, 32, 0.01, None), b"null pointer")
    assert lib.casmvs_abn8_workspace_bytes(0, 8, 32) == 0 and lib.casmvs_abn8_workspace_bytes(1, 8, 32) == 128
    refused(lib.casmvs_depth_ce_forward(_p(), _p(), _p(), None, _p(), _p(), _p(), _p(), _p(), 0, 1, 0, 16, 1, None), b"D=0")
    refused(lib.casmvs_depth_ce_forward(_p(), _p(), _p(), None, _p(), _p(), _p(), _p(), _p(), 0, 2, 4, 1 << 30, 1, None), b"2^31")
    refused(lib.casmvs_depth_ce_forward(_p(), None, _p(), None, _p(), _p(), _p(), _p(), _p(), 0, 1, 4, 16, 1, None), b"null pointer")
    refused(lib.casmvs_depth_ce_forward(_p(), _p(), _p(), None, _p(), _p(), _p(), None, _p(), 0, 1, 4, 16, 1, None), b"null pointer")
    refused(lib.casmvs_depth_ce_backward(_p(), _p(), _p(), _p(), None, _p(), 0, 1, 4, 16, None), b"null pointer")
    refused(lib.casmvs_depth_ce_forward(_p(), _p(), _p(), None, _p(12), _p(), _p(), _p(), _p(), 0, 1, 4, 16, 1, None), b"8-byte")
    refused(lib.casmvs_depth_ce_forward(_p(), _p(), _p(), None, _p(), _p(), _p(), _p(), _p(12), 0, 1, 4, 16, 1, None), b"8-byte")
    refused(lib.casmvs_depth_ce_backward(_p(), _p(12), _p(), _p(), _p(), _p(), 0, 1, 4, 16, None), b"8-byte")
    assert lib.casmvs_depth_ce_workspace_bytes(0, 4, 16) == 0


def test_layer_norm_module_is_a_norm_act():
    model = M.CascadeMVSNet(norm_act=M.LayerNormAct)
    assert not model.feature.foldable and not model.cost_reg_0.foldable and M.CascadeMVSNet(norm_act=M.ABN).feature.foldable
    keys = set(model.state_dict())
    assert not [k for k in keys if "running" in k] and "feature.conv0.0.bn.weight" in keys and "cost_reg_2.conv11.1.bias" in keys
    assert keys == {k for k in M.CascadeMVSNet(norm_act=M.ABN).state_dict() if "running" not in k}
    assert M.LayerNormAct(4).leaky_slope() == 0.01 and M.LayerNormAct(4, activation="relu").leaky_slope() == 0.0
    assert M.LayerNormAct(4, activation="identity").leaky_slope() == 1.0 and M.LayerNormAct(4, affine=False).weight is None
    with pytest.raises(RuntimeError, match="elu"):
        M.LayerNormAct(4, activation="elu").leaky_slope()
    assert model.checkpoint_mode == "f32" and model.return_cost is False


@pytest.mark.skipif(not (os.path.isfile(emulation.CLANG) or shutil.which(emulation.CLANG)), reason="needs a clang++ with ext_vector_type / _Float16 / __bf16 (ROCm's)")
def test_operator_kernels_run_on_the_cpu(tmp_path):
    exe = emulation._compile(str(tmp_path), "run_kernels13")
    emulation._run(exe, ["layer_norm f32", "layer_norm bf16", "layer_norm f16", "pack8 f32", "abn8", "depth_ce f32", "depth_ce bf16"])
