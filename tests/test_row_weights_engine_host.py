"""What a decoder stack accepts as adapters, checked on the host: the engine's own method on an engine without kernels."""
from types import SimpleNamespace

import pytest
import torch

from vox_serve_b200 import ops
from vox_serve_b200._lib import VoxB200Error
from vox_serve_b200.engine import LlamaAdapters, LlamaDims, LlamaEngine

DIMS = LlamaDims(128, 2, 2, 1, 64, 256, 100)


def _engine(dims=DIMS, rows=16):
    eng = object.__new__(LlamaEngine)
    eng.dims, eng.max_rows, eng.device, eng.adapters = dims, rows, torch.device("cpu"), None
    eng.split_qkv = eng.split_o = eng.split_down = 2
    eng.qkv_w = (dims.num_attention_heads + 2 * dims.num_key_value_heads) * dims.head_dim
    eng.w = SimpleNamespace(layers=[{"gu": SimpleNamespace(N=2 * dims.intermediate_size)}])
    eng.hidden = torch.zeros(rows, dims.hidden_size)
    return eng


def test_adapters_are_set_once():
    """captured steps hold the addresses of the banks and of the planes: neither changes afterwards"""
    eng, one = _engine(), LlamaAdapters(DIMS, 2, 8, device="cpu")
    eng.set_adapters(one)
    held = eng.adapter_planes.data_ptr(), eng.adapter_gu.data_ptr()
    eng.set_adapters(one)
    assert (eng.adapter_planes.data_ptr(), eng.adapter_gu.data_ptr()) == held
    with pytest.raises(VoxB200Error, match="already"):
        eng.set_adapters(LlamaAdapters(DIMS, 2, 8, device="cpu"))
    assert eng.adapters is one and (eng.adapter_planes.data_ptr(), eng.adapter_gu.data_ptr()) == held


@pytest.mark.parametrize("dims", [LlamaDims(128, 2, 1, 2, 64, 256, 100), LlamaDims(128, 2, 4, 2, 32, 256, 100), LlamaDims(128, 2, 4, 1, 64, 256, 100),
                                  LlamaDims(128, 3, 2, 1, 64, 256, 100), LlamaDims(64, 2, 2, 1, 64, 256, 100), LlamaDims(128, 2, 2, 1, 64, 512, 100)])
def test_adapters_of_another_model(dims):
    """another head count or key head count as well, with q | k | v as wide as before or not.  (4 + 2 2 heads of 32 give the same matrices as 2 + 2 1 heads of 64: those go.)"""
    eng, other = _engine(), LlamaAdapters(dims, 2, 8, device="cpu")
    if LlamaAdapters.shapes(dims) == LlamaAdapters.shapes(DIMS) and dims.num_hidden_layers == DIMS.num_hidden_layers:
        eng.set_adapters(other)
        return
    with pytest.raises(VoxB200Error, match="another model"):
        eng.set_adapters(other)
    assert eng.adapters is None


def test_adapters_on_another_device():
    eng = _engine()
    eng.hidden = torch.zeros(16, 128, device="meta")
    with pytest.raises(VoxB200Error, match="cpu"):
        eng.set_adapters(LlamaAdapters(DIMS, 2, 8, device="cpu"))


def test_plans_that_are_not_the_step_s():
    """refused before the step writes anything"""
    eng = _engine()
    eng.set_adapters(LlamaAdapters(DIMS, 2, 8, device="cpu"))
    for slots, rows in ((3, 4), (2, 3), (2, 5)):
        plan = ops.LoraPlan(8, slots, device="cpu")
        plan.n_rows = rows
        with pytest.raises(VoxB200Error, match="plan of adapters"):
            eng.forward(None, None, 4, adapters=plan)
