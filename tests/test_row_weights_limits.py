"""Sizes and addresses that the operators whose weights a row brings with it would take wrongly: refused on the host, by the Python classes and by the C entry points."""
import ctypes

import pytest
import torch

from vox_serve_b200 import _lib, ops
from vox_serve_b200._lib import VoxB200Error

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32


@pytest.mark.parametrize("rows", [2 ** 21 + 1, 2 ** 31, 2 ** 32 + 1, 2 ** 33 + 64])
def test_plans_of_too_many_rows(rows):
    """2^32 + 1 rows are 1 to a C int: a table of one row's size, which a step of a thousand would have written past"""
    with pytest.raises(VoxB200Error, match="rows"):
        ops.LoraPlan(rows, 4, device="cpu")
    assert ops.LoraPlan(2 ** 10, 4, device="cpu").tiles.numel() * 4 == _lib.load().vb_lora_plan_bytes(2 ** 10, 4)


@pytest.mark.parametrize("args", [(1, 2 ** 24 + 8, (8,), 1), (1, 2 ** 32 + 8, (8,), 1), (1, 8, (2 ** 24 + 8,), 1), (1, 8, (8, 2 ** 32 + 8), 1)])
def test_banks_of_too_large_matrices(args):
    with pytest.raises(VoxB200Error, match="2\\^24"):
        ops.LoraBank(*args, device="meta")


def _packed(n, k, rows):
    return ops.PackedWeight(torch.zeros(8, dtype=torch.uint8), n, k, rows)


@pytest.mark.parametrize("width,ff,shared", [(2 ** 32 + 8, 64, 0), (2 ** 24 + 8, 64, 0), (72, 2 ** 17 + 64, 0), (72, 64, 2 ** 17 + 64), (72, 2 ** 32 + 64, 0)])
def test_experts_of_too_large_matrices(width, ff, shared):
    n = 4 * ff + shared
    with pytest.raises(VoxB200Error, match="at most"):
        ops.MoeWeights(_packed(2 * n, width, 128), _packed(width, n, 128), 4, width, ff, shared)


def _room():
    buf = torch.zeros(1 << 16, dtype=torch.uint8)
    return buf, (buf.data_ptr() + 255) // 256 * 256


def _refused(rc, words):
    assert rc != 0 and words in _lib.load().vb_last_error().decode(), _lib.load().vb_last_error()


def test_unaligned_banks_and_plans():
    buf, at = _room()
    lib = _lib.load()
    widths = (ctypes.c_int32 * 4)(32)
    good = [at, at, at, 2, 16, 64, 1]
    for i, by in ((0, 8), (1, 2), (2, 2)):
        bad = list(good)
        bad[i] += by
        bank = _lib.LoraBankStruct(*bad, widths)
        assert lib.vb_lora_workspace_bytes(ctypes.addressof(bank), 100) == 0
        _refused(lib.vb_lora(at, 32, None, 32, 1, at, 64, ctypes.addressof(bank), at, 4, at, 1 << 12, None), "bank must be 16-byte aligned")
    bank = _lib.LoraBankStruct(*good, widths)
    _refused(lib.vb_lora(at, 32, None, 32, 1, at, 64, ctypes.addressof(bank), at + 4, 4, at, 1 << 12, None), "plan must be 16-byte aligned")
    _refused(lib.vb_lora_plan(at, at + 2, 4, 2, None), "ids 4-byte")
    bank = _lib.LoraBankStruct(at, at, at, 2, 16, 2 ** 24 + 8, 1, widths)
    _refused(lib.vb_lora(at, 32, None, 32, 1, at, 2 ** 25, ctypes.addressof(bank), at, 4, at, 1 << 12, None), "a multiple of 8")


@pytest.mark.parametrize("which", ["up", "down", "y", "ids", "bias", "table"])
def test_unaligned_experts(which):
    buf, at = _room()
    lib = _lib.load()
    by = {k: 0 for k in ("up", "down", "y", "ids", "bias", "table")}
    by[which] = 8 if which in ("up", "down") else 2
    weights = _lib.MoeWeightsStruct(at + by["up"], at + by["down"], 64, 4, 64, 0, 128, 0, 0.0, 1.0)
    router = _lib.MoeRouterStruct(at, at + by["bias"], None, at + by["table"], 3 if which in ("ids", "table") else 0, 2, 0, 0, 16)
    _refused(lib.vb_moe_layer(at + by["y"], 64, at, 64, ctypes.addressof(weights), ctypes.addressof(router), at + by["ids"], 2, at, 1 << 15, None), "aligned")


def test_experts_on_two_devices():
    """a call compares its rows with one of them"""
    up, down = _packed(2 * 4 * 64, 72, 128), _packed(72, 4 * 64, 128)
    ops.MoeWeights(up, down, 4, 72, 64)
    with pytest.raises(VoxB200Error, match="meta"):
        ops.MoeWeights(up, ops.PackedWeight(torch.zeros(8, dtype=torch.uint8, device="meta"), 72, 4 * 64, 128), 4, 72, 64)
