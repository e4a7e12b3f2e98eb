"""Which layers microscaled weights leave alone, and that a user is told; calls with nothing in them."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

from vllm_tgis_adapter_amd import ops
from vllm_tgis_adapter_amd.engine.worker import Worker
from vllm_tgis_adapter_amd.parallel.layers import ColumnParallelLinear, RowParallelLinear


@pytest.mark.parametrize("method,bits", [("mxfp4", 6), ("mxfp4a4", 4)])
def test_layers_of_no_whole_blocks_are_named(method, bits, capsys):
    model = nn.ModuleDict({"fits": ColumnParallelLinear(64, 8, dtype=torch.float32),
                           "ragged": RowParallelLinear(48, 8, dtype=torch.float32)})
    Worker._quantize_model(SimpleNamespace(
        model=model, device="cpu", _quantize_model_mx=lambda m: Worker._quantize_model_mx(
            SimpleNamespace(model=model, device="cpu"), m)), method)
    assert model["fits"].mx_act_bits == bits and model["fits"].weight_q.shape == (8, 32)
    assert model["ragged"].mx_act_bits is None and model["ragged"].weight.shape == (8, 48)
    said = capsys.readouterr().out
    assert "quantized 1 " in said and "left 1 " in said and "ragged" in said
    assert model["ragged"](torch.ones(2, 48)).shape == (2, 8)


def test_nothing_is_said_where_all_are_rounded(capsys):
    model = nn.ModuleDict({"fits": ColumnParallelLinear(64, 8, dtype=torch.float32)})
    Worker._quantize_model_mx(SimpleNamespace(model=model, device="cpu"), "mxfp4")
    assert "left" not in capsys.readouterr().out


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_single_values_and_rows_without_blocks(device):
    """The same answers on the CPU and on the GPU."""
    one = torch.ones((), device=device)
    byte = torch.ones((), dtype=torch.uint8, device=device)
    wq, scales = ops.quantize_mx(torch.ones(6, 64, device=device))
    seg = torch.tensor([0, 1, 1], dtype=torch.int32, device=device)
    for call in (lambda: ops.quantize_mx(one), lambda: ops.dequantize_mx(wq, byte),
                 lambda: ops.linear_mx(one, wq, scales), lambda: ops.gated_mx(one, wq, scales),
                 lambda: ops.moe_gemm_mx(one, wq.view(2, 3, -1), scales.view(2, 3, -1), seg, False)):
        with pytest.raises(ValueError):
            call()
    for bits in (4, 6):
        y = ops.dequantize_mx(wq[:, :0], scales[:, :0], bits, torch.float16)
        assert y.shape == (6, 0) and y.dtype == torch.float16
