"""Which layers microscaled weights leave alone, and that a user is told."""

from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

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
