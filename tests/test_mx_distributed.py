"""Microscaled weights over two ranks (gloo on the CPU): layers cut by rows and by inputs, a mixture
cut inside its experts and one with whole experts a rank, an engine."""

import pytest
import torch

import mx_oracle as oracle
from test_distributed import _run_spawn, _setup_dist
from test_mx_exact import exact_rows

HIDDEN, INTER, TOKENS, BITS = 128, 192, 7, 6


def _close(got, want, off) -> bool:
    return bool(((got.double() - want).abs() <= oracle.rounded_off(want, off, got.dtype)).all())


def _values(w) -> torch.Tensor:
    return oracle.quantize(w, 4)[2]


def _layers(rank, world):
    """Each rank's shard is rounded by itself: blocks are those of the whole matrix."""
    from vllm_tgis_adapter_amd.parallel.layers import (
        MergedColumnParallelLinear, RowParallelLinear, quantize_module_mx_,
    )

    g = torch.Generator().manual_seed(1)
    x = torch.randn(TOKENS, HIDDEN, generator=g)
    gate, up = (torch.randn(INTER, HIDDEN, generator=g) for _ in range(2))
    down = torch.randn(HIDDEN, INTER, generator=g)
    column = MergedColumnParallelLinear(HIDDEN, [INTER, INTER], dtype=torch.float32)
    column.load_full_weights([gate, up])
    row = RowParallelLinear(INTER, HIDDEN, dtype=torch.float32)
    row.load_full_weight(down)
    quantize_module_mx_(column, BITS)
    quantize_module_mx_(row, BITS)
    mine = slice(rank * INTER // world, (rank + 1) * INTER // world)
    h = column.gated(x)
    want, off = oracle.gated(x, torch.cat([_values(gate)[mine], _values(up)[mine]]), BITS)
    columns = _close(h, want, off)
    # the whole activation, as each rank has a part of it
    whole = torch.randn(TOKENS, INTER, generator=g)
    y = row(whole[:, mine].contiguous())
    want, magnitude = oracle.product(whole, _values(down), BITS)
    return {"columns": columns, "rows": _close(y, want, oracle.sums_off(magnitude, INTER + 1))}


def _mixture(rank, world, ep):
    """A token's experts one by one, of weights rounded as a whole."""
    from vllm_tgis_adapter_amd import ops
    from vllm_tgis_adapter_amd.engine.config import ModelConfig
    from vllm_tgis_adapter_amd.models.mixtral import MoEBlock

    cfg = ModelConfig.from_model_arg("tiny-mixtral", dtype="float32")
    cfg.expert_parallel = ep
    cfg.num_experts_per_tok = 3
    block = MoEBlock(cfg)
    assert block.ep == ep
    g = torch.Generator().manual_seed(7)
    experts, inter, hidden = cfg.num_experts, cfg.intermediate_size, cfg.hidden_size
    gate = torch.randn(experts, hidden, generator=g) * 0.2
    w13 = torch.randn(experts, 2 * inter, hidden, generator=g) * 0.2
    w2 = torch.randn(experts, hidden, inter, generator=g) * 0.2
    # (each rank has rows of its own, with whole experts; sums of the first product are exact in
    # any order, so that the second one's rows round to the same codes here and there)
    x = exact_rows(TOKENS, hidden, BITS, torch.Generator().manual_seed(rank if ep else 0), "cpu").float()
    block.gate.data.copy_(gate)
    if ep:
        own = slice(block.expert0, block.expert0 + block.experts_per_rank)
        block.w13.data.copy_(w13[own])
        block.w2.data.copy_(w2[own])
    else:
        part = inter // world
        mine = slice(rank * part, (rank + 1) * part)
        block.w13.data[:, :part].copy_(w13[:, :inter][:, mine])
        block.w13.data[:, part:].copy_(w13[:, inter:][:, mine])
        block.w2.data.copy_(w2[:, :, mine])
    assert block.quantize_mx_(BITS) == 2
    got = block(x)
    weights, ids = ops.topk_softmax(x @ gate.T, cfg.num_experts_per_tok)
    want, off = torch.zeros(TOKENS, hidden, dtype=torch.float64), 0
    for t in range(TOKENS):
        for j in range(cfg.num_experts_per_tok):
            e = int(ids[t, j])
            # (what the second product rounds: results of the first in 32 bits, whose blocks
            # lie inside a rank's part)
            h = ops.gated_mx(x[t:t + 1], *ops.quantize_mx(w13[e]), BITS)
            y, magnitude = oracle.product(h, _values(w2[e]), BITS)
            share = float(weights[t, j])
            want[t] += share * y[0]
            # its sums, one of two ranks, its weighting and the sums of a token's experts
            off = max(off, float(oracle.sums_off(magnitude, inter + 8).max()))
    return {"mixture": bool(((got.double() - want).abs() <= off).all())}


def _engine(rank, world):
    from vllm_tgis_adapter_amd.engine import EngineConfig, LLMEngine, ModelConfig
    from vllm_tgis_adapter_amd.engine.config import CacheConfig, SchedulerConfig
    from vllm_tgis_adapter_amd.engine.worker import Worker
    from test_mx import generate

    cfg = EngineConfig(
        model_config=ModelConfig.from_model_arg("tiny-llama", dtype="float32"),
        cache_config=CacheConfig(block_size=16, num_gpu_blocks=128),
        scheduler_config=SchedulerConfig(max_num_seqs=4, max_num_batched_tokens=128),
        device="cpu", tensor_parallel_size=world, load_synthetic_weights=True,
        quantization="mxfp4")
    if rank:
        worker = Worker(cfg)
        worker.init_kv_cache()
        worker.worker_loop()
        return {}
    engine = LLMEngine(cfg)
    tokens = generate(engine)
    engine.worker.stop_workers()
    rounded = [m for m in engine.worker.model.modules() if getattr(m, "mx_act_bits", None) == 6]
    return {"tokens": [len(t) for t in tokens] == [8, 8], "layers": len(rounded) == 8}


WORK = {"layers": _layers, "mixture": lambda r, w: _mixture(r, w, False),
        "whole experts": lambda r, w: _mixture(r, w, True), "engine": _engine}


def _worker(what, rank, world, port, q):
    try:
        _setup_dist(rank, world, port)
        q.put((rank, WORK[what](rank, world)))
    except Exception:
        import traceback

        q.put((rank, "ERROR " + traceback.format_exc()))
    finally:
        import torch.distributed as dist

        if dist.is_initialized():
            dist.destroy_process_group()


@pytest.mark.parametrize("what", list(WORK))
def test_two_ranks(what):
    from functools import partial

    for rank, payload in _run_spawn(partial(_worker, what), 2).items():
        assert all(payload.values()), (rank, payload)
