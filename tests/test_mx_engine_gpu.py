"""Microscaled weights where a model uses them: mixtures of all types."""

import pytest
import torch

from vllm_tgis_adapter_amd import ops

pytestmark = pytest.mark.gpu


def mixture(dtype: str, bits: int, top: int):
    from vllm_tgis_adapter_amd.engine.config import ModelConfig
    from vllm_tgis_adapter_amd.models.mixtral import MoEBlock

    torch.manual_seed(top)
    cfg = ModelConfig.from_model_arg("tiny-mixtral", dtype=dtype)
    cfg.num_experts, cfg.num_experts_per_tok = 8, top
    block = MoEBlock(cfg).cuda()
    for p in block.parameters():
        p.data.normal_(std=0.1)
    assert block.quantize_mx_(bits) == 2
    return block, cfg.hidden_size


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("tokens,top", [(1, 2), (37, 2), (150, 5)])
def test_mixture_block(tokens, top, dtype, bits):
    """Types without a router of their own: each token's experts, weighted."""
    block, hidden = mixture(dtype, bits, top)
    g = torch.Generator("cuda").manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(block.gate.dtype)
    got = block(x)
    weights, ids = ops.topk_softmax(torch.nn.functional.linear(x, block.gate), top)
    flat = ids.flatten()
    order = flat.argsort(stable=True)
    seg = torch.zeros(block.num_experts + 1, dtype=torch.int32, device="cuda")
    seg[1:] = torch.bincount(flat, minlength=block.num_experts).cumsum(0)
    xs = x[order // top]
    h = ops.moe_gemm_mx(xs, block.w13_q, block.w13_scale, seg, True, act_bits=bits)
    ye = torch.empty(tokens * top, hidden, dtype=x.dtype, device="cuda")
    ye[order] = ops.moe_gemm_mx(h, block.w2_q, block.w2_scale, seg, False, act_bits=bits)
    terms = ye.double().view(tokens, top, -1) * weights.to(x.dtype).double()[..., None]
    want, size = terms.sum(1), terms.abs().sum(1)
    # each term is rounded once and each sum of up to `top` of them once: half a step each, of
    # no more than the sum of the rounded terms' sizes
    info = torch.finfo(x.dtype)
    off = (1 + top) * info.eps / 2 * (1 + info.eps) * size + 2 * top * info.smallest_normal * info.eps
    assert ((got.double() - want).abs() <= off).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_a_mixture_repeats_itself(dtype):
    """Sums of a token's experts are taken in one order, whatever is done at the same time."""
    block, hidden = mixture(dtype, 6, 5)
    x = torch.randn(300, hidden, device="cuda").to(block.gate.dtype)
    first = block(x)
    for _ in range(20):
        assert torch.equal(block(x), first)
