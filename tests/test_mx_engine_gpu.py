"""Microscaled weights where a model uses them: each product of an engine's steps against 64 bits,
mixtures of all types, layers with adapters."""

import pytest
import torch

import mx_oracle as oracle
import test_lora_layers_gpu as adapters_of
from test_mx import generate
from test_mx_exact import widened
from vllm_tgis_adapter_amd import ops

pytestmark = pytest.mark.gpu


def eager_engine(model: str, method, dtype: str):
    from vllm_tgis_adapter_amd.engine import LLMEngine
    from vllm_tgis_adapter_amd.engine.config import (
        CacheConfig, EngineConfig, ModelConfig, SchedulerConfig,
    )

    return LLMEngine(EngineConfig(
        model_config=ModelConfig.from_model_arg(model, dtype=dtype),
        cache_config=CacheConfig(block_size=16),
        scheduler_config=SchedulerConfig(max_num_seqs=4, max_num_batched_tokens=512),
        device="cuda", quantization=method, seed=0, enforce_eager=True))


def right(got, x, wq, scales, gated: bool, bits: int) -> bool:
    """One product's results, its rows as they came in."""
    values = widened(wq.cpu(), scales.cpu())
    if gated:
        want, off = oracle.gated(x, values, bits)
    else:
        want, magnitude = oracle.product(x, values, bits)
        off = oracle.sums_off(magnitude, x.shape[1])
    off = oracle.rounded_off(want, off, got.dtype)
    return bool(((got.cpu().double() - want).abs() <= off).all())


@pytest.mark.parametrize("dtype,method", [
    ("bfloat16", "mxfp4"), ("bfloat16", "mxfp4a4"), ("float16", "mxfp4"), ("float32", "mxfp4")])
@pytest.mark.parametrize("model", ["tiny-llama", "tiny-mixtral"])
def test_products_of_an_engine(model, dtype, method, monkeypatch):
    """One sequence, then two: every step goes through these products and no others, with the
    model's weights rounded as the format says."""
    bits = 4 if method == "mxfp4a4" else 6
    layers = 2
    plain, eng = (eager_engine(model, m, dtype) for m in (None, method))
    stored = dict(eng.worker.model.named_buffers())
    rounded = 0
    for name, w in plain.worker.model.named_parameters():
        name = name + "_q" if name.endswith((".w13", ".w2")) else name.replace(".weight", ".weight_q")
        if name not in stored:
            continue
        codes, scales, _ = oracle.quantize(w.reshape(-1, w.shape[-1]), 4)
        assert torch.equal(stored[name].cpu().view(-1, w.shape[-1] // 2), oracle.pack(codes, 4))
        assert torch.equal(stored[name[:-1] + "scale"].cpu().view(-1, w.shape[-1] // 32), scales)
        rounded += 1
    assert rounded == 4 * layers

    calls = {"linear": 0, "gated": 0, "experts": 0}
    linear, gated, experts = ops.linear_mx, ops.gated_mx, ops.moe_gemm_mx

    def count_linear(x, wq, scales, bias=None, act_bits=4):
        y = linear(x, wq, scales, bias, act_bits)
        assert bias is None and act_bits == bits and right(y, x, wq, scales, False, bits)
        calls["linear"] += 1
        return y

    def count_gated(x, wq, scales, act_bits=4):
        y = gated(x, wq, scales, act_bits)
        assert act_bits == bits and right(y, x, wq, scales, True, bits)
        calls["gated"] += 1
        return y

    def count_experts(x, wq, scales, seg_off, gate, rows=None, act_bits=4):
        y = experts(x, wq, scales, seg_off, gate, rows, act_bits)
        off = seg_off.tolist()
        xs = x if rows is None else x[rows.long()]
        assert act_bits == bits and off[-1] == xs.shape[0]
        for e, (a, b) in enumerate(zip(off, off[1:])):
            assert a == b or right(y[a:b], xs[a:b], wq[e], scales[e], gate, bits)
        calls["experts"] += 1
        return y

    monkeypatch.setattr(ops, "linear_mx", count_linear)
    monkeypatch.setattr(ops, "gated_mx", count_gated)
    monkeypatch.setattr(ops, "moe_gemm_mx", count_experts)
    steps = []
    forward = eng.worker.model.forward
    monkeypatch.setattr(eng.worker.model, "forward",
                        lambda *a, **k: (steps.append(1), forward(*a, **k))[1])
    for requests in (1, 2):
        assert all(len(t) == 6 for t in generate(eng, requests, 6))
    mixture = model == "tiny-mixtral"
    n = len(steps) * layers
    assert n >= 12 * layers
    assert calls == ({"linear": 2 * n, "gated": 0, "experts": 2 * n} if mixture
                     else {"linear": 3 * n, "gated": n, "experts": 0})


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


@pytest.mark.parametrize("kind", ["qkv", "o", "gate"])
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("tokens", [1, 17, 65])
def test_layers_with_adapters(kind, bits, tokens):
    """A layer's rows are rounded for its weight and not for the adapters'."""
    from vllm_tgis_adapter_amd.engine import lora
    from vllm_tgis_adapter_amd.parallel import layers

    g = torch.Generator("cuda").manual_seed(tokens + bits)
    adapters = adapters_of._adapters(g, 16)
    mod, _, projs = adapters_of._layer(g, kind, 16)
    layers.quantize_module_mx_(mod, bits)
    weight = widened(mod.weight_q, mod.weight_scale)
    x = adapters_of._normal(g, tokens, adapters_of.HIDDEN)
    ids = torch.tensor([0, 3, 5, 8, 9], device="cuda")[
        torch.randint(5, (tokens,), generator=g, device="cuda")].int()
    lora._STACK_CACHE.clear()
    lora._RECENT_SETS.clear()
    lora.set_context(ids, adapters)
    try:
        got = mod.gated(x, lora=(0, projs)) if kind == "gate" else mod(x, lora=(0, projs))
    finally:
        lora.clear_context()
        lora._STACK_CACHE.clear()
        lora._RECENT_SETS.clear()
    deltas, off = adapters_of._want(x, torch.zeros_like(weight), projs, adapters, ids)
    q = oracle.quantize(x, bits)[2].cuda()
    base = q @ weight.T
    # the base's sums, its rounding ahead of the deltas, the deltas' own (their hidden values are
    # rounded to bf16: half a step of each of 16, at most)
    off = off + oracle.sums_off(q.abs() @ weight.abs().T, x.shape[1]) + 2 ** -8 * base.abs()
    for number, a in adapters.items():
        mine = ids == number
        for name, lo, hi in projs:
            if (0, name) in a.weights:
                wa, wb = (t.double() for t in a.weights[(0, name)])
                inner = (x.double()[mine] @ wa.T).abs()
                off[mine, lo:hi] += 2 ** -7 * a.scaling * inner @ wb.abs().T
    want = base + deltas
    if kind == "gate":
        off = off + 2 ** -8 * want.abs()
        (gate, up), (og, ou) = want.chunk(2, 1), off.chunk(2, 1)
        want = torch.nn.functional.silu(gate) * up
        off = 1.1 * og * (up.abs() + ou) + ou * gate.abs() + 1e-5 * want.abs()
    err = (got.double() - want).abs()
    assert (err <= 2 ** -8 * (want.abs() + off) + off + 1e-7).all()
