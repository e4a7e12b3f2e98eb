"""Microscaled products captured and replayed whose launches share scratch memory: K cut in parts
that a second launch adds up, codes of x from a launch ahead, the largest tiles."""

import pytest
import torch

import mx_oracle as oracle
from vllm_tgis_adapter_amd import ops

pytestmark = pytest.mark.gpu

# rows of a tile, columns, K cut, rows, outputs, inputs, experts, bits, gated, type
FORMS = [
    (64, 128, True, 48, 502, 8192, 0, 6, False, torch.float16),
    (64, 128, True, 130, 500, 14336, 3, 4, False, torch.bfloat16),
    (64, 224, False, 61, 24601, 2816, 0, 6, True, torch.bfloat16),
    (128, 128, True, 512, 4096, 14336, 0, 6, False, torch.bfloat16),
    (128, 128, True, 200, 502, 14336, 3, 4, True, torch.float32),
    (128, 256, True, 66, 8201, 14336, 0, 6, False, torch.float32),
    (128, 256, False, 260, 12001, 1056, 0, 6, False, torch.float16),
    (256, 256, False, 1030, 4096, 288, 0, 4, True, torch.float16),
    (256, 256, True, 2060, 500, 28672, 2, 6, True, torch.bfloat16),
]


def captured(call):
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    return graph, y


@pytest.mark.parametrize("bm,bn,cut,rows,n,k,experts,bits,gated,dtype", FORMS)
def test_replays_are_the_eager_results(bm, bn, cut, rows, n, k, experts, bits, gated, dtype):
    """Rows, a bias and segments change between replays; a second graph of the same weights is
    replayed beside the first, on a stream of its own."""
    plan = ops._C.mx_plan(rows, n, k, experts, bits, gated)
    assert plan[2:4] == (bm, bn) and (plan[4] > 1) == cut
    g = torch.Generator("cuda").manual_seed(rows)
    lead = (*((experts,) if experts else ()), n * (2 if gated else 1))
    codes = torch.randint(0, 256, (*lead, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(118, 121, (*lead, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    bias = torch.zeros(n, device="cuda", dtype=dtype) if not experts and not gated else None
    seg = torch.zeros(experts + 1, device="cuda", dtype=torch.int32)
    inputs = [torch.zeros(rows, k, device="cuda", dtype=dtype) for _ in range(2)]

    def call(x):
        if experts:
            return ops.moe_gemm_mx(x, codes, scales, seg, gated, act_bits=bits)
        if gated:
            return ops.gated_mx(x, codes, scales, bits)
        return ops.linear_mx(x, codes, scales, bias, bits)

    seg[1:] = rows
    (one, y1), (two, y2) = (captured(lambda x=x: call(x)) for x in inputs)
    side = torch.cuda.Stream()
    for turn in range(4):
        for x in inputs:
            x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        if bias is not None:
            bias.copy_(torch.randn(n, generator=g, device="cuda"))
        if experts:
            seg[1:experts] = rows * turn // 3
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(2):
            one.replay()
            with torch.cuda.stream(side):
                two.replay()
        torch.cuda.synchronize()
        for x, y in zip(inputs, (y1, y2)):
            assert torch.equal(y, call(x))


def test_rows_of_a_graph_are_right():
    """A product in two parts, replayed, against 64 bits."""
    rows, n, k = 512, 4096, 14336
    assert ops._C.mx_plan(rows, n, k, 0, 6, False)[2:] == (128, 128, 2)
    wq, scales, values = oracle.weights(n, k, 5)
    wq, scales, values = wq.cuda(), scales.cuda(), values.cuda()
    x = torch.zeros(rows, k, device="cuda", dtype=torch.float16)
    bias = torch.zeros(n, device="cuda", dtype=torch.float16)
    graph, y = captured(lambda: ops.linear_mx(x, wq, scales, bias, 6))
    for seed in range(3):
        g = torch.Generator("cuda").manual_seed(seed)
        x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        bias.copy_(torch.randn(n, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        q = oracle.quantize(x, 6)[2].cuda()
        want = q @ values.T + bias.double()
        off = oracle.sums_off(q.abs() @ values.abs().T + bias.double().abs(), k + 1)
        assert ((y.double() - want).abs() <= oracle.rounded_off(want, off, y.dtype)).all()
