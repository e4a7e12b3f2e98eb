"""Microscaled products whose sums are exact in 32 bits, in whatever order: results are the exact
sums rounded once, so that one lost input, a sum held in fewer bits or a bias added twice shows.

Rows are numbers of their format with a magnitude in the top binade in each block, so that rounding
leaves them as they are.  Products are whole multiples of a unit of 2^-12 (steps of 1/8 and 1/2,
block scales of at least 2^-1 and 2^-7), biases too, and the sum of all magnitudes stays below
2^24 units, which is looked at for each case."""

import pytest
import torch

import mx_oracle as oracle
from vllm_tgis_adapter_amd import ops

TYPES = [torch.bfloat16, torch.float16, torch.float32]
UNIT = 2.0 ** -12


def exact_rows(rows: int, k: int, bits: int, g, device) -> torch.Tensor:
    grid = oracle.numbers(bits).to(device)
    x = grid[torch.randint(0, len(grid), (rows, k // 32, 32), generator=g, device=device)]
    x[..., 0] = 4.0
    x = torch.where(torch.rand(x.shape, generator=g, device=device) < 0.5, -x, x)
    scale = torch.randint(-1, 1, (rows, k // 32, 1), generator=g, device=device)
    return (x * torch.exp2(scale.double())).view(rows, k)


def random_weights(shape, k: int, g, device):
    codes = torch.randint(0, 256, (*shape, k // 2), generator=g, device=device, dtype=torch.uint8)
    scales = torch.randint(120, 122, (*shape, k // 32), generator=g, device=device, dtype=torch.uint8)
    return codes, scales


def widened(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = oracle.numbers(4).to(codes.device)
    table = torch.cat([table, -table])
    values = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    values = values.view(*scales.shape, 32) * torch.exp2(scales.double() - 127)[..., None]
    return values.flatten(-2)


def is_exact(got: torch.Tensor, x: torch.Tensor, w: torch.Tensor, bias, gated: bool) -> None:
    """Results of rows x (64 bits) and weights w."""
    y, magnitude = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        y, magnitude = y + bias.double(), magnitude + bias.double().abs()
    assert magnitude.max() < 2 ** 24 * UNIT
    if not gated:
        assert torch.equal(got, y.to(got.dtype))
        return
    g, u = y.chunk(2, dim=1)
    want = g * torch.sigmoid(g) * u
    # of the exponential: its argument's rounding and that of log2(e), |g| half steps and a
    # quarter of them, and a handful for itself, the sum, the division and the products
    own = (1.25 * g.abs() + 12) * 2.0 ** -24 * want.abs() + 1e-36
    assert ((got.double() - want).abs() <= oracle.rounded_off(want, own, got.dtype)).all()


def check(rows, n, k, experts, bits, gated, device):
    g = torch.Generator(device).manual_seed(rows * n + k + experts)
    shape = (n * (2 if gated else 1),)
    x = exact_rows(rows, k, bits, g, device)
    codes, scales = random_weights((experts, *shape) if experts else shape, k, g, device)
    bias = None
    if not experts and not gated:   # multiples of 2^-5 up to 4: whole units, 7 bits
        bias = torch.randint(-128, 129, (n,), generator=g, device=device) / 32
    if experts:
        cuts = torch.randint(0, rows + 1, (experts - 1,), generator=torch.Generator().manual_seed(n))
        bounds = [0, *sorted(cuts.tolist()), rows]
        seg = torch.tensor(bounds, dtype=torch.int32, device=device)
    for dtype in TYPES:
        rounded = x.to(dtype)
        assert torch.equal(rounded.double(), x)
        if experts:
            got = ops.moe_gemm_mx(rounded, codes, scales, seg, gated, act_bits=bits)
        elif gated:
            got = ops.gated_mx(rounded, codes, scales, bits)
        else:
            got = ops.linear_mx(rounded, codes, scales, bias.to(dtype), bits)
        assert got.dtype == dtype and got.shape == (rows, n)
        if not experts:
            is_exact(got, x, widened(codes, scales), bias, gated)
            continue
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if b > a:
                is_exact(got[a:b], x[a:b], widened(codes[e], scales[e]), None, gated)


@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("rows,n,k,experts,gated", [
    (3, 14, 32, 0, False), (2, 5, 28672, 0, False), (2, 5, 14336, 0, True), (9, 6, 288, 4, True),
    (9, 6, 4096, 4, False)])
def test_plain_path(rows, n, k, experts, bits, gated):
    check(rows, n, k, experts, bits, gated, "cpu")


# (rounded inside, rows of a tile, columns), parts of K, rows, outputs, inputs, experts, bits, gated
FORMS = [
    ((True, 16, 0), False, 1, 502, 28672, 0, 4, False),
    ((True, 16, 0), False, 16, 9001, 1056, 0, 6, False),
    ((True, 16, 0), False, 3, 9001, 8192, 0, 4, False),
    ((True, 16, 0), False, 3, 5001, 8192, 0, 6, True),
    ((True, 16, 0), False, 40, 501, 288, 4, 6, True),
    ((True, 16, 0), False, 30, 1001, 4096, 8, 4, False),
    ((False, 32, 0), False, 20, 502, 2048, 0, 4, True),
    ((False, 32, 0), False, 20, 501, 2048, 0, 4, False),
    ((False, 32, 0), False, 100, 501, 288, 4, 6, False),
    ((False, 64, 0), False, 40, 502, 288, 0, 6, False),
    ((False, 64, 0), False, 129, 501, 288, 4, 4, True),
    ((False, 16, 128), True, 13, 501, 28672, 0, 6, False),
    ((False, 16, 128), False, 20, 2050, 28672, 8, 6, False),
    ((False, 16, 128), True, 20, 501, 14336, 3, 4, False),
    ((False, 32, 128), True, 20, 501, 28672, 0, 6, False),
    ((False, 32, 128), False, 20, 8201, 14336, 0, 4, True),
    ((False, 32, 128), False, 130, 2050, 14336, 8, 4, False),
    ((False, 32, 128), True, 61, 501, 28672, 3, 6, False),
    ((False, 64, 128), True, 61, 501, 28672, 0, 6, False),
    ((False, 64, 128), True, 64, 501, 28672, 0, 4, True),
    ((False, 64, 128), True, 100, 502, 4096, 0, 4, False),
    ((False, 64, 128), False, 100, 501, 288, 0, 6, False),
    ((False, 64, 128), False, 260, 2050, 28672, 8, 4, False),
    ((False, 64, 128), True, 130, 501, 14336, 3, 6, False),
    ((False, 64, 224), False, 61, 24601, 2816, 0, 6, True),
    ((False, 64, 224), False, 61, 49202, 2816, 0, 4, False),
    ((False, 64, 224), False, 260, 3001, 28672, 8, 6, True),
    ((False, 64, 256), False, 40, 32701, 2816, 0, 6, True),
    ((False, 64, 256), False, 300, 8187, 2048, 8, 6, False),
    ((False, 128, 128), True, 1030, 501, 8192, 0, 4, False),
    ((False, 128, 128), False, 200, 8201, 288, 0, 6, False),
    ((False, 128, 128), True, 66, 2050, 28672, 0, 6, False),
    ((False, 128, 128), False, 520, 3001, 1056, 8, 4, False),
    ((False, 128, 128), True, 200, 501, 28672, 3, 4, True),
    ((False, 128, 256), True, 66, 8201, 14336, 0, 6, False),
    ((False, 128, 256), False, 260, 12001, 1056, 0, 6, False),
    ((False, 128, 256), False, 2000, 4093, 4128, 0, 4, False),
    ((False, 128, 256), True, 66, 2050, 28672, 0, 6, True),
    ((False, 128, 256), False, 260, 8201, 1056, 3, 6, False),
    ((False, 128, 256), True, 200, 2050, 28672, 3, 6, False),
    ((False, 256, 256), False, 1030, 8201, 288, 0, 6, False),
    ((False, 256, 256), False, 2060, 4097, 288, 0, 4, False),
    ((False, 256, 256), True, 130, 12001, 28672, 0, 4, False),
    ((False, 256, 256), False, 260, 12001, 14336, 0, 6, True),
    ((False, 256, 256), False, 520, 8201, 288, 8, 6, False),
    ((False, 256, 256), True, 2060, 1001, 28672, 3, 6, False),
    ((False, 256, 256), True, 2060, 501, 28672, 2, 6, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("form,cut,rows,n,k,experts,bits,gated", FORMS)
def test_form(form, cut, rows, n, k, experts, bits, gated):
    """Each tile, whole K and cut, plain with a bias and gated, dense and by experts, in all types,
    rows of outputs that are not whole fours among them."""
    plan = ops._C.mx_plan(rows, n, k, experts, bits, gated)
    assert plan[1:4] == form and (plan[4] > 1) == cut
    check(rows, n, k, experts, bits, gated, "cuda")


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [4, 6])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [3, 40, 300])
def test_small_numbers(m, dtype, bits, device):
    """Rows, terms and results below a type's least normal number: one term a result, and sums
    of 32 equal ones, are the exact ones rounded once."""
    g = torch.Generator().manual_seed(m)
    one, all_ = torch.zeros(8, 64), torch.zeros(8, 64)
    one[:, :8] = torch.eye(8)
    all_[:, :32] = 1.0
    for of_x in (-149, -140, -133, -127, -126, -125, -24, -20, -16):
        x = (torch.randn(m, 64, generator=g).double() * 2.0 ** of_x).to(dtype)
        flat = torch.full((m, 64), 2.0 ** of_x, dtype=torch.float64).to(dtype)
        for of_w in (-20, 0, 20):
            wq, scales = (t.to(device) for t in ops.quantize_mx(one * 2.0 ** of_w))
            want = oracle.quantize(x, bits)[2][:, :8] * 2.0 ** of_w
            got = ops.linear_mx(x.to(device), wq, scales, act_bits=bits).cpu()
            assert torch.equal(got, want.to(dtype)), (of_x, of_w)
            wq, scales = (t.to(device) for t in ops.quantize_mx(all_ * 2.0 ** of_w))
            want = oracle.quantize(flat, bits)[2][:, :8] * 32 * 2.0 ** of_w
            got = ops.linear_mx(flat.to(device), wq, scales, act_bits=bits).cpu()
            assert torch.equal(got, want.to(dtype)), (of_x, of_w)
