"""Products whose K is shared into planes of sums of any size: a plane starts where the one before ends, on 16 bytes or
not. And outputs that start where their caller says."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


def operands(M, N, K):
    """Whole numbers, whose sums are exact in 32 bits and most of them in bfloat16's 8 not."""
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    make = lambda *shape: torch.randint(-3, 4, shape, generator=g, device=DEV).bfloat16()  # noqa: E731
    return make(M, K), make(N, K)


SIZES = [(163, 143, 928), (129, 78, 968), (65, 77, 512), (127, 131, 2048), (199, 257, 1024), (255, 33, 4096), (131, 129, 640)]


@pytest.mark.parametrize("M,N,K", SIZES)
def test_planes_of_odd_sizes(ops, M, N, K):
    x, w = operands(M, N, K)
    want = x.double() @ w.double().T
    for splits in sorted({2, 3, ops._one_tile_plan(M, N, K)[0]}):
        planes = torch.full((splits, M, N), 7.0, device=DEV)
        ops.gemm_tc(x, w, planes, N, 1, 128, splits, M * N, constant_operand=2)
        assert torch.equal(planes.double().sum(0), want), splits
    got = ops.gemm_bf16(x, w, None, torch.float32, allow_planes=True)
    got = got.sum(torch.float32) if isinstance(got, ops.Planes) else got
    assert torch.equal(got.double(), want)
    assert torch.equal(ops.gemm_bf16(x, w), want.bfloat16())


@pytest.mark.parametrize("M,N,K", SIZES)
def test_adapters_beside_them(ops, M, N, K):
    x, w = operands(M, N, K)
    g = torch.Generator(device=DEV).manual_seed(K)
    a = torch.zeros(3, 8, K, dtype=torch.bfloat16, device=DEV)
    a[:, :, :200:7] = 1.0
    b = torch.randint(-2, 3, (3, N, 8), generator=g, device=DEV).bfloat16()
    index = torch.randint(-1, 3, (M,), generator=g, device=DEV, dtype=torch.int32)
    bank = ops.AdapterBank(a, b, torch.tensor([1.0, 0.5, 2.0], device=DEV))
    want = x.double() @ w.double().T
    for s in range(3):
        rows = (index == s).nonzero()[:, 0]
        want[rows] += float(bank.scales[s]) * (x[rows].double() @ a[s].double().T) @ b[s].double().T
    assert torch.equal(ops.adapted_product(x, w, bank, index, out_dtype=torch.float32).double(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 4, 8])
@pytest.mark.parametrize("M,N,K", [(300, 264, 256), (700, 512, 512), (2100, 256, 128)])
def test_outputs_that_start_anywhere(ops, M, N, K, shift, dtype):
    x, w = operands(M, N, K)
    flat = torch.full((M * (N + 8) + 16,), 7.0, dtype=dtype, device=DEV)
    out = flat[shift:shift + M * (N + 8)].view(M, N + 8)[:, :N]
    ops.gemm_bf16(x, w, out)
    assert torch.equal(out, (x.double() @ w.double().T).to(dtype))
    flat[shift:shift + M * (N + 8)].view(M, N + 8)[:, :N] = 7.0
    assert (flat == 7.0).all()


@pytest.mark.parametrize("act", ["silu", "clamped"])
@pytest.mark.parametrize("shift", [0, 1, 4, 8])
@pytest.mark.parametrize("M,I,K", [(40, 132, 256), (100, 200, 256), (300, 132, 256), (700, 256, 512), (2100, 136, 128)])
def test_gated_outputs_that_start_anywhere(ops, M, I, K, shift, act):
    """The same bits as in rows of their own, and nothing beside them."""
    x, w = operands(M, 2 * I, K)
    x, w = x * 0.1, w * 0.1
    clamp = ops.GluClamp(7.0, 1.7, 1.0, None) if act == "clamped" else None
    want = ops.gemm_bf16_silu_mul(x, w, torch.empty(M, I, dtype=torch.bfloat16, device=DEV), act=act, clamp=clamp)
    flat = torch.full((M * (I + 12) + 16,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = flat[shift:shift + M * (I + 12)].view(M, I + 12)[:, :I]
    ops.gemm_bf16_silu_mul(x, w, out, act=act, clamp=clamp)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert (flat == 7.0).all()
