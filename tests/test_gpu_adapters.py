"""A shared projection with low-rank adapters beside it, against the plain form in 64 bits."""
import numpy as np
import pytest
import torch

import plain_requests as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


def case(ops, T, K, N, R, S, dtype, seed=0, pad=0, index=None):
    g = torch.Generator().manual_seed(seed + 1000 * T + K + N + R)
    normal = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    x = normal(T, K + pad).to(dtype).to(DEV)[:, :K]
    w = (normal(N, K) * 0.05).to(dtype).to(DEV)
    a = (normal(S, R, K) / K ** 0.5).to(dtype).to(DEV)
    b = (normal(S, N, R) * 0.2).to(dtype).to(DEV)
    scales = (0.5 + torch.rand(S, generator=g)).to(DEV)
    if index is None:
        index = torch.randint(-1, S + 1, (T,), generator=g)  # S: outside of the bank
    index = torch.as_tensor(index, dtype=torch.int32).to(DEV)
    return x, w, ops.AdapterBank(a, b, scales), index


def check(ops, x, w, bank, index, y, out_bf16):
    host = lambda t: t.float().cpu().numpy()  # noqa: E731
    want, size, much = plain.adapted(host(x), host(w), host(bank.a), host(bank.b), host(bank.scales),
                                     index.cpu().numpy())
    terms = x.shape[1] + bank.rank + 8
    bound = plain.adapted_bound(want, size, much, terms, out_bf16)
    if x.dtype == torch.bfloat16 and not out_bf16:
        bound += 2.0 ** -8 * size
    off = np.abs(host(y).astype(np.float64) - want)
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("K,N,R,S", [(256, 512, 16, 4), (520, 200, 24, 3), (1024, 328, 64, 9)])
def test_against_the_plain_form(ops, T, K, N, R, S, dtype):
    x, w, bank, index = case(ops, T, K, N, R, S, dtype)
    check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), dtype == torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K,N,R", [(8, 8, 8), (64, 1, 8), (72, 77, 40), (100, 50, 16), (33, 17, 8), (4096, 1024, 512),
                                   (2048, 2048, 96), (1000, 4104, 128)])
@pytest.mark.parametrize("T", [1, 5, 40, 200])
def test_odd_sizes(ops, T, K, N, R, dtype):
    x, w, bank, index = case(ops, T, K, N, R, 2, dtype)
    check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), dtype == torch.bfloat16)


@pytest.mark.parametrize("T", [3, 12, 50, 150, 700])
def test_rows_of_a_wider_buffer_and_32_bit_results(ops, T):
    x, w, bank, index = case(ops, T, 512, 264, 32, 3, torch.bfloat16, pad=24)
    y = ops.adapted_product(x, w, bank, index, out_dtype=torch.float32)
    assert y.dtype == torch.float32
    check(ops, x, w, bank, index, y, False)


@pytest.mark.parametrize("index", ["none", "one", "blocks", "every"])
@pytest.mark.parametrize("T", [16, 48, 256, 777])
def test_how_adapters_lie_among_the_tokens(ops, T, index):
    S = 64
    which = {"none": np.full(T, -1), "one": np.zeros(T), "blocks": np.arange(T) * 5 // T - 1,
             "every": np.arange(T) % S}[index]
    x, w, bank, index = case(ops, T, 512, 384, 16, S, torch.bfloat16, index=which.astype(np.int32))
    check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), True)


@pytest.mark.parametrize("T", [8, 40, 300])
def test_a_row_depends_on_its_own_adapter_alone(ops, T):
    """Wild numbers in slots that no row has reach nobody, and neither do those of another row's `a`. (A
    finite `b` is the caller's part: behind the projection's own K, zeros meet the b of the block's other
    adapters, and zero times infinity is no zero.)"""
    x, w, bank, index = case(ops, T, 512, 264, 16, 4, torch.bfloat16, index=np.arange(T) % 3)
    want = ops.adapted_product(x, w, bank, index)
    bank.a[3], bank.b[3] = float("nan"), float("inf")
    assert torch.equal(ops.adapted_product(x, w, bank, index), want)
    bank.a[1, 3:] = float("nan")
    bank.scales[1] = float("inf")
    got = ops.adapted_product(x, w, bank, index)
    others = (index != 1).nonzero()[:, 0]
    assert torch.equal(got[others], want[others])
    assert not torch.isfinite(got[(index == 1).nonzero()[:, 0]]).any()


def test_without_an_adapter_it_is_the_product(ops):
    for T in (1, 16, 48, 300):
        x, w, bank, index = case(ops, T, 1024, 512, 16, 2, torch.bfloat16, index=np.full(T, -1))
        got = ops.adapted_product(x, w, bank, index).float()
        want = (x.double() @ w.double().T).float()
        assert torch.allclose(got, want, rtol=2.0 ** -8 * 1.01, atol=1024 * 2.0 ** -24 * 1024 * 0.05)


@pytest.mark.parametrize("K,N,R,S", [(512, 384, 64, 24), (520, 132, 48, 20), (4096, 640, 128, 40), (72, 1000, 200, 58)])
@pytest.mark.parametrize("T", [17, 24, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_many_adapters_behind_the_products_k(ops, T, K, N, R, S, out):
    """Up to as many as may ride there, all of them among the rows or a few; N past the last tile of 128."""
    for index in (np.arange(T) * 7 % S, np.where(np.arange(T) % 3 == 0, S - 1, -1), np.arange(T) % (S + 2) - 1):
        x, w, bank, index = case(ops, T, K, N, R, S, torch.bfloat16, pad=16, index=index.astype(np.int32))
        check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index, out_dtype=out), out == torch.bfloat16)


@pytest.mark.parametrize("T,K,N,R,S", [(300, 4096, 512, 64, 3), (300, 4096, 512, 64, 100), (257, 8200, 264, 32, 5), (700, 4096, 136, 128, 9),
                                       (130, 16384, 200, 200, 70), (1025, 4104, 72, 16, 2), (64, 16392, 264, 64, 20),
                                       (40, 26216, 136, 64, 3)])
def test_rank_numbers_on_the_tensor_cores(ops, T, K, N, R, S):
    """Where they leave rows for a pass behind the projection's sums, or planes for a few rows' product."""
    assert ops._low_pays(T, K, S, R) and not ops._planes_pay(T, N, S, R)
    for index in (None, (np.arange(T) * 5 // T % S).astype(np.int32)):
        x, w, bank, index = case(ops, T, K, N, R, S, torch.bfloat16, index=index)
        check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), True)


@pytest.fixture
def behind_k(ops, monkeypatch):
    """The paired product with the adapters behind its K, whatever the sizes' rule says."""
    monkeypatch.setattr(ops, "_planes_pay", lambda T, N, slots, rank: T > 64 and N >= 128)
    return ops


@pytest.mark.parametrize("T", [65, 128, 130, 255, 256, 257, 300, 777])
@pytest.mark.parametrize("K,N,R,S", [(64, 128, 8, 1), (512, 200, 24, 3), (520, 1024, 64, 9), (1032, 136, 200, 4), (256, 648, 16, 64)])
def test_behind_the_paired_products_k(behind_k, T, K, N, R, S):
    for index in (None, (np.arange(T) * 3 // T % S).astype(np.int32), np.arange(T, dtype=np.int32) % S):
        x, w, bank, index = case(behind_k, T, K, N, R, S, torch.bfloat16, pad=8, index=index)
        check(behind_k, x, w, bank, index, behind_k.adapted_product(x, w, bank, index), True)
    check(behind_k, x, w, bank, index, behind_k.adapted_product(x, w, bank, index, out_dtype=torch.float32), False)


def test_behind_the_paired_products_k_a_row_depends_on_its_own_adapter_alone(behind_k):
    test_a_row_depends_on_its_own_adapter_alone(behind_k, 300)
    test_a_row_depends_on_its_own_adapter_alone(behind_k, 70)


def test_behind_the_paired_products_k_on_another_stream_and_replayed(behind_k):
    test_on_another_stream_and_replayed(behind_k)
    test_prompts_and_single_tokens_on_two_streams(behind_k)


@pytest.mark.parametrize("T,N,R", [(1, 16640, 512), (5, 16400, 128), (8, 16392, 64), (9, 8200, 64), (13, 2000, 256), (16, 16400, 16)])
@pytest.mark.parametrize("scaled", [False, True])
def test_a_few_rows_of_wide_projections(ops, T, N, R, scaled):
    """Where a few rows' adapters leave the weight-streaming product's epilogue; a norm's row scale is then
    the results' as well."""
    K = 256
    x, w, bank, index = case(ops, T, K, N, R, 4, torch.bfloat16)
    assert ops._rows_pay(T, N, 4, R)
    if not scaled:
        check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), True)
        return
    shares = torch.rand(16, 16, device=DEV) * 40
    y = ops.adapted_product(ops.RowScaled(x.contiguous(), shares, 1e-5), w, bank, index).float().cpu().numpy().astype(np.float64)
    host = lambda t: t.float().cpu().numpy()  # noqa: E731
    scale = 1 / np.sqrt(host(shares).astype(np.float64).sum(0)[:T] / K + 1e-5)
    want, size, much = (v * scale[:, None] for v in plain.adapted(
        host(x), host(w), host(bank.a), host(bank.b), host(bank.scales), index.cpu().numpy()))
    bound = plain.adapted_bound(want, size, much, K + bank.rank + 40, True)
    assert (np.abs(y - want) <= bound).all(), (np.abs(y - want) / bound).max()


@pytest.mark.parametrize("N", [64, 256])  # the rank numbers as rows, and as planes behind K
@pytest.mark.parametrize("T", [8192, 8193, 8200, 16500])
def test_more_tokens_than_one_launch_takes(ops, T, N):
    x, w, bank, index = case(ops, T, 64, N, 8, 3, torch.bfloat16, pad=8)
    check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), True)


@pytest.mark.parametrize("T", [5, 300, 7000])
@pytest.mark.parametrize("S", [1024, 1025, 3000])
def test_banks_of_thousands_of_places(ops, T, S):
    """More than the tensor cores' kernel keeps its marks for; blocks with as many adapters as tokens."""
    x, w, bank, index = case(ops, T, 64, 256, 8, S, torch.bfloat16)
    check(ops, x, w, bank, index, ops.adapted_product(x, w, bank, index), True)


def test_prompts_and_single_tokens_on_two_streams(ops):
    """One bank and index for projections of prompts and of single tokens, in turn and on two streams."""
    x, w, bank, index = case(ops, 600, 512, 4096, 16, 4, torch.bfloat16)
    few = [x[i:i + 3].contiguous() for i in range(0, 30, 3)]
    of_few = [index[i:i + 3].contiguous() for i in range(0, 30, 3)]
    want, want_few = ops.adapted_product(x, w, bank, index), [
        ops.adapted_product(t, w, bank, i) for t, i in zip(few, of_few)]
    torch.cuda.synchronize()
    side, got_few = torch.cuda.Stream(), []
    for _ in range(3):
        got = ops.adapted_product(x, w, bank, index)
        with torch.cuda.stream(side), ops.scratch_owner("adapters beside"):
            got_few = [ops.adapted_product(t, w, bank, i) for t, i in zip(few, of_few)]
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert all(torch.equal(g, v) for g, v in zip(got_few, want_few))
    ops.release_scratch("adapters beside")


@pytest.mark.parametrize("S,T", [(1000, 3), (1000, 16), (1000, 40), (1000, 70), (1400, 20), (1000, 600)])
def test_banks_past_32_bits(ops, S, T):
    """7 GB of B and more: the last places' rows lie behind 2^32 bytes and 2^31 numbers."""
    K, N, R = 64, 16640, 136
    x, w, small, _ = case(ops, T, K, N, R, 2, torch.bfloat16)
    a = torch.zeros(S, R, K, dtype=torch.bfloat16, device=DEV)
    b = torch.zeros(S, N, R, dtype=torch.bfloat16, device=DEV)
    assert b.numel() > 1 << 31
    a[-2:], b[-2:] = small.a, small.b
    scales = torch.zeros(S, device=DEV)
    scales[-2:] = small.scales
    index = torch.arange(T, dtype=torch.int32, device=DEV) % 2
    got = ops.adapted_product(x, w, ops.AdapterBank(a, b, scales), index + S - 2)
    check(ops, x, w, small, index, got, True)


# The weight-streaming product's other epilogues, with adapters in their sums
def sums_of(x, w, bank, index, scale=1.0):
    """The sums in 64 bits, and what 32-bit ones may be off by."""
    host = lambda t: t.float().cpu().numpy()  # noqa: E731
    want, _, much = plain.adapted(host(x), host(w), host(bank.a), host(bank.b), host(bank.scales), index.cpu().numpy())
    return want, (x.shape[1] + bank.rank + 8) * 2.0 ** -24 * much


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T", [1, 3, 8, 9, 16, 17, 32, 40, 64, 70])
@pytest.mark.parametrize("K,I,R,S", [(256, 128, 16, 4), (520, 100, 48, 3), (2048, 1024, 128, 9)])
def test_gated_pairs(ops, T, K, I, R, S, act):
    x, w, bank, index = case(ops, T, K, 2 * I, R, S, torch.bfloat16)
    out = torch.empty(T, I, dtype=torch.bfloat16, device=DEV)
    assert ops.adapted_epilogue_fits(x, w, bank) == (T <= 16) and ops.adapted_rows_fit(x, w, bank) == (17 <= T <= 64)
    ops.adapted_silu_mul(x, w, bank, index, out, act=act)
    sums, off = sums_of(x, w, bank, index)
    if T > 16:  # the rank numbers may be bfloat16 there
        _, size, _ = plain.adapted(*(t.float().cpu().numpy() for t in (x, w, bank.a, bank.b, bank.scales)),
                                   index.cpu().numpy())
        off = off + 2.0 ** -8 * size
    gate, up, d_gate, d_up = sums[:, ::2], sums[:, 1::2], off[:, ::2], off[:, 1::2]
    if act == "silu":
        value = gate / (1 + np.exp(-gate))
    else:
        value = 0.5 * gate * (1 + np.tanh(np.sqrt(2 / np.pi) * (gate + 0.044715 * gate ** 3)))
    # both activations have slopes below 1.13; 2^-20 of the value for their own exponentials
    want = value * up
    bound = 1.13 * d_gate * (np.abs(up) + d_up) + np.abs(value) * d_up + (2.0 ** -8 * 1.01 + 2.0 ** -20) * np.abs(want) + 1e-30
    assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("T", [1, 5, 8, 9, 16, 17, 40, 64])
@pytest.mark.parametrize("K,N,R,S,scale", [(256, 128, 16, 4, 1.0), (520, 200, 48, 3, 0.5), (4096, 2048, 64, 9, 1.0)])
def test_sums_into_the_residual_rows(ops, T, K, N, R, S, scale):
    x, w, bank, index = case(ops, T, K, N, R, S, torch.bfloat16)
    g = torch.Generator().manual_seed(T)
    before, gamma = torch.randn(T, N, generator=g).to(DEV), torch.rand(N, generator=g).to(DEV)
    resid = before.clone()
    got = ops.adapted_residual(x, w, bank, index, residual=ops.ResidualSink(resid, gamma, 1e-5, scale))
    sums, off = sums_of(x, w, bank, index)
    if T > 16:
        _, size, _ = plain.adapted(*(t.float().cpu().numpy() for t in (x, w, bank.a, bank.b, bank.scales)),
                                   index.cpu().numpy())
        off = off + 2.0 ** -8 * size
    if T > 16 and scale != 1.0:  # that product adds its sums as they are
        assert isinstance(got, ops.Planes) and torch.equal(resid, before)
        return
    assert isinstance(got, ops.NormPending)
    want = before.double().cpu().numpy() + scale * sums
    bound = scale * off + 2.0 ** -23 * (np.abs(want) + scale * np.abs(sums))
    assert (np.abs(resid.double().cpu().numpy() - want) <= bound).all()
    assert torch.equal(got.values, (resid * gamma).bfloat16())
    squares = resid.double().square().sum(1)
    assert torch.allclose(got.shares.double().sum(0)[:T], squares, rtol=1e-5)
    # without a sink, and for more rows than the kernel takes: 32-bit sums
    planes = ops.adapted_residual(x, w, bank, index)
    off = np.abs(planes.sum(torch.float32).double().cpu().numpy() - sums) - off
    assert isinstance(planes, ops.Planes) and (off <= 2.0 ** -24 * np.abs(sums)).all()


@pytest.mark.parametrize("pairing", ["half", "interleaved"])
@pytest.mark.parametrize("T", [1, 6, 8, 13, 16, 17, 40, 64])
@pytest.mark.parametrize("A,Kh,D,rot", [(4, 2, 16, 16), (6, 3, 32, 32), (3, 1, 48, 32), (8, 2, 128, 128), (2, 2, 64, 0)])
@pytest.mark.parametrize("scaled", [False, True])
def test_rotated_projections(ops, A, Kh, D, rot, T, pairing, scaled):
    """Against the 32-bit sums' own rotation: both round once, what they round differs by their sums' order."""
    K, N = 264, (A + 2 * Kh) * D
    x, w, bank, index = case(ops, T, K, N, 24, 5, torch.bfloat16)
    inv_freq = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float32) / max(rot, 1))).to(DEV)
    as_int = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    positions, seqs = as_int([(37 * t) % 700 for t in range(T)]), as_int([-1 if t == 5 else 0 for t in range(T)])
    table = torch.arange(11, dtype=torch.int32, device=DEV).view(1, 11)
    ops_args = (positions, seqs, table, inv_freq, rot)
    caches = [torch.zeros(11, Kh, 64, D, dtype=torch.bfloat16, device=DEV) for _ in range(4)]
    given = ops.RowScaled(x.contiguous(), torch.rand(16, (T + 15) // 16 * 16, device=DEV) * 40 + 1, 1e-5) if scaled else x
    if T <= 16:
        q = ops.gemm_skinny_rope(given, w, *ops_args, caches[0], caches[1], A, Kh, D, pairing=pairing,
                                 adapters=(bank, index))
    else:
        if pairing == "half":
            pytest.skip("that product rotates neighbours")
        assert ops.qkv_rows_rope_fusable(given, w, rot, D, caches[0], pairing) and ops.adapted_rows_fit(given, w, bank)
        q = ops.gemm_rows_rope(given, w, *ops_args, caches[0], caches[1], A, Kh, D, adapters=(bank, index))
        # (without the cache's rows its weights would be fewer than the bank's)
        with pytest.raises(ops.KernelError):
            ops.gemm_rows_rope(given, w, *ops_args, None, None, A, Kh, D, write_cache=False, adapters=(bank, index))
    sums = ops.adapted_product(given, w, bank, index, out_dtype=torch.float32)
    q2 = ops.rope_kv_write(ops.Planes(sums[None].clone()), *ops_args, caches[2], caches[3], A, Kh, D,
                           dtype=torch.bfloat16, pairing=pairing)
    live = [t for t in range(T) if t != 5]
    most = float(sums.abs().max())
    for one, two in ((q[live], q2[live]), (caches[0], caches[2]), (caches[1], caches[3])):
        one, two = one.float(), two.float()
        # a rounding each, and 32-bit sums of K + 24 products of which none passes the largest sum by much
        assert ((one - two).abs() <= 2.0 ** -7 * torch.maximum(one.abs(), two.abs()) + 2.0 ** -15 * most).all()


def test_no_tokens(ops):
    x, w, bank, index = case(ops, 0, 64, 32, 8, 1, torch.bfloat16, index=[])
    assert ops.adapted_product(x, w, bank, index).shape == (0, 32)


@pytest.mark.parametrize("T", [9, 16, 40])
def test_a_row_scaled_input(ops, T):
    """What a norm leaves for the products behind it: scale_t * values. A few tokens' product is linear in
    the scale and takes it behind its sums; otherwise the rows are scaled first, and rounded again (2^-8 of
    every factor, so of the products' absolute sum)."""
    K = 512
    x, w, bank, index = case(ops, T, K, 256, 16, 3, torch.bfloat16)
    shares = torch.rand(32, (T + 15) // 16 * 16, device=DEV) * 40
    scaled = ops.RowScaled(x.contiguous(), shares, 1e-5)
    y = ops.adapted_product(scaled, w, bank, index).float().cpu().numpy().astype(np.float64)
    host = lambda t: t.float().cpu().numpy()  # noqa: E731
    scale = 1 / np.sqrt(host(shares).astype(np.float64).sum(0)[:T] / K + 1e-5)
    want, size, much = plain.adapted(host(x), host(w), host(bank.a), host(bank.b), host(bank.scales),
                                     index.cpu().numpy())
    want, size, much = (v * scale[:, None] for v in (want, size, much))
    bound = plain.adapted_bound(want, size, much, K + bank.rank + 40, True) + (2.0 ** -8 * much if T > 16 else 0)
    assert (np.abs(y - want) <= bound).all(), (np.abs(y - want) / bound).max()


def test_on_another_stream_and_replayed(ops):
    for T in (4, 40, 300):
        x, w, bank, index = case(ops, T, 1024, 768, 32, 5, torch.bfloat16)
        want = ops.adapted_product(x, w, bank, index)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side), ops.scratch_owner(("adapters", T)):
            got = ops.adapted_product(x, w, bank, index)
            side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = ops.adapted_product(x, w, bank, index)
        x.copy_(x.flip(0))
        index.copy_(index.flip(0))
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        check(ops, x, w, bank, index, captured, True)
        ops.release_scratch(("adapters", T))
