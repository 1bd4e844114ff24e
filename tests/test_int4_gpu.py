"""4-bit products on the GPU against the weight that (q, scale, zero) stand for, in 64 bits.

Tolerance: a bf16 result sums two products for each k, x (16 + q) and -x (16 + zero), in fp32, an
fp16 result one, x (q - zero); each group's sum is scaled and added to the others. So
the sum is off by at most (terms + groups + 10) fp32 steps (2^-23) of its terms'
magnitudes, and the result's rounding adds half a step of its type (fp16: 2^-25)."""
import pytest
import torch

from pytorch_distributed_matmul_benchmark_amd import ops

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _weight(lead, N, K, G, dtype, zero, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + N + 3 * K)
    q = torch.randint(0, 256, (*lead, N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scale = ((0.5 + torch.rand(*lead, N, K // G, device="cuda", generator=g)) * 0.05).to(dtype)
    z = torch.randint(0, 16, scale.shape, device="cuda", generator=g, dtype=torch.uint8) if zero else None
    return q, scale, z


def _values(q, scale, zero):
    """(weight, bound on a term's magnitude factor) [.., N, K] in float64"""
    G = q.shape[-1] * 2 // scale.shape[-1]
    v = torch.stack((q % 16, q // 16), -1).flatten(-2).double()
    z = (torch.full_like(scale, 8).double() if zero is None else zero.double()).repeat_interleave(G, -1)
    s = scale.double().repeat_interleave(G, -1)
    big = s.abs() * (32 + v + z) if scale.dtype == torch.bfloat16 else s.abs() * (v - z).abs()
    return s * (v - z), big


def _close(got, x, w, big, groups):
    exact, mag = x.double() @ w.t(), x.double().abs() @ big.t()
    terms = x.shape[1] * (2 if got.dtype == torch.bfloat16 else 1)
    bound = torch.finfo(got.dtype).eps / 2 * exact.abs() * 1.01 + (terms + groups + 10) * 2.0 ** -23 * mag + 2.0 ** -25
    off = (got.double() - exact).abs()
    assert bool((off <= bound).all()), f"off by {(off / bound).max().item():.3g} of the bound"


@pytest.mark.parametrize("M,N,K,G", [
    (1, 1, 32, 32), (1, 16, 128, 128), (1, 4096, 4096, 128), (3, 77, 96, 32), (7, 300, 192, 64),
    (16, 1023, 1024, 256), (17, 130, 544, 32), (32, 256, 2048, 2048), (33, 515, 320, 64),
    (64, 200, 640, 128), (100, 384, 1536, 512), (200, 1000, 1056, 32), (515, 640, 1024, 64)])
@pytest.mark.parametrize("zero", [False, True], ids=["sym", "zero"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_one_weight(dtype, zero, M, N, K, G):
    q, s, z = _weight((), N, K, G, DT[dtype], zero)
    x = torch.randn(M, K, device="cuda").to(DT[dtype])
    y = ops.int4_matmul(x, q, s, z)
    _close(y, x, *_values(q, s, z), K // G)


# enough columns that the rows are taken 16, 32, 64 and 64 (of 128 columns) a tile
@pytest.mark.parametrize("M,N,K", [(33, 5400, 2048), (64, 8001, 640), (130, 5000, 1152), (500, 4090, 768)])
@pytest.mark.parametrize("G,zero", [(32, True), (64, False), (64, True), (128, True), (128, False)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_many_columns(dtype, G, zero, M, N, K):
    q, s, z = _weight((), N, K, G, DT[dtype], zero)
    x = torch.randn(M, K, device="cuda").to(DT[dtype])
    _close(ops.int4_matmul(x, q, s, z), x, *_values(q, s, z), K // G)


@pytest.mark.parametrize("sizes,behind,N,K,G", [
    ([1], 0, 40, 64, 32), ([0, 3, 1, 0], 2, 136, 256, 64), ([1] * 66, 0, 48, 128, 128),
    ([17, 0, 40, 2], 0, 100, 416, 32), ([100, 64, 1], 5, 272, 768, 256),
    ([100, 64, 1, 70], 3, 4100, 416, 32), ([30, 0, 32, 20], 70, 5000, 1024, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_expert_weights(dtype, sizes, behind, N, K, G):
    dt, T = DT[dtype], sum(sizes) + behind
    q, s, z = _weight((len(sizes),), N, K, G, dt, True)
    x = torch.randn(T, K, device="cuda").to(dt)
    x[T - behind:] = float("nan")
    ends = torch.tensor(sizes).cumsum(0).cuda()
    y = ops.int4_matmul(x, q, s, z, ends=ends)
    out = torch.full_like(y, 9.0)
    assert ops.int4_matmul(x, q, s, z, ends=ends.int(), out=out) is out
    assert bool((y[T - behind:] == 0).all()) and bool((out[T - behind:] == 9).all())
    assert torch.equal(y[:T - behind], out[:T - behind])
    w, big = _values(q, s, z)
    lo = 0
    for e, n in enumerate(sizes):
        if n:
            _close(y[lo:lo + n], x[lo:lo + n], w[e], big[e], K // G)
        lo += n


def test_each_nibble_lands_on_its_k():
    """Unit rows pick out single weights, exactly: scale 1, every value of q - zero."""
    K = 256
    for dt in DT.values():
        q, _, z = _weight((), 48, K, 32, dt, True)
        s = torch.ones(48, K // 32, device="cuda", dtype=dt)
        y = ops.int4_matmul(torch.eye(K, device="cuda", dtype=dt), q, s, z)
        assert torch.equal(y.double(), _values(q, s, z)[0].t())


def test_views():
    q, s, z = _weight((), 72, 160, 32, torch.bfloat16, True)
    big = torch.full((9, 171), float("nan"), device="cuda", dtype=torch.bfloat16)
    x = big[1:8, 3:163]
    x.copy_(torch.randn(7, 160, device="cuda"))
    want = ops.int4_matmul(x.contiguous(), q, s, z)
    out = torch.zeros(7, 80, device="cuda", dtype=torch.bfloat16)[:, 5:77]
    assert torch.equal(ops.int4_matmul(x, q, s, z, out=out), want)
    assert torch.equal(ops.int4_matmul(x.t().contiguous().t(), q, s, z), want)
    shifted = torch.zeros(q.numel() + 1, device="cuda", dtype=torch.uint8)[1:].view(q.shape)
    shifted.copy_(q)
    assert torch.equal(ops.int4_matmul(x, shifted, s, z), want)


def test_infinities_stay_in_their_rows():
    q, s, z = _weight((), 64, 256, 64, torch.float16, True)
    x = torch.randn(20, 256, device="cuda").half()
    clean = ops.int4_matmul(x, q, s, z)
    x[3, 7] = float("inf")
    y = ops.int4_matmul(x, q, s, z)
    keep = torch.arange(20, device="cuda") != 3
    assert torch.equal(y[keep], clean[keep]) and not bool(y[3].isfinite().any())


def test_no_rows():
    q, s, z = _weight((), 64, 256, 64, torch.float16, True)
    assert ops.int4_matmul(torch.zeros(0, 256, device="cuda").half(), q, s, z).shape == (0, 64)
    assert ops.int4_matmul(torch.zeros(3, 256, device="cuda").half(), q[:0], s[:0], z[:0]).shape == (3, 0)


def test_captured_graph_and_repeats():
    q, s, z = _weight((4,), 320, 512, 128, torch.bfloat16, True)
    x = torch.randn(24, 512, device="cuda").bfloat16()
    ends = torch.tensor([6, 12, 18, 24], device="cuda")
    ops.int4_matmul(x, q, s, z, ends=ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.int4_matmul(x, q, s, z, ends=ends)
        y1 = ops.int4_matmul(x, q[1], s[1], z[1])
    for k, sizes in enumerate(([6, 6, 6, 6], [0, 24, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0], [6, 6, 6, 6])):
        ends.copy_(torch.tensor(sizes).cumsum(0))
        x.copy_(torch.randn(24, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.int4_matmul(x, q, s, z, ends=ends))
        assert torch.equal(y1, ops.int4_matmul(x, q[1], s[1], z[1]))


def test_quantised_weight_end_to_end():
    g = torch.Generator(device="cuda").manual_seed(8)
    w = torch.randn(512, 200, device="cuda", generator=g).bfloat16()
    x = torch.randn(5, 512, device="cuda", generator=g).bfloat16()
    for sym in (False, True):
        q, s, z = ops.int4_quantize(w, 128, sym)
        _close(ops.int4_matmul(x, q, s, z), x, *_values(q, s, z), 4)


@pytest.mark.parametrize("T", [3, 40, 200])
def test_offsets_past_32_bits(T):
    """Expert weights of more than 4 GiB: the last expert's last columns."""
    E, N, K, G = 5, 131080, 16384, 128
    q = torch.empty(E, N, K // 2, device="cuda", dtype=torch.uint8).random_(0, 256)
    s = torch.full((E, N, K // G), 0.01, device="cuda", dtype=torch.float16)
    s[:, -3:] = 0.02
    x = torch.randn(T, K, device="cuda").half()
    ends = torch.tensor([0, 0, 0, T // 2, T], device="cuda")
    y = ops.int4_matmul(x, q, s, ends=ends)
    for e, rows in ((3, slice(0, T // 2)), (4, slice(T // 2, T))):
        _close(y[rows, -40:], x[rows], *_values(q[e, -40:], s[e, -40:], None), K // G)


@pytest.mark.parametrize("G,zero", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("M", [1, 4, 13])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_long_sums_of_many_columns(dtype, M, G, zero):
    N, K = 8300, 6272 if G == 128 else 6240 if G == 32 else 6208
    q, s, z = _weight((), N, K, G, DT[dtype], zero)
    x = torch.randn(M, K, device="cuda").to(DT[dtype])
    _close(ops.int4_matmul(x, q, s, z), x, *_values(q, s, z), K // G)
