"""4-bit products of whole numbers, where every fp32 sum is exact: compared bit for bit with the
64-bit result rounded once."""
import pytest
import torch
from test_int4_gpu import DT, _values, _weight

from pytorch_distributed_matmul_benchmark_amd import ops

pytestmark = pytest.mark.gpu


def _same(y, x, q, s, z):
    want = (x.double() @ _values(q, s, z)[0].t()).to(y.dtype)
    assert torch.equal(y, want), f"{(y != want).sum().item()} of {y.numel()} differ"


@pytest.mark.parametrize("M", [1, 20, 100])
@pytest.mark.parametrize("zero", [False, True], ids=["sym", "zero"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_an_outlier_of_zero_weights_leaves_no_trace(dtype, zero, M):
    """One value of 2^18 (fp16: 2^15) a row, whose weights are zero, among whole numbers up to 3: every
    product is below 31 x 2^18 and with the 255 others every sum below 2^23 + 255 x 3 x 31 < 2^24."""
    K, N, big = 256, 200, 2.0 ** 18 if dtype == "bf16" else 2.0 ** 15
    q, _, z = _weight((), N, K, 64, DT[dtype], zero)
    s = torch.ones(N, K // 64, device="cuda", dtype=DT[dtype])
    x = torch.randint(-3, 4, (M, K), device="cuda").to(DT[dtype])
    nothing = (z if zero else torch.full_like(s, 8).byte()).repeat_interleave(32, -1)  # of each byte's group
    at = torch.arange(M, device="cuda") % 16 + 16 * (torch.arange(M, device="cuda") % 7)  # each place of a dword
    q[:, at // 2] = (nothing | nothing << 4)[:, at // 2]
    x[torch.arange(M, device="cuda"), at] = big
    y = ops.int4_matmul(x, q, s, z)
    _same(y, x, q, s, z)


def test_large_finite_rows():
    """2^122 times a weight of up to 15: 31 x 2^122 is below the fp32 range's end, 3.4e38."""
    K, N = 256, 96
    q, s, z = _weight((), N, K, 128, torch.bfloat16, True)
    s.fill_(2.0 ** -20)
    x = torch.zeros(K, K, device="cuda", dtype=torch.bfloat16)
    x.fill_diagonal_(2.0 ** 122)
    for rows in (x[:1], x[:16], x):
        _same(ops.int4_matmul(rows, q, s, z), rows, q, s, z)


@pytest.mark.parametrize("ends", [False, True])
def test_rows_far_apart(ends):
    """The last tokens' rows of a batch of long sequences: more than 2^23 elements from row to row."""
    K, N = 256, 96
    q, s, z = _weight((2,) if ends else (), N, K, 64, torch.bfloat16, True)
    far = torch.empty(3, 2049, 4096, device="cuda", dtype=torch.bfloat16)[:, -1, -K:]
    far.copy_(torch.randn(3, K, device="cuda"))
    assert far.stride(0) > 1 << 23
    kw = {"ends": torch.tensor([1, 3], device="cuda")} if ends else {}
    assert torch.equal(ops.int4_matmul(far, q, s, z, **kw), ops.int4_matmul(far.contiguous(), q, s, z, **kw))


def test_refusals_name_their_reason():
    K = (1 << 23) + 128
    q = torch.zeros(1, K // 2, device="cuda", dtype=torch.uint8)
    s = torch.ones(1, K // 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^23"):
        ops.int4_matmul(torch.zeros(1, K, device="cuda", dtype=torch.bfloat16), q, s)
    q, s, x = q[:, :64].contiguous(), s[:, :1].contiguous(), torch.zeros(2, 128, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="do not overlap"):
        ops.int4_matmul(x, q, s, out=torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16).expand(2, 1))
    with pytest.raises(RuntimeError, match="gradient"):
        ops.int4_matmul(x, q, s, out=torch.zeros(2, 1, device="cuda", dtype=torch.bfloat16, requires_grad=True))


def _whole(lead, M, N, K, G, dtype, zero):
    """x of -3 .. 3, scales 1/4 .. 2: a group's sum stays below 128 x 3 x 31 and the sum of all, in quarters, below
    4 x 2 x 3 x 15 K < 2^24 for K up to 46603."""
    assert 4 * 2 * 3 * 15 * K < 2 ** 24
    q, s, z = _weight(lead, N, K, G, dtype, zero)
    s = 2.0 ** torch.randint(-2, 2, s.shape, device="cuda").to(dtype)
    return torch.randint(-3, 4, (M, K), device="cuda").to(dtype), q, s, z


# long sums, partial last chunks (K % 128 = 32, 64, 96) and every group size, on each kernel and tile height
@pytest.mark.parametrize("M,N,K,G", [
    (1, 4096, 4096, 128), (1, 4096, 4096, 32), (1, 8200, 8192, 128), (4, 8300, 6208, 64), (13, 8300, 6272, 128),
    (13, 8300, 6240, 32), (16, 11007, 4096, 32), (16, 1023, 1024, 256), (17, 130, 544, 32), (32, 256, 2048, 2048),
    (25, 1024, 5600, 32), (33, 5400, 2080, 32), (47, 10176, 4480, 128), (64, 8001, 672, 32), (100, 8192, 4096, 64),
    (100, 384, 1536, 512), (130, 5000, 1152, 64), (500, 4090, 768, 128), (515, 640, 1056, 32)])
@pytest.mark.parametrize("zero", [False, True], ids=["sym", "zero"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_whole_numbers(dtype, zero, M, N, K, G):
    x, q, s, z = _whole((), M, N, K, G, DT[dtype], zero)
    y = ops.int4_matmul(x, q, s, z)
    _same(y, x, q, s, z)
    # (one matrix instruction's k less would show)
    assert not torch.equal(y, (x[:, :-32].double() @ _values(q, s, z)[0].t()[:-32]).to(y.dtype))


@pytest.mark.parametrize("sizes,N,K,G", [
    ([1] * 66, 1408, 2048, 128), ([0, 3, 1, 0], 8192, 6240, 32), ([17, 0, 40, 2], 100, 416, 32),
    ([100, 64, 1, 70], 4100, 4192, 32), ([30, 0, 32, 20], 5000, 1024, 64), ([9] * 8, 1416, 4128, 32)])
@pytest.mark.parametrize("zero", [False, True], ids=["sym", "zero"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_whole_numbers_of_experts(dtype, zero, sizes, N, K, G):
    x, q, s, z = _whole((len(sizes),), sum(sizes), N, K, G, DT[dtype], zero)
    y = ops.int4_matmul(x, q, s, z, ends=torch.tensor(sizes).cumsum(0).cuda())
    lo = 0
    for e, n in enumerate(sizes):
        _same(y[lo:lo + n], x[lo:lo + n], q[e], s[e], None if z is None else z[e])
        lo += n
