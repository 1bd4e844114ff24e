"""Expert-grouped products where a sum ends inside a K-tile, beside what must not reach it."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from test_grouped_gpu import DT, _close, _data, _ends, _reduce_exact, _rows_exact

from pytorch_distributed_matmul_benchmark_amd import ops

pytestmark = pytest.mark.gpu


def _beside_nan(t):
    """t with 16 bytes of NaN behind every row."""
    b = torch.full((*t.shape[:-1], t.shape[-1] + 8), float("nan"), device="cuda", dtype=t.dtype)
    b[..., :-8] = t
    return b[..., :-8]


# K-tiles of 64 on the large tiles: 7, 9, 13 and 23, the last one of 8 to 56 k
@pytest.mark.parametrize("K", [392, 424, 552, 776, 1416])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_large_tiles_end_inside_a_k_tile(dtype, K):
    """All three products of a layer whose sums are K long, on the large tiles, with NaN beside every row."""
    dt, T, wide, sizes = DT[dtype], 4096, 2048, [2100, 1996]

    ends = _ends(sizes)
    # y = x @ w, column-major weights
    x, w = _data(T, K, wide, 2, dt, colmajor=True)
    got = ops.grouped_matmul(_beside_nan(x), _beside_nan(w.transpose(1, 2)).transpose(1, 2), ends)
    _close(got, _rows_exact(x, w, ends), _rows_exact(x.abs(), w.abs(), ends), K)
    # dx = dy @ w^T, row-major weights of K columns; dw of K columns
    x, w = _data(T, wide, K, 2, dt)
    dy, _ = _data(T, K, 1, 1, dt, seed=3)
    xs, ws = _beside_nan(x).requires_grad_(), _beside_nan(w).requires_grad_()
    dx, dw = torch.autograd.grad(ops.native_grouped_matmul(xs, ws, ends), (xs, ws), _beside_nan(dy))
    wt = w.transpose(1, 2)
    _close(dx, _rows_exact(dy, wt, ends), _rows_exact(dy.abs(), wt.abs(), ends), K)
    _close(dw, _reduce_exact(x, dy, ends), _reduce_exact(x.abs(), dy.abs(), ends), max(sizes))


def test_an_infinite_weight_stays_in_its_column_of_the_large_tiles():
    T, K, N = 4096, 424, 2048
    x, w = _data(T, K, N, 2, torch.bfloat16, colmajor=True)
    ends = _ends([2000, 2096])
    clean = ops.grouped_matmul(x, w, ends)
    w[1, :56, 700] = float("inf")  # contiguous columns: right behind column 699's last k
    y = ops.grouped_matmul(x, w, ends)
    assert not bool(y[2000:, 700].isfinite().any())
    y[2000:, 700] = clean[2000:, 700]
    assert torch.equal(y, clean)


@pytest.mark.parametrize("K", [520, 1416])
def test_large_tiles_of_ragged_experts_end_inside_a_k_tile(K):
    """Tiles of several experts in one stream: the K-tile that ends a sum is fetched while the tile before it,
    another expert's, is multiplied."""
    sizes = [700, 0, 513, 1, 900, 1100, 300]
    x, w = _data(sum(sizes) + 30, K, 2568, len(sizes), torch.bfloat16, colmajor=True)
    x[sum(sizes):] = float("nan")
    ends = _ends(sizes)
    y = ops.grouped_matmul(x, _beside_nan(w.transpose(1, 2)).transpose(1, 2), ends)
    x[sum(sizes):] = 0
    _close(y, _rows_exact(x, w, ends), _rows_exact(x.abs(), w.abs(), ends), K)


@pytest.mark.parametrize("T,M,N", [(9, 24, 40), (1500, 264, 520), (9, 1, 40), (9, 24, 1)])
def test_weight_gradients_into_interleaved_matrices(T, M, N):
    """out[e] as rows e, e + E, ... of one matrix: rows apart that do not overlap."""
    x, _ = _data(T, M, 1, 1, torch.bfloat16)
    dy, _ = _data(T, N, 1, 1, torch.bfloat16, seed=5)
    ends = _ends([T // 2, 0, T - T // 2])
    buf = torch.full((M, 3, N + 3), 5.0, device="cuda", dtype=torch.bfloat16)
    out = buf[:, :, :N].transpose(0, 1)
    assert ops.grouped_weight_grad(x, dy, ends, out=out) is out
    assert torch.equal(out, ops.grouped_weight_grad(x, dy, ends)) and bool((buf[:, :, N:] == 5).all())
    with pytest.raises(ValueError, match="overlap"):
        ops.grouped_weight_grad(x, dy, ends, out=out[:1].expand(3, M, N))
    if M > 1 and N > 1:
        with pytest.raises(ValueError, match="overlap"):  # matrices one row apart
            ops.grouped_weight_grad(x, dy, ends, out=buf.view(-1).as_strided((3, M, N), (N, N, 1)))


def test_forward_mode_tangents_are_refused():
    x, w, ends = torch.randn(4, 32, device="cuda"), torch.randn(2, 32, 8, device="cuda"), _ends([1, 3])
    q, s, z = ops.int4_quantize(w[0].half(), 32)
    leaf = x.clone().requires_grad_()
    y = ops.native_grouped_matmul(leaf, w, ends)
    with fwAD.dual_level():
        def dual(t):
            return fwAD.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.grouped_matmul(dual(x), w, ends), lambda: ops.grouped_matmul(x, dual(w), ends),
                     lambda: ops.grouped_weight_grad(dual(x), x, ends), lambda: ops.grouped_weight_grad(x, dual(x), ends),
                     lambda: ops.grouped_matmul(x, w, ends, out=dual(torch.zeros(4, 8, device="cuda"))),
                     lambda: ops.int4_matmul(dual(x.half()), q, s, z), lambda: ops.int4_matmul(x.half(), q, dual(s), z),
                     lambda: ops.native_grouped_matmul(dual(x), w, ends),
                     lambda: torch.autograd.grad(y, leaf, dual(torch.ones_like(y)), retain_graph=True)):
            with pytest.raises(RuntimeError, match="forward.mode|jvp"):
                call()
        assert ops.grouped_matmul(x, w, ends).shape == (4, 8)


def _far(t, at=3):
    """t with its last dimension's rows more than 8 MB apart, at an odd element, NaN between them."""
    b = torch.full((*t.shape[:-1], (1 << 23) // t.element_size() + 9), float("nan"), device="cuda", dtype=t.dtype)
    b[..., at:at + t.shape[-1]] = t
    return b[..., at:at + t.shape[-1]]


# from few rows to many, short sums and long ones (which several sets of waves share)
@pytest.mark.parametrize("sizes,K,N", [
    ([2, 0, 3], 70, 40), ([1], 1, 3), ([2, 0, 3], 1101, 37), ([20, 0, 13], 2056, 40), ([40, 0, 50], 1101, 37),
    ([100, 50, 70], 1101, 136), ([100, 50, 70], 201, 37), ([600, 700], 130, 40)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_rows_far_apart(dtype, sizes, K, N):
    """Strides past 8 MB, which are read by the element at the edges: of the rows, of the weights in both
    layouts, of what the weights' gradient sums."""
    T, E, ends = sum(sizes) + 2, len(sizes), _ends(sizes)
    x, w = _data(T, K, N, E, DT[dtype])
    dy, _ = _data(T, N, 1, 1, DT[dtype], seed=3)
    x[T - 2:], dy[T - 2:] = float("nan"), float("inf")
    x0, dy0 = x.nan_to_num(), dy.nan_to_num(posinf=0)
    want = _rows_exact(x0, w, ends), _rows_exact(x0.abs(), w.abs(), ends), K
    if T <= 300:
        _close(ops.grouped_matmul(_far(x), w, ends), *want)
        _close(ops.grouped_weight_grad(_far(x), _far(dy), ends), _reduce_exact(x0, dy0, ends),
               _reduce_exact(x0.abs(), dy0.abs(), ends), max(sizes))
    if K <= 300:
        _close(ops.grouped_matmul(x, _far(w), ends), *want)
    _close(ops.grouped_matmul(x, _far(w.transpose(1, 2)).transpose(1, 2), ends), *want)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_rows_and_long_gradients_far_apart(dtype):
    x, w = _data(6000, 72, 1200, 1, DT[dtype])
    ends = _ends([5990])
    y = ops.grouped_matmul(x, _far(w.transpose(1, 2)).transpose(1, 2), ends)
    _close(y, _rows_exact(x, w, ends), _rows_exact(x.abs(), w.abs(), ends), 72)
    x, _ = _data(1700, 40, 1, 1, DT[dtype])
    dy, _ = _data(1700, 70, 1, 1, DT[dtype], seed=3)
    ends = _ends([1000, 650])
    _close(ops.grouped_weight_grad(_far(x), dy, ends), _reduce_exact(x, dy, ends),
           _reduce_exact(x.abs(), dy.abs(), ends), 1000)
    both, out = w[:, :70, :40].expand(2, -1, -1), torch.full((1700, (1 << 23) // x.element_size() + 9), 2.0,
                                                            device="cuda", dtype=DT[dtype])[:, 1:41]
    ops.grouped_matmul(dy, both, ends, out=out)
    assert torch.equal(out[:1650], ops.grouped_matmul(dy, both, ends)[:1650]) and bool((out[1650:] == 2).all())


@pytest.mark.parametrize("derive", [lambda w: w.transpose(1, 2), lambda w: w.bfloat16().transpose(1, 2),
                                    lambda w: (w * 2).transpose(1, 2)], ids=["view", "cast", "computed"])
def test_capture_beside_a_living_eager_graph_of_what_an_operand_comes_from(derive):
    """A weight that is used through a view or a cast: the leaf behind it decides."""
    leaf = torch.randn(2, 24, 16, device="cuda", requires_grad=True)
    ends = torch.tensor([2, 4], device="cuda")
    x = torch.randn(4, 16, device="cuda").to(derive(leaf.detach()).dtype)
    alive = ops.native_grouped_matmul(x, derive(leaf), ends)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.native_grouped_matmul(x, derive(leaf), ends)
    eager = derive(leaf)
    del alive
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="still alive"):  # the operand's own graph, from before the capture
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.native_grouped_matmul(x, eager, ends)
    del eager
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.native_grouped_matmul(x, derive(leaf), ends)
        torch.autograd.grad(y, leaf, torch.ones_like(y))
        del y
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.native_grouped_matmul(x, derive(leaf), ends)
        (dw,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    for i in range(3):
        with torch.no_grad():
            leaf.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        again = leaf.detach().clone().requires_grad_()
        want = ops.native_grouped_matmul(x, derive(again), ends)
        assert torch.equal(y, want)
        assert torch.equal(dw, torch.autograd.grad(want, again, torch.ones_like(want))[0])
