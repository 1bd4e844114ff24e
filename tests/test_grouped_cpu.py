"""Expert-grouped and 4-bit products without a GPU: refusals, the CPU path, the
quantiser's error bound, gradients against differences."""
import pytest
import torch

from pytorch_distributed_matmul_benchmark_amd import ops


def _ends(*sizes, dtype=torch.int32):
    return torch.tensor(sizes).cumsum(0).to(dtype)


def _exact(x, w, ends):
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64)
    lo = 0
    for e, hi in enumerate(ends.tolist()):
        y[lo:hi] = x[lo:hi].double() @ w[e].double()
        lo = hi
    return y


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cpu_path_matches_the_definition(dtype):
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(9, 5, generator=g).to(dtype), torch.randn(4, 5, 3, generator=g).to(dtype)
    ends = _ends(2, 0, 5, 1)  # an empty expert, one row behind the last
    y = ops.grouped_matmul(x, w, ends)
    # 5 products: the sum is off by at most 6 fp32 steps of the sum of magnitudes, then one rounding
    bound = 6 * 2.0 ** -23 * _exact(x.abs(), w.abs(), ends) + torch.finfo(dtype).eps / 2 * _exact(x, w, ends).abs()
    assert bool(((y.double() - _exact(x, w, ends)).abs() <= bound * 1.01).all())
    assert bool((y[8:] == 0).all())
    out = torch.full_like(y, 7.0)
    assert ops.grouped_matmul(x, w, ends, out=out) is out
    assert torch.equal(out[:8], y[:8]) and bool((out[8:] == 7).all())
    dw = ops.grouped_weight_grad(x, y, ends)
    assert dw.shape == w.shape and bool((dw[1] == 0).all())


def test_ends_outside_the_rows_are_held_inside():
    x, w = torch.randn(4, 3), torch.randn(3, 3, 2)
    y = ops.grouped_matmul(x, w, torch.tensor([-5, 2, 99]))
    assert torch.allclose(y[:2], x[:2] @ w[1]) and torch.allclose(y[2:], x[2:] @ w[2])


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(7, 4, generator=g, requires_grad=True)
    w = torch.randn(3, 6, 4, generator=g).transpose(1, 2).detach().requires_grad_()  # column-major
    c = torch.randn(7, 6, generator=g)
    ends = _ends(3, 0, 3)
    dx, dw = torch.autograd.grad((ops.native_grouped_matmul(x, w, ends) * c).sum(), (x, w))
    assert dw.stride() == w.stride() and bool((dx[6:] == 0).all()) and bool((dw[1] == 0).all())
    for leaf, grad in ((x, dx), (w, dw)):
        d = torch.randn(leaf.shape, generator=g)
        lo, hi = ((leaf.detach() + s * d) for s in (-0.5, 0.5))
        f = [(_exact(v, w.detach(), ends) if leaf is x else _exact(x.detach(), v, ends)) for v in (lo, hi)]
        diff = ((f[1] - f[0]) * c.double()).sum()  # exact: the product is linear in each factor
        # <= 42 products of <= 4 terms, each within a few fp32 steps of values below 50
        assert abs((grad.double() * d.double()).sum() - diff) < 42 * 8 * 2.0 ** -24 * 50


def test_a_shared_weight_sums_its_gradients():
    w = torch.randn(1, 4, 3, requires_grad=True)
    x = torch.randn(5, 4)
    y = ops.native_grouped_matmul(x, w.expand(2, 4, 3), _ends(2, 3))
    (dw,) = torch.autograd.grad(y.sum(), w)
    assert torch.allclose(dw[0], x.t() @ torch.ones(5, 3), atol=1e-5)


X, W, E = torch.zeros(4, 32), torch.zeros(2, 32, 8), torch.tensor([1, 4], dtype=torch.int32)


@pytest.mark.parametrize("err,call", [
    (ValueError, lambda: ops.grouped_matmul(X[0], W, E)),
    (ValueError, lambda: ops.grouped_matmul(X, W[0], E)),
    (ValueError, lambda: ops.grouped_matmul(X[:, :9], W, E)),
    (ValueError, lambda: ops.grouped_matmul(X, W[:0], E[:0])),
    (ValueError, lambda: ops.grouped_matmul(X, W, E[:1])),
    (ValueError, lambda: ops.grouped_matmul(X, W, E[None])),
    (TypeError, lambda: ops.grouped_matmul(X, W, E.float())),
    (TypeError, lambda: ops.grouped_matmul(X, W, [1, 4])),
    (TypeError, lambda: ops.grouped_matmul(X, W.half(), E)),
    (TypeError, lambda: ops.grouped_matmul(X.double(), W.double(), E)),
    (ValueError, lambda: ops.grouped_matmul(X, W, E, out=torch.zeros(4, 9))),
    (ValueError, lambda: ops.grouped_matmul(X, W, E, out=torch.zeros(4, 8).half())),
    (RuntimeError, lambda: ops.grouped_matmul(X.clone().requires_grad_(), W, E)),
    (ValueError, lambda: ops.grouped_weight_grad(X, X[:3], E)),
    (ValueError, lambda: ops.grouped_weight_grad(X, X[0], E)),
    (TypeError, lambda: ops.grouped_weight_grad(X, X.half(), E)),
    (ValueError, lambda: ops.grouped_weight_grad(X, X, E[:0])),
    (ValueError, lambda: ops.grouped_weight_grad(X, X, E, out=torch.zeros(2, 32, 31))),
    (RuntimeError, lambda: ops.grouped_weight_grad(X, X.clone().requires_grad_(), E)),
])
def test_grouped_refusals(err, call):
    with pytest.raises(err):
        call()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 256])
def test_quantise_round_trip(group, symmetric):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(2, 256, 5, generator=g).half()
    w[0, :32] = 0  # an all-zero group
    q, scale, zero = ops.int4_quantize(w, group, symmetric)
    assert q.shape == (2, 5, 128) and scale.shape == (2, 5, 256 // group) and (zero is None) == symmetric
    back = ops.int4_dequantize(q, scale, zero)
    # half a step, and what rounding the scale to fp16 leaves at the range's end (15 steps of
    # 2^-11), plus half a step for a rounded zero point that the range's ends are cut by
    step = scale.float().repeat_interleave(group, -1).transpose(-1, -2)
    allowed = step * (0.5 + 15 * 2.0 ** -11 + (0.0 if symmetric else 0.5))
    assert bool(((back - w.float()).abs() <= allowed * 1.001).all())
    # even k in the low half
    assert int(q[1, 3, 7] & 15) == int((back[1, 14, 3] / scale[1, 3, 14 // group]).round()
                                       + (8 if symmetric else zero[1, 3, 14 // group]))


def test_int4_cpu_path():
    g = torch.Generator().manual_seed(4)
    w = torch.randn(3, 64, 6, generator=g).bfloat16()
    q, s, z = ops.int4_quantize(w, 32)
    x = torch.randn(5, 64, generator=g).bfloat16()
    full = ops.int4_dequantize(q, s, z).double()
    y = ops.int4_matmul(x, q[1], s[1], z[1])
    ref = x.double() @ full[1]
    assert bool(((y.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 70 * 2.0 ** -23 * (x.double().abs() @ full[1].abs())).all())
    ends = _ends(1, 0, 3)
    y = ops.int4_matmul(x, q, s, z, ends=ends)
    assert torch.equal(y[1:4], ops.int4_matmul(x[1:4], q[2], s[2], z[2])) and bool((y[4:] == 0).all())


def _q():
    return ops.int4_quantize(torch.randn(64, 8).half(), 32)


@pytest.mark.parametrize("err,call", [
    (TypeError, lambda q, s, z, x: ops.int4_matmul(x.float(), q, s, z)),
    (TypeError, lambda q, s, z, x: ops.int4_matmul(x.bfloat16(), q, s, z)),
    (TypeError, lambda q, s, z, x: ops.int4_matmul(x, q.int(), s, z)),
    (TypeError, lambda q, s, z, x: ops.int4_matmul(x, q, s, z.int())),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x[0], q, s, z)),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x[:, :32], q, s, z)),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q, s[:4], z)),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q, s, z[:, :1])),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q, torch.cat((s, s), 1), None)),  # groups of 16
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q[None], s[None], z[None])),  # experts without ends
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q, s, z, ends=torch.tensor([2]))),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q[None], s[None], z[None], ends=torch.tensor([1, 2]))),
    (ValueError, lambda q, s, z, x: ops.int4_matmul(x, q, s, z, out=torch.zeros(2, 9).half())),
    (RuntimeError, lambda q, s, z, x: ops.int4_matmul(x.requires_grad_(), q, s, z)),
    (ValueError, lambda q, s, z, x: ops.int4_quantize(torch.zeros(64, 8).half(), 48)),
    (ValueError, lambda q, s, z, x: ops.int4_quantize(torch.zeros(96, 8).half(), 64)),
    (ValueError, lambda q, s, z, x: ops.int4_quantize(torch.zeros(192, 8).half(), 192)),
    (TypeError, lambda q, s, z, x: ops.int4_quantize(torch.zeros(64, 8), 32)),
])
def test_int4_refusals(err, call):
    q, s, z = _q()
    with pytest.raises(err):
        call(q, s, z, torch.zeros(2, 64).half())
