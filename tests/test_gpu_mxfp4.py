"""4-bit microscaled weights on the device, against plain computations in 64 bits.

Tolerances.  A BF16 output is the exact value rounded once: off by at most 2^-8 of it, so the 2-norm of all errors is below 2^-8
of the outputs' (the sums' own errors are far below that for the inputs here).  A single output may also be off by its 32-bit sum:
K additions that lose at most 2^-23 each of the sum of the terms' magnitudes.  A gradient through the gated pair is
rounded twice (the projections' gradients, which feed the product, and the result): 2^-7."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from _util import Abi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


@pytest.fixture(scope="module")
def pkg():
    import bf16_huffman_infer_b200
    return bf16_huffman_infer_b200


def normal(*shape, seed=0, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def plain_quantised(a):
    """The format's values of a matrix, by distance to the grid in double precision (ties to the even code), and its scale bytes."""
    v = a.double().cpu().view(a.shape[0], -1, 32)
    top = v.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top).exponent - 1 - 2, -127).clamp(min=-127)
    q = torch.ldexp(v.abs(), -e).clamp(max=6)
    dist = (q[..., None] - GRID).abs()
    # of two codes at the same distance the even one comes first in this order
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[dist[..., order].argmin(-1)]
    value = torch.ldexp(GRID[code], e) * torch.where(torch.signbit(v), -1.0, 1.0)
    return value.view(a.shape), (e + 127).squeeze(-1).to(torch.uint8)


def made(pkg, M, K, seed=0, std=0.02):
    """(weight, its dense values in 64 bits)"""
    w = pkg.MXFP4Weight.compress(normal(M, K, seed=seed, std=std), to_cpu=False)
    return w, w.get_weight().double()


def close(y, want, magnitudes, K):
    """Each output within a rounding and its sum's error, and all of them within a rounding by the 2-norm."""
    err = (y.double() - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + magnitudes * (K * 2.0 ** -23)).all()), float((err - want.abs() * 2.0 ** -8).max())
    assert float(err.norm()) <= 2.0 ** -8 * float(want.norm()) + 1e-30
    return True


SHAPES = [(1, 32), (16, 128), (17, 96), (130, 512), (250, 2080), (1024, 4096), (300, 18944)]
ROWS = [1, 2, 3, 5, 8, 9, 16, 17, 32, 33, 48, 64, 100, 128, 129, 200, 257, 700]


# ---- quantisation ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", SHAPES[:6])
def test_quantised_values(pkg, M, K, dtype):
    a = normal(M, K, std=0.02, dtype=dtype)
    w = pkg.MXFP4Weight.compress(a, to_cpu=False)
    value, byte = plain_quantised(a)
    assert torch.equal(w.get_weight().double().cpu(), value)
    assert torch.equal(w.packed()[1].cpu(), byte)
    codes, scales = w.packed()
    again = pkg.MXFP4Weight.from_packed(codes, scales)
    assert torch.equal(again.codes, w.codes) and torch.equal(again.scales, w.scales)      # padding included
    assert all(torch.equal(x, y.cpu()) for x, y in zip(pkg.MXFP4Weight.compress(a.cpu()).buffers(), w.buffers()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantisation_at_the_edges(pkg, dtype):
    """Every midpoint and its neighbours, both signs, at scales down to the smallest and up to the largest; zeros and blocks of zeros."""
    marks = torch.tensor([0, 0.125, 0.25, 0.375, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.5], dtype=torch.float64)
    info = torch.finfo(dtype)
    rows = []
    for e in ([-14, -3, 0, 12] if dtype == torch.float16 else [-133, -130, -127, -126, -124, -60, 0, 60, 124, 125]):
        for lead in (4.0, 6.0, 7.5):
            if lead * 2.0 ** e > info.max:
                continue
            row = torch.zeros(64, dtype=torch.float64)
            row[:19], row[19], row[32:51], row[51] = marks * 2.0 ** e, lead * 2.0 ** e, -marks * 2.0 ** e, -lead * 2.0 ** e
            rows.append(row.clamp(min=-lead * 2.0 ** e, max=lead * 2.0 ** e))
    a = torch.stack(rows + [torch.zeros(64, dtype=torch.float64)]).to(dtype)
    w = pkg.MXFP4Weight.compress(a.to(DEV), to_cpu=False)
    value, byte = plain_quantised(a)
    assert torch.equal(w.packed()[1].cpu(), byte)
    assert torch.equal(w.get_weight().double().cpu(), value)


def test_infinities_and_nans_make_their_block_nan(pkg):
    a = normal(20, 160, std=0.02)
    a[3, 40], a[7, 0], a[19, 159] = float("inf"), float("nan"), -float("inf")
    w = pkg.MXFP4Weight.compress(a, to_cpu=False)
    dense = w.get_weight().view(20, 5, 32)
    want = torch.zeros(20, 5, dtype=torch.bool, device=DEV)
    want[3, 1] = want[7, 0] = want[19, 4] = True
    assert torch.equal(dense.isnan().all(-1), want) and torch.equal(dense.isnan().any(-1), want)
    for rows in (1, 40):
        y = F.linear(normal(rows, 160, seed=1), w)
        assert torch.equal(y.isnan().all(0), want.any(1)) and torch.equal(y.isnan().any(0), want.any(1))


@pytest.mark.parametrize("M,K", SHAPES)
def test_plain_order_as_on_the_host(pkg, M, K):
    """Codes and scales of every value, NaN scales and padding among them; slices and odd addresses."""
    g = torch.Generator().manual_seed(M)
    codes = torch.randint(0, 256, (M + 2, K // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(0, 256, (M + 2, K // 32), dtype=torch.uint8, generator=g)
    scales[0, 0] = 255
    on = codes.to(DEV), scales.to(DEV)
    shifted = torch.empty(codes.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(codes.shape).copy_(codes)
    for part in (slice(0, M), slice(1, M + 1), slice(2, M + 2)):
        want = pkg.MXFP4Weight.from_packed(codes[part], scales[part])
        for c, s in (on, (shifted, on[1]), (on[0].T.contiguous().T, on[1].T.contiguous().T), (on[0], on[1].view(torch.float8_e8m0fnu))):
            got = pkg.MXFP4Weight.from_packed(c[part], s[part])
            assert torch.equal(got.codes.cpu(), want.codes) and torch.equal(got.scales.cpu(), want.scales)
    for c, s in ((on[0], scales), (codes, on[1])):
        with pytest.raises(RuntimeError):
            pkg.MXFP4Weight.from_packed(c, s)


def test_quantisation_of_other_layouts(pkg):
    a = normal(64, 256, std=0.02)
    want = pkg.MXFP4Weight.compress(a, to_cpu=False).get_weight()
    shifted = torch.empty(64 * 256 + 1, dtype=a.dtype, device=DEV)[1:].view(64, 256).copy_(a)
    for view in (a.T.contiguous().T, torch.cat([a, a], 1)[:, :256], shifted, nn_parameter(a)):
        assert torch.equal(pkg.MXFP4Weight.compress(view, to_cpu=False).get_weight(), want)
    for bad in (a.double(), a[0], a[:, :40], a[:0], a.int()):
        with pytest.raises((AssertionError, ValueError)):
            pkg.MXFP4Weight.compress(bad)


def nn_parameter(a):
    return torch.nn.Parameter(a.clone())


# ---- the product -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("M,K", SHAPES)
def test_product(pkg, M, K, rows):
    w, dense = made(pkg, M, K, seed=M + K)
    x, bias = normal(rows, K, seed=rows), normal(M, seed=3)
    mag = x.double().abs() @ dense.abs().T
    assert close(F.linear(x, w), x.double() @ dense.T, mag, K)
    assert close(F.linear(x, w, bias), x.double() @ dense.T + bias.double(), mag + bias.double().abs(), K)


@pytest.mark.parametrize("rows", [9, 13, 16])
@pytest.mark.parametrize("M,K", [(2100, 2080), (2101, 6880), (24003, 416), (23700, 7840), (6000, 12288)])
def test_nine_to_sixteen_rows(pkg, M, K, rows):
    """Weights that are large enough for the kernel of few rows: a few steps an SM and many, X in one piece and in several."""
    w, dense = made(pkg, M, K, seed=M + K, std=1.5 / math.sqrt(K))
    x, bias = normal(rows, K, seed=rows), normal(M, seed=3)
    mag = x.double().abs() @ dense.abs().T + bias.double().abs()
    want = x.double() @ dense.T + bias.double()
    assert close(F.linear(x, w, bias), want, mag, K)
    if M % 2 == 0:
        g, u = want.chunk(2, -1)
        want = act64(g, "gelu") * u
        pre = torch.empty(rows, M, device=DEV)
        h = pkg.ops.gated_mxfp4(x, w.codes, w.scales, M, bias, 1, pre)
        assert float((h.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
        assert bool(((pre.double() - torch.cat([g, u], -1)).abs() <= mag * (K * 2.0 ** -23)).all())


@pytest.mark.parametrize("rows", [17, 20, 24])
@pytest.mark.parametrize("M,K", [(24003, 416), (23700, 7840), (24002, 96)])
def test_seventeen_to_24_rows(pkg, M, K, rows):
    test_nine_to_sixteen_rows(pkg, M, K, rows)


@pytest.mark.parametrize("rows", [9, 16, 24])
@pytest.mark.parametrize("byte", [0, 60, 200, 240, 252])
def test_scales_of_the_whole_range_in_many_steps(pkg, byte, rows):
    g = torch.Generator().manual_seed(rows + byte)
    M, K = 45000, 96
    w = pkg.MXFP4Weight.from_packed(torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g).to(DEV), torch.full((M, K // 32), byte, dtype=torch.uint8, device=DEV))
    dense = w.get_weight().double()
    x = torch.ldexp(torch.randn(rows, K, generator=g).double(), torch.tensor(min(127 - byte, 120))).to(torch.bfloat16).to(DEV)
    want, mag = x.double() @ dense.T, x.double().abs() @ dense.abs().T
    assert bool(((F.linear(x, w).double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23) + K * 2.0 ** -134).all())


def test_product_of_other_layouts(pkg):
    w, dense = made(pkg, 130, 512)
    for rows in (3, 70):
        x = normal(rows, 512, seed=rows)
        want = F.linear(x, w)
        shifted = torch.empty(rows * 512 + 1, dtype=x.dtype, device=DEV)[1:].view(rows, 512).copy_(x)
        for view in (x.T.contiguous().T, torch.cat([x, x], 1)[:, 512:], shifted):
            assert torch.equal(F.linear(view, w), want)
        assert torch.equal(F.linear(x.view(1, rows, 1, 512), w), want.view(1, rows, 1, 130))
    assert torch.equal(F.linear(x[0], w), F.linear(x[:1], w)[0])
    assert F.linear(x[:0], w).shape == (0, 130) and F.linear(x.new_empty(2, 0, 512), w).shape == (2, 0, 130)
    one = normal(1, 512)
    assert torch.equal(F.linear(one.expand(40, 512), w), F.linear(one.repeat(40, 1), w))


@pytest.mark.parametrize("rows", [2, 40])
def test_values_far_apart(pkg, rows):
    """Rows of X and blocks of K whose magnitudes differ by many powers of two; scales from tiny to huge."""
    g = torch.Generator().manual_seed(rows)
    M, K = 48, 512
    codes = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(60, 200, (M, 1), dtype=torch.uint8, generator=g) + torch.randint(0, 9, (M, K // 32), dtype=torch.uint8, generator=g)
    w = pkg.MXFP4Weight.from_packed(codes.to(DEV), scales.to(DEV))
    dense = w.get_weight().double()
    x = torch.randn(rows, K, generator=g).double() * torch.exp2(torch.randint(-40, 20, (rows, 1), generator=g).double()) \
        * torch.exp2(torch.randint(-20, 1, (rows, K), generator=g).double())
    x = x.to(torch.bfloat16).to(DEV)
    want, mag = x.double() @ dense.T, x.double().abs() @ dense.abs().T
    err = (F.linear(x, w).double() - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23)).all())


@pytest.mark.parametrize("rows", [1, 4, 20, 70])
def test_infinities_and_nans_in_x(pkg, rows):
    w, dense = made(pkg, 64, 384)
    x = normal(rows, 384, seed=5)
    clean = F.linear(x, w)
    x[0, 130] = float("inf")
    if rows > 1:
        x[1, 7] = float("nan")
    y = F.linear(x, w)
    col = dense[:, 130]
    assert torch.equal(y[0].isnan(), col == 0) and torch.equal(y[0][col != 0], torch.where(col > 0, math.inf, -math.inf)[col != 0].to(y.dtype))
    if rows > 1:
        assert bool(y[1].isnan().all())
        assert torch.equal(y[2:], clean[2:])


@pytest.mark.parametrize("byte", [0, 1, 30, 126, 127, 128, 200, 231, 232, 240, 251, 252])
@pytest.mark.parametrize("rows", [1, 8, 9, 16, 33, 200])
def test_scales_of_the_whole_range(pkg, rows, byte):
    """One scale throughout, from the smallest to the largest whose values are finite, and X the other way: products near one."""
    g = torch.Generator().manual_seed(rows + byte)
    M, K = 150, 416
    codes = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g)
    w = pkg.MXFP4Weight.from_packed(codes.to(DEV), torch.full((M, K // 32), byte, dtype=torch.uint8, device=DEV))
    dense = w.get_weight().double()
    grid = torch.cat([GRID, -GRID])
    assert torch.equal(dense.cpu(), torch.ldexp(torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).view(M, K), torch.tensor(byte - 127)))
    x = torch.ldexp(torch.randn(rows, K, generator=g).double(), torch.tensor(min(127 - byte, 120))).to(torch.bfloat16).to(DEV)
    want, mag = x.double() @ dense.T, x.double().abs() @ dense.abs().T
    # and half of BF16's and the products' smallest steps, for terms that are below
    assert bool(((F.linear(x, w).double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23) + K * 2.0 ** -134).all())
    gate, up = want.chunk(2, -1)
    gate_mag, up_mag = mag.chunk(2, -1)
    # the sums' errors as above, through |act'| <= 1.1; the function's own error, a few units of 2^-23 of arguments up to 60 (where it is not small)
    slack = 1.1 * gate_mag * K * 2.0 ** -23 * (up.abs() + up_mag * K * 2.0 ** -23) + act64(gate, "silu").abs() * up_mag * K * 2.0 ** -23
    want = act64(gate, "silu") * up
    assert bool(((pkg.gated_mxfp4(x, w).double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -14) + slack + 2.0 ** -100).all())


@pytest.mark.parametrize("rows", [1, 8])
def test_sums_that_overflow(pkg, rows):
    """Few rows: outputs beyond the range are infinities of their sign, their neighbours (the other rows, the bias) are what they were."""
    M, K = 40, 4096
    g = torch.Generator().manual_seed(rows)
    codes = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g)
    scales = torch.full((M, K // 32), 120, dtype=torch.uint8)
    scales[::2, 40] = 250
    codes[::2, 40 * 16:41 * 16] = 0x11                           # 0.5 2^123 throughout a block
    w = pkg.MXFP4Weight.from_packed(codes.to(DEV), scales.to(DEV))
    x = torch.randn(rows, K, generator=g).to(torch.bfloat16)
    x[:, 40 * 32:41 * 32] = torch.tensor([2.0, -2.0] * rows).to(x.dtype)[:rows, None]      # 32 2^123 = 2^128
    x = x.to(DEV)
    y, bias = F.linear(x, w), normal(M, seed=3)
    assert torch.equal(y[:, ::2], torch.where(x[:, 40 * 32, None] > 0, math.inf, -math.inf).to(y.dtype).expand(rows, M // 2))
    dense = w.get_weight().double()[1::2]
    mag = x.double().abs() @ dense.abs().T
    assert bool(((y[:, 1::2].double() - x.double() @ dense.T).abs() <= (x.double() @ dense.T).abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23)).all())
    assert torch.equal(F.linear(x, w, bias)[:, ::2], y[:, ::2])


def test_refused_calls(pkg):
    w, _ = made(pkg, 64, 128)
    x = normal(2, 128)
    for bad in (x.float(), x.half(), x.cpu()):
        with pytest.raises(AssertionError):
            F.linear(bad, w)
    for bad in (x[:, :96], normal(2, 160), x.new_empty(())):
        with pytest.raises(RuntimeError):
            F.linear(bad, w)
    bias = normal(64)
    for bad in (bias[1:], bias.float(), bias.cpu(), bias[None], bias[0]):
        with pytest.raises(RuntimeError):
            F.linear(x, w, bad)
    with pytest.raises(ValueError):
        pkg.gated_mxfp4(x, w, activation="relu")
    odd, _ = made(pkg, 63, 128)
    with pytest.raises(RuntimeError):
        pkg.gated_mxfp4(x, odd)
    ops, pre = pkg.ops, torch.empty(2, 64, device=DEV)
    for bad in (lambda: ops.forward_mxfp4(x, w.codes[:3], w.scales, 64, None), lambda: ops.forward_mxfp4(x, w.codes, w.scales, 65, None),
                lambda: ops.forward_mxfp4(x, w.codes, w.scales, 64, bias[1:]), lambda: ops.forward_mxfp4(x.T, w.codes, w.scales, 64, None),
                lambda: ops.forward_mxfp4(x.view(-1)[1:129], w.codes, w.scales, 64, None), lambda: ops.mxfp4_quantize(x, w.codes, w.scales),
                lambda: ops.mxfp4_linear_grad(x[:, :60].contiguous(), w.codes, w.scales, 64, 128), lambda: ops.dense_mxfp4(w.codes, w.scales, 64, 100),
                lambda: ops.gated_mxfp4(x, w.codes, w.scales, 64, None, 3, None), lambda: ops.gated_mxfp4(x, w.codes, w.scales, 64, None, 0, pre[:1]),
                lambda: ops.mxfp4_gated_grad(pre, x, 0), lambda: ops.mxfp4_gated_grad(pre, x[:, :32].contiguous(), -1)):
        with pytest.raises(RuntimeError):
            bad()


# ---- its gradient --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 3, 9, 40, 129, 300])
@pytest.mark.parametrize("M,K", SHAPES)
def test_gradient_of_the_product(pkg, M, K, rows):
    w, dense = made(pkg, M, K, seed=M + K)
    x, bias = normal(rows, K, seed=rows).requires_grad_(), normal(M, seed=3).requires_grad_()
    y = F.linear(x, w, bias)
    assert torch.equal(y.detach(), F.linear(x.detach(), w, bias.detach()))
    dy = normal(rows, M, seed=9)
    dx, db = torch.autograd.grad(y, (x, bias), dy)
    assert close(dx, dy.double() @ dense, dy.double().abs() @ dense.abs(), M)
    assert close(db, dy.double().sum(0), dy.double().abs().sum(0), rows)


def test_gradient_by_differences(pkg):
    """(f(x + h) - f(x)) / h for the sum of squares / 2 of the outputs, in 64 bits outside the product."""
    w, dense = made(pkg, 96, 256)
    x = normal(12, 256, seed=2).requires_grad_()
    y = F.linear(x, w)
    dx, = torch.autograd.grad((y.float() ** 2).sum() / 2, x)

    def f(v):
        return float(((v @ dense.T) ** 2).sum() / 2)

    x0 = x.detach().double()
    g = torch.Generator().manual_seed(0)
    for _ in range(5):
        d = torch.randn(12, 256, generator=g).double().to(DEV)
        numeric = (f(x0 + 1e-4 * d) - f(x0 - 1e-4 * d)) / 2e-4
        # y and dx are rounded: each by at most 2^-8 of its norm
        assert abs(numeric - float((dx.double() * d).sum())) <= 2.0 ** -7 * float(dx.double().norm() * d.norm())


def test_gradients_of_views_and_broadcasts(pkg):
    w, dense = made(pkg, 72, 256)
    x = normal(1, 256, seed=2).requires_grad_()
    y = F.linear(x.expand(24, 256), w)
    y.sum().backward()                                           # dy is an expanded scalar
    want = dense.sum(0)
    assert float((x.grad[0].double() / 24 - want).norm()) <= 2.0 ** -7 * float(want.norm())        # the rows' gradients and their sum are rounded
    x = normal(4, 6, 256, seed=3).requires_grad_()
    F.linear(x, w).transpose(0, 1).contiguous().sum().backward()
    assert x.grad.shape == x.shape
    e = x.new_empty(0, 256).requires_grad_()
    F.linear(e, w).sum().backward()
    assert e.grad.shape == (0, 256)


def test_gradients_of_one_vector(pkg):
    w, dense = made(pkg, 72, 256)
    x, bias, dy = normal(256, seed=2), normal(72, seed=3), normal(72, seed=4)
    leaf, b = x.clone().requires_grad_(), bias.clone().requires_grad_()
    y = F.linear(leaf, w, b)
    assert torch.equal(y.detach(), F.linear(x[None], w, bias)[0])
    dx, db = torch.autograd.grad(y, (leaf, b), dy)
    assert torch.equal(db, dy) and close(dx, dy.double() @ dense, dy.double().abs() @ dense.abs(), 72)
    h = pkg.gated_mxfp4(leaf, w, b)
    dx, db = torch.autograd.grad(h, (leaf, b), dy[:36])
    many, bs = x[None].clone().requires_grad_(), bias.clone().requires_grad_()
    want = torch.autograd.grad(pkg.gated_mxfp4(many, w, bs), (many, bs), dy[None, :36])
    assert torch.equal(dx, want[0][0]) and torch.equal(db, want[1])


def test_other_derivatives(pkg):
    w, dense = made(pkg, 72, 256)
    x, t, bias = normal(5, 256), normal(5, 256, seed=1), normal(72, seed=2)
    layer = pkg.CompressedLinear(w, None)
    y, tangent = torch.func.jvp(layer, (x,), (t,))
    assert torch.equal(y, layer(x)) and torch.equal(tangent, layer(t))
    xs = torch.stack([x, t])
    assert torch.equal(torch.func.vmap(layer)(xs), layer(xs))
    assert torch.equal(torch.func.vmap(lambda v, b: F.linear(v, w, b), in_dims=(None, 0))(x, torch.stack([bias, -bias])),
                       torch.stack([F.linear(x, w, bias), F.linear(x, w, -bias)]))
    got = torch.func.grad(lambda v: layer(v).float().sum())(x)
    x.requires_grad_()
    dx, = torch.autograd.grad(layer(x).float().sum(), x, create_graph=True)
    assert torch.equal(got, dx.detach())
    # dx is linear in dy, which does not depend on x here; through a square it does
    y = layer(x)
    dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    ddx, = torch.autograd.grad(dx.float().sum(), x)
    want = 2 * (torch.ones(5, 256, device=DEV, dtype=torch.float64) @ dense.T) @ dense
    assert float((ddx.double() - want).norm()) <= 2.0 ** -6 * float(want.norm())                    # four roundings on the way


@pytest.mark.parametrize("wide,other", [(75 * 256, 512), (76 * 256 - 90, 2080), (2 * 74 * 256 + 256 * 20, 800)])
@pytest.mark.parametrize("rows", [30, 150])
def test_tiles_of_a_last_round(pkg, wide, other, rows):
    """A few tiles more than whole rounds over the pairs of SMs, forward (gated and not) and backward."""
    w, dense = made(pkg, wide, other, std=1.5 / math.sqrt(other))
    x = normal(rows, other, seed=rows)
    mag = x.double().abs() @ dense.abs().T
    want = x.double() @ dense.T
    assert close(F.linear(x, w), want, mag, other)
    g, u = want.chunk(2, -1)
    want = act64(g, "silu") * u
    assert float((pkg.gated_mxfp4(x, w).double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
    w, dense = made(pkg, other, wide // 32 * 32)
    dy = normal(rows, other, seed=rows + 1)
    assert close(pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, other, wide // 32 * 32), dy.double() @ dense, dy.double().abs() @ dense.abs(), other)


# ---- the gated pair --------------------------------------------------------------------------------------------------------
def act64(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    return F.gelu(g, approximate="tanh" if name == "gelu_tanh" else "none")


GATED = [(1, 32), (8, 128), (13, 96), (65, 512), (200, 2080), (1024, 1024), (50, 8192)]


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 33, 64, 130, 300])
@pytest.mark.parametrize("inter,K", GATED)
def test_gated(pkg, inter, K, rows, activation):
    w, dense = made(pkg, 2 * inter, K, seed=inter + K, std=1.5 / math.sqrt(K))
    x, bias, dh = normal(rows, K, seed=rows), normal(2 * inter, seed=3), normal(rows, inter, seed=4)
    for b in (None, bias):
        x64 = x.double().requires_grad_()
        b64 = None if b is None else b.double().requires_grad_()
        g, u = F.linear(x64, dense, b64).chunk(2, -1)
        want = act64(g, activation) * u
        h = pkg.gated_mxfp4(x, w, b, activation)
        assert float((h.double() - want.detach()).norm()) <= 2.0 ** -8 * float(want.detach().norm())
        leaf = x.clone().requires_grad_()
        bleaf = None if b is None else b.clone().requires_grad_()
        again = pkg.gated_mxfp4(leaf, w, bleaf, activation)
        assert torch.equal(again.detach(), h)
        leaves = [v for v in (leaf, bleaf) if v is not None]
        for got, ref in zip(torch.autograd.grad(again, leaves, dh), torch.autograd.grad(want, [v for v in (x64, b64) if v is not None], dh.double())):
            assert float((got.double() - ref).norm()) <= 2.0 ** -7 * float(ref.norm())


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [2, 40])
def test_gated_far_from_zero(pkg, rows, activation):
    """Gates from -60 to 60 and far beyond: neither overflow nor cancellation shows in value or gradient."""
    inter, K = 64, 128
    codes = torch.zeros(2 * inter, K // 2, dtype=torch.uint8)
    codes[:, 0] = 2                                              # element 0 has the code of 1
    w = pkg.MXFP4Weight.from_packed(codes.to(DEV), torch.full((2 * inter, K // 32), 127, dtype=torch.uint8, device=DEV))
    x = torch.zeros(rows, K, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = torch.linspace(-60, 60, rows, device=DEV).to(x.dtype)
    shift = torch.linspace(-30, 30, inter, device=DEV).to(x.dtype)
    bias = torch.cat([shift, torch.ones(inter, device=DEV, dtype=x.dtype)])
    x64 = x.double().requires_grad_()
    g, u = x64[:, :1] + bias[:inter].double(), x64[:, :1] + 1
    if activation == "gelu":
        want = g * torch.special.ndtr(g) * u
    elif activation == "gelu_tanh":
        want = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u
    else:
        want = g * torch.sigmoid(g) * u
    leaf = x.clone().requires_grad_()
    h = pkg.gated_mxfp4(leaf, w, bias, activation)
    err = (h.double() - want).abs().detach()
    # a rounding of the result; the function's own error, a few units of 2^-23 of arguments up to 90
    assert bool((err <= want.detach().abs() * (2.0 ** -8 + 2.0 ** -14) + 1e-12).all())
    dx, = torch.autograd.grad(h.float().sum(), leaf)
    ref, = torch.autograd.grad(want.sum(), x64)
    assert float((dx.double() - ref).norm()) <= 2.0 ** -7 * float(ref.norm())
    far = x.clone()
    far[:, 0] = torch.where(far[:, 0] < 0, -1e5, 1e5).to(far.dtype)
    assert bool(pkg.gated_mxfp4(far, w, bias, activation).isfinite().all())


def plain_activation(g, name):
    """act(g) and act'(g) in 64 bits, without cancellation for negative g."""
    if name == "gelu":
        s, ds = torch.special.erfc(-g / math.sqrt(2)) / 2, torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    else:
        k = 2 * math.sqrt(2 / math.pi)
        z, dz = (g, torch.ones_like(g)) if name == "silu" else (k * (g + 0.044715 * g ** 3), k * (1 + 3 * 0.044715 * g * g))
        s = torch.sigmoid(z)
        ds = s * torch.sigmoid(-z) * dz
    return g * s, s + g * ds


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_tails_of_the_activations(pkg, activation):
    """Where the exponential leaves the range of normal numbers, value by value."""
    lo = {"silu": -102.0, "gelu": -13.0, "gelu_tanh": -9.9}[activation]
    gates = torch.linspace(lo, 0, 97).to(torch.bfloat16)
    K = 32
    w = pkg.MXFP4Weight.from_packed(torch.tensor([[2] + [0] * 15, [32] + [0] * 15], dtype=torch.uint8, device=DEV),      # the first element, the second
                                    torch.full((2, 1), 127, dtype=torch.uint8, device=DEV))
    x = torch.zeros(97, K, dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = gates, 1
    want = plain_activation(gates.double(), activation)[0].to(DEV)
    few = torch.cat([pkg.gated_mxfp4(x[i:i + 8].to(DEV), w, None, activation) for i in range(0, 97, 8)])[:, 0].double()
    many = pkg.gated_mxfp4(x.to(DEV), w, None, activation)[:, 0].double()
    for got in (few, many):
        # a rounding (half a step of 2^-133 for the smallest); arguments up to 102 with a few units of 2^-24 of their own; a 32-bit exponential in steps of
        # 2^-149, times a gate up to 102
        assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** -134 + 2.0 ** -141).all()), (got, want)


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("inter", [64, 65])
def test_gradient_of_the_activations(pkg, inter, activation):
    g = torch.cat([torch.linspace(-30, 30, 2 * inter - 6), torch.tensor([-1e30, -1e20, -1e5, 1e5, 1e20, 1e30])]).view(2, inter).to(DEV)
    u, dh = normal(2, inter, seed=1, dtype=torch.float32), normal(2, inter, seed=2)
    dpre = pkg.ops.mxfp4_gated_grad(torch.cat([g, u], 1), dh, {"silu": 0, "gelu": 1, "gelu_tanh": 2}[activation])[:, :2 * inter].double()
    a, da = plain_activation(g.double(), activation)
    da = torch.where(g.abs() > 1e4, (g > 0).double(), da)         # the formula's limits, where it leaves 64 bits
    for got, want in ((dpre[:, :inter], dh.double() * u.double() * da), (dpre[:, inter:], dh.double() * a)):
        # a rounding; act' in 32 bits: terms up to 1.6 (9, gelu_tanh's inner derivative times g (1 - s)) with a few units of 2^-23, arguments up to 30
        assert bool(((got - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -14) + (dh.double() * u.double()).abs() * 2.0 ** -14 + 1e-30).all())


def test_gated_layouts_and_empties(pkg):
    w, dense = made(pkg, 80, 256, std=0.1)
    x = normal(2, 3, 256)
    h = pkg.gated_mxfp4(x, w)
    assert h.shape == (2, 3, 40) and torch.equal(pkg.gated_mxfp4(x.transpose(0, 1).contiguous().transpose(0, 1), w), h)
    assert pkg.gated_mxfp4(x[:0], w).shape == (0, 3, 40)
    e = x[:0].clone().requires_grad_()
    pkg.gated_mxfp4(e, w).sum().backward()
    assert e.grad.shape == e.shape
    leaf = x.clone().requires_grad_()
    pkg.gated_mxfp4(leaf, w).sum().backward()                    # an expanded scalar as gradient
    assert leaf.grad.shape == x.shape
    y = pkg.gated_mxfp4(leaf, w)
    dx, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


# ---- streams, graphs, launches --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 16, 40, 200])
def test_same_results_every_time(pkg, rows):
    w, _ = made(pkg, 1000, 4096)
    x = normal(rows, 4096).requires_grad_()
    y = F.linear(x, w)
    dx, = torch.autograd.grad(y, x, y.detach())
    for _ in range(5):
        again = F.linear(x, w)
        assert torch.equal(again, y) and torch.equal(torch.autograd.grad(again, x, y.detach())[0], dx)


def test_captured_and_on_two_streams(pkg):
    """Two graphs of a block's products, replayed on two streams at once and then on new inputs, against eager calls."""
    up, _ = made(pkg, 2 * 1000, 512, seed=1, std=0.05)
    down, _ = made(pkg, 512, 1024, seed=2, std=0.05)             # 1000 gated values padded by hand to a multiple of 32

    def block(x):
        h = F.pad(pkg.gated_mxfp4(x, up), (0, 24))
        return x + F.linear(h, down)

    graphs = []
    for rows in (2, 50):
        x = normal(rows, 512, seed=rows)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(block(x))
        graphs.append((graph, x, y, torch.cuda.Stream()))
    for seed in range(3):
        for _, x, _, _ in graphs:
            x.copy_(normal(*x.shape, seed=10 + seed))
        torch.cuda.synchronize()
        for graph, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
                graph.replay()
        torch.cuda.synchronize()
        for _, x, y, _ in graphs:
            assert torch.equal(y, block(block(x)))


def test_backward_in_a_graph(pkg):
    """A whole training step of a block's products captured, on another stream, and replayed on new inputs."""
    up, _ = made(pkg, 2 * 96, 256, seed=1, std=0.09)
    down, _ = made(pkg, 256, 96, seed=2, std=0.1)

    def step(x, dy):
        leaf = x.detach().requires_grad_()
        return torch.autograd.grad(F.linear(pkg.gated_mxfp4(leaf, up), down), leaf, dy)[0]

    for rows in (3, 150):
        x, dy = normal(rows, 256, seed=rows), normal(rows, 256, seed=rows + 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step(x, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            dx = step(x, dy)
        graph.replay()
        assert torch.equal(dx, eager)
        x.copy_(normal(rows, 256, seed=7))
        dy.copy_(normal(rows, 256, seed=8))
        graph.replay()
        assert torch.equal(dx, step(x, dy))


def test_no_wait_ran_out(pkg):
    """After products of every kind the kernels' status is clean."""
    abi, status = Abi(), ctypes.c_int(-1)
    abi.check(abi.lib.bhi_debug_status(ctypes.byref(status)))    # what earlier calls left
    w, _ = made(pkg, 600, 2048)
    for rows in (1, 8, 16, 17, 100, 400):
        x = normal(rows, 2048).requires_grad_()
        (F.linear(x, w).sum() + pkg.gated_mxfp4(x, w).sum()).backward()
    abi.check(abi.lib.bhi_debug_status(ctypes.byref(status)))
    assert status.value == 0


def test_results_are_whole_for_the_next_kernel(pkg):
    """A chain of products, each of which may start while the one before is still running, against the same with waits between."""
    ws = [made(pkg, 2048, 2048, seed=s, std=0.022)[0] for s in range(3)]
    x = normal(1, 2048)
    y = x
    for i in range(60):
        y = F.linear(y, ws[i % 3])
    z = x
    for i in range(60):
        z = F.linear(z, ws[i % 3])
        torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_first_call_of_a_thread(pkg):
    """A thread that has made no CUDA call of its own yet, as those of the autograd engine, on the tiled products."""
    import threading
    w, _ = made(pkg, 96, 256)
    x, dy = normal(64, 256), normal(64, 96)
    want = F.linear(x, w), pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, 96, 256)
    got, calls = {}, {
        "y": lambda: pkg.ops.forward_mxfp4(x, w.codes, w.scales, 96, None),
        "dx": lambda: pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, 96, 256),
    }
    for name, call in calls.items():
        def run(name=name, call=call):
            got[name] = call()
            torch.cuda.current_stream().synchronize()
        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
    assert torch.equal(got["y"], want[0]) and torch.equal(got["dx"], want[1])
