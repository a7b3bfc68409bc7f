"""The forms of the product of few rows that large weights and long rows take (two tiles of the weight a step, X in several chunks), against
plain computations in 64 bits.  Tolerances: an output is its 32-bit sum rounded to BF16 once, off by at most 2^-8 of itself and K 2^-23 of the
sum of its terms' magnitudes."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def pkg():
    import bf16_huffman_infer_b200
    return bf16_huffman_infer_b200


def weight(pkg, M, K):
    g = torch.Generator(device=DEV).manual_seed(M + K)
    return pkg.MXFP4Weight.from_packed(torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g, device=DEV),
                                       torch.randint(112, 121, (M, K // 32), dtype=torch.uint8, generator=g, device=DEV))


def normal(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(torch.bfloat16)


def sums(x, w, bias):
    """(sums, sums of the terms' magnitudes) in 64 bits, some rows of the weight at a time"""
    parts = [p.double() for p in w.get_weight().split(4096)]
    x, bias = x.double(), bias.double()
    return torch.cat([x @ p.T for p in parts], 1) + bias, torch.cat([x.abs() @ p.abs().T for p in parts], 1) + bias.abs()


# two CTAs an SM where rows * K is at most 8192, one beyond; odd numbers of tiles, M not a multiple of 16
@pytest.mark.parametrize("rows", [1, 3, 8])
@pytest.mark.parametrize("M,K", [(37888, 96), (37888, 2080), (45003, 96), (45003, 416), (45003, 2080), (40009, 8224)])
def test_two_tiles_a_step(pkg, M, K, rows):
    w, x, bias = weight(pkg, M, K), normal(rows, K, seed=rows), normal(M, seed=3)
    want, mag = sums(x, w, bias)
    for y, z in ((F.linear(x, w, bias), want), (F.linear(x, w), want - bias.double())):
        assert bool(((y.double() - z).abs() <= z.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23)).all())


@pytest.mark.parametrize("rows,M,K", [(8, 37889, 14336), (7, 38005, 18944), (8, 1000, 18944), (5, 530, 40000), (16, 23700, 14336), (24, 23700, 8224)])
def test_x_in_several_chunks(pkg, rows, M, K):
    w, x, bias = weight(pkg, M, K), normal(rows, K, seed=rows), normal(M, seed=3)
    want, mag = sums(x, w, bias)
    assert bool(((F.linear(x, w, bias).double() - want).abs() <= want.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23)).all())


@pytest.mark.parametrize("rows,inter,K", [(8, 520, 18944), (8, 521, 18944), (6, 1300, 40000), (16, 12000, 14336), (20, 12001, 8224)])
def test_gated_with_x_in_several_chunks(pkg, rows, inter, K):
    w, x, bias = weight(pkg, 2 * inter, K), normal(rows, K, seed=rows) * 2.0 ** -8, normal(2 * inter, seed=3)
    want, mag = sums(x, w, bias)
    pre = torch.empty(rows, 2 * inter, device=DEV)
    h = pkg.ops.gated_mxfp4(x, w.codes, w.scales, 2 * inter, bias, 0, pre)
    assert torch.equal(h, pkg.gated_mxfp4(x, w, bias))
    assert bool(((pre.double() - want).abs() <= mag * (K * 2.0 ** -23)).all())
    g, u = pre.double().chunk(2, -1)                             # from the projections as they are: a rounding, some units of 2^-23 in silu
    want = g * torch.sigmoid(g) * u
    assert bool(((h.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** -100).all())
