"""4-bit products under ``torch.autocast``: what F.linear does there to a dense BF16 weight."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def pkg():
    import bf16_huffman_infer_b200
    return bf16_huffman_infer_b200


def normal(*shape, seed=0, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_inputs_are_cast(pkg, rows, dtype):
    w = pkg.MXFP4Weight.compress(normal(96, 256, std=0.1), to_cpu=False)
    x, bias, dy = normal(rows, 256, seed=1, dtype=dtype), normal(96, seed=2), normal(rows, 96, seed=3, dtype=torch.bfloat16)
    layer = pkg.CompressedLinear(w, nn.Parameter(bias))
    gated = pkg.GatedMXFP4(w, nn.Parameter(bias), "silu")
    low, low_bias = x.to(torch.bfloat16), bias.to(torch.bfloat16)
    calls = [(lambda v: F.linear(v, w, bias), lambda v: F.linear(v, w, low_bias), dy), (layer, lambda v: F.linear(v, w, low_bias), dy),
             (lambda v: pkg.gated_mxfp4(v, w, bias, "gelu"), lambda v: pkg.gated_mxfp4(v, w, low_bias, "gelu"), dy[:, :48]),
             (gated, lambda v: pkg.gated_mxfp4(v, w, low_bias), dy[:, :48])]
    for call, plain, g in calls:
        leaf, want_leaf = x.clone().requires_grad_(), low.clone().requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = call(leaf)
        want = plain(want_leaf)
        assert y.dtype == torch.bfloat16 and torch.equal(y, want)
        dx, = torch.autograd.grad(y, leaf, g)
        assert dx.dtype == dtype and torch.equal(dx, torch.autograd.grad(want, want_leaf, g)[0].to(dtype))


def test_other_types_are_refused(pkg):
    w = pkg.MXFP4Weight.compress(normal(96, 256, std=0.1), to_cpu=False)
    x = normal(3, 256)
    for call in (lambda v: F.linear(v, w), lambda v: pkg.gated_mxfp4(v, w)):
        with pytest.raises(AssertionError):
            call(x)
        with torch.autocast("cuda", dtype=torch.float16), pytest.raises(AssertionError):
            call(x)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            for bad in (x.double(), x.int(), x.cpu()):
                with pytest.raises(AssertionError):
                    call(bad)


def test_gated_pair_refuses_other_derivatives(pkg):
    w = pkg.MXFP4Weight.compress(normal(96, 256, std=0.1), to_cpu=False)
    x, t = normal(3, 256, dtype=torch.bfloat16), normal(3, 256, seed=1, dtype=torch.bfloat16)
    for call in (lambda: torch.func.jvp(lambda v: pkg.gated_mxfp4(v, w), (x,), (t,)), lambda: torch.func.vmap(lambda v: pkg.gated_mxfp4(v, w))(x),
                 lambda: torch.func.grad(lambda v: pkg.gated_mxfp4(v, w).float().sum())(x)):
        with pytest.raises(RuntimeError):
            call()
