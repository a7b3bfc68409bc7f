"""Checkpoints with 4-bit layers into skeletons of any type and initialisation, on the host."""
import copy

import pytest
import torch
from torch import nn

from bf16_huffman_infer_b200 import CompressedLinear, GatedMLP, GatedMXFP4, MXFP4Weight, load_compressed, save_compressed
from test_mxfp4_blocks import Block, Clamped, filled


def weight(M, K, seed):
    g = torch.Generator().manual_seed(seed)
    return MXFP4Weight.from_packed(torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g),
                                   torch.randint(110, 130, (M, K // 32), dtype=torch.uint8, generator=g))


def bias(n):
    return nn.Parameter(torch.arange(n).to(torch.bfloat16), requires_grad=False)


class Model(nn.Module):
    def __init__(self, block=Block, act=None, **factory):
        super().__init__()
        self.mlp = block(act, bias=True, **factory)
        self.out = nn.Linear(64, 40, **{"dtype": torch.bfloat16, **factory})
        self.norm = nn.LayerNorm(64, **{"dtype": torch.bfloat16, **factory})


@pytest.fixture
def saved(tmp_path):
    model = Model()
    model.mlp = GatedMLP(GatedMXFP4(weight(192, 64, 1), bias(192), "silu"), CompressedLinear(weight(64, 96, 2), bias(64)))
    model.out = CompressedLinear(weight(40, 64, 3), bias(40))
    path = str(tmp_path / "model.safetensors")
    save_compressed(model, path)
    return model, path


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("fill", [None, 0.0, float("nan")])
def test_skeletons_of_any_type(saved, dtype, fill):
    model, path = saved
    skeleton = Model(dtype=dtype).eval()
    loaded = load_compressed(skeleton if fill is None else filled(skeleton, fill), path)
    assert isinstance(loaded.mlp, GatedMLP) and not loaded.mlp.training and not loaded.mlp.gate_up.training
    want = {k: v for k, v in model.state_dict().items() if not k.startswith("norm")}
    for k, v in want.items():
        got = loaded.state_dict()[k]
        assert got.dtype == v.dtype and torch.equal(got, v), k   # biases among them: the products take BF16 ones
    assert loaded.norm.weight.dtype == dtype


def test_skeleton_without_storage(saved):
    model, path = saved
    with torch.device("meta"):
        skeleton = Model()
    skeleton.norm = copy.deepcopy(model.norm)
    loaded = load_compressed(skeleton, path)
    assert all(not t.is_meta and torch.equal(t, model.state_dict()[k]) for k, t in loaded.state_dict().items())


def test_skeletons_of_another_block(saved):
    _, path = saved
    for skeleton in (Model(Clamped), Model(Clamped, dtype=torch.float32), filled(Model(Clamped), 0.0), Model(act=nn.GELU())):
        before = dict(skeleton.named_modules())
        with pytest.raises(ValueError):
            load_compressed(skeleton, path)
        assert dict(skeleton.named_modules()) == before
