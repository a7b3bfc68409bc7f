"""A decoder with every linear layer rounded to 4-bit floats: against the same model over the rounded matrices, graphed, saved and
loaded, and with gradients flowing through its frozen weights."""
import copy

import pytest
import torch
from torch import nn

from test_gpu_model import _same_decoding, _tiny_model

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rounded(model, converted):
    """``model`` with the matrices that ``converted`` multiplies by."""
    from bf16_huffman_infer_b200 import CompressedLinear
    from bf16_huffman_infer_b200.functional import FusedCompressedLinear, _FusedSlice
    from bf16_huffman_infer_b200.mxfp4 import GatedMLP
    model = copy.deepcopy(model).to(DEV)
    with torch.no_grad():
        for name, mod in converted.named_modules():
            if isinstance(mod, CompressedLinear):
                model.get_submodule(name).weight.copy_(mod.weight.get_weight())
            elif isinstance(mod, GatedMLP):
                gate, up = mod.gate_up.weight.get_weight().chunk(2)
                model.get_submodule(name).gate_proj.weight.copy_(gate)
                model.get_submodule(name).up_proj.weight.copy_(up)
            elif isinstance(mod, _FusedSlice):
                assert isinstance(mod._owner, FusedCompressedLinear)
                a, b = mod._owner.splits[mod.index]
                model.get_submodule(name).weight.copy_(mod._owner.weight.get_weight()[a:b])
    return model


@pytest.fixture(scope="module", params=[True, False], ids=["stacked", "separate"])
def models(request):
    from bf16_huffman_infer_b200 import convert_all_linear
    from bf16_huffman_infer_b200.mxfp4 import GatedMLP
    cfg, model = _tiny_model()
    converted = copy.deepcopy(model).to(DEV)
    convert_all_linear(converted, min_out_features=256, progress=False, algo="mxfp4", fuse_siblings=request.param)
    assert not any(isinstance(m, nn.Linear) for m in converted.modules())
    assert sum(isinstance(m, GatedMLP) for m in converted.modules()) == (cfg.num_hidden_layers if request.param else 0)
    return cfg, model, converted


@pytest.mark.parametrize("batch,length", [(1, 1), (2, 9), (3, 70)])
def test_logits(models, batch, length):
    cfg, model, converted = models
    ids = torch.randint(0, cfg.vocab_size, (batch, length), generator=torch.Generator().manual_seed(1)).to(DEV)
    with torch.no_grad():
        got, want = converted(ids).logits.float(), _rounded(model, converted)(ids).logits.float()
    # sums in another order, and the gated pair is rounded once where the separate layers round four times
    assert float((got - want).norm() / want.norm()) < 0.02


def test_graphed_generation(models):
    from transformers import StaticCache
    from bf16_huffman_infer_b200 import get_graphed_model
    cfg, _, converted = models
    ids = torch.randint(0, cfg.vocab_size, (2, 8), generator=torch.Generator().manual_seed(0)).to(DEV)
    kw = dict(max_new_tokens=12, min_new_tokens=12, do_sample=False, output_logits=True, return_dict_in_generate=True)
    with torch.no_grad():
        eager = converted.generate(ids, past_key_values=StaticCache(config=cfg, max_cache_len=64), disable_compile=True, **kw)
    graphed = get_graphed_model(converted, StaticCache(config=cfg, max_cache_len=64))
    run = graphed.generate(ids, **kw)
    assert graphed.graph_stats["replays"] >= 10
    assert _same_decoding(run, eager, "mxfp4") >= 1


def test_saved_and_loaded(models, tmp_path):
    from bf16_huffman_infer_b200 import load_compressed, save_compressed
    cfg, model, converted = models
    path = str(tmp_path / "model.safetensors")
    save_compressed(converted, path)
    fresh = load_compressed(copy.deepcopy(model), path).to(DEV)
    ids = torch.randint(0, cfg.vocab_size, (1, 20), generator=torch.Generator().manual_seed(2)).to(DEV)
    with torch.no_grad():
        assert torch.equal(fresh(ids).logits, converted(ids).logits)


def test_gradient_through_the_frozen_model(models):
    cfg, model, converted = models
    plain = _rounded(model, converted)
    e = (torch.randn(2, 30, cfg.hidden_size, generator=torch.Generator().manual_seed(3)) * 0.1).to(torch.bfloat16).to(DEV)
    grads = []
    for m in (converted, plain):
        for p in m.parameters():
            p.requires_grad_(False)
        leaf = e.clone().requires_grad_()
        m(inputs_embeds=leaf).logits.float().pow(2).mean().backward()
        grads.append(leaf.grad.double())
    # some forty roundings of 2^-8 on the way down and up again, in both
    assert float((grads[0] - grads[1]).norm() / grads[1].norm()) < 0.1


def test_convert_of_one_layer():
    from bf16_huffman_infer_b200 import CompressedLinear, convert
    linear = nn.Linear(256, 100, dtype=torch.bfloat16)
    for where in ("cpu", DEV):
        layer = convert(linear.to(where), "one", disable_precision_check=False, algo="mxfp4")
        assert isinstance(layer, CompressedLinear) and layer.weight.codes.device.type == torch.device(where).type
        x = torch.randn(4, 256, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
        y = layer.to(DEV)(x)
        want = x.double() @ layer.weight.get_weight().double().T + layer.bias.double()
        assert float((y.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
    with pytest.raises(AssertionError):
        convert(nn.Linear(256, 100).to(DEV), "fp32", algo="mxfp4")
    with pytest.raises(ValueError):
        convert(nn.Linear(40, 100, dtype=torch.bfloat16).to(DEV), "narrow", algo="mxfp4")
