"""Row sharding of models with 4-bit layers on the host: which layers become which, and the arena that none of them needs."""
import pytest
import torch
from torch import nn

from bf16_huffman_infer_b200 import CompressedLinear, GatedMLP, GatedMXFP4, MXFP4Weight
from bf16_huffman_infer_b200.functional import FusedCompressedLinear, _FusedSlice
from bf16_huffman_infer_b200.tensor_parallel import PeerArena, PeerRowShardedLinear, RowShardedLinear, shard_model_linears


def weight(M, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    return MXFP4Weight.from_packed(torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g),
                                   torch.randint(110, 130, (M, K // 32), dtype=torch.uint8, generator=g))


def model_of_4_bit_layers():
    model = nn.Module()
    model.out = CompressedLinear(weight(96, 64, 1), nn.Parameter(torch.arange(96.0).to(torch.bfloat16), requires_grad=False))
    owner = FusedCompressedLinear(weight(64 + 32, 64, 2), None, [(0, 64), (64, 96)])
    model.q, model.k = _FusedSlice(owner, 0, True), _FusedSlice(owner, 1, False)
    model.mlp = GatedMLP(GatedMXFP4(weight(2 * 32, 64, 3), None, "silu"), CompressedLinear(weight(64, 32, 4), None))
    model.odd = CompressedLinear(weight(33, 64, 5), None)
    return model, owner


@pytest.mark.parametrize("rank", [0, 1])
@pytest.mark.parametrize("with_arena", [False, True])
def test_layers_of_a_sharded_model(rank, with_arena):
    model, owner = model_of_4_bit_layers()
    full = {"out": model.out.weight.packed(), "fused": owner.weight.packed(), "down": model.mlp.down_proj.weight.packed()}
    bias = model.out.bias.clone()
    arena = PeerArena(torch.device("cpu")) if with_arena else None
    shard_model_linears(model, rank, 2, arena=arena)
    assert type(model.out) is RowShardedLinear and type(model.mlp.down_proj) is RowShardedLinear and type(owner.sharded) is RowShardedLinear
    assert type(model.mlp.gate_up) is GatedMXFP4 and type(model.odd) is CompressedLinear
    for name, layer in (("out", model.out), ("fused", owner.sharded), ("down", model.mlp.down_proj)):
        rows = layer.out_features // 2
        for got, want in zip(layer.local.weight.packed(), full[name]):
            assert torch.equal(got, want[rank * rows:(rank + 1) * rows])
    assert torch.equal(model.out.local.bias, bias[rank * 48:(rank + 1) * 48])


def test_an_arena_without_layers_is_committed():
    model, _ = model_of_4_bit_layers()
    arena = PeerArena(torch.device("cpu"))
    shard_model_linears(model, 0, 1, arena=arena)
    arena.commit()
    assert arena.buffer is not None and arena.buffer.numel() == 0
    with pytest.raises(AssertionError):
        arena.commit()
    with pytest.raises(AssertionError):
        arena.add(64)


def test_no_exchange_layer_of_a_4_bit_weight():
    with pytest.raises(TypeError):
        PeerRowShardedLinear.from_full(CompressedLinear(weight(64, 32), None), PeerArena(torch.device("cpu")))
