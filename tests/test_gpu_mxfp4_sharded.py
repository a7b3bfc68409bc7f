"""Row sharding of a model with 4-bit and lossless layers on one rank: the arena holds what exchanges, the rest computes as before."""
import pytest
import torch
from torch import nn

from _util import make_weight

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("lossless", [False, True])
@pytest.mark.parametrize("with_arena", [False, True])
def test_one_rank(lossless, with_arena):
    from bf16_huffman_infer_b200 import CompressedLinear, HuffmanWeight, MXFP4Weight
    from bf16_huffman_infer_b200.tensor_parallel import PeerArena, RowShardedLinear, shard_model_linears
    a, b = (make_weight(512, 512, seed).to(DEV) for seed in (1, 2))
    model = nn.Sequential(CompressedLinear(MXFP4Weight.compress(a, to_cpu=False), None),
                          CompressedLinear(HuffmanWeight.compress(b).to(DEV) if lossless else MXFP4Weight.compress(b, to_cpu=False), None)).to(DEV)
    x = torch.randn(4, 512, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    with torch.no_grad():
        want = model(x)
    arena = PeerArena(torch.device(DEV)) if with_arena else None
    shard_model_linears(model, 0, 1, arena=arena)
    if arena is not None:
        arena.commit()
    assert type(model[0]) is RowShardedLinear
    with torch.no_grad():
        for _ in range(2):
            assert torch.equal(model(x), want)
