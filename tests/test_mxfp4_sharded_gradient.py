"""The gradient through a row-sharded 4-bit layer, two ranks over gloo with a plain product in the kernel's place."""
import os
import socket

import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn.functional as F

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def _worker(rank, world, port, out):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from bf16_huffman_infer_b200 import CompressedLinear, MXFP4Weight
        from bf16_huffman_infer_b200.tensor_parallel import RowShardedLinear

        class Plain(CompressedLinear):
            def forward(self, x):
                codes, scales = self.weight.packed()
                v = GRID[torch.stack([codes & 15, codes >> 4], -1).long()].view(*scales.shape, 32)
                return F.linear(x, torch.ldexp(v, (scales.int() - 127)[..., None]).flatten(1), self.bias)

        g = torch.Generator().manual_seed(0)
        full = Plain(MXFP4Weight.from_packed(torch.randint(0, 256, (96, 32), dtype=torch.uint8, generator=g), torch.randint(120, 128, (96, 2), dtype=torch.uint8, generator=g)), None)
        layer = RowShardedLinear.from_full(full, rank, world)
        layer.local = Plain(layer.local.weight, layer.local.bias)
        x, dy = torch.randn(2, 3, 64, generator=g), torch.randn(2, 3, 96, generator=g)
        leaves = [x.clone().requires_grad_() for _ in range(2)]
        want, got = full(leaves[0]), layer(leaves[1])
        # x reaches the loss on two ways, as past a residual
        grads = [torch.autograd.grad((y * dy).sum() + v.square().sum(), v)[0] for y, v in zip((want, got), leaves)]
        # sums of 64 and of 96 terms, of magnitude 2.5 on average, in another order: each addition loses at most 2^-23 of the magnitudes' sum
        ok = bool(torch.allclose(got, want, rtol=0, atol=64 * 160 * 2.0 ** -23)) and bool(torch.allclose(grads[1], grads[0], rtol=0, atol=96 * 250 * 2.0 ** -23))
        with torch.no_grad():
            ok = ok and not layer(leaves[1]).requires_grad
        out[rank] = ok and not layer(x).requires_grad
    finally:
        dist.destroy_process_group()


def test_gradient_of_a_sharded_layer():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    with mp.Manager() as mgr:
        out = mgr.dict()
        mp.spawn(_worker, args=(2, port, out), nprocs=2, join=True)
        assert dict(out) == {0: True, 1: True}
