"""4-bit microscaled weights on the host: the order in memory and what is refused."""
import ctypes

import pytest
import torch
import torch.nn.functional as F

from _util import LIB
from bf16_huffman_infer_b200 import GatedMXFP4, MXFP4Weight, gated_mxfp4, linear_mxfp4, ops

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def packed_weight(M, K, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(110, 130, (M, K // 32), dtype=torch.uint8, generator=g)
    return codes, scales


@pytest.mark.parametrize("M,K", [(1, 32), (16, 128), (17, 96), (33, 160), (128, 512)])
def test_packed_and_back(M, K):
    codes, scales = packed_weight(M, K)
    w = MXFP4Weight.from_packed(codes, scales)
    assert w.shape == (M, K) and tuple(w.codes.shape) == ((M + 15) // 16, (K + 127) // 128, 16, 4, 16)
    back = w.packed()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)


def test_order_of_the_buffers():
    """One element at a time: element e of quarter t of block j is nibble e / 2 + 4 (e odd) of word j of the row in quarter t."""
    for k in range(256):
        codes = torch.zeros(18, 128, dtype=torch.uint8)
        codes[17, k // 2] = 5 << (4 * (k % 2))
        w = MXFP4Weight.from_packed(codes, torch.full((18, 8), 127, dtype=torch.uint8))
        group, j, t, e = k // 128, k % 128 // 32, k % 32 // 8, k % 8
        nibble = e // 2 + 4 * (e % 2)
        want = torch.zeros(2, 2, 16, 4, 16, dtype=torch.uint8)
        want[1, group, 1, t, 4 * j + nibble // 2] = 5 << (4 * (nibble % 2))
        assert torch.equal(w.codes, want)
    scales = torch.arange(18 * 8, dtype=torch.uint8).view(18, 8)
    w = MXFP4Weight.from_packed(torch.zeros(18, 128, dtype=torch.uint8), scales)
    assert torch.equal(w.scales[1, 1, 1], scales[17, 4:]) and torch.equal(w.scales[0, 0, 3], scales[3, :4]) and int(w.scales[1, :, 2:].sum()) == 0


def test_nan_blocks_hold_no_codes():
    codes, scales = packed_weight(16, 128)
    scales[3, 1] = 255
    w = MXFP4Weight.from_packed(codes, scales)
    back = w.packed()[0].view(16, 4, 16)
    assert int(back[3, 1].sum()) == 0 and torch.equal(back[2], codes.view(16, 4, 16)[2])


def test_e8m0_scales_are_taken():
    codes, scales = packed_weight(16, 128)
    w = MXFP4Weight.from_packed(codes, scales.view(torch.float8_e8m0fnu))
    assert torch.equal(w.packed()[1], scales)


def test_refused_buffers():
    codes, scales = packed_weight(16, 128)
    for c, s in [(codes[:, :-1], scales), (codes, scales[:, :-1]), (codes[:-1], scales), (codes.int(), scales), (codes, scales.int()), (codes[0], scales[0])]:
        with pytest.raises(ValueError):
            MXFP4Weight.from_packed(c, s)
    w = MXFP4Weight.from_packed(codes, scales)
    for args in [(w.codes, w.scales, 17, 128), (w.codes, w.scales, 16, 129), (w.codes, w.scales, 16, 160), (w.codes, w.scales, 0, 128), (w.codes.int(), w.scales, 16, 128),
                 (w.codes, w.scales[..., :3], 16, 128)]:
        with pytest.raises(ValueError):
            MXFP4Weight(*args)
    with pytest.raises(ValueError):
        GatedMXFP4(w, None, "relu")
    with pytest.raises(ValueError):
        GatedMXFP4(MXFP4Weight.from_packed(codes[:15], scales[:15]), None, "silu")


def test_no_computation_on_the_host():
    codes, scales = packed_weight(16, 128)
    w = MXFP4Weight.from_packed(codes, scales)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    with pytest.raises(AssertionError):
        linear_mxfp4(x, w)
    with pytest.raises(AssertionError):
        F.linear(x, w)
    with pytest.raises(AssertionError):
        gated_mxfp4(x, w)
    with pytest.raises(AssertionError):
        w.get_weight()
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.forward_mxfp4(x, w.codes, w.scales, 16, None)
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.mxfp4_quantize(x, w.codes, w.scales)


def test_only_linear_takes_the_weight():
    w = MXFP4Weight.from_packed(*packed_weight(16, 128))
    with pytest.raises(TypeError):
        F.bilinear(torch.zeros(1, 4), torch.zeros(1, 4), w)


def test_operator_schemas():
    ns = torch.ops.bf16_huffman_infer
    for name, sig in {
        "mxfp4_quantize": "(Tensor W, Tensor(a!) codes, Tensor(b!) scales) -> ()",
        "mxfp4_from_packed": "(Tensor packed, Tensor packed_scales, Tensor(a!) codes, Tensor(b!) scales) -> ()",
        "dense_mxfp4": "(Tensor codes, Tensor scales, int M, int K) -> Tensor",
        "forward_mxfp4": "(Tensor X, Tensor codes, Tensor scales, int M, Tensor? bias) -> Tensor",
        "mxfp4_linear_grad": "(Tensor dY, Tensor codes, Tensor scales, int M, int K) -> Tensor",
        "mxfp4_gated_grad": "(Tensor pre, Tensor dH, int activation) -> Tensor",
    }.items():
        assert str(getattr(ns, name).default._schema) == f"bf16_huffman_infer::{name}{sig}"


def test_refusals_of_the_library():
    """The C entry points look at sizes, pointers and types before they touch a device."""
    lib = ctypes.CDLL(LIB)
    lib.bhi_last_error.restype = ctypes.c_char_p
    p, odd, none, n = ctypes.c_void_p(256), ctypes.c_void_p(264), ctypes.c_void_p(0), ctypes.c_int
    most, refused = (1 << 24) + 32, 1
    weights = [(none, p, 16, 128), (p, none, 16, 128), (odd, p, 16, 128), (p, odd, 16, 128), (p, p, 0, 128), (p, p, 16, 0), (p, p, 16, 48), (p, p, most, 128), (p, p, 16, most)]
    for c, s, M, K in weights:
        assert lib.bhi_mxfp4_quantize(p, n(0), n(M), n(K), c, s, none) == refused
        assert lib.bhi_mxfp4_from_packed(p, p, n(M), n(K), c, s, none) == refused
        assert lib.bhi_mxfp4_dense(c, s, n(M), n(K), p, none) == refused
        assert lib.bhi_mxfp4_linear(c, s, n(M), n(K), p, none, p, n(1), none) == refused
        assert lib.bhi_mxfp4_linear_grad(c, s, n(M), n(K), p, n(max(M, 8) // 8 * 8), p, n(1), none) == refused
        assert lib.bhi_mxfp4_gated(c, s, n(M // 2), n(K), p, none, n(0), p, none, n(1), none) == refused
    assert lib.bhi_mxfp4_quantize(odd, n(0), n(16), n(128), p, p, none) == refused
    assert lib.bhi_mxfp4_quantize(p, n(3), n(16), n(128), p, p, none) == refused
    for codes, scales in [(none, p), (p, none), (ctypes.c_void_p(258), p)]:
        assert lib.bhi_mxfp4_from_packed(codes, scales, n(16), n(128), p, p, none) == refused
    assert lib.bhi_mxfp4_dense(p, p, n(16), n(128), odd, none) == refused
    for x, y, rows in [(none, p, 1), (odd, p, 1), (p, none, 1), (p, p, 0), (p, p, -1), (p, p, (1 << 30) + 1)]:
        assert lib.bhi_mxfp4_linear(p, p, n(16), n(128), x, none, y, n(rows), none) == refused
        assert lib.bhi_mxfp4_linear_grad(p, p, n(16), n(128), x, n(16), y, n(rows), none) == refused
        assert lib.bhi_mxfp4_gated(p, p, n(8), n(128), x, none, n(0), y, none, n(rows), none) == refused
    for ld in (8, 17, 20):
        assert lib.bhi_mxfp4_linear_grad(p, p, n(16), n(128), p, n(ld), p, n(1), none) == refused
    for act in (-1, 3):
        assert lib.bhi_mxfp4_gated(p, p, n(8), n(128), p, none, n(act), p, none, n(1), none) == refused
        assert lib.bhi_mxfp4_gated_grad(p, p, n(8), n(act), p, n(16), n(1), none) == refused
    for pre, dh, out, inter, ld, rows in [(none, p, p, 8, 16, 1), (p, none, p, 8, 16, 1), (p, p, none, 8, 16, 1), (odd, p, p, 8, 16, 1), (p, p, p, 0, 16, 1),
                                          (p, p, p, 8, 12, 1), (p, p, p, 8, 18, 1), (p, p, p, 8, 16, 0), (p, p, p, 8, 16, (1 << 30) + 1)]:
        assert lib.bhi_mxfp4_gated_grad(pre, dh, n(inter), n(0), out, n(ld), n(rows), none) == refused
    assert lib.bhi_last_error()


def test_rows_of_a_weight():
    codes, scales = packed_weight(50, 96)
    w = MXFP4Weight.from_packed(codes, scales)
    part = w.rows(7, 41)
    assert part.shape == (34, 96)
    assert torch.equal(part.packed()[0], codes[7:41]) and torch.equal(part.packed()[1], scales[7:41])
    from bf16_huffman_infer_b200.tensor_parallel import shard_rows
    parts = [shard_rows(w, r, 3).packed() for r in range(3)]
    assert torch.equal(torch.cat([p[0] for p in parts]), codes) and torch.equal(torch.cat([p[1] for p in parts]), scales)


class _Block(torch.nn.Module):
    def __init__(self, act, scale=1.0, extra=False):
        super().__init__()
        self.gate_proj, self.up_proj = (torch.nn.Linear(64, 96, bias=False, dtype=torch.bfloat16) for _ in range(2))
        self.down_proj = torch.nn.Linear(96, 64, bias=False, dtype=torch.bfloat16)
        self.act_fn = act
        self.scale = scale
        if extra:
            self.norm = torch.nn.LayerNorm(96)

    def forward(self, x):
        return self.down_proj(self.act_fn(self.gate_proj(x)) * self.up_proj(x) * self.scale)


def test_which_blocks_are_gated():
    from bf16_huffman_infer_b200.functional import _is_gated_mlp, fuse_gated_mlps
    from torch import nn
    assert _is_gated_mlp(_Block(nn.SiLU())) == "silu"
    assert _is_gated_mlp(_Block(nn.GELU())) == "gelu"
    assert _is_gated_mlp(_Block(nn.GELU(approximate="tanh"))) == "gelu_tanh"
    hooked = _Block(nn.SiLU())
    hooked.up_proj.register_forward_hook(lambda m, a, o: o)
    empty = _Block(nn.SiLU())
    empty.up_proj.weight.data.fill_(float("nan"))
    assert _is_gated_mlp(empty) == "silu"
    for other in (_Block(nn.ReLU()), _Block(nn.SiLU(), scale=2.0), _Block(nn.SiLU(), extra=True), hooked, _Block(nn.SiLU()).float(), nn.SiLU(), nn.Linear(4, 4)):
        assert _is_gated_mlp(other) is None
    with pytest.raises(ValueError):
        fuse_gated_mlps(nn.Sequential(_Block(nn.SiLU())), algo="huffman")


def test_refused_checkpoint_entries():
    from torch import nn
    from bf16_huffman_infer_b200.checkpoint import _validate
    model = nn.Sequential(_Block(nn.SiLU()), nn.Linear(64, 32))
    good = {"0": {"kind": "gated", "bias": False, "activation": "silu", "algo": "mxfp4", "shape": [192, 64]},
            "1": {"kind": "linear", "bias": True, "algo": "mxfp4", "shape": [32, 64]}}
    _validate(model, {"modules": good, "slices": {}})
    for name, change in [("0", {"shape": [96, 64]}), ("0", {"activation": "gelu"}), ("0", {"algo": "huffman"}), ("1", {"shape": [64, 32]}), ("1", {"shape": None}),
                         ("1", {"kind": "gated", "activation": "silu"})]:
        bad = {**good, name: {**good[name], **change}}
        with pytest.raises(ValueError):
            _validate(model, {"modules": bad, "slices": {}})
