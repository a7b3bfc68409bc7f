"""Scale bytes under which codes leave BF16's range, in the plain order: the same values under another scale, or NaN."""
import pytest
import torch

from bf16_huffman_infer_b200 import MXFP4Weight

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def values(codes, scales):
    """In 64 bits, of the plain order; a block whose scale is NaN, or that has a value beyond the range, is NaN."""
    v = GRID[torch.stack([codes & 15, codes >> 4], -1).long()].view(*scales.shape, 32)
    v = torch.ldexp(v, (scales.int() - 127)[..., None])
    none = (scales == 255) | (v.abs() >= 2.0 ** 128).any(-1)
    return torch.where(none[..., None], torch.nan, v)


def every_code_under(byte):
    """Rows of a block of one code each, all sixteen, then blocks with one code in one place among small ones."""
    one = torch.arange(16, dtype=torch.uint8)[:, None].expand(16, 16) * 17
    mixed = torch.full((16 * 32, 16), 0x10, dtype=torch.uint8)
    for i in range(32):
        for c in range(16):
            mixed[16 * i + c, i // 2] = c << 4 if i % 2 else 0x10 | c
    codes = torch.cat([one, mixed])
    return codes, torch.full((codes.shape[0], 1), byte, dtype=torch.uint8)


@pytest.mark.parametrize("byte", [0, 125, 251, 252, 253, 254, 255])
def test_values_are_kept_or_nan(byte):
    codes, scales = every_code_under(byte)
    w = MXFP4Weight.from_packed(codes, scales)
    got, want = values(*w.packed()), values(codes, scales)
    assert torch.equal(got.isnan(), want.isnan())
    there = ~want.isnan()
    assert torch.equal(got[there], want[there]) and torch.equal(torch.signbit(got[there]), torch.signbit(want[there]))
    assert set(w.scales.unique().tolist()) <= {0, byte if byte < 253 else 252, 255}


def test_blocks_side_by_side():
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (40, 160 // 2), dtype=torch.uint8, generator=g) & 0x99      # codes up to 0.5
    scales = torch.randint(245, 256, (40, 5), dtype=torch.uint8, generator=g)
    codes[::7, 20] |= 0x60
    w = MXFP4Weight.from_packed(codes, scales)
    got, want = values(*w.packed()), values(codes, scales)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num()) and bool(want.isnan().any())
