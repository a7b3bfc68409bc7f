"""Products of 4-bit weights where few rows of X meet the ends of the number range, against plain computations in 64 bits.

Tolerances.  An output is its 32-bit sum rounded to BF16 once: off by at most 2^-8 of itself and, for the sum, by K additions that lose at
most 2^-23 each of the sum of the terms' magnitudes; K halves of BF16's smallest step, 2^-134, for what lies below the normal numbers."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# rows of X and the weight's shape: every form of the kernel for few rows (two tiles of the weight a step from 256 rows an SM on)
FORMS = [(1, 40, 512), (3, 40, 2080), (8, 40, 2080), (1, 40000, 128), (8, 40000, 160), (8, 40000, 1056), (5, 3000, 4128), (9, 24003, 416), (16, 24000, 416), (16, 2100, 2080),
         (17, 24002, 160), (24, 24002, 416), (24, 23700, 2080), (40, 130, 416)]


@pytest.fixture(scope="module")
def pkg():
    import bf16_huffman_infer_b200
    return bf16_huffman_infer_b200


def weight(pkg, M, K, seed, lo=120, hi=128):
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (M, K // 2), dtype=torch.uint8, generator=g, device=DEV)
    return codes, torch.randint(lo, hi, (M, K // 32), dtype=torch.uint8, generator=g, device=DEV)


def within(y, want, mag, K):
    err = (y.double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + mag * (K * 2.0 ** -23) + K * 2.0 ** -134
    assert bool((err <= bound).all()), (float((err / bound.clamp(min=1e-300)).max()), int((err > bound).sum()))


def gated64(z, mag, K):
    """silu(g) u of projections in 64 bits, and how far the sums' errors may move it (|silu'| <= 1.1)"""
    (g, u), (mg, mu) = z.chunk(2, -1), mag.chunk(2, -1)
    a = g * torch.sigmoid(g)
    slack = 1.1 * mg * K * 2.0 ** -23 * (u.abs() + mu * K * 2.0 ** -23) + a.abs() * mu * K * 2.0 ** -23
    return a * u, slack + (a * u).abs() * 2.0 ** -14              # the function's own error, some units of 2^-23 of arguments


@pytest.mark.parametrize("rows,M,K", FORMS)
@pytest.mark.parametrize("spread", [30, 34, 45, 90])
def test_x_far_apart_inside_a_group(pkg, rows, M, K, spread):
    """Neighbouring values of X up to 2^spread apart, and weights that are zero wherever X is large: what is left is all that counts."""
    codes, scales = weight(pkg, M, K, spread)
    g = torch.Generator(device=DEV).manual_seed(rows + spread)
    x = torch.randn(rows, K, generator=g, device=DEV)
    small = torch.rand(K, generator=g, device=DEV) < 0.7
    small[:2] = torch.tensor([False, True], device=DEV)
    x = torch.where(small, x * 2.0 ** -spread, x)
    x[:, 0] = 1.0
    x = x.to(torch.bfloat16)
    keep = torch.where(small[0::2], 0x0F, 0) + torch.where(small[1::2], 0xF0, 0)
    codes[: M // 2 * 2: 2] &= keep.to(torch.uint8)               # every other row
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dense = w.get_weight().double()
    want, mag = x.double() @ dense.T, x.double().abs() @ dense.abs().T
    within(F.linear(x, w), want, mag, K)
    if M % 2 == 0:
        h, slack = gated64(want, mag, K)
        err = (pkg.gated_mxfp4(x, w).double() - h).abs()
        assert bool((err <= h.abs() * 2.0 ** -8 + slack + 2.0 ** -134).all())


@pytest.mark.parametrize("rows,M,K", FORMS)
@pytest.mark.parametrize("byte", [0, 1, 2, 3])
@pytest.mark.parametrize("spread", [26, 29, 31])
def test_x_far_apart_under_the_smallest_scales(pkg, rows, M, K, byte, spread):
    """The same with X up to 2^100 and scales of 2^-127 and little more: what is left are ordinary numbers."""
    codes, scales = weight(pkg, M, K, spread, byte, byte + 1)
    g = torch.Generator(device=DEV).manual_seed(rows + spread)
    x = (1 + torch.rand(rows, K, generator=g, device=DEV)) * 2.0 ** (100 - spread)
    x[:, ::128] = 2.0 ** 100
    x = x.to(torch.bfloat16)
    codes[:, ::64] &= 0xF0                                       # zero codes where X is large
    codes[:, 1:] &= 0x11                                         # and others up to 0.5
    codes[:, 4:] = 0                                             # few of them: a sum of one group
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dense = w.get_weight().double()
    within(F.linear(x, w), x.double() @ dense.T, x.double().abs() @ dense.abs().T, K)


@pytest.mark.parametrize("rows", [1, 8, 16])
def test_one_row_far_apart_leaves_the_others(pkg, rows):
    """A chunk of K whose X is far apart in one row is multiplied in another way; every row keeps its tolerance, chunk by chunk."""
    M, K = 24000, 16384                                          # X in several chunks from eight rows on
    codes, scales = weight(pkg, M, K, 1)
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dense = w.get_weight()
    for at in (5, K - 3):
        x = torch.randn(rows, K, generator=torch.Generator(device=DEV).manual_seed(at), device=DEV)
        x[rows // 2, at] = 2.0 ** -50
        x = x.to(torch.bfloat16)
        want = torch.cat([x.double() @ part.double().T for part in dense.split(4000)], 1)
        mag = torch.cat([x.double().abs() @ part.double().abs().T for part in dense.split(4000)], 1)
        within(F.linear(x, w), want, mag, K)


@pytest.mark.parametrize("rows", [1, 3, 8, 16, 24])
def test_sums_of_infinities_and_nans_in_x(pkg, rows):
    """A row with infinities of one sign, of both, or a NaN, next to rows without: classes of results term by term."""
    M, K = 24002, 416
    codes, scales = weight(pkg, M, K, 7)
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dense = w.get_weight().double()
    x = torch.randn(rows, K, generator=torch.Generator(device=DEV).manual_seed(rows), device=DEV).to(torch.bfloat16)
    clean = F.linear(x, w)
    for values in ([(3, math.inf)], [(3, math.inf), (200, math.inf)], [(3, math.inf), (5, -math.inf)], [(415, math.nan)], [(0, 3e38), (1, -math.inf)]):
        v = x.clone()
        for at, value in values:
            v[0, at] = value
        special = ~v[0].isfinite()
        terms = v[0, special].double() * dense[:, special]
        y = F.linear(v, w)
        want = terms.sum(1)
        assert torch.equal(y[0].isnan(), want.isnan()) and torch.equal(y[0][~want.isnan()].double(), want[~want.isnan()])
        assert torch.equal(y[1:], clean[1:])


def test_a_row_with_a_nan_takes_little_time_of_its_own(pkg):
    """Its outputs are NaNs by the products as they are: nothing is computed once more (which took eighteen times as long)."""
    M, K, rows = 40000, 4096, 8
    w = pkg.MXFP4Weight.from_packed(*weight(pkg, M, K, 3))
    x = torch.randn(rows, K, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    nan = x.clone()
    nan[0, 5] = math.nan

    def time(v):
        best = math.inf
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda.synchronize()
            a.record()
            for _ in range(20):
                F.linear(v, w)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    time(x)
    assert time(nan) < 5 * time(x)


def test_overflow_inside_is_not_the_outputs(pkg):
    """Scales near 2^104, under which the FP16 sums of four blocks overflow while the outputs, X being small, do not."""
    for rows in (1, 8, 16):
        for byte in (229, 231, 233, 250):
            M, K = (24000, 512) if rows > 8 else (40, 512)
            codes = torch.full((M, K // 2), 0x77, dtype=torch.uint8, device=DEV)
            w = pkg.MXFP4Weight.from_packed(codes, torch.full((M, K // 32), byte, dtype=torch.uint8, device=DEV))
            x = torch.full((rows, K), 2.0 ** -70 * 1.9921875, device=DEV, dtype=torch.bfloat16)
            want = x.double().sum(1, keepdim=True) * 6 * 2.0 ** (byte - 127)
            assert torch.equal(F.linear(x, w).double(), want.to(torch.bfloat16).double().expand(rows, M))


@pytest.mark.parametrize("rows,M,K", FORMS)
@pytest.mark.parametrize("byte", [191, 192, 231, 252, 253, 254, 255])
def test_large_scales_in_some_rows(pkg, rows, M, K, byte):
    """Scales from 2^64 on in a few blocks, those among them under which codes leave the range: every form agrees with the dense matrix, zeros in X
    included, and the other rows of the weight keep their tolerance."""
    codes, scales = weight(pkg, M, K, byte)
    g = torch.Generator(device=DEV).manual_seed(rows + byte)
    at = torch.randint(0, M, (5,), generator=g, device=DEV)
    scales[at, torch.randint(0, K // 32, (5,), generator=g, device=DEV)] = byte
    x = torch.randn(rows, K, generator=g, device=DEV) * 2.0 ** -30
    x[:, torch.rand(K, generator=g, device=DEV) < 0.3] = 0.0
    x[0] = 0.0
    x = x.to(torch.bfloat16)
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dense = w.get_weight()
    assert bool(dense.isnan().any()) == (byte > 252) and not bool(dense.isinf().any())
    wide = dense.double()
    clean = torch.where(wide.isfinite(), wide, 0)
    bad = torch.nonzero(~wide.isfinite().all(1))[:, 0]
    want, mag = x.double() @ clean.T, x.double().abs() @ clean.abs().T
    for m in bad.tolist():                                       # NaNs term by term
        want[:, m] = (x.double() * wide[m]).sum(1)
    y = F.linear(x, w)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.isinf(), want.isinf()) and torch.equal(y[y.isinf()].double(), want[y.isinf()])
    fine = want.isfinite()
    within(y[fine], want[fine], mag[fine], K)


@pytest.mark.parametrize("rows", [1, 8, 16, 40])
@pytest.mark.parametrize("code,byte", [(7, 253), (6, 253), (5, 253), (4, 254), (3, 254), (15, 254), (11, 254), (1, 254)])
def test_codes_beyond_the_range(pkg, rows, code, byte):
    """Values that BF16 just has and just has not, few rows and many alike."""
    M = 24000 if rows == 16 else 32                              # FP16 products and BF16 ones of few rows
    w = pkg.MXFP4Weight.from_packed(torch.full((M, 64), code * 17, dtype=torch.uint8, device=DEV), torch.full((M, 4), byte, dtype=torch.uint8, device=DEV))
    dense = w.get_weight().double()
    value = [0, 0.5, 1, 1.5, 2, 3, 4, 6][code & 7] * 2.0 ** (byte - 127) * (-1 if code & 8 else 1)
    fits = abs(value) < 2.0 ** 128
    assert bool((dense == value).all() if fits else dense.isnan().all())
    for x in (torch.full((rows, 128), 2.0 ** -100, device=DEV), torch.eye(128, device=DEV)[:rows] * 2.0 ** -60, torch.zeros(rows, 128, device=DEV)):
        x = x.to(torch.bfloat16)
        y = F.linear(x, w).double()
        want = x.double().sum(1, keepdim=True).expand(rows, M) * value
        assert torch.equal(y, want) if fits else bool(y.isnan().all())


def test_plain_order_beyond_the_range_as_on_the_host(pkg):
    from test_mxfp4_range import every_code_under
    for byte in range(250, 256):
        codes, scales = every_code_under(byte)
        codes, scales = codes[:528].view(-1, 3 * 16), scales[:528].view(-1, 3)      # blocks side by side
        want, got = pkg.MXFP4Weight.from_packed(codes, scales), pkg.MXFP4Weight.from_packed(codes.to(DEV), scales.to(DEV))
        assert torch.equal(got.codes.cpu(), want.codes) and torch.equal(got.scales.cpu(), want.scales)


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("byte", [0, 1, 60, 127, 128, 200, 251, 252])
def test_input_gradient_under_scales_of_the_whole_range(pkg, rows, byte):
    M, K = 150, 416
    w = pkg.MXFP4Weight.from_packed(*weight(pkg, M, K, byte, byte, byte + 1))
    dense = w.get_weight().double()
    g = torch.Generator(device=DEV).manual_seed(rows + byte)
    dy = torch.ldexp(torch.randn(rows, 152, generator=g, device=DEV).double(), torch.tensor(min(127 - byte, 120), device=DEV)).to(torch.bfloat16)
    dx = pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, M, K)  # two columns more than the weight has rows: not read
    dy = dy[:, :M].double()
    within(dx, dy @ dense, dy.abs() @ dense.abs(), M)


@pytest.mark.parametrize("rows", [1, 40])
def test_input_gradient_of_nan_blocks_and_of_nans(pkg, rows):
    """A NaN block makes its 32 columns NaN, a NaN in dy its row; nothing else."""
    M, K = 150, 416
    codes, scales = weight(pkg, M, K, 5)
    scales[149, 2], scales[3, 12] = 255, 255
    w = pkg.MXFP4Weight.from_packed(codes, scales)
    dy = torch.randn(rows, 152, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    dy[:, 150:] = math.nan                                       # past the weight's rows
    want = torch.zeros(rows, K, dtype=torch.bool, device=DEV)
    want[:, 64:96] = want[:, 384:416] = True
    assert torch.equal(pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, M, K).isnan(), want)
    dy[rows // 2, 7] = math.nan
    want[rows // 2] = True
    assert torch.equal(pkg.ops.mxfp4_linear_grad(dy, w.codes, w.scales, M, K).isnan(), want)
