"""GPU tests of the scores, by kernel: scales at the ends of fp32, and how each stores.

Which kernel a call takes follows from its sizes: up to 128 columns one that sums nothing up (ONE), for longer rows one with items in the
lanes (ROWS), or one with users there for more than 128 users and square blocks (SQUARE), each with tiles of several widths."""
import pytest
import torch

from test_gpu_row_ops import DEV, TYPES, U, check_product, flag, gen, half, within

pytestmark = pytest.mark.gpu

# users, items, columns, rows to a scale of the items
KERNELS = {
    "ONE, 16 users a tile": (5, 200, 128, 1), "ONE, 32": (40, 200, 128, 128), "ONE, 256": (200, 18_944, 128, 1), "ONE, 64, no whole tile": (64, 18_945, 100, 128),
    "ROWS, 16": (5, 200, 256, 1), "ROWS, 32": (129, 200, 300, 1), "ROWS, 32, squares": (128, 200, 256, 128), "ROWS, 256": (200, 18_944, 256, 1),
    "SQUARE, 128": (129, 200, 256, 128), "SQUARE, 256": (129, 18_944, 256, 128),
}


def of_value(rows, width, value):
    return torch.full((rows, -(-width // 16) * 16), float(value), device=DEV).to(torch.float8_e4m3fn)[:, :width]


def powers(shape, exponent):
    return torch.full(shape, 2.0 ** exponent, dtype=torch.float64, device=DEV).float()


@pytest.mark.parametrize("kernel", KERNELS)
def test_scales_that_make_up_for_one_another(mascot, kernel):
    """One scale or the product of both is far outside of what fp32 holds next to the sum; the score is not.  All steps are exact: a block's
    sum has seven significant bits, and the scales are powers of two."""
    m, n, width, each = KERNELS[kernel]
    blocks = -(-width // 128)
    for value, ea, eb in ((448, -110, 110), (448, 110, -110), (448, -126, 120), (448, -75, -75), (448, -149, 20), (448, 20, -149), (2 ** -9, 66, 66), (2 ** -9, 127, 10)):
        a, b = of_value(m, width, value), of_value(n, width, value)
        sa, sb = powers((blocks, m), ea), powers((blocks, -(-n // each)), eb)
        want = value * value * width * 2.0 ** (ea + eb)
        assert 2.0 ** -126 <= want < 2.0 ** 128
        f = flag()
        got = mascot.rows_product(a, sa, b, sb, flags=f)
        assert f.item() == 0 and (got.double() == want).all(), (value, ea, eb, want, got[0, 0].item())
        # one row of either side with ordinary scales between the others
        sa[:, m // 2], sb[:, -1] = 1, 1
        a.view(torch.uint8)[m // 2], b.view(torch.uint8)[:] = 0x38, 0x38          # ones
        got = mascot.rows_product(a, sa, b, sb)
        last = (n - 1) // each * each
        assert (got[m // 2, last:] == width).all()


@pytest.mark.parametrize("kernel", KERNELS)
def test_scales_over_all_of_fp32(mascot, kernel):
    """Scales from subnormal ones to 2^120, a different one in each place: right wherever the terms and sums are numbers of fp32."""
    m, n, width, each = KERNELS[kernel]
    g = gen(m + n + width)
    blocks = -(-width // 128)

    def scales(count, low, high):
        e = torch.randint(low, high, (blocks, count), generator=g, device=DEV).double()
        return (torch.exp2(e) * (1 + torch.rand(blocks, count, generator=g, device=DEV, dtype=torch.float64))).float()
    a = (torch.randn(m, width, generator=g, device=DEV) * 40).to(torch.float8_e4m3fn)
    b = (torch.randn(n, width, generator=g, device=DEV) * 40).to(torch.float8_e4m3fn)
    up = -(-width // 16) * 16
    a, b = (torch.nn.functional.pad(x.view(torch.uint8), (0, up - width)).view(torch.float8_e4m3fn)[:, :width] for x in (a, b))
    sa, sb = scales(m, -140, 120), scales(-(-n // each), -140, 120)
    sa[:, 0] = 0                                            # no rounding hides these
    each_a = sa.t().repeat_interleave(128, 1)[:, :width].double()
    each_b = sb.t().repeat_interleave(each, 0)[:n].repeat_interleave(128, 1)[:, :width].double()
    va, vb = a.double() * each_a, b.double() * each_b
    want, mass = va @ vb.t(), va.abs() @ vb.abs().t()
    got = mascot.rows_product(a, sa, b, sb)
    # as in check_product, and half a step of the smallest numbers for each rounding: the scaled sum and the addition of a block
    tol = 2 * (min(width, 128) + 4 + blocks) * 2 * U * mass + want.abs() * half(torch.float32) * 1.01 + 2 * blocks * 2.0 ** -150
    fits = mass < 2.0 ** 126                                # neither a term nor a partial sum leaves fp32
    assert fits.float().mean() > 0.3 and (want[fits].abs() > 2.0 ** -126).float().mean() > 0.3
    within(torch.where(fits, got.double(), 0.0), torch.where(fits, want, 0.0), tol)


@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("m,width,each", [(129, 129, 128), (300, 256, 128), (130, 256, 1), (70, 300, 1), (120, 256, 128)])
@pytest.mark.parametrize("n", [264, 262, 263, 18_944, 18_942])
def test_long_rows_into_strided_scores(mascot, dst, m, width, each, n):
    """Rows of scores at 16-, 4- and 2-byte boundaries, and nothing written beside them."""
    for extra, offset in ((0, 0), (8, 0), (0, 1), (2, 2), (1, 0)):
        if n > 1000 and (extra, offset) not in ((0, 0), (2, 2), (1, 0)):
            continue
        store = torch.full((m * (n + extra) + offset + 9,), 5.0, device=DEV, dtype=dst)
        out = store[offset:offset + m * (n + extra)].view(m, n + extra)[:, :n]
        check_product(mascot, m, n, width, each, dst, out=out)
        rest = torch.ones_like(store, dtype=torch.bool)
        rest[offset:offset + m * (n + extra)].view(m, n + extra)[:, :n] = False
        assert (store[rest] == 5).all()


@pytest.mark.parametrize("kernel", KERNELS)
def test_a_row_of_zeros_meets_a_nan(mascot, kernel):
    """Scores of a row of zeros are zeros but for the item that holds a NaN."""
    m, n, width, each = KERNELS[kernel]
    a, b = of_value(m, width, 1), of_value(n, width, 1)
    a.view(torch.uint8)[2] = 0
    b.view(torch.uint8)[77, 3] = 0xff
    blocks = -(-width // 128)
    got = mascot.rows_product(a, powers((blocks, m), 0), b, powers((blocks, -(-n // each)), 3))
    want = torch.full((m, n), 8.0 * width, device=DEV)
    want[2] = 0
    want[:, 77] = float("nan")
    assert torch.equal(got.nan_to_num(-1), want.nan_to_num(-1))
