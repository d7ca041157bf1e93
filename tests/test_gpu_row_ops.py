"""GPU tests of the operators on factor rows against plain implementations in 64 bits.

Tolerances are bounds, not measurements: u = 2^-24 is half a step of fp32, `half(t)` that of the output's type.  A sum of n
terms in fp32, in whatever order, is off by at most n * u * (sum of the terms' magnitudes) to first order; twice that is
allowed for the higher orders.  Where sums must be exact the terms are small integers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
DEV = "cuda"


def half(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def some_ids(n, rows, g, dtype=torch.int32, pad=0.1, hot=0.3):
    """Ids over all rows, a share of them one row, a share -1."""
    i = torch.randint(0, rows, (n,), generator=g, device=DEV)
    i[torch.rand(n, generator=g, device=DEV) < hot] = rows // 2
    i[torch.rand(n, generator=g, device=DEV) < pad] = -1
    return i.to(dtype)


def within(got, want, tol, what=""):
    got, tol = got.double(), torch.as_tensor(tol, dtype=torch.float64, device=DEV).expand_as(want)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first {got[bad][:3].tolist()} for {want[bad][:3].tolist()}"


def strided(t, extra, offset=0):
    """The same values in rows of a longer stride, at an offset of so many elements."""
    rows, width = t.shape
    store = torch.zeros(rows * (width + extra) + offset, dtype=torch.float32, device=DEV).to(t.dtype)
    v = store[offset:offset + rows * (width + extra)].view(rows, width + extra)[:, :width]
    (v.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else v).copy_(t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t)
    return v


def flag():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ---- lookup ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("width", [1, 3, 8, 33, 64, 100, 128, 200, 520])
@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
def test_lookup(mascot, width, src, dst):
    g = gen(width)
    table = torch.randn(77, width, generator=g, device=DEV).to(src)
    for n, dtype in ((1, torch.int32), (5, torch.int64), (1003, torch.int32)):
        ids = some_ids(n, 77, g, dtype)
        want = torch.cat([table.double() * 1.7, torch.zeros(1, width, dtype=torch.float64, device=DEV)])[ids.long()]
        tol = want.abs() * (2 * U + half(dst)) * 1.01 + (2.0 ** -24 if dst == torch.float16 else 0)      # subnormal steps of binary16
        f = flag()
        within(mascot.rows_lookup(table, ids, scale=1.7, out_dtype=dst, flags=f), want, tol)
        assert f.item() == 0
        odd = strided(table, 5, 1)
        out = strided(torch.full((n, width), 9.0, device=DEV, dtype=dst), 3)
        assert mascot.rows_lookup(odd, ids, scale=1.7, out=out) is out
        within(out, want, tol, "strided")
        four = strided(table, 8, 0)
        within(mascot.rows_lookup(four, ids, scale=1.7, out_dtype=dst), want, tol, "stride in pieces")


def test_lookup_of_bad_ids_and_empty_tables(mascot):
    table = torch.ones(10, 64, device=DEV)
    for dtype, bad in ((torch.int32, [10, -2, 2 ** 31 - 1, -2 ** 31]), (torch.int64, [10, -2, 2 ** 32, 2 ** 32 + 3, 2 ** 62, -2 ** 63])):
        for b in bad:
            f = flag()
            out = mascot.rows_lookup(table, torch.tensor([3, b, -1, 4], dtype=dtype, device=DEV), flags=f)
            assert out.sum(1).tolist() == [64, 0, 0, 64] and f.item() == mascot.FLAG_BAD_ID
    empty = torch.empty(0, 64, device=DEV)
    assert (mascot.rows_lookup(empty, torch.tensor([-1, -1], device=DEV)) == 0).all()
    f = flag()
    assert (mascot.rows_lookup(empty, torch.tensor([0, -1], device=DEV), flags=f) == 0).all() and f.item() == mascot.FLAG_BAD_ID
    assert mascot.rows_lookup(table, torch.empty(0, dtype=torch.int64, device=DEV)).shape == (0, 64)
    # nothing but the named rows is read: the others may hold anything
    table[3] = float("nan")
    assert torch.isfinite(mascot.rows_lookup(table, torch.tensor([1, -1, 2], device=DEV))).all()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("width", [1, 100, 128, 300])
def test_lookup_of_a_quantised_table(mascot, width, block_rows):
    g = gen(width)
    x = torch.randn(300, width, generator=g, device=DEV) * torch.exp2(torch.randint(-30, 30, (300, 1), generator=g, device=DEV).float())
    q, s = mascot.rows_quantize(x, block_rows)
    scales = s.t().repeat_interleave(block_rows, 0)[:300].repeat_interleave(128, 1)[:, :width].double()
    ids = some_ids(1000, 300, g)
    for dst in TYPES:
        want = torch.cat([q.double() * scales * 0.25, torch.zeros(1, width, dtype=torch.float64, device=DEV)])[ids.long()].to(dst)     # all steps but the last are exact
        assert torch.equal(mascot.rows_lookup(q, ids, scale=0.25, table_scale=s, out_dtype=dst), want)
    assert mascot.rows_lookup(strided(q, 7, 3), ids, table_scale=s).dtype == torch.float32


# ---- gradient of a lookup ------------------------------------------------------------------------------------------
def plain_gradient(grad, ids, rows, scale):
    """(sums, sums of magnitudes, terms per row)"""
    at = torch.where((ids >= 0) & (ids < rows), ids.long(), rows)
    s = torch.zeros(rows + 1, grad.shape[1], dtype=torch.float64, device=DEV).index_add_(0, at, grad.double())[:-1] * scale
    m = torch.zeros(rows + 1, grad.shape[1], dtype=torch.float64, device=DEV).index_add_(0, at, grad.double().abs())[:-1] * abs(scale)
    return s, m, torch.bincount(at, minlength=rows + 1)[:-1].double()[:, None]


# one chunk and less; one block's sort and one entry more; tiles with and without a scan; one, two and three digits
@pytest.mark.parametrize("n,rows", [(1, 1), (2, 5), (15, 3), (16, 3), (17, 40), (1000, 7), (12_287, 900), (12_288, 900), (12_289, 900), (12_289, 1), (40_000, 1023), (40_000, 1024),
                                    (32_768, 900), (32_769, 900), (131_072, 100_000), (200_001, 50), (140_001, 1_200_000), (1_048_575, 3000), (1_200_001, 300_000), (1_050_000, 200)])
def test_gradient_is_exact_on_integers(mascot, n, rows):
    g = gen(n + rows)
    for width, dtype, src in ((4, torch.int32, torch.float32), (7, torch.int64, torch.bfloat16), (132, torch.int32, torch.float16)):
        if rows * width > 20_000_000:
            width = 4
        ids = some_ids(n, rows, g, dtype)
        grad = torch.randint(-8, 9, (n, width), generator=g, device=DEV).to(src)
        want, _, _ = plain_gradient(grad, ids, rows, 2.0)
        out = torch.full((rows, width), float("nan"), device=DEV)
        f = flag()
        got = mascot.rows_gradient(grad, ids, rows, scale=2.0, out=out, flags=f)
        assert got is out and torch.equal(got.double(), want) and f.item() == 0
        base = torch.randint(-8, 9, (rows, width), generator=g, device=DEV).float()
        got = mascot.rows_gradient(grad, ids, rows, scale=2.0, out=base.clone(), accumulate=True)
        assert torch.equal(got.double(), want + base.double())


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("width", [5, 64, 100, 260])
def test_gradient(mascot, src, dst, width):
    g = gen(width)
    n, rows = 20_011, 501
    ids = some_ids(n, rows, g, hot=0.1)
    grad = torch.randn(n, width, generator=g, device=DEV).to(src)
    want, mass, terms = plain_gradient(grad, ids, rows, 0.3)
    sums = 2 * (terms + 2) * U * mass
    got = mascot.rows_gradient(grad, ids, rows, scale=0.3, out_dtype=dst)
    within(got, want, sums + want.abs() * half(dst) * 1.01 + (2.0 ** -24 if dst == torch.float16 else 0))
    again = mascot.rows_gradient(strided(grad, 4), ids, rows, scale=0.3, out=strided(torch.ones(rows, width, device=DEV).to(dst), 12))
    assert torch.equal(again, got)                    # same order of the sums, whatever the strides
    odd = mascot.rows_gradient(strided(grad, 3, 1), ids, rows, scale=0.3, out=strided(torch.ones(rows, width, device=DEV).to(dst), 1, 1))
    assert torch.equal(odd, got)
    base = torch.randn(rows, width, generator=g, device=DEV).to(dst)
    got = mascot.rows_gradient(grad, ids, rows, scale=0.3, out=base.clone(), accumulate=True)
    whole = want + base.double()
    within(got, whole, sums + whole.abs() * (half(dst) + 2 * U) * 1.01 + (2.0 ** -24 if dst == torch.float16 else 0), "accumulate")
    untouched = terms[:, 0] == 0
    assert torch.equal(got[untouched], base[untouched])


def test_gradient_of_a_long_table(mascot):
    """Keys of more than 24 bits: three digits of ten."""
    rows, n = 40_000_000, 70_000
    ids = some_ids(n, rows, gen(4), torch.int64)
    grad = torch.randint(-8, 9, (n, 1), generator=gen(5), device=DEV).half()
    want, _, _ = plain_gradient(grad, ids, rows, 1.0)
    assert torch.equal(mascot.rows_gradient(grad, ids, rows, out_dtype=torch.float32).double(), want)


@pytest.mark.parametrize("n", [3000, 300_000, 2_300_000])
def test_gradient_of_one_row(mascot, n):
    """All ids the same: a row over every chunk, more than a block's warps of them."""
    grad = torch.randint(-3, 4, (n, 8), generator=gen(n), device=DEV).float()
    ids = torch.full((n,), 2, device=DEV)
    got = mascot.rows_gradient(grad, ids, 4)
    want = torch.zeros(4, 8, device=DEV, dtype=torch.float64)
    want[2] = grad.double().sum(0)
    assert torch.equal(got.double(), want)


def test_gradient_of_long_and_short_rows_side_by_side(mascot):
    """Runs of every length next to one another: parts of rows that begin, cover and end chunks."""
    g = gen(1)
    lengths = torch.cat([torch.arange(1, 200), torch.tensor([1, 5000, 1, 1, 40_000, 2, 15, 16, 17, 31, 32, 33, 70_000, 1])])
    ids = torch.repeat_interleave(torch.arange(lengths.numel()), lengths).to(DEV)
    grad = torch.randint(-4, 5, (ids.numel(), 33), generator=g, device=DEV).float()
    order = torch.randperm(ids.numel(), generator=g, device=DEV)
    want, _, _ = plain_gradient(grad, ids, lengths.numel(), 1.0)
    for i, x in ((ids, grad), (ids[order], grad[order])):
        assert torch.equal(mascot.rows_gradient(x, i, lengths.numel()).double(), want)


def test_gradient_bad_ids_empty_inputs_and_scratch(mascot):
    grad = torch.ones(4, 64, device=DEV)
    f = flag()
    got = mascot.rows_gradient(grad, torch.tensor([1, 5, -1, -7], device=DEV), 5, flags=f)
    assert got.sum(1).tolist() == [0, 64, 0, 0, 0] and f.item() == mascot.FLAG_BAD_ID
    none = torch.full((4,), -1, device=DEV)
    f = flag()
    assert (mascot.rows_gradient(grad, none, 5, out=torch.ones(5, 64, device=DEV), flags=f) == 0).all() and f.item() == 0
    assert (mascot.rows_gradient(grad, none, 5, out=torch.ones(5, 64, device=DEV), accumulate=True) == 1).all()
    assert (mascot.rows_gradient(grad[:0], none[:0], 5, out=torch.ones(5, 64, device=DEV)) == 0).all()
    assert mascot.rows_gradient(grad, none, 0).shape == (0, 64)
    f = flag()
    mascot.rows_gradient(grad, none + 1, 0, flags=f)
    assert f.item() == mascot.FLAG_BAD_ID
    # places that name no row may hold anything, and so may the scratch
    grad[2:] = float("nan")
    ids = torch.tensor([1, 1, -1, -1], device=DEV)
    ws = torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV)
    assert mascot.rows_gradient(grad, ids, 3, workspace=ws).sum(1).tolist() == [0, 128, 0]
    with pytest.raises(mascot.MascotError):
        mascot.rows_gradient(grad, ids, 3, workspace=ws[:64])


def test_rows_far_into_a_table(mascot):
    """Offsets beyond 2^32 elements."""
    rows = 2 ** 32 // 128 + 1000
    table = torch.zeros(rows, 128, dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([0, rows - 1, rows - 2, rows - 1, 2 ** 25, 2 ** 25 - 1], device=DEV)
    table[ids] = torch.arange(6, device=DEV)[:, None].bfloat16()
    table[rows - 1] = 3
    assert mascot.rows_lookup(table, ids)[:, 127].tolist() == [0, 3, 2, 3, 4, 5]
    got = mascot.rows_gradient(torch.ones(6, 128, device=DEV), ids, rows, out=table)
    assert got[ids][:, 5].tolist() == [1, 2, 1, 2, 1, 1] and float(got.float().sum() if rows < 1000 else got.sum(dtype=torch.float32)) == 6 * 128


# ---- preference loss -------------------------------------------------------------------------------------------------
def pairs(n, users, items, width, dtype, seed, id_type=torch.int32, pad=0.05):
    g = gen(seed)
    P = (torch.randn(users, width, generator=g, device=DEV) * width ** -0.25).to(dtype)
    Q = (torch.randn(items, width, generator=g, device=DEV) * width ** -0.25).to(dtype)
    u, i, j = some_ids(n, users, g, id_type, pad), some_ids(n, items, g, id_type, 0.0), some_ids(n, items, g, id_type, pad, 0.0)
    return P, Q, u, i, j, torch.randn(n, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV) + 0.1


def plain_pairs(P, Q, u, i, j, beta, eps, ref, w, scale):
    there = (u >= 0) & (i >= 0) & (j >= 0)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    P, Q = P.double().requires_grad_(), Q.double().requires_grad_()
    p, qi, qj = P[u.long().clamp(min=0)], Q[i.long().clamp(min=0)], Q[j.long().clamp(min=0)]
    m = (p * (qi - qj)).sum(1)
    m = torch.where(there, m, zero)
    m.retain_grad()
    z = beta * (m - (ref.double() if ref is not None else 0))
    loss = (1 - eps) * torch.nn.functional.softplus(-z, threshold=1e9) + eps * torch.nn.functional.softplus(z, threshold=1e9)
    loss = torch.where(there, loss * (w.double() if w is not None else 1), zero)
    dP, dQ, c = torch.autograd.grad(loss.sum(), [P, Q, m])
    mass = (p.abs() * (qi.abs() + qj.abs())).sum(1).detach()
    return loss.detach(), m.detach(), torch.where(there, c, zero), dP * scale, dQ * scale, mass


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 5, 64, 100, 128, 300])
@pytest.mark.parametrize("plain", [True, False])
def test_pair_loss(mascot, dtype, width, plain):
    for n, id_type in ((1, torch.int32), (3, torch.int64), (1037, torch.int32)):
        P, Q, u, i, j, ref, w = pairs(n, 60, 30, width, dtype, width + n, id_type)
        beta, eps = (1.0, 0.0) if plain else (0.6, 0.15)
        if plain:
            ref = w = None
        loss, m, c, _, _, mass = plain_pairs(P, Q, u, i, j, beta, eps, ref, w, 1.0)
        f = flag()
        got = mascot.pair_loss(P, Q, u, i, j, beta=beta, smoothing=eps, reference=ref, weight=w, flags=f)
        assert f.item() == 0
        # margin: differences, products and sums of `width` terms; z: two roundings more of |beta| (|m| + |ref|)
        tol_m = 2 * (width + 2) * U * mass
        tol_z = beta * (tol_m + 3 * U * (m.abs() + (ref.double().abs() if ref is not None else 0)))
        weight = w.double() if w is not None else 1.0
        within(got[1], m, tol_m, "margin")
        # the loss changes by at most w for a unit of z, coef by beta * w / 4; expf, log1pf and the rest: 16 steps of what they give
        within(got[0], loss, weight * (tol_z + 16 * U * (1 + loss / weight)), "loss")
        within(got[2], c, weight * beta * (tol_z / 4 + 16 * U), "coef")
        odd = mascot.pair_loss(strided(P, 3, 1), strided(Q, 1, 1), u, i, j, beta=beta, smoothing=eps, reference=ref, weight=w)
        within(odd[1], m, tol_m, "margin, strided")


def test_pair_loss_at_its_ends(mascot):
    """Large margins, weights of zero, no rows: nothing but the pair itself is touched."""
    P = torch.tensor([[1.0], [1e3], [-1e3], [float("inf")], [float("nan")], [3e38]], device=DEV)
    Q = torch.tensor([[1.0], [0.0], [10.0]], device=DEV)
    u = torch.tensor([1, 2, 3, 4, 4, -1, 5, 0], device=DEV)
    i = torch.tensor([0, 0, 0, 0, 0, 0, 2, 1], device=DEV)
    j = torch.tensor([1, 1, 1, 1, 1, 1, 1, 1], device=DEV)
    w = torch.tensor([1.0, 1, 1, 1, 0, 1, 1, 1], device=DEV)
    loss, m, c = mascot.pair_loss(P, Q, u, i, j, weight=w)
    assert loss[:3].tolist() == [0, 1000, 0] and c[:3].tolist() == [0, -1, 0]
    assert math.isnan(loss[3]) and math.isnan(c[3])
    assert loss[4:6].tolist() == [0, 0] and c[4:6].tolist() == [0, 0] and m[5].item() == 0
    assert loss[6].item() == 0 and c[6].item() == 0 and m[6].item() == float("inf")
    assert m[7].item() == 0 and abs(loss[7].item() - math.log(2)) < 1e-6 and c[7].item() == -0.5
    # coef 0 and padding add nothing, whatever the rows hold
    dP, dQ = mascot.pair_gradient(P, Q, u[4:7], i[4:7], j[4:7], c[4:7])
    assert (dP == 0).all() and (dQ == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("width", [3, 16, 64, 100, 128, 260])
def test_pair_gradient(mascot, dtype, dst, width):
    for n, users, items, id_type in ((1, 4, 3, torch.int64), (700, 60, 30, torch.int32), (4096, 300, 5, torch.int32), (9001, 2000, 100, torch.int32)):
        P, Q, u, i, j, ref, w = pairs(n, users, items, width, dtype, width + n, id_type)
        _, _, c, dP, dQ, _ = plain_pairs(P, Q, u, i, j, 0.7, 0.1, ref, w, 0.25)
        coef = c.float()                                     # half a step of fp32 off, in every term
        there = (u >= 0) & (i >= 0) & (j >= 0)
        U_, I, J = (x.long().clamp(min=0) for x in (u, i, j))
        cp = torch.where(there, c.abs(), 0.0)[:, None]
        massP = torch.zeros_like(dP).index_add_(0, U_, cp * (Q.double()[I].abs() + Q.double()[J].abs())) * 0.25
        massQ = torch.zeros_like(dQ).index_add_(0, I, cp * P.double()[U_].abs()).index_add_(0, J, cp * P.double()[U_].abs()) * 0.25
        f = flag()
        gotP, gotQ = mascot.pair_gradient(P, Q, u, i, j, coef, scale=0.25, out_dtype=dst, flags=f)
        assert f.item() == 0
        tiny = 2.0 ** -24 if dst == torch.float16 else 0
        countP = torch.bincount(U_, minlength=users).double()[:, None]
        countQ = (torch.bincount(I, minlength=items) + torch.bincount(J, minlength=items)).double()[:, None]
        within(gotP, dP, 2 * (countP + 4) * U * massP + dP.abs() * half(dst) * 1.01 + tiny, "dP")
        within(gotQ, dQ, 2 * (countQ + 4) * U * massQ + dQ.abs() * half(dst) * 1.01 + tiny, "dQ")
        both = torch.zeros(max(users, items), 2 * width + 4, device=DEV).to(dst)
        a, b = mascot.pair_gradient(strided(P, 5, 1), strided(Q, 2, 1), u, i, j, coef, scale=0.25, dP=both[:users, :width], dQ=both[:items, width + 4:])
        assert torch.equal(a, gotP) and torch.equal(b, gotQ)
        bP, bQ = torch.randn(users, width, device=DEV).to(dst), torch.randn(items, width, device=DEV).to(dst)
        aP, aQ = mascot.pair_gradient(P, Q, u, i, j, coef, scale=0.25, dP=bP.clone(), dQ=bQ.clone(), accumulate=True)
        for got, base, d, mass, count in ((aP, bP, dP, massP, countP), (aQ, bQ, dQ, massQ, countQ)):
            whole = base.double() + d
            within(got, whole, 2 * (count + 4) * U * mass + whole.abs() * (half(dst) + 2 * U) * 1.01 + tiny, "accumulate")


@pytest.mark.parametrize("n,users,items", [(1, 2, 2), (171, 5, 2), (1366, 900, 40), (10_923, 3000, 40), (150_001, 70_000, 900), (400_003, 70_000, 9000)])
def test_pair_gradient_is_exact_on_integers(mascot, n, users, items):
    g = gen(5)
    P = torch.randint(-2, 3, (users, 64), generator=g, device=DEV).float()
    Q = torch.randint(-2, 3, (items, 64), generator=g, device=DEV).float()
    u, i, j = some_ids(n, users, g), some_ids(n, items, g), some_ids(n, items, g)
    coef = torch.randint(-2, 3, (n,), generator=g, device=DEV).float()
    there = (u >= 0) & (i >= 0) & (j >= 0)
    U_, I, J, c = u.long().clamp(min=0), i.long().clamp(min=0), j.long().clamp(min=0), torch.where(there, coef, 0.0).double()[:, None]
    dP = torch.zeros(users, 64, dtype=torch.float64, device=DEV).index_add_(0, U_, c * (Q[I] - Q[J]))
    dQ = torch.zeros(items, 64, dtype=torch.float64, device=DEV).index_add_(0, I, c * P[U_]).index_add_(0, J, -c * P[U_])
    gotP, gotQ = mascot.pair_gradient(P, Q, u, i, j, coef)
    assert torch.equal(gotP.double(), dP) and torch.equal(gotQ.double(), dQ)
    f = flag()
    a, b = 7 % n, 9 % n
    u[a], j[b] = users, items
    mascot.pair_gradient(P, Q, u, i, j, coef, flags=f)
    assert f.item() == mascot.FLAG_BAD_ID
    f = flag()
    loss, m, c = mascot.pair_loss(P, Q, u, i, j, flags=f)
    assert f.item() == mascot.FLAG_BAD_ID and loss[[a, b]].tolist() == [0, 0] and c[[a, b]].tolist() == [0, 0]


def test_pair_tables_without_rows(mascot):
    """Pairs that name rows of an empty table add nothing, and say so."""
    P, Q = torch.empty(0, 64, device=DEV), torch.ones(3, 64, device=DEV)
    u = torch.tensor([0, -1], device=DEV)
    f = flag()
    loss, m, c = mascot.pair_loss(P, Q, u, u.clamp(min=0), u.clamp(min=0), flags=f)
    assert loss.tolist() == [0, 0] and f.item() == mascot.FLAG_BAD_ID
    f = flag()
    dP, dQ = mascot.pair_gradient(P, Q, u, u.clamp(min=0), u.clamp(min=0), torch.ones(2, device=DEV), dP=torch.empty(0, 64, device=DEV), dQ=torch.ones(3, 64, device=DEV), flags=f)
    assert dP.shape == (0, 64) and (dQ == 0).all() and f.item() == mascot.FLAG_BAD_ID
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert all(t.shape == (0,) for t in mascot.pair_loss(Q, Q, none, none, none))
    dP, dQ = mascot.pair_gradient(Q, Q, none, none, none, torch.empty(0, device=DEV), dP=torch.ones(3, 64, device=DEV), dQ=torch.ones(3, 64, device=DEV))
    assert (dP == 0).all() and (dQ == 0).all()


def test_two_streams_at_once(mascot):
    """Calls in flight on two streams, each with scratch of its own, do not touch one another."""
    args = [pairs(60_000, 5000, 700, 64, torch.float32, s) for s in (1, 2)]
    def both(a):
        P, Q, u, i, j, ref, w = a
        c = mascot.pair_loss(P, Q, u, i, j, weight=w)[2]
        return mascot.pair_gradient(P, Q, u, i, j, c)
    want = [[t.clone() for t in both(a)] for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(20):
        got = []
        for a, st in zip(args, streams):
            with torch.cuda.stream(st):
                got.append(both(a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


def test_pair_gradient_against_differences(mascot):
    """dloss / dP and dQ by central differences of the loss, in steps that fp32 resolves."""
    P, Q, u, i, j, ref, w = pairs(40, 6, 5, 8, torch.float32, 3)
    loss, m, c = mascot.pair_loss(P, Q, u, i, j, beta=0.8, smoothing=0.1, reference=ref, weight=w)
    dP, dQ = mascot.pair_gradient(P, Q, u, i, j, c)
    h = 2.0 ** -6
    for t, d in ((P, dP), (Q, dQ)):
        for r in range(t.shape[0]):
            for k in range(t.shape[1]):
                was = t[r, k].item()
                sums = []
                for x in (was + h, was - h):
                    t[r, k] = x
                    sums.append(mascot.pair_loss(P, Q, u, i, j, beta=0.8, smoothing=0.1, reference=ref, weight=w)[0].double().sum().item())
                t[r, k] = was
                # differences of fp32 losses (about 40 of them, each some 2^-22 off) over 2 h, and h^2 / 6 of a third derivative below 40 * 4^3 / 8
                assert abs((sums[0] - sums[1]) / (2 * h) - d[r, k].item()) < 40 * 2.0 ** -21 / (2 * h) + h * h / 6 * 320


def test_pair_of_one_item_adds_nothing(mascot):
    P, Q = torch.ones(2, 64, device=DEV), torch.ones(3, 64, device=DEV)
    u, i = torch.tensor([0, 1], device=DEV), torch.tensor([1, 2], device=DEV)
    loss, m, c = mascot.pair_loss(P, Q, u, i, i)
    assert m.tolist() == [0, 0] and c.tolist() == [-0.5, -0.5]
    dP, dQ = mascot.pair_gradient(P, Q, u, i, i, c)
    assert (dP == 0).all() and (dQ == 0).all()


# ---- quantisation ------------------------------------------------------------------------------------------------------
def plain_quantize(x, block_rows):
    """(q, scales) from the definition, in 64 bits."""
    rows, width = x.shape
    y = x.double()
    r, c = torch.arange(rows, device=DEV) // block_rows, torch.arange(width, device=DEV) // 128
    rb, cb = -(-rows // block_rows), -(-width // 128)
    top = torch.zeros(cb * rb, dtype=torch.float64, device=DEV)
    top.scatter_reduce_(0, (c[None, :] * rb + r[:, None]).reshape(-1), torch.where(torch.isfinite(y), y.abs(), 0.0).reshape(-1), "amax")
    m, e = torch.frexp(top / 448)                     # the exponent of a power of two above: e, or e - 1 where top / 448 is one itself
    s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), torch.where(m == 0.5, e - 1, e).clamp(min=-126)), 1.0).view(cb, rb)
    z = y / s[c[None, :], r[:, None]]
    step = torch.ldexp(torch.ones_like(z), (torch.frexp(z)[1] - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(y), torch.round(z / step) * step, float("nan")), s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (3, 129), (128, 128), (130, 100), (257, 512), (300, 515)])
def test_quantize(mascot, dtype, block_rows, rows, width):
    g = gen(rows + width)
    x = torch.randn(rows, width, generator=g, device=DEV)
    x = (x * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g, device=DEV).float())).to(dtype)
    x[:, ::7] *= 2.0 ** -11
    x[0, 0] = 0
    want, s = plain_quantize(x, block_rows)
    for src in (x, strided(x, 4), strided(x, 3, 1)):
        q, scale = mascot.rows_quantize(src, block_rows)
        assert torch.equal(scale.double(), s) and torch.equal(q.double(), want)
    q = strided(torch.zeros(rows, width, device=DEV).to(torch.float8_e4m3fn), 5, 2)
    assert mascot.rows_quantize(x, block_rows, q=q)[0] is q and torch.equal(q.double(), want)


def test_quantize_borders_and_what_is_not_finite(mascot):
    rows = [[448.0, 1, 0, -448], [449.0, 1, 2, 3], [448.0 * 2 ** 20, 1, 2, 3], [0.0, 0, -0.0, 0], [2.0 ** -140, 0, 0, 2.0 ** -149], [3.4e38, -3.4e38, 1, 0],
            [float("inf"), 7, -3, 0.5], [float("nan"), float("-inf"), 5, 0], [float("nan"), float("inf"), 0, 0], [17.0, 18, 19, 16], [-17.0, -18, -19, 0.001]]
    x = torch.tensor(rows, device=DEV)
    want, s = plain_quantize(x, 1)
    q, scale = mascot.rows_quantize(x)
    assert torch.equal(scale.double(), s)
    assert torch.equal(torch.isnan(q.float()), ~torch.isfinite(x))
    assert torch.equal(q.double().nan_to_num(0), want.nan_to_num(0))
    q, scale = mascot.rows_quantize(x, 128)
    want, s = plain_quantize(x, 128)
    assert torch.equal(scale.double(), s) and torch.equal(q.double().nan_to_num(0), want.nan_to_num(0))
    assert mascot.rows_quantize(x[:0])[0].shape == (0, 4)


def test_quantize_and_lookup_write_rows_and_no_more(mascot):
    """What lies between the rows, and behind the last one, stays as it was."""
    for width in (100, 97, 128):
        store = torch.full((5 * 160 + 7,), 77, dtype=torch.uint8, device=DEV)
        q = store[3 * (width == 97):].as_strided((5, width), (160, 1), 3 * (width == 97)).view(torch.float8_e4m3fn)
        mascot.rows_quantize(torch.ones(5, width, device=DEV), q=q)
        mark = torch.zeros_like(store)
        mark.as_strided((5, width), (160, 1), 3 * (width == 97)).fill_(1)
        assert (store[mark == 0] == 77).all() and (store[mark == 1] != 77).all()
        out = torch.full((5 * 160 + 7,), 7.0, device=DEV)
        mascot.rows_lookup(torch.ones(9, width, device=DEV), torch.arange(5, device=DEV), out=out.as_strided((5, width), (160, 1), 3 * (width == 97)))
        assert (out[mark == 0] == 7).all() and (out[mark == 1] == 1).all()
        out.fill_(7)
        mascot.rows_gradient(torch.ones(2, width, device=DEV), torch.tensor([1, 4], device=DEV), 5, out=out.as_strided((5, width), (160, 1), 3 * (width == 97)))
        assert (out[mark == 0] == 7).all() and out[mark == 1].sum().item() == 2 * width


# ---- scores ----------------------------------------------------------------------------------------------------------
def quantised(rows, width, seed, block_rows=1, any_scale=False):
    g = gen(seed)
    x = torch.randn(rows, width, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))
    q = (x * 50).clamp(-448, 448).to(torch.float8_e4m3fn)
    blocks = (-(-width // 128), -(-rows // block_rows))
    s = torch.rand(blocks, generator=g, device=DEV) + 0.25 if any_scale else torch.exp2(torch.randint(-8, 3, blocks, generator=g, device=DEV).float())
    each = s.t().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :width].double()
    store = torch.full((rows, -(-width // 16) * 16), 0x7f, dtype=torch.uint8, device=DEV)      # NaN behind the width: not read
    store[:, :width] = q.view(torch.uint8)
    return store.view(torch.float8_e4m3fn)[:, :width], s, q.double() * each


def check_product(mascot, m, n, width, block_rows, dst, seed=0, any_scale=True, out=None):
    a, sa, va = quantised(m, width, seed + 1, 1, any_scale)
    b, sb, vb = quantised(n, width, seed + 2, block_rows, any_scale)
    want, mass = va @ vb.t(), va.abs() @ vb.abs().t()
    f = flag()
    got = mascot.rows_product(a, sa, b, sb, out_dtype=None if out is not None else dst, out=out, flags=f)
    assert f.item() == 0
    # a step of fp32 (addends may be cut, not rounded) of the magnitudes for each addition, three roundings for the scales of a block
    tol = 2 * (min(width, 128) + 4 + -(-width // 128)) * 2 * U * mass + want.abs() * half(dst) * 1.01 + (2.0 ** -24 if dst == torch.float16 else 0)
    big = want.abs() > 65000 if dst == torch.float16 else torch.zeros_like(want, dtype=torch.bool)
    within(torch.where(big, 0.0, got.double()), torch.where(big, 0.0, want), tol, f"{m} x {n} x {width}")


@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 63, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("n", [1, 31, 127, 128, 129, 1000])
def test_product_sizes(mascot, m, n):
    check_product(mascot, m, n, 64, 1, torch.float32)
    check_product(mascot, m, n, 128, 128, torch.bfloat16)


@pytest.mark.parametrize("width", [1, 15, 16, 17, 31, 32, 33, 64, 100, 127, 128, 129, 160, 255, 256, 257, 384, 1000, 4096])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dst", TYPES)
def test_product_widths(mascot, width, block_rows, dst):
    check_product(mascot, 70, 300, width, block_rows, dst)
    check_product(mascot, 3, 260, width, block_rows, dst)


@pytest.mark.parametrize("m,n,width", [(1, 100_003, 128), (20, 20_001, 128), (50, 20_001, 300), (100, 20_001, 64), (120, 20_001, 520), (1000, 20_011, 64), (4096, 5000, 128), (513, 2049, 1024), (900, 12_345, 384)])
def test_product_of_many_tiles(mascot, m, n, width):
    check_product(mascot, m, n, width, 1, torch.float32)
    check_product(mascot, m, n, width, 128, torch.float16, any_scale=False)


@pytest.mark.parametrize("dst", TYPES)
def test_product_into_strided_rows(mascot, dst):
    for extra, offset in ((0, 1), (1, 0), (3, 3), (8, 0)):
        store = torch.full((70 * (200 + extra) + offset + 9,), 5.0, device=DEV, dtype=dst)
        out = store[offset:offset + 70 * (200 + extra)].view(70, 200 + extra)[:, :200]
        check_product(mascot, 70, 200, 128, 1, dst, out=out)
        rest = torch.ones_like(store, dtype=torch.bool)
        rest[offset:offset + 70 * (200 + extra)].view(70, 200 + extra)[:, :200] = False
        assert (store[rest] == 5).all()


def test_product_of_nan_zero_and_large_scales(mascot):
    """A NaN and an infinite scale concern their own row and column only; large scales do not overflow on the way."""
    a, sa, va = quantised(5, 256, 1)
    b, sb, vb = quantised(200, 256, 2)
    a, b = a.clone(), b.clone()
    a.view(torch.uint8)[2, 130] = 0x7f
    b.view(torch.uint8)[77, 3] = 0xff
    sa[1, 3] = float("inf")
    got = mascot.rows_product(a, sa, b, sb)
    bad = torch.zeros(5, 200, dtype=torch.bool, device=DEV)
    bad[2], bad[3], bad[:, 77] = True, True, True
    assert torch.equal(torch.isfinite(got), ~bad)
    one = torch.full((1, 128), 1.0, device=DEV).to(torch.float8_e4m3fn)
    big, small = torch.full((1, 1), 2.0 ** 100, device=DEV), torch.full((1, 1), 2.0 ** -120, device=DEV)
    assert mascot.rows_product(one, big, one, small).item() == 2.0 ** -13
    zero = torch.zeros(3, 128, device=DEV).to(torch.float8_e4m3fn)
    assert (mascot.rows_product(zero, torch.ones(1, 3, device=DEV), b[:, :128], sb[:1].contiguous()).nan_to_num(0) == 0).all()
    assert mascot.rows_product(a[:0], sa[:, :0].contiguous(), b, sb).shape == (0, 200)


# ---- as they are used ----------------------------------------------------------------------------------------------------
def test_streams_and_graphs(mascot):
    """The calls run on torch's current stream and can be captured; a graph with scratch of its own may be replayed next to another."""
    P, Q, u, i, j, ref, w = pairs(20_000, 3000, 500, 64, torch.float32, 1)

    def step():
        loss, m, c = mascot.pair_loss(P, Q, u, i, j, reference=ref)
        dP, dQ = mascot.pair_gradient(P, Q, u, i, j, c, scale=0.5)
        rows = mascot.rows_lookup(P, u, scale=3.0)
        back = mascot.rows_gradient(rows, u, 3000)
        q, s = mascot.rows_quantize(Q)
        qu, su = mascot.rows_quantize(rows[:40])
        return loss, m, dP, dQ, rows, back, q.float(), s, mascot.rows_product(qu, su, q, s)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    was = P.clone()
    for round_ in range(3):
        P.copy_(was * (round_ + 1))
        for _, out in graphs:
            for t in out:
                t.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    P.copy_(was)


def test_equal_calls_give_equal_bits(mascot):
    P, Q, u, i, j, ref, w = pairs(100_000, 3000, 500, 128, torch.bfloat16, 2)
    first = None
    for _ in range(3):
        loss, m, c = mascot.pair_loss(P, Q, u, i, j)
        got = (loss, m, c, *mascot.pair_gradient(P, Q, u, i, j, c, out_dtype=torch.float32), mascot.rows_gradient(P[u.long().clamp(min=0)], u, 3000, out_dtype=torch.float32))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_train_from_preferences_and_answer(mascot):
    """A run of all of them: steps on pairs against a frozen model, then scores of all items for a batch of users from tables in
    8 bits.  The steps follow the same steps in 64 bits, the scores those of the quantised rows."""
    n, users, items, k = 6000, 400, 90, 64
    P, Q, u, i, j, _, _ = pairs(n, users, items, k, torch.float32, 9, pad=0.02)
    P64, Q64 = P.double(), Q.double()
    ref = mascot.pair_loss(P, Q, u, i, j)[1]
    for step in range(3):
        loss, m, c = mascot.pair_loss(P, Q, u, i, j, beta=0.5, reference=ref)
        dP, dQ = mascot.pair_gradient(P, Q, u, i, j, c, scale=1.0)
        _, m64, _, gP, gQ, _ = plain_pairs(P64, Q64, u, i, j, 0.5, 0.0, ref, None, 1.0)
        P, Q, P64, Q64 = P - 0.05 * dP, Q - 0.05 * dQ, P64 - 0.05 * gP, Q64 - 0.05 * gQ
        # errors of a step are some hundred units of 2^-24 of the sums of a popular row (about 2,000 terms below 1); three steps
        within(P, P64, 3 * 0.05 * 2000 * 2000 * U / 10, f"P after step {step}")
        within(Q, Q64, 3 * 0.05 * 2000 * 2000 * U / 10, f"Q after step {step}")
    batch = torch.tensor([5, 17, -1, 399, 5], device=DEV)
    rows = mascot.rows_lookup(P, batch)
    assert torch.equal(rows[0], P[5]) and (rows[2] == 0).all()
    qa, sa = mascot.rows_quantize(rows)
    qb, sb = mascot.rows_quantize(Q)
    scores = mascot.rows_product(qa, sa, qb, sb)
    va, vb = qa.double() * sa.t().double(), qb.double() * sb.t().double()
    within(scores, va @ vb.t(), 2 * (k + 6) * 2 * U * (va.abs() @ vb.abs().t()))
    assert (scores[2] == 0).all() and torch.equal(scores[0], scores[4])
    # and back: the gradient of what a lookup gave, by position
    g = torch.ones_like(rows)
    back = mascot.rows_gradient(g, batch, users, scale=2.0)
    assert back[5].tolist() == [4.0] * k and back[17].tolist() == [2.0] * k and back.sum().item() == 4 * 2.0 * k


def test_python_face_refuses(mascot):
    x, i = torch.zeros(4, 64, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    q, s = mascot.rows_quantize(x)
    for f in (lambda: mascot.rows_lookup(x.t(), i), lambda: mascot.rows_lookup(x.double(), i), lambda: mascot.rows_lookup(x, i.cpu()), lambda: mascot.rows_lookup(x, i.float()),
              lambda: mascot.rows_lookup(x[0], i), lambda: mascot.rows_lookup(x, i, out=torch.zeros(3, 63, device=DEV)), lambda: mascot.rows_lookup(q, i),
              lambda: mascot.rows_lookup(q, i, table_scale=s[:, :3].contiguous()), lambda: mascot.rows_lookup(x[:1].expand(4, 64), i),
              lambda: mascot.rows_lookup(x, i, flags=torch.zeros(2, dtype=torch.int32, device=DEV)), lambda: mascot.rows_lookup(x, torch.zeros(6, dtype=torch.int32, device=DEV)[::2]),
              lambda: mascot.rows_gradient(x, i, 4), lambda: mascot.rows_gradient(x[:3], i, 4, accumulate=True), lambda: mascot.rows_gradient(x[:3], i, 4, out=x),
              lambda: mascot.pair_loss(x, x, i, i, i, weight=torch.zeros(4, device=DEV)), lambda: mascot.pair_gradient(x, x, i, i, i, torch.zeros(3, device=DEV), dP=x, dQ=x.clone()),
              lambda: mascot.rows_quantize(x, 2), lambda: mascot.rows_quantize(q), lambda: mascot.rows_product(q, s, q, s[:, :3].contiguous()),
              lambda: mascot.rows_product(q, s, x, s), lambda: mascot.rows_product(q, s, q, s, out=torch.zeros(4, 5, device=DEV))):
        with pytest.raises(mascot.MascotError) as e:
            f()
        assert e.value.status == mascot.ERR_BAD_ARG
    host = torch.zeros(4, 64)
    rows = mascot.Rows(host.data_ptr(), 4, 64, 64, 0)
    out = torch.zeros(3, 64, device=DEV)
    rc = mascot.load().mascot_rows_lookup(rows, None, 0, mascot.Ids(i.data_ptr(), 3, 64, 0), 1.0, mascot.Rows(out.data_ptr(), 3, 64, 64, 0), None, None)
    assert rc == mascot.ERR_BAD_ARG and b"not memory of the current device" in mascot.load().mascot_last_error(None)
