"""GPU tests of the calls around the operators on factor rows: what they take from, and leave to, the program that makes them."""
import ctypes as C

import pytest
import torch

from test_gpu_row_ops import DEV, gen

pytestmark = pytest.mark.gpu


def some_calls(mascot):
    """Each operator as a function without arguments that returns its outputs, all of them there before the call but for those of the pair loss."""
    g = gen(3)
    P, Q = torch.randn(50, 64, generator=g, device=DEV), torch.randn(300, 64, generator=g, device=DEV)
    u = torch.randint(0, 50, (40_000,), generator=g, device=DEV)
    i, j = (torch.randint(0, 300, (40_000,), generator=g, device=DEV) for _ in range(2))
    rows, back = torch.empty(40_000, 64, device=DEV), torch.empty(50, 64, device=DEV)
    dP, dQ, scores = torch.empty_like(P), torch.empty_like(Q), torch.empty(50, 300, device=DEV)
    coef = torch.randn(40_000, generator=g, device=DEV)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device=DEV)
    (qp, sp), (qq, sq), (qs, ss) = mascot.rows_quantize(P), mascot.rows_quantize(Q), mascot.rows_quantize(Q, 128)
    few = slice(0, 100)
    return {
        "lookup": lambda: mascot.rows_lookup(P, u, out=rows),
        "lookup from 8 bits": lambda: mascot.rows_lookup(qp, u, table_scale=sp, out=rows),
        "gradient": lambda: mascot.rows_gradient(rows, u, 50, out=back, workspace=ws),
        "gradient, few": lambda: mascot.rows_gradient(rows[few], u[few], 50, out=back, workspace=ws),
        "gradient, none": lambda: mascot.rows_gradient(rows[:0], u[:0], 50, out=back, workspace=ws),
        "loss": lambda: mascot.pair_loss(P, Q, u, i, j),
        "pairs": lambda: mascot.pair_gradient(P, Q, u, i, j, coef, dP=dP, dQ=dQ, workspace=ws),
        "quantize": lambda: mascot.rows_quantize(Q, q=qq, scale=sq),
        "quantize, squares": lambda: mascot.rows_quantize(Q, 128, q=qs, scale=ss),
        "product": lambda: mascot.rows_product(qp, sp, qq, sq, out=scores),
    }


CALLS = ["lookup", "lookup from 8 bits", "gradient", "gradient, few", "gradient, none", "loss", "pairs", "quantize", "quantize, squares", "product"]


def bits(out):
    return [t.clone().view(torch.uint8) for t in (out if isinstance(out, tuple) else (out,))]


@pytest.mark.parametrize("name", CALLS)
def test_an_old_error_of_the_caller_is_not_the_calls(mascot, name):
    """A CUDA call of the program failed and nobody has asked for the thread's last error yet: the operators do their work all the same, report
    no error, and leave that one where it is."""
    call = some_calls(mascot)[name]
    want = bits(call())
    call()                                                  # outputs that torch allocates come from its cache from here on
    torch.cuda.synchronize()
    runtime = C.CDLL("libcudart.so.12")
    assert runtime.cudaSetDevice(9999) == 101               # no such device: refused by the host, nothing else happens
    try:
        got = call()
    finally:
        left = runtime.cudaGetLastError()
    assert left == 101
    assert all(torch.equal(a, b) for a, b in zip(bits(got), want))


def test_tensors_that_require_gradients_are_refused_while_gradients_are_recorded(mascot):
    """A call that autograd does not see must not lose a gradient without a word; under no_grad, and with detached tensors, all is as ever."""
    P, Q = torch.randn(8, 64, device=DEV), torch.randn(9, 64, device=DEV)
    i = torch.tensor([0, 3, -1], device=DEV)
    c, w = torch.ones(3, device=DEV), torch.ones(3, device=DEV)
    (q, s), x = mascot.rows_quantize(Q), torch.randn(3, 64, device=DEV)
    out = torch.empty(3, 64, device=DEV)
    calls = [
        (lambda t: mascot.rows_lookup(t, i), P), (lambda t: mascot.rows_lookup(P, i, out=t), out), (lambda t: mascot.rows_lookup(q, i, table_scale=t), s),
        (lambda t: mascot.rows_gradient(t, i, 8), x), (lambda t: mascot.rows_gradient(x, i, 8, out=t), P.clone()),
        (lambda t: mascot.pair_loss(t, Q, i, i, i), P), (lambda t: mascot.pair_loss(P, t, i, i, i), Q), (lambda t: mascot.pair_loss(P, Q, i, i, i, reference=t), w),
        (lambda t: mascot.pair_loss(P, Q, i, i, i, weight=t), w), (lambda t: mascot.pair_gradient(t, Q, i, i, i, c), P), (lambda t: mascot.pair_gradient(P, t, i, i, i, c), Q),
        (lambda t: mascot.pair_gradient(P, Q, i, i, i, t), c), (lambda t: mascot.rows_quantize(t), Q), (lambda t: mascot.rows_product(q, t, q, s), s),
    ]
    for call, t in calls:
        leaf = t.clone().requires_grad_()
        with pytest.raises(mascot.MascotError) as e:
            call(leaf)
        assert e.value.status == mascot.ERR_BAD_ARG and "requires a gradient" in str(e.value)
        with pytest.raises(mascot.MascotError):
            call(leaf * 1)                                  # as refused: the product of one
        with torch.no_grad():
            under = bits(call(leaf))
        assert all(torch.equal(a, b) for a, b in zip(under, bits(call(leaf.detach())))), "the same under no_grad and detached"


def test_what_a_call_writes_counts_as_changed(mascot):
    """Autograd finds out that a tensor which it saved has been written into."""
    P, Q = torch.randn(8, 64, device=DEV), torch.randn(9, 64, device=DEV)
    i, c = torch.tensor([0, 3, -1], device=DEV), torch.ones(3, device=DEV)
    q, s = mascot.rows_quantize(Q)
    x, big = torch.randn(3, 64, device=DEV), torch.empty(9, 9, device=DEV)
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    dP, dQ = torch.zeros_like(P), torch.zeros_like(Q)
    wide = torch.zeros(3, 128, device=DEV)
    for call, written in (
        (lambda: mascot.rows_lookup(P, i, out=wide[:, 64:], flags=flags), [wide, flags]),
        (lambda: mascot.rows_gradient(x, i, 8, out=dP, accumulate=True, workspace=ws), [dP, ws]),
        (lambda: mascot.pair_loss(P, Q, i, i, i, flags=flags), [flags]),
        (lambda: mascot.pair_gradient(P, Q, i, i, i, c, dP=dP, dQ=dQ, workspace=ws), [dP, dQ, ws]),
        (lambda: mascot.rows_quantize(Q, q=q, scale=s), [q, s]),
        (lambda: mascot.rows_product(q, s, q, s, out=big), [big]),
    ):
        before, inputs = [t._version for t in written], [t._version for t in (P, Q, i, c, x)]
        call()
        assert all(t._version > v for t, v in zip(written, before))
        assert inputs == [t._version for t in (P, Q, i, c, x)]
    weight = torch.ones(3, 64, device=DEV, requires_grad=True)
    saved = torch.zeros(3, 64, device=DEV)
    loss = (weight * saved).sum()
    mascot.rows_lookup(P, i, out=saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        inside = torch.empty(3, 64, device=DEV)
        assert mascot.rows_lookup(P, i, out=inside) is inside
    assert mascot.rows_lookup(P, i, out=inside) is inside
