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
