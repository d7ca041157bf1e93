"""CPU tests of the operators on factor rows: what the C ABI refuses before it touches a GPU, and the pure functions.  Addresses are
made up: nothing here is launched, with or without a GPU."""
import ctypes as C

import pytest

AT = 1 << 44            # not an address of anything
GAP = 1 << 36


def rows(mascot, n, width, type_=0, at=0, stride=None, data=None):
    return mascot.Rows(AT + at * GAP if data is None else data, n, width if stride is None else stride, width, type_)


def ids(mascot, n, at=8, bits=32, data=None, reserved=0):
    return mascot.Ids(AT + at * GAP if data is None else data, n, bits, reserved)


def refused(mascot, rc, *words):
    assert rc == mascot.ERR_BAD_ARG, rc
    text = mascot.load().mascot_last_error(None).decode()
    for w in words:
        assert w in text, text


def reached_the_device(mascot, rc):
    """All arguments were taken: what is missing is a GPU, or memory of one at the made-up address."""
    import torch
    if torch.cuda.is_available():
        refused(mascot, rc, "not memory of the current device")
    else:
        assert rc == mascot.ERR_NO_DEVICE


def lookup(mascot, table, i, out, scales=None, block_rows=0):
    return mascot.load().mascot_rows_lookup(table, scales, block_rows, i, 1.0, out, None, None)


def test_lookup_refuses(mascot):
    M = mascot
    t, i, o = rows(M, 10, 64), ids(M, 5), rows(M, 5, 64, at=1)
    reached_the_device(M, lookup(M, t, i, o))
    refused(M, lookup(M, None, i, o), "table", "null")
    refused(M, lookup(M, t, None, o), "ids", "null")
    refused(M, lookup(M, t, i, None), "out", "null")
    refused(M, lookup(M, rows(M, 10, 64, 7), i, o), "table")
    refused(M, lookup(M, t, i, rows(M, 5, 64, M.E4M3, 1)), "out")
    refused(M, lookup(M, rows(M, 10, 64, stride=63), i, o), "stride")
    refused(M, lookup(M, rows(M, 10, 0), i, o), "width")
    refused(M, lookup(M, rows(M, 10, 65537), i, o), "width")
    refused(M, lookup(M, rows(M, 1 << 31, 64), i, o), "rows")
    refused(M, lookup(M, rows(M, 10, 64, data=0), i, o), "table", "null")
    refused(M, lookup(M, rows(M, 10, 64, data=AT + 2), i, o), "table", "address")
    refused(M, lookup(M, t, ids(M, 5, bits=16), o), "bits")
    refused(M, lookup(M, t, ids(M, 5, reserved=1), o), "reserved")
    refused(M, lookup(M, t, ids(M, 5, data=AT + 8 * GAP + 4, bits=64), o), "ids", "address")
    refused(M, lookup(M, t, i, rows(M, 6, 64, at=1)), "out", "each id")
    refused(M, lookup(M, t, i, rows(M, 5, 32, at=1)), "out", "width")
    refused(M, lookup(M, t, i, rows(M, 5, 64)), "overlap")
    refused(M, lookup(M, t, i, rows(M, 5, 64, data=AT + 8 * GAP)), "overlap")
    refused(M, lookup(M, rows(M, 10, 64, M.E4M3), i, o), "block_rows")
    refused(M, lookup(M, rows(M, 10, 64, M.E4M3), i, o, None, 1), "table_scale")
    refused(M, lookup(M, t, i, o, AT + 3 * GAP, 1), "MASCOT_E4M3")
    reached_the_device(M, lookup(M, rows(M, 10, 64, M.E4M3), i, o, AT + 3 * GAP, 128))
    # two column halves of one matrix share no element
    reached_the_device(M, lookup(M, rows(M, 10, 64, stride=128), i, rows(M, 5, 64, stride=128, data=AT + 256)))
    refused(M, lookup(M, rows(M, 10, 64, stride=128), i, rows(M, 5, 64, stride=128, data=AT + 252)), "overlap")
    assert lookup(M, t, ids(M, 0), rows(M, 0, 64, at=1)) == M.OK       # nothing to do


def test_gradient_refuses(mascot):
    M = mascot

    def call(g, i, o, ws=AT + 4 * GAP, size=1 << 30, accumulate=0):
        return M.load().mascot_rows_gradient(g, i, 1.0, o, accumulate, ws, size, None, None)
    g, i, o = rows(M, 5, 64), ids(M, 5), rows(M, 10, 64, at=1)
    reached_the_device(M, call(g, i, o))
    refused(M, call(rows(M, 5, 64, M.E4M3), i, o), "grad")
    refused(M, call(rows(M, 4, 64), i, o), "grad", "each id")
    refused(M, call(g, i, rows(M, 10, 65, at=1)), "out", "width")
    refused(M, call(g, i, o, None), "workspace")
    refused(M, call(g, i, o, size=100), "workspace")
    refused(M, call(g, i, o, AT + 4 * GAP + 8), "workspace", "aligned")
    refused(M, call(g, i, o, AT + GAP), "workspace", "overlap")
    refused(M, call(g, i, o, AT), "workspace", "overlap")
    refused(M, call(g, i, rows(M, 10, 64)), "overlap")
    assert call(rows(M, 0, 64), ids(M, 0), o, accumulate=1) == M.OK
    reached_the_device(M, call(rows(M, 0, 64), ids(M, 0), o, None, 0))          # clears the table


def test_pair_loss_refuses(mascot):
    M = mascot

    def call(P, Q, u, i, j, beta=1.0, eps=0.0, outs=(AT + 5 * GAP, AT + 6 * GAP, AT + 7 * GAP), ref=None, w=None):
        return M.load().mascot_pair_loss(P, Q, u, i, j, beta, eps, ref, w, *outs, None, None)
    P, Q = rows(M, 10, 64), rows(M, 8, 64, at=1)
    u, i, j = ids(M, 5, 8), ids(M, 5, 9), ids(M, 5, 10)
    reached_the_device(M, call(P, Q, u, i, j))
    reached_the_device(M, call(P, Q, u, i, i, outs=(None, AT + 5 * GAP, None)))
    refused(M, call(P, rows(M, 8, 32, at=1), u, i, j), "one width")
    refused(M, call(P, rows(M, 8, 64, M.F16, 1), u, i, j), "one type")
    refused(M, call(P, rows(M, 8, 64, M.E4M3, 1), u, i, j), "Q")
    refused(M, call(P, Q, u, ids(M, 4, 9), j), "one count")
    for eps in (-0.1, 1.5, float("nan")):
        refused(M, call(P, Q, u, i, j, eps=eps), "smoothing")
    for beta in (float("inf"), float("nan")):
        refused(M, call(P, Q, u, i, j, beta=beta), "beta")
    refused(M, call(P, Q, u, i, j, outs=(None, None, None)), "no output")
    refused(M, call(P, Q, u, i, j, outs=(AT + 5 * GAP, AT + 5 * GAP + 8, None)), "overlap")
    refused(M, call(P, Q, u, i, j, outs=(AT + 5 * GAP, None, None), ref=AT + 5 * GAP), "reference", "overlap")
    refused(M, call(P, Q, u, i, j, outs=(AT, None, None)), "P", "overlap")
    refused(M, call(P, Q, u, i, j, outs=(AT + 5 * GAP + 2, None, None)), "address")
    assert call(P, Q, ids(M, 0), ids(M, 0), ids(M, 0)) == M.OK


def test_pair_gradient_refuses(mascot):
    M = mascot

    def call(P, Q, dP, dQ, u=ids(M, 5, 8), i=ids(M, 5, 9), j=ids(M, 5, 10), coef=AT + 11 * GAP, ws=AT + 4 * GAP, size=1 << 30):
        return M.load().mascot_pair_gradient(P, Q, u, i, j, coef, 1.0, dP, dQ, 0, ws, size, None, None)
    P, Q, dP, dQ = rows(M, 10, 64), rows(M, 8, 64, at=1), rows(M, 10, 64, at=2), rows(M, 8, 64, at=3)
    reached_the_device(M, call(P, Q, dP, dQ))
    refused(M, call(P, Q, dP, rows(M, 9, 64, at=3)), "shapes")
    refused(M, call(P, Q, dP, rows(M, 8, 64, M.BF16, 3)), "one type")
    refused(M, call(P, Q, dP, dP), "shapes")
    refused(M, call(P, Q, dP, rows(M, 8, 64, at=2)), "dP", "dQ", "overlap")
    refused(M, call(P, Q, rows(M, 10, 64, at=1), dQ), "overlap")
    refused(M, call(P, Q, dP, dQ, coef=None), "coef")
    refused(M, call(P, Q, dP, dQ, ws=AT + 11 * GAP), "coef", "overlap")
    refused(M, call(P, Q, dP, dQ, size=64), "workspace")
    refused(M, call(rows(M, 1 << 30, 64), rows(M, 1 << 30, 64, at=1), rows(M, 1 << 30, 64, at=2), rows(M, 1 << 30, 64, at=3)), "2^31")
    # the two gradients may be columns of one matrix
    reached_the_device(M, call(P, rows(M, 10, 64, at=1), rows(M, 10, 64, stride=128, at=2), rows(M, 10, 64, stride=128, data=AT + 2 * GAP + 256)))


def test_quantize_and_product_refuse(mascot):
    M = mascot

    def quantize(x, q, block_rows=1, scale=AT + 5 * GAP):
        return M.load().mascot_rows_quantize(x, block_rows, q, scale, None)
    x, q = rows(M, 10, 100), rows(M, 10, 100, M.E4M3, 1, 112)
    reached_the_device(M, quantize(x, q))
    refused(M, quantize(x, rows(M, 10, 100, 0, 1)), "q", "E4M3")
    refused(M, quantize(rows(M, 10, 100, M.E4M3), q), "x")
    refused(M, quantize(x, rows(M, 10, 101, M.E4M3, 1)), "q", "shape")
    refused(M, quantize(x, q, 2), "block_rows")
    refused(M, quantize(x, q, scale=None), "scale")
    refused(M, quantize(x, q, scale=AT), "overlap")
    refused(M, quantize(x, rows(M, 10, 100, M.E4M3, data=AT)), "overlap")
    assert quantize(rows(M, 0, 100), rows(M, 0, 100, M.E4M3, 1)) == M.OK

    def product(a, b, o, each=1, sa=AT + 5 * GAP, sb=AT + 6 * GAP):
        return M.load().mascot_rows_product(a, sa, b, sb, each, o, None, None)
    a, b, o = rows(M, 6, 100, M.E4M3, 0, 112), rows(M, 10, 100, M.E4M3, 1, 112), rows(M, 6, 10, M.BF16, 2)
    reached_the_device(M, product(a, b, o))
    reached_the_device(M, product(a, b, o, 128))
    refused(M, product(rows(M, 6, 100, M.F16), b, o), "a", "E4M3")
    refused(M, product(a, rows(M, 10, 99, M.E4M3, 1, 112), o), "one width")
    refused(M, product(a, b, rows(M, 6, 11, 0, 2)), "out")
    refused(M, product(a, b, rows(M, 6, 10, M.E4M3, 2)), "out")
    refused(M, product(a, b, rows(M, 6, 10, 0, 2, 9)), "out", "stride")
    refused(M, product(a, b, o, 64), "b_block_rows")
    refused(M, product(a, b, o, sa=None), "null")
    refused(M, product(rows(M, 6, 100, M.E4M3, 0, 104), b, o), "16 bytes")
    refused(M, product(a, rows(M, 10, 100, M.E4M3, stride=112, data=AT + GAP + 8), o), "16 bytes")
    refused(M, product(a, b, rows(M, 6, 10, data=AT)), "overlap")
    assert product(rows(M, 0, 100, M.E4M3, 0, 112), b, rows(M, 0, 10, 0, 2)) == M.OK


def test_workspace_sizes(mascot):
    M, n = mascot, C.c_uint64()
    lib = M.load()
    assert lib.mascot_rows_gradient_workspace(0, 1000, 64, C.byref(n)) == M.OK and n.value == 0
    last = 0
    for count in (1, 100, 12_288, 12_289, 1 << 20, 1 << 22):
        assert lib.mascot_rows_gradient_workspace(count, 1000, 64, C.byref(n)) == M.OK
        assert n.value > last
        last = n.value
    assert last < 64 * (1 << 22)                     # far less than the gradients themselves
    for args in ((1 << 31, 10, 64), (10, 1 << 31, 64), (10, 10, 0), (10, 10, 1 << 20)):
        refused(M, lib.mascot_rows_gradient_workspace(*args, C.byref(n)), "out of range")
    refused(M, lib.mascot_rows_gradient_workspace(1, 1, 1, None), "null")
    refused(M, lib.mascot_pair_gradient_workspace(1 << 30, 10, 10, 64, C.byref(n)), "out of range")
    refused(M, lib.mascot_pair_gradient_workspace(10, 1 << 30, 1 << 30, 64, C.byref(n)), "out of range")
    assert lib.mascot_pair_gradient_workspace(10, 10, 10, 64, C.byref(n)) == M.OK and n.value > 0


def test_struct_layout(mascot):
    assert C.sizeof(mascot.Rows) == 32 and C.sizeof(mascot.Ids) == 24


def test_tensors_off_the_gpu_are_refused(mascot):
    import torch
    x = torch.zeros(3, 64)
    i = torch.zeros(3, dtype=torch.int32)
    q = x.to(torch.float8_e4m3fn)
    s = torch.ones(1, 3)
    for f in (lambda: mascot.rows_lookup(x, i), lambda: mascot.rows_gradient(x, i, 3), lambda: mascot.pair_loss(x, x, i, i, i),
              lambda: mascot.pair_gradient(x, x, i, i, i, torch.zeros(3)), lambda: mascot.rows_quantize(x), lambda: mascot.rows_product(q, s, q, s)):
        with pytest.raises(mascot.MascotError) as e:
            f()
        assert e.value.status == mascot.ERR_BAD_ARG and "GPU" in str(e.value)


def test_a_reader_that_gave_up_spoils_nothing(tmp_path):
    """csrc/reader.h, the rule of the scores' kernel for a warp whose wait ran out: whatever the order in which warps take their turns, what
    the others store is right or NaN, and all come to their end.  Going on as if nothing had been leaves wrong finite scores."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = str(tmp_path / "reader_check")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-I", os.path.join(root, "icdm-2021_mascot_b200", "csrc"), os.path.join(root, "tests", "reader_check.cpp"), "-o", exe])

    def run(rule, barrier, group):
        return [int(x) for x in subprocess.run([exe, rule, str(barrier), str(group)], capture_output=True, text=True, check=True).stdout.split()]
    for group in (1, 2, 4):
        whole = run("reader", -1, group)
        assert whole[:2] == [0, 0] and whole[2] == 400 * 40 * 4 * group              # nothing gives up: all scores, all right
        for barrier in (0, 1):
            wrong, nan, right = run("reader", barrier, group)
            assert wrong == 0 and nan > 0 and right > 0 and nan + right == whole[2]
    assert run("always", 0, 1)[0] > 0 and run("always", 1, 2)[0] > 0


def test_odd_addresses_are_refused(mascot):
    """Every pointer to 4-byte elements, the flag word of every entry included: a load or an atomic at an odd address would fault."""
    M, lib = mascot, mascot.load()
    t, i, o = rows(M, 10, 64), ids(M, 5), rows(M, 5, 64, at=1)
    e4m3, g = rows(M, 10, 64, M.E4M3), rows(M, 5, 64, at=2)
    u, p, n = ids(M, 5, 8), ids(M, 5, 9), ids(M, 5, 10)
    dP, dQ = rows(M, 10, 64, at=3), rows(M, 10, 64, at=4)
    a, b, s = rows(M, 5, 64, M.E4M3), rows(M, 10, 64, M.E4M3, 1), rows(M, 5, 10, M.BF16, 2)
    x, q = rows(M, 10, 64, at=5), rows(M, 10, 64, M.E4M3, 6)
    f = [AT + k * GAP for k in range(11, 16)]
    calls = {                              # a call with its 4-byte pointers, in order; each name as in the messages
        "lookup": (lambda w: lib.mascot_rows_lookup(e4m3, w[0], 1, i, 1.0, o, w[1], None), ["table_scale", "flags"]),
        "gradient": (lambda w: lib.mascot_rows_gradient(g, i, 1.0, dP, 0, AT + 7 * GAP, 1 << 30, w[0], None), ["flags"]),
        "loss": (lambda w: lib.mascot_pair_loss(t, t, u, p, n, 1.0, 0.0, w[0], w[1], w[2], None, None, w[3], None), ["reference", "weight", "loss", "flags"]),
        "pairs": (lambda w: lib.mascot_pair_gradient(t, t, u, p, n, w[0], 1.0, dP, dQ, 0, AT + 7 * GAP, 1 << 30, w[1], None), ["coef", "flags"]),
        "quantize": (lambda w: lib.mascot_rows_quantize(x, 1, q, w[0], None), ["scale"]),
        "product": (lambda w: lib.mascot_rows_product(a, w[0], b, w[1], 1, s, w[2], None), ["a_scale", "b_scale", "flags"]),
    }
    for call, names in calls.values():
        at = f[:len(names)]
        reached_the_device(M, call(at))
        for k, name in enumerate(names):
            for off in (1, 2, 3):
                refused(M, call(at[:k] + [at[k] + off] + at[k + 1:]), name, "address")


def test_kernels_end_with_no_copy_under_way():
    """Whatever a kernel copies into shared memory asynchronously has arrived when it ends: the memory is another block's then."""
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "icdm-2021_mascot_b200", "csrc")
    seen = []
    for name in sorted(os.listdir(csrc)):
        if name.endswith(".cu"):
            for body in re.split(r"(?=\n(?:template <[^\n]*>\n)?__global__ )", open(os.path.join(csrc, name)).read())[1:]:
                if re.search(r"cp_commit\(|fetch_piece<|fetch_word\(|cp\.async\.commit", body):
                    kernel = re.search(r"(\w+)\(const", body).group(1)
                    seen.append(kernel)
                    assert re.search(r"cp\.async\.wait_all|cp_wait<0>", body), f"{name}: {kernel}"
    assert {"reduce_kernel", "product_kernel"} <= set(seen), seen


def test_what_autograd_is_told(mascot):
    """The two halves of it on the CPU, where the calls themselves stop at the device."""
    import torch
    leaf = torch.zeros(2, 3, requires_grad=True)
    for refuse in (lambda: mascot._rows("P", leaf, leaf.device), lambda: mascot._plain("weight", leaf[0], torch.float32, leaf.device, (3,))):
        with pytest.raises(mascot.MascotError) as e:
            refuse()
        assert e.value.status == mascot.ERR_BAD_ARG and "requires a gradient" in str(e.value)
        with torch.no_grad():
            refuse()
    t = torch.zeros(4, 4)
    was = t._version
    mascot._changed(None, t[1:])
    assert t._version == was + 1
    with torch.inference_mode():
        inside = torch.zeros(2)
    mascot._changed(inside)


def test_workspace_on_both_sides_of_the_one_launch_sort(mascot):
    """Up to 32,768 entries one cluster sorts, and needs neither keys nor counts; one entry more needs both: 4 bytes an entry, and 1024 counts
    for each of 17 tiles of 2,048 entries and their sums."""
    lib, n = mascot.load(), C.c_uint64()

    def rows(count):
        assert lib.mascot_rows_gradient_workspace(count, 1000, 64, C.byref(n)) == mascot.OK
        return n.value

    def pairs(count):
        assert lib.mascot_pair_gradient_workspace(count, 600, 400, 64, C.byref(n)) == mascot.OK
        return n.value
    more = 4 * 32_769 + 4 * 1024 * 17 + 4 * 1024
    assert more <= rows(32_769) - rows(32_768) < more + 5000
    assert more <= pairs(10_923) - pairs(10_922) < more + 10_000            # 32,769 and 32,766 entries
    assert rows(32_768) - rows(32_767) < 5000 and rows(32_770) - rows(32_769) < 5000
