"""ctypes binding of libmascot.so - the thin Python face of the C ABI in include/mascot.h.

Used by the tests, the benchmark and the smoke test; the production host code is the C++
command line (cli/quantized_mf.cpp, cli/test_mf.cpp).  There is no fallback: if the shared library
is missing or no CUDA device is usable, calls raise.
"""
import ctypes as C
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("MASCOT_LIB_PATH", os.path.join(HERE, "libmascot.so"))

RATING = np.dtype([("r", np.float32), ("u", np.uint32), ("i", np.uint32)])

V_MASCOT, V_AFP, V_MUPPET, V_MPT, V_SGD, V_NAIVE, V_MEMQUANT, V_SWITCH_ONLY = 1, 2, 3, 4, 5, 6, 7, 8

OK, ERR_BAD_ARG, ERR_CUDA, ERR_OOM, ERR_STATE, ERR_NO_DEVICE, ERR_TIMEOUT, ERR_UNSUPPORTED, ERR_COMM = \
    0, -1, -2, -3, -4, -5, -6, -7, -8

EXPORTS = [
    "mascot_abi_info", "mascot_config_default", "mascot_create", "mascot_destroy", "mascot_last_error", "mascot_status_string",
    "mascot_set_ratings", "mascot_init_factors", "mascot_set_factors", "mascot_train_epoch", "mascot_eval_rmse",
    "mascot_get_factors", "mascot_get_group_info", "mascot_get_index_maps", "mascot_get_sample_stats",
    "mascot_get_test_ratings", "mascot_promote_group", "mascot_reload_train", "mascot_stream_source_index", "mascot_get_stream_order", "mascot_rmse_host", "mascot_rmse_device", "mascot_rmse_device_noalloc",
    "mascot_set_ratings_sharded", "mascot_is_check_epoch", "mascot_stats_begin", "mascot_train_segment", "mascot_stats_fetch",
    "mascot_stats_apply", "mascot_item_rows", "mascot_sync", "mascot_get_stream", "mascot_eval_sq_error", "mascot_train_epoch_streamed",
    "mascot_release_scratch", "mascot_release_cached", "mascot_comm_unique_id", "mascot_shard_init", "mascot_shard_set_ratings", "mascot_shard_train_epoch",
    "mascot_shard_eval_rmse", "mascot_shard_gather_factors", "mascot_shard_info", "mascot_shard_schedule", "mascot_probe_read_bandwidth", "mascot_get_timings", "mascot_get_worker_count",
    "mascot_rows_lookup", "mascot_rows_gradient", "mascot_rows_gradient_workspace", "mascot_pair_loss", "mascot_pair_gradient",
    "mascot_pair_gradient_workspace", "mascot_rows_quantize", "mascot_rows_product",
]

COMM_ID_BYTES = 128


class Config(C.Structure):
    _fields_ = [
        ("lambda_", C.c_float), ("learning_rate", C.c_float), ("decay", C.c_float), ("sample_ratio", C.c_float),
        ("error_threshold", C.c_float), ("interval", C.c_uint32), ("user_group_num", C.c_uint32),
        ("item_group_num", C.c_uint32), ("k", C.c_uint32), ("num_workers", C.c_uint32), ("epoch", C.c_uint32),
        ("thread_block_size", C.c_uint32), ("version", C.c_uint32), ("is_yahoo", C.c_uint32),
        ("deterministic", C.c_uint32), ("shuffle", C.c_uint32), ("seed", C.c_uint64), ("device", C.c_int32),
        ("muppet_width", C.c_uint32), ("plain_user_stores", C.c_uint32), ("l2_item_window", C.c_uint32), ("no_class_partition", C.c_uint32), ("run_window_log2", C.c_uint32), ("reserved", C.c_uint32 * 2),
    ]


class EpochStats(C.Structure):
    _fields_ = [
        ("updates", C.c_uint64), ("lr", C.c_float), ("kernel_ms", C.c_float), ("total_ms", C.c_float),
        ("error_check", C.c_uint32), ("promoted_user_groups", C.c_uint32), ("promoted_item_groups", C.c_uint32),
        ("kernel_launches", C.c_uint32), ("workers", C.c_uint32), ("pass_bits", C.c_uint32),
        ("algorithmic_bytes", C.c_uint64),
    ]


class Rows(C.Structure):
    """mascot_rows: a matrix in device memory."""
    _fields_ = [("data", C.c_void_p), ("rows", C.c_uint64), ("stride", C.c_uint64), ("width", C.c_uint32), ("type", C.c_uint32)]


class Ids(C.Structure):
    """mascot_ids: a vector of ids in device memory."""
    _fields_ = [("data", C.c_void_p), ("count", C.c_uint64), ("bits", C.c_uint32), ("reserved", C.c_uint32)]


class MascotError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"libmascot status {status}: {message}")
        self.status = status


_lib = None


def load():
    """dlopen libmascot.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise OSError(f"{LIB_PATH} is missing - run `python icdm-2021_mascot_b200/build.py`")
        L = C.CDLL(LIB_PATH)
        L.mascot_last_error.restype = C.c_char_p
        L.mascot_last_error.argtypes = [C.c_void_p]
        L.mascot_status_string.restype = C.c_char_p
        L.mascot_status_string.argtypes = [C.c_int]
        rows, ids, ptr = C.POINTER(Rows), C.POINTER(Ids), C.c_void_p
        L.mascot_rows_lookup.argtypes = [rows, ptr, C.c_uint32, ids, C.c_float, rows, ptr, ptr]
        L.mascot_rows_gradient.argtypes = [rows, ids, C.c_float, rows, C.c_int, ptr, C.c_uint64, ptr, ptr]
        L.mascot_rows_gradient_workspace.argtypes = [C.c_uint64, C.c_uint64, C.c_uint32, C.POINTER(C.c_uint64)]
        L.mascot_pair_loss.argtypes = [rows, rows, ids, ids, ids, C.c_float, C.c_float, ptr, ptr, ptr, ptr, ptr, ptr, ptr]
        L.mascot_pair_gradient.argtypes = [rows, rows, ids, ids, ids, ptr, C.c_float, rows, rows, C.c_int, ptr, C.c_uint64, ptr, ptr]
        L.mascot_pair_gradient_workspace.argtypes = [C.c_uint64, C.c_uint64, C.c_uint64, C.c_uint32, C.POINTER(C.c_uint64)]
        L.mascot_rows_quantize.argtypes = [rows, C.c_uint32, rows, ptr, ptr]
        L.mascot_rows_product.argtypes = [rows, ptr, rows, ptr, C.c_uint32, rows, ptr, ptr]
        ver, csz, ssz = C.c_uint32(), C.c_uint32(), C.c_uint32()
        L.mascot_abi_info(C.byref(ver), C.byref(csz), C.byref(ssz))
        if (csz.value, ssz.value) != (C.sizeof(Config), C.sizeof(EpochStats)):
            raise OSError(f"libmascot ABI mismatch: library structs are {csz.value}/{ssz.value} bytes, "
                          f"binding expects {C.sizeof(Config)}/{C.sizeof(EpochStats)}")
        _lib = L
    return _lib


def _ptr(a):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def default_config(**overrides):
    cfg = Config()
    load().mascot_config_default(C.byref(cfg))
    for key, val in overrides.items():
        setattr(cfg, "lambda_" if key in ("lambda", "lam") else key, val)
    return cfg


def as_ratings(a):
    a = np.ascontiguousarray(a)
    if a.dtype != RATING:
        a = a.reshape(-1, 3).astype(np.uint32, copy=False).view(RATING).reshape(-1)
    return a


def make_ratings(u, i, r):
    out = np.empty(len(r), RATING)
    out["u"], out["i"], out["r"] = u, i, r
    return out


class Engine:
    """One libmascot handle."""

    def __init__(self, cfg):
        self._lib = load()
        self.cfg = cfg
        self._h = C.c_void_p()
        rc = self._lib.mascot_create(C.byref(cfg), C.byref(self._h))
        if rc != OK:
            raise MascotError(rc, self._lib.mascot_last_error(None).decode())
        self.k = int(cfg.k)
        self.n_users = self.n_items = 0
        self.n_train = self.n_test = 0

    def _check(self, rc):
        if rc != OK:
            raise MascotError(rc, self._lib.mascot_last_error(self._h).decode())

    def close(self):
        if self._h:
            self._lib.mascot_destroy(self._h)
            self._h = C.c_void_p()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_ratings(self, train, test, n_users, n_items):
        train, test = as_ratings(train), as_ratings(test)
        self._check(self._lib.mascot_set_ratings(self._h, _ptr(train), C.c_uint64(train.size), _ptr(test),
                                                 C.c_uint64(test.size), C.c_uint32(n_users), C.c_uint32(n_items)))
        self.n_users, self.n_items, self.n_train, self.n_test = n_users, n_items, train.size, test.size

    def set_ratings_raw(self, train_ptr, n_train, test_ptr, n_test, n_users, n_items):
        """Same call with raw host addresses (e.g. pinned buffers owned by the caller)."""
        self._check(self._lib.mascot_set_ratings(self._h, C.c_void_p(train_ptr), C.c_uint64(n_train), C.c_void_p(test_ptr),
                                                 C.c_uint64(n_test), C.c_uint32(n_users), C.c_uint32(n_items)))
        self.n_users, self.n_items, self.n_train, self.n_test = n_users, n_items, n_train, n_test

    # ---- sharded training building blocks ----
    def set_ratings_sharded(self, train, segment_offsets, test, n_users, n_items, user_degree=None, item_degree=None):
        train, test = as_ratings(train), as_ratings(test)
        seg = np.ascontiguousarray(segment_offsets, np.uint64)
        ud = None if user_degree is None else np.ascontiguousarray(user_degree, np.uint32)
        idg = None if item_degree is None else np.ascontiguousarray(item_degree, np.uint32)
        self._check(self._lib.mascot_set_ratings_sharded(self._h, _ptr(train), C.c_uint64(train.size), _ptr(seg), C.c_uint32(seg.size - 1),
                                                         _ptr(test), C.c_uint64(test.size), C.c_uint32(n_users), C.c_uint32(n_items),
                                                         _ptr(ud), _ptr(idg)))
        self.n_users, self.n_items, self.n_train, self.n_test = n_users, n_items, train.size, test.size

    def is_check_epoch(self, epoch):
        return bool(self._lib.mascot_is_check_epoch(self._h, C.c_uint32(epoch)))

    def stats_begin(self):
        self._check(self._lib.mascot_stats_begin(self._h))

    def train_segment(self, epoch, segment, collect_stats=False, wait=True):
        st = EpochStats() if wait else None
        self._check(self._lib.mascot_train_segment(self._h, C.c_uint32(epoch), C.c_uint32(segment), C.c_uint32(1 if collect_stats else 0),
                                                   C.byref(st) if wait else None))
        return st

    def stats_fetch(self):
        ug, ig = len(self.group_info(0)[0]), len(self.group_info(1)[0])
        out = [np.empty(ug * self.k, np.float32), np.empty(ig * self.k, np.float32), np.empty(ug, np.float32), np.empty(ig, np.float32)]
        self._check(self._lib.mascot_stats_fetch(self._h, *[_ptr(a) for a in out]))
        return out

    def stats_apply(self, epoch, gsum_p, gsum_q, nsum_p, nsum_q):
        arrs = [np.ascontiguousarray(a, np.float32) for a in (gsum_p, gsum_q, nsum_p, nsum_q)]
        pu, pi = C.c_uint32(), C.c_uint32()
        self._check(self._lib.mascot_stats_apply(self._h, C.c_uint32(epoch), *[_ptr(a) for a in arrs], C.byref(pu), C.byref(pi)))
        return pu.value, pi.value

    def item_rows(self, row_begin, row_end):
        p16, b16, p32, b32 = C.c_void_p(), C.c_uint64(), C.c_void_p(), C.c_uint64()
        self._check(self._lib.mascot_item_rows(self._h, C.c_uint32(row_begin), C.c_uint32(row_end), C.byref(p16), C.byref(b16),
                                               C.byref(p32), C.byref(b32)))
        return (p16.value or 0, b16.value), (p32.value or 0, b32.value)

    def sync(self):
        self._check(self._lib.mascot_sync(self._h))

    def stream_handle(self):
        """Address of the engine's cudaStream_t (for ordering a caller's own device work on it)."""
        st = C.c_void_p()
        self._check(self._lib.mascot_get_stream(self._h, C.byref(st)))
        return st.value or 0

    def eval_sq_error(self):
        s, n = C.c_double(), C.c_uint64()
        self._check(self._lib.mascot_eval_sq_error(self._h, C.byref(s), C.byref(n)))
        return s.value, n.value

    def reload_train_raw(self, train_ptr, n_train):
        """Replace the training stream from a raw host address (the per-step input path)."""
        self._check(self._lib.mascot_reload_train(self._h, C.c_void_p(train_ptr), C.c_uint64(n_train)))
        self.n_train = n_train

    def train_epoch_streamed_raw(self, epoch, train_ptr, n_train):
        """One epoch over a rating array in host memory (upload overlapped with the updates)."""
        st = EpochStats()
        self._check(self._lib.mascot_train_epoch_streamed(self._h, C.c_uint32(epoch), C.c_void_p(train_ptr), C.c_uint64(n_train), C.byref(st)))
        self.n_train = n_train
        return st

    def train_epoch_streamed(self, epoch, train):
        train = as_ratings(train)
        return self.train_epoch_streamed_raw(epoch, train.ctypes.data, train.size)

    def reload_train(self, train):
        train = as_ratings(train)
        self.reload_train_raw(train.ctypes.data, train.size)

    # ---- sharded training inside the library (one engine per GPU, NCCL between them) ----
    def shard_init(self, comm_id, rank, world, blocks_per_gpu=1, timeout_ms=0):
        """Join the group identified by the 128 bytes `comm_id` (see comm_unique_id)."""
        buf = (C.c_ubyte * COMM_ID_BYTES).from_buffer_copy(bytes(comm_id))
        self._check(self._lib.mascot_shard_init(self._h, buf, C.c_uint32(rank), C.c_uint32(world), C.c_uint32(blocks_per_gpu),
                                                C.c_uint32(timeout_ms)))

    def shard_set_ratings(self, train, test, n_users, n_items):
        train, test = as_ratings(train), as_ratings(test)
        self.shard_set_ratings_raw(train.ctypes.data, train.size, test.ctypes.data, test.size, n_users, n_items)

    def shard_set_ratings_raw(self, train_ptr, n_train, test_ptr, n_test, n_users, n_items):
        self._check(self._lib.mascot_shard_set_ratings(self._h, C.c_void_p(train_ptr), C.c_uint64(n_train), C.c_void_p(test_ptr),
                                                       C.c_uint64(n_test), C.c_uint32(n_users), C.c_uint32(n_items)))
        info = self.shard_info()
        self.n_users, self.n_items, self.n_train, self.n_test = n_users, n_items, info["local_ratings"], info["local_test_ratings"]

    def shard_train_epoch(self, epoch):
        st = EpochStats()
        self._check(self._lib.mascot_shard_train_epoch(self._h, C.c_uint32(epoch), C.byref(st)))
        return st

    def shard_eval_rmse(self):
        v = C.c_double()
        self._check(self._lib.mascot_shard_eval_rmse(self._h, C.byref(v)))
        return v.value

    def shard_gather_factors(self):
        self._check(self._lib.mascot_shard_gather_factors(self._h))

    def shard_info(self):
        r, w, b, n, nt, sent = C.c_uint32(), C.c_uint32(), C.c_uint32(), C.c_uint64(), C.c_uint64(), C.c_uint64()
        self._check(self._lib.mascot_shard_info(self._h, C.byref(r), C.byref(w), C.byref(b), C.byref(n), C.byref(nt), C.byref(sent)))
        return dict(rank=r.value, world=w.value, blocks=b.value, local_ratings=n.value, local_test_ratings=nt.value, bytes_sent=sent.value)

    def release_scratch(self):
        self._check(self._lib.mascot_release_scratch(self._h))

    def init_factors(self):
        self._check(self._lib.mascot_init_factors(self._h))

    def set_factors(self, P, Q):
        P = np.ascontiguousarray(P, np.float32)
        Q = np.ascontiguousarray(Q, np.float32)
        assert P.size == self.n_users * self.k and Q.size == self.n_items * self.k
        self._check(self._lib.mascot_set_factors(self._h, _ptr(P), _ptr(Q)))

    def train_epoch(self, epoch):
        st = EpochStats()
        self._check(self._lib.mascot_train_epoch(self._h, C.c_uint32(epoch), C.byref(st)))
        return st

    def eval_rmse(self):
        v = C.c_double()
        self._check(self._lib.mascot_eval_rmse(self._h, C.byref(v)))
        return v.value

    def get_factors(self, order=0):
        P = np.empty((self.n_users, self.k), np.float32)
        Q = np.empty((self.n_items, self.k), np.float32)
        self._check(self._lib.mascot_get_factors(self._h, _ptr(P), _ptr(Q), C.c_int(order)))
        return P, Q

    def group_info(self, side):
        n = C.c_uint32()
        self._check(self._lib.mascot_get_group_info(self._h, C.c_int(side), C.byref(n), None, None, None))
        end = np.empty(n.value, np.uint32)
        prec = np.empty(n.value, np.uint8)
        err = np.empty(n.value, np.float32)
        self._check(self._lib.mascot_get_group_info(self._h, C.c_int(side), C.byref(n), _ptr(end), _ptr(prec), _ptr(err)))
        return end, prec, err

    def promote_group(self, side, group):
        self._check(self._lib.mascot_promote_group(self._h, C.c_int(side), C.c_uint32(group)))

    def index_maps(self):
        u = np.empty(self.n_users, np.uint32)
        i = np.empty(self.n_items, np.uint32)
        self._check(self._lib.mascot_get_index_maps(self._h, _ptr(u), _ptr(i)))
        return u, i

    def sample_stats(self):
        ug, ig = len(self.group_info(0)[0]), len(self.group_info(1)[0])
        gp = np.empty(ug * self.k, np.float32)
        gq = np.empty(ig * self.k, np.float32)
        np_ = np.empty(ug, np.float32)
        nq = np.empty(ig, np.float32)
        self._check(self._lib.mascot_get_sample_stats(self._h, _ptr(gp), _ptr(gq), _ptr(np_), _ptr(nq)))
        return gp, gq, np_, nq

    def test_ratings(self, order=1):
        out = np.empty(self.n_test, RATING)
        self._check(self._lib.mascot_get_test_ratings(self._h, _ptr(out), C.c_int(order)))
        return out

    def stream_order(self):
        out = np.empty(self.n_train, np.uint32)
        self._check(self._lib.mascot_get_stream_order(self._h, _ptr(out)))
        return out

    def stream_source_index(self, pos):
        v = C.c_uint64()
        self._check(self._lib.mascot_stream_source_index(self._h, C.c_uint64(pos), C.byref(v)))
        return v.value


def write_binary_ratings(path, records, n_users, n_items):
    """Write the binary rating file of the command-line tools (cli/io_formats.h): `records` is an (n, 3)
    uint32 view or a RATING array with compact ids."""
    recs = as_ratings(records)
    header = np.zeros(1, np.dtype([("magic", "<u4"), ("version", "<u4"), ("n", "<u8"), ("n_users", "<u4"), ("n_items", "<u4"),
                                   ("flags", "<u4"), ("reserved", "<u4")]))
    header["magic"], header["version"], header["n"] = 0x5243534d, 1, recs.size
    header["n_users"], header["n_items"], header["flags"] = n_users, n_items, 1
    with open(path, "wb") as f:
        f.write(header.tobytes())
        recs.tofile(f)


def comm_unique_id():
    """128 opaque bytes naming a new group of sharded engines (made by one rank, carried to the others)."""
    buf = (C.c_ubyte * COMM_ID_BYTES)()
    rc = load().mascot_comm_unique_id(buf)
    if rc != OK:
        raise MascotError(rc, load().mascot_last_error(None).decode())
    return bytes(buf)


def shard_schedule(world, blocks_per_gpu, rank, step):
    """(block trained, rank it is sent to, block that arrives, rank it comes from) - needs no device."""
    out = [C.c_uint32() for _ in range(4)]
    rc = load().mascot_shard_schedule(C.c_uint32(world), C.c_uint32(blocks_per_gpu), C.c_uint32(rank), C.c_uint32(step),
                                      *[C.byref(o) for o in out])
    if rc != OK:
        raise MascotError(rc, "bad schedule arguments")
    return tuple(o.value for o in out)


def probe_read_bandwidth(nbytes, passes=20, device=0):
    """GB/s of 128-bit L2-only loads over a buffer of `nbytes` (L2-resident when small, HBM when large)."""
    v = C.c_double()
    rc = load().mascot_probe_read_bandwidth(C.c_int(device), C.c_uint64(nbytes), C.c_uint32(passes), C.byref(v))
    if rc != OK:
        raise MascotError(rc, load().mascot_last_error(None).decode())
    return v.value


def release_cached():
    """Gives back the device memory, pinned memory and threads that the library keeps between calls."""
    rc = load().mascot_release_cached()
    if rc != OK:
        raise MascotError(rc, load().mascot_last_error(None).decode())


def rmse_host(P, Q, test, k, device=0):
    """Handle-free evaluation of fp32 factors on host buffers (the test_mf path)."""
    L = load()
    P = np.ascontiguousarray(P, np.float32)
    Q = np.ascontiguousarray(Q, np.float32)
    test = as_ratings(test)
    v = C.c_double()
    rc = L.mascot_rmse_host(_ptr(P), C.c_uint32(P.size // k), _ptr(Q), C.c_uint32(Q.size // k), C.c_uint32(k),
                            _ptr(test), C.c_uint64(test.size), C.c_int(device), C.byref(v))
    if rc != OK:
        raise MascotError(rc, L.mascot_last_error(None).decode())
    return v.value


# ---- operators on factor rows in device memory: torch tensors in, torch tensors out, on torch's current stream ----
# Outputs that the caller does not hand over, and scratch, come from torch's allocator, so that the calls can be captured
# into a torch.cuda.graph.  `flags` is an int32 tensor of one element that gathers FLAG_BAD_ID and FLAG_GAVE_UP.
# Autograd does not see these calls, and a gradient must not get lost in one: while gradients are recorded, a tensor that requires one is
# refused (as torch does for its own calls with out=), and what a call writes into counts as changed.

F32, F16, BF16, E4M3 = 0, 1, 2, 3
FLAG_BAD_ID, FLAG_GAVE_UP = 1, 2
_ops = None


class _Ops:
    """torch and what the calls below look up in it, once."""
    def __init__(self):
        import torch
        self.torch = torch
        self.types = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3}
        self.bits = {torch.int32: 32, torch.int64: 64}
        self.recording = torch.is_grad_enabled
        self.changed = torch.autograd.graph.increment_version
        # the raw handle where torch offers it: the stream object around it costs 2 us a call
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _torch_ops():
    global _ops
    if _ops is None:
        _ops = _Ops()
    return _ops


def _refuse(message):
    raise MascotError(ERR_BAD_ARG, message)


def _unrecorded(what, t):
    """Refuses a tensor that requires a gradient while gradients are recorded."""
    if _torch_ops().recording():
        _refuse(f"{what}: requires a gradient, which this call does not record: make it under torch.no_grad(), or with {what}.detach(); "
                "rows_gradient and pair_gradient compute the gradients of rows_lookup and pair_loss")


def _changed(*tensors):
    """Tells autograd that a call has written into these tensors of the caller's (None: not the caller's)."""
    for t in tensors:
        if t is not None and not t.is_inference():
            _torch_ops().changed(t)


def _rows(what, t, device):
    """The Rows of a 2-d tensor on `device` whose rows are contiguous."""
    if t.requires_grad:
        _unrecorded(what, t)
    kind = _torch_ops().types.get(t.dtype)
    if kind is None:
        _refuse(f"{what}: must be float32, float16, bfloat16 or float8_e4m3fn, not {t.dtype}")
    if t.dim() != 2:
        _refuse(f"{what}: must have two dimensions")
    if t.device != device:
        _refuse(f"{what}: is on {t.device}, not on {device}")
    rows, width = t.shape
    stride, step = t.stride()
    if width > 1 and step != 1:
        _refuse(f"{what}: elements of a row must lie one after the other")
    if rows > 1 and stride < width:
        _refuse(f"{what}: rows overlap")
    return Rows(t.data_ptr(), rows, stride if rows > 1 else max(width, stride), width, kind)


def _id_vector(what, t, device):
    bits = _torch_ops().bits.get(t.dtype)
    if bits is None:
        _refuse(f"{what}: must be int32 or int64, not {t.dtype}")
    if t.dim() != 1 or not t.is_contiguous():
        _refuse(f"{what}: must be a contiguous vector")
    if t.device != device:
        _refuse(f"{what}: is on {t.device}, not on {device}")
    return Ids(t.data_ptr(), t.shape[0], bits, 0)


def _plain(what, t, dtype, device, shape):
    """Address of a contiguous tensor of that type, device and shape; None stays None."""
    if t is None:
        return None
    if t.requires_grad:
        _unrecorded(what, t)
    if t.dtype != dtype or t.device != device or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        _refuse(f"{what}: must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    return t.data_ptr()


def _flag_word(flags, device):
    return _plain("flags", flags, _torch_ops().torch.int32, device, (1,))


def _device_of(what, t):
    if not t.is_cuda:
        _refuse(f"{what}: must be on a GPU; libmascot has no CPU path")
    return t.device


def _call(device, name, *args):
    """A call on `device`, on torch's current stream there."""
    ops = _torch_ops()
    cuda, f = ops.torch.cuda, getattr(load(), name)
    if cuda.current_device() == device.index:
        rc = f(*args, ops.stream(device.index))
    else:
        with cuda.device(device):
            rc = f(*args, ops.stream(device.index))
    if rc != OK:
        raise MascotError(rc, load().mascot_last_error(None).decode())


def _result(what, out, shape, dtype, like):
    """`out` where it fits, else a new tensor on the device of `like`."""
    if out is None:
        return like.new_empty(shape) if dtype == like.dtype else like.new_empty(shape, dtype=dtype)
    if tuple(out.shape) != tuple(shape):
        _refuse(f"{what}: must have shape {tuple(shape)}")
    if dtype is not None and out.dtype != dtype:
        _refuse(f"{what}: must be {dtype}")
    return out


def _scale_rows(what, scale, rows, width, device):
    """Rows that share a scale (1 or 128), by the shape of `scale`: [column blocks, row blocks]."""
    blocks = -(-width // 128)
    each = 128 if rows > 1 and tuple(scale.shape) == (blocks, -(-rows // 128)) else 1
    return each, _plain(what, scale, _torch_ops().torch.float32, device, (blocks, -(-rows // each)))


def rows_lookup(table, ids, scale=1.0, table_scale=None, out=None, out_dtype=None, flags=None):
    """out[j] = scale * table[ids[j]], zeros where ids[j] is -1 (mascot_rows_lookup).  A float8_e4m3fn table comes with its
    scales, `table_scale` of rows_quantize; the result is float32 then unless out_dtype says otherwise."""
    device = _device_of("table", table)
    t, i = _rows("table", table, device), _id_vector("ids", ids, device)
    each, ts = 0, None
    if table_scale is not None:
        each, ts = _scale_rows("table_scale", table_scale, t.rows, t.width, device)
    if out_dtype is None and out is None:
        out_dtype = _torch_ops().torch.float32 if t.type == E4M3 else table.dtype
    given, out = out, _result("out", out, (i.count, t.width), out_dtype, table)
    _call(device, "mascot_rows_lookup", t, ts, each, i, scale, _rows("out", out, device), _flag_word(flags, device))
    _changed(given, flags)
    return out


def _workspace(workspace, name, like, device, *sizes):
    need = C.c_uint64()
    if getattr(load(), name)(*sizes, C.byref(need)) != OK:
        _refuse(load().mascot_last_error(None).decode())
    if workspace is None:
        workspace = like.new_empty(need.value, dtype=_torch_ops().torch.uint8)
    elif not workspace.is_contiguous() or workspace.device != device:
        _refuse(f"workspace: must be a contiguous tensor on {device}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def rows_gradient(grad, ids, rows, scale=1.0, out=None, out_dtype=None, accumulate=False, workspace=None, flags=None):
    """out[r] = scale * sum of grad[j] over the j with ids[j] == r, for r < rows (mascot_rows_gradient); with `accumulate` added
    to what `out` holds."""
    device = _device_of("grad", grad)
    g, i = _rows("grad", grad, device), _id_vector("ids", ids, device)
    if accumulate and out is None:
        _refuse("accumulate: needs an out")
    given, out = out, _result("out", out, (rows, g.width), out_dtype if out_dtype is not None or out is not None else grad.dtype, grad)
    keep, ws, size = _workspace(workspace, "mascot_rows_gradient_workspace", grad, device, i.count, rows, g.width)
    _call(device, "mascot_rows_gradient", g, i, scale, _rows("out", out, device), 1 if accumulate else 0, ws, size, _flag_word(flags, device))
    _changed(given, workspace, flags)
    return out


def pair_loss(P, Q, users, preferred, other, beta=1.0, smoothing=0.0, reference=None, weight=None, flags=None):
    """(loss, margin, coef) of the preference loss on pairs, fp32 vectors (mascot_pair_loss)."""
    device = _device_of("P", P)
    torch = _torch_ops().torch
    p, q = _rows("P", P, device), _rows("Q", Q, device)
    u, i, j = _id_vector("users", users, device), _id_vector("preferred", preferred, device), _id_vector("other", other, device)
    n = u.count
    ref, w = _plain("reference", reference, torch.float32, device, (n,)), _plain("weight", weight, torch.float32, device, (n,))
    loss, margin, coef = P.new_empty((3, n), dtype=torch.float32).unbind(0)
    _call(device, "mascot_pair_loss", p, q, u, i, j, beta, smoothing, ref, w, loss.data_ptr(), margin.data_ptr(), coef.data_ptr(),
          _flag_word(flags, device))
    _changed(flags)
    return loss, margin, coef


def pair_gradient(P, Q, users, preferred, other, coef, scale=1.0, dP=None, dQ=None, out_dtype=None, accumulate=False, workspace=None, flags=None):
    """(dP, dQ): gradients of the sum of scale * loss, from the coef of pair_loss (mascot_pair_gradient); with `accumulate`
    added to what dP and dQ hold."""
    device = _device_of("P", P)
    p, q = _rows("P", P, device), _rows("Q", Q, device)
    u, i, j = _id_vector("users", users, device), _id_vector("preferred", preferred, device), _id_vector("other", other, device)
    if accumulate and (dP is None or dQ is None):
        _refuse("accumulate: needs dP and dQ")
    given = dP, dQ
    dP = _result("dP", dP, P.shape, out_dtype if out_dtype is not None or dP is not None else P.dtype, P)
    dQ = _result("dQ", dQ, Q.shape, out_dtype if out_dtype is not None or dQ is not None else Q.dtype, Q)
    c = _plain("coef", coef, _torch_ops().torch.float32, device, (u.count,))
    keep, ws, size = _workspace(workspace, "mascot_pair_gradient_workspace", P, device, u.count, p.rows, q.rows, p.width)
    _call(device, "mascot_pair_gradient", p, q, u, i, j, c, scale, _rows("dP", dP, device), _rows("dQ", dQ, device), 1 if accumulate else 0, ws,
          size, _flag_word(flags, device))
    _changed(*given, workspace, flags)
    return dP, dQ


def rows_quantize(x, block_rows=1, q=None, scale=None):
    """(q, scale): x as float8_e4m3fn with a power-of-two scale for each block of `block_rows` (1 or 128) rows by 128 columns, scale
    [column blocks, row blocks] (mascot_rows_quantize).  A q of the call's own making has rows of a multiple of 128 bytes."""
    device = _device_of("x", x)
    torch = _torch_ops().torch
    r = _rows("x", x, device)
    given = q, scale
    if q is None:
        q = torch.empty((r.rows, -(-r.width // 128) * 128), dtype=torch.float8_e4m3fn, device=device)[:, :r.width]
    else:
        q = _result("q", q, (r.rows, r.width), torch.float8_e4m3fn, x)
    shape = (-(-r.width // 128), -(-r.rows // block_rows) if block_rows > 0 else 0)
    if scale is None:
        scale = torch.empty(shape, dtype=torch.float32, device=device)
    s = _plain("scale", scale, torch.float32, device, shape)
    _call(device, "mascot_rows_quantize", r, block_rows, _rows("q", q, device), s)
    _changed(*given)
    return q, scale


def rows_product(a, a_scale, b, b_scale, out=None, out_dtype=None, flags=None):
    """out[m][n] = the product of row m of a and row n of b, both float8_e4m3fn with their scales (mascot_rows_product): a with one
    for each row and 128 columns, b for each 1 or 128 rows; float32 unless out_dtype says otherwise."""
    device = _device_of("a", a)
    torch = _torch_ops().torch
    x, y = _rows("a", a, device), _rows("b", b, device)
    sa = _plain("a_scale", a_scale, torch.float32, device, (-(-x.width // 128), x.rows))
    each, sb = _scale_rows("b_scale", b_scale, y.rows, y.width, device)
    given, out = out, _result("out", out, (x.rows, y.rows), out_dtype if out_dtype is not None or out is not None else torch.float32, a)
    _call(device, "mascot_rows_product", x, sa, y, sb, each, _rows("out", out, device), _flag_word(flags, device))
    _changed(given, flags)
    return out
