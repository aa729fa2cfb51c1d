"""ctypes binding of libepsp.so (include/epsp.h) for the Python test and bench
harness.  Every call goes through the C ABI; torch tensors are only used as
device allocations (their data_ptr() is passed as a plain pointer).

The native library is mandatory: importing this module raises when
libepsp.so is missing or does not export the ABI.  There is no fallback.
"""
from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, c_char_p, c_double, c_float, c_int32, c_size_t, c_uint32, c_uint64, c_void_p

HERE = os.path.dirname(os.path.abspath(__file__))
# EPSP_LIB names another build of the same library (for example a tuning
# variant); by default the in-tree build next to this file is loaded.
LIB_PATH = os.environ.get("EPSP_LIB") or os.path.join(HERE, "libepsp.so")

OK, INVALID_ARGUMENT, PREFILL, UNSUPPORTED, OUT_OF_MEMORY, IO, INTERNAL, UNAVAILABLE = 0, 2, 6, 9, 10, 11, 12, 13
F32, F16, BF16 = 0, 1, 2
E4M3, I8 = 3, 4  # of an 8-bit cache

# Every symbol include/epsp.h declares.
EXPORTS = [
    "ep_sp_create", "ep_sp_reserve", "ep_sp_destroy", "ep_sp_set_qg_bound", "ep_sp_get_qg_bound",
    "ep_sp_set_ext", "ep_sp_set_k_matrix", "ep_sp_get_k_matrix_size", "ep_sp_set_prefill_mode",
    "ep_sp_get_prefill_mode", "ep_sp_set_ffn_skip", "ep_sp_get_ffn_skip", "ep_sp_reset",
    "ep_sp_query_blocks", "ep_sp_attend_layer", "ep_sp_prefill", "ep_sp_ffn_compact", "ep_sp_ffn_scatter",
    "ep_sp_sync_status", "ep_sp_last_error", "ep_sp_error_name", "ep_sp_chunk_plan", "ep_sp_ffn_auto_mask",
    "ep_sp_ffn_parse", "ep_sp_parse_config", "ep_sp_profile_enable", "ep_sp_profile_read", "ep_sp_layer_work",
    "ep_sp_select_pages_noalloc", "ep_sp_select_layer", "ep_sp_attend_rows", "ep_sp_xchg_alloc",
    "ep_sp_xchg_open", "ep_sp_xchg_attach", "ep_sp_xchg_slot", "ep_sp_attend_rows_xchg", "ep_sp_xchg_wait",
    "ep_sp_select_heads", "ep_sp_attend_ctas", "ep_sp_attend_ctas_xchg", "ep_sp_attention_grid", "ep_sp_balance_ctas",
    "ep_sp_cta_work", "ep_sp_set_attn_tiles", "ep_sp_get_attn_tiles", "ep_sp_append_kv",
    "ep_sp_set_f32_attention", "ep_sp_get_f32_attention", "ep_sp_get_pooled_pages", "ep_sp_set_head_routing",
    "ep_sp_get_head_routing", "ep_sp_set_paged_kv", "ep_sp_xchg_attach_buffers", "ep_sp_xchg_bytes",
    "ep_sp_decode_bytes", "ep_sp_decode_layer", "ep_sp_prompt_weights_bytes", "ep_sp_prompt_weights",
    "ep_sp_evict_bytes", "ep_sp_evict_layer", "ep_sp_profile_read_families",
    "ep_sp_pack_kv", "ep_sp_unpack_kv", "ep_sp_decode8_bytes", "ep_sp_decode8_layer", "ep_sp_count_refs",
    "ep_sp_fork_bytes", "ep_sp_fork_seqs", "ep_sp_resize_bytes", "ep_sp_resize_seqs", "ep_sp_compact_bytes",
    "ep_sp_compact_pool", "ep_sp_profile_read_family",
]
NUM_KERNELS = 6  # EP_SP_NUM_KERNELS
KERNEL_NAMES = ["k1_pool_pages", "k2_select_pages", "k3_sparse_attention", "k4_compact", "k4_scatter",
                "k5_exchange_wait"]
NUM_FAMILIES = 9  # EP_SP_NUM_FAMILIES
FAMILY_NAMES = KERNEL_NAMES + ["k6_decode", "k7_prompt_weights", "k8_evict"]
FAMILY_PACK, FAMILY_PAGES = 9, 10  # of profile_family alone
XCHG_HANDLE_BYTES = 64


class Config(ctypes.Structure):
    _fields_ = [
        ("n_layer", c_int32), ("n_head", c_int32), ("n_head_kv", c_int32), ("head_dim", c_int32),
        ("dtype", c_int32), ("out_dtype", c_int32), ("max_ctx", c_int32), ("page_size", c_int32),
        ("device", c_int32), ("kv_head_offset", c_int32), ("n_head_kv_total", c_int32), ("kq_scale", c_float),
    ]


class PrefillOptions(ctypes.Structure):
    _fields_ = [
        ("chunk_size", c_uint32), ("enable_chunking", c_int32), ("enable_qg_bound", c_int32),
        ("qg_sel_pages", c_uint32), ("qg_local_rows", c_uint32), ("qg_pool_pages", c_uint32),
    ]


class PrefillStats(ctypes.Structure):
    _fields_ = [
        ("chunks", c_uint32), ("query_gating", c_int32), ("attn_fallback", c_int32), ("qg_groups", c_uint32),
        ("chunk_attn_rows", c_uint32),
    ]


class KvBatchDesc(ctypes.Structure):
    """ep_sp_kv_batch."""

    _fields_ = [
        ("n_seq", c_int32), ("max_kv_len", c_int32), ("kv_lens", c_void_p), ("block_tables", c_void_p),
        ("table_stride", c_int32), ("block_rows", c_int32), ("pool_rows", c_int32), ("seq_rows", c_int32),
    ]


class Kv8Desc(ctypes.Structure):
    """ep_sp_kv8."""

    _fields_ = [("type", c_int32), ("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p)]


class PagesDesc(ctypes.Structure):
    """ep_sp_pages."""

    _fields_ = [
        ("n_seq", c_int32), ("table_stride", c_int32), ("block_rows", c_int32), ("pool_blocks", c_int32),
        ("kv_lens", c_void_p), ("block_tables", c_void_p), ("refs", c_void_p),
    ]


class PoolDesc(ctypes.Structure):
    """ep_sp_pool."""

    _fields_ = [("rows", c_void_p), ("block_bytes", c_size_t)]


def _load() -> ctypes.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"libepsp.so not built ({LIB_PATH}); run __graft_entry__.build()")
    lib = ctypes.CDLL(LIB_PATH)
    missing = [s for s in EXPORTS if not hasattr(lib, s)]
    if missing:
        raise ImportError(f"libepsp.so lacks {missing}")
    P = c_void_p
    sig = {
        "ep_sp_create": (c_int32, [POINTER(Config), POINTER(P)]),
        "ep_sp_reserve": (c_int32, [P]),
        "ep_sp_destroy": (None, [P]),
        "ep_sp_set_qg_bound": (c_int32, [P, c_int32, c_int32, c_int32, c_int32]),
        "ep_sp_get_qg_bound": (c_int32, [P]),
        "ep_sp_set_ext": (c_int32, [P, c_int32, c_int32, c_int32]),
        "ep_sp_set_k_matrix": (c_int32, [P, POINTER(c_int32), c_size_t]),
        "ep_sp_get_k_matrix_size": (c_int32, [P]),
        "ep_sp_set_prefill_mode": (None, [P, c_int32]),
        "ep_sp_get_prefill_mode": (c_int32, [P]),
        "ep_sp_set_ffn_skip": (None, [P, c_uint64]),
        "ep_sp_get_ffn_skip": (c_uint64, [P]),
        "ep_sp_reset": (c_int32, [P]),
        "ep_sp_query_blocks": (c_int32, [P, c_int32, POINTER(c_int32)]),
        "ep_sp_attend_layer": (c_int32, [P, c_int32, P, P, P, c_int32, c_int32, P, P, P, c_int32, P]),
        "ep_sp_prefill": (c_int32, [P, POINTER(PrefillOptions), c_int32, POINTER(P), POINTER(P), POINTER(P),
                                    POINTER(P), c_int32, c_int32, POINTER(PrefillStats), P]),
        "ep_sp_ffn_compact": (c_int32, [P, c_int32, P, P, c_int32, c_int32, P, P, P, P]),
        "ep_sp_ffn_scatter": (c_int32, [P, c_int32, P, P, P, P, c_int32, c_int32, P]),
        "ep_sp_sync_status": (c_int32, [P, P]),
        "ep_sp_last_error": (c_char_p, [P]),
        "ep_sp_error_name": (c_char_p, [c_int32]),
        "ep_sp_chunk_plan": (c_int32, [c_uint32, c_uint32, c_uint32, POINTER(c_uint32), c_int32, POINTER(c_int32)]),
        "ep_sp_ffn_auto_mask": (c_int32, [c_int32, c_double, POINTER(c_uint64)]),
        "ep_sp_ffn_parse": (c_int32, [c_char_p, c_int32, POINTER(c_uint64), ctypes.c_char_p, c_int32]),
        "ep_sp_parse_config": (c_int32, [c_char_p, POINTER(PrefillOptions)]),
        "ep_sp_profile_enable": (c_int32, [P, c_int32]),
        "ep_sp_profile_read": (c_int32, [P, POINTER(c_double), POINTER(ctypes.c_int64)]),
        "ep_sp_layer_work": (c_int32, [P, c_int32, c_int32, c_int32, POINTER(c_double)]),
        "ep_sp_select_pages_noalloc": (c_int32, [P, c_int32, P, P, c_int32, c_int32, P, P, c_int32, P]),
        "ep_sp_select_layer": (c_int32, [P, c_int32, P, P, P, c_int32, c_int32, P, P, c_int32, P]),
        "ep_sp_attend_rows": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, c_int32, P, P]),
        "ep_sp_xchg_alloc": (c_int32, [P, c_int32, c_int32, POINTER(P), P]),
        "ep_sp_xchg_open": (c_int32, [P, P, POINTER(P)]),
        "ep_sp_xchg_attach": (c_int32, [P, c_int32, c_int32, POINTER(P)]),
        "ep_sp_xchg_slot": (c_int32, [P, c_int32, POINTER(P)]),
        "ep_sp_attend_rows_xchg": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, P]),
        "ep_sp_xchg_wait": (c_int32, [P, c_int32, c_int32, P]),
        "ep_sp_select_heads": (c_int32, [P, c_int32, P, P, P, c_int32, c_int32, c_int32, c_int32, P]),
        "ep_sp_attend_ctas": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, c_int32, P, P]),
        "ep_sp_attend_ctas_xchg": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, P]),
        "ep_sp_attention_grid": (c_int32, [P, c_int32, POINTER(c_int32)]),
        "ep_sp_balance_ctas": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, POINTER(c_int32)]),
        "ep_sp_cta_work": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, c_int32, POINTER(c_double)]),
        "ep_sp_set_attn_tiles": (c_int32, [P, c_int32]),
        "ep_sp_get_attn_tiles": (c_int32, [P]),
        "ep_sp_append_kv": (c_int32, [P, c_int32, P, P, c_int32, P, P, c_int32, P]),
        "ep_sp_set_f32_attention": (c_int32, [P, c_int32]),
        "ep_sp_get_f32_attention": (c_int32, [P]),
        "ep_sp_get_pooled_pages": (c_int32, [P, P, P, c_int32, P]),
        "ep_sp_set_head_routing": (c_int32, [P, c_int32, c_double]),
        "ep_sp_get_head_routing": (c_int32, [P, POINTER(c_int32), POINTER(c_double)]),
        "ep_sp_set_paged_kv": (c_int32, [P, c_int32, P, c_int32, c_int32]),
        "ep_sp_xchg_attach_buffers": (c_int32, [P, c_int32, c_int32, c_int32, c_int32, POINTER(P), P]),
        "ep_sp_xchg_bytes": (c_int32, [P, c_int32, c_int32, POINTER(c_size_t)]),
        "ep_sp_decode_bytes": (c_int32, [P, c_int32, c_int32, c_int32, POINTER(c_size_t)]),
        "ep_sp_decode_layer": (c_int32, [P, c_int32, POINTER(KvBatchDesc), P, P, P, P, P, P, P, c_int32, P, c_size_t,
                                         P]),
        "ep_sp_prompt_weights_bytes": (c_int32, [P, c_int32, c_int32, c_int32, POINTER(c_size_t)]),
        "ep_sp_prompt_weights": (c_int32, [P, c_int32, P, P, c_int32, c_int32, c_int32, c_int32, P, c_int32, P,
                                           c_size_t, P]),
        "ep_sp_evict_bytes": (c_int32, [P, c_int32, c_int32, c_int32, POINTER(c_size_t)]),
        "ep_sp_evict_layer": (c_int32, [P, c_int32, POINTER(KvBatchDesc), P, P, P, c_int32, c_int32, c_int32, c_int32,
                                        POINTER(KvBatchDesc), P, P, P, c_int32, P, P, P, c_size_t, P]),
        "ep_sp_profile_read_families": (c_int32, [P, c_int32, POINTER(c_double), POINTER(ctypes.c_int64)]),
        "ep_sp_profile_read_family": (c_int32, [P, c_int32, POINTER(c_double), POINTER(ctypes.c_int64)]),
        "ep_sp_pack_kv": (c_int32, [P, c_int32, POINTER(KvBatchDesc), P, P, P, POINTER(KvBatchDesc), POINTER(Kv8Desc),
                                    P]),
        "ep_sp_unpack_kv": (c_int32, [P, c_int32, POINTER(KvBatchDesc), POINTER(Kv8Desc), P, POINTER(KvBatchDesc), P, P,
                                      P]),
        "ep_sp_decode8_bytes": (c_int32, [P, c_int32, c_int32, POINTER(c_size_t)]),
        "ep_sp_decode8_layer": (c_int32, [P, c_int32, POINTER(KvBatchDesc), P, P, P, POINTER(Kv8Desc), P, P, c_size_t,
                                          P]),
        "ep_sp_count_refs": (c_int32, [P, POINTER(PagesDesc), P]),
        "ep_sp_fork_bytes": (c_int32, [P, POINTER(PagesDesc), POINTER(c_size_t)]),
        "ep_sp_fork_seqs": (c_int32, [P, POINTER(PagesDesc), P, P, P, c_size_t, P]),
        "ep_sp_resize_bytes": (c_int32, [P, POINTER(PagesDesc), POINTER(c_size_t)]),
        "ep_sp_resize_seqs": (c_int32, [P, POINTER(PagesDesc), P, POINTER(PoolDesc), c_int32, P, c_size_t, P]),
        "ep_sp_compact_bytes": (c_int32, [P, POINTER(PagesDesc), POINTER(c_size_t)]),
        "ep_sp_compact_pool": (c_int32, [P, POINTER(PagesDesc), POINTER(PoolDesc), c_int32, P, P, c_size_t, P]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


lib = _load()


class EpspError(RuntimeError):
    def __init__(self, rc: int, msg: str):
        super().__init__(f"{error_name(rc)} ({rc}): {msg}")
        self.rc = rc


def error_name(rc: int) -> str:
    return lib.ep_sp_error_name(rc).decode()


def _ptr(t) -> int | None:
    if t is None:
        return None
    return t.data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        import torch

        return torch.cuda.current_stream().cuda_stream
    return stream if isinstance(stream, int) else stream.cuda_stream


class _CudaArray:
    def __init__(self, ptr, shape, typestr):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3, "strides": None}


def device_view(ptr: int, shape, dtype: int):
    """torch tensor aliasing `shape` elements of device memory at ptr (no copy),
    e.g. an exchange slot: device_view(ctx.xchg_slot(s), (n_tok, heads, d), BF16)."""
    import torch

    typestr = {F32: "<f4", F16: "<f2", BF16: "<i2"}[dtype]
    t = torch.as_tensor(_CudaArray(ptr, shape, typestr), device="cuda")
    return t.view(torch.bfloat16) if dtype == BF16 else t


def _torch_dtypes():
    import torch

    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16, "i32": torch.int32}


_DTYPES: dict = {}  # the torch types of F32, F16, BF16 and "i32", filled by the first batch or context call


_RAW_STREAM = []  # torch's direct query of a device's current stream, where it has one


def _current_stream(device):
    """The raw current stream of a device (the direct query takes a tenth of the time)."""
    if not _RAW_STREAM:
        import torch

        _RAW_STREAM.append(getattr(torch._C, "_cuda_getCurrentRawStream", None)
                           or (lambda d: torch.cuda.current_stream(d).cuda_stream))
    return _RAW_STREAM[0](device)


def _dtype(code):
    if not _DTYPES:
        _DTYPES.update(_torch_dtypes())
    return _DTYPES[code]


def _check(name, t, dtype, shape, device):
    """The library sees plain pointers: what a tensor is must be checked here."""
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return
    if t.dtype is not dtype:
        raise ValueError(f"{name} is {t.dtype}, not {dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous (strides {tuple(t.stride())})")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not cuda:{device}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")


class KvBatch:
    """A batch of sequences in one layer's cache (ep_sp_kv_batch).  kv_lens: int32 [n_seq] on the device (None for an
    eviction's destination, with n_seq given).  Paged: block_tables int32 [n_seq][entries] on the device, block_rows
    and pool_rows; contiguous: block_rows 0 and seq_rows rows from one sequence to the next.  Keeps its tensors
    alive; kv_lens and the tables may be rewritten in place between calls."""

    def __init__(self, kv_lens, max_kv_len, block_tables=None, block_rows=0, pool_rows=0, seq_rows=0, n_seq=None):
        ref = kv_lens if kv_lens is not None else block_tables
        if kv_lens is None and n_seq is None:
            raise ValueError("a batch without kv_lens needs n_seq")
        self.n_seq = int(n_seq) if n_seq is not None else kv_lens.shape[0]
        self.kv_lens, self.block_tables = kv_lens, block_tables
        self.device = None if ref is None else ref.get_device()
        if kv_lens is not None:
            _check("kv_lens", kv_lens, _dtype("i32"), (self.n_seq,), self.device)
        entries = 0
        if block_rows:
            if block_tables is None:
                raise ValueError("block_rows without block_tables")
            _check("block_tables", block_tables, _dtype("i32"), (self.n_seq, block_tables.shape[-1]), self.device)
            entries = block_tables.shape[1]
        self.rows = pool_rows if block_rows else self.n_seq * seq_rows
        self.desc = KvBatchDesc(self.n_seq, max_kv_len, _ptr(kv_lens), _ptr(block_tables) if block_rows else None,
                                entries, block_rows, pool_rows, seq_rows)
        self.ref = ctypes.byref(self.desc)


def _code8(dtype):
    import torch

    code = {torch.float8_e4m3fn: E4M3, torch.int8: I8}.get(dtype)
    if code is None:
        raise ValueError(f"an 8-bit cache is torch.float8_e4m3fn or torch.int8, not {dtype}")
    return code


class Kv8:
    """One layer's cache in 8 bits (ep_sp_kv8): k, v [rows][n_head_kv][head_dim] of torch.float8_e4m3fn or torch.int8,
    k_scale, v_scale f32 [rows / page_size][n_head_kv].  Keeps its tensors alive."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.type, self.device = _code8(k.dtype), k.get_device()
        if k.dim() != 3 or k_scale.dim() != 2 or k.shape[0] % max(1, k_scale.shape[0]):
            raise ValueError("k is [rows][n_head_kv][head_dim], k_scale [rows / page_size][n_head_kv]")
        _check("v", v, k.dtype, k.shape, self.device)
        _check("k", k, k.dtype, k.shape, self.device)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _check(name, t, _dtype(F32), (k_scale.shape[0], k.shape[1]), self.device)
        self.rows = k.shape[0]
        self.page = self.rows // k_scale.shape[0] if k_scale.shape[0] else 0
        self.desc = Kv8Desc(self.type, k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self.ref = ctypes.byref(self.desc)


class Pages:
    """Sequences and the blocks they hold (ep_sp_pages): kv_lens int32 [n_seq], block_tables int32 [n_seq][entries],
    refs int32 [pool_blocks], all on the device and rewritten by the calls.  Keeps its tensors alive."""

    def __init__(self, kv_lens, block_tables, refs, block_rows):
        i32, self.device = _dtype("i32"), kv_lens.get_device()
        self.kv_lens, self.block_tables, self.refs, self.n_seq = kv_lens, block_tables, refs, kv_lens.shape[0]
        _check("kv_lens", kv_lens, i32, (self.n_seq,), self.device)
        _check("block_tables", block_tables, i32, (self.n_seq, block_tables.shape[-1]), self.device)
        _check("refs", refs, i32, (refs.shape[0],), self.device)
        self.blocks, self.block_rows = refs.shape[0], block_rows
        self.desc = PagesDesc(self.n_seq, block_tables.shape[1], block_rows, self.blocks, kv_lens.data_ptr(),
                              block_tables.data_ptr(), refs.data_ptr())
        self.ref = ctypes.byref(self.desc)


class Pools:
    """The pools that follow a set of block tables: tensors (K, V, scales, of any layers and types) whose storage is
    [blocks][bytes of a block].  Keeps its tensors alive."""

    def __init__(self, tensors, blocks):
        self.tensors, self.blocks, self.fits, self.shapes = list(tensors), blocks, None, {}
        if not self.tensors:
            raise ValueError("no pools")
        self.device = self.tensors[0].get_device()
        self.desc = (PoolDesc * len(self.tensors))()
        for i, t in enumerate(self.tensors):
            if not t.is_contiguous() or t.get_device() != self.device:
                raise ValueError(f"pool {i} must be contiguous and on the device of the others")
            if t.nbytes == 0 or t.nbytes % (4 * blocks):
                raise ValueError(f"pool {i} is not {blocks} blocks of whole 4-byte words")
            self.desc[i] = PoolDesc(t.data_ptr(), t.nbytes // blocks)
            self.shapes.setdefault((t.shape, t.dtype), i)


class Context:
    """One ep_sp_ctx.  Methods return the C status code; `check()` raises."""

    def __init__(self, *, n_layer, n_head, n_head_kv, head_dim, dtype=BF16, out_dtype=None, max_ctx,
                 page_size=32, device=0, kv_head_offset=0, n_head_kv_total=0, kq_scale=0.0):
        self.cfg = Config(n_layer, n_head, n_head_kv, head_dim, dtype, dtype if out_dtype is None else out_dtype,
                          max_ctx, page_size, device, kv_head_offset, n_head_kv_total, kq_scale)
        self._pool_rows = 0  # rows of the pools of set_paged_kv
        self._facts = None   # see _fast
        self.h = c_void_p()
        rc = lib.ep_sp_create(ctypes.byref(self.cfg), ctypes.byref(self.h))
        if rc != OK:
            raise EpspError(rc, "ep_sp_create")

    def close(self):
        if self.h:
            lib.ep_sp_destroy(self.h)
            self.h = c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self, rc: int) -> int:
        if rc != OK:
            raise EpspError(rc, self.last_error())
        return rc

    def last_error(self) -> str:
        return lib.ep_sp_last_error(self.h).decode()

    # controls -----------------------------------------------------------
    def reserve(self):
        return lib.ep_sp_reserve(self.h)

    def set_qg_bound(self, enabled, sel_pages, local_pages, pool_pages=0):
        return lib.ep_sp_set_qg_bound(self.h, enabled, sel_pages, local_pages, pool_pages)

    def qg_bound(self):
        return lib.ep_sp_get_qg_bound(self.h)

    def set_ext(self, per_kv_head, q_subblock, max_gather_rows):
        return lib.ep_sp_set_ext(self.h, per_kv_head, q_subblock, max_gather_rows)

    def set_k_matrix(self, values):
        vals = [int(x) for x in values]
        arr = (c_int32 * max(1, len(vals)))(*vals) if vals else None
        return lib.ep_sp_set_k_matrix(self.h, arr, len(vals))

    def k_matrix_size(self):
        return lib.ep_sp_get_k_matrix_size(self.h)

    def set_prefill_mode(self, on):
        lib.ep_sp_set_prefill_mode(self.h, 1 if on else 0)

    def prefill_mode(self):
        return lib.ep_sp_get_prefill_mode(self.h)

    def set_ffn_skip(self, mask):
        lib.ep_sp_set_ffn_skip(self.h, mask)

    def ffn_skip(self):
        return lib.ep_sp_get_ffn_skip(self.h)

    def reset(self):
        return lib.ep_sp_reset(self.h)

    def query_blocks(self, n_tok):
        n = c_int32()
        rc = lib.ep_sp_query_blocks(self.h, n_tok, ctypes.byref(n))
        return rc, n.value

    def sync_status(self, stream=None):
        return lib.ep_sp_sync_status(self.h, _stream(stream))

    # compute ------------------------------------------------------------
    def attend_layer(self, layer, q, k, v, kv_len, n_tok, out, sel=None, cnt=None, sel_cap=0, stream=None):
        return lib.ep_sp_attend_layer(self.h, layer, _ptr(q), _ptr(k), _ptr(v), kv_len, n_tok, _ptr(out),
                                      _ptr(sel), _ptr(cnt), sel_cap, _stream(stream))

    def select_layer(self, layer, q, k, v, kv_len, n_tok, sel=None, cnt=None, sel_cap=0, stream=None):
        return lib.ep_sp_select_layer(self.h, layer, _ptr(q), _ptr(k), _ptr(v), kv_len, n_tok, _ptr(sel), _ptr(cnt),
                                      sel_cap, _stream(stream))

    def attend_rows(self, layer, kv_len, n_tok, row_begin, row_end, out, stream=None):
        return lib.ep_sp_attend_rows(self.h, layer, kv_len, n_tok, row_begin, row_end, _ptr(out), _stream(stream))

    # ---------------------------------------------- head-parallel exchange
    def xchg_alloc(self, rows, n_slots, ipc=True):
        """Allocates this rank's exchange buffer; returns (base, handle bytes or None)."""
        base = c_void_p()
        h = ctypes.create_string_buffer(XCHG_HANDLE_BYTES) if ipc else None
        self.check(lib.ep_sp_xchg_alloc(self.h, rows, n_slots, ctypes.byref(base), h))
        return base.value, (h.raw if ipc else None)

    def xchg_open(self, handle: bytes):
        base = c_void_p()
        buf = ctypes.create_string_buffer(handle, XCHG_HANDLE_BYTES)
        self.check(lib.ep_sp_xchg_open(self.h, buf, ctypes.byref(base)))
        return base.value

    def xchg_attach(self, rank, bases):
        arr = (c_void_p * len(bases))(*bases)
        return lib.ep_sp_xchg_attach(self.h, len(bases), rank, arr)

    def xchg_attach_buffers(self, rows, n_slots, rank, bases, mc_base=None):
        arr = (c_void_p * len(bases))(*bases)
        return lib.ep_sp_xchg_attach_buffers(self.h, rows, n_slots, len(bases), rank, arr, mc_base)

    def xchg_bytes(self, rows, n_slots):
        n = c_size_t()
        self.check(lib.ep_sp_xchg_bytes(self.h, rows, n_slots, ctypes.byref(n)))
        return n.value

    def xchg_slot(self, slot):
        p = c_void_p()
        self.check(lib.ep_sp_xchg_slot(self.h, slot, ctypes.byref(p)))
        return p.value

    def attend_rows_xchg(self, layer, kv_len, n_tok, row_begin, row_end, slot, stream=None):
        return lib.ep_sp_attend_rows_xchg(self.h, layer, kv_len, n_tok, row_begin, row_end, slot, _stream(stream))

    def xchg_wait(self, slot, rows, stream=None):
        return lib.ep_sp_xchg_wait(self.h, slot, rows, _stream(stream))

    def attend_ctas_xchg(self, layer, kv_len, n_tok, cta_begin, cta_end, slot, stream=None):
        return lib.ep_sp_attend_ctas_xchg(self.h, layer, kv_len, n_tok, cta_begin, cta_end, slot, _stream(stream))

    # ------------------------------------------------- splitting a layer
    def select_heads(self, layer, q, k, v, kv_len, n_tok, head_begin, head_end, stream=None):
        return lib.ep_sp_select_heads(self.h, layer, _ptr(q), _ptr(k), _ptr(v), kv_len, n_tok, head_begin, head_end,
                                      _stream(stream))

    def attend_ctas(self, layer, kv_len, n_tok, cta_begin, cta_end, out, stream=None):
        return lib.ep_sp_attend_ctas(self.h, layer, kv_len, n_tok, cta_begin, cta_end, _ptr(out), _stream(stream))

    def attention_grid(self, n_tok):
        n = c_int32()
        self.check(lib.ep_sp_attention_grid(self.h, n_tok, ctypes.byref(n)))
        return n.value

    def append_kv(self, layer, k_new, v_new, n_new, k_cache, v_cache, kv_pos, stream=None):
        return lib.ep_sp_append_kv(self.h, layer, _ptr(k_new), _ptr(v_new), n_new, _ptr(k_cache), _ptr(v_cache),
                                   kv_pos, _stream(stream))

    def set_attn_tiles(self, tiles_per_cta):
        return lib.ep_sp_set_attn_tiles(self.h, tiles_per_cta)

    def attn_tiles(self):
        return lib.ep_sp_get_attn_tiles(self.h)

    def set_paged_kv(self, block_rows, block_table=None, n_entries=0, pool_rows=0):
        rc = lib.ep_sp_set_paged_kv(self.h, block_rows, _ptr(block_table), n_entries, pool_rows)
        if rc == OK:
            self._pool_rows = pool_rows if block_rows else 0
        return rc

    # ------------------------------- answering from and shrinking the cache
    def _fast(self):
        """(torch type, output type, f32, int32, device, n_head, n_head_kv, head_dim), read once: a ctypes field costs
        as much as a check."""
        f = self._facts
        if f is None:
            c = self.cfg
            f = self._facts = (_dtype(c.dtype), _dtype(c.out_dtype), _dtype(F32), _dtype("i32"), c.device, c.n_head,
                               c.n_head_kv, c.head_dim)
        return f

    def _cache_tensors(self, kv, k, v, what=("k", "v")):
        dt, _, _, _, dev, _, heads, d = self._facts or self._fast()
        if kv.device is not None and kv.device != dev:
            raise ValueError(f"the batch is on cuda:{kv.device}, not cuda:{dev}")
        need = kv.rows * heads * d
        tail = (heads, d)
        # rows in any number of leading dimensions; both at once when all is well (an attribute of a tensor takes
        # 50 to 150 ns)
        shape = k.shape
        if (k.dtype is dt and v.dtype is dt and k.get_device() == dev and v.get_device() == dev and k.is_contiguous()
                and v.is_contiguous() and shape[-2:] == tail and v.shape == shape and k.numel() >= need):
            return
        for name, t in zip(what, (k, v)):
            _check(name, t, dt, t.shape[:-2] + tail, dev)
            if t.numel() < need:
                raise ValueError(f"{name} holds fewer than the batch's {kv.rows} rows")

    def _workspace(self, t):
        if t is None:
            return None, 0
        if not t.is_contiguous() or t.get_device() != self._fast()[4]:
            raise ValueError(f"the workspace must be a contiguous tensor on cuda:{self.cfg.device}")
        return t.data_ptr(), t.nbytes

    def decode_bytes(self, n_seq, max_kv_len, with_acc=False):
        n = c_size_t()
        self.check(lib.ep_sp_decode_bytes(self.h, n_seq, max_kv_len, 1 if with_acc else 0, ctypes.byref(n)))
        return n.value

    def decode_layer(self, layer, kv, q, k, v, out, workspace, k_new=None, v_new=None, acc=None, stream=None):
        """kv: KvBatch; q, out [n_seq][n_head][head_dim]; k, v the cache's rows; k_new, v_new [n_seq][n_head_kv]
        [head_dim]; acc f32 [n_seq][n_head_kv][stride].  Raises ValueError for a tensor of another type, shape,
        layout or device; returns the status code."""
        dt, odt, f32, _, dev, heads, kvh, d = self._facts or self._fast()
        self._cache_tensors(kv, k, v)
        n_seq = kv.n_seq
        _check("q", q, dt, (n_seq, heads, d), dev)
        _check("out", out, odt, (n_seq, heads, d), dev)
        p_k, p_v, p_acc, wide = None, None, None, 0
        if k_new is not None:
            _check("k_new", k_new, dt, (n_seq, kvh, d), dev)
            p_k = k_new.data_ptr()
        if v_new is not None:
            _check("v_new", v_new, dt, (n_seq, kvh, d), dev)
            p_v = v_new.data_ptr()
        if acc is not None:
            wide = acc.shape[-1]
            _check("acc", acc, f32, (n_seq, kvh, wide), dev)
            p_acc = acc.data_ptr()
        ws, n = self._workspace(workspace)
        return lib.ep_sp_decode_layer(self.h, layer, kv.ref, q.data_ptr(), p_k, p_v, k.data_ptr(), v.data_ptr(),
                                      out.data_ptr(), p_acc, wide, ws, n,
                                      _current_stream(dev) if stream is None else self._stream(stream))

    def prompt_weights_bytes(self, kv_len, n_tok, row_begin):
        n = c_size_t()
        self.check(lib.ep_sp_prompt_weights_bytes(self.h, kv_len, n_tok, row_begin, ctypes.byref(n)))
        return n.value

    def prompt_weights(self, layer, q, k, kv_len, n_tok, row_begin, acc, workspace, accumulate=False, stream=None):
        """q [n_tok][n_head][head_dim]; k the cache (paged under set_paged_kv); acc f32 [n_head_kv][stride]."""
        dt, _, f32, _, dev, heads, kvh, d = self._fast()
        _check("q", q, dt, (n_tok, heads, d), dev)
        rows, wide = k.shape[0], acc.shape[-1]
        _check("k", k, dt, (rows, kvh, d), dev)
        if rows < (self._pool_rows or kv_len):
            raise ValueError(f"k holds {rows} rows, the call reads {self._pool_rows or kv_len}")
        _check("acc", acc, f32, (kvh, wide), dev)
        ws, n = self._workspace(workspace)
        return lib.ep_sp_prompt_weights(self.h, layer, q.data_ptr(), k.data_ptr(), kv_len, n_tok, row_begin,
                                        1 if accumulate else 0, acc.data_ptr(), wide, ws, n,
                                        self._stream(stream))

    def evict_bytes(self, n_seq, max_kv_len, n_keep):
        n = c_size_t()
        self.check(lib.ep_sp_evict_bytes(self.h, n_seq, max_kv_len, n_keep, ctypes.byref(n)))
        return n.value

    def evict_layer(self, layer, src, k, v, acc, n_keep, sink_rows, recent_rows, dst, k_dst, v_dst, workspace,
                    acc_dst=None, new_lens=None, kept_rows=None, stream=None):
        """src, dst: KvBatch (the same object and tensors compact in place); acc f32 [n_seq][n_head_kv][stride];
        acc_dst likewise; new_lens int32 [n_seq]; kept_rows int32 [n_seq][n_head_kv][n_keep]."""
        _, _, f32, i32, dev, _, kvh, _ = self._facts or self._fast()
        self._cache_tensors(src, k, v)
        self._cache_tensors(dst, k_dst, v_dst, ("k_dst", "v_dst"))
        n_seq = src.n_seq
        wide = acc.shape[-1]
        _check("acc", acc, f32, (n_seq, kvh, wide), dev)
        p_acc, wide_dst, p_lens, p_kept = None, 0, None, None
        if acc_dst is not None:
            wide_dst = acc_dst.shape[-1]
            _check("acc_dst", acc_dst, f32, (n_seq, kvh, wide_dst), dev)
            p_acc = acc_dst.data_ptr()
        if new_lens is not None:
            _check("new_lens", new_lens, i32, (n_seq,), dev)
            p_lens = new_lens.data_ptr()
        if kept_rows is not None:
            _check("kept_rows", kept_rows, i32, (n_seq, kvh, n_keep), dev)
            p_kept = kept_rows.data_ptr()
        ws, n = self._workspace(workspace)
        return lib.ep_sp_evict_layer(self.h, layer, src.ref, k.data_ptr(), v.data_ptr(), acc.data_ptr(), wide,
                                     n_keep, sink_rows, recent_rows, dst.ref, k_dst.data_ptr(), v_dst.data_ptr(),
                                     p_acc, wide_dst, p_lens, p_kept, ws, n,
                                     _current_stream(dev) if stream is None else self._stream(stream))

    # ------------------------------------------------- the cache in 8 bits
    def _cache8_tensors(self, kv, c8, what="the 8-bit cache"):
        _, _, _, _, dev, _, heads, d = self._facts or self._fast()
        if c8.device != dev or (kv.device is not None and kv.device != dev):
            raise ValueError(f"{what} or its batch is not on cuda:{dev}")
        if c8.k.shape[1:] != (heads, d):
            raise ValueError(f"{what} has rows of shape {tuple(c8.k.shape[1:])}, not {(heads, d)}")
        if c8.rows != c8.page * c8.k_scale.shape[0] or c8.page != self.cfg.page_size:
            raise ValueError(f"{what} has {c8.k_scale.shape[0]} scales for {c8.rows} rows in pages of {self.cfg.page_size}")
        if c8.rows < kv.rows:
            raise ValueError(f"{what} holds fewer than the batch's {kv.rows} rows")

    def _first(self, first, n_seq):
        if first is None:
            return None
        _check("first", first, self._fast()[3], (n_seq,), self._fast()[4])
        return first.data_ptr()

    def pack_kv(self, layer, src, k, v, dst, cache, first=None, stream=None):
        """Rows [first, src.kv_lens) of k, v (src: KvBatch) into cache (Kv8, laid out by dst: KvBatch)."""
        self._cache_tensors(src, k, v)
        self._cache8_tensors(dst, cache)
        return lib.ep_sp_pack_kv(self.h, layer, src.ref, k.data_ptr(), v.data_ptr(), self._first(first, src.n_seq),
                                 dst.ref, cache.ref, self._stream(stream))

    def unpack_kv(self, layer, src, cache, dst, k, v, first=None, stream=None):
        """Rows [first, src.kv_lens) of cache (Kv8, src: KvBatch) into k, v (dst: KvBatch)."""
        self._cache8_tensors(src, cache)
        self._cache_tensors(dst, k, v)
        return lib.ep_sp_unpack_kv(self.h, layer, src.ref, cache.ref, self._first(first, src.n_seq), dst.ref,
                                   k.data_ptr(), v.data_ptr(), self._stream(stream))

    def decode8_bytes(self, n_seq, max_kv_len):
        n = c_size_t()
        self.check(lib.ep_sp_decode8_bytes(self.h, n_seq, max_kv_len, ctypes.byref(n)))
        return n.value

    def decode8_layer(self, layer, kv, q, cache, out, workspace, k_new=None, v_new=None, stream=None):
        """decode_layer over a Kv8; k_new, v_new go into it first."""
        dt, odt, _, _, dev, heads, kvh, d = self._facts or self._fast()
        self._cache8_tensors(kv, cache)
        n_seq = kv.n_seq
        _check("q", q, dt, (n_seq, heads, d), dev)
        _check("out", out, odt, (n_seq, heads, d), dev)
        p_k, p_v = None, None
        if k_new is not None:
            _check("k_new", k_new, dt, (n_seq, kvh, d), dev)
            p_k = k_new.data_ptr()
        if v_new is not None:
            _check("v_new", v_new, dt, (n_seq, kvh, d), dev)
            p_v = v_new.data_ptr()
        ws, n = self._workspace(workspace)
        return lib.ep_sp_decode8_layer(self.h, layer, kv.ref, q.data_ptr(), p_k, p_v, cache.ref, out.data_ptr(), ws, n,
                                       _current_stream(dev) if stream is None else self._stream(stream))

    # --------------------------------------------- blocks of paged caches
    def _pages(self, pages, pools=None):
        dev = self._fast()[4]
        if pools is not None and pools.fits != (self._facts, pages.blocks, pages.block_rows):
            self._pool_rows_fit(pages, pools)
        if pages.device != dev or (pools is not None and pools.device != dev):
            raise ValueError(f"the pages or pools are not on cuda:{dev}")
        if pools is not None and pools.blocks != pages.blocks:
            raise ValueError(f"the pools have {pools.blocks} blocks, the counts {pages.blocks}")

    def _pool_rows_fit(self, pages, pools):
        """A tensor that is seen to hold cache rows or pages' scales has as many as the blocks (or one a block); looked
        at once, the shapes stay."""
        _, _, f32, _, _, _, heads, d = self._fast()
        rows = pages.blocks * pages.block_rows
        for (shape, dtype), i in pools.shapes.items():
            n = shape.numel() // (heads * d) if len(shape) > 2 and shape[-2:] == (heads, d) else None
            if len(shape) == 2 and dtype == f32 and shape[1] == heads:
                n = shape[0]
            if n is not None and n not in (rows, rows // self.cfg.page_size, pages.blocks):
                raise ValueError(f"pool {i} of shape {tuple(shape)} is not {pages.blocks} blocks of "
                                 f"{pages.block_rows} rows")
        pools.fits = (self._facts, pages.blocks, pages.block_rows)

    def _seq_ints(self, name, t, n_seq):
        _check(name, t, self._fast()[3], (n_seq,), self._fast()[4])
        return t.data_ptr()

    def _bytes(self, fn, pages):
        n = c_size_t()
        rc = fn(self.h, pages.ref, ctypes.byref(n))
        if rc != OK:
            raise EpspError(rc, "pages")
        return n.value

    def count_refs(self, pages, stream=None):
        self._pages(pages)
        return lib.ep_sp_count_refs(self.h, pages.ref, self._stream(stream))

    def fork_bytes(self, pages):
        return self._bytes(lib.ep_sp_fork_bytes, pages)

    def fork_seqs(self, pages, parents, workspace, lens=None, stream=None):
        """parents int32 [n_seq] (-1: empty the sequence); lens int32 [n_seq] or None: all of the parent's rows."""
        self._pages(pages)
        ws, n = self._workspace(workspace)
        return lib.ep_sp_fork_seqs(self.h, pages.ref, self._seq_ints("parents", parents, pages.n_seq),
                                   None if lens is None else self._seq_ints("lens", lens, pages.n_seq), ws, n,
                                   self._stream(stream))

    def resize_bytes(self, pages):
        return self._bytes(lib.ep_sp_resize_bytes, pages)

    def resize_seqs(self, pages, new_lens, pools, workspace, stream=None):
        """new_lens int32 [n_seq]; pools: Pools."""
        self._pages(pages, pools)
        ws, n = self._workspace(workspace)
        return lib.ep_sp_resize_seqs(self.h, pages.ref, self._seq_ints("new_lens", new_lens, pages.n_seq), pools.desc,
                                     len(pools.tensors), ws, n, self._stream(stream))

    def compact_bytes(self, pages):
        return self._bytes(lib.ep_sp_compact_bytes, pages)

    def compact_pool(self, pages, pools, workspace, n_used=None, stream=None):
        """n_used int32 [1] or None: receives the number of blocks in use."""
        self._pages(pages, pools)
        p_used = None if n_used is None else self._seq_ints("n_used", n_used, 1)
        ws, n = self._workspace(workspace)
        return lib.ep_sp_compact_pool(self.h, pages.ref, pools.desc, len(pools.tensors), p_used, ws, n,
                                      self._stream(stream))

    def profile_family(self, family):
        """(milliseconds, launches) of one family since the last ep_sp_profile_enable."""
        ms, n = c_double(), ctypes.c_int64()
        self.check(lib.ep_sp_profile_read_family(self.h, family, ctypes.byref(ms), ctypes.byref(n)))
        return ms.value, n.value

    def profile_families(self):
        """{family name: (milliseconds, launches)} since the last ep_sp_profile_enable."""
        ms, n = (c_double * NUM_FAMILIES)(), (ctypes.c_int64 * NUM_FAMILIES)()
        self.check(lib.ep_sp_profile_read_families(self.h, NUM_FAMILIES, ms, n))
        return {name: (ms[i], n[i]) for i, name in enumerate(FAMILY_NAMES)}

    def _stream(self, stream):
        """The given stream, or the current one of the context's device."""
        if stream is None:
            return _current_stream(self._fast()[4])
        return stream if isinstance(stream, int) else stream.cuda_stream

    def set_head_routing(self, mode, threshold):
        return lib.ep_sp_set_head_routing(self.h, mode, threshold)

    def head_routing(self):
        m, t = c_int32(), c_double()
        self.check(lib.ep_sp_get_head_routing(self.h, ctypes.byref(m), ctypes.byref(t)))
        return m.value, t.value

    def pooled_pages(self, pages, counts, cap, stream=None):
        return lib.ep_sp_get_pooled_pages(self.h, _ptr(pages), _ptr(counts), cap, _stream(stream))

    def set_f32_attention(self, mode):
        return lib.ep_sp_set_f32_attention(self.h, mode)

    def f32_attention(self):
        return lib.ep_sp_get_f32_attention(self.h)

    def cta_work(self, layer, kv_len, n_tok, cta_begin, cta_end):
        out = (c_double * 3)()
        self.check(lib.ep_sp_cta_work(self.h, layer, kv_len, n_tok, cta_begin, cta_end, out))
        return list(out)

    def balance_ctas(self, layer, kv_len, n_tok, n_parts):
        cuts = (c_int32 * (n_parts + 1))()
        self.check(lib.ep_sp_balance_ctas(self.h, layer, kv_len, n_tok, n_parts, cuts))
        return list(cuts)

    def prefill(self, opts: PrefillOptions, qs, ks, vs, outs, n_tokens, n_ubatch, stream=None):
        n = len(qs)
        arr = lambda ts: (c_void_p * n)(*[t.data_ptr() for t in ts])  # noqa: E731
        stats = PrefillStats()
        rc = lib.ep_sp_prefill(self.h, ctypes.byref(opts), n, arr(qs), arr(ks), arr(vs), arr(outs), n_tokens,
                               n_ubatch, ctypes.byref(stats), _stream(stream))
        return rc, stats

    def select_pages_noalloc(self, layer, q, k, kv_len, n_tok, sel, cnt, sel_cap, stream=None):
        return lib.ep_sp_select_pages_noalloc(self.h, layer, _ptr(q), _ptr(k), kv_len, n_tok, _ptr(sel), _ptr(cnt),
                                              sel_cap, _stream(stream))

    def ffn_compact(self, layer, x, keep, n_rows, hidden, x_kept, row_ids, n_keep, stream=None):
        return lib.ep_sp_ffn_compact(self.h, layer, _ptr(x), _ptr(keep), n_rows, hidden, _ptr(x_kept),
                                     _ptr(row_ids), _ptr(n_keep), _stream(stream))

    def ffn_scatter(self, layer, ffn_out, residual, row_ids, n_keep, n_rows, hidden, stream=None):
        return lib.ep_sp_ffn_scatter(self.h, layer, _ptr(ffn_out), _ptr(residual), _ptr(row_ids), _ptr(n_keep),
                                     n_rows, hidden, _stream(stream))


# host-side planning (no device) -----------------------------------------
def chunk_plan(n_tokens, chunk_size, n_ubatch, cap=1 << 16):
    buf = (c_uint32 * (2 * cap))()
    n = c_int32()
    rc = lib.ep_sp_chunk_plan(n_tokens, chunk_size, n_ubatch, buf, cap, ctypes.byref(n))
    if rc != OK:
        return rc, []
    return rc, [(buf[2 * i], buf[2 * i + 1]) for i in range(n.value)]


def ffn_auto_mask(n_layer, ratio):
    out = c_uint64()
    rc = lib.ep_sp_ffn_auto_mask(n_layer, ratio, ctypes.byref(out))
    return rc, out.value


def ffn_parse(spec, n_layer):
    out = c_uint64()
    warn = ctypes.create_string_buffer(64)
    rc = lib.ep_sp_ffn_parse(None if spec is None else spec.encode(), n_layer, ctypes.byref(out), warn, 64)
    return rc, out.value, warn.value.decode()


def parse_config(path):
    o = PrefillOptions(0, 1, 0, 8, 0, 0)
    rc = lib.ep_sp_parse_config(path.encode(), ctypes.byref(o))
    return rc, o
