"""Python mirror of the reference's ``fe::cuda`` KV/attention operator
interface (Cambridgebit/FlashEngine.cpp include/fe/native_cuda.hpp:6-14), over
the fe_kv C ABI. Device buffers are torch CUDA tensors (PyTorch is only the
allocator and stream provider here); per-step plan metadata are host arrays.

Names, argument meaning and error behaviour follow the reference:
``create_plan``/``AttentionPlan``, ``prepare_plan``, ``attention``, ``store``;
a failing call raises (the reference throws std::runtime_error).
"""
from __future__ import annotations

import array
import ctypes

import numpy as np

from . import _lib
from ._lib import FE_DTYPE_BF16, FE_DTYPE_F16, FeError, check

_P = ctypes.c_void_p


_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch

        _TORCH = torch
    return _TORCH


def _ptr(t):
    if t is None:
        return None
    return _P(t.data_ptr())


def _stream(stream):
    if stream is None:
        torch = _torch()
        return _P(torch.cuda.current_stream().cuda_stream)
    if hasattr(stream, "cuda_stream"):
        return _P(stream.cuda_stream)
    return _P(int(stream))


def dtype_code(t) -> int:
    torch = _torch()
    if t.dtype == torch.bfloat16:
        return FE_DTYPE_BF16
    if t.dtype == torch.float16:
        return FE_DTYPE_F16
    raise TypeError(f"unsupported dtype {t.dtype}; expected float16 or bfloat16")


def _host_i32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a, dtype=np.int32))


def _require_device_i32(t):
    torch = _torch()
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is torch.int32 and
            t.is_contiguous()):
        raise ValueError("expected a contiguous int32 CUDA tensor")


# ---------------------------------------------------------------------------
# fe::cuda::store  (include/fe/native_cuda.hpp:14)
# ---------------------------------------------------------------------------

def store(k, v, kc, vc, slots, rows=None, width=None, bf16=None, stream=None, cache_slots=None):
    """Scatter rows of k/v into the pools through `slots` (int64, device).
    Rows with a negative slot are skipped, as in the reference CUDA kernel."""
    lib = _lib.load()
    rows = int(slots.shape[0]) if rows is None else int(rows)
    width = int(k.numel() // max(rows, 1)) if width is None else int(width)
    dtype = dtype_code(kc) if bf16 is None else (FE_DTYPE_BF16 if bf16 else FE_DTYPE_F16)
    cache_slots = int(kc.numel() // width) if cache_slots is None else int(cache_slots)
    check(lib.fe_kv_append(_ptr(k), _ptr(v), _ptr(kc), _ptr(vc), _ptr(slots), rows, width, dtype,
                           cache_slots, _stream(stream)), "store")


# ---------------------------------------------------------------------------
# fe::cuda::rope / accept  (include/fe/native_cuda.hpp:13,15) and the fused
# rope + store (no reference counterpart)
# ---------------------------------------------------------------------------

def rope(q, k, pos, cache, stream=None):
    """Rotate q [rows, hq, dim] and k [rows, hkv, dim] in place with the fp32
    cache [max_positions, rotary_dim] (cos | sin); rotary_dim = the cache's
    width (dim for full rotary, less for partial rotary); pos: int64 [rows]."""
    lib = _lib.load()
    rows, hkv, dim = (int(x) for x in k.shape)
    hq = int(q.shape[1]) if q is not None else 0
    check(lib.fe_rope(_ptr(q) if q is not None else None, _ptr(k), _ptr(pos), _ptr(cache), rows,
                      hq, hkv, dim, int(cache.shape[1]), int(cache.shape[0]), dtype_code(k),
                      _stream(stream)), "rope")


def rope_append(q, k, v, kc, vc, slots, pos, cache, k_out=None, stream=None):
    """rope + store in one launch: q rotated in place, rotated k (and v) written
    to the pools [cache_slots, hkv*dim] through `slots`; the rotated keys also
    go to `k_out` when given (it may be `k`). The rotary width is the cache's
    width, as in rope()."""
    lib = _lib.load()
    rows, hkv, dim = (int(x) for x in k.shape)
    hq = int(q.shape[1])
    cache_slots = int(kc.numel() // (hkv * dim))
    check(lib.fe_rope_append(_ptr(q), _ptr(k), _ptr(v), _ptr(k_out) if k_out is not None else None,
                             _ptr(kc), _ptr(vc), _ptr(slots), _ptr(pos), _ptr(cache), rows, hq, hkv,
                             dim, int(cache.shape[1]), int(cache.shape[0]), dtype_code(k),
                             cache_slots, _stream(stream)), "rope_append")


def accept(draft, verify, out, stream=None):
    """Greedy acceptance: draft int64 [batch, k], verify [batch, k+1],
    out [batch, k+2] (device)."""
    lib = _lib.load()
    batch = int(verify.shape[0])
    k = int(verify.shape[1]) - 1
    check(lib.fe_accept(_ptr(draft), _ptr(verify), _ptr(out), batch, k, _stream(stream)),
          "accept")


# ---------------------------------------------------------------------------
# block copy / copy-on-write and page clearing (no reference counterpart)
# ---------------------------------------------------------------------------

def copy_blocks(k_pools, v_pools, src, dst, ntok, page, width, num_pages_total, dtype=None,
                stream=None):
    """Copy token rows [0, ntok[c]) of page src[c] onto page dst[c] in every
    layer's K and V pool. src/dst/ntok: int32 device tensors."""
    lib = _lib.load()
    n = len(k_pools)
    if n != len(v_pools):
        raise ValueError("k_pools and v_pools differ in length")
    kp = (_P * max(n, 1))(*[t.data_ptr() for t in k_pools])
    vp = (_P * max(n, 1))(*[t.data_ptr() for t in v_pools])
    dtype = dtype_code(k_pools[0]) if dtype is None else int(dtype)
    check(lib.fe_kv_copy_blocks(kp, vp, n, _ptr(src), _ptr(dst), _ptr(ntok), int(src.shape[0]),
                                int(page), int(width), int(num_pages_total), dtype,
                                _stream(stream)), "copy_blocks")


def fork_copies(parent_tables, child_tables, fork_lens, page):
    """Copy-on-write lists for forked sequences (host only): for fork f, the
    pages of the first fork_lens[f] tokens that child_tables[f] does not share
    with parent_tables[f] become (src, dst, ntok) entries for copy_blocks.
    Returns three int32 numpy arrays. Raises FeError on tables that would let
    one sequence write a page the other reads (a shared partial tail)."""
    lib = _lib.load()
    n = len(parent_tables)
    if len(child_tables) != n or len(fork_lens) != n:
        raise ValueError("one parent table, child table and fork length per fork")
    pt = [np.asarray(t, np.int32) for t in parent_tables]
    ct = [np.asarray(t, np.int32) for t in child_tables]
    poff = _host_i32(np.concatenate([[0], np.cumsum([len(t) for t in pt])]))
    coff = _host_i32(np.concatenate([[0], np.cumsum([len(t) for t in ct])]))
    pcat = _host_i32(np.concatenate(pt) if n else np.zeros(1, np.int32))
    ccat = _host_i32(np.concatenate(ct) if n else np.zeros(1, np.int32))
    lens = np.ascontiguousarray(np.asarray(fork_lens, np.int64))
    cap = int(sum(-(-int(L) // int(page)) for L in lens)) if n else 0
    src, dst, ntok = (np.zeros(max(cap, 1), np.int32) for _ in range(3))
    count = ctypes.c_int(0)
    hp = lambda a: a.ctypes.data_as(_P)  # noqa: E731
    check(lib.fe_kv_fork_copies(n, hp(pcat), hp(poff), hp(ccat), hp(coff), hp(lens), int(page),
                                hp(src), hp(dst), hp(ntok), cap, ctypes.byref(count)),
          "fork_copies")
    k = count.value
    return src[:k].copy(), dst[:k].copy(), ntok[:k].copy()


def clear_pages(pools, pages, page, width, num_pages_total, dtype=None, stream=None):
    """Zero whole pages (int32 device tensor `pages`) of every pool."""
    lib = _lib.load()
    n = len(pools)
    arr = (_P * max(n, 1))(*[t.data_ptr() for t in pools])
    dtype = dtype_code(pools[0]) if dtype is None else int(dtype)
    check(lib.fe_kv_clear_pages(arr, n, _ptr(pages), int(pages.shape[0]), int(page), int(width),
                                int(num_pages_total), dtype, _stream(stream)), "clear_pages")


def gather(pool, out, kv, pages, last, row_offset, batch, max_len, page, width, dtype=None,
           stream=None):
    """Dense copy of whole sequences' KV rows (device int32 metadata)."""
    lib = _lib.load()
    dtype = dtype_code(pool) if dtype is None else int(dtype)
    check(lib.fe_kv_gather(_ptr(pool), _ptr(out), _ptr(kv), _ptr(pages), _ptr(last),
                           _ptr(row_offset), int(batch), int(max_len), int(page), int(width), dtype,
                           _stream(stream)), "gather")


def paged_decode_noalloc(q, k_pool, v_pool, out, kv, pages, last, batch, hq, hkv, page,
                        num_blocks, max_pages, dtype=None, stream=None):
    """Decode attention through fe_paged_decode_noalloc: no plan and no
    device allocation (split-K scratch is a fixed array inside the library).
    kv/pages/last are int32 DEVICE tensors; one query row per sequence."""
    lib = _lib.load()
    dtype = dtype_code(q) if dtype is None else int(dtype)
    check(lib.fe_paged_decode_noalloc(_ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(out), _ptr(kv),
                                      _ptr(pages), _ptr(last), int(batch), int(hq), int(hkv),
                                      int(page), int(num_blocks), int(max_pages), dtype,
                                      _stream(stream)), "paged_decode_noalloc")


def device_errors(stream=None) -> int:
    """Read and clear the device-side error bits (FE_DEVERR_*)."""
    lib = _lib.load()
    bits = ctypes.c_uint32(0)
    check(lib.fe_device_errors(_stream(stream), ctypes.byref(bits)), "device_errors")
    return int(bits.value)


# ---------------------------------------------------------------------------
# fe::cuda::create_plan / destroy_plan / prepare_plan / attention
# (include/fe/native_cuda.hpp:7-10)
# ---------------------------------------------------------------------------

class AttentionPlan:
    """Owns an fe_attn_plan. `prepare` takes host metadata (as
    fe::cuda::prepare_plan); `attention` takes device tensors."""

    _create = "fe_attn_plan_create"

    def __init__(self, hq, hkv, dim, page, max_batch, max_pages, bf16, blocks):
        self.lib = _lib.load()
        h = _P()
        dtype = FE_DTYPE_BF16 if bf16 else FE_DTYPE_F16
        check(getattr(self.lib, self._create)(int(hq), int(hkv), int(dim), int(page),
                                              int(max_batch), int(max_pages), dtype, int(blocks),
                                              ctypes.byref(h)), "create_plan")
        self.handle = h
        self.hq, self.hkv, self.dim, self.page = hq, hkv, dim, page
        self.bf16, self.blocks = bool(bf16), blocks

    def prepare(self, qo, kv, pages, last, batch=None, rows=None, graph=False, stream=None):
        qo, kv, pages, last = _host_i32(qo), _host_i32(kv), _host_i32(pages), _host_i32(last)
        batch = kv.shape[0] - 1 if batch is None else int(batch)
        rows = int(qo[batch]) if rows is None else int(rows)
        check(self.lib.fe_attn_plan_prepare(self.handle, qo.ctypes.data_as(_P),
                                            kv.ctypes.data_as(_P), pages.ctypes.data_as(_P),
                                            last.ctypes.data_as(_P), batch, rows, int(bool(graph)),
                                            _stream(stream)), "prepare_plan")

    def prepare_device(self, qo, kv, pages, last, batch, rows, stream=None):
        """fe_attn_plan_prepare_device: the same metadata as `prepare`, as
        int32 DEVICE tensors; the work lists are built on the GPU (graph mode,
        nothing read back, capturable in a CUDA graph)."""
        for t in (qo, kv, pages, last):
            _require_device_i32(t)
        check(self.lib.fe_attn_plan_prepare_device(self.handle, _ptr(qo), _ptr(kv), _ptr(pages),
                                                   _ptr(last), int(batch), int(rows),
                                                   _stream(stream)), "prepare_plan_device")

    def step_prepare_device(self, block_tables, starts, rows_per_seq, slots, positions,
                            stream=None):
        """fe_step_prepare_device: slot mapping and work lists on the GPU from
        int32 block tables [batch, stride] and start positions [batch] (< 0:
        graph padding entry); writes int64 slots / positions [batch *
        rows_per_seq]."""
        _require_device_i32(block_tables)
        _require_device_i32(starts)
        batch, stride = int(block_tables.shape[0]), int(block_tables.shape[1])
        if int(starts.shape[0]) != batch:
            raise ValueError("starts must have one entry per block-table row")
        torch = _torch()
        for t in (slots, positions):
            if t.dtype != torch.int64 or not t.is_cuda or t.numel() < batch * rows_per_seq:
                raise ValueError("slots / positions: int64 CUDA tensors of batch*rows_per_seq")
        check(self.lib.fe_step_prepare_device(self.handle, _ptr(block_tables), stride, _ptr(starts),
                                              batch, int(rows_per_seq), _ptr(slots),
                                              _ptr(positions), _stream(stream)),
              "step_prepare_device")

    def device_meta(self, total_pages=None, nbytes=1 << 22, stream=None) -> dict:
        """The plan's device metadata (what the kernels read), copied back and
        unpacked (parse_meta)."""
        buf = np.zeros(int(nbytes), np.uint8)
        check(self.lib.fe_attn_plan_debug_device_meta(self.handle, buf.ctypes.data_as(_P),
                                                      int(nbytes), _stream(stream)),
              "debug_device_meta")
        return parse_meta(buf, total_pages)

    def host_meta(self) -> dict:
        """The host copy of the last host-side prepare's metadata."""
        return _host_meta(self.lib, self.handle)

    def attention(self, q, k, v, out, causal=True, stream=None, lists=None):
        """fe_attn_run; `lists` (FE_ATTN_LISTS_DECODE / _ROWS) runs only part
        of the prepared work (fe_attn_run_lists)."""
        if lists is None:
            check(self.lib.fe_attn_run(self.handle, _ptr(q), _ptr(k), _ptr(v), _ptr(out),
                                       int(bool(causal)), _stream(stream)), "attention")
        else:
            check(self.lib.fe_attn_run_lists(self.handle, _ptr(q), _ptr(k), _ptr(v), _ptr(out),
                                             int(bool(causal)), int(lists), _stream(stream)),
                  "attention")

    def info(self) -> dict:
        inf = _lib.PlanInfo()
        check(self.lib.fe_attn_plan_get_info(self.handle, ctypes.byref(inf)), "plan_info")
        return {name: getattr(inf, name) for name, _ in _lib.PlanInfo._fields_}

    def close(self):
        if getattr(self, "handle", None):
            self.lib.fe_attn_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---------------------------------------------------------------------------
# 8-bit KV cache (no reference counterpart)
# ---------------------------------------------------------------------------

class Kv8Pool:
    """One layer's K or V in 8 bits: `codes` [cache_slots, hkv, dim] in
    float8_e4m3fn and `exps` uint8 [cache_slots / 16, hkv], the biased
    exponents of the scales of 16 slots (value = code * 2 ** (exp - 127)).
    Both contiguous CUDA tensors on one device; they may be slices of larger
    tensors that hold all layers. A pool is made once and keeps its tensors,
    so what a call needs of them (shape, device, addresses) is read here."""

    __slots__ = ("codes", "exps", "shape", "device", "index", "codes_ptr", "exps_ptr")

    def __init__(self, codes, exps):
        torch = _torch()
        for name, t, dt, nd in (("codes", codes, torch.float8_e4m3fn, 3),
                                ("exps", exps, torch.uint8, 2)):
            if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dt and
                    t.dim() == nd and t.is_contiguous()):
                raise ValueError(f"{name}: expected a contiguous {nd}-d {dt} CUDA tensor")
        if codes.shape[0] % _lib.FE_KV8_BLOCK or \
                tuple(exps.shape) != (codes.shape[0] // _lib.FE_KV8_BLOCK, codes.shape[1]):
            raise ValueError(f"exps {tuple(exps.shape)} do not fit codes {tuple(codes.shape)}: "
                             "one row per 16 slots")
        if exps.get_device() != codes.get_device():
            raise ValueError("codes and exps are on different devices")
        self.codes, self.exps = codes, exps
        self.shape, self.device = tuple(codes.shape), codes.device
        self.index = codes.get_device()
        self.codes_ptr, self.exps_ptr = codes.data_ptr(), exps.data_ptr()

    @classmethod
    def empty(cls, num_blocks, page, hkv, dim, device="cuda"):
        """A zeroed pool of num_blocks pages and the padding page."""
        torch = _torch()
        slots = (int(num_blocks) + 1) * int(page)
        codes = torch.zeros(slots, hkv, dim, dtype=torch.uint8, device=device)
        exps = torch.full((slots // _lib.FE_KV8_BLOCK, hkv), 127, dtype=torch.uint8, device=device)
        return cls(codes.view(torch.float8_e4m3fn), exps)

    @property
    def cache_slots(self):
        return self.shape[0]


# These calls are short enough on the GPU that a decode step is bound by the
# host; their checks read each tensor attribute once and pass plain integers.
# Kernels run on the current device: what they are given has to be there.

def _kv8_device():
    return _torch()._C._cuda_getDevice()


def _kv8_stream(stream, device):
    if stream is None:
        return _torch()._C._cuda_getCurrentRawStream(device)
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _kv8_rows(name, t, dtype, shape, device):
    """Address of a contiguous tensor of this dtype and shape on CUDA device
    `device`."""
    if t is None:
        raise ValueError(f"{name} is missing")
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{name}: expected a contiguous {dtype} tensor {tuple(shape)} on the current "
                     f"device (cuda:{device}), got {t.dtype} {tuple(t.shape)} {tuple(t.stride())} "
                     f"on {t.device}")


def _kv8_pools(device, *pools):
    """Pools of a call on CUDA device `device`."""
    for p in pools:
        if p.index != device:
            raise ValueError(f"a pool is on {p.device}, the current device is cuda:{device}")


def _kv8_lists(device, *lists):
    """Contiguous int32 tensors on CUDA device `device`."""
    torch = _torch()
    tensor, i32 = torch.Tensor, torch.int32
    for t in lists:
        if not (isinstance(t, tensor) and t.dtype is i32 and t.get_device() == device and
                t.is_contiguous()):
            raise ValueError("expected a contiguous int32 tensor on the current device "
                             f"(cuda:{device})")


def append_kv8(q, k, v, kpool, vpool, slots, pos=None, cache=None, q_out=None, stream=None):
    """rope_append into 8-bit pools, one launch: q [rows, hq, dim] rotated into
    `q_out` (default: in place; q may be None), k [rows, hkv, dim] rotated and
    v quantised into `kpool` / `vpool` through `slots` (int64 [rows]). pos int64
    [rows] and cache fp32 [max_positions, rotary_dim] as in rope(); cache None
    rotates nothing. Rows of one 16-slot block must be adjacent and in order."""
    torch = _torch()
    shape, dt = k.shape, k.dtype
    pool = kpool.shape
    if len(shape) != 3 or pool != vpool.shape or shape[1:] != pool[1:]:
        raise ValueError(f"k {tuple(shape)} and pools {pool}, {vpool.shape} do not fit")
    rows, hkv, dim = shape
    if dt is torch.bfloat16:
        code = FE_DTYPE_BF16
    elif dt is torch.float16:
        code = FE_DTYPE_F16
    else:
        raise ValueError(f"k: expected float16 or bfloat16, got {dt}")
    device = _kv8_device()
    if kpool.index != device or vpool.index != device:
        _kv8_pools(device, kpool, vpool)
    if k.get_device() != device or not k.is_contiguous():
        raise ValueError(f"k: expected a contiguous tensor on the current device (cuda:{device})")
    vp = _kv8_rows("v", v, dt, shape, device)
    hq = rot = most = 0
    qp = op = pp = cp = None
    if q is not None:
        qs = q.shape
        hq = qs[1] if len(qs) == 3 else -1
        qp = op = _kv8_rows("q", q, dt, (rows, hq, dim), device)
        if q_out is not None:
            op = _kv8_rows("q_out", q_out, dt, qs, device)
    sp = _kv8_rows("slots", slots, torch.int64, (rows,), device)
    if cache is not None:
        cs = cache.shape
        most, rot = cs
        if rot:
            pp = _kv8_rows("pos", pos, torch.int64, (rows,), device)
            cp = _kv8_rows("cache", cache, torch.float32, cs, device)
    rc = _lib.load().fe_kv8_append(qp, op, k.data_ptr(), vp, kpool.codes_ptr, vpool.codes_ptr,
                                   kpool.exps_ptr, vpool.exps_ptr, sp, pp, cp, rows, hq, hkv, dim,
                                   rot, most, code, pool[0], _kv8_stream(stream, device))
    if rc:
        check(rc, "append_kv8")


def gather_kv8(pool, out, kv, pages, last, row_offset, max_len, page, stream=None):
    """Whole sequences' values from an 8-bit pool into rows of `out` [rows,
    hkv, dim] (16-bit), metadata as gather(): int32 CUDA tensors. A sequence
    whose rows reach past `out`, or whose pages past `pages`, is skipped and
    flagged (device_errors)."""
    device = _kv8_device()
    _kv8_pools(device, pool)
    _kv8_lists(device, kv, pages, last, row_offset)
    batch = last.numel()
    if not last.shape == row_offset.shape == (batch,) or kv.shape != (batch + 1,):
        raise ValueError("last and row_offset must have one entry per sequence, kv one more")
    slots, hkv, dim = pool.shape
    rows, odd = divmod(out.numel(), hkv * dim)
    if odd or out.get_device() != device or not out.is_contiguous():
        raise ValueError("out: expected a contiguous tensor [rows, hkv, dim] on the current device "
                         f"(cuda:{device})")
    check(_lib.load().fe_kv8_gather_within(pool.codes_ptr, pool.exps_ptr, out.data_ptr(),
                                           rows, kv.data_ptr(), pages.data_ptr(), pages.numel(),
                                           last.data_ptr(), row_offset.data_ptr(), batch, max_len,
                                           page, hkv, dim, dtype_code(out), slots,
                                           _kv8_stream(stream, device)), "gather_kv8")


def copy_blocks_kv8(k_pools, v_pools, src, dst, ntok, page, stream=None):
    """copy_blocks for 8-bit pools (lists of Kv8Pool, one per layer): codes
    and scales. src/dst/ntok: int32 CUDA tensors."""
    n = len(k_pools)
    if n != len(v_pools):
        raise ValueError("k_pools and v_pools differ in length")
    device = _kv8_device()
    _kv8_lists(device, src, dst, ntok)
    if not src.shape == dst.shape == ntok.shape:
        raise ValueError("src, dst and ntok differ in length")
    if n == 0:
        return
    shape = k_pools[0].shape
    ptrs = [[p.codes_ptr for p in side if p.index == device and p.shape == shape]
            for side in (k_pools, v_pools)] + \
        [[p.exps_ptr for p in side] for side in (k_pools, v_pools)]
    if len(ptrs[0]) != n or len(ptrs[1]) != n:
        _kv8_pools(device, *k_pools, *v_pools)
        raise ValueError("the layers' pools differ in shape")
    arrays = [array.array("Q", p) for p in ptrs]
    check(_lib.load().fe_kv8_copy_blocks(*[a.buffer_info()[0] for a in arrays], n, src.data_ptr(),
                                         dst.data_ptr(), ntok.data_ptr(), src.shape[0], page,
                                         shape[1], shape[2], shape[0] // page,
                                         _kv8_stream(stream, device)), "copy_blocks_kv8")


def _kv8_metadata(qo, kv, last, batch):
    """The lengths that a prepare of `batch` sequences reads."""
    if batch < 0 or qo.shape[0] <= batch or kv.shape[0] <= batch or last.shape[0] < batch:
        raise ValueError(f"{batch} sequences need {batch + 1} entries of qo and kv and {batch} of "
                         f"last, got {qo.shape[0]}, {kv.shape[0]} and {last.shape[0]}")


class Kv8Plan(AttentionPlan):
    """An attention plan over 8-bit pools: prepared like any other plan;
    `attention` takes Kv8Pools. bf16: the dtype of q and out."""

    _create = "fe_kv8_plan_create"

    def __init__(self, hq, hkv, dim, page, max_batch, max_pages, bf16, blocks):
        super().__init__(hq, hkv, dim, page, max_batch, max_pages, bf16, blocks)
        torch = _torch()
        self.pool_shape = ((int(blocks) + 1) * int(page), int(hkv), int(dim))
        self.dtype = torch.bfloat16 if bf16 else torch.float16
        self.rows = 0  # query rows of the last prepare
        self.index = _kv8_device()

    def _device(self):
        """The current device, which has to be the plan's."""
        device = _kv8_device()
        if self.index != device:
            raise ValueError(f"the plan is for cuda:{self.index}, the current device is "
                             f"cuda:{device}")
        return device

    def prepare(self, qo, kv, pages, last, batch=None, rows=None, graph=False, stream=None):
        self._device()
        qo, kv, pages, last = _host_i32(qo), _host_i32(kv), _host_i32(pages), _host_i32(last)
        batch = kv.shape[0] - 1 if batch is None else int(batch)
        _kv8_metadata(qo, kv, last, batch)
        if pages.shape[0] < kv[batch]:
            raise ValueError(f"{pages.shape[0]} pages, kv counts {kv[batch]}")
        super().prepare(qo, kv, pages, last, batch, rows, graph, stream)
        self.rows = int(qo[batch])

    def prepare_device(self, qo, kv, pages, last, batch, rows, stream=None):
        _kv8_lists(self._device(), qo, kv, pages, last)
        _kv8_metadata(qo, kv, last, int(batch))
        super().prepare_device(qo, kv, pages, last, batch, rows, stream)
        self.rows = int(rows)

    def step_prepare_device(self, block_tables, starts, rows_per_seq, slots, positions,
                            stream=None):
        device = self._device()
        _kv8_lists(device, block_tables, starts)
        for t in (slots, positions):
            if t.get_device() != device or not t.is_contiguous():
                raise ValueError("slots / positions: contiguous int64 tensors on the current "
                                 f"device (cuda:{device})")
        super().step_prepare_device(block_tables, starts, rows_per_seq, slots, positions, stream)
        self.rows = int(block_tables.shape[0]) * int(rows_per_seq)

    def attention(self, q, kpool, vpool, out, causal=True, stream=None):
        if kpool.shape != self.pool_shape or vpool.shape != self.pool_shape:
            raise ValueError(f"pools of shape {kpool.shape}, {vpool.shape}: the plan is for "
                             f"{self.pool_shape}")
        shape = (q.shape[0], self.hq, self.dim)
        if shape[0] < self.rows:
            raise ValueError(f"q has {shape[0]} rows, the plan was prepared for {self.rows}")
        device = self._device()
        if kpool.index != device or vpool.index != device:
            _kv8_pools(device, kpool, vpool)
        check(self.lib.fe_kv8_attn_run(self.handle, _kv8_rows("q", q, self.dtype, shape, device),
                                       kpool.codes_ptr, vpool.codes_ptr, kpool.exps_ptr,
                                       vpool.exps_ptr,
                                       _kv8_rows("out", out, self.dtype, shape, device),
                                       1 if causal else 0, _kv8_stream(stream, device)),
              "attention")


def create_plan(hq, hkv, dim, page, max_batch, max_pages, bf16, blocks) -> AttentionPlan:
    return AttentionPlan(hq, hkv, dim, page, max_batch, max_pages, bf16, blocks)


def destroy_plan(plan: AttentionPlan):
    plan.close()


def prepare_plan(plan: AttentionPlan, qo, kv, pages, last, batch, rows, graph=False, stream=None):
    plan.prepare(qo, kv, pages, last, batch, rows, graph, stream)


def attention(plan: AttentionPlan, q, k, v, output, causal=True, stream=None):
    plan.attention(q, k, v, output, causal, stream)


# ---------------------------------------------------------------------------
# host-only planner (test hook): inspect the work list without a GPU
# ---------------------------------------------------------------------------

ITEM_DTYPE = np.dtype([("seq", "<i4"), ("kvh", "<i2"), ("key_mode", "<i2"), ("rb0", "<i4"),
                       ("nrb", "<i4"), ("kt0", "<i4"), ("kt1", "<i4"), ("part", "<i4"),
                       ("group", "<i4")])
GROUP_DTYPE = np.dtype([("nsplit", "<i4"), ("part0", "<i4"), ("rec_floats", "<i4"),
                        ("rows", "<i4"), ("seq", "<i4"), ("kvh", "<i4"), ("row0", "<i4"),
                        ("rows_per_head", "<i4")])
SEQ_DTYPE = np.dtype([("q_row0", "<i4"), ("qrows", "<i4"), ("length", "<i4"),
                      ("page_off", "<i4")])


def _host_meta(lib, handle) -> dict:
    """The host copy of the last host-side prepare's metadata, unpacked."""
    n = ctypes.c_int64(0)
    check(lib.fe_attn_plan_debug_meta(handle, None, 0, ctypes.byref(n)), "meta")
    buf = np.zeros(n.value, dtype=np.uint8)
    check(lib.fe_attn_plan_debug_meta(handle, buf.ctypes.data_as(_P), n.value, ctypes.byref(n)),
          "meta")
    return parse_meta(buf)


def parse_meta(buf: np.ndarray, total_pages: int | None = None) -> dict:
    """Unpack a plan's metadata blob (fe_attn_plan.h layout; section order
    from the header's offsets). `total_pages` defaults to everything between
    the pages offset and the end (the host planner puts the pages last)."""
    h = buf[:128].view(np.int32)
    out = {"batch": int(h[18]), "rows": int(h[19]), "chunk_tiles": int(h[23]),
           "dec_heads": int(h[24]), "views": []}
    seqs_off, pages_off = int(h[20]), int(h[21])
    batch = out["batch"]
    out["seqs"] = buf[seqs_off:seqs_off + SEQ_DTYPE.itemsize * batch].view(SEQ_DTYPE)
    # lists: 0 = row work (non-causal), 1 = row work (causal), 2 = decode work
    for c in range(3):
        n_items, n_groups, grid = int(h[0 + c]), int(h[3 + c]), int(h[6 + c])
        co, io, go = int(h[9 + c]), int(h[12 + c]), int(h[15 + c])
        view = {
            "grid": grid,
            "n_items": n_items,
            "cta_off": (buf[co:co + 4 * (grid + 1)].view(np.int32) if grid
                        else np.zeros(1, np.int32)),
            "items": buf[io:io + ITEM_DTYPE.itemsize * n_items].view(ITEM_DTYPE),
            "groups": buf[go:go + GROUP_DTYPE.itemsize * n_groups].view(GROUP_DTYPE),
        }
        out["views"].append(view)
    end = int(h[22]) if total_pages is None else pages_off + 4 * int(total_pages)
    out["pages"] = buf[pages_off:end].view(np.int32)
    out["buf"] = buf
    return out


class HostPlan:
    """fe_attn_plan_create_host: validates metadata and builds the work list
    on the host for `grid_cap` CTAs, without touching a GPU."""

    _create = "fe_attn_plan_create_host"

    def __init__(self, hq, hkv, dim, page, max_batch, max_pages, bf16, blocks, grid_cap=296):
        self.lib = _lib.load()
        h = _P()
        dtype = FE_DTYPE_BF16 if bf16 else FE_DTYPE_F16
        check(getattr(self.lib, self._create)(int(hq), int(hkv), int(dim), int(page),
                                              int(max_batch), int(max_pages), dtype, int(blocks),
                                              int(grid_cap), ctypes.byref(h)), "create_host")
        self.handle = h
        self.G = hq // hkv

    def prepare(self, qo, kv, pages, last, batch=None, rows=None, graph=False):
        qo, kv, pages, last = _host_i32(qo), _host_i32(kv), _host_i32(pages), _host_i32(last)
        batch = kv.shape[0] - 1 if batch is None else int(batch)
        rows = int(qo[batch]) if rows is None else int(rows)
        check(self.lib.fe_attn_plan_prepare(self.handle, qo.ctypes.data_as(_P),
                                            kv.ctypes.data_as(_P), pages.ctypes.data_as(_P),
                                            last.ctypes.data_as(_P), batch, int(rows),
                                            int(bool(graph)), None), "prepare_plan")
        return self.meta()

    def meta(self) -> dict:
        return _host_meta(self.lib, self.handle)

    def close(self):
        if getattr(self, "handle", None):
            self.lib.fe_attn_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class HostKv8Plan(HostPlan):
    """HostPlan with the lists of a Kv8Plan."""

    _create = "fe_kv8_plan_create_host"


__all__ = ["Kv8Pool", "Kv8Plan", "HostKv8Plan", "append_kv8", "gather_kv8", "copy_blocks_kv8",
           "store", "copy_blocks", "paged_decode_noalloc", "clear_pages", "gather", "device_errors", "AttentionPlan",
           "create_plan", "destroy_plan", "prepare_plan", "attention", "HostPlan", "FeError",
           "dtype_code", "ITEM_DTYPE", "GROUP_DTYPE", "SEQ_DTYPE", "parse_meta"]
