"""Python binding of the B200 paged-attention library (libnvb.so).

This mirrors the checked wrappers the reference's Rust device layer puts in
front of its C ABI (src/gpu.rs:482-509 tensor extents / alignment / aliasing,
src/gpu.rs:775-995 qkv_rope_cached, paged_attention and flash_attention),
for torch tensors. Every call goes through the C ABI declared in
include/nvb_attention.h; there is no CPU or PyTorch fallback: if the CUDA
library is missing, loading fails loudly.

The package directory is named ``nano-vllm-rs_b200`` (not importable with a
plain ``import``); load it with ``__graft_entry__.load_package()`` which
registers it as ``nano_vllm_rs_b200``.
"""
from __future__ import annotations

import bisect
import ctypes
import os
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
LIB_DIR = PKG_DIR / "_lib"
LIB_PATH = LIB_DIR / "libnvb.so"
HOST_LIB_PATH = LIB_DIR / "libnvb_host.so"
INCLUDE_DIR = PKG_DIR.parent / "include"

_lib = None
_host = None

c_int, c_float, c_void_p, c_char_p = ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_char_p
_P = c_void_p
_LL = ctypes.c_longlong


def _declare(lib):
    sig = {
        "nvb_paged_fwd": [_P] * 8 + [c_int] * 9 + [_P] * 3,
        "nvb_paged_fwd_ex": [_P] * 8 + [c_int] * 9 + [_P] * 3 + [c_int],
        "nvb_num_splits": [c_int] * 5,
        "nvb_attention": [_P] * 8 + [c_int] * 9,
        "nvb_attention_splitkv": [_P] * 8 + [c_int] * 9 + [_P, c_int],
        "nvb_qkv_rope_cached": [_P] * 9 + [c_int] * 6 + [c_float, _P, c_int],
        "nvb_qkv_rope": [_P] * 9 + [c_int] * 6 + [c_float, c_float],
        "nvb_rope_cache": [_P, _P, c_int, c_int, c_float],
        "nvb_capture_begin": [_P],
        "nvb_capture_end": [_P, ctypes.POINTER(c_void_p)],
        "nvb_capture_abort": [_P],
        "nvb_graph_replay": [_P, _P],
        "nvb_graph_destroy": [_P],
        "nvb_device_error": [ctypes.POINTER(c_int)],
        "nvb_clear_device_error": [],
        "nvb_paged_decode_gather": [_P] * 8 + [c_int] * 8 + [_P] * 4 + [c_int, c_int, ctypes.c_uint],
        "nvb_paged_decode_gather_capturable": [_P] * 8 + [c_int] * 8 + [_P] * 5 + [c_int, c_int],
        "nvb_paged_tree_fwd": [_P] * 9 + [c_int] * 10 + [_P] * 3 + [c_int],
        "nvb_tree_num_splits": [c_int] * 6,
        "nvb_tree_parts": [c_int],
        "nvb_cache_copy_pages": [_P] * 3 + [c_int] + [_P] * 3 + [c_int] * 5,
        "nvb_cache_compact_paths": [_P] * 3 + [c_int] + [_P] * 6 + [c_int] * 7,
        "nvb_latent_store": [_P, _P, _LL, _P, _P, _P, _P, _P, _LL, _LL, _P, _LL, _LL] + [c_int] * 5 + [c_float, _P, c_int],
        "nvb_latent_gather": [_P] * 5 + [_LL, _P, _LL] + [c_int] * 5,
        "nvb_paged_latent_fwd": [_P] * 7 + [c_int] * 7 + [c_float, _P, _P, _LL],
        "nvb_latent_scratch_floats": [c_int],
        "nvb_latent_prefill_fwd": [_P] * 4 + [_LL] + [_P] * 3 + [c_int] * 5 + [c_float, _P],
        "nvb_peer_buffer_create": [ctypes.c_size_t, ctypes.POINTER(c_void_p), _P],
        "nvb_peer_buffer_open": [_P, ctypes.POINTER(c_void_p)],
        "nvb_peer_buffer_close": [_P],
        "nvb_peer_buffer_free": [_P],
    }
    for name, args in sig.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = None if name in ("nvb_capture_abort", "nvb_graph_destroy") else c_int
    lib.nvb_latent_scratch_floats.restype = _LL
    for name in ("nvb_last_error", "nvb_version"):
        getattr(lib, name).restype = c_char_p
        getattr(lib, name).argtypes = []


def library():
    """Loads libnvb.so (built by ``build.py``); raises if it is missing."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: run __graft_entry__.build() first")
        lib = ctypes.CDLL(str(LIB_PATH))
        _declare(lib)
        _lib = lib
    return _lib


class NvbError(RuntimeError):
    pass


def _check(code: int):
    if code != 0:
        msg = library().nvb_last_error().decode(errors="replace")
        raise NvbError(f"libnvb: {msg} (status {code})")


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _stream(stream=None):
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _tensor(t, shape, dtype, name):
    """Extent/dtype/contiguity check, like Gpu::tensor (src/gpu.rs:482-501)."""
    if t is None:
        raise NvbError(f"{name} is required")
    if not t.is_cuda:
        raise NvbError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise NvbError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise NvbError(f"{name} must be contiguous")
    need = 1
    for d in shape:
        need *= int(d)
    if t.numel() < need:
        raise NvbError(f"{name} has {t.numel()} elements, needs {need} for shape {tuple(shape)}")


def _span(t):
    start = t.data_ptr()
    return start, start + t.numel() * t.element_size()


def _distinct(output, inputs, name):
    """Rejects an output that overlaps an input (src/gpu.rs:502-509)."""
    o0, o1 = _span(output)
    for t in inputs:
        if t is None:
            continue
        a0, a1 = _span(t)
        if o0 < a1 and a0 < o1:
            raise NvbError(f"{name} aliases an input or another output")


def _refuse(t, shape, dtype, name, device):
    if t.get_device() != device:
        raise NvbError(f"{name} is on {t.device}, the current device is cuda:{device}")
    if t.dtype is not dtype:
        raise NvbError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise NvbError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise NvbError(f"{name} must be contiguous")


def _pointers(arguments, written, device):
    """Addresses of the arguments (name, tensor or None, shape, type): each of
    that shape and type, contiguous and on the device, and none that is in
    `written` overlapping another."""
    pointers, spans = [], []
    for name, t, shape, dtype in arguments:
        if t is None:
            pointers.append(None)
            continue
        if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != device:
            _refuse(t, shape, dtype, name, device)
        p = t.data_ptr()
        pointers.append(p)
        spans.append((p, p + t.nbytes, name))
    spans.sort()
    end, held = 0, False
    for a, z, name in spans:
        if a < end and a < z and (held or name in written):
            raise NvbError(f"{name} overlaps another argument")
        if z > end:
            end, held = z, name in written
    return pointers


def _raw_stream(stream, device):
    """The stream's handle; that of the device's current stream without one."""
    import torch

    return stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(device)


def num_splits(batch, q_heads, kv_heads, max_k, num_sms):
    return library().nvb_num_splits(batch, q_heads, kv_heads, max_k, num_sms)


def splitkv_scratch(num_splits_, batch, q_heads, device):
    """Caller-owned FP32 split-KV scratch (lse_accum, out_accum)."""
    import torch

    lse_accum = torch.empty(num_splits_, batch, q_heads, dtype=torch.float32, device=device)
    out_accum = torch.empty(num_splits_, batch, q_heads, 128, dtype=torch.float32, device=device)
    return lse_accum, out_accum


def peer_buffer_create(nbytes):
    """A zeroed device buffer of this GPU to share with the node's other ranks:
    returns (device pointer, 64-byte CUDA IPC handle)."""
    ptr = c_void_p()
    handle = ctypes.create_string_buffer(64)
    _check(library().nvb_peer_buffer_create(nbytes, ctypes.byref(ptr), handle))
    return ptr.value, handle.raw


def peer_buffer_open(handle):
    """Maps another rank's buffer (its IPC handle) into this process."""
    ptr = c_void_p()
    buf = ctypes.create_string_buffer(bytes(handle), 64)
    _check(library().nvb_peer_buffer_open(buf, ctypes.byref(ptr)))
    return ptr.value


def peer_buffer_close(ptr):
    _check(library().nvb_peer_buffer_close(c_void_p(ptr)))


def peer_buffer_free(ptr):
    _check(library().nvb_peer_buffer_free(c_void_p(ptr)))


def paged_decode_gather(q, k, v, out_local, cu_q, kv_lens, block_table, *, batch, max_k, q_heads, kv_heads,
                        block_size, table_stride, num_blocks, num_splits, lse_accum, out_accum, peer_out, peer_flag,
                        rank, epoch, stream=None, check=True):
    """Decode of this rank's kv heads with the combine fused into the
    all-gather of the outputs (nvb_paged_decode_gather): `peer_out` and
    `peer_flag` are every rank's output and flag device pointers (ints)."""
    import torch

    world = len(peer_out)
    if check:
        _tensor(q, (batch, q_heads, 128), torch.bfloat16, "q")
        _tensor(out_local, (batch, q_heads, 128), torch.bfloat16, "out_local")
        for t, nm in ((k, "k"), (v, "v")):
            _tensor(t, (num_blocks, block_size, kv_heads, 128), torch.bfloat16, nm)
        _tensor(cu_q, (batch + 1,), torch.int32, "cu_q")
        _tensor(kv_lens, (batch,), torch.int32, "kv_lens")
        _tensor(block_table, (batch, table_stride), torch.int32, "block_table")
        if num_splits > 1:
            _tensor(lse_accum, (num_splits, batch, q_heads), torch.float32, "lse_accum")
            _tensor(out_accum, (num_splits, batch, q_heads, 128), torch.float32, "out_accum")
        if len(peer_flag) != world or not 1 <= world <= 8:
            raise ValueError("peer_out and peer_flag need one pointer per rank (1..8 ranks)")
    outs = (c_void_p * world)(*peer_out)
    flags = (c_void_p * world)(*peer_flag)
    _check(library().nvb_paged_decode_gather(
        _stream(stream), _ptr(q), _ptr(k), _ptr(v), _ptr(out_local), _ptr(cu_q), _ptr(kv_lens), _ptr(block_table),
        batch, max_k, q_heads, kv_heads, block_size, table_stride, num_blocks, num_splits, _ptr(lse_accum),
        _ptr(out_accum), ctypes.cast(outs, c_void_p), ctypes.cast(flags, c_void_p), world, rank, epoch))


def paged_decode_gather_capturable(q, k, v, out_local, cu_q, kv_lens, block_table, *, batch, max_k, q_heads,
                                   kv_heads, block_size, table_stride, num_blocks, num_splits, lse_accum, out_accum,
                                   peer_out0, peer_out1, peer_flag, rank, stream=None, check=True):
    """nvb_paged_decode_gather_capturable: the same step with the epoch kept
    in device memory (slot len(peer_flag) of this rank's flags), so that a
    CUDA graph can capture it once; step n writes output set n & 1
    (`peer_out1` for odd n)."""
    import torch

    world = len(peer_out0)
    if check:
        _tensor(q, (batch, q_heads, 128), torch.bfloat16, "q")
        _tensor(out_local, (batch, q_heads, 128), torch.bfloat16, "out_local")
        for t, nm in ((k, "k"), (v, "v")):
            _tensor(t, (num_blocks, block_size, kv_heads, 128), torch.bfloat16, nm)
        _tensor(cu_q, (batch + 1,), torch.int32, "cu_q")
        _tensor(kv_lens, (batch,), torch.int32, "kv_lens")
        _tensor(block_table, (batch, table_stride), torch.int32, "block_table")
        if num_splits > 1:
            _tensor(lse_accum, (num_splits, batch, q_heads), torch.float32, "lse_accum")
            _tensor(out_accum, (num_splits, batch, q_heads, 128), torch.float32, "out_accum")
        if len(peer_out1) != world or len(peer_flag) != world or not 1 <= world <= 8:
            raise ValueError("peer_out0, peer_out1 and peer_flag need one pointer per rank (1..8 ranks)")
    o0 = (c_void_p * world)(*peer_out0)
    o1 = (c_void_p * world)(*peer_out1)
    flags = (c_void_p * world)(*peer_flag)
    _check(library().nvb_paged_decode_gather_capturable(
        _stream(stream), _ptr(q), _ptr(k), _ptr(v), _ptr(out_local), _ptr(cu_q), _ptr(kv_lens), _ptr(block_table),
        batch, max_k, q_heads, kv_heads, block_size, table_stride, num_blocks, num_splits, _ptr(lse_accum),
        _ptr(out_accum), ctypes.cast(o0, c_void_p), ctypes.cast(o1, c_void_p), ctypes.cast(flags, c_void_p), world,
        rank))


def paged_fwd(q, k, v, out, cu_q, kv_lens, block_table, *, batch, max_q, max_k, q_heads, kv_heads,
              block_size, table_stride, num_blocks, num_splits=1, lse=None, lse_accum=None,
              out_accum=None, stream=None, check=True):
    """Paged attention through nvb_paged_fwd_ex (the bounded entry point).

    Same argument meaning as the reference's Gpu::flash_attention
    (src/gpu.rs:890-995) / nvr_flash_fwd.
    """
    import torch

    total_q = q.shape[0]
    if check:
        for t, nm in ((q, "q"), (out, "out")):
            _tensor(t, (total_q, q_heads, 128), torch.bfloat16, nm)
        for t, nm in ((k, "k"), (v, "v")):
            _tensor(t, (num_blocks, block_size, kv_heads, 128), torch.bfloat16, nm)
        _tensor(cu_q, (batch + 1,), torch.int32, "cu_q")
        _tensor(kv_lens, (batch,), torch.int32, "kv_lens")
        _tensor(block_table, (batch, table_stride), torch.int32, "block_table")
        if lse is not None:
            _tensor(lse, (batch, q_heads, max_q), torch.float32, "lse")
        if num_splits > 1:
            _tensor(lse_accum, (num_splits, batch, q_heads), torch.float32, "lse_accum")
            _tensor(out_accum, (num_splits, batch, q_heads, 128), torch.float32, "out_accum")
        inputs = [q, k, v, cu_q, kv_lens, block_table]
        outputs = [out, lse, lse_accum, out_accum]
        for i, o in enumerate(outputs):
            if o is not None:
                _distinct(o, inputs + [x for x in outputs[:i] if x is not None], "output")
    lib = library()
    _check(lib.nvb_paged_fwd_ex(_stream(stream), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(cu_q),
                                _ptr(kv_lens), _ptr(block_table), batch, total_q, max_q, max_k, q_heads,
                                kv_heads, block_size, table_stride, num_splits, _ptr(lse), _ptr(lse_accum),
                                _ptr(out_accum), num_blocks))


_sm_counts = {}


def _num_sms(device):
    count = _sm_counts.get(device)
    if count is None:
        import torch

        count = _sm_counts[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return count


def tree_num_splits(batch, max_q, q_heads, kv_heads, max_k, num_sms=None):
    """Split count of paged_tree_fwd for a GPU of num_sms SMs (default: the current device's)."""
    if num_sms is None:
        import torch

        num_sms = _num_sms(torch.cuda.current_device())
    return library().nvb_tree_num_splits(batch, max_q, q_heads, kv_heads, max_k, num_sms)


def tree_scratch(num_splits_, total_q, q_heads, device):
    """Caller-owned FP32 scratch (lse_accum, out_accum) of paged_tree_fwd: one row of each for each of the
    nvb_tree_parts(num_splits) parts; (None, None) where it needs none."""
    parts = library().nvb_tree_parts(num_splits_)
    if parts == 1:
        return None, None
    return splitkv_scratch(parts, total_q, q_heads, device)


def paged_tree_fwd(q, k, v, out, cu_q, kv_lens, block_table, tree_mask, *, batch, max_q, max_k, q_heads, kv_heads,
                   block_size, table_stride, num_blocks, num_splits=1, lse=None, lse_accum=None, out_accum=None,
                   stream=None, check=True):
    """Attention of drafted trees over the paged cache (nvb_paged_tree_fwd).

    Queries cu_q[b]..cu_q[b + 1] are sequence b's nodes, whose keys are the
    last of its kv_lens[b] keys in the same order; tree_mask [total_q, words]
    int64 has bit t % 64 of word t // 64 set where a node attends to node t
    (host.tree_mask). The keys before the tree are visible to all. lse, where
    given, is [total_q, q_heads]. lse_accum and out_accum: tree_scratch of
    num_splits (or more parts).
    """
    import torch

    total_q, words, device = q.shape[0], tree_mask.shape[-1], torch.cuda.current_device()
    if check:
        bf16, i32, f32 = torch.bfloat16, torch.int32, torch.float32
        rows, cache = (total_q, q_heads, 128), (num_blocks, block_size, kv_heads, 128)
        lse_parts = out_parts = 1
        if lse_accum is not None or out_accum is not None:
            parts = library().nvb_tree_parts(num_splits)
            lse_parts, out_parts = (parts if t is None else max((parts, *t.shape[:1])) for t in (lse_accum, out_accum))
        pointers = _pointers(
            (("q", q, rows, bf16), ("k", k, cache, bf16), ("v", v, cache, bf16), ("out", out, rows, bf16),
             ("cu_q", cu_q, (batch + 1,), i32), ("kv_lens", kv_lens, (batch,), i32),
             ("block_table", block_table, (batch, table_stride), i32),
             ("tree_mask", tree_mask, (total_q, words), torch.int64), ("lse", lse, (total_q, q_heads), f32),
             ("lse_accum", lse_accum, (lse_parts, total_q, q_heads), f32),
             ("out_accum", out_accum, (out_parts, total_q, q_heads, 128), f32)),
            ("out", "lse", "lse_accum", "out_accum"), device)
    else:
        pointers = [t.data_ptr() if t is not None else None
                    for t in (q, k, v, out, cu_q, kv_lens, block_table, tree_mask, lse, lse_accum, out_accum)]
    _check(library().nvb_paged_tree_fwd(_raw_stream(stream, device), *pointers[:8], words, batch, total_q, max_q,
                                        max_k, q_heads, kv_heads, block_size, table_stride, num_splits, *pointers[8:],
                                        num_blocks))


class CacheLayers:
    """The K and V caches of a model's layers ([num_blocks, block_size,
    kv_heads, head_dim] BF16 each), checked once, for the copies below. Keeps
    the tensors alive."""

    def __init__(self, k_caches, v_caches):
        import torch

        k_caches, v_caches = list(k_caches), list(v_caches)
        if not k_caches or len(k_caches) != len(v_caches):
            raise NvbError(f"{len(k_caches)} K caches and {len(v_caches)} V caches")
        if k_caches[0].dim() != 4:
            raise NvbError("a cache must be [num_blocks, block_size, kv_heads, head_dim]")
        self.shape, self.layers = tuple(k_caches[0].shape), len(k_caches)
        self.device = torch.cuda.current_device()
        names = [(f"{n}[{i}]", t) for n, ts in (("k_caches", k_caches), ("v_caches", v_caches)) for i, t in enumerate(ts)]
        pointers = _pointers([(n, t, self.shape, torch.bfloat16) for n, t in names], [n for n, _ in names], self.device)
        self._tensors = k_caches + v_caches
        self._starts = sorted(pointers)
        self._bytes = k_caches[0].numel() * 2
        self._k = (c_void_p * self.layers)(*pointers[:self.layers])
        self._v = (c_void_p * self.layers)(*pointers[self.layers:])

    def _pointers(self, arguments, written=()):
        """Addresses of the arguments, checked; none may lie in a cache."""
        import torch

        if self.device != torch.cuda.current_device():
            raise NvbError(f"the caches are on cuda:{self.device}, the current device is "
                           f"cuda:{torch.cuda.current_device()}")
        pointers = _pointers(arguments, written, self.device)
        for (name, t, shape, dtype), p in zip(arguments, pointers):
            if p is None:
                continue
            i = bisect.bisect_right(self._starts, p + t.nbytes - 1) - 1
            if i >= 0 and p < self._starts[i] + self._bytes:
                raise NvbError(f"{name} lies in a cache")
        return pointers


def cache_copy_pages(layers, src, dst, rows=None, *, stream=None):
    """Copies page src[i] to page dst[i] in every cache of `layers` (a
    CacheLayers), its first rows[i] tokens where rows is given
    (nvb_cache_copy_pages). src, dst and rows are int32 CUDA tensors; no page
    may be the target of two pairs, nor a target and a source."""
    import torch

    num_blocks, block_size, kv_heads, head_dim = layers.shape
    pairs, i32 = src.numel(), torch.int32
    pointers = layers._pointers((("src", src, (pairs,), i32), ("dst", dst, (pairs,), i32), ("rows", rows, (pairs,), i32)))
    _check(library().nvb_cache_copy_pages(_raw_stream(stream, layers.device), layers._k, layers._v, layers.layers,
                                          *pointers, pairs, kv_heads, head_dim, block_size, num_blocks))


def cache_compact_paths(layers, cu_q, kv_lens, block_table, path, counts, new_kv_lens, *, stream=None):
    """Moves the K and V rows of each sequence's accepted path (path and counts
    of model.layer_verify) together behind its context, in every cache of
    `layers` (a CacheLayers), and writes the lengths that are left to
    new_kv_lens (nvb_cache_compact_paths)."""
    import torch

    num_blocks, block_size, kv_heads, head_dim = layers.shape
    batch, i32 = kv_lens.numel(), torch.int32
    if path.dim() != 2 or block_table.dim() != 2:
        raise NvbError("path and block_table must have a row for each sequence")
    table_stride, path_stride = block_table.shape[1], path.shape[1]
    pointers = layers._pointers(
        (("cu_q", cu_q, (batch + 1,), i32), ("kv_lens", kv_lens, (batch,), i32),
         ("block_table", block_table, (batch, table_stride), i32), ("path", path, (batch, path_stride), i32),
         ("counts", counts, (batch,), i32), ("new_kv_lens", new_kv_lens, (batch,), i32)), ("new_kv_lens",))
    _check(library().nvb_cache_compact_paths(_raw_stream(stream, layers.device), layers._k, layers._v, layers.layers,
                                             *pointers, batch, path_stride, kv_heads, head_dim, block_size,
                                             table_stride, num_blocks))


LATENT_DIM, LATENT_ROPE, LATENT_WIDTH = 512, 64, 576  # of a row of the latent cache


def _refuse_misfit(arguments, device):
    """The error for the first of the arguments (name, tensor, shape, type, whether only its last dimension has to be
    contiguous) that does not fit; what they overlap the library checks."""
    for name, t, shape, dtype, rows in arguments:
        if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not (rows or t.is_contiguous()):
            _refuse(t, shape, dtype, name, device)
        if rows and t.stride(-1) != 1:
            raise NvbError(f"{name}'s last dimension must be contiguous")
    raise NvbError("the arguments do not fit")


def _latent_cache(cache):
    if cache.dim() != 3 or cache.shape[2] != LATENT_WIDTH:
        raise NvbError(f"cache must be [num_blocks, block_size, {LATENT_WIDTH}], got {tuple(cache.shape)}")
    return cache.shape


def latent_store(kv, weight, positions, slots, cache, *, rope_table, eps=1e-6, q=None, q_out=None, interleaved=False,
                 stream=None):
    """Appends a step's latents to the latent cache and rotates the queries'
    rotary parts (nvb_latent_store).

    kv [rows, 576] (its rows may be slices of longer ones): 512 latent values,
    normalised with `weight` [512] and `eps`, and 64 key values, rotated by
    positions [rows] int32; row r goes to slot slots[r] of cache [num_blocks,
    block_size, 576]. q and q_out [rows, heads, 64] are slices of the queries:
    q_out is q itself (the default) or does not overlap it. kv None rotates
    queries only (weight, slots and cache None). rope_table [positions, 64]:
    host.rope_table.
    """
    import torch

    device, i32, bf16 = torch.cuda.current_device(), torch.int32, torch.bfloat16
    if kv is None and q is None:
        raise NvbError("kv or q is required")
    if positions is None or rope_table is None or rope_table.dim() != 2:
        raise NvbError("positions [rows] and rope_table [positions, 64] are required")
    if kv is not None and kv.dim() != 2:
        raise NvbError("kv must be [rows, 576]")
    rows, max_positions = (kv if kv is not None else q).shape[0], rope_table.shape[0]
    heads = num_blocks = block_size = kv_stride = 0
    kv_at = weight_at = slots_at = cache_at = q_at = out_at = None
    strides = out_strides = (0, 0)
    at = positions.data_ptr(), rope_table.data_ptr()
    fine = (positions.dtype is i32 and positions.shape == (rows,) and positions.is_contiguous()
            and positions.get_device() == device and rope_table.dtype is torch.float32
            and rope_table.shape[1] == LATENT_ROPE and rope_table.is_contiguous() and rope_table.get_device() == device)
    if kv is not None:
        if weight is None or slots is None or cache is None:
            raise NvbError("weight, slots and cache go with kv")
        num_blocks, block_size, _ = _latent_cache(cache)
        kv_at, weight_at, slots_at, cache_at = kv.data_ptr(), weight.data_ptr(), slots.data_ptr(), cache.data_ptr()
        kv_stride = kv.stride(0) if rows > 1 else LATENT_WIDTH
        fine = (fine and kv.dtype is bf16 and kv.shape == (rows, LATENT_WIDTH) and kv.stride(1) == 1
                and kv.get_device() == device and weight.dtype is bf16 and weight.shape == (LATENT_DIM,)
                and weight.is_contiguous() and weight.get_device() == device and slots.dtype is i32
                and slots.shape == (rows,) and slots.is_contiguous() and slots.get_device() == device
                and cache.dtype is bf16 and cache.is_contiguous() and cache.get_device() == device)
    elif weight is not None or slots is not None or cache is not None:
        raise NvbError("weight, slots and cache go with kv")
    if q is not None:
        if q.dim() != 3:
            raise NvbError("q must be [rows, heads, 64]")
        if q_out is None:
            q_out = q
        heads, strides, out_strides = q.shape[1], q.stride(), q_out.stride()
        q_at, out_at = q.data_ptr(), q_out.data_ptr()
        if rows == 1 or heads == 1:  # strides of such dimensions say nothing
            keep = (rows > 1, heads > 1, 1)
            strides, out_strides = ([s * k for s, k in zip(x, keep)] for x in (strides, out_strides))
        shape = (rows, heads, LATENT_ROPE)
        fine = (fine and q.dtype is bf16 and q.shape == shape and strides[-1] == 1 and q.get_device() == device
                and q_out.dtype is bf16 and q_out.shape == shape and out_strides[-1] == 1
                and q_out.get_device() == device)
    elif q_out is not None:
        raise NvbError("q_out goes with q")
    if not fine:
        arguments = [("positions", positions, (rows,), i32, False),
                     ("rope_table", rope_table, (max_positions, LATENT_ROPE), torch.float32, False)]
        if kv is not None:
            arguments += [("kv", kv, (rows, LATENT_WIDTH), bf16, True), ("weight", weight, (LATENT_DIM,), bf16, False),
                          ("slots", slots, (rows,), i32, False), ("cache", cache, cache.shape, bf16, False)]
        if q is not None:
            arguments += [("q", q, shape, bf16, True), ("q_out", q_out, shape, bf16, True)]
        _refuse_misfit(arguments, device)
    _check(library().nvb_latent_store(
        _raw_stream(stream, device), kv_at, kv_stride, weight_at, at[0], slots_at, cache_at, q_at, strides[0],
        strides[1], out_at, out_strides[0], out_strides[1], rows, heads, interleaved, block_size, num_blocks, eps,
        at[1], max_positions))


def latent_gather(cache, block_table, cu_k, latent, rope, *, stream=None):
    """Copies the first cu_k[b + 1] - cu_k[b] cached rows of every sequence to
    latent [total_k, 512] and rope [total_k, 64] (nvb_latent_gather); both may
    be slices of longer rows."""
    import torch

    device, i32, bf16 = torch.cuda.current_device(), torch.int32, torch.bfloat16
    num_blocks, block_size, _ = shape = _latent_cache(cache)
    if block_table.dim() != 2 or latent.dim() != 2 or rope.dim() != 2:
        raise NvbError("block_table and latent must have rows")
    (batch, table_stride), total_k = block_table.shape, latent.shape[0]
    if not (cache.dtype is bf16 and cache.is_contiguous() and cache.get_device() == device
            and block_table.dtype is i32 and block_table.is_contiguous() and block_table.get_device() == device
            and cu_k.dtype is i32 and cu_k.shape == (batch + 1,) and cu_k.is_contiguous()
            and cu_k.get_device() == device
            and latent.dtype is bf16 and latent.shape[1] == LATENT_DIM and latent.stride(1) == 1
            and latent.get_device() == device
            and rope.dtype is bf16 and rope.shape == (total_k, LATENT_ROPE) and rope.stride(1) == 1
            and rope.get_device() == device):
        _refuse_misfit((("cache", cache, shape, bf16, False), ("block_table", block_table, block_table.shape, i32, False),
                        ("cu_k", cu_k, (batch + 1,), i32, False), ("latent", latent, (total_k, LATENT_DIM), bf16, True),
                        ("rope", rope, (total_k, LATENT_ROPE), bf16, True)), device)
    strides = (latent.stride(0), rope.stride(0)) if total_k > 1 else (LATENT_DIM, LATENT_ROPE)
    _check(library().nvb_latent_gather(_raw_stream(stream, device), cache.data_ptr(), block_table.data_ptr(),
                                       cu_k.data_ptr(), latent.data_ptr(), strides[0], rope.data_ptr(), strides[1],
                                       batch, total_k, block_size, table_stride, num_blocks))


def latent_scratch(device):
    """FP32 scratch of paged_latent_fwd on `device`, whatever the batch; calls that may overlap need their own."""
    import torch

    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    return torch.empty(library().nvb_latent_scratch_floats(_num_sms(index)), dtype=torch.float32, device=device)


def paged_latent_fwd(q, cache, out, cu_q, kv_lens, block_table, *, max_q, scale, scratch, lse=None, stream=None):
    """Absorbed attention over the paged latent cache (nvb_paged_latent_fwd).

    q [total_q, heads, 576] attends to cache [num_blocks, block_size, 576], out
    [total_q, heads, 512] takes the weighted sums of its first 512 values, lse,
    where given, [total_q, heads]. Sequence b's queries cu_q[b]..cu_q[b + 1] are
    the last of its kv_lens[b] tokens. max_q: the most queries of a sequence.
    scratch: latent_scratch.
    """
    import torch

    device, bf16, i32, f32 = torch.cuda.current_device(), torch.bfloat16, torch.int32, torch.float32
    num_blocks, block_size, _ = shape = _latent_cache(cache)
    if q.dim() != 3 or block_table.dim() != 2 or scratch is None:
        raise NvbError("q must be [total_q, heads, 576], block_table a row for each sequence, scratch latent_scratch's")
    (total_q, heads, width), (batch, table_stride) = q.shape, block_table.shape
    if not (q.dtype is bf16 and width == LATENT_WIDTH and q.is_contiguous() and q.get_device() == device
            and cache.dtype is bf16 and cache.is_contiguous() and cache.get_device() == device
            and out.dtype is bf16 and out.shape == (total_q, heads, LATENT_DIM) and out.is_contiguous()
            and out.get_device() == device
            and cu_q.dtype is i32 and cu_q.shape == (batch + 1,) and cu_q.is_contiguous()
            and cu_q.get_device() == device
            and kv_lens.dtype is i32 and kv_lens.shape == (batch,) and kv_lens.is_contiguous()
            and kv_lens.get_device() == device
            and block_table.dtype is i32 and block_table.is_contiguous() and block_table.get_device() == device
            and scratch.dtype is f32 and scratch.is_contiguous() and scratch.get_device() == device
            and (lse is None or lse.dtype is f32 and lse.shape == (total_q, heads) and lse.is_contiguous()
                 and lse.get_device() == device)):
        arguments = [("q", q, (total_q, heads, LATENT_WIDTH), bf16, False), ("cache", cache, shape, bf16, False),
                     ("out", out, (total_q, heads, LATENT_DIM), bf16, False), ("cu_q", cu_q, (batch + 1,), i32, False),
                     ("kv_lens", kv_lens, (batch,), i32, False),
                     ("block_table", block_table, block_table.shape, i32, False),
                     ("scratch", scratch, scratch.shape, f32, False)]
        _refuse_misfit(arguments + ([("lse", lse, (total_q, heads), f32, False)] if lse is not None else []), device)
    _check(library().nvb_paged_latent_fwd(
        _raw_stream(stream, device), q.data_ptr(), cache.data_ptr(), out.data_ptr(), cu_q.data_ptr(),
        kv_lens.data_ptr(), block_table.data_ptr(), batch, total_q, max_q, heads, block_size, table_stride, num_blocks,
        scale, lse.data_ptr() if lse is not None else None, scratch.data_ptr(), scratch.numel()))


def latent_prefill_fwd(q, kv, k_rope, out, cu_q, cu_k, *, max_q, scale, lse=None, stream=None):
    """Causal attention over expanded latent keys and values (nvb_latent_prefill_fwd).

    q [total_q, heads, 192] (128 values and the 64 rotated ones), kv [total_k,
    heads, 256] (128 key values and 128 values a head), k_rope [total_k, 64]
    (rows may be slices of longer ones), out [total_q, heads, 128], lse, where
    given, [total_q, heads]. Sequence b's queries are the last of its keys
    cu_k[b]..cu_k[b + 1]. max_q: the most queries of a sequence.
    """
    import torch

    device, bf16, i32, f32 = torch.cuda.current_device(), torch.bfloat16, torch.int32, torch.float32
    if q.dim() != 3 or kv.dim() != 3 or k_rope.dim() != 2:
        raise NvbError("q must be [total_q, heads, 192], kv [total_k, heads, 256]")
    (total_q, heads, width), total_k, batch = q.shape, kv.shape[0], cu_q.numel() - 1
    if not (q.dtype is bf16 and width == 192 and q.is_contiguous() and q.get_device() == device
            and kv.dtype is bf16 and kv.shape == (total_k, heads, 256) and kv.is_contiguous()
            and kv.get_device() == device
            and k_rope.dtype is bf16 and k_rope.shape == (total_k, LATENT_ROPE) and k_rope.stride(1) == 1
            and k_rope.get_device() == device
            and out.dtype is bf16 and out.shape == (total_q, heads, 128) and out.is_contiguous()
            and out.get_device() == device
            and cu_q.dtype is i32 and cu_q.dim() == 1 and cu_q.is_contiguous() and cu_q.get_device() == device
            and cu_k.dtype is i32 and cu_k.shape == (batch + 1,) and cu_k.is_contiguous()
            and cu_k.get_device() == device
            and (lse is None or lse.dtype is f32 and lse.shape == (total_q, heads) and lse.is_contiguous()
                 and lse.get_device() == device)):
        arguments = [("q", q, (total_q, heads, 192), bf16, False), ("kv", kv, (total_k, heads, 256), bf16, False),
                     ("k_rope", k_rope, (total_k, LATENT_ROPE), bf16, True),
                     ("out", out, (total_q, heads, 128), bf16, False), ("cu_q", cu_q, (batch + 1,), i32, False),
                     ("cu_k", cu_k, (batch + 1,), i32, False)]
        _refuse_misfit(arguments + ([("lse", lse, (total_q, heads), f32, False)] if lse is not None else []), device)
    _check(library().nvb_latent_prefill_fwd(
        _raw_stream(stream, device), q.data_ptr(), kv.data_ptr(), k_rope.data_ptr(),
        k_rope.stride(0) if total_k > 1 else LATENT_ROPE, out.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), batch,
        total_q, total_k, max_q, heads, scale, lse.data_ptr() if lse is not None else None))


def attention(q, kcache, vcache, positions, seq_indices, tables, out, *, rows, q_heads, kv_heads, head_dim,
              block_size, num_blocks, table_stride, batch, max_context, scratch=None, partitions=1,
              stream=None):
    """Native-form paged attention (Gpu::paged_attention, src/gpu.rs:829-887)."""
    import torch

    _tensor(q, (rows, q_heads, head_dim), torch.bfloat16, "q")
    _tensor(out, (rows, q_heads, head_dim), torch.bfloat16, "out")
    for t, nm in ((kcache, "kcache"), (vcache, "vcache")):
        _tensor(t, (num_blocks, block_size, kv_heads, head_dim), torch.bfloat16, nm)
    _tensor(positions, (rows,), torch.int32, "positions")
    _tensor(seq_indices, (rows,), torch.int32, "seq_indices")
    _tensor(tables, (batch, table_stride), torch.int32, "tables")
    _distinct(out, [q, kcache, vcache, positions, seq_indices, tables], "out")
    lib = library()
    if partitions > 1:
        _tensor(scratch, (rows * q_heads * partitions * (head_dim + 2),), torch.float32, "scratch")
        _check(lib.nvb_attention_splitkv(_stream(stream), _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(positions),
                                         _ptr(seq_indices), _ptr(tables), _ptr(out), rows, q_heads, kv_heads,
                                         head_dim, block_size, num_blocks, table_stride, batch, max_context,
                                         _ptr(scratch), partitions))
    else:
        _check(lib.nvb_attention(_stream(stream), _ptr(q), _ptr(kcache), _ptr(vcache), _ptr(positions),
                                 _ptr(seq_indices), _ptr(tables), _ptr(out), rows, q_heads, kv_heads, head_dim,
                                 block_size, num_blocks, table_stride, batch, max_context))


def qkv_rope_cached(qkv, q_weight, k_weight, positions, slots, qout, kcache, vcache, *, rows, q_heads, kv_heads,
                    head_dim, block_size, num_blocks, eps, rope_cache, max_positions, stream=None, check=True):
    """Fused norm + RoPE + KV store (Gpu::qkv_rope_cached, src/gpu.rs:775-825)."""
    import torch

    if check:
        _tensor(qkv, (rows, q_heads + 2 * kv_heads, head_dim), torch.bfloat16, "qkv")
        _tensor(q_weight, (head_dim,), torch.bfloat16, "q_weight")
        _tensor(k_weight, (head_dim,), torch.bfloat16, "k_weight")
        _tensor(positions, (rows,), torch.int32, "positions")
        _tensor(slots, (rows,), torch.int32, "slots")
        _tensor(qout, (rows, q_heads, head_dim), torch.bfloat16, "qout")
        for t, nm in ((kcache, "kcache"), (vcache, "vcache")):
            _tensor(t, (num_blocks, block_size, kv_heads, head_dim), torch.bfloat16, nm)
        _tensor(rope_cache, (max_positions, head_dim), torch.float32, "rope_cache")
        inputs = [qkv, q_weight, k_weight, positions, slots, rope_cache]
        _distinct(qout, inputs + [kcache, vcache], "qout")
        _distinct(kcache, inputs + [vcache], "kcache")
        _distinct(vcache, inputs, "vcache")
    _check(library().nvb_qkv_rope_cached(_stream(stream), _ptr(qkv), _ptr(q_weight), _ptr(k_weight),
                                         _ptr(positions), _ptr(slots), _ptr(qout), _ptr(kcache), _ptr(vcache),
                                         rows, q_heads, kv_heads, head_dim, block_size, num_blocks, float(eps),
                                         _ptr(rope_cache), max_positions))


def qkv_rope(qkv, q_weight, k_weight, positions, slots, qout, kcache, vcache, *, rows, q_heads, kv_heads, head_dim,
             block_size, num_blocks, eps, theta, stream=None):
    """Fused norm + RoPE + KV store with in-kernel angles (nv_qkv_rope)."""
    _check(library().nvb_qkv_rope(_stream(stream), _ptr(qkv), _ptr(q_weight), _ptr(k_weight), _ptr(positions),
                                  _ptr(slots), _ptr(qout), _ptr(kcache), _ptr(vcache), rows, q_heads, kv_heads,
                                  head_dim, block_size, num_blocks, float(eps), float(theta)))


def rope_cache(cache, positions, head_dim, theta, stream=None):
    import torch

    _tensor(cache, (positions, head_dim), torch.float32, "rope_cache")
    _check(library().nvb_rope_cache(_stream(stream), _ptr(cache), positions, head_dim, float(theta)))


def device_error():
    code = c_int(0)
    _check(library().nvb_device_error(ctypes.byref(code)))
    return code.value


def clear_device_error():
    _check(library().nvb_clear_device_error())


class Graph:
    """A captured CUDA graph (mirrors Gpu::capture / Graph, src/gpu.rs:511-533,
    1128-1146). Keeps references to the tensors the capture used so their
    memory outlives the graph."""

    def __init__(self, handle, keep):
        self._handle = handle
        self._keep = keep

    def replay(self, stream=None):
        _check(library().nvb_graph_replay(self._handle, _stream(stream)))

    def close(self):
        if self._handle:
            library().nvb_graph_destroy(self._handle)
            self._handle = None
            self._keep = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_captures = []  # what each capture that is under way keeps


def _hold(*tensors):
    """Keeps the memory that a call allocated for itself for the graph that is being captured."""
    if _captures:
        _captures[-1].extend(tensors)


def capture(fn, keep=(), stream=None):
    """Captures the device work `fn()` enqueues on `stream` into a Graph, which
    keeps `keep` and the workspaces that the calls in `fn` allocate."""
    s = _stream(stream)
    lib = library()
    _check(lib.nvb_capture_begin(s))
    kept = list(keep)
    _captures.append(kept)
    try:
        fn()
    except BaseException:
        lib.nvb_capture_abort(s)
        raise
    finally:
        _captures[:] = [c for c in _captures if c is not kept]
    handle = ctypes.c_void_p(0)
    _check(lib.nvb_capture_end(s, ctypes.byref(handle)))
    return Graph(handle, kept)


def version():
    return library().nvb_version().decode()


from . import workloads  # noqa: E402  (seeded benchmark inputs)
from . import engine  # noqa: E402,F401  (continuous-batching scheduler, libnvb_host.so)
from . import model  # noqa: E402,F401  (Qwen3 runner, libnvb_model.so)
