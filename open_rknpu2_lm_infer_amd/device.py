"""Device-resident use of the C ABI (rk_npu_hip.h) with torch tensors.

torch provides device memory and streams only; every computation is a
hip_matmul kernel launched through the C ABI on torch's current stream.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Dict, List, Optional, Tuple

from . import _ffi as F
from .attention import KV_FORMATS
from .npu import NpuError, _Handle, _Shared, check, ensure, int32

_DT = {}


def _dtype_code(t) -> int:
    if not _DT:
        import torch
        _DT.update({torch.float32: F.RK_NPU_HIP_F32, torch.float16: F.RK_NPU_HIP_F16})
    code = _DT.get(t.dtype)
    if code is None:
        raise NpuError(f"unsupported activation dtype {t.dtype}")
    return code


def current_stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class DeviceContext:
    """One context + allocation domain; owns weights and workspaces."""

    def __init__(self, domain_id: int = 0, device: Optional[str] = None):
        self.shared = _Shared(domain_id, device)
        self._ws: Dict[Tuple[int, int, int, int], _Handle] = {}

    @property
    def domain(self):
        return self.shared.domain.raw

    def weights(self, bits: int, codes, scales) -> "DeviceWeights":
        """codes: int8 [K][N] cuda tensor, scales: f32 [N] cuda tensor."""
        import torch
        ensure(codes.is_cuda and scales.is_cuda and codes.dtype == torch.int8 and scales.dtype == torch.float32,
               "device weights need cuda int8 codes and f32 scales")
        codes = codes.contiguous()
        scales = scales.contiguous()
        k, n = codes.shape
        L = F.lib()
        torch.cuda.synchronize()
        if bits == 4:
            raw = L.rk_npu_hip_w4a8_weights_create_device(self.domain, ctypes.byref(F.rk_npu_i4_weight_config(k, n, 0)),
                                                          ctypes.c_void_p(codes.data_ptr()),
                                                          ctypes.c_void_p(scales.data_ptr()))
            h = _Handle(raw, L.rk_npu_w4a8_weights_free, "W4 weights", self.shared)
        else:
            raw = L.rk_npu_hip_f32i8f32_weights_create_device(self.domain,
                                                              ctypes.byref(F.rk_npu_matmul_weight_config(k, n, k)),
                                                              ctypes.c_void_p(codes.data_ptr()),
                                                              ctypes.c_void_p(scales.data_ptr()))
            h = _Handle(raw, L.rk_npu_f32i8f32_weights_free, "W8 weights", self.shared)
        return DeviceWeights(h, bits, k, n)

    def weights_from_checkpoint(self, bits: int, k: int, parts) -> "DeviceWeights":
        """Weights from checkpoint storage on the device, fused along N in order.
        parts: (data, scales, fmt) with data a cuda tensor of int32 words
        [n][ceil(k*bits/32)] (fmt RK_NPU_HIP_PACK_QUANTIZED) or int8 codes [n][k]
        (RK_NPU_HIP_INT_QUANTIZED, bits 8) and scales f32 [n]."""
        import torch
        torch.cuda.synchronize()
        arr = (F.rk_npu_hip_checkpoint_part * len(parts))()
        n_total = 0
        keep = []
        for i, (data, scales, fmt) in enumerate(parts):
            ensure(data.is_cuda and scales.is_cuda and scales.dtype == torch.float32, "checkpoint parts must be on the GPU")
            data, scales = data.contiguous(), scales.contiguous()
            keep += [data, scales]
            arr[i] = F.rk_npu_hip_checkpoint_part(data.data_ptr(), scales.data_ptr(), data.shape[0], fmt)
            n_total += data.shape[0]
        L = F.lib()
        raw = L.rk_npu_hip_weights_create_checkpoint(self.domain, bits, k, arr, len(parts))
        free = L.rk_npu_w4a8_weights_free if bits == 4 else L.rk_npu_f32i8f32_weights_free
        h = _Handle(raw, free, f"W{bits} weights from checkpoint storage", self.shared)
        return DeviceWeights(h, bits, k, n_total)

    def workspace(self, bits: int, rows: int, k: int, n: int, cached: bool = True) -> _Handle:
        """The context's workspace for (bits, rows, k, n), created on first use;
        cached=False creates a new one (sized by the plan switches in force,
        e.g. for split-K partials under HM_SPLITS) and does not keep it."""
        key = (bits, rows, k, n)
        if not cached:
            saved = self._ws.pop(key, None)
            try:
                return self.workspace(bits, rows, k, n)
            finally:
                self._ws.pop(key, None)
                if saved is not None:
                    self._ws[key] = saved
        if key not in self._ws:
            L = F.lib()
            if bits == 4:
                cfg = F.rk_npu_w4a8_config()
                opt = F.rk_npu_w4a8_options()
                L.rk_npu_w4a8_config_init(ctypes.byref(cfg), rows, n, k)
                L.rk_npu_w4a8_options_init(ctypes.byref(opt))
                self._ws[key] = _Handle(L.rk_npu_w4a8_workspace_create_ex(self.domain, ctypes.byref(cfg),
                                                                          ctypes.byref(opt)),
                                        L.rk_npu_w4a8_workspace_free, "W4 workspace", self.shared)
            else:
                st = F.rk_npu_matmul_strategy()
                st.op_kind = F.RK_NPU_MATMUL_F32I8F32_DYNAMIC
                st.M, st.N, st.K, st.k_tile = rows, n, k, k
                self._ws[key] = _Handle(L.rk_npu_matmul_workspace_create(self.domain, ctypes.byref(st)),
                                        L.rk_npu_matmul_workspace_free, "W8 workspace", self.shared)
        return self._ws[key]

    def attention_workspace(self, cache, own: bool = False) -> _Handle:
        """The context's attention workspace for the geometry of a cache (KvCacheQ8 or KvPages), created on
        first use (rk_npu_attention_f16_prepare); own: a new one, for calls that
        overlap others (a second stream, graphs launched side by side)."""
        c = cache.config.attention
        key = ("attention", c.query_heads, c.kv_heads, c.head_dim, c.softmax_scale, c.mask_mode, c.max_query_rows)
        if not own and key in self._ws:
            return self._ws[key]
        raw = ctypes.c_void_p()
        check(F.lib().rk_npu_attention_f16_prepare(self.domain, ctypes.byref(c), ctypes.byref(raw)),
              "prepare attention")
        ws = _Handle(raw.value, F.lib().rk_npu_attention_f16_workspace_free, "attention workspace", self.shared)
        if not own:
            self._ws[key] = ws
        return ws


class DeviceWeights:
    def __init__(self, handle: _Handle, bits: int, k: int, n: int):
        self.handle, self.bits, self.k, self.n = handle, bits, k, n

    def bytes(self) -> int:
        """Algorithmic weight bytes: codes at storage width plus f32 scales."""
        return self.k * self.n * self.bits // 8 + 4 * self.n


def linear(ctx: DeviceContext, w: DeviceWeights, x, out, rows: int, swiglu: bool = False, ws=None, stream=None):
    ws = ws or ctx.workspace(w.bits, rows, w.k, w.n)
    rc = F.lib().rk_npu_hip_linear_run(ws.raw, w.handle.raw, w.bits, ctypes.c_void_p(x.data_ptr()), _dtype_code(x),
                                       ctypes.c_void_p(out.data_ptr()), _dtype_code(out), rows,
                                       F.RK_NPU_HIP_SWIGLU if swiglu else F.RK_NPU_HIP_PLAIN,
                                       stream if stream is not None else current_stream())
    check(rc, "device linear")


def ffn(ctx: DeviceContext, gate_up: DeviceWeights, down: DeviceWeights, x, out, rows: int, gws=None, dws=None,
        stream=None):
    gws = gws or ctx.workspace(gate_up.bits, rows, gate_up.k, gate_up.n)
    dws = dws or ctx.workspace(down.bits, rows, down.k, down.n)
    rc = F.lib().rk_npu_hip_ffn_run(gws.raw, gate_up.handle.raw, gate_up.bits, dws.raw, down.handle.raw, down.bits,
                                    ctypes.c_void_p(x.data_ptr()), _dtype_code(x), ctypes.c_void_p(out.data_ptr()),
                                    _dtype_code(out), rows, stream if stream is not None else current_stream())
    check(rc, "device FFN")


def _stream(stream, t):
    """`stream`, or torch's current one on the tensor's GPU (as a number: a Stream
    object takes 2 us to make, a third of a call that reads a short cache)."""
    import torch
    return stream if stream is not None else torch._C._cuda_getCurrentRawStream(t.get_device())


class KvCacheQ8:
    """A KV cache of one sequence in 8 bits (rk_npu_attention_q8.h): fmt "i8" or
    "e4m3", one scale for each `block` tokens (32, 64 or 128) and KV head, the
    tokens after the last complete block in fp16. Holds up to `capacity` tokens,
    allocated at once unless initial_capacity is smaller (append on the device
    allocates nothing: reserve first).

    Arrays are cuda tensors [heads][rows][head_dim], f16 or f32, any strides of
    heads and rows (the transposed view of a token-major projection, say)."""

    def __init__(self, ctx: DeviceContext, query_heads: int, kv_heads: int, head_dim: int, softmax_scale: float,
                 capacity: int, fmt: str = "i8", block: int = 32, causal: bool = True, max_query_rows: int = 128,
                 initial_capacity: Optional[int] = None):
        ensure(fmt in KV_FORMATS, f"KV format must be one of {sorted(KV_FORMATS)}")
        initial = capacity if initial_capacity is None else initial_capacity
        for name, value in (("query_heads", query_heads), ("kv_heads", kv_heads), ("head_dim", head_dim),
                            ("capacity", capacity), ("max_query_rows", max_query_rows), ("initial_capacity", initial),
                            ("block", block)):
            int32(value, name)
        L = F.lib()
        cfg = F.rk_npu_hip_attention_q8_config()
        L.rk_npu_hip_attention_q8_config_init(ctypes.byref(cfg))
        a = cfg.attention
        a.query_heads, a.kv_heads, a.head_dim, a.softmax_scale = query_heads, kv_heads, head_dim, softmax_scale
        a.max_query_rows, a.max_capacity = max_query_rows, capacity
        a.initial_capacity = initial
        a.mask_mode = F.RK_NPU_ATTENTION_F16_CAUSAL if causal else F.RK_NPU_ATTENTION_F16_NO_MASK
        cfg.format, cfg.block = KV_FORMATS[fmt], block
        raw = ctypes.c_void_p()
        check(L.rk_npu_hip_attention_q8_cache_create(ctx.domain, ctypes.byref(cfg), ctypes.byref(raw)),
              "create the 8-bit KV cache")
        self.handle = _Handle(raw.value, L.rk_npu_hip_attention_q8_cache_free, "8-bit KV cache", ctx.shared)
        self.ctx, self.config = ctx, cfg
        self._kv, self._query = (kv_heads, head_dim), (query_heads, head_dim)

    def info(self) -> F.rk_npu_attention_f16_cache_info:
        info = F.rk_npu_attention_f16_cache_info()
        check(F.lib().rk_npu_hip_attention_q8_cache_get_info(self.handle.raw, ctypes.byref(info)), "8-bit KV info")
        return info

    @property
    def length(self) -> int:
        return self.info().length

    def bytes(self) -> int:
        info = self.info()
        return info.key_bytes + info.value_bytes + info.tail_bytes

    def reserve(self, capacity: int) -> None:
        check(F.lib().rk_npu_hip_attention_q8_cache_reserve(self.ctx.shared.ctx.raw, self.handle.raw,
                                                           int32(capacity, "capacity")),
              "reserve the 8-bit KV cache")

    def truncate(self, length: int) -> None:
        """Keeps the first `length` tokens; exact within the open block and the last complete one."""
        check(F.lib().rk_npu_hip_attention_q8_cache_truncate(self.handle.raw, int32(length, "length")),
              "truncate the 8-bit KV cache")

    def append(self, k, v, stream=None) -> None:
        """Appends k and v, [kv_heads][rows][head_dim]."""
        shape = k.shape
        ensure(shape == v.shape, "k and v must have the same shape")
        kh, vh = _heads(k, *self._kv), _heads(v, *self._kv)
        check(F.lib().rk_npu_hip_attention_q8_device_append(self.handle.raw, ctypes.byref(kh), ctypes.byref(vh),
                                                            shape[1], _stream(stream, k)),
              "append to the 8-bit KV cache")

    def read(self, first: int, k, v, stream=None) -> None:
        """The values of tokens first.. into k and v, [kv_heads][rows][head_dim]."""
        shape = k.shape
        ensure(shape == v.shape, "k and v must have the same shape")
        kh, vh = _heads(k, *self._kv), _heads(v, *self._kv)
        check(F.lib().rk_npu_hip_attention_q8_device_read(self.handle.raw, int32(first, "first"), shape[1],
                                                          ctypes.byref(kh), ctypes.byref(vh), _stream(stream, k)),
              "read the 8-bit KV cache")


def _heads(t, heads: int, head_dim: int) -> F.rk_npu_hip_heads:
    shape, stride = t.shape, t.stride()
    if not (len(shape) == 3 and shape[0] == heads and shape[2] == head_dim and stride[2] == 1 and t.is_cuda):
        raise NpuError(f"attention arrays are cuda [{heads}][rows][{head_dim}] tensors with contiguous rows")
    if shape[1] >= 2 ** 31:
        int32(shape[1], "rows")
    code = _DT.get(t.dtype)
    return F.rk_npu_hip_heads(t.data_ptr(), _dtype_code(t) if code is None else code, stride[0], stride[1])


def attention_q8(ctx: DeviceContext, cache: KvCacheQ8, q, out, position: int, ws=None, stream=None):
    """Attention of the rows q [query_heads][rows][head_dim], the first at
    `position`, over the cache's tokens. ws: the context's workspace of this
    geometry, which calls on one stream share."""
    shape = q.shape
    ensure(shape == out.shape, "q and out must have the same shape")
    ws = ws or ctx.attention_workspace(cache)
    qh, oh = _heads(q, *cache._query), _heads(out, *cache._query)
    check(F.lib().rk_npu_hip_attention_q8_device_run(ws.raw, cache.handle.raw, ctypes.byref(qh), shape[1],
                                                     int32(position, "position"), ctypes.byref(oh),
                                                     _stream(stream, q)), "8-bit KV attention")


def _ints(t, name: str, shape) -> int:
    """The address of a cuda int32 tensor of this shape, its last dimension contiguous."""
    import torch
    if not (t.is_cuda and t.dtype == torch.int32 and tuple(t.shape) == tuple(shape) and
            (t.shape[-1] <= 1 or t.stride(-1) == 1)):
        raise NpuError(f"{name} is a cuda int32 tensor {list(shape)}, contiguous")
    return t.data_ptr()


class PagedBatch:
    """The sequences of a call on a KvPages (rk_npu_attention_paged.h), in cuda int32
    tensors that are read when the work runs: table [sequences][pages], the page of
    token t being table[s][t // page]; lengths [sequences], the call's rows among
    them; row_offsets [sequences + 1], sequence s having rows row_offsets[s] to
    row_offsets[s + 1], or None: row s. No sequence has more than max_rows rows or
    max_tokens tokens (default: what the table and the pages' capacity hold)."""

    def __init__(self, table, lengths, row_offsets=None, max_rows: int = 1, max_tokens: Optional[int] = None):
        ensure(len(table.shape) == 2 and len(lengths.shape) == 1, "a table is [sequences][pages], lengths [sequences]")
        n = lengths.shape[0]
        self._tensors = table, lengths, row_offsets
        self.sequences, self.max_rows, self.max_tokens = n, int32(max_rows, "max_rows"), max_tokens
        if max_tokens is not None:
            int32(max_tokens, "max_tokens")
        self._stride = int32(table.shape[1] if n <= 1 else table.stride(0), "the table's stride")
        ensure(n <= 1 or self._stride >= table.shape[1], "the table's rows overlap")
        self._columns = table.shape[1]
        self._at = (_ints(lengths, "lengths", (n,)),
                    None if row_offsets is None else _ints(row_offsets, "row_offsets", (n + 1,)),
                    _ints(table, "table", (n, self._columns)), self._stride)

    @property
    def table(self):
        return self._tensors[0]

    @property
    def lengths(self):
        return self._tensors[1]

    @property
    def row_offsets(self):
        return self._tensors[2]

    def _raw(self, rows: int, page: int, capacity: int = F.RK_NPU_HIP_PAGED_MAX_TOKENS) -> F.rk_npu_hip_paged_batch:
        most, tokens = self._columns * page, self.max_tokens
        if tokens is None:
            tokens = min(most, capacity)
        elif tokens > most:
            raise NpuError(f"the table holds {most} tokens a sequence, max_tokens is {tokens}")
        if rows >= 2 ** 31:
            int32(rows, "rows")
        return F.rk_npu_hip_paged_batch(self.sequences, rows, min(self.max_rows, rows), tokens, *self._at)


class KvPages:
    """A pool of `pages` pages of `page` tokens (16 to 256) of fp16 K and V for many
    sequences (rk_npu_attention_paged.h), none longer than `capacity` tokens (default:
    the pool's). append rotates the first rotary_dim dims of K and query rows by
    positions times rope_theta^(-2j / rotary_dim), or times frequencies[j] (a
    sequence of rotary_dim / 2 floats), pairs (j, j + rotary_dim / 2) or, interleaved,
    (2j, 2j + 1).

    Arrays are cuda tensors [heads][rows][head_dim], f16 or f32, any strides of
    heads and rows."""

    def __init__(self, ctx: DeviceContext, query_heads: int, kv_heads: int, head_dim: int, softmax_scale: float,
                 pages: int, page: int = 64, capacity: Optional[int] = None, causal: bool = True, rotary_dim: int = 0,
                 rope_theta: float = 10000.0, interleaved: bool = False, frequencies=None):
        capacity = min(pages * page, F.RK_NPU_HIP_PAGED_MAX_TOKENS) if capacity is None else capacity
        for name, value in (("query_heads", query_heads), ("kv_heads", kv_heads), ("head_dim", head_dim),
                            ("pages", pages), ("page", page), ("capacity", capacity), ("rotary_dim", rotary_dim)):
            int32(value, name)
        L = F.lib()
        cfg = F.rk_npu_hip_attention_paged_config()
        L.rk_npu_hip_attention_paged_config_init(ctypes.byref(cfg))
        a = cfg.attention
        a.query_heads, a.kv_heads, a.head_dim, a.softmax_scale = query_heads, kv_heads, head_dim, softmax_scale
        a.max_query_rows, a.max_capacity, a.initial_capacity = 1, capacity, 0
        a.mask_mode = F.RK_NPU_ATTENTION_F16_CAUSAL if causal else F.RK_NPU_ATTENTION_F16_NO_MASK
        cfg.page, cfg.pages, cfg.rotary_dim, cfg.interleaved, cfg.rope_theta = page, pages, rotary_dim, interleaved, rope_theta
        if frequencies is not None:
            frequencies = [float(f) for f in frequencies]
            ensure(2 * len(frequencies) == rotary_dim, "there are rotary_dim / 2 frequencies")
            if frequencies:
                cfg.frequencies = (ctypes.c_double * len(frequencies))(*frequencies)
        raw = ctypes.c_void_p()
        check(L.rk_npu_hip_attention_paged_pool_create(ctx.domain, ctypes.byref(cfg), ctypes.byref(raw)),
              "create the KV pages")
        self.handle = _Handle(raw.value, L.rk_npu_hip_attention_paged_pool_free, "KV pages", ctx.shared)
        self.ctx, self.config, self.page, self.capacity = ctx, cfg, page, capacity
        self._kv, self._query = (kv_heads, head_dim), (query_heads, head_dim)

    def bytes(self) -> int:
        sizes = F.rk_npu_attention_f16_sizes()
        check(F.lib().rk_npu_hip_attention_paged_query(ctypes.byref(self.config), ctypes.byref(sizes)), "KV pages' sizes")
        return sizes.key_bytes + sizes.value_bytes

    def check(self) -> None:
        """Waits for the calls made and raises where the device found a wrong length, offset or page since the last check."""
        check(F.lib().rk_npu_hip_attention_paged_status(self.handle.raw), "a length, row offset or page out of range")

    def append(self, batch: PagedBatch, k, v, q=None, q_out=None, positions=None, stream=None) -> None:
        """Puts the batch's rows k and v, [kv_heads][rows][head_dim], into their pages, k
        rotated, and the query rows q, rotated, into q_out (q itself, or another array).
        positions: cuda int32 [rows], by default the rows' tokens."""
        shape = k.shape
        rows = shape[1] if len(shape) == 3 else 0
        if shape != v.shape:
            raise NpuError("k and v must have the same shape")
        kh, vh = _heads(k, *self._kv), _heads(v, *self._kv)
        if (q is None) != (q_out is None):
            raise NpuError("q and q_out come together")
        qh = oh = at = None
        if q is not None:
            qh, oh = _heads(q, *self._query), _heads(q_out, *self._query)
            if q.shape[1] != rows or q_out.shape[1] != rows:
                raise NpuError("q, q_out and k must have the same rows")
        if positions is not None:
            at = _ints(positions, "positions", (rows,))
        check(F.lib().rk_npu_hip_attention_paged_append(self.handle.raw, batch._raw(rows, self.page, self.capacity), kh, vh, at, qh, oh,
                                                        _stream(stream, k)), "append to the KV pages")

    def read(self, batch: PagedBatch, k, v, stream=None) -> None:
        """The batch's rows as the pages hold them, into k and v, [kv_heads][rows][head_dim]."""
        shape = k.shape
        if shape != v.shape:
            raise NpuError("k and v must have the same shape")
        kh, vh = _heads(k, *self._kv), _heads(v, *self._kv)
        check(F.lib().rk_npu_hip_attention_paged_read(self.handle.raw, batch._raw(shape[1], self.page, self.capacity), kh, vh,
                                                      _stream(stream, k)), "read the KV pages")


def attention_paged(ctx: DeviceContext, pages: KvPages, batch: PagedBatch, q, out, ws=None, stream=None):
    """Attention of the batch's rows q [query_heads][rows][head_dim] over their
    sequences' pages. ws: the context's workspace of this geometry, which calls on
    one stream share."""
    shape = q.shape
    if shape != out.shape:
        raise NpuError("q and out must have the same shape")
    ws = ws or ctx.attention_workspace(pages)
    qh, oh = _heads(q, *pages._query), _heads(out, *pages._query)
    check(F.lib().rk_npu_hip_attention_paged_run(ws.raw, pages.handle.raw, batch._raw(shape[1], pages.page, pages.capacity), qh, oh,
                                                 _stream(stream, q)), "attention over the KV pages")


@contextlib.contextmanager
def plan_switch(name: str, value: int):
    """Sets one of the library's plan switches (rk_npu_hip_set_switch, e.g.
    HM_GEMM_VARIANT) for the body of the with-block, then restores it."""
    L = F.lib()
    prev = ctypes.c_int()
    check(L.rk_npu_hip_set_switch(name.encode(), int(value), ctypes.byref(prev)), f"set switch {name}")
    try:
        yield
    finally:
        check(L.rk_npu_hip_set_switch(name.encode(), prev.value, None), f"restore switch {name}")


class KernelProfile:
    """rk_npu_hip_profile_* as a context manager; .stats after exit."""

    def __init__(self, max_launches: int = 65536):
        self.max_launches = max_launches
        self.stats: List[dict] = []

    def __enter__(self):
        check(F.lib().rk_npu_hip_profile_begin(self.max_launches), "profile begin")
        return self

    def __exit__(self, *exc):
        L = F.lib()
        L.rk_npu_hip_profile_end()
        cap = 4096
        arr = (F.rk_npu_hip_kernel_stat * cap)()
        n = ctypes.c_int()
        check(L.rk_npu_hip_profile_read(arr, cap, ctypes.byref(n)), "profile read")
        self.stats = [dict(kind=s.kind, bits=s.bits, epilogue=s.epilogue, rows=s.rows, K=s.K, N=s.N,
                           launches=s.launches, total_ms=s.total_ms, name=s.name.decode())
                      for s in arr[:min(n.value, cap)]]
        return False
