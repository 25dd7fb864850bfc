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

    def attention_workspace(self, cache: "KvCacheQ8", own: bool = False) -> _Handle:
        """The context's attention workspace for the cache's geometry, created on
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
    int32(shape[1], "rows")
    return F.rk_npu_hip_heads(t.data_ptr(), _dtype_code(t), stride[0], stride[1])


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
