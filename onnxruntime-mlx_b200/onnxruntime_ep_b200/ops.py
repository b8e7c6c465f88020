"""Kernel-level bindings: call the extern "C" entry points of include/b200ep.h on torch CUDA
tensors (torch provides device memory and the current stream; the arithmetic is the library's).

Each function validates shapes the way the reference's handlers do and raises B200EPError on a
non-zero status.  Nothing here falls back to another implementation.
"""

from __future__ import annotations

import ctypes

from . import check, load_library

DT = {"float32": 1, "float16": 10, "bfloat16": 16}


class GqaParams(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int64), ("seq", ctypes.c_int64), ("num_heads", ctypes.c_int64),
        ("kv_heads", ctypes.c_int64), ("head_size", ctypes.c_int64), ("cap", ctypes.c_int64),
        ("max_seq", ctypes.c_int64), ("rotary_half", ctypes.c_int64), ("do_rotary", ctypes.c_int32),
        ("interleaved", ctypes.c_int32), ("packed_qkv", ctypes.c_int32),
        ("local_window", ctypes.c_int32), ("scale", ctypes.c_float), ("qk_norm_eps", ctypes.c_float),
        ("bias_batch", ctypes.c_int64), ("bias_total", ctypes.c_int64),
    ]


class PagedParams(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32), ("num_tokens", ctypes.c_int32), ("num_heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32), ("head_size", ctypes.c_int32), ("num_blocks", ctypes.c_int32),
        ("block_size", ctypes.c_int32), ("max_blocks", ctypes.c_int32), ("max_seq", ctypes.c_int32),
        ("rotary_half", ctypes.c_int32), ("do_rotary", ctypes.c_int32), ("interleaved", ctypes.c_int32),
        ("scale", ctypes.c_float),
    ]


class PagedQ8Params(ctypes.Structure):
    _fields_ = [
        ("batch", ctypes.c_int32), ("num_tokens", ctypes.c_int32), ("num_heads", ctypes.c_int32),
        ("kv_heads", ctypes.c_int32), ("head_size", ctypes.c_int32), ("num_blocks", ctypes.c_int32),
        ("block_size", ctypes.c_int32), ("max_blocks", ctypes.c_int32), ("max_seq", ctypes.c_int32),
        ("rotary_half", ctypes.c_int32), ("do_rotary", ctypes.c_int32), ("interleaved", ctypes.c_int32),
        ("cache_type", ctypes.c_int32), ("scale", ctypes.c_float), ("query_stride", ctypes.c_int64),
        ("key_stride", ctypes.c_int64), ("value_stride", ctypes.c_int64),
    ]


_configured = False


_TYPE = {}   # torch dtype -> ONNX TensorProto code, of rows
_CACHE = {}  # ... and of 8-bit caches


def _lib():
    global _configured, torch
    L = load_library()
    if not _configured:
        import torch

        _TYPE.update({torch.float32: 1, torch.float16: 10, torch.bfloat16: 16})
        _CACHE.update({torch.int8: 3, torch.float8_e4m3fn: 17})
        vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float
        L.b200ep_matmulnbits.argtypes = [vp, vp, vp, vp, vp, i32, i64, i64, i64, i32, i32, vp]
        L.b200ep_matmulnbits_dequant.argtypes = [vp, vp, vp, vp, i32, i32, i64, i64, i32, i32, vp]
        L.b200ep_rms_norm.argtypes = [vp, vp, vp, i32, i64, i64, f32, vp]
        L.b200ep_skip_rms_norm.argtypes = [vp, vp, vp, vp, vp, i32, i64, i64, f32, vp]
        L.b200ep_gqa_workspace_size.argtypes = [ctypes.POINTER(GqaParams)]
        L.b200ep_gqa_workspace_size.restype = ctypes.c_size_t
        L.b200ep_group_query_attention.argtypes = (
            [ctypes.POINTER(GqaParams)] + [vp] * 12 + [i32, vp, ctypes.c_size_t, vp])
        L.b200ep_matmulnbits_prepack_size.argtypes = [i64, i64, i32, i32, ctypes.POINTER(ctypes.c_size_t)]
        L.b200ep_matmulnbits_prepack.argtypes = [vp, vp, vp, i32, i64, i64, i32, i32, vp, vp]
        L.b200ep_matmulnbits_prepacked.argtypes = [vp, vp, vp, i32, i64, i64, i64, i32, i32, vp]
        L.b200ep_device_error.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int), i32]
        L.b200ep_paged_attention.argtypes = [ctypes.POINTER(PagedParams)] + [vp] * 11 + [i32, vp]
        L.b200ep_gqa_sliding_workspace_size.argtypes = [ctypes.POINTER(GqaParams), i32]
        L.b200ep_gqa_sliding_workspace_size.restype = ctypes.c_size_t
        L.b200ep_group_query_attention_sliding.argtypes = (
            [ctypes.POINTER(GqaParams)] + [vp] * 11 + [i32, vp, ctypes.c_size_t, vp])
        q8 = ctypes.POINTER(PagedQ8Params)
        L.b200ep_paged_kv_quantize.argtypes = [q8] + [vp] * 11 + [i32, vp]
        L.b200ep_paged_kv_dequantize.argtypes = [q8] + [vp] * 8 + [i64, i32, vp]
        L.b200ep_paged_attention_quantized_workspace_size.argtypes = [q8]
        L.b200ep_paged_attention_quantized_workspace_size.restype = ctypes.c_size_t
        L.b200ep_paged_attention_quantized.argtypes = [q8] + [vp] * 13 + [i32, vp, ctypes.c_size_t, vp]
        L.b200ep_sample.argtypes = [vp] * 8 + [i64] * 4 + [i32, vp]
        _configured = True
    return L


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device=None):
    import torch

    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _dt(t) -> int:
    return DT[str(t.dtype).replace("torch.", "")]


def device_error(clear: bool = True) -> tuple[int, int]:
    code, detail = ctypes.c_int(0), ctypes.c_int(0)
    check(_lib().b200ep_device_error(ctypes.byref(code), ctypes.byref(detail), int(clear)))
    return code.value, detail.value


def matmulnbits(a, b, scales, zero_points=None, *, K, N, bits=4, block_size=32, out=None):
    """com.microsoft MatMulNBits: a [..., K] -> [..., N] (all float tensors share a dtype)."""
    import torch

    assert a.is_cuda and a.shape[-1] == K and a.is_contiguous()
    M = a.numel() // K
    if out is None:
        out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
    check(_lib().b200ep_matmulnbits(_p(a), _p(b), _p(scales), _p(zero_points), _p(out), _dt(a), M, N, K,
                                    bits, block_size, _stream(a.device)))
    return out


def matmulnbits_dequant(b, scales, zero_points=None, *, K, N, bits=4, block_size=32, out_dtype=None):
    import torch

    out_dtype = out_dtype or torch.float32
    w = torch.empty(N, K, dtype=out_dtype, device=b.device)
    check(_lib().b200ep_matmulnbits_dequant(_p(b), _p(scales), _p(zero_points), _p(w), _dt(scales),
                                            DT[str(out_dtype).replace("torch.", "")], N, K, bits,
                                            block_size, _stream(b.device)))
    return w


def matmulnbits_prepack(b, scales, zero_points=None, *, K, N, bits=4, block_size=32):
    """Repack ORT-layout int4 weights into tensor-core group records; returns the device buffer."""
    import torch

    size = ctypes.c_size_t(0)
    check(_lib().b200ep_matmulnbits_prepack_size(N, K, bits, block_size, ctypes.byref(size)))
    packed = torch.empty(int(size.value), dtype=torch.uint8, device=b.device)
    check(_lib().b200ep_matmulnbits_prepack(_p(b), _p(scales), _p(zero_points), _dt(scales), N, K, bits, block_size,
                                            _p(packed), _stream(b.device)))
    return packed


def matmulnbits_prepacked(a, packed, *, K, N, bits=4, block_size=32, out=None):
    import torch

    M = a.numel() // K
    if out is None:
        out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
    check(_lib().b200ep_matmulnbits_prepacked(_p(a), _p(packed), _p(out), _dt(a), M, N, K, bits, block_size,
                                              _stream(a.device)))
    return out


def rms_norm(x, gamma, eps, out=None):
    import torch

    hidden = x.shape[-1]
    out = torch.empty_like(x) if out is None else out
    check(_lib().b200ep_rms_norm(_p(x), _p(gamma), _p(out), _dt(x), x.numel() // hidden, hidden, eps,
                                 _stream(x.device)))
    return out


def skip_rms_norm(x, skip, gamma, eps, *, residual=True):
    import torch

    hidden = x.shape[-1]
    y = torch.empty_like(x)
    r = torch.empty_like(x) if residual else None
    check(_lib().b200ep_skip_rms_norm(_p(x), _p(skip), _p(gamma), _p(y), _p(r), _dt(x), x.numel() // hidden,
                                      hidden, eps, _stream(x.device)))
    return y, r


def gqa_params(*, batch, seq, num_heads, kv_heads, head_size, cap, cos_cache=None, do_rotary=1,
               interleaved=0, packed_qkv=0, local_window=-1, scale=0.0, qk_norm_eps=1e-6,
               attention_bias=None) -> GqaParams:
    p = GqaParams()
    p.batch, p.seq, p.num_heads, p.kv_heads, p.head_size, p.cap = batch, seq, num_heads, kv_heads, head_size, cap
    p.max_seq = 0 if cos_cache is None else cos_cache.shape[0]
    p.rotary_half = 0 if cos_cache is None else cos_cache.shape[1]
    p.do_rotary = int(bool(do_rotary) and cos_cache is not None)
    p.interleaved, p.packed_qkv, p.local_window = int(interleaved), int(packed_qkv), int(local_window)
    p.scale, p.qk_norm_eps = float(scale), float(qk_norm_eps)
    if attention_bias is not None:
        p.bias_batch, p.bias_total = attention_bias.shape[0], attention_bias.shape[-1]
    return p


def group_query_attention(query, key, value, kv_key, kv_value, seqlens_k, cos_cache=None, sin_cache=None,
                          *, num_heads, kv_heads, scale=0.0, do_rotary=1, interleaved=0, local_window=-1,
                          q_norm=None, k_norm=None, qk_norm_eps=1e-6, attention_bias=None, out=None,
                          workspace=None):
    """GroupQueryAttention over the shared KV buffers kv_key/kv_value [B, HK, cap, D] (in place)."""
    import torch

    packed = key is None
    B, S, W = query.shape
    D = W // (num_heads + 2 * kv_heads) if packed else W // num_heads
    p = gqa_params(batch=B, seq=S, num_heads=num_heads, kv_heads=kv_heads, head_size=D, cap=kv_key.shape[2],
                   cos_cache=cos_cache, do_rotary=do_rotary, interleaved=interleaved, packed_qkv=packed,
                   local_window=local_window, scale=scale, qk_norm_eps=qk_norm_eps,
                   attention_bias=attention_bias)
    if out is None:
        out = torch.empty(B, S, num_heads * D, dtype=query.dtype, device=query.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(_lib().b200ep_group_query_attention(
        ctypes.byref(p), _p(query), _p(key), _p(value), _p(kv_key), _p(kv_value), _p(seqlens_k),
        _p(cos_cache), _p(sin_cache), _p(q_norm), _p(k_norm), _p(attention_bias), _p(out), _dt(query),
        _p(workspace), ws_bytes, _stream(query.device)))
    return out


def group_query_attention_sliding(query, key, value, past_key, past_value, seqlens_k, cos_cache=None,
                                  sin_cache=None, *, num_heads, kv_heads, local_window, scale=0.0, do_rotary=1,
                                  interleaved=0, present_key=None, present_value=None, out=None):
    """GroupQueryAttention with sliding_window_cache = 1: returns (out, present_key, present_value);
    present defaults to the past buffers (updated in place)."""
    import torch

    packed = key is None
    B, S, W = query.shape
    D = W // (num_heads + 2 * kv_heads) if packed else W // num_heads
    p = gqa_params(batch=B, seq=S, num_heads=num_heads, kv_heads=kv_heads, head_size=D, cap=past_key.shape[2],
                   cos_cache=cos_cache, do_rotary=do_rotary, interleaved=interleaved, packed_qkv=packed,
                   local_window=local_window, scale=scale)
    present_key = past_key if present_key is None else present_key
    present_value = past_value if present_value is None else present_value
    if out is None:
        out = torch.empty(B, S, num_heads * D, dtype=query.dtype, device=query.device)
    check(_lib().b200ep_group_query_attention_sliding(
        ctypes.byref(p), _p(query), _p(key), _p(value), _p(past_key), _p(past_value), _p(present_key),
        _p(present_value), _p(seqlens_k), _p(cos_cache), _p(sin_cache), _p(out), _dt(query), None, 0,
        _stream(query.device)))
    return out, present_key, present_value


def gqa_workspace_size(**kw) -> int:
    return int(_lib().b200ep_gqa_workspace_size(ctypes.byref(gqa_params(**kw))))


def paged_attention(query, key, value, key_cache, value_cache, cumulative_seqlens, past_seqlens, block_table,
                    cos_cache=None, sin_cache=None, *, num_heads, kv_heads, scale=0.0, interleaved=0, out=None):
    """com.microsoft PagedAttention: packed rows [num_tokens, H*D]; caches [num_blocks, block_size, HK, D]
    updated in place; control tensors int32 on the device."""
    import torch

    T, W = query.shape
    D = W // num_heads
    batch = cumulative_seqlens.numel() - 1
    p = PagedParams()
    p.batch, p.num_tokens, p.num_heads, p.kv_heads, p.head_size = batch, T, num_heads, kv_heads, D
    p.num_blocks, p.block_size = key_cache.shape[0], key_cache.shape[1]
    p.max_blocks = block_table.numel() // batch
    p.do_rotary = int(cos_cache is not None)
    p.max_seq = 0 if cos_cache is None else cos_cache.shape[0]
    p.rotary_half = 0 if cos_cache is None else cos_cache.shape[1]
    p.interleaved, p.scale = int(interleaved), float(scale)
    if out is None:
        out = torch.empty(T, num_heads * D, dtype=query.dtype, device=query.device)
    check(_lib().b200ep_paged_attention(
        ctypes.byref(p), _p(query), _p(key), _p(value), _p(key_cache), _p(value_cache), _p(cumulative_seqlens),
        _p(past_seqlens), _p(block_table), _p(cos_cache), _p(sin_cache), _p(out), _dt(query),
        _stream(query.device)))
    return out


# The bindings of the 8-bit cache and of sampling run once per decode step and layer: they check with few
# attribute reads, hand addresses to ctypes as integers, and keep the parameter structs of geometries seen.
_q8_structs = {}


def _q8_fail(what):
    raise ValueError("paged 8-bit cache: " + what)


def _q8_cache(key_cache, value_cache, key_scales, value_scales, block_table, batch):
    """Checks the cache's tensors the way the kernels rely on them; returns the pages' shape."""
    shape, dtype = key_cache.shape, key_cache.dtype
    if dtype not in _CACHE or value_cache.dtype != dtype:
        _q8_fail("key_cache and value_cache must both be int8 or float8_e4m3fn")
    if len(shape) != 4 or value_cache.shape != shape:
        _q8_fail("caches must be [num_blocks, kv_heads, block_size, head_size]")
    rows = shape[:3]
    if key_scales.shape != rows or value_scales.shape != rows or key_scales.dtype != torch.float32 or (
            value_scales.dtype != torch.float32):
        _q8_fail("scales must be float32 [num_blocks, kv_heads, block_size]")
    if not (key_cache.is_contiguous() and value_cache.is_contiguous() and key_scales.is_contiguous()
            and value_scales.is_contiguous()):
        _q8_fail("caches and scales must be contiguous")
    if block_table.dtype != torch.int32 or not block_table.is_contiguous() or batch and (
            block_table.numel() % batch or block_table.dim() > 1 and block_table.shape[0] != batch):
        _q8_fail("block_table must be a contiguous int32 [batch, max_blocks]")
    return shape


def _q8_rows(name, x, width, dtype, tokens):
    """Packed rows [T, width]; the rows may be slices of wider ones.  Returns the row stride."""
    if x.shape != (tokens, width):
        _q8_fail(f"{name} must be [{tokens}, {width}]")
    if x.dtype != dtype:
        _q8_fail(f"{name} must be {dtype}")
    row, one = x.stride()
    if one != 1 or tokens > 1 and row < width:
        _q8_fail(f"the elements of a row of {name} must be contiguous")
    return row if tokens > 1 else width


def _q8_control(cumulative_seqlens, past_seqlens, cos_cache, sin_cache, dtype):
    """Checks lengths and angles; returns (sequences, rows and columns of the cos / sin caches)."""
    batch = past_seqlens.numel()
    if cumulative_seqlens.dtype != torch.int32 or not cumulative_seqlens.is_contiguous():
        _q8_fail("cumulative_seqlens must be contiguous int32")
    if past_seqlens.dtype != torch.int32 or not past_seqlens.is_contiguous():
        _q8_fail("past_seqlens must be contiguous int32")
    if cumulative_seqlens.numel() != batch + 1:
        _q8_fail("cumulative_seqlens must have one entry more than past_seqlens")
    if cos_cache is None or sin_cache is None:
        if cos_cache is not sin_cache:
            _q8_fail("cos_cache and sin_cache come together")
        return batch, 0, 0
    shape = cos_cache.shape
    if cos_cache.dtype != dtype or sin_cache.dtype != dtype or len(shape) != 2 or sin_cache.shape != shape or not (
            cos_cache.is_contiguous() and sin_cache.is_contiguous()):
        _q8_fail("cos / sin must be contiguous [max_seq, rotary_half] of the rows' type")
    return batch, shape[0], shape[1]


def _q8_struct(batch, tokens, heads, pages, cache_type, max_blocks, max_seq, half, interleaved, scale, strides):
    key = (batch, tokens, heads, pages, cache_type, max_blocks, max_seq, half, interleaved, scale, strides)
    ref = _q8_structs.get(key)
    if ref is None:
        if len(_q8_structs) >= 4096:  # (every batch size and prompt length is a geometry)
            _q8_structs.clear()
        blocks, kv_heads, block, head = pages
        ref = _q8_structs[key] = ctypes.byref(PagedQ8Params(
            batch, tokens, heads, kv_heads, head, blocks, block, max_blocks, max_seq, half, int(half > 0),
            int(interleaved), cache_type, scale, *strides))
    return ref


def _device(*tensors):
    """The CUDA device that all of the tensors (None: one that was not given) are on."""
    at = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != at or at < 0:
            raise ValueError("the tensors must be on one CUDA device")
    return at


def _raw_stream(device):
    return torch._C._cuda_getCurrentRawStream(device)


def _current_device():
    return torch._C._cuda_getDevice()


def _launch(device, entry, *args):
    """Calls an entry point on the device's current stream (its last argument).  It launches on the current device, so
    the tensors' is made that one."""
    if _current_device() == device:
        check(entry(*args, _raw_stream(device)))
    else:
        with torch.cuda.device(device):
            check(entry(*args, _raw_stream(device)))


def paged_kv_quantize(key, value, key_cache, value_cache, key_scales, value_scales, cumulative_seqlens,
                      past_seqlens, block_table, cos_cache=None, sin_cache=None, *, interleaved=0):
    """Write packed key / value rows [T, kv_heads * D] (the key after RoPE) into 8-bit pages, in place:
    codes [num_blocks, kv_heads, block_size, D] int8 or float8_e4m3fn, scales float32
    [num_blocks, kv_heads, block_size].  Rows may be slices of a packed projection."""
    L = _lib()
    dtype = key.dtype
    batch, max_seq, half = _q8_control(cumulative_seqlens, past_seqlens, cos_cache, sin_cache, dtype)
    pages = _q8_cache(key_cache, value_cache, key_scales, value_scales, block_table, batch)
    T, width = key.shape[0], pages[1] * pages[3]
    strides = (0, _q8_rows("key", key, width, dtype, T), _q8_rows("value", value, width, dtype, T))
    p = _q8_struct(batch, T, 0, pages, _CACHE[key_cache.dtype], block_table.numel() // batch if batch else 1, max_seq,
                   half, interleaved, 0.0, strides)
    device = _device(key, value, key_cache, value_cache, key_scales, value_scales, cumulative_seqlens, past_seqlens,
                     block_table, cos_cache, sin_cache)
    _launch(
        device, L.b200ep_paged_kv_quantize, p, key.data_ptr(), value.data_ptr(), key_cache.data_ptr(),
        value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), cumulative_seqlens.data_ptr(),
        past_seqlens.data_ptr(), block_table.data_ptr(), half and cos_cache.data_ptr(), half and sin_cache.data_ptr(),
        _TYPE.get(dtype, 0))


def paged_kv_dequantize(key_cache, value_cache, key_scales, value_scales, seqlens, block_table, *, cap=None,
                        dtype=None, key=None, value=None):
    """Read the first seqlens[b] positions of each sequence out of 8-bit pages: (key, value), each
    [B, kv_heads, cap, D] of ``dtype`` with zeros from seqlens[b] on — GroupQueryAttention's shared-buffer
    layout.  ``cap`` and ``dtype`` are taken from ``key`` / ``value`` when those are given."""
    L = _lib()
    if seqlens.dtype != torch.int32 or not seqlens.is_contiguous():
        _q8_fail("seqlens must be contiguous int32")
    B = seqlens.numel()
    pages = _q8_cache(key_cache, value_cache, key_scales, value_scales, block_table, B)
    if key is None and value is None:
        if cap is None:
            _q8_fail("cap is needed when no output is given")
        shape = (B, pages[1], cap, pages[3])
        device = _device(key_cache, value_cache, key_scales, value_scales, seqlens, block_table)
        key = torch.empty(shape, dtype=dtype or torch.float16, device=key_cache.device)
        value = torch.empty_like(key)
    else:
        if key is None or value is None:
            _q8_fail("key and value come together")
        cap = key.shape[2] if key.dim() == 4 else -1
        if key.shape != (B, pages[1], cap, pages[3]) or value.shape != key.shape or (
                value.dtype != key.dtype) or not (key.is_contiguous() and value.is_contiguous()):
            _q8_fail("outputs must be contiguous [B, kv_heads, cap, D] of one type")
        device = _device(key_cache, value_cache, key_scales, value_scales, seqlens, block_table, key, value)
    p = _q8_struct(B, 0, 0, pages, _CACHE[key_cache.dtype], block_table.numel() // B if B else 1, 0, 0, 0, 0.0,
                   (0, 0, 0))
    _launch(
        device, L.b200ep_paged_kv_dequantize, p, key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(),
        value_scales.data_ptr(), seqlens.data_ptr(), block_table.data_ptr(), key.data_ptr(), value.data_ptr(), cap,
        _TYPE.get(key.dtype, 0))
    return key, value


def paged_attention_quantized_workspace_size(*, num_heads, kv_heads, head_size) -> int:
    p = PagedQ8Params()
    p.num_heads, p.kv_heads, p.head_size = num_heads, kv_heads, head_size
    return int(_lib().b200ep_paged_attention_quantized_workspace_size(ctypes.byref(p)))


def paged_attention_quantized(query, key, value, key_cache, value_cache, key_scales, value_scales,
                              cumulative_seqlens, past_seqlens, block_table, cos_cache=None, sin_cache=None, *,
                              num_heads, kv_heads, scale=0.0, interleaved=0, out=None, workspace=None):
    """PagedAttention over 8-bit pages (see paged_kv_quantize): packed query rows [T, num_heads * D], RoPE'd
    here, each attending to its sequence's positions up to its own.  ``key`` / ``value`` (both or neither)
    are first written into the pages.  ``workspace``: a uint8 tensor of at least
    paged_attention_quantized_workspace_size bytes, any contents; allocated on the current stream when
    absent."""
    L = _lib()
    dtype = query.dtype
    batch, max_seq, half = _q8_control(cumulative_seqlens, past_seqlens, cos_cache, sin_cache, dtype)
    pages = _q8_cache(key_cache, value_cache, key_scales, value_scales, block_table, batch)
    if pages[1] != kv_heads:
        _q8_fail(f"the cache holds {pages[1]} kv heads, not {kv_heads}")
    T, D = query.shape[0], pages[3]
    strides = _q8_rows("query", query, num_heads * D, dtype, T)
    if key is None and value is None:
        strides = (strides, 0, 0)
    else:
        if key is None or value is None:
            _q8_fail("key and value come together, or neither")
        strides = (strides, _q8_rows("key", key, kv_heads * D, dtype, T),
                   _q8_rows("value", value, kv_heads * D, dtype, T))
    device = _device(query, key_cache, value_cache, key_scales, value_scales, cumulative_seqlens, past_seqlens,
                     block_table, key, value, cos_cache, sin_cache, out, workspace)
    if out is None:
        out = torch.empty((T, num_heads * D), dtype=dtype, device=query.device)
    elif out.shape != (T, num_heads * D) or out.dtype != dtype or not out.is_contiguous():
        _q8_fail("out must be contiguous [T, num_heads * D] of the query's type")
    p = _q8_struct(batch, T, num_heads, pages, _CACHE[key_cache.dtype], block_table.numel() // batch if batch else 1,
                   max_seq, half, interleaved, scale, strides)
    if workspace is None:
        workspace = torch.empty(L.b200ep_paged_attention_quantized_workspace_size(p), dtype=torch.uint8,
                                device=query.device)
    elif not workspace.is_contiguous():
        _q8_fail("workspace must be contiguous")
    _launch(
        device, L.b200ep_paged_attention_quantized, p, query.data_ptr(), key if key is None else key.data_ptr(),
        value if value is None else value.data_ptr(),
        key_cache.data_ptr(), value_cache.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
        cumulative_seqlens.data_ptr(), past_seqlens.data_ptr(), block_table.data_ptr(),
        half and cos_cache.data_ptr(), half and sin_cache.data_ptr(), out.data_ptr(), _TYPE.get(dtype, 0),
        workspace.data_ptr(), workspace.nbytes)
    return out


def _per_row(name, x, dtype, B):
    if x is None:
        return None
    if x.dtype != dtype or x.shape != (B,) or not x.is_contiguous():
        raise ValueError(f"sample: {name} must be contiguous {dtype} [{B}]")
    return x.data_ptr()


def sample(logits, noise, temperature=None, top_k=None, top_p=None, min_p=None, *, tokens=None, logprobs=None):
    """Draw one token per row of ``logits`` [B, V]: (tokens int64 [B], logprobs float32 [B]).  ``noise``: float32
    [B, V] of standard exponential numbers (``torch.empty(B, V).exponential_()``).  ``temperature`` (0: the largest
    logit), ``top_k`` int32 (<= 0: all), ``top_p`` (>= 1: all) and ``min_p`` (<= 0: all) are [B] or None.  Rows may
    be slices of wider ones.  tokens is -1 where every logit is -inf or NaN."""
    L = _lib()
    shape = logits.shape
    if len(shape) != 2 or noise.shape != shape:
        raise ValueError("sample: logits and noise must both be [B, V]")
    if noise.dtype != torch.float32:
        raise ValueError("sample: noise must be float32")
    B, V = shape
    (lr, lc), (nr, nc) = logits.stride(), noise.stride()
    if V > 1 and (lc != 1 or nc != 1) or B > 1 and (lr < V or nr < V):
        raise ValueError("sample: the elements of a row of logits and of noise must be contiguous")
    f32 = torch.float32
    args = (_per_row("temperature", temperature, f32, B), _per_row("top_k", top_k, torch.int32, B),
            _per_row("top_p", top_p, f32, B), _per_row("min_p", min_p, f32, B))
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.numel() != B or not tokens.is_contiguous()):
        raise ValueError(f"sample: tokens must be contiguous int64 with {B} entries")
    if logprobs is not None and (logprobs.dtype != f32 or logprobs.shape != (B,) or not logprobs.is_contiguous()):
        raise ValueError(f"sample: logprobs must be contiguous float32 [{B}]")
    device = _device(logits, noise, temperature, top_k, top_p, min_p, tokens, logprobs)
    if tokens is None:
        tokens = torch.empty(B, dtype=torch.int64, device=logits.device)
    if logprobs is None:
        logprobs = torch.empty(B, dtype=f32, device=logits.device)
    _launch(device, L.b200ep_sample, logits.data_ptr(), noise.data_ptr(), *args, tokens.data_ptr(), logprobs.data_ptr(),
            B, V, lr if B > 1 else 0, nr if B > 1 else 0, _TYPE.get(logits.dtype, 0))
    return tokens, logprobs
