"""Direct-op front end: device tensors in, device tensors out, via the C ABI.

torch is used only as the allocator of device memory and as the source of the
current HIP stream; every computation runs in libgomlx_hip.so.

`stream` is a HIP stream's handle.  A call on one that is not torch's current stream orders
nothing: its inputs, and the outputs and workspace that the caller gives, must be ready there
(an event, a wait), and so must its outputs be before the current stream reads them.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import call

_DT = {
    torch.float32: _lib.DT_FLOAT32,
    torch.bfloat16: _lib.DT_BFLOAT16,
    torch.float16: _lib.DT_FLOAT16,
    torch.int32: _lib.DT_INT32,
    torch.int64: _lib.DT_INT64,
    torch.bool: _lib.DT_BOOL,
    torch.uint8: _lib.DT_UINT8,
    torch.int8: _lib.DT_INT8,
    torch.int16: _lib.DT_INT16,
}
for _name, _code in (("uint16", "DT_UINT16"), ("uint32", "DT_UINT32"), ("uint64", "DT_UINT64")):
    if hasattr(torch, _name) and hasattr(_lib, _code):
        _DT[getattr(torch, _name)] = getattr(_lib, _code)


def dtype_code(dt: torch.dtype) -> int:
    try:
        return _DT[dt]
    except KeyError:
        raise TypeError(f"gomlx_hip: unsupported dtype {dt}") from None


def _stream(stream=None) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return int(stream)


def _stream_of(handle, device):
    """torch's stream of a handle (ExternalStream takes 0 for a new stream)."""
    return torch.cuda.ExternalStream(int(handle), device=device) if int(handle) else torch.cuda.default_stream(device)


def _empty(shape, dtype, device, stream=None) -> torch.Tensor:
    """An output or a workspace of a call on `stream` (a handle; None: the current stream).
    torch reuses memory in the order of the stream that it was allocated on, so it comes
    from `stream`'s own: work still queued on the current stream for whoever had the memory
    before cannot meet the call.  Freed, it waits for the current stream's uses too."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(_stream_of(stream, device)):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(torch.cuda.current_stream(device))
    return t


def _empty_like(x: torch.Tensor, stream=None) -> torch.Tensor:
    """torch.empty_like as _empty."""
    if stream is None:
        return torch.empty_like(x)
    with torch.cuda.stream(_stream_of(stream, x.device)):
        t = torch.empty_like(x)
    t.record_stream(torch.cuda.current_stream(x.device))
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("gomlx_hip ops take device tensors")


def _rows(x: torch.Tensor):
    if not x.is_contiguous():
        raise ValueError("row kernels need a contiguous input")
    n = x.shape[-1] if x.dim() else 1
    return x.numel() // max(n, 1), n


def softmax(x: torch.Tensor, log: bool = False, out=None, stream=None) -> torch.Tensor:
    """Softmax (log-softmax) over the last axis."""
    _check_dev(x)
    rows, n = _rows(x)
    y = _empty_like(x, stream) if out is None else out
    call("ghip_softmax_rows", dtype_code(x.dtype), x.data_ptr(), y.data_ptr(), rows, n,
         int(log), _stream(stream))
    return y


def scale_mask_softmax(x: torch.Tensor, scale: float, causal: bool, bmask=None, out=None,
                       stream=None) -> torch.Tensor:
    """softmax(x * scale + mask) over the last axis of x [..., sq, sk]."""
    _check_dev(x, bmask)
    sq, sk = x.shape[-2], x.shape[-1]
    rows = x.numel() // sk
    y = _empty_like(x, stream) if out is None else out
    call("ghip_scale_mask_softmax_rows", dtype_code(x.dtype), x.data_ptr(), y.data_ptr(), rows,
         sq, sk, float(scale), int(causal), _ptr(bmask), _stream(stream))
    return y


def rmsnorm(x: torch.Tensor, gamma=None, eps: float = 1e-6, out=None, stream=None):
    _check_dev(x, gamma)
    rows, n = _rows(x)
    y = _empty_like(x, stream) if out is None else out
    call("ghip_rmsnorm_rows", dtype_code(x.dtype), x.data_ptr(), _ptr(gamma), y.data_ptr(),
         rows, n, float(eps), _stream(stream))
    return y


def layernorm(x: torch.Tensor, gamma=None, beta=None, eps: float = 1e-5, out=None, stream=None):
    _check_dev(x, gamma, beta)
    rows, n = _rows(x)
    y = _empty_like(x, stream) if out is None else out
    call("ghip_layernorm_rows", dtype_code(x.dtype), x.data_ptr(), _ptr(gamma), _ptr(beta),
         y.data_ptr(), rows, n, float(eps), _stream(stream))
    return y


def gemm_workspace(a_dtype, out_dtype, B: int, M: int, N: int, K: int, device, stream=None):
    """Workspace for ghip_gemm_batched_ws / ghip_gemm_grouped_ws (None when a
    product of these sizes never splits its contraction), for calls on `stream`."""
    n = _lib.load().ghip_gemm_workspace_bytes(dtype_code(a_dtype), dtype_code(out_dtype or a_dtype), B, M, N, K)
    return _empty((n,), torch.uint8, device, stream) if n > 0 else None


def gemm(a: torch.Tensor, b: torch.Tensor, out_dtype=None, out=None, stream=None, k_split: bool = True,
         workspace=None):
    """c[b] = a[b] @ b[b] for a [B,M,K] / [M,K], b [B,K,N] / [K,N]; any strides.
    k_split: with a workspace (`workspace`, or one allocated here), so few-tile
    products with a long contraction split it (ghip_gemm_batched_ws)."""
    _check_dev(a, b)
    squeeze = a.dim() == 2
    a3 = a.unsqueeze(0) if a.dim() == 2 else a
    b3 = b.unsqueeze(0) if b.dim() == 2 else b
    B, M, K = a3.shape
    B2, K2, N = b3.shape
    if K != K2 or (B2 != B and B2 != 1):
        raise ValueError(f"gemm: shapes {tuple(a.shape)} x {tuple(b.shape)}")
    odt = out_dtype or a.dtype
    c = _empty((B, M, N), odt, a.device, stream) if out is None else out.view(B, M, N)
    sb_b = b3.stride(0) if B2 == B else 0
    if k_split and workspace is None:
        workspace = gemm_workspace(a.dtype, odt, B, M, N, K, a.device, stream)
    ws_ptr = workspace.data_ptr() if (k_split and workspace is not None) else None
    ws_bytes = workspace.numel() * workspace.element_size() if ws_ptr is not None else 0
    call("ghip_gemm_batched_ws", dtype_code(a.dtype), dtype_code(odt), B, M, N, K,
         a3.data_ptr(), a3.stride(0), a3.stride(1), a3.stride(2),
         b3.data_ptr(), sb_b, b3.stride(1), b3.stride(2),
         c.data_ptr(), c.stride(0), c.stride(1), c.stride(2), ws_ptr, ws_bytes, _stream(stream))
    return c[0] if squeeze else c


def gemm_grouped(a: torch.Tensor, bs, out_dtype=None, outs=None, stream=None, k_split: bool = True,
                 workspace=None):
    """[a @ b for b in bs] in one call (ghip_gemm_grouped_ws): a [M,K], every b [K,N]
    with the same strides; returns the list of [M,N] results.  k_split as in gemm."""
    import ctypes
    _check_dev(a, *bs)
    M, K = a.shape
    K2, N = bs[0].shape
    if K != K2 or any(b.shape != bs[0].shape or b.stride() != bs[0].stride() for b in bs):
        raise ValueError("gemm_grouped: every b must be [K, N] with the same strides")
    odt = out_dtype or a.dtype
    cs = [_empty((M, N), odt, a.device, stream) for _ in bs] if outs is None else list(outs)
    if any(c.stride() != cs[0].stride() or c.stride(1) != 1 for c in cs):
        raise ValueError("gemm_grouped: outputs need one row stride and unit column stride")
    bp = (ctypes.c_void_p * len(bs))(*[b.data_ptr() for b in bs])
    cp = (ctypes.c_void_p * len(cs))(*[c.data_ptr() for c in cs])
    if k_split and workspace is None:
        workspace = gemm_workspace(a.dtype, odt, 1, M, N, K, a.device, stream)
    ws_ptr = workspace.data_ptr() if (k_split and workspace is not None) else None
    ws_bytes = workspace.numel() * workspace.element_size() if ws_ptr is not None else 0
    call("ghip_gemm_grouped_ws", dtype_code(a.dtype), dtype_code(odt), len(bs), M, N, K, a.data_ptr(),
         a.stride(0), a.stride(1), bp, bs[0].stride(0), bs[0].stride(1), cp, cs[0].stride(0), ws_ptr, ws_bytes,
         _stream(stream))
    return cs


def softmax_axis(x: torch.Tensor, axis: int, log: bool = False, out=None, stream=None) -> torch.Tensor:
    """Softmax (log-softmax) over a middle axis of a contiguous tensor (the column
    kernel: x read as [outer, n, inner])."""
    _check_dev(x)
    if not x.is_contiguous():
        raise ValueError("softmax_axis: contiguous input required")
    axis = axis % x.dim()
    outer = 1
    for d in x.shape[:axis]:
        outer *= d
    inner = 1
    for d in x.shape[axis + 1:]:
        inner *= d
    y = _empty_like(x, stream) if out is None else out
    call("ghip_softmax_cols", dtype_code(x.dtype), x.data_ptr(), y.data_ptr(), outer, x.shape[axis], inner,
         int(log), _stream(stream))
    return y


def copy(src: torch.Tensor, out: torch.Tensor, stream=None) -> torch.Tensor:
    """out[...] = src[...] for tensors of one shape and element size, any strides."""
    import ctypes
    _check_dev(src, out)
    if tuple(src.shape) != tuple(out.shape) or src.element_size() != out.element_size():
        raise ValueError(f"copy: {tuple(src.shape)} x{src.element_size()} -> {tuple(out.shape)} x{out.element_size()}")
    r = src.dim()
    arr = ctypes.c_int64 * max(r, 1)
    call("ghip_copy_strided", src.element_size(), src.data_ptr(), out.data_ptr(), r,
         arr(*src.shape), arr(*src.stride()), arr(*out.stride()), _stream(stream))
    return out


def _strides3(t: torch.Tensor):
    """(batch, head, sequence) element strides of a [B, H, S, D] view."""
    import ctypes
    if t.stride(3) != 1:
        raise ValueError("sdpa: the head dim must be contiguous")
    return (ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2))


def sdpa_workspace(q: torch.Tensor, Hkv: int, Sk: int, causal: bool, stream=None):
    """Workspace for ghip_sdpa_fwd_masked_ws (None when the shape takes no key split), for
    calls on `stream`."""
    B, H, Sq, D = q.shape
    n = _lib.load().ghip_sdpa_workspace_bytes(dtype_code(q.dtype), B, H, Hkv, Sq, Sk, D, int(causal))
    return _empty((n,), torch.uint8, q.device, stream) if n > 0 else None


def sdpa(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool,
         out=None, stream=None, kv_split: bool = True, workspace=None):
    """Fused attention: q [B,H,Sq,D], k / v [B,Hkv,Sk,D] (any strides with a contiguous
    head dim, e.g. BSHD storage viewed as BHSD) -> out [B,H,Sq,D].  kv_split: with a
    workspace (`workspace`, or one allocated here), so small grids split their key
    range (ghip_sdpa_fwd_masked_ws)."""
    return sdpa_masked(q, k, v, None, scale, causal, out=out, stream=stream, kv_split=kv_split,
                       workspace=workspace)


def _mask_strides(mask: torch.Tensor, B, H, Sq, Sk):
    """Element strides of `mask` broadcast to [B, H, Sq, Sk] over its trailing axes
    (0 on missing and size-1 axes)."""
    import ctypes
    st = [0, 0, 0, 0]
    off = 4 - mask.dim()
    for i in range(mask.dim()):
        if mask.shape[i] != 1:
            if mask.shape[i] != (B, H, Sq, Sk)[off + i]:
                raise ValueError(f"mask {tuple(mask.shape)} does not broadcast to {(B, H, Sq, Sk)}")
            st[off + i] = mask.stride(i)
    return (ctypes.c_int64 * 4)(*st)


def sdpa_masked(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask, scale: float, causal: bool,
                out=None, stream=None, kv_split: bool = True, workspace=None):
    """sdpa with a bool keep-mask or an additive mask (q's dtype) of any rank that
    broadcasts to the scores [B, H, Sq, Sk] (mask None: none)."""
    _check_dev(q, k, v, *([mask] if mask is not None else []))
    B, H, Sq, D = q.shape
    _, Hkv, Sk, _ = k.shape
    o = _empty((B, H, Sq, D), q.dtype, q.device, stream) if out is None else out
    mdt = -1 if mask is None else dtype_code(mask.dtype)
    ms = None if mask is None else _mask_strides(mask, B, H, Sq, Sk)
    ws = (workspace if workspace is not None else sdpa_workspace(q, Hkv, Sk, causal, stream)) if kv_split else None
    call("ghip_sdpa_fwd_masked_ws", dtype_code(q.dtype), q.data_ptr(), k.data_ptr(), v.data_ptr(),
         o.data_ptr(), B, H, Hkv, Sq, Sk, D, _strides3(q), _strides3(k), _strides3(v),
         _strides3(o), _ptr(mask), mdt, ms, float(scale), int(causal), _ptr(ws),
         0 if ws is None else ws.numel(), _stream(stream))
    return o


def scale_mask_softmax_ex(x: torch.Tensor, scale: float, causal: bool, mask=None, out=None, stream=None):
    """softmax(x * scale + mask) over the last axis of scores x [B, H, Sq, Sk]."""
    _check_dev(x, mask)
    B, H, Sq, Sk = x.shape
    y = _empty_like(x, stream) if out is None else out
    mdt = -1 if mask is None else dtype_code(mask.dtype)
    ms = None if mask is None else _mask_strides(mask, B, H, Sq, Sk)
    call("ghip_scale_mask_softmax_rows_ex", dtype_code(x.dtype), x.data_ptr(), y.data_ptr(), B, H, Sq, Sk,
         float(scale), int(causal), _ptr(mask), mdt, ms, _stream(stream))
    return y


def _launch(dev: torch.device, name: str, stream, *args):
    """Calls entry point `name` with `dev` current, on `stream` (None: dev's current one)."""
    n = dev.index
    if n != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            call(name, *args, _stream(stream))
    else:
        # The current stream's handle alone: a torch.cuda.Stream object costs 3 us.
        call(name, *args, torch._C._cuda_getCurrentRawStream(n) if stream is None else int(stream))


def _given(what: str, ws):
    """A caller's workspace: its bytes must lie one after the other."""
    if not ws.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous")
    return ws


def _one_device(first: torch.Tensor, *ts) -> torch.device:
    """The device that every tensor lies on."""
    dev = first.device
    if not first.is_cuda:
        raise ValueError("gomlx_hip ops take device tensors")
    n = dev.index
    for t in ts:
        if t is not None and t.get_device() != n:  # (-1: the host)
            raise ValueError(f"gomlx_hip: tensors on device {dev} and {t.device}")
    return dev


def _like(what: str, t: torch.Tensor, shape, dtype):
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)} where {dtype} {tuple(shape)} is needed")


def _ints(what: str, t, n: int):
    """A dense int32 [n] operand (None stays None)."""
    if t is not None and (t.dtype != torch.int32 or t.shape != (n,) or (n > 1 and t.stride(0) != 1)):
        _like(what, t, (n,), torch.int32)
        raise ValueError(f"{what}: must be contiguous")


_I3 = ctypes.c_int64 * 3


def _rows3(what: str, t: torch.Tensor):
    """The strides of a tensor's first three axes; the last one must be contiguous."""
    b, h, s, d = t.stride()
    if d != 1 and t.shape[3] != 1:
        raise ValueError(f"{what}: the head dim must be contiguous")
    return _I3(b, h, s)


def _window_shapes(q, k, v, q_start, lens):
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("sdpa_window: q [B, H, Sq, D] and k / v [B, Hkv, Sk, D] are needed")
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    _like("sdpa_window: k", k, (B, Hkv, Sk, D), q.dtype)
    _like("sdpa_window: v", v, (B, Hkv, Sk, D), q.dtype)
    _ints("sdpa_window: lens", lens, B)
    return (B, H, Hkv, Sq, Sk, D), Sk - Sq if q_start is None else int(q_start)


def sdpa_window(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                q_start=None, lens=None, with_lse: bool = False, out=None, lse=None, stream=None):
    """Causal attention over the last `window` keys (0: all) and the first `sinks` ones:
    q [B, H, Sq, D] at positions q_start.. (None: the last Sq of the Sk keys), k / v
    [B, Hkv, Sk, D], any strides with a contiguous head dim; lens: int32 [B], the
    sequences' lengths (queries past them: zeros).  Returns o [B, H, Sq, D], with_lse: (o,
    lse [B, H, Sq] float32), what sdpa_window_grad takes.  Wraps ghip_sdpa_window_fwd."""
    dev = _one_device(q, k, v, lens, out, lse)
    dims, start = _window_shapes(q, k, v, q_start, lens)
    B, H, _, Sq, _, D = dims
    if out is None:
        out = _empty((B, H, Sq, D), q.dtype, dev, stream)
    else:
        _like("sdpa_window: out", out, (B, H, Sq, D), q.dtype)
    if lse is not None:
        _like("sdpa_window: lse", lse, (B, H, Sq), torch.float32)
        if not lse.is_contiguous():
            raise ValueError("sdpa_window: lse must be contiguous")
    elif with_lse:
        lse = _empty((B, H, Sq), torch.float32, dev, stream)
    _launch(dev, "ghip_sdpa_window_fwd", stream, dtype_code(q.dtype), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            out.data_ptr(), _ptr(lse), *dims, _rows3("q", q), _rows3("k", k), _rows3("v", v), _rows3("out", out), start,
            int(window), int(sinks), _ptr(lens), float(scale))
    return (out, lse) if with_lse else out


def sdpa_window_grad_workspace(q: torch.Tensor, k: torch.Tensor, window: int = 0, sinks: int = 0, q_start=None,
                               stream=None):
    """Workspace for sdpa_window_grad at these sizes, for calls on `stream`."""
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    n = _lib.load().ghip_sdpa_window_bwd_workspace_bytes(dtype_code(q.dtype), B, H, Hkv, Sq, Sk, D,
                                                         Sk - Sq if q_start is None else int(q_start), int(window),
                                                         int(sinks))
    return _empty((n,), torch.uint8, q.device, stream)


def sdpa_window_grad(d_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                     lse: torch.Tensor, scale: float, window: int = 0, sinks: int = 0, q_start=None, lens=None,
                     outs=None, workspace=None, stream=None):
    """(dq, dk, dv) of sdpa_window from its inputs, its o and lse, and d_out, the gradient
    of o.  outs: the three tensors to write.  Wraps ghip_sdpa_window_bwd."""
    dev = _one_device(d_out, q, k, v, o, lse, lens, workspace, *(outs or ()))
    dims, start = _window_shapes(q, k, v, q_start, lens)
    B, H, Hkv, Sq, Sk, D = dims
    _like("sdpa_window_grad: o", o, q.shape, q.dtype)
    _like("sdpa_window_grad: d_out", d_out, q.shape, q.dtype)
    _like("sdpa_window_grad: lse", lse, (B, H, Sq), torch.float32)
    if not lse.is_contiguous():
        raise ValueError("sdpa_window_grad: lse must be contiguous")
    if outs is None:
        dq = _empty((B, H, Sq, D), q.dtype, dev, stream)
        dk = _empty((B, Hkv, Sk, D), q.dtype, dev, stream)
        dv = _empty((B, Hkv, Sk, D), q.dtype, dev, stream)
    else:
        dq, dk, dv = outs
        _like("sdpa_window_grad: dq", dq, q.shape, q.dtype)
        _like("sdpa_window_grad: dk", dk, k.shape, q.dtype)
        _like("sdpa_window_grad: dv", dv, k.shape, q.dtype)
    if workspace is None:
        ws = sdpa_window_grad_workspace(q, k, window, sinks, q_start, stream)
    else:
        ws = _given("sdpa_window_grad", workspace)
    _launch(dev, "ghip_sdpa_window_bwd", stream, dtype_code(q.dtype), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            o.data_ptr(), d_out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dims,
            _rows3("q", q), _rows3("k", k), _rows3("v", v), _rows3("o", o), _rows3("d_out", d_out), _rows3("dq", dq),
            _rows3("dk", dk), _rows3("dv", dv), start, int(window), int(sinks), _ptr(lens), float(scale), ws.data_ptr(),
            ws.numel() * ws.element_size())
    return dq, dk, dv


def _check_cache(what, k_cache, v_cache, block_table, B, Hkv, D, dtype):
    """(num_pages, page_size, max_pages, table stride) of caches viewed as [page, Hkv, token, D]."""
    shape = k_cache.shape
    if len(shape) != 4:
        raise ValueError(f"{what}: the caches are [pages, Hkv, page_size, D]")
    pages, heads, size, dim = shape
    if heads != Hkv or dim != D or k_cache.dtype != dtype:
        _like(f"{what}: k_cache", k_cache, (pages, Hkv, size, D), dtype)
    _like(f"{what}: v_cache", v_cache, shape, dtype)
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B:
        raise ValueError(f"{what}: block_table is int32 [{B}, pages of a sequence]")
    step, one = block_table.stride()
    per = block_table.shape[1]
    if per > 1 and one != 1:
        raise ValueError(f"{what}: a sequence's table entries must be contiguous")
    return pages, size, per, step


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              block_table: torch.Tensor, starts: torch.Tensor, counts=None, stream=None):
    """Writes k / v [B, Hkv, S, D] into the pages of k_cache / v_cache (viewed as [pages,
    Hkv, page_size, D], any strides with a contiguous head dim) as tokens starts[b] + i, i <
    counts[b] (None: S), of the sequences whose pages block_table [B, pages] names.  Wraps
    ghip_kv_append."""
    dev = _one_device(k, v, k_cache, v_cache, block_table, starts, counts)
    shape = k.shape
    if len(shape) != 4:
        raise ValueError("kv_append: k / v [B, Hkv, S, D] are needed")
    B, Hkv, S, D = shape
    _like("kv_append: v", v, shape, k.dtype)
    pages, size, per, ts = _check_cache("kv_append", k_cache, v_cache, block_table, B, Hkv, D, k.dtype)
    _ints("kv_append: starts", starts, B)
    _ints("kv_append: counts", counts, B)
    _launch(dev, "ghip_kv_append", stream, k.element_size(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), B, S, Hkv, D, pages, size, per, block_table.data_ptr(), ts, starts.data_ptr(),
            _ptr(counts), _rows3("k", k), _rows3("v", v), _rows3("k_cache", k_cache), _rows3("v_cache", v_cache))


def sdpa_paged_workspace(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, stream=None):
    """Workspace for sdpa_paged at these sizes (None when the sequences never split), for
    calls on `stream`."""
    B, H, D = q.shape
    n = _lib.load().ghip_sdpa_paged_workspace_bytes(dtype_code(q.dtype), B, H, k_cache.shape[1], D, k_cache.shape[2],
                                                    block_table.shape[1])
    return _empty((n,), torch.uint8, q.device, stream) if n > 0 else None


def sdpa_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
               lens: torch.Tensor, scale: float, window: int = 0, sinks: int = 0, out=None, stream=None,
               split: bool = True, workspace=None):
    """Attention of one new token a sequence, q [B, H, D] at position lens[b] - 1, over its
    pages (as kv_append wrote them), under sdpa_window's window and sinks.  split: with a
    workspace (`workspace`, or one allocated here), so the sequences' tokens are dealt out
    over the card.  Wraps ghip_sdpa_paged."""
    dev = _one_device(q, k_cache, v_cache, block_table, lens, out, workspace)
    if q.dim() != 3:
        raise ValueError("sdpa_paged: q [B, H, D] is needed")
    B, H, D = q.shape
    Hkv = k_cache.shape[1] if k_cache.dim() == 4 else 0
    pages, size, per, ts = _check_cache("sdpa_paged", k_cache, v_cache, block_table, B, Hkv, D, q.dtype)
    _ints("sdpa_paged: lens", lens, B)
    if out is None:
        out = _empty((B, H, D), q.dtype, dev, stream)
    else:
        _like("sdpa_paged: out", out, (B, H, D), q.dtype)
    for what, t in (("q", q), ("out", out)):
        if t.stride(2) != 1 and D != 1:
            raise ValueError(f"sdpa_paged: {what}'s head dim must be contiguous")
    ws = None
    if split and workspace is None:
        ws = sdpa_paged_workspace(q, k_cache, block_table, stream)
    elif split:
        ws = _given("sdpa_paged", workspace)
    _launch(dev, "ghip_sdpa_paged", stream, dtype_code(q.dtype), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
            out.data_ptr(), B, H, Hkv, D, pages, size, per, block_table.data_ptr(), ts, lens.data_ptr(),
            _I3(q.stride(0), q.stride(1)), _rows3("k_cache", k_cache), _rows3("v_cache", v_cache),
            _I3(out.stride(0), out.stride(1)), int(window), int(sinks), float(scale), _ptr(ws),
            0 if ws is None else ws.numel() * ws.element_size())
    return out


def _new(like: torch.Tensor, shape, stream, dtype=None) -> torch.Tensor:
    """_empty on the device (and of the type) of another tensor."""
    if stream is None:
        return like.new_empty(shape) if dtype is None else like.new_empty(shape, dtype=dtype)
    return _empty(shape, dtype or like.dtype, like.device, stream)


def _new_like(t: torch.Tensor, stream, dtype=None) -> torch.Tensor:
    """_new of another tensor's shape, contiguous (at two thirds of its cost)."""
    if stream is None:
        return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)
    return _empty(t.shape, dtype or t.dtype, t.device, stream)


def _rope(what: str, freqs, positions, sections, interleaved, B: int, S: int, D: int):
    """The GHipRope of a call on B sequences of S tokens (None: nothing is turned)."""
    if freqs is None:
        if positions is not None or sections is not None:
            raise ValueError(f"{what}: positions and sections go with freqs")
        return None
    if freqs.dtype != torch.float32 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise ValueError(f"{what}: freqs is a contiguous float32 vector, one value a pair")
    pairs, axes, at, step = freqs.shape[0], 1, None, (0, 0, 0)
    if positions is not None:
        if positions.dtype != torch.int32 or positions.dim() not in (2, 3) or positions.shape[-2:] != (B, S):
            raise ValueError(f"{what}: positions is int32 [{B}, {S}] or [axes, {B}, {S}]")
        at, step = positions.data_ptr(), positions.stride()
        if len(step) == 3:
            axes = positions.shape[0]
        else:
            step = (0, *step)
    if sections is None:
        sections = (pairs,)
    if len(sections) != axes or axes > 4:
        raise ValueError(f"{what}: {len(sections)} sections for {axes} axes of positions (1 to 4)")
    return _lib.Rope(at, *step, axes, *sections, *(0,) * (4 - axes), freqs.data_ptr(), 2 * pairs, interleaved)


def rope(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, sections=None, interleaved: bool = False,
         inverse: bool = False, out=None, stream=None) -> torch.Tensor:
    """Rotary positions: pair i of each row of x [B, H, S, D] (any strides with a contiguous head
    dim) turned by positions * freqs[i]; positions int32 [B, S], or [axes, B, S] with `sections`,
    the number of pairs that each axis turns.  freqs: float32 [rotary_dim / 2]; interleaved: pairs
    are neighbours, else half a rotary_dim apart.  inverse: turned back, the gradient of x from
    that of the output.  out may be x.  Wraps ghip_rope."""
    dev = _one_device(x, positions, freqs, out)
    if x.dim() != 4:
        raise ValueError("rope: x [B, H, S, D] is needed")
    B, H, S, D = x.shape
    if positions is None or freqs is None:
        raise ValueError("rope: positions and freqs are needed")
    r = _rope("rope", freqs, positions, sections, interleaved, B, S, D)
    if out is None:
        out = _new_like(x, stream)
    else:
        _like("rope: out", out, x.shape, x.dtype)
    _launch(dev, "ghip_rope", stream, dtype_code(x.dtype), x.data_ptr(), out.data_ptr(), B, H, S, D, _rows3("x", x),
            _rows3("out", out), r, inverse)
    return out


def _new_tokens(what, q, k, v, q_out, stream):
    """(B, H, Hkv, S, D), q_out and the strides of an append's operands."""
    if k.dim() != 4 or (q is not None and q.dim() != 4):
        raise ValueError(f"{what}: q [B, H, S, D] and k / v [B, Hkv, S, D] are needed")
    B, Hkv, S, D = k.shape
    _like(f"{what}: v", v, k.shape, k.dtype)
    if q is None:
        if q_out is not None:
            raise ValueError(f"{what}: q_out goes with q")
        return (B, 0, Hkv, S, D), None, (None, None, _rows3("k", k), _rows3("v", v))
    H = q.shape[1]
    _like(f"{what}: q", q, (B, H, S, D), k.dtype)
    if q_out is None:
        q_out = _new_like(q, stream)
    else:
        _like(f"{what}: q_out", q_out, q.shape, q.dtype)
    return (B, H, Hkv, S, D), q_out, (_rows3("q", q), _rows3("q_out", q_out), _rows3("k", k), _rows3("v", v))


def kv_append_rope(q, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, starts: torch.Tensor, freqs, counts=None, positions=None, sections=None,
                   interleaved: bool = False, q_out=None, stream=None):
    """kv_append with rotary positions on the way: k is turned as rope does and v copied into the
    pages, q [B, H, S, D] (None: none) is turned into q_out, which is returned (it may be q).
    positions None: token i of sequence b is at starts[b] + i; freqs None: nothing is turned.
    Wraps ghip_kv_append_rope."""
    what = "kv_append_rope"
    dev = _one_device(k, q, v, k_cache, v_cache, block_table, starts, freqs, counts, positions, q_out)
    (B, H, Hkv, S, D), q_out, steps = _new_tokens(what, q, k, v, q_out, stream)
    pages, size, per, ts = _check_cache(what, k_cache, v_cache, block_table, B, Hkv, D, k.dtype)
    _ints(f"{what}: starts", starts, B)
    _ints(f"{what}: counts", counts, B)
    r = _rope(what, freqs, positions, sections, interleaved, B, S, D)
    _launch(dev, "ghip_kv_append_rope", stream, dtype_code(k.dtype), _ptr(q), _ptr(q_out), k.data_ptr(), v.data_ptr(),
            k_cache.data_ptr(), v_cache.data_ptr(), B, H, Hkv, S, D, pages, size, per, block_table.data_ptr(), ts,
            starts.data_ptr(), _ptr(counts), *steps, _rows3("k_cache", k_cache), _rows3("v_cache", v_cache), r)
    return q_out


def kv4_cache(num_pages: int, page_size: int, Hkv: int, D: int, device="cuda"):
    """A paged cache's storage for keys (or values) in 4 bits: (codes [num_pages, Hkv, page_size,
    D / 2], scales [num_pages, Hkv, page_size, 4 ceil(D / 128)]), uint8, all zeros."""
    return (torch.zeros((num_pages, Hkv, page_size, D // 2), dtype=torch.uint8, device=device),
            torch.zeros((num_pages, Hkv, page_size, (D + 127) // 128 * 4), dtype=torch.uint8, device=device))


def _kv4(what, k_cache, v_cache, block_table, B, Hkv, D):
    """The two GHipKv4 of caches (codes, scales) viewed as [page, Hkv, token, ...], and
    (num_pages, page_size, max_pages, table stride)."""
    shape = k_cache[0].shape
    if len(shape) != 4 or shape[1] != Hkv or shape[3] * 2 != D:
        raise ValueError(f"{what}: codes are [pages, {Hkv}, page_size, {D // 2}]")
    pages, _, size, half = shape
    wide = pages, Hkv, size, (D + 127) // 128 * 4
    made = []
    for name, (codes, scales) in (("k_cache", k_cache), ("v_cache", v_cache)):
        if codes.shape != shape or scales.shape != wide or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            _like(f"{what}: {name}'s codes", codes, shape, torch.uint8)
            _like(f"{what}: {name}'s scales", scales, wide, torch.uint8)
        a, b, c, one = codes.stride()
        e, f, g, uno = scales.stride()
        if (one != 1 and half != 1) or uno != 1:
            raise ValueError(f"{what}: a row's codes and scales must be contiguous")
        made.append(_lib.Kv4(codes.data_ptr(), scales.data_ptr(), a, b, c, e, f, g))
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B:
        raise ValueError(f"{what}: block_table is int32 [{B}, pages of a sequence]")
    step, one = block_table.stride()
    per = block_table.shape[1]
    if per > 1 and one != 1:
        raise ValueError(f"{what}: a sequence's table entries must be contiguous")
    return made, (pages, size, per, step)


def kv4_append_rope(q, k: torch.Tensor, v: torch.Tensor, k_cache, v_cache, block_table: torch.Tensor,
                    starts: torch.Tensor, freqs, counts=None, positions=None, sections=None, interleaved: bool = False,
                    q_out=None, stream=None):
    """kv_append_rope into caches of 4 bits, (codes, scales) as kv4_cache makes them: E2M1 values
    and a power of two for each 32.  D: a multiple of 32.  Wraps ghip_kv4_append_rope."""
    what = "kv4_append_rope"
    dev = _one_device(k, q, v, *k_cache, *v_cache, block_table, starts, freqs, counts, positions, q_out)
    (B, H, Hkv, S, D), q_out, steps = _new_tokens(what, q, k, v, q_out, stream)
    (kc, vc), (pages, size, per, ts) = _kv4(what, k_cache, v_cache, block_table, B, Hkv, D)
    _ints(f"{what}: starts", starts, B)
    _ints(f"{what}: counts", counts, B)
    r = _rope(what, freqs, positions, sections, interleaved, B, S, D)
    _launch(dev, "ghip_kv4_append_rope", stream, dtype_code(k.dtype), _ptr(q), _ptr(q_out), k.data_ptr(), v.data_ptr(),
            kc, vc, B, H, Hkv, S, D, pages, size, per, block_table.data_ptr(), ts, starts.data_ptr(), _ptr(counts),
            *steps, r)
    return q_out


def kv4_read(k_cache, v_cache, block_table: torch.Tensor, tokens: int, lens=None, dtype=torch.bfloat16, outs=None,
             stream=None):
    """(k, v) [B, Hkv, tokens, D]: each sequence's first tokens out of caches of 4 bits, as the
    values they hold; zeros past lens[b] (int32 [B]; None: none) and on pages out of range.
    What sdpa_window takes for a later chunk of a prompt.  Wraps ghip_kv4_read."""
    what = "kv4_read"
    dev = _one_device(*k_cache, *v_cache, block_table, lens, *(outs or ()))
    B = block_table.shape[0]
    if k_cache[0].dim() != 4:
        raise ValueError(f"{what}: the caches are [pages, Hkv, page_size, ...]")
    Hkv, D = k_cache[0].shape[1], 2 * k_cache[0].shape[3]
    (kc, vc), (pages, size, per, ts) = _kv4(what, k_cache, v_cache, block_table, B, Hkv, D)
    _ints(f"{what}: lens", lens, B)
    shape = (B, Hkv, int(tokens), D)
    if outs is None:
        k = _new(k_cache[0], shape, stream, dtype)
        v = _new_like(k, stream)
    else:
        k, v = outs
        _like(f"{what}: k", k, shape, k.dtype)
        _like(f"{what}: v", v, shape, k.dtype)
    _launch(dev, "ghip_kv4_read", stream, dtype_code(k.dtype), kc, vc, k.data_ptr(), v.data_ptr(), B, Hkv, int(tokens),
            D, pages, size, per, block_table.data_ptr(), ts, _ptr(lens), _rows3("k", k), _rows3("v", v))
    return k, v


def sdpa_paged_kv4_workspace(q: torch.Tensor, k_cache, block_table: torch.Tensor, stream=None):
    """Workspace for sdpa_paged_kv4 at these sizes (None when the sequences never split), for
    calls on `stream`."""
    B, H, D = q.shape
    _, Hkv, size, _ = k_cache[0].shape
    n = _lib.load().ghip_sdpa_paged_kv4_workspace_bytes(B, H, Hkv, D, size, block_table.shape[1])
    return _new(q, (n,), stream, torch.uint8) if n > 0 else None


def sdpa_paged_kv4(q: torch.Tensor, k_cache, v_cache, block_table: torch.Tensor, lens: torch.Tensor, scale: float,
                   window: int = 0, sinks: int = 0, out=None, stream=None, split: bool = True, workspace=None):
    """sdpa_paged over caches of 4 bits, (codes, scales) each, as kv4_append_rope wrote them.
    Wraps ghip_sdpa_paged_kv4."""
    what = "sdpa_paged_kv4"
    dev = _one_device(q, *k_cache, *v_cache, block_table, lens, out, workspace)
    if q.dim() != 3:
        raise ValueError(f"{what}: q [B, H, D] is needed")
    B, H, D = q.shape
    Hkv = k_cache[0].shape[1] if k_cache[0].dim() == 4 else 0
    (kc, vc), (pages, size, per, ts) = _kv4(what, k_cache, v_cache, block_table, B, Hkv, D)
    _ints(f"{what}: lens", lens, B)
    if out is None:
        out = _new_like(q, stream)
    else:
        _like(f"{what}: out", out, (B, H, D), q.dtype)
    (qb, qh, qd), (ob, oh, od) = q.stride(), out.stride()
    if (qd != 1 or od != 1) and D != 1:
        raise ValueError(f"{what}: the head dim of q and out must be contiguous")
    ws = None
    if split and workspace is None:
        ws = sdpa_paged_kv4_workspace(q, k_cache, block_table, stream)
    elif split:
        ws = _given(what, workspace)
    _launch(dev, "ghip_sdpa_paged_kv4", stream, dtype_code(q.dtype), q.data_ptr(), kc, vc, out.data_ptr(), B, H, Hkv, D,
            pages, size, per, block_table.data_ptr(), ts, lens.data_ptr(), _I3(qb, qh), _I3(ob, oh), int(window), int(sinks),
            float(scale), _ptr(ws), 0 if ws is None else ws.numel() * ws.element_size())
    return out


def _logits(what: str, logits, ids):
    """The row stride of logits [N, V] beside ids [N]."""
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits [N, V] are needed")
    if logits.stride(1) != 1 and logits.shape[1] != 1:
        raise ValueError(f"{what}: a row's logits must be contiguous")
    _ints(f"{what}: ids", ids, logits.shape[0])
    return logits.stride(0)


def token_logprobs_workspace(logits: torch.Tensor, top: int = 0, stream=None):
    """Workspace for token_logprobs at these sizes (None where a row is never shared), for calls
    on `stream`."""
    n = _lib.load().ghip_token_logprobs_workspace_bytes(dtype_code(logits.dtype), *logits.shape, int(top))
    return _new(logits, (n,), stream, torch.uint8) if n > 0 else None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, top: int = 0, scale: float = 1.0, outs=None, stream=None,
                   split: bool = True, workspace=None):
    """(logp, entropy, lse, top_logps, top_ids) of rows of logits [N, V] times scale (1 /
    temperature): the log probability of each row's token ids [N] (int32; outside [0, V): 0),
    the entropy and the log-sum-exp of the row (float32 [N]), and the log probabilities and
    indices of the `top` largest logits, larger first, equal ones by index ([N, top]; None
    where top is 0).  outs: the five tensors to write.  split: with a workspace (`workspace`, or
    one allocated here), so few rows are shared out over the card.  Wraps ghip_token_logprobs."""
    what = "token_logprobs"
    dev = _one_device(logits, ids, workspace, *(outs or ()))
    step = _logits(what, logits, ids)
    N, V = logits.shape
    top = int(top)
    if outs is None:
        logp = _new_like(ids, stream, torch.float32)
        best = _new(logp, (N, top), stream) if top > 0 else None
        outs = (logp, _new_like(logp, stream), _new_like(logp, stream), best,
                None if best is None else _new_like(best, stream, torch.int32))
    else:
        outs = tuple(outs)
        for i, (t, shape) in enumerate(zip(outs, ((N,), (N,), (N,), (N, top), (N, top)), strict=True)):
            if t is None and (i < 3 or top > 0):
                raise ValueError(f"{what}: five outputs are needed (the last two may be None where top is 0)")
            if t is not None:
                _like(f"{what}: output {i}", t, shape, torch.int32 if i == 4 else torch.float32)
                if not t.is_contiguous():
                    raise ValueError(f"{what}: outputs must be contiguous")
    ws = None
    if split and workspace is None:
        ws = token_logprobs_workspace(logits, top, stream)
    elif split:
        ws = _given(what, workspace)
    _launch(dev, "ghip_token_logprobs", stream, dtype_code(logits.dtype), logits.data_ptr(), step, ids.data_ptr(), N, V, top,
            float(scale), outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), _ptr(outs[3]), _ptr(outs[4]), _ptr(ws),
            0 if ws is None else ws.numel() * ws.element_size())
    return outs


def token_logprobs_grad(logits: torch.Tensor, ids: torch.Tensor, lse: torch.Tensor, d_logp, entropy=None, d_entropy=None,
                        scale: float = 1.0, out=None, stream=None) -> torch.Tensor:
    """The gradient of logits from those of token_logprobs' logp and entropy (float32 [N]; one of
    them may be None), with the lse and, beside d_entropy, the entropy that it gave.  out may be
    logits.  Wraps ghip_token_logprobs_grad."""
    what = "token_logprobs_grad"
    dev = _one_device(logits, ids, lse, d_logp, entropy, d_entropy, out)
    step = _logits(what, logits, ids)
    N, V = logits.shape
    if lse is None or (d_logp is None and d_entropy is None) or (d_entropy is not None and entropy is None):
        raise ValueError(f"{what}: lse and d_logp or d_entropy (with entropy) are needed")
    for name, t in (("lse", lse), ("d_logp", d_logp), ("entropy", entropy), ("d_entropy", d_entropy)):
        if t is not None:
            _like(f"{what}: {name}", t, (N,), torch.float32)
            if not t.is_contiguous():
                raise ValueError(f"{what}: {name} must be contiguous")
    if out is None:
        out = _new_like(logits, stream)
    else:
        _like(f"{what}: out", out, (N, V), logits.dtype)
        if out.stride(1) != 1 and V != 1:
            raise ValueError(f"{what}: a row of out must be contiguous")
    _launch(dev, "ghip_token_logprobs_grad", stream, dtype_code(logits.dtype), logits.data_ptr(), step, ids.data_ptr(),
            lse.data_ptr(), _ptr(entropy), _ptr(d_logp), _ptr(d_entropy), N, V, float(scale), out.data_ptr(), out.stride(0))
    return out


def gather_rows(table: torch.Tensor, ids: torch.Tensor, out=None, stream=None):
    """out[i] = table[clamp(ids[i])] for an embedding table [V, ...]."""
    _check_dev(table, ids)
    if ids.dtype != torch.int32 or not ids.is_contiguous() or not table.is_contiguous():
        raise ValueError("gather_rows: contiguous table and int32 ids required")
    V = table.shape[0]
    row_bytes = table[0].numel() * table.element_size()
    o = _empty((ids.numel(),) + tuple(table.shape[1:]), table.dtype, table.device, stream) if out is None else out
    call("ghip_gather_rows", table.data_ptr(), V, row_bytes, ids.data_ptr(), ids.numel(),
         o.data_ptr(), _stream(stream))
    return o.view(tuple(ids.shape) + tuple(table.shape[1:])) if out is None else o


def argminmax(x: torch.Tensor, axis: int, is_min: bool = False, out_dtype=torch.int32,
              stream=None):
    _check_dev(x)
    if not x.is_contiguous():
        raise ValueError("argminmax: contiguous input required")
    ax = axis % x.dim()
    outer = 1
    for d in x.shape[:ax]:
        outer *= d
    inner = 1
    for d in x.shape[ax + 1:]:
        inner *= d
    o = _empty(tuple(x.shape[:ax]) + tuple(x.shape[ax + 1:]), out_dtype, x.device, stream)
    call("ghip_argminmax", dtype_code(x.dtype), x.data_ptr(), outer, x.shape[ax], inner,
         int(is_min), dtype_code(out_dtype), o.data_ptr(), _stream(stream))
    return o


def iota(shape, axis: int, dtype=torch.int32, device="cuda", stream=None):
    o = _empty(tuple(shape), dtype, device, stream)
    ax = axis % len(shape)
    outer = 1
    for d in shape[:ax]:
        outer *= d
    inner = 1
    for d in shape[ax + 1:]:
        inner *= d
    call("ghip_iota", dtype_code(dtype), o.data_ptr(), outer, shape[ax], inner, _stream(stream))
    return o
