"""Operator API with the factory shape of the reference's TileLang kernels
(soraku_inference/acceleration/tilelang_kernels.py:34-254): ``factory(*shape)``
returns ``kernel(*inputs) -> out`` with the output allocated
(``out_idx=[-1]``).  Inputs are contiguous torch tensors on the HIP device;
matrices may be float32 or bfloat16 (FP32 accumulation).  Masking writes -inf
as the native path does (model.py:582-584), not -1e30 (tilelang_kernels.py:31).
"""

from __future__ import annotations

import ctypes as C
import functools
import operator

from . import _lib
from ._lib import check, lib


def _ptr(t) -> C.c_void_p:
    if not t.is_cuda:
        raise ValueError("operands must live on the HIP device")
    if not t.is_contiguous():
        raise ValueError("operands must be contiguous (fast_generate.py:94-97)")
    return C.c_void_p(t.data_ptr())


def _stream(t) -> C.c_void_p:
    import torch

    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _wdtype(t) -> int:
    import torch

    if t.dtype == torch.float32:
        return _lib.SK_F32
    if t.dtype == torch.bfloat16:
        return _lib.SK_BF16
    raise ValueError(f"matrix dtype {t.dtype} not supported (float32 or bfloat16)")


def _empty(ref, *shape):
    import torch

    return torch.empty(*shape, device=ref.device, dtype=torch.float32)


def add_rmsnorm(B: int, D: int, eps: float):
    """out = rmsnorm(hidden + prefix) * w (tilelang_kernels.py:34-55)."""
    def kernel(hidden, prefix, weight):
        out = _empty(hidden, B, D)
        check(lib().sk_op_add_rmsnorm(_stream(hidden), B, D, eps, _ptr(hidden), _ptr(prefix),
                                      _ptr(weight), _ptr(out)))
        return out
    return kernel


def rmsnorm(B: int, D: int, eps: float):
    """tilelang_kernels.py:58-78."""
    def kernel(x, weight):
        out = _empty(x, B, D)
        check(lib().sk_op_rmsnorm(_stream(x), B, D, eps, _ptr(x), _ptr(weight), _ptr(out)))
        return out
    return kernel


def swiglu_gemv(B: int, I: int, D: int):
    """act = silu(x Wg^T) * (x Wu^T) (tilelang_kernels.py:81-112)."""
    def kernel(x, wg, wu):
        if wg.dtype != wu.dtype:
            raise ValueError("gate and up must share a dtype")
        out = _empty(x, B, I)
        check(lib().sk_op_swiglu_gemv(_stream(x), B, I, D, _wdtype(wg), _ptr(x), _ptr(wg), _ptr(wu),
                                      _ptr(out)))
        return out
    return kernel


def down_residual_gemv(B: int, D: int, I: int):
    """y = act Wd^T + residual (tilelang_kernels.py:115-143)."""
    def kernel(act, wd, residual):
        out = _empty(act, B, D)
        check(lib().sk_op_down_residual_gemv(_stream(act), B, D, I, _wdtype(wd), _ptr(act), _ptr(wd),
                                             _ptr(residual), _ptr(out)))
        return out
    return kernel


def classifier_gemv(B: int, V: int, D: int):
    """logits = body Wq^T + bias (tilelang_kernels.py:146-173)."""
    def kernel(body, wq, bias):
        out = _empty(body, B, V)
        check(lib().sk_op_classifier_gemv(_stream(body), B, V, D, _wdtype(wq), _ptr(body), _ptr(wq),
                                          _ptr(bias), _ptr(out)))
        return out
    return kernel


def frame_embed(R: int, Q: int, V: int, D: int, scale: float):
    """out[r] = scale * sum_q table[q, codes[r, q]] (tilelang_kernels.py:176-196)."""
    def kernel(codes, table):
        out = _empty(table, R, D)
        check(lib().sk_op_frame_embed(_stream(table), R, Q, V, D, scale, _ptr(codes), _ptr(table),
                                      _ptr(out)))
        return out
    return kernel


def prefix_add(B: int, V: int, D: int, scale: float):
    """out = prefix + table_q[code] * scale (tilelang_kernels.py:199-216)."""
    def kernel(prefix, table_q, code):
        out = _empty(prefix, B, D)
        check(lib().sk_op_prefix_add(_stream(prefix), B, V, D, scale, _ptr(prefix), _ptr(table_q),
                                     _ptr(code), _ptr(out)))
        return out
    return kernel


def sampling_prep(V: int, bos_id: int, pad_id: int, eos_id: int):
    """out = logits / T with BOS/PAD (and EOS if flagged) masked
    (tilelang_kernels.py:219-254)."""
    def kernel(logits, temperature, mask_eos):
        out = _empty(logits, V)
        check(lib().sk_op_sampling_prep(_stream(logits), V, bos_id, pad_id, eos_id, _ptr(logits),
                                        _ptr(temperature), _ptr(mask_eos), _ptr(out)))
        return out
    return kernel


def sample(V: int, bos_id: int, eos_id: int, pad_id: int):
    """Fused CFG + masks + temperature + top-k/top-p + explicit-uniform draw
    (model.py:579-595,686-708); ``kernel(logits[rows, V], ...) -> int64[1]``."""
    def kernel(logits, *, cfg_scale: float, q: int, mask_eos_q0: bool, temperature: float,
               top_k, top_p, u: float):
        import torch

        rows = logits.shape[0]
        out = torch.empty(1, device=logits.device, dtype=torch.int64)
        check(lib().sk_op_sample(_stream(logits), rows, V, _ptr(logits), float(cfg_scale), int(q),
                                 int(bool(mask_eos_q0)), bos_id, eos_id, pad_id, float(temperature),
                                 int(top_k or 0), float(top_p or 0.0), float(u), _ptr(out)))
        return out
    return kernel


# ---- attention over a cache in pages (no counterpart in the reference) ----
# Pools k_pages / v_pages [n_pages, Hkv, page, hd] (float32 or bfloat16), table
# [S, width] int32 (any row stride, so a slice of a wider one will do), starts
# [S + 1] and lens [S] int32, all on the HIP device: sequence s's new tokens are
# the packed rows starts[s]:starts[s + 1] and lens[s] its length with them.  Calls are
# planned from rows per sequence and width: single tokens and chunks belong in calls of their
# own, and a wide table is passed as a slice that the longest sequence fills.
# include/soraku_mi355x.h holds the whole contract.
#
# A single-token call runs for 4 to 25 us on the GPU, so the host's part is kept
# short: one pass of cheap checks, the raw stream handle, no Stream or pointer
# objects.

class _Torch:
    """What these operators use of torch, looked up once."""

    def __init__(self):
        import torch

        self.f32, self.bf16, self.i32, self.u8 = torch.float32, torch.bfloat16, torch.int32, torch.uint8
        self.i8, self.i64, self.f64 = torch.int8, torch.int64, torch.float64
        self.empty, self.empty_like, self.on = torch.empty, torch.empty_like, torch.cuda.device
        self.stream, self.device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        self.codes = {torch.float32: _lib.SK_F32, torch.bfloat16: _lib.SK_BF16}
        self.lib = lib()


@functools.lru_cache(maxsize=None)
def _torch() -> _Torch:
    return _Torch()


def _need(t, name, dtype, at, shape):
    """t's address; t must be contiguous, of that type and shape, on device number ``at``."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != at or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {shape} on HIP device {at}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}{'' if t.is_contiguous() else ', not contiguous'}")
    return t.data_ptr()


def _int32(**sizes):
    """The sizes; a foreign call would cut them down to their lowest 32 bits."""
    for name, n in sizes.items():
        if operator.index(n) >> 31 not in (0, -1):
            raise ValueError(f"{name} must be a 32-bit integer, got {n}")
    return map(operator.index, sizes.values())


def _table(t, name, dtype, at, S):
    """(address, row stride, entries per row) of a page table."""
    if t.dtype is not dtype or t.get_device() != at or t.dim() != 2 or t.shape[0] != S:
        raise ValueError(f"{name} must be an int32 tensor [{S}, pages] on HIP device {at}")
    width, (stride, step) = t.shape[1], t.stride()
    if (S | width) >> 31:
        raise ValueError(f"{name} must be smaller than 2^31 x 2^31")
    if (width > 1 and step != 1) or (S > 1 and stride < width):
        raise ValueError(f"{name}'s rows must be contiguous and apart")
    return t.data_ptr(), stride if S > 1 else width, width


def _pool(k_pages, v_pages, Hkv, page, hd, codes):
    """(device number, pages, addresses of K and V, type code)."""
    if not k_pages.is_cuda:
        raise ValueError("operands must live on the HIP device")
    if k_pages.dim() != 4 or k_pages.dtype not in codes:
        raise ValueError("pages must be [n_pages, Hkv, page, hd], float32 or bfloat16")
    dt, at, n = k_pages.dtype, k_pages.get_device(), k_pages.shape[0]
    shape = (n, Hkv, page, hd)
    kp = _need(k_pages, "k_pages", dt, at, shape)
    return at, n, kp, None if v_pages is None else _need(v_pages, "v_pages", dt, at, shape), codes[dt]


def _code(t, codes):
    if t.dtype not in codes:
        raise ValueError(f"dtype {t.dtype} not supported (float32 or bfloat16)")
    if t.shape[0] >> 31:
        raise ValueError("too many tokens")
    return codes[t.dtype]


def _call(T, fn, at, *args):
    """fn(stream, *args) on device ``at`` and its current stream."""
    if at == T.device():
        check(fn(T.stream(at), *args))
    else:
        with T.on(at):
            check(fn(T.stream(at), *args))


@functools.lru_cache(maxsize=1024)
def _attention_workspace(*sizes) -> int:
    n = C.c_int64()
    check(lib().sk_op_paged_attention_workspace(*sizes, C.byref(n)))
    return n.value


@functools.lru_cache(maxsize=1024)
def _mass_workspace(*sizes) -> int:
    n = C.c_int64()
    check(lib().sk_op_paged_attention_mass_workspace(*sizes, C.byref(n)))
    return n.value


def paged_append(Hq: int, Hkv: int, hd: int, page: int, eps: float):
    """New tokens into the cache: per-head RMSNorm of q and k (gains ``[hd]``, or
    both None for none), rotation by ``positions * inv_freq``, k and v to
    their slots; returns q ``[T, Hq, hd]`` of qkv's dtype (``out``, if given).
    ``mass`` (accounts, ``[n_pages, Hkv, page]`` float32) is set to 0 at the new slots."""
    Hq, Hkv, hd, page = _int32(Hq=Hq, Hkv=Hkv, hd=hd, page=page)

    def kernel(qkv, q_gain, k_gain, inv_freq, positions, starts, lens, table, k_pages, v_pages, mass=None, out=None):
        T = _torch()
        f32, i32 = T.f32, T.i32
        at, n, kp, vp, kd = _pool(k_pages, v_pages, Hkv, page, hd, T.codes)
        xd, dt, rows, S = _code(qkv, T.codes), qkv.dtype, qkv.shape[0], lens.shape[0]
        tp, stride, width = _table(table, "table", i32, at, S)
        if out is None:
            out = T.empty(rows, Hq, hd, device=k_pages.device, dtype=dt)
        _call(T, T.lib.sk_op_paged_append, at, rows, S, Hq, Hkv, hd, page, n, width, stride, xd, kd, eps,
              _need(qkv, "qkv", dt, at, (rows, (Hq + 2 * Hkv) * hd)),
              None if q_gain is None else _need(q_gain, "q_gain", f32, at, (hd,)),
              None if k_gain is None else _need(k_gain, "k_gain", f32, at, (hd,)),
              _need(inv_freq, "inv_freq", f32, at, (hd // 2,)), _need(positions, "positions", i32, at, (rows,)),
              _need(starts, "starts", i32, at, (S + 1,)), _need(lens, "lens", i32, at, (S,)), tp, kp, vp,
              None if mass is None else _need(mass, "mass", f32, at, (n, Hkv, page)),
              _need(out, "out", dt, at, (rows, Hq, hd)))
        return out
    return kernel


def paged_attention(Hq: int, Hkv: int, hd: int, page: int, scale: float | None = None, window: int = 0,
                    sinks: int = 0):
    """out ``[T, Hq, hd]`` = softmax(scale q k^T) v of the new tokens over their
    sequences' slots, causal; with a ``window`` only the last ``window`` slots and the
    first ``sinks``.  ``scale`` defaults to hd ** -0.5.  ``lse`` ``[T, Hq]`` float32,
    if given, receives the softmax's logarithms.  Tokens that see nothing give 0 and -inf."""
    Hq, Hkv, hd, page, window, sinks = _int32(Hq=Hq, Hkv=Hkv, hd=hd, page=page, window=window, sinks=sinks)
    scale = hd ** -0.5 if scale is None else float(scale)

    def kernel(q, k_pages, v_pages, table, starts, lens, out=None, lse=None):
        T = _torch()
        i32 = T.i32
        at, n, kp, vp, kd = _pool(k_pages, v_pages, Hkv, page, hd, T.codes)
        xd, dt, rows, S = _code(q, T.codes), q.dtype, q.shape[0], lens.shape[0]
        tp, stride, width = _table(table, "table", i32, at, S)
        shape = (rows, Hq, hd)
        if out is None:
            out = T.empty_like(q)
        size = _attention_workspace(rows, S, Hq, Hkv, hd, page, width, xd, kd, window, sinks)
        ws = T.empty(size, device=k_pages.device, dtype=T.u8) if size else None
        _call(T, T.lib.sk_op_paged_attention, at, rows, S, Hq, Hkv, hd, page, n, width, stride, xd, kd, scale, window,
              sinks, _need(q, "q", dt, at, shape), kp, vp, tp, _need(starts, "starts", i32, at, (S + 1,)),
              _need(lens, "lens", i32, at, (S,)), _need(out, "out", dt, at, shape),
              None if lse is None else _need(lse, "lse", T.f32, at, (rows, Hq)), ws.data_ptr() if size else None, size)
        return out
    return kernel


def paged_attention_mass(Hq: int, Hkv: int, hd: int, page: int, scale: float | None = None, window: int = 0,
                         sinks: int = 0):
    """Adds the weight every slot got in the ``paged_attention`` call of the same
    arguments (its ``q`` and ``lse``) to ``mass`` ``[n_pages, Hkv, page]`` float32, summed over
    tokens and the query heads that share a key head; returns ``mass``."""
    Hq, Hkv, hd, page, window, sinks = _int32(Hq=Hq, Hkv=Hkv, hd=hd, page=page, window=window, sinks=sinks)
    scale = hd ** -0.5 if scale is None else float(scale)

    def kernel(q, lse, k_pages, table, starts, lens, mass):
        T = _torch()
        f32, i32 = T.f32, T.i32
        at, n, kp, _, kd = _pool(k_pages, None, Hkv, page, hd, T.codes)
        xd, rows, S = _code(q, T.codes), q.shape[0], lens.shape[0]
        tp, stride, width = _table(table, "table", i32, at, S)
        size = _mass_workspace(rows, S, Hq, Hkv, hd, page, width, xd, kd)
        ws = T.empty(size, device=k_pages.device, dtype=T.u8) if size else None
        _call(T, T.lib.sk_op_paged_attention_mass, at, rows, S, Hq, Hkv, hd, page, n, width, stride, xd, kd, scale, window,
              sinks, _need(q, "q", q.dtype, at, (rows, Hq, hd)), _need(lse, "lse", f32, at, (rows, Hq)), kp, tp,
              _need(starts, "starts", i32, at, (S + 1,)), _need(lens, "lens", i32, at, (S,)),
              _need(mass, "mass", f32, at, (n, Hkv, page)), ws.data_ptr() if size else None, size)
        return mass
    return kernel


def paged_evict(Hkv: int, hd: int, page: int, keep: int, sinks: int = 0, recent: int = 0):
    """Cuts caches back to ``keep`` slots per key head: the first ``sinks``, the last
    ``recent``, and of the others those of the largest accounts (ties to the lowest slot) move in
    order, with their accounts, to the pages of ``to`` ``[S, pages]``, none of which may be in ``table``.
    Returns the new lengths ``[S]`` and the old slots ``[S, Hkv, keep]`` (-1 past the length), int32."""
    Hkv, hd, page, keep, sinks, recent = _int32(Hkv=Hkv, hd=hd, page=page, keep=keep, sinks=sinks, recent=recent)

    def kernel(k_pages, v_pages, mass, table, lens, to):
        T = _torch()
        i32 = T.i32
        at, n, kp, vp, kd = _pool(k_pages, v_pages, Hkv, page, hd, T.codes)
        S, dev = lens.shape[0], k_pages.device
        tp, stride, width = _table(table, "table", i32, at, S)
        dp, to_stride, to_width = _table(to, "to", i32, at, S)
        new_lens = T.empty(S, device=dev, dtype=i32)
        kept = T.empty((S, Hkv, keep), device=dev, dtype=i32)
        _call(T, T.lib.sk_op_paged_evict, at, S, Hkv, hd, page, n, width, stride, kd, keep, sinks, recent, kp, vp,
              _need(mass, "mass", T.f32, at, (n, Hkv, page)), tp, _need(lens, "lens", i32, at, (S,)), dp, to_stride,
              to_width, new_lens.data_ptr(), kept.data_ptr())
        return new_lens, kept
    return kernel


# ---- projections with 8-bit weights (no counterpart in the reference) ----
# A matrix [N, K] is held as codes [N, Kp] int8 (Kp: K up to a multiple of 128, zeros behind)
# and scales [N] float32, one per row; int8_rows makes them, once, when weights are loaded.
# Activations are float32 or bfloat16 and become codes, row by row, inside int8_linear.

@functools.lru_cache(maxsize=1024)
def _linear_workspace(*sizes) -> int:
    n = C.c_int64()
    check(lib().sk_op_int8_linear_workspace(*sizes, C.byref(n)))
    return n.value


def _matrix(t, name, K, codes):
    """(device number, rows, type code) of a contiguous [rows, K] tensor of float32 or bfloat16."""
    if not t.is_cuda:
        raise ValueError("operands must live on the HIP device")
    if t.dim() != 2 or t.shape[1] != K or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor [rows, {K}], got {tuple(t.shape)}"
                         f"{'' if t.is_contiguous() else ', not contiguous'}")
    return t.get_device(), t.shape[0], _code(t, codes)


def int8_rows(K: int):
    """``kernel(x[R, K]) -> codes [R, Kp] int8, scales [R] float32``: each row as the nearest whole
    numbers of 127 x / max|x| and the scale max|x| / 127."""
    K, = _int32(K=K)

    def kernel(x):
        T = _torch()
        at, rows, xd = _matrix(x, "x", K, T.codes)
        codes = x.new_empty(rows, -(-K // 128) * 128, dtype=T.i8)
        scales = x.new_empty(rows, dtype=T.f32)
        _call(T, T.lib.sk_op_int8_rows, at, rows, K, xd, x.data_ptr(), codes.data_ptr(), scales.data_ptr())
        return codes, scales
    return kernel


def int8_linear(N: int, K: int, act: str | None = None, eps: float | None = None):
    """out ``[M, N]`` = act(x W^T + bias) + residual with W as ``codes`` [N, Kp] and ``scales`` [N] of
    ``int8_rows``; of x's dtype.  ``act="swiglu"``: W has 2 N rows, gate rows first, and act is
    silu(gate) * up.  With ``eps`` x is normalised first (RMSNorm, ``gain`` [K] or none).  ``out`` may be
    ``residual`` itself."""
    N, K = _int32(N=N, K=K)
    if act not in (None, "swiglu"):
        raise ValueError(f"act must be None or 'swiglu', got {act!r}")
    both, kp = (2 * N if act else N), -(-K // 128) * 128
    act = _lib.SK_ACT_SWIGLU if act else _lib.SK_ACT_NONE
    if eps is not None and not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    eps = -1.0 if eps is None else float(eps)

    def kernel(x, codes, scales, gain=None, bias=None, residual=None, out=None):
        T = _torch()
        f32, dt = T.f32, x.dtype
        at, rows, xd = _matrix(x, "x", K, T.codes)
        shape = (rows, N)
        if out is None:
            out = x.new_empty(rows, N)
            op = out.data_ptr()
        else:
            op = _need(out, "out", dt, at, shape)
        size = _linear_workspace(rows, N, K, xd, act)
        ws = x.new_empty(size, dtype=T.u8) if size else None
        _call(T, T.lib.sk_op_int8_linear, at, rows, N, K, xd, act, eps, x.data_ptr(),
              None if gain is None else _need(gain, "gain", f32, at, (K,)), _need(codes, "codes", T.i8, at, (both, kp)),
              _need(scales, "scales", f32, at, (both,)), None if bias is None else _need(bias, "bias", f32, at, (both,)),
              None if residual is None else _need(residual, "residual", dt, at, shape), op,
              ws.data_ptr() if size else None, size)
        return out
    return kernel


# ---- sampling by row (sample for a batch, model.py:686-708) ----

@functools.lru_cache(maxsize=1024)
def _sample_workspace(*sizes) -> int:
    n = C.c_int64()
    check(lib().sk_op_sample_rows_workspace(*sizes, C.byref(n)))
    return n.value


def sample_rows(V: int, cfg: bool = False):
    """One id per row of logits ``[R, V]`` (float32 or bfloat16; rows may be apart) from the uniform draws
    ``u`` [R] float64: ``kernel(logits, u, temperature=None, top_k=None, top_p=None, min_p=None,
    cfg_scale=None, allowed=None, out=None, logprob=None, kept=None) -> int64[R]``.

    Parameters are tensors [R] on the device (``top_k`` int32, the others float32) or None for none of
    it; a temperature that is not above 0 is greedy.  With ``cfg`` the logits are ``[R, 2, V]``, cond and
    uncond, merged with ``cfg_scale``.  ``allowed``: bits of the ids that may be drawn, int32 ``[R or 1, ceil(V / 32)]``.
    ``logprob`` [R] float32 and ``kept`` [R] int32, if given, receive the drawn id's log-probability among the
    kept ones, and their number.  A row without candidates gives -1."""
    V, = _int32(V=V)
    words = (V + 31) // 32

    def kernel(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, cfg_scale=None, allowed=None, out=None,
               logprob=None, kept=None):
        T = _torch()
        f32, i32 = T.f32, T.i32
        if not logits.is_cuda:
            raise ValueError("operands must live on the HIP device")
        at, dim, shape, step = logits.get_device(), 3 if cfg else 2, logits.shape, logits.stride()
        if len(shape) != dim or shape[-1] != V or (cfg and shape[1] != 2):
            raise ValueError(f"logits must be [rows, {'2, ' if cfg else ''}{V}], got {tuple(shape)}")
        rows, dt = shape[0], _code(logits, T.codes)
        stride = step[-2] if cfg or rows > 1 else V
        if (V > 1 and step[-1] != 1) or stride < V or (cfg and rows > 1 and step[0] != 2 * stride):
            raise ValueError("logits' rows must be contiguous and evenly apart")
        if cfg != (cfg_scale is not None):
            raise ValueError("cfg_scale comes with cfg")
        n = (rows,)
        if out is None:
            out = logits.new_empty(rows, dtype=T.i64)
            op = out.data_ptr()
        else:
            op = _need(out, "out", T.i64, at, n)
        apart = 0
        if allowed is not None:
            if allowed.dim() != 2 or allowed.shape[0] not in (1, rows):
                raise ValueError(f"allowed must be int32 [{rows} or 1, {words}]")
            _need(allowed, "allowed", i32, at, (allowed.shape[0], words))
            apart = words if allowed.shape[0] == rows else 0
        size = _sample_workspace(rows, V, dt)
        ws = logits.new_empty(size, dtype=T.u8) if size else None
        _call(T, T.lib.sk_op_sample_rows, at, rows, V, dt, logits.data_ptr(), stride, _need(u, "u", T.f64, at, n),
              None if temperature is None else _need(temperature, "temperature", f32, at, n),
              None if top_k is None else _need(top_k, "top_k", i32, at, n),
              None if top_p is None else _need(top_p, "top_p", f32, at, n),
              None if min_p is None else _need(min_p, "min_p", f32, at, n),
              None if cfg_scale is None else _need(cfg_scale, "cfg_scale", f32, at, n),
              None if allowed is None else allowed.data_ptr(), apart, op,
              None if logprob is None else _need(logprob, "logprob", f32, at, n),
              None if kept is None else _need(kept, "kept", i32, at, n), ws.data_ptr() if size else None, size)
        return out
    return kernel
