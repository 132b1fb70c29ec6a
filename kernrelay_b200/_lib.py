"""ctypes binding of libkernrelay.so's B200 extension ABI (include/kernrelay_b200.h).

Everything here calls into the CUDA library; there is no Python or CPU fallback.
If the library is missing the import of the wrappers fails loudly.
"""
from __future__ import annotations

import ctypes
import json
import os
from array import array
from pathlib import Path

_PKG = Path(__file__).resolve().parent
_LIB = None

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_long = ctypes.c_long
c_float = ctypes.c_float
c_size_t = ctypes.c_size_t
c_char_p = ctypes.c_char_p
c_u64 = ctypes.c_uint64
c_u32p = ctypes.POINTER(ctypes.c_uint32)
c_i64 = ctypes.c_int64


class KVCacheDesc(ctypes.Structure):
    """krb_kv_cache of include/kernrelay_b200.h."""
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("dtype", c_int), ("layers", c_int),
                ("pages", c_int), ("heads", c_int), ("page_size", c_int), ("head_dim", c_int),
                ("k_stride", ctypes.c_int64 * 4), ("v_stride", ctypes.c_int64 * 4)]


def lib_path() -> Path:
    env = os.environ.get("KERNRELAY_LIB")
    return Path(env) if env else _PKG / "libkernrelay.so"


# (name, restype, argtypes) of every exported symbol of include/kernrelay.h and
# include/kernrelay_b200.h; tests check the library exports exactly these.
SIGNATURES = [
    ("kr_version", c_char_p, []),
    ("kr_plan_run", c_int, [c_char_p, c_int, c_int, c_char_p, c_char_p, c_char_p]),
    ("kr_qwen_run", c_int, [c_char_p, c_char_p, c_int, c_int, c_int, c_int, c_char_p, c_size_t]),
    ("kr_qwen_pp_run", c_int, [c_char_p, c_char_p, c_int, c_int, c_int, c_int, c_int, c_int,
                               c_char_p, c_size_t]),
    ("kr_qwen_tp_run", c_int, [c_char_p, c_char_p, c_int, c_int, c_int, c_int, c_int, c_int,
                               c_char_p, c_size_t]),
    ("kr_qwen_profile_many", c_int, [c_char_p, c_char_p, c_int, c_int, c_char_p, c_size_t]),
    ("krb_last_error", c_char_p, []),
    ("krb_device_count", c_int, []),
    ("krb_synth_normal_host", c_int, [c_char_p, c_u64, ctypes.c_double, ctypes.c_double, c_u64,
                                      c_u64, c_void_p]),
    ("krb_gemm_bf16", c_int, [c_void_p, c_long, c_void_p, c_long, c_void_p, c_long, c_void_p,
                              c_int, c_int, c_int, c_int, c_void_p]),
    ("krb_gemm_f32out", c_int, [c_void_p, c_long, c_void_p, c_long, c_void_p, c_long, c_int, c_int,
                                c_int, c_int, c_void_p]),
    ("krb_gemm_silu_bf16", c_int, [c_void_p, c_long, c_void_p, c_long, c_void_p, c_long, c_int,
                                   c_int, c_int, c_int, c_void_p]),
    ("krb_gemm_qkv_rope_bf16", c_int, [c_void_p, c_long, c_void_p, c_long, c_void_p, c_long,
                                       c_void_p, c_int, c_int, c_int, c_int, c_int, c_void_p,
                                       c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_long,
                                       c_void_p]),
    ("krb_rmsnorm_bf16", c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_float,
                                 c_void_p]),
    ("krb_add_rmsnorm_bf16", c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                     c_int, c_int, c_float, c_void_p]),
    ("krb_add_rmsnorm_res_f32", c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int,
                                        c_int, c_float, c_void_p]),
    ("krb_embed_bf16", c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p,
                               c_void_p]),
    ("krb_qk_norm_rope_bf16", c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p,
                                      c_void_p, c_void_p, c_float, c_void_p]),
    ("krb_attention_prefill_bf16", c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                           c_float, c_int, c_void_p, c_void_p]),
    ("krb_qk_norm_rope_paged", c_int, [c_void_p, c_int, c_void_p, c_i64, c_void_p, c_i64, c_void_p,
                                       c_void_p, c_int, c_int, c_void_p, c_void_p, c_int,
                                       c_void_p, c_void_p, c_float, c_void_p, c_void_p]),
    ("krb_attention_paged", c_int, [c_void_p, c_int, c_void_p, c_i64, c_void_p, c_i64, c_int,
                                    c_int, c_void_p, c_i64, c_int, c_void_p, c_void_p, c_int,
                                    c_int, c_void_p, c_i64, c_int, c_float, c_void_p, c_size_t,
                                    c_void_p, c_void_p]),
    ("krb_attention_paged_workspace", c_size_t, [c_void_p, c_int, c_int]),
    ("krb_kv_copy_pages", c_int, [c_void_p, c_void_p, c_void_p, c_int, c_void_p]),
    ("krb_kv_commit", c_int, [c_void_p, c_void_p, c_i64, c_int, c_void_p, c_void_p, c_i64, c_int,
                              c_void_p, c_int, c_void_p, c_void_p]),
    ("krb_relay_down_single", c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                      c_int, c_int, c_int, c_int, c_float, c_int, c_void_p,
                                      c_void_p]),
    ("krb_relay_down_single_noalloc", c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                              c_void_p, c_int, c_int, c_int, c_int, c_float,
                                              c_int, c_void_p, c_void_p]),
    ("krb_relay_timeout_probe", c_int, [c_int, c_int, c_int, c_int, c_float, c_u32p]),
    ("krb_relay_plan", c_int, [c_int, c_int, c_int, c_int, c_int, c_int, c_char_p, c_size_t]),
    ("krb_plan_check", c_int, [c_char_p, c_char_p, c_size_t]),
    ("krb_engine_create", c_int, [c_char_p, c_char_p, c_int, c_int, c_int, c_int, c_int,
                                  ctypes.POINTER(c_void_p)]),
    ("krb_microdag_create", c_int, [c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_char_p,
                                    c_u64, ctypes.POINTER(c_void_p)]),
    ("krb_engine_destroy", None, [c_void_p]),
    ("krb_engine_ipc_handle", c_int, [c_void_p, c_void_p, c_size_t]),
    ("krb_engine_open_peers", c_int, [c_void_p, c_void_p, c_size_t]),
    ("krb_nccl_unique_id", c_int, [c_void_p, c_size_t]),
    ("krb_engine_init_nccl", c_int, [c_void_p, c_void_p, c_size_t]),
    ("krb_engines_link", c_int, [ctypes.POINTER(c_void_p), c_int]),
    ("krb_engines_init_nccl", c_int, [ctypes.POINTER(c_void_p), c_int]),
    ("krb_engine_capture", c_int, [c_void_p]),
    ("krb_engine_run", c_int, [c_void_p]),
    ("krb_engine_run_host", c_int, [c_void_p, c_void_p, c_void_p]),
    ("krb_engine_sync", c_int, [c_void_p]),
    ("krb_engine_stream", c_int, [c_void_p, ctypes.POINTER(c_void_p)]),
    ("krb_engine_status", c_int, [c_void_p, c_u32p]),
    ("krb_engine_stage_times", c_int, [c_void_p, c_char_p, c_size_t]),
    ("krb_engine_verify", c_int, [c_void_p, c_char_p, c_size_t]),
    ("krb_engine_last_logits", c_int, [c_void_p, c_void_p, c_int]),
    ("krb_engine_final_hidden", c_int, [c_void_p, c_void_p, c_size_t]),
    ("krb_engine_final_x", c_int, [c_void_p, c_void_p, c_size_t]),
    ("krb_engine_layer_dump", c_int, [c_void_p, c_int]),
    ("krb_engine_layer_hidden", c_int, [c_void_p, c_int, c_void_p, c_size_t]),
    ("krb_engine_info", c_int, [c_void_p, c_char_p, c_size_t]),
    ("krb_engine_relay_trace", c_int, [c_void_p, c_void_p, c_size_t, ctypes.POINTER(c_size_t)]),
]


def lib():
    global _LIB
    if _LIB is None:
        p = lib_path()
        if not p.exists():
            raise FileNotFoundError(
                f"{p} is missing; build it with `python -m kernrelay_b200.build`")
        L = ctypes.CDLL(str(p))
        for name, res, args in SIGNATURES:
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _LIB = L
    return _LIB


class KrbError(RuntimeError):
    pass


def check(rc: int, what: str = ""):
    if rc != 0:
        msg = lib().krb_last_error().decode(errors="replace")
        raise KrbError(f"{what}: {msg}" if what else msg)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _addr(t):
    return None if t is None else t.data_ptr()


def _empty(shape, dtype, like, stream):
    """A tensor on `like`'s device that this call's kernels on `stream` use: allocated on that
    stream, so that the allocator does not hand its memory to another stream's work too early."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    import torch
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _raw_stream(stream, index):
    """cudaStream_t of `stream`, or of the current stream of device `index`."""
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(index)


def _stream(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


# ---------------------------------------------------------------- tensor-level op wrappers
def gemm(A, B, bias=None, out=None, bn=0, stream=None):
    """C = A @ B.T (+bias): A [M,K], B [N,K] bf16 contiguous (row pitch may differ)."""
    import torch
    M, K = A.shape
    N = B.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.bfloat16, device=A.device)
    check(lib().krb_gemm_bf16(_ptr(A), A.stride(0), _ptr(B), B.stride(0), _ptr(out), out.stride(0),
                              _ptr(bias), M, N, K, bn, _stream(stream)), "gemm")
    return out


def gemm_f32(A, B, out=None, bn=0, stream=None):
    """fp32 C = A @ B.T (unrounded)."""
    import torch
    M, K = A.shape
    N = B.shape[0]
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=A.device)
    check(lib().krb_gemm_f32out(_ptr(A), A.stride(0), _ptr(B), B.stride(0), _ptr(out),
                                out.stride(0), M, N, K, bn, _stream(stream)), "gemm_f32")
    return out


def gemm_silu(A, Bgu, n_out, bn, out=None, stream=None):
    import torch
    M, K = A.shape
    if out is None:
        out = torch.empty((M, n_out), dtype=torch.bfloat16, device=A.device)
    check(lib().krb_gemm_silu_bf16(_ptr(A), A.stride(0), _ptr(Bgu), Bgu.stride(0), _ptr(out),
                                   out.stride(0), M, n_out, K, bn, _stream(stream)), "gemm_silu")
    return out


def interleave_gate_up(Wg, Wu, bn):
    """[I, K] gate and up rows -> the gate/up block interleave used by gemm_silu."""
    import torch
    I, K = Wg.shape
    half = bn // 2
    nblk = (I + half - 1) // half
    out = torch.zeros((nblk * bn, K), dtype=Wg.dtype, device=Wg.device)
    for b in range(nblk):
        lo, hi = b * half, min(I, (b + 1) * half)
        out[b * bn: b * bn + (hi - lo)] = Wg[lo:hi]
        out[b * bn + half: b * bn + half + (hi - lo)] = Wu[lo:hi]
    return out


def rmsnorm(x, gamma, eps, out=None, stream=None):
    import torch
    rows, H = x.shape
    out = torch.empty_like(x) if out is None else out
    check(lib().krb_rmsnorm_bf16(_ptr(x), _ptr(gamma), _ptr(out), None, rows, H, eps,
                                 _stream(stream)), "rmsnorm")
    return out


def add_rmsnorm(a, b, gamma, eps, stream=None):
    import torch
    rows, H = a.shape
    y = torch.empty_like(a)
    s = torch.empty_like(a)
    check(lib().krb_add_rmsnorm_bf16(_ptr(a), _ptr(b), _ptr(gamma), _ptr(y), None, _ptr(s), rows,
                                     H, eps, _stream(stream)), "add_rmsnorm")
    return y, s


def add_rmsnorm_res(res, delta, gamma, eps, stream=None):
    """fp32 residual form: (y bf16, sum fp32) with sum = res + delta."""
    import torch
    rows, H = res.shape
    y = torch.empty((rows, H), dtype=torch.bfloat16, device=res.device)
    s = torch.empty_like(res)
    check(lib().krb_add_rmsnorm_res_f32(_ptr(res), _ptr(delta), _ptr(gamma), _ptr(y), _ptr(s), rows,
                                        H, eps, _stream(stream)), "add_rmsnorm_res")
    return y, s


def embed(ids, table, status=None, stream=None):
    import torch
    S = ids.shape[0]
    V, H = table.shape
    out = torch.empty((S, H), dtype=torch.bfloat16, device=table.device)
    check(lib().krb_embed_bf16(_ptr(ids), _ptr(table), _ptr(out), S, H, V, _ptr(status),
                               _stream(stream)), "embed")
    return out


def gemm_qkv_rope(A, B, HQ, HKV, D, cos, sin, bias=None, q_norm=None, k_norm=None, eps=1e-6,
                  vt=None, stream=None):
    """Fused QKV GEMM (+bias) with per-head QK-norm and RoPE in the epilogue; with `vt`
    (fp16 [HKV*D, ldvt >= M]) the v heads are also written transposed."""
    import torch
    M, K = A.shape
    N = (HQ + 2 * HKV) * D
    out = torch.empty((M, N), dtype=torch.bfloat16, device=A.device)
    check(lib().krb_gemm_qkv_rope_bf16(_ptr(A), A.stride(0), _ptr(B), B.stride(0), _ptr(out),
                                       out.stride(0), _ptr(bias), M, K, HQ, HKV, D, _ptr(cos),
                                       _ptr(sin), _ptr(q_norm), _ptr(k_norm), eps, _ptr(vt),
                                       vt.stride(0) if vt is not None else 0, _stream(stream)),
          "gemm_qkv_rope")
    return out


def qk_norm_rope(qkv, HQ, HKV, D, cos, sin, q_norm=None, k_norm=None, eps=1e-6, stream=None):
    S = qkv.shape[0]
    check(lib().krb_qk_norm_rope_bf16(_ptr(qkv), S, HQ, HKV, D, _ptr(cos), _ptr(sin), _ptr(q_norm),
                                      _ptr(k_norm), eps, _stream(stream)), "qk_norm_rope")
    return qkv


def attention(qkv, HQ, HKV, D, scale, impl=0, status=None, stream=None):
    """Causal GQA attention over the fused qkv buffer with the tcgen05 kernel (head_dim 64
    or 128); impl 0 and 2 both select it."""
    import torch
    S = qkv.shape[0]
    out = torch.empty((S, HQ * D), dtype=torch.bfloat16, device=qkv.device)
    check(lib().krb_attention_prefill_bf16(_ptr(qkv), _ptr(out), S, HQ, HKV, D, scale, impl,
                                           _ptr(status), _stream(stream)), "attention")
    return out


# ---------------------------------------------------------------- paged K/V cache
class KVCache:
    """A paged K/V cache in the caller's tensors: k and v of the same shape [pages, heads,
    page_size, head_dim], or [layers, pages, ...], bf16 or fp16, head_dim contiguous, the other
    axes of any strides (pass `x.transpose(-3, -2)` where the slot axis is stored outside the
    heads').  page_size: a power of two from 8 on; head_dim 64 or 128.  The handle keeps the
    tensors; make it once per cache.

    The operators below run on the current stream of the cache's device, or on stream=.  Outputs and
    workspaces that a call allocates belong to that stream; that its inputs are ready on it, and live
    until it is done with them (torch's record_stream), is the caller's, as in torch."""

    def __init__(self, k, v):
        import torch
        if k.shape != v.shape or k.dim() not in (4, 5):
            raise KrbError("KVCache: k and v must be [pages, heads, page_size, head_dim] or "
                           "[layers, pages, heads, page_size, head_dim]")
        if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float16):
            raise KrbError("KVCache: k and v must both be bf16 or both fp16")
        if k.device != v.device:
            raise KrbError("KVCache: k and v on different devices")
        if k.stride(-1) != 1 or v.stride(-1) != 1:
            raise KrbError("KVCache: head_dim must be contiguous")
        self.k, self.v, self.dtype, self.index = k, v, k.dtype, k.get_device()
        sizes = ((1,) + tuple(k.shape))[-5:]
        self.layers, self.pages, self.heads, self.page_size, self.head_dim = sizes
        strides = [((0,) + tuple(t.stride()))[-5:-1] for t in (k, v)]
        self.desc = KVCacheDesc(k.data_ptr(), v.data_ptr(), int(k.dtype == torch.float16), *sizes,
                                *((c_i64 * 4)(*s) for s in strides))
        self.ref = ctypes.addressof(self.desc)
        self._workspaces = {}  # (HQ, max_q) -> bytes

    def attention_workspace(self, HQ, max_q):
        """Bytes of attention_paged's workspace (krb_attention_paged_workspace)."""
        n = self._workspaces.get((HQ, max_q))
        if n is None:
            import torch
            if not 0 <= max_q < 2 ** 31:  # a C int would take it modulo 2^32
                raise KrbError(f"attention_paged: bad max_q {max_q}")
            if self.index < 0:
                raise KrbError("KVCache: the cache is not on a GPU")
            with torch.cuda.device(self.index):
                n = lib().krb_attention_paged_workspace(self.ref, HQ, max_q)
            if not n:
                raise KrbError(lib().krb_last_error().decode(errors="replace"))
            self._workspaces[HQ, max_q] = n
        return n


def _is(t, dtype, index, dim):
    """A dim-d tensor of dtype on CUDA device `index` whose last axis is contiguous.  These
    operators' smallest calls take a few microseconds, so their checks are kept as cheap (row
    pitches below: rows that are never stepped over may have any stride)."""
    return (t.dtype is dtype and t.get_device() == index and t.dim() == dim
            and (t.stride()[-1] == 1 or t.shape[-1] <= 1))


def _refuse(what, name, t, dtype, dim):
    raise KrbError(f"{what}: {name} must be a {dim}-d {dtype} tensor on the cache's device with its "
                   f"last axis contiguous, got {t.dim()}-d {t.dtype} on {t.device}, strides "
                   f"{tuple(t.stride())}")


def _check_layer(what, cache, layer):
    if not 0 <= layer < cache.layers:
        raise KrbError(f"{what}: no such layer ({layer} of {cache.layers})")


def _enter(cache):
    """None where the cache's device is the current one, else the context to call again in."""
    import torch
    if cache.index < 0:
        raise KrbError("KVCache: the cache is not on a GPU")
    if torch._C._cuda_getDevice() == cache.index:  # a CUDA tensor exists: CUDA is initialised
        return None
    return torch.cuda.device(cache.index)


def qk_norm_rope_paged(qkv, cache, positions, slots, HQ, cos, sin, q_norm=None, k_norm=None,
                       eps=1e-6, layer=0, out=None, status=None, stream=None):
    """Per-head norms (optional) and RoPE at positions[n] for the q and k heads of
    qkv [N, (HQ+2*HKV)*D]; returns the rotated q [N, HQ*D] and writes the k and v heads to slot
    slots[n] = page * page_size + offset of the cache's `layer` (-1: not written).  positions and
    slots int64 [N]; cos / sin bf16 [max_pos, D].  out may be the q columns of qkv and may not overlap it
    otherwise."""
    import torch
    what, dt, index, i64, bf = "qk_norm_rope_paged", cache.dtype, cache.index, torch.int64, torch.bfloat16
    if not _is(qkv, dt, index, 2):
        _refuse(what, "qkv", qkv, dt, 2)
    if not _is(positions, i64, index, 1):
        _refuse(what, "positions", positions, i64, 1)
    if not _is(slots, i64, index, 1):
        _refuse(what, "slots", slots, i64, 1)
    if not _is(cos, bf, index, 2):
        _refuse(what, "cos", cos, bf, 2)
    if not _is(sin, bf, index, 2):
        _refuse(what, "sin", sin, bf, 2)
    _check_layer(what, cache, layer)
    D = cache.head_dim
    N, width = qkv.shape
    if width != (HQ + 2 * cache.heads) * D:
        raise KrbError(f"{what}: qkv rows must hold (HQ + 2*HKV) * head_dim values")
    if positions.shape[0] != N or slots.shape[0] != N:
        raise KrbError(f"{what}: positions and slots must have one entry per row of qkv")
    max_pos, columns = cos.shape
    if columns != D or sin.shape != cos.shape or (max_pos > 1 and (cos.stride(0) != D or sin.stride(0) != D)):
        raise KrbError(f"{what}: cos and sin must be contiguous [max_pos, head_dim]")
    if q_norm is not None and not (_is(q_norm, bf, index, 1) and q_norm.shape[0] == D):
        _refuse(what, "q_norm [head_dim]", q_norm, bf, 1)
    if k_norm is not None and not (_is(k_norm, bf, index, 1) and k_norm.shape[0] == D):
        _refuse(what, "k_norm [head_dim]", k_norm, bf, 1)
    if status is not None and not (_is(status, torch.int32, index, 1) and len(status)):
        _refuse(what, "status [1]", status, torch.int32, 1)
    if out is not None and not (_is(out, dt, index, 2) and out.shape == (N, HQ * D)):
        _refuse(what, "out [N, HQ*head_dim]", out, dt, 2)
    if (on := _enter(cache)) is not None:
        with on:
            return qk_norm_rope_paged(qkv, cache, positions, slots, HQ, cos, sin, q_norm, k_norm,
                                      eps, layer, out, status, stream)
    if out is None:
        out = qkv.new_empty((N, HQ * D)) if stream is None else _empty((N, HQ * D), dt, qkv, stream)
    many = N > 1
    check(lib().krb_qk_norm_rope_paged(
        cache.ref, layer, qkv.data_ptr(), qkv.stride(0) if many else width, out.data_ptr(),
        out.stride(0) if many else HQ * D,
        positions.data_ptr(), slots.data_ptr(), N, HQ, cos.data_ptr(), sin.data_ptr(), max_pos,
        _addr(q_norm), _addr(k_norm), eps, _addr(status), _raw_stream(stream, index)), what)
    return out


def attention_paged(q, cache, page_table, kv_lens, q_starts, max_q, scale, mask=None, layer=0,
                    out=None, workspace=None, status=None, stream=None):
    """Attention of each sequence's new tokens (rows q_starts[b]:q_starts[b+1] of q [N, HQ*D],
    already appended) over its cached positions: all kv_lens[b] - T_b positions before them and,
    of the new ones, those up to itself (mask None) or those of its mask bits (int32 [N, words],
    bit j % 32 of word j / 32 for new token j; a tree of drafted tokens).  page_table int32
    [B, max_pages], kv_lens int32 [B], q_starts int32 [B+1], all on the device; max_q: no less
    than any T_b.  out may not overlap q.  Rows that belong to no sequence, and those of a sequence that
    the device refuses (status), are not written: in the default out, a fresh tensor, they hold
    whatever its memory held.  workspace: a uint8 tensor of cache.attention_workspace(HQ, max_q) bytes
    that no other call uses until this one is done (default: allocated per call).  stream: see KVCache."""
    import torch
    what, dt, index, i32 = "attention_paged", cache.dtype, cache.index, torch.int32
    if not _is(q, dt, index, 2):
        _refuse(what, "q", q, dt, 2)
    if not _is(page_table, i32, index, 2):
        _refuse(what, "page_table", page_table, i32, 2)
    if not _is(kv_lens, i32, index, 1):
        _refuse(what, "kv_lens", kv_lens, i32, 1)
    if not _is(q_starts, i32, index, 1):
        _refuse(what, "q_starts", q_starts, i32, 1)
    _check_layer(what, cache, layer)
    N, width = q.shape
    HQ = width // cache.head_dim
    if HQ * cache.head_dim != width:
        raise KrbError(f"{what}: q rows must hold HQ * head_dim values")
    B, max_pages = page_table.shape
    if kv_lens.shape[0] != B or q_starts.shape[0] != B + 1:
        raise KrbError(f"{what}: page_table, kv_lens and q_starts must be of the same batch")
    words = ldm = 0
    if mask is not None:
        if not _is(mask, i32, index, 2):
            _refuse(what, "mask", mask, i32, 2)
        rows, words = mask.shape
        if rows != N:
            raise KrbError(f"{what}: mask must have one row per row of q")
        if not words and N:  # a tensor without elements has no address: it would pass for no mask
            raise KrbError(f"{what}: mask must have words of 32 bits for max_q tokens")
        ldm = mask.stride(0) if N > 1 else words
    if status is not None and not (_is(status, i32, index, 1) and len(status)):
        _refuse(what, "status [1]", status, i32, 1)
    if out is not None and not (_is(out, dt, index, 2) and out.shape == q.shape):
        _refuse(what, "out [N, HQ*head_dim]", out, dt, 2)
    if workspace is not None and not _is(workspace, torch.uint8, index, 1):
        _refuse(what, "workspace", workspace, torch.uint8, 1)
    if (on := _enter(cache)) is not None:
        with on:
            return attention_paged(q, cache, page_table, kv_lens, q_starts, max_q, scale, mask,
                                   layer, out, workspace, status, stream)
    need = cache.attention_workspace(HQ, max_q) if N and B else 0
    many = N > 1
    if out is None:
        out = torch.empty_like(q) if stream is None else _empty((N, width), dt, q, stream)
    if workspace is None:
        workspace = _empty((need,), torch.uint8, q, stream)
    check(lib().krb_attention_paged(
        cache.ref, layer, q.data_ptr(), q.stride(0) if many else width, out.data_ptr(),
        out.stride(0) if many else width, N, HQ, page_table.data_ptr(),
        page_table.stride(0) if B > 1 else max_pages, max_pages, kv_lens.data_ptr(),
        q_starts.data_ptr(), B, max_q, _addr(mask), ldm, words, scale, workspace.data_ptr(),
        workspace.shape[0], _addr(status), _raw_stream(stream, index)), what)
    return out


def kv_copy_pages(cache, src, dst, stream=None):
    """Copy page src[i] to page dst[i], K and V of all layers (a fork's page of its own, or pages
    moved together).  src, dst: host sequences of page numbers (bytes, too, element by element); no
    page is written twice, or both read and written."""
    what, n = "kv_copy_pages", len(src)
    if len(dst) != n:
        raise KrbError(f"{what}: src and dst differ in length")
    if getattr(src, "is_cuda", False) or getattr(dst, "is_cuda", False):
        raise KrbError(f"{what}: src and dst must be host integers, not tensors on a GPU")
    try:
        # through a list: array() takes bytes-like objects for memory of its entries
        src, dst = (array("i", x.tolist() if hasattr(x, "tolist") else list(x)) for x in (src, dst))
    except (TypeError, OverflowError) as e:
        raise KrbError(f"{what}: src and dst must be host integers ({e})") from None
    if len(src) != n or len(dst) != n:
        raise KrbError(f"{what}: src and dst must be flat sequences of host integers")
    if (on := _enter(cache)) is not None:
        with on:
            return kv_copy_pages(cache, src, dst, stream)
    check(lib().krb_kv_copy_pages(cache.ref, src.buffer_info()[0], dst.buffer_info()[0], n,
                                  _raw_stream(stream, cache.index)), what)


def kv_commit(cache, page_table, bases, accepted, counts, status=None, stream=None):
    """Keep the accepted tokens of verified drafts: K and V of position bases[b] + accepted[b][i]
    move to position bases[b] + i for i < counts[b], all layers.  accepted int32 [B, A], ascending
    strictly from >= 0 per sequence; bases, counts int32 [B]; page_table as in attention_paged."""
    import torch
    what, index, i32 = "kv_commit", cache.index, torch.int32
    if not _is(page_table, i32, index, 2):
        _refuse(what, "page_table", page_table, i32, 2)
    if not _is(accepted, i32, index, 2):
        _refuse(what, "accepted", accepted, i32, 2)
    if not _is(bases, i32, index, 1):
        _refuse(what, "bases", bases, i32, 1)
    if not _is(counts, i32, index, 1):
        _refuse(what, "counts", counts, i32, 1)
    B, A = accepted.shape
    rows, max_pages = page_table.shape
    if rows != B or bases.shape[0] != B or counts.shape[0] != B:
        raise KrbError(f"{what}: page_table, bases, accepted and counts must be of the same batch")
    if status is not None and not (_is(status, i32, index, 1) and len(status)):
        _refuse(what, "status [1]", status, i32, 1)
    if (on := _enter(cache)) is not None:
        with on:
            return kv_commit(cache, page_table, bases, accepted, counts, status, stream)
    check(lib().krb_kv_commit(
        cache.ref, page_table.data_ptr(), page_table.stride(0) if B > 1 else max_pages, max_pages,
        bases.data_ptr(), accepted.data_ptr(), accepted.stride(0) if B > 1 else A, A, counts.data_ptr(), B, _addr(status),
        _raw_stream(stream, index)), what)


def relay_down_single(act, w_down, resid, gamma, tiles, eps, bn=0, status=None, stream=None):
    """resid fp32 [S,H] -> (sum fp32 [S,H], x bf16 [S,H])."""
    import torch
    S, K = act.shape
    H = w_down.shape[0]
    s = torch.empty((S, H), dtype=torch.float32, device=act.device)
    x = torch.empty((S, H), dtype=torch.bfloat16, device=act.device)
    check(lib().krb_relay_down_single(_ptr(act), _ptr(w_down), _ptr(resid), _ptr(gamma), _ptr(s),
                                      _ptr(x), S, H, K, tiles, eps, bn, _ptr(status),
                                      _stream(stream)), "relay_down_single")
    return s, x


def relay_down_single_noalloc(act, w_down, resid, gamma, tiles, eps, bn=0, status=None,
                              stream=None, out=None):
    """krb_relay_down_single_noalloc: same results as relay_down_single, no device
    allocation inside the library call (asynchronous on `stream`).  `out` may
    pass preallocated (sum fp32 [S,H], x bf16 [S,H])."""
    import torch
    S, K = act.shape
    H = w_down.shape[0]
    if out is None:
        out = (torch.empty((S, H), dtype=torch.float32, device=act.device),
               torch.empty((S, H), dtype=torch.bfloat16, device=act.device))
    s, x = out
    check(lib().krb_relay_down_single_noalloc(_ptr(act), _ptr(w_down), _ptr(resid), _ptr(gamma),
                                              _ptr(s), _ptr(x), S, H, K, tiles, eps, bn,
                                              _ptr(status), _stream(stream)),
          "relay_down_single_noalloc")
    return s, x


def synth_normal(name: str, seed: int, std: float, n: int, offset: int = 0, mean: float = 0.0):
    """bf16 bit pattern (uint16 numpy array) of a synthetic tensor (host, no GPU)."""
    import numpy as np
    out = np.empty(n, dtype=np.uint16)
    check(lib().krb_synth_normal_host(name.encode(), seed, std, mean, offset, n,
                                      out.ctypes.data_as(ctypes.c_void_p)), "synth")
    return out


def relay_timeout_probe(S, H, K, tiles, timeout_ms):
    """Status word of a relay whose only peer never runs (see kernrelay_b200.h)."""
    v = ctypes.c_uint32()
    check(lib().krb_relay_timeout_probe(S, H, K, tiles, timeout_ms, ctypes.byref(v)), "probe")
    return v.value


def relay_plan(S, H, tiles, k, rank, bn):
    buf = ctypes.create_string_buffer(1 << 16)
    rc = lib().krb_relay_plan(S, H, tiles, k, rank, bn, buf, len(buf))
    if rc != 0:
        raise KrbError(buf.value.decode(errors="replace"))
    return json.loads(buf.value.decode())


def plan_check(schedule_json):
    """Validate a schedule.json like kr_plan_run (no GPU needed); raises KrbError."""
    buf = ctypes.create_string_buffer(1 << 16)
    rc = lib().krb_plan_check(str(schedule_json).encode(), buf, len(buf))
    if rc != 0:
        raise KrbError(json.loads(buf.value.decode()).get("error", "plan check failed"))
    return json.loads(buf.value.decode())


# ---------------------------------------------------------------- per-rank engine
class Engine:
    """One rank of a prefill: owns its weights, activations and (split modes)
    its relay region.  For tp modes the ranks are wired with open_peers (split)
    or init_nccl (baseline) after all engines exist."""

    def __init__(self, model_dir, mode, seq, rank=0, world=1, device=0, tiles=4, _handle=None):
        h = _handle
        if h is None:
            h = c_void_p()
            check(lib().krb_engine_create(str(model_dir).encode(), mode.encode(), seq, rank, world,
                                          device, tiles, ctypes.byref(h)), "engine_create")
        self.h = h
        self.rank, self.world, self.device = rank, world, device

    @classmethod
    def microdag(cls, seq, hidden, intermediate, mode, rank=0, world=1, device=0, tiles=4,
                 seed=1234):
        """The isolated TP-MLP micro-DAG (krb_microdag_create): this rank's down GEMM over
        X_r, W_r, the reduction over the ranks and the Add+RMSNorm with R."""
        h = c_void_p()
        check(lib().krb_microdag_create(seq, hidden, intermediate, tiles, rank, world, device,
                                        mode.encode(), seed, ctypes.byref(h)), "microdag_create")
        return cls(None, mode, seq, rank=rank, world=world, device=device, tiles=tiles, _handle=h)

    def final_hidden(self):
        """fp32 [S, H] residual after the last layer (micro-DAG: h = R + sum of partials)."""
        import numpy as np
        info = self.info()
        n = info["seq"] * info["H"]
        out = np.empty(n, dtype=np.float32)
        check(lib().krb_engine_final_hidden(self.h, out.ctypes.data_as(c_void_p), n), "final_hidden")
        return out.reshape(info["seq"], info["H"])

    def final_x(self):
        """fp16 [S, H] final normed rows as fp32 numpy (micro-DAG: x = RMSNorm(h))."""
        import numpy as np
        info = self.info()
        n = info["seq"] * info["H"]
        out = np.empty(n, dtype=np.float16)
        check(lib().krb_engine_final_x(self.h, out.ctypes.data_as(c_void_p), n), "final_x")
        return out.astype(np.float32).reshape(info["seq"], info["H"])

    def close(self):
        if self.h:
            lib().krb_engine_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def ipc_handle(self) -> bytes:
        buf = ctypes.create_string_buffer(64)
        check(lib().krb_engine_ipc_handle(self.h, buf, 64), "ipc_handle")
        return buf.raw

    def open_peers(self, handles: list[bytes]):
        blob = b"".join(handles)
        buf = ctypes.create_string_buffer(blob, len(blob))
        check(lib().krb_engine_open_peers(self.h, buf, len(blob)), "open_peers")

    @staticmethod
    def nccl_unique_id() -> bytes:
        buf = ctypes.create_string_buffer(128)
        check(lib().krb_nccl_unique_id(buf, 128), "nccl_unique_id")
        return buf.raw

    def init_nccl(self, uid: bytes):
        buf = ctypes.create_string_buffer(uid, len(uid))
        check(lib().krb_engine_init_nccl(self.h, buf, len(uid)), "init_nccl")

    @staticmethod
    def link(engines):
        arr = (c_void_p * len(engines))(*[e.h for e in engines])
        check(lib().krb_engines_link(arr, len(engines)), "engines_link")

    @staticmethod
    def init_nccl_all(engines):
        arr = (c_void_p * len(engines))(*[e.h for e in engines])
        check(lib().krb_engines_init_nccl(arr, len(engines)), "engines_init_nccl")

    def capture(self):
        check(lib().krb_engine_capture(self.h), "capture")

    def run(self):
        check(lib().krb_engine_run(self.h), "run")

    def run_host(self, ids_pinned, logits_pinned):
        check(lib().krb_engine_run_host(self.h, c_void_p(ids_pinned.data_ptr()),
                                        None if logits_pinned is None else
                                        c_void_p(logits_pinned.data_ptr())), "run_host")

    def sync(self):
        check(lib().krb_engine_sync(self.h), "sync")

    def stream_ptr(self) -> int:
        p = c_void_p()
        check(lib().krb_engine_stream(self.h, ctypes.byref(p)), "stream")
        return p.value or 0

    def status(self) -> int:
        v = ctypes.c_uint32()
        check(lib().krb_engine_status(self.h, ctypes.byref(v)), "status")
        return v.value

    def _json(self, fn, cap=1 << 16):
        buf = ctypes.create_string_buffer(cap)
        rc = fn(self.h, buf, cap)
        if rc != 0:
            raise KrbError(buf.value.decode(errors="replace"))
        return json.loads(buf.value.decode())

    def stage_times(self):
        return self._json(lib().krb_engine_stage_times)

    def verify(self):
        return self._json(lib().krb_engine_verify)

    def info(self):
        return self._json(lib().krb_engine_info)

    def last_logits(self):
        import numpy as np
        n = self.info()["V"]
        out = np.empty(n, dtype=np.float32)
        check(lib().krb_engine_last_logits(self.h, out.ctypes.data_as(c_void_p), n), "last_logits")
        return out

    TRACE_SLOTS = 48  # kTraceSlots in csrc/relay.cuh

    def relay_trace(self):
        """[grid, 48] globaltimer stamps of the last relay launch (KRB_RELAY_TRACE=1);
        slot meanings in csrc/relay.cuh (kTraceSlots)."""
        import numpy as np
        out = np.zeros(4096 * self.TRACE_SLOTS, dtype=np.uint64)
        n = c_size_t()
        check(lib().krb_engine_relay_trace(self.h, out.ctypes.data_as(c_void_p), out.size,
                                           ctypes.byref(n)), "relay_trace")
        return out[: n.value].reshape(-1, self.TRACE_SLOTS) if n.value else None

    def layer_dump(self, on=True):
        check(lib().krb_engine_layer_dump(self.h, 1 if on else 0), "layer_dump")

    def layer_hidden(self, layer):
        """fp32 residual stream after `layer` as numpy [S, H]."""
        import numpy as np
        info = self.info()
        n = info["seq"] * info["H"]
        out = np.empty(n, dtype=np.float32)
        check(lib().krb_engine_layer_hidden(self.h, layer, out.ctypes.data_as(c_void_p), n),
              "layer_hidden")
        return out.reshape(info["seq"], info["H"])
