"""Python host layer over libkq's C ABI (include/kq.h).

Mirrors the reference's per-kernel call surface: the parameter structs
(GemvParams int4-gemv/src/kernels.metal:42-49, VQParams
vq-gemv/src/kernels.metal:32-37, MoEParams moe-fused/src/kernels.metal:22-35)
and one call per hot-path kernel, taking device buffers. Buffers are torch
tensors on the GPU (torch is only the allocator/stream provider here) or raw
device addresses (int). Every call goes through libkq; there is no fallback:
if the library is missing or a call fails, a KQError is raised.
"""
import ctypes as C
import os
import struct
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "_lib", "libkq.so")

KQ_OK, KQ_EINVAL, KQ_ENULL, KQ_EALIGN, KQ_EUNSUPPORTED, KQ_EWORKSPACE, KQ_EHIP = range(7)
F16, BF16, F32 = 0, 1, 2
PATH_AUTO, PATH_VALU, PATH_MFMA, PATH_SCALAR = 0, 1, 2, 3
MOE_PATH_AUTO, MOE_PATH_LAUNCHES, MOE_PATH_ONE, MOE_PATH_ATOMIC = 0, 1, 2, 3  # KQ_MOE_PATH_*
MOE_WS_ERR_OFFSET = 128  # KQ_MOE_WS_ERR_OFFSET

# every symbol include/kq.h declares
EXPORTS = ("kq_status_str", "kq_last_hip_error", "kq_version", "kq_int4_gemv",
           "kq_int4_gemv_path", "kq_int4_gemv_cfg", "kq_xsum32", "kq_stream_read",
           "kq_stream_read_cfg", "kq_stream_read_out",
           "kq_vq_gemv", "kq_moe_default_desc", "kq_moe_workspace_size",
           "kq_moe_workspace_init", "kq_moe_workspace_error", "kq_moe_router_topk", "kq_moe_gate_up_swiglu",
           "kq_moe_down_combine", "kq_moe_block", "kq_moe_block_path", "kq_moe_block_noalloc",
           "kq_moe_unfused_workspace_size",
           "kq_moe_block_unfused", "kq_vq_quantize_workspace_size", "kq_vq_quantize",
           "kq_kv_write", "kq_kv_read", "kq_kv_attn_workspace_size", "kq_kv_attn",
           "kq_rope_freqs", "kq_rope", "kq_kv_write_rope",
           "kq_kv_tree", "kq_kv_attn_tree_workspace_size", "kq_kv_attn_tree",
           "kq_draft_verify_workspace_size", "kq_draft_verify", "kq_kv_keep")


class KQError(RuntimeError):
    def __init__(self, status, where):
        self.status = status
        msg = lib().kq_status_str(status).decode()
        if status == KQ_EHIP:
            msg += f" (hipError {lib().kq_last_hip_error()})"
        super().__init__(f"{where}: {msg} [kq_status {status}]")


class MoEDesc(C.Structure):
    """kq_moe_desc: MoEParams without its derived fields."""
    _fields_ = [("hidden", C.c_uint32), ("inter", C.c_uint32), ("n_experts", C.c_uint32),
                ("top_k", C.c_uint32), ("blob", C.c_uint64), ("off_gate", C.c_uint64),
                ("off_up", C.c_uint64), ("off_down", C.c_uint64), ("sub_w", C.c_uint64),
                ("sub_s", C.c_uint64), ("sub_b", C.c_uint64), ("sub_bi", C.c_uint64)]

    def as_dict(self):
        return {f: getattr(self, f) for f, _ in self._fields_}


class _KVCacheC(C.Structure):
    """kq_kv_cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_exp", C.c_void_p), ("v_exp", C.c_void_p),
                ("type", C.c_uint32), ("n_pages", C.c_uint32), ("page", C.c_uint32),
                ("block", C.c_uint32), ("heads", C.c_uint32), ("head_dim", C.c_uint32)]


class _KVBatchC(C.Structure):
    """kq_kv_batch."""
    _fields_ = [("pages", C.c_void_p), ("kv_len", C.c_void_p), ("q_start", C.c_void_p),
                ("n_seq", C.c_uint32), ("max_pages", C.c_uint32), ("max_q", C.c_uint32),
                ("n_rows", C.c_uint32), ("max_len", C.c_uint32)]


class _KVRowsC(C.Structure):
    """kq_kv_rows."""
    _fields_ = [("p", C.c_void_p), ("row", C.c_int64), ("head", C.c_int64)]


class _KVAttnC(C.Structure):
    """kq_kv_attn_desc."""
    _fields_ = [("q_heads", C.c_uint32), ("scale", C.c_float), ("causal", C.c_uint32),
                ("window", C.c_uint32), ("sinks", C.c_void_p)]


class _KVNodesC(C.Structure):
    """kq_kv_nodes."""
    _fields_ = [("mask", C.c_void_p), ("pos", C.c_void_p), ("words", C.c_uint32)]


class _RopeC(C.Structure):
    """kq_rope_desc."""
    _fields_ = [("inv_freq", C.c_void_p), ("rot", C.c_uint32), ("layout", C.c_uint32),
                ("amplitude", C.c_double), ("inverse", C.c_uint32)]


class _RopeScalingC(C.Structure):
    """kq_rope_scaling."""
    _fields_ = [("kind", C.c_uint32), ("rot", C.c_uint32), ("base", C.c_double), ("factor", C.c_double),
                ("low", C.c_double), ("high", C.c_double), ("original", C.c_double)]


_lib = None


def lib():
    """Load libkq.so. Raises if it was not built: there is no CPU fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"libkq not built: {LIB_PATH} is missing "
                               "(run __graft_entry__.build() or kernels_amd/build.py)")
        L = C.CDLL(LIB_PATH)
        vp, u32, i32, sz = C.c_void_p, C.c_uint32, C.c_int, C.c_size_t
        L.kq_status_str.argtypes = [i32]
        L.kq_status_str.restype = C.c_char_p
        L.kq_last_hip_error.restype = i32
        L.kq_version.restype = C.c_char_p
        L.kq_int4_gemv.argtypes = [vp, vp, vp, i32, vp, vp, i32, u32, u32, u32, u32, vp]
        L.kq_int4_gemv_path.argtypes = [vp, vp, vp, i32, vp, vp, i32, u32, u32, u32, u32, i32, vp]
        L.kq_int4_gemv_cfg.argtypes = [vp, vp, vp, i32, vp, vp, i32, u32, u32, u32, u32, i32,
                                       i32, i32, vp]
        L.kq_xsum32.argtypes = [vp, vp, u32, u32, vp]
        L.kq_stream_read.argtypes = [vp, sz, vp, vp]
        L.kq_stream_read_cfg.argtypes = [vp, sz, vp, u32, u32, vp]
        L.kq_stream_read_out.argtypes = [vp, sz, vp, u32, u32, u32, vp]
        L.kq_vq_gemv.argtypes = [vp, vp, vp, vp, vp, i32, u32, u32, u32, u32, u32, vp]
        L.kq_moe_default_desc.argtypes = [C.POINTER(MoEDesc)]
        L.kq_moe_default_desc.restype = None
        L.kq_moe_workspace_size.argtypes = [C.POINTER(MoEDesc), u32]
        L.kq_moe_workspace_size.restype = sz
        L.kq_moe_workspace_init.argtypes = [vp, sz, vp]
        L.kq_moe_workspace_error.argtypes = [vp, sz, C.POINTER(u32), i32, vp]
        L.kq_moe_router_topk.argtypes = [vp, i32, vp, i32, u32, C.POINTER(MoEDesc), vp, vp, vp,
                                         vp, sz, vp]
        L.kq_moe_gate_up_swiglu.argtypes = [vp, C.POINTER(MoEDesc), vp, vp, vp, u32, vp, sz, vp]
        L.kq_moe_down_combine.argtypes = [vp, C.POINTER(MoEDesc), vp, vp, vp, vp, i32, u32, vp,
                                          sz, vp]
        L.kq_moe_block.argtypes = [vp, C.POINTER(MoEDesc), vp, i32, vp, i32, u32, vp, vp, vp, vp,
                                   vp, i32, vp, sz, vp]
        L.kq_moe_block_path.argtypes = [vp, C.POINTER(MoEDesc), vp, i32, vp, i32, u32, vp, vp, vp,
                                        vp, vp, i32, vp, sz, i32, vp]
        L.kq_moe_block_noalloc.argtypes = [vp, C.POINTER(MoEDesc), vp, i32, vp, i32, u32, vp, vp,
                                           vp, vp, vp, i32, vp]
        L.kq_moe_unfused_workspace_size.argtypes = [C.POINTER(MoEDesc)]
        L.kq_moe_unfused_workspace_size.restype = sz
        L.kq_moe_block_unfused.argtypes = [vp, C.POINTER(MoEDesc), vp, i32, vp, i32, u32, vp, vp,
                                           vp, vp, vp, i32, vp, sz, C.POINTER(u32), vp]
        L.kq_vq_quantize_workspace_size.argtypes = [u32, u32, u32, u32, u32]
        L.kq_vq_quantize_workspace_size.restype = sz
        L.kq_vq_quantize.argtypes = [vp, i32, u32, u32, u32, u32, u32, u32, C.c_uint64, vp, vp,
                                     vp, vp, sz, vp]
        # the structs of the key/value cache's calls: by reference, or packed (bytes)
        L.kq_kv_write.argtypes = [vp, vp, vp, vp, i32, vp]
        L.kq_kv_read.argtypes = [vp, vp, vp, vp, i32, vp]
        L.kq_kv_attn_workspace_size.argtypes = [vp, vp, u32]
        L.kq_kv_attn_workspace_size.restype = sz
        L.kq_kv_attn.argtypes = [vp, vp, vp, vp, vp, i32, vp, vp, sz, vp]
        L.kq_rope_freqs.argtypes = [C.POINTER(_RopeScalingC), vp, C.POINTER(C.c_double)]
        L.kq_rope.argtypes = [vp, vp, vp, vp, u32, u32, u32, i32, vp]
        L.kq_kv_write_rope.argtypes = [vp, vp, vp, vp, vp, vp, u32, vp, vp, i32, vp]
        L.kq_kv_tree.argtypes = [vp, vp, vp, u32, vp, u32, vp]
        L.kq_kv_attn_tree_workspace_size.argtypes = [vp, vp, u32]
        L.kq_kv_attn_tree_workspace_size.restype = sz
        L.kq_kv_attn_tree.argtypes = [vp, vp, vp, vp, vp, vp, i32, vp, vp, sz, vp]
        L.kq_draft_verify_workspace_size.argtypes = [u32, u32, u32]
        L.kq_draft_verify_workspace_size.restype = sz
        L.kq_draft_verify.argtypes = [vp, vp, vp, vp, vp, sz, vp]
        L.kq_kv_keep.argtypes = [vp, vp, vp, vp, vp]
        for name in EXPORTS:
            if name not in ("kq_status_str", "kq_last_hip_error", "kq_version",
                            "kq_moe_default_desc", "kq_moe_workspace_size",
                            "kq_moe_unfused_workspace_size", "kq_vq_quantize_workspace_size",
                            "kq_kv_attn_workspace_size", "kq_kv_attn_tree_workspace_size",
                            "kq_draft_verify_workspace_size"):
                getattr(L, name).restype = i32
        _lib = L
    return _lib


def _ptr(t):
    """Device address of a torch tensor (or an int address, or None)."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_current = None  # (raw stream of a device, current device): torch's own, without a Stream object


def _stream(stream):
    if stream is None:
        global _current
        if _current is None:
            import torch
            torch.cuda.init()
            _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        return _current[0](_current[1]())
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _check(st, where):
    if st != KQ_OK:
        raise KQError(st, where)


_dtypes = None


def _dt(t):
    global _dtypes
    if _dtypes is None:
        import torch
        _dtypes = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
    return _dtypes[t.dtype]


# ---------------------------------------------------------------------------
# int4 GEMV
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class GemvParams:
    """GemvParams (int4-gemv/src/kernels.metal:42-49); derived fields are
    properties, validated by the library (K % 32, G in {32,64,128})."""
    M: int
    K: int
    G: int = 64

    @property
    def words_pr(self):
        return self.K // 8

    @property
    def groups_pr(self):
        return self.K // self.G

    @property
    def chunks_pg(self):
        return self.G // 32


def int4_gemv(W, SB, x, y, P: GemvParams, B=None, batch=1, sb_dtype=F16, path=PATH_AUTO,
              stream=None, rows=0, unroll=0):
    """y = dequant(W, SB[, B]) . x  (y: [batch][M], fp16 or fp32 by tensor dtype).

    SB alone = interleaved (scale, bias) pairs (the v4-v6 layout,
    int4-gemv/src/main.mm:198-199); SB and B = separate scale and bias arrays
    (the v0-v3 layout). rows/unroll > 0 forces the launch shape."""
    ydt = y if isinstance(y, int) else _dt(y)
    if isinstance(y, int):
        raise TypeError("pass y as a tensor so its dtype is known")
    s = _stream(stream)
    if rows or unroll:
        st = lib().kq_int4_gemv_cfg(_ptr(W), _ptr(SB), _ptr(B), sb_dtype, _ptr(x), _ptr(y), ydt,
                                    P.M, P.K, P.G, batch, path, rows, unroll, s)
    elif path != PATH_AUTO:
        st = lib().kq_int4_gemv_path(_ptr(W), _ptr(SB), _ptr(B), sb_dtype, _ptr(x), _ptr(y), ydt,
                                     P.M, P.K, P.G, batch, path, s)
    else:
        st = lib().kq_int4_gemv(_ptr(W), _ptr(SB), _ptr(B), sb_dtype, _ptr(x), _ptr(y), ydt,
                                P.M, P.K, P.G, batch, s)
    _check(st, "kq_int4_gemv")


def xsum32(x, xs, K, batch=1, stream=None):
    _check(lib().kq_xsum32(_ptr(x), _ptr(xs), K, batch, _stream(stream)), "kq_xsum32")


def stream_read(src, nbytes, sink, stream=None, unroll=0, threads=0):
    """Streaming-read ceiling; unroll/threads > 0 set the launch shape of the
    reference's sweep (int4-gemv/src/main.mm:294-334)."""
    if unroll or threads:
        _check(lib().kq_stream_read_cfg(_ptr(src), nbytes, _ptr(sink), unroll, threads,
                                        _stream(stream)), "kq_stream_read_cfg")
    else:
        _check(lib().kq_stream_read(_ptr(src), nbytes, _ptr(sink), _stream(stream)),
               "kq_stream_read")


def stream_read_out(src, nbytes, out, out_elems, unroll, threads, stream=None):
    """The streaming read, then out_elems 2-byte values written across the
    grid (a GEMV's output store): the ceiling of a kernel that stores y."""
    _check(lib().kq_stream_read_out(_ptr(src), nbytes, _ptr(out), out_elems, unroll, threads,
                                    _stream(stream)), "kq_stream_read_out")


# ---------------------------------------------------------------------------
# VQ GEMV
# ---------------------------------------------------------------------------
@dataclass(frozen=True)
class VQParams:
    """VQParams (vq-gemv/src/kernels.metal:32-37) plus the two format knobs:
    rows_per_cb (codebook block height; M = one codebook per matrix, the
    reference) and scale_group (32 = the reference; K = one scale per row)."""
    M: int
    K: int
    rows_per_cb: int
    scale_group: int = 32
    cb_size: int = 256

    @property
    def chunks_pr(self):
        return self.K // 32


def vq_gemv(IDX, Cb, S, x, y, P: VQParams, batch=1, stream=None):
    _check(lib().kq_vq_gemv(_ptr(IDX), _ptr(Cb), _ptr(S), _ptr(x), _ptr(y), _dt(y), P.M, P.K,
                            P.rows_per_cb, P.scale_group, batch, _stream(stream)), "kq_vq_gemv")


def vq_quantize_workspace_size(M, K, rows_per_cb, scale_group, sample=200_000):
    n = lib().kq_vq_quantize_workspace_size(M, K, rows_per_cb, scale_group, sample)
    if n == 0:
        raise KQError(KQ_EINVAL, "kq_vq_quantize_workspace_size")
    return n


def vq_quantize(W, IDX, Cb, S, M, K, rows_per_cb, scale_group, ws, ws_bytes, iters=25,
                sample=200_000, seed=0, w_dtype=None, stream=None):
    """quantize_matrix (vq-gemv/quant/pq_quantize.py:28-83) on the GPU: W
    [M][K] (float32, float16 or bfloat16 tensor) into IDX u8 [M][K/2], Cb
    fp16 [blocks][256][2] and S fp16 [M][K/scale_group]."""
    _check(lib().kq_vq_quantize(_ptr(W), _dt(W) if w_dtype is None else w_dtype, M, K,
                                rows_per_cb, scale_group, iters, sample, seed, _ptr(IDX),
                                _ptr(Cb), _ptr(S), _ptr(ws), ws_bytes, _stream(stream)),
           "kq_vq_quantize")


# ---------------------------------------------------------------------------
# MoE block
# ---------------------------------------------------------------------------
def moe_default_desc():
    d = MoEDesc()
    lib().kq_moe_default_desc(C.byref(d))
    return d


def moe_workspace_size(desc, batch):
    n = lib().kq_moe_workspace_size(C.byref(desc), batch)
    if n == 0:
        raise KQError(KQ_EINVAL, "kq_moe_workspace_size")
    return n


def moe_workspace_init(ws, nbytes, stream=None):
    _check(lib().kq_moe_workspace_init(_ptr(ws), nbytes, _stream(stream)), "kq_moe_workspace_init")


def moe_workspace_error(ws, nbytes, clear=False, stream=None):
    """The workspace's error word after the stream's earlier work (synchronises
    the stream); non-zero: a one-launch block on it gave up waiting."""
    v = C.c_uint32(0)
    _check(lib().kq_moe_workspace_error(_ptr(ws), nbytes, C.byref(v), int(bool(clear)),
                                        _stream(stream)), "kq_moe_workspace_error")
    return v.value


def moe_router_topk(R, x, idx, wgt, desc, ws, ws_bytes, batch=1, xh=None, stream=None):
    _check(lib().kq_moe_router_topk(_ptr(R), _dt(R), _ptr(x), _dt(x), batch, C.byref(desc),
                                    _ptr(idx), _ptr(wgt), _ptr(xh), _ptr(ws), ws_bytes,
                                    _stream(stream)), "kq_moe_router_topk")


def moe_gate_up_swiglu(pool, desc, idx, xh, H, ws, ws_bytes, batch=1, stream=None):
    _check(lib().kq_moe_gate_up_swiglu(_ptr(pool), C.byref(desc), _ptr(idx), _ptr(xh), _ptr(H),
                                       batch, _ptr(ws), ws_bytes, _stream(stream)),
           "kq_moe_gate_up_swiglu")


def moe_down_combine(pool, desc, idx, wgt, H, y, ws, ws_bytes, batch=1, stream=None):
    _check(lib().kq_moe_down_combine(_ptr(pool), C.byref(desc), _ptr(idx), _ptr(wgt), _ptr(H),
                                     _ptr(y), _dt(y), batch, _ptr(ws), ws_bytes, _stream(stream)),
           "kq_moe_down_combine")


def moe_block(pool, desc, R, x, idx, wgt, H, y, ws, ws_bytes, batch=1, xh=None, stream=None,
              path=None):
    """encodeFused (moe-fused/src/main.mm:176-206): router_topk ->
    gate_up_swiglu -> down_combine on one stream. path (MOE_PATH_*): the
    launch structure (None: kq_moe_block, the same as MOE_PATH_AUTO);
    MOE_PATH_ATOMIC is the reference's atomic sum(h) form at 1-2 tokens
    (moe-fused/src/kernels.metal:400-487)."""
    if path is None:
        _check(lib().kq_moe_block(_ptr(pool), C.byref(desc), _ptr(R), _dt(R), _ptr(x), _dt(x),
                                  batch, _ptr(idx), _ptr(wgt), _ptr(xh), _ptr(H), _ptr(y), _dt(y),
                                  _ptr(ws), ws_bytes, _stream(stream)), "kq_moe_block")
    else:
        _check(lib().kq_moe_block_path(_ptr(pool), C.byref(desc), _ptr(R), _dt(R), _ptr(x),
                                       _dt(x), batch, _ptr(idx), _ptr(wgt), _ptr(xh), _ptr(H),
                                       _ptr(y), _dt(y), _ptr(ws), ws_bytes, path,
                                       _stream(stream)), "kq_moe_block_path")


MOE_NOALLOC_WS_BYTES = 1 << 20  # KQ_MOE_NOALLOC_WS_BYTES


def moe_block_noalloc(pool, desc, R, x, idx, wgt, H, y, batch=1, xh=None, stream=None):
    """moe_block on libkq's per-GPU static workspace: no allocation, no
    workspace argument (no reference counterpart; for callers that cannot
    allocate). Calls that overlap on one GPU race."""
    _check(lib().kq_moe_block_noalloc(_ptr(pool), C.byref(desc), _ptr(R), _dt(R), _ptr(x), _dt(x),
                                      batch, _ptr(idx), _ptr(wgt), _ptr(xh), _ptr(H), _ptr(y),
                                      _dt(y), _stream(stream)), "kq_moe_block_noalloc")


def moe_unfused_workspace_size(desc):
    n = lib().kq_moe_unfused_workspace_size(C.byref(desc))
    if n == 0:
        raise KQError(KQ_EINVAL, "kq_moe_unfused_workspace_size")
    return n


def moe_block_unfused(pool, desc, R, x, idx, wgt, H, y, ws, ws_bytes, batch=1, xh=None,
                      stream=None):
    """encodeUnfused (moe-fused/src/main.mm:208-284): the block one operation
    per launch. Returns the number of kernel launches it made."""
    n = C.c_uint32(0)
    _check(lib().kq_moe_block_unfused(_ptr(pool), C.byref(desc), _ptr(R), _dt(R), _ptr(x), _dt(x),
                                      batch, _ptr(idx), _ptr(wgt), _ptr(xh), _ptr(H), _ptr(y),
                                      _dt(y), _ptr(ws), ws_bytes, C.byref(n), _stream(stream)),
           "kq_moe_block_unfused")
    return n.value


# ---------------------------------------------------------------------------
# 8-bit key/value cache, and the attention that reads it
# ---------------------------------------------------------------------------
KV_I8, KV_E4M3 = 0, 1  # kq_kv_type

# kq_kv_batch, kq_kv_rows, kq_kv_attn_desc and kq_draft as bytes: a call makes up to four of them, and a
# ctypes.Structure costs several times as much
_pack_batch, _pack_rows, _pack_attn, _pack_draft = (struct.Struct("@" + f).pack for f in ("3P5I4x", "Pqq", "If2IP", "2P2q5P5I4x"))


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _here(t, dtype, shape, what):
    """t: a contiguous tensor of this type and shape."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")


class KVCache:
    """kq_kv_cache over four contiguous tensors, kept alive with it:

    k [n_pages][heads][page][head_dim] and v [n_pages][heads][page/16][head_dim][16]
    of torch.int8 or torch.float8_e4m3fn, k_exp and v_exp uint8
    [n_pages][heads][page/block]: a code c stands for c * 2^(exp - 127)."""

    def __init__(self, k, v, k_exp, v_exp):
        import torch
        types = {torch.int8: KV_I8, torch.float8_e4m3fn: KV_E4M3}
        _need(k.dtype in types, f"k: int8 or float8_e4m3fn, not {k.dtype}")
        _need(k.dim() == 4 and k_exp.dim() == 3, "k: [n_pages][heads][page][head_dim], "
              "k_exp: [n_pages][heads][page/block]")
        n, heads, page, dim = k.shape
        blocks = k_exp.shape[2]
        _need(blocks and page % blocks == 0 and page % 16 == 0, "k_exp: [n_pages][heads][page/block]")
        _here(k, k.dtype, k.shape, "k")
        _here(v, k.dtype, (n, heads, page // 16, dim, 16), "v")
        _here(k_exp, torch.uint8, (n, heads, blocks), "k_exp")
        _here(v_exp, torch.uint8, (n, heads, blocks), "v_exp")
        _need(len({t.device for t in (k, v, k_exp, v_exp)}) == 1, "the cache's tensors are on one device")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device = k.get_device()
        self.heads, self.head_dim, self.page, self.block = heads, dim, page, page // blocks
        self.scale = dim ** -0.5
        self._c = _KVCacheC(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), types[k.dtype],
                            n, page, page // blocks, heads, dim)
        self._ref = C.byref(self._c)


def kv_cache(n_pages, heads, head_dim, page=16, block=16, dtype=None, device=None):
    """A new KVCache of zeros (dtype: torch.int8, the default, or torch.float8_e4m3fn)."""
    import torch
    _need(page % 16 == 0 and block > 0 and page % block == 0, "page: a multiple of block and of 16")
    dtype, device = dtype or torch.int8, device or "cuda"
    codes = [torch.zeros(s, dtype=torch.int8, device=device).view(dtype)
             for s in ((n_pages, heads, page, head_dim), (n_pages, heads, page // 16, head_dim, 16))]
    exps = [torch.full((n_pages, heads, page // block), 63, dtype=torch.uint8, device=device)
            for _ in range(2)]
    return KVCache(*codes, *exps)


class KVBatch:
    """kq_kv_batch: the sequences of a step, as every layer's calls take them.

    pages int32 [n_seq][max_pages], kv_len int32 [n_seq] (the step's tokens
    included), q_start int32 [n_seq + 1] or None (max_q rows each); max_len and
    max_q are the host's bounds. The tensors may be refilled between calls."""

    def __init__(self, pages, kv_len, max_len, q_start=None, max_q=1):
        import torch
        _need(pages.dim() == 2 and kv_len.dim() == 1, "pages: [n_seq][max_pages], kv_len: [n_seq]")
        n = kv_len.shape[0]
        _here(pages, torch.int32, (n, pages.shape[1]), "pages")
        _here(kv_len, torch.int32, (n,), "kv_len")
        if q_start is not None:
            _here(q_start, torch.int32, (n + 1,), "q_start")
        _need(0 <= max_len < 2**32 and 0 <= max_q < 2**32, "max_len, max_q: 32-bit")
        _need(len({t.device for t in (pages, kv_len, q_start) if t is not None}) == 1,
              "the batch's tensors are on one device")
        self.pages, self.kv_len, self.q_start = pages, kv_len, q_start
        self.device, self.n_seq, self.max_q, self.max_len = pages.get_device(), n, max_q, max_len
        self._args = (_ptr(pages), _ptr(kv_len), _ptr(q_start) or 0, n, pages.shape[1], max_q)

    def _packed(self, rows):
        return _pack_batch(*self._args, rows, self.max_len)


def _kv_rows(t, shape, dtype, what):
    """kq_kv_rows of a tensor of this shape [rows][heads][head_dim] and type."""
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{what}: a {dtype} tensor {tuple(shape)}, not {t.dtype} {tuple(t.shape)}")
    row, head, one = t.stride()
    if one != 1 and shape[0]:
        raise ValueError(f"{what}: contiguous in its last dimension, not strides {t.stride()}")
    return _pack_rows(t.data_ptr(), row, head)


def _kv_call(cache, batch, stream, *tensors):
    """The call's stream; refuses tensors of another device than the current one, whose stream it is."""
    s = _stream(stream)
    if _current is None:
        _stream(None)
    d = _current[1]()
    if cache.device != d or batch.device != d:
        raise ValueError(f"the cache and the batch are on the current device ({d})")
    for t in tensors:
        if t is not None and t.get_device() != d:
            raise ValueError(f"every tensor of the call is on the current device ({d})")
    return s


def _kv_move(f, where, cache, batch, k, v, stream):
    s = _kv_call(cache, batch, stream, k, v)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or shape[1] != cache.heads or shape[2] != cache.head_dim:
        raise ValueError(f"k: [n_rows][{cache.heads}][{cache.head_dim}], not {tuple(shape)}")
    a, b = _kv_rows(k, shape, dtype, "k"), _kv_rows(v, shape, dtype, "v")
    _check(f(cache._ref, batch._packed(shape[0]), a, b, _dt(k), s), where)


def kv_write(cache, batch, k, v, stream=None):
    """The newest tokens' keys and values [n_rows][heads][head_dim] (float16 or
    bfloat16, any row and head strides) into the cache."""
    _kv_move(lib().kq_kv_write, "kq_kv_write", cache, batch, k, v, stream)


def kv_read(cache, batch, k, v, stream=None):
    """The batch's newest tokens out of the cache into k and v
    [n_rows][heads][head_dim] (float16, bfloat16 or float32)."""
    _kv_move(lib().kq_kv_read, "kq_kv_read", cache, batch, k, v, stream)


def _kv_attn_size(f, where, cache, batch, q_heads):
    rows = 0 if batch.q_start is not None else min(batch.n_seq * batch.max_q, 2**32 - 1)  # with q_start any number
    n = f(cache._ref, batch._packed(rows), q_heads)
    if n == 0:
        raise KQError(KQ_EINVAL, where)
    return n


def kv_attn_workspace_size(cache, batch, q_heads):
    return _kv_attn_size(lib().kq_kv_attn_workspace_size, "kq_kv_attn_workspace_size", cache, batch, q_heads)


def _kv_attn(f, where, cache, batch, nodes, q, out, ws, ws_bytes, scale, causal, window, sinks, lse, stream):
    s = _kv_call(cache, batch, stream, q, out, sinks, lse, None if isinstance(ws, int) else ws)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError(f"q: [n_rows][q_heads][{cache.head_dim}], not {tuple(shape)}")
    rows, q_heads, _ = shape
    a, b = _kv_rows(q, shape, dtype, "q"), _kv_rows(out, shape, dtype, "out")
    if sinks is not None and (_dt(sinks) != F32 or sinks.shape != (q_heads,) or not sinks.is_contiguous()):
        raise ValueError(f"sinks: a contiguous float32 tensor [{q_heads}]")
    if lse is not None and (_dt(lse) != F32 or lse.shape != (rows, q_heads) or not lse.is_contiguous()):
        raise ValueError(f"lse: a contiguous float32 tensor [{rows}][{q_heads}]")
    if not 0 <= window < 2**32:
        raise ValueError("window: 32-bit")
    d = _pack_attn(q_heads, cache.scale if scale is None else scale, bool(causal), window, _ptr(sinks) or 0)
    _check(f(cache._ref, batch._packed(rows), d, *nodes, a, b, _dt(q), _ptr(lse), _ptr(ws), ws_bytes, s), where)


def kv_attn(cache, batch, q, out, ws, ws_bytes, scale=None, causal=True, window=0, sinks=None, lse=None,
            stream=None):
    """Attention of the rows q [n_rows][q_heads][head_dim] over their sequences in
    the cache, into out (float16 or bfloat16 both). scale: None is
    1 / sqrt(head_dim). window > 0: a row sees its own and the window - 1 tokens
    before. sinks: float32 [q_heads]. lse: float32 [n_rows][q_heads], written."""
    _kv_attn(lib().kq_kv_attn, "kq_kv_attn", cache, batch, (), q, out, ws, ws_bytes, scale, causal, window, sinks, lse, stream)


# ---------------------------------------------------------------------------
# Trees of drafted tokens
# ---------------------------------------------------------------------------
class KVTree:
    """kq_kv_nodes over contiguous tensors, kept alive with it: mask int32 [n_rows][words], bit t of a row: it sees
    its sequence's row t; pos int32 [n_rows], which attention with a window reads, or None."""

    def __init__(self, mask, pos=None):
        import torch
        _need(mask.dim() == 2, "mask: [n_rows][words]")
        _here(mask, torch.int32, mask.shape, "mask")
        if pos is not None:
            _here(pos, torch.int32, (mask.shape[0],), "pos")
            _need(pos.device == mask.device, "mask and pos are on one device")
        self.mask, self.pos, self.device = mask, pos, mask.get_device()
        self._c = _KVNodesC(mask.data_ptr(), _ptr(pos) or 0, mask.shape[1])
        self._ref = C.byref(self._c)


def kv_tree(batch, parent, mask, pos=None, window=0, stream=None):
    """Masks int32 [n_rows][words], words * 32 >= max_q, and positions int32 [n_rows] of the trees that parent int32
    [n_rows] describes (a row's parent among its sequence's rows), for all the layers' calls of a step. Returns their
    KVTree. window > 0: a row sees the nearest `window` of the rows it continues, itself among them."""
    s = _on_current(stream, batch.kv_len, parent, mask, pos)
    tree = KVTree(mask, pos)
    rows = mask.shape[0]
    _ints(parent, rows, "parent")
    _need(0 <= window < 2**32, "window: 32-bit")
    _check(lib().kq_kv_tree(batch._packed(rows), _ptr(parent), _ptr(mask), mask.shape[1], _ptr(pos), window, s), "kq_kv_tree")
    return tree


def kv_attn_tree_workspace_size(cache, batch, q_heads):
    return _kv_attn_size(lib().kq_kv_attn_tree_workspace_size, "kq_kv_attn_tree_workspace_size", cache, batch, q_heads)


def kv_attn_tree(cache, batch, tree, q, out, ws, ws_bytes, scale=None, window=0, sinks=None, lse=None, stream=None):
    """kv_attn of a tree's rows: each over the tokens before the batch's rows of its sequence (window > 0: behind its
    position less the window) and the rows that its mask names."""
    if tree.device != cache.device or tree.mask.shape[0] != q.shape[0]:
        raise ValueError(f"tree: of {q.shape[0]} rows, on the cache's device")
    _kv_attn(lib().kq_kv_attn_tree, "kq_kv_attn_tree", cache, batch, (tree._ref,), q, out, ws, ws_bytes, scale, True, window, sinks,
             lse, stream)


_int32 = _float32 = None  # torch's, from the first call on


def _ints(t, n, what):
    """t: a contiguous int32 tensor [n]."""
    global _int32, _float32
    if _int32 is None:
        import torch
        _int32, _float32 = torch.int32, torch.float32
    if t.dtype is not _int32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        _here(t, _int32, (n,), what)


def draft_verify_workspace_size(n_seq, max_q, vocab):
    n = lib().kq_draft_verify_workspace_size(n_seq, max_q, vocab)
    if n == 0:
        raise KQError(KQ_EINVAL, "kq_draft_verify_workspace_size")
    return n


def _probabilities(t, what):
    """The shape of a float32 tensor of rows, contiguous and at any stride."""
    if t.dim() != 2 or t.dtype is not _float32 or (t.stride(1) != 1 and t.shape[1] > 1 and t.shape[0]):
        raise ValueError(f"{what}: a float32 tensor of rows, contiguous in its last dimension, not {t.dtype} {tuple(t.shape)} of strides {t.stride()}")
    return t.shape


def draft_verify(p, token, u, keep, n_keep, out, ws, ws_bytes, q=None, q_index=None, parent=None, start=None, stream=None):
    """Drafted tokens against the target's probabilities p float32 [n_rows][vocab] (any row stride), with given
    random numbers u float32 [n_rows]: kept rows into keep int32 [n_seq][max_q], how many into n_keep int32 [n_seq], their
    tokens and the one behind them into out int32 [n_seq][max_q].

    token: int32 [n_rows]. parent: int32 [n_rows] (None: a chain). start: int32 [n_seq + 1] (None: max_q rows
    each). q: float32 [n_q][vocab], the probabilities that the tokens were drawn from, row q_index[i] (int32 [n_rows],
    -1: picked outright) or i for row i; None: all were picked outright."""
    s = _on_current(stream, p, token, u, keep, n_keep, out, q, q_index, parent, start, None if isinstance(ws, int) else ws)
    _need(keep.dim() == 2 and p.dim() == 2, "keep: [n_seq][max_q], p: [n_rows][vocab]")
    n_seq, max_q = keep.shape
    _ints(n_keep, n_seq, "n_keep")
    rows, vocab = _probabilities(p, "p")
    _ints(token, rows, "token")
    if out.shape != keep.shape or out.dtype is not _int32 or not out.is_contiguous() or keep.dtype is not _int32 or not keep.is_contiguous():
        raise ValueError(f"keep, out: contiguous int32 tensors [{n_seq}][{max_q}]")
    if u.dtype is not _float32 or u.dim() != 1 or u.numel() != rows or not u.is_contiguous():
        raise ValueError(f"u: a contiguous float32 tensor [{rows}]")
    for t, n, what in ((parent, rows, "parent"), (start, n_seq + 1, "start"), (q_index, rows, "q_index")):
        if t is not None:
            _ints(t, n, what)
    at_q = n_q = q_row = 0
    if q is not None:
        n_q, wide = _probabilities(q, "q")
        if wide != vocab or (q_index is None and n_q < rows):
            raise ValueError(f"q: {'a row for each of p' if q_index is None else 'rows'}, {vocab} wide, not {tuple(q.shape)}")
        at_q, q_row = q.data_ptr(), q.stride(0)
    d = _pack_draft(p.data_ptr(), at_q, p.stride(0), q_row, _ptr(q_index) or 0, token.data_ptr(), _ptr(parent) or 0, _ptr(start) or 0,
                    u.data_ptr(), n_seq, max_q, rows, n_q, vocab)
    _check(lib().kq_draft_verify(d, keep.data_ptr(), n_keep.data_ptr(), out.data_ptr(), _ptr(ws), ws_bytes, s), "kq_draft_verify")


def kv_keep(cache, batch, keep, n_keep, stream=None):
    """The rows keep[i][:n_keep[i]] (int32 [n_seq][max_q] and [n_seq], as draft_verify leaves them) of each sequence's
    newest tokens moved together in the cache; the sequence then ends behind them, which is for kv_len to say."""
    s = _kv_call(cache, batch, stream, keep, n_keep)
    _ints(n_keep, batch.n_seq, "n_keep")
    if keep.dtype is not _int32 or keep.shape != (batch.n_seq, batch.max_q) or not keep.is_contiguous():
        raise ValueError(f"keep: a contiguous int32 tensor [{batch.n_seq}][{batch.max_q}]")
    rows = batch.n_seq * batch.max_q if batch.q_start is None else 0x7FFF0000 - 1  # with q_start: no tensor has them
    _check(lib().kq_kv_keep(cache._ref, batch._packed(rows), keep.data_ptr(), n_keep.data_ptr(), s), "kq_kv_keep")


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
ROPE_KINDS = ("plain", "linear", "ntk", "bands", "yarn")  # kq_rope_kind


def rope_freqs(rot, base=10000.0, kind="plain", factor=1.0, low=1.0, high=None, original=0.0, device=None):
    """(inv_freq float32 [rot/2] on the device, amplitude): the frequencies of rotary positions, as they are
    or for contexts `factor` times as long as the `original` tokens (kq_rope_freqs; high: 4 in bands, 32 in yarn)."""
    import torch
    _need(kind in ROPE_KINDS, f"kind: one of {', '.join(ROPE_KINDS)}")
    _need(0 <= rot < 2**32, "rot: 32-bit")
    got, amplitude = (C.c_float * max(min(rot, 512) // 2, 1))(), C.c_double(0.0)  # beyond 512 the call refuses
    d = _RopeScalingC(ROPE_KINDS.index(kind), rot, base, factor, low, (32.0 if kind == "yarn" else 4.0) if high is None else high,
                      original)
    _check(lib().kq_rope_freqs(C.byref(d), got, C.byref(amplitude)), "kq_rope_freqs")
    return torch.tensor(list(got), dtype=torch.float32, device=device or "cuda"), amplitude.value


class Rope:
    """kq_rope_desc over a contiguous float32 tensor [rot/2] of frequencies, kept alive with it.

    pairs: columns (2i, 2i + 1) are turned together, else (i, i + rot/2). inverse:
    the other way, which is the gradient."""

    def __init__(self, inv_freq, pairs=False, amplitude=1.0, inverse=False):
        import torch
        _need(inv_freq.dim() == 1, "inv_freq: [rot/2]")
        _here(inv_freq, torch.float32, inv_freq.shape, "inv_freq")
        self.inv_freq, self.device, self.rot = inv_freq, inv_freq.get_device(), 2 * inv_freq.shape[0]
        self._c = _RopeC(inv_freq.data_ptr(), self.rot, bool(pairs), amplitude, bool(inverse))
        self._ref = C.byref(self._c)


def _on_current(stream, *tensors):
    """The call's stream; refuses tensors of another device than the current one, whose stream it is."""
    s = _stream(stream)
    if _current is None:
        _stream(None)
    d = _current[1]()
    for t in tensors:
        if t is not None and t.get_device() != d:
            raise ValueError(f"every tensor of the call is on the current device ({d})")
    return s


def _positions(pos, rows):
    if pos is None:
        return None
    _ints(pos, rows, "pos")
    return pos.data_ptr()


def rope(x, out, pos, rope, stream=None):
    """x [n_rows][heads][head_dim] (float16, bfloat16 or float32, any row and head strides) turned into out, which
    may be x; pos: int32 [n_rows], each row's position."""
    s = _on_current(stream, x, out, pos)
    _need(rope.device == _current[1](), "the rotation's frequencies are on the current device")
    shape, dtype = x.shape, x.dtype
    if len(shape) != 3:
        raise ValueError(f"x: [n_rows][heads][head_dim], not {tuple(shape)}")
    a, b = _kv_rows(x, shape, dtype, "x"), _kv_rows(out, shape, dtype, "out")
    at = _positions(pos, shape[0])
    _check(lib().kq_rope(rope._ref, at, a, b, *shape, _dt(x), s), "kq_rope")


def kv_write_rope(cache, batch, rope, k, v, q=None, q_out=None, pos=None, stream=None):
    """kv_write with the keys turned on their way into the cache, and q [n_rows][q_heads][head_dim] into q_out
    (which may be q). pos: int32 [n_rows], or None: the rows' places in their sequences."""
    s = _kv_call(cache, batch, stream, k, v, q, q_out, pos, rope.inv_freq)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 3 or shape[1] != cache.heads or shape[2] != cache.head_dim:
        raise ValueError(f"k: [n_rows][{cache.heads}][{cache.head_dim}], not {tuple(shape)}")
    _need((q is None) == (q_out is None), "q and q_out: both or none")
    a, b = _kv_rows(k, shape, dtype, "k"), _kv_rows(v, shape, dtype, "v")
    at = _positions(pos, shape[0])
    x = y = None
    heads = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != shape[0] or q.shape[2] != shape[2]:
            raise ValueError(f"q: [{shape[0]}][q_heads][{shape[2]}], not {tuple(q.shape)}")
        heads = q.shape[1]
        x, y = _kv_rows(q, q.shape, dtype, "q"), _kv_rows(q_out, q.shape, dtype, "q_out")
    _check(lib().kq_kv_write_rope(cache._ref, batch._packed(shape[0]), rope._ref, at, x, y, heads, a, b, _dt(k), s),
           "kq_kv_write_rope")
