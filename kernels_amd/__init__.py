"""kernels_amd -- MI355X (gfx950) decode hot path: int4 GEMV / skinny GEMM,
VQ dequant-GEMV, the three-kernel MoE block and an 8-bit key/value cache with
its attention, behind libkq's C ABI.

`kernels_amd.kq` is the host layer (ctypes over include/kq.h);
`kernels_amd.gen` builds the seeded synthetic inputs of the benchmark configs.
"""
from . import kq  # noqa: F401
from .kq import (GemvParams, KQError, KVBatch, KVCache, MoEDesc, VQParams, int4_gemv,  # noqa: F401
                 kv_attn, kv_attn_workspace_size, kv_cache, kv_read, kv_write, lib, moe_block,
                 moe_default_desc, moe_down_combine, moe_gate_up_swiglu, moe_router_topk,
                 moe_workspace_init, moe_workspace_size, stream_read, vq_gemv, xsum32)

__all__ = ["kq", "GemvParams", "VQParams", "MoEDesc", "KQError", "lib", "int4_gemv", "vq_gemv",
           "xsum32", "stream_read", "moe_default_desc", "moe_workspace_size",
           "moe_workspace_init", "moe_router_topk", "moe_gate_up_swiglu", "moe_down_combine",
           "moe_block", "KVCache", "KVBatch", "kv_cache", "kv_write", "kv_read", "kv_attn",
           "kv_attn_workspace_size"]
