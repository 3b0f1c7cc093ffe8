/*
 * kq.h -- C ABI of libkq, the MI355X (gfx950) decode hot path:
 *   int4 group-affine GEMV / batched skinny GEMM, codebook (VQ) dequant-GEMV,
 *   the three-kernel MoE block (router top-k, gathered gate/up + SwiGLU,
 *   gathered down + weighted combine), an 8-bit paged key/value cache with the
 *   attention that reads it, and a step of speculative decoding over it (rotary
 *   positions, trees of drafted tokens, their verification).
 *
 * Every entry point is stream-ordered and asynchronous: it validates its
 * arguments on the host, enqueues kernels on `stream` and returns. Nothing
 * here allocates device memory, synchronises, prints or exits. All pointers
 * are caller-owned device pointers (W, IDX and X 16-byte aligned). Errors are
 * reported as kq_status; kq_last_hip_error() gives the HIP code behind
 * KQ_EHIP.
 *
 * The reference (Apple Metal) exposes this path only as per-kernel call
 * surfaces encoded by its Objective-C++ harnesses; each declaration below
 * cites the kernel and the encode site it replaces (paths are relative to the
 * reference repository root).
 */
#ifndef KQ_H
#define KQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same type as hipStream_t; NULL is the default stream. */
typedef struct ihipStream_t* kq_stream_t;

typedef enum kq_status {
    KQ_OK = 0,
    KQ_EINVAL = 1,        /* shape or argument violates the format contract */
    KQ_ENULL = 2,         /* a required pointer is NULL */
    KQ_EALIGN = 3,        /* a pointer is not aligned as required */
    KQ_EUNSUPPORTED = 4,  /* well-formed but not implemented (dtype, batch) */
    KQ_EWORKSPACE = 5,    /* workspace NULL or smaller than required */
    KQ_EHIP = 6           /* the HIP runtime rejected a launch */
} kq_status;

typedef enum kq_dtype { KQ_F16 = 0, KQ_BF16 = 1, KQ_F32 = 2 } kq_dtype;

/* Kernel family used by kq_int4_gemv_path (0 picks by batch size).
 * KQ_PATH_SCALAR: the debug scalar kernel, one thread per (row, token) with
 * a plain per-chunk loop and no staging, after gemv_int4_scalar (v0,
 * int4-gemv/src/kernels.metal:71-95) -- slow, for checking the fast paths
 * on the device; AUTO never picks it.
 * KQ_PATH_MFMA: the matrix cores, G <= 128 with K % 128 == 0 (separate scales and
 * biases 8-byte aligned); separate ones with G = 128 and K / 128 odd, K >= 256,
 * run the skinny matrix-core kernels instead of int4_mfma. */
typedef enum kq_int4_path {
    KQ_PATH_AUTO = 0,
    KQ_PATH_VALU = 1,
    KQ_PATH_MFMA = 2,
    KQ_PATH_SCALAR = 3
} kq_int4_path;

const char* kq_status_str(kq_status s);
/* hipError_t of the last KQ_EHIP returned on this host thread (0 if none). */
int kq_last_hip_error(void);
/* Library version string, e.g. "kq 0.1 gfx950". */
const char* kq_version(void);

/* ------------------------------------------------------------------------
 * int4 group-affine GEMV / skinny GEMM
 *
 *   Y[b, m] = sum_k (S[m, k/G] * q[m, k] + B[m, k/G]) * X[b, k]
 *   q[m, k] = (W[m, k/8] >> 4*(k%8)) & 0xF          (low nibble = lowest k)
 *
 * W  : uint32 [M][K/8], row-major.
 * S,B: per (row, group) scale and bias, dtype sb_dtype (KQ_F16 or KQ_BF16).
 *      B == NULL selects the interleaved layout: S points at SB[M][K/G][2]
 *      (scale, bias) pairs. B != NULL selects separate S[M][K/G], B[M][K/G].
 * X  : fp16 [batch][K].  Y: [batch][M] of y_dtype (KQ_F16 or KQ_F32).
 * Accumulation is fp32. Constraints: K % 32 == 0, G in {32, 64, 128},
 * K % G == 0, 1 <= batch <= 16, M >= 1. The activations are staged in LDS,
 * which bounds K (K <= 29120 on the VALU path); a shape no path takes
 * returns KQ_EUNSUPPORTED.
 *
 * Replaces: gemv_int4_wide_unroll (v6, interleaved SB)
 *   int4-gemv/src/kernels.metal:397-448, encoded by addGemv
 *   int4-gemv/src/main.mm:353-377,404-408; and the split-S/B layout of
 *   gemv_int4_scalar / gemv_int4_simd int4-gemv/src/kernels.metal:71-136.
 *   batch > 1 has no reference kernel (it is the per-row batch-1 op).
 * ------------------------------------------------------------------------ */
kq_status kq_int4_gemv(const uint32_t* W, const void* S, const void* B, kq_dtype sb_dtype,
                       const uint16_t* X, void* Y, kq_dtype y_dtype,
                       uint32_t M, uint32_t K, uint32_t G, uint32_t batch,
                       kq_stream_t stream);

/* kq_int4_gemv with the kernel family forced (VALU dot2 path, MFMA
 * 16x16x32 path, or the debug scalar kernel); used to measure the crossover
 * and to cross-check the paths. Same contract (the scalar kernel has no K
 * limit beyond it). */
kq_status kq_int4_gemv_path(const uint32_t* W, const void* S, const void* B, kq_dtype sb_dtype,
                            const uint16_t* X, void* Y, kq_dtype y_dtype,
                            uint32_t M, uint32_t K, uint32_t G, uint32_t batch,
                            kq_int4_path path, kq_stream_t stream);

/* Tuning entry point: kq_int4_gemv with the kernel family and launch shape
 * forced; 0 = automatic for either field.
 * VALU: rows = K parts P per workgroup (a divisor of the number of 2048-k
 * steps), unroll = ring depth D (2, 4, 8).
 * MFMA: rows = K parts P per workgroup (a divisor of K/128; at most 8 with
 * 2 or 4 tiles per wave, else 16), unroll = 10 * T + D with T the 16-row
 * tiles per wave and D its ring depth in steps: 12, 24 or 42.
 * The launch shape given is the one that runs.
 * Returns KQ_EUNSUPPORTED for a shape the family cannot run. Used by the
 * benchmark sweeps and the tests. */
kq_status kq_int4_gemv_cfg(const uint32_t* W, const void* S, const void* B, kq_dtype sb_dtype,
                           const uint16_t* X, void* Y, kq_dtype y_dtype,
                           uint32_t M, uint32_t K, uint32_t G, uint32_t batch,
                           kq_int4_path path, int rows, int unroll, kq_stream_t stream);

/* xs[b, j] = sum_{i<32} X[b, 32j + i] in fp32, for j < K/32.
 * Replaces: xsum32 int4-gemv/src/kernels.metal:54-65 (encoded at
 * int4-gemv/src/main.mm:247-258). kq_int4_gemv computes this itself. */
kq_status kq_xsum32(const uint16_t* X, float* xs, uint32_t K, uint32_t batch,
                    kq_stream_t stream);

/* Streaming read of `bytes` (multiple of 16) from src, XOR-folded; writes to
 * sink[0] only if the fold is all ones. The bandwidth ceiling.
 * Replaces: stream_read int4-gemv/src/kernels.metal:260-283. */
kq_status kq_stream_read(const void* src, size_t bytes, uint32_t* sink, kq_stream_t stream);

/* kq_stream_read with the launch shape of the reference's ceiling sweep:
 * `unroll` (1, 2, 4 or 8) independent loads in flight per thread, over
 * `threads` threads (a multiple of 256). kq_stream_read uses the best
 * shape measured on MI355X (unroll 1, 2048 x 256 threads).
 * Replaces: stream_read with function constant UNROLL and its dispatch
 * size int4-gemv/src/kernels.metal:260-283, swept by
 * int4-gemv/src/main.mm:294-334. */
kq_status kq_stream_read_cfg(const void* src, size_t bytes, uint32_t* sink, uint32_t unroll,
                             uint32_t threads, kq_stream_t stream);

/* kq_stream_read_cfg that then writes `out_elems` 2-byte values to out: lane
 * 0 of every wave of the grid writes its fold to out[w], out[w + waves], ...
 * -- a GEMV's output store (y of out_elems rows, written from every XCD)
 * after the same read. No counterpart in the reference: a measurement entry,
 * so that a kernel that must store its output is also compared with a read
 * that pays for the same store at the end of its launch. */
kq_status kq_stream_read_out(const void* src, size_t bytes, uint16_t* out, uint32_t out_elems,
                             uint32_t unroll, uint32_t threads, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * Codebook (VQ, d = 2, 256 entries) dequant-GEMV
 *
 *   Y[b, m] = sum_i S[m, 2i / scale_group] *
 *             ( C[m / rows_per_cb][IDX[m, i]][0] * X[b, 2i]
 *             + C[m / rows_per_cb][IDX[m, i]][1] * X[b, 2i+1] )
 *
 * IDX: uint8 [M][K/2].  C: fp16 [ceil(M/rows_per_cb)][256][2].
 * S  : fp16 [M][K/scale_group].  X: fp16 [batch][K].  Y: [batch][M].
 * rows_per_cb = M and scale_group = 32 is the reference format;
 * rows_per_cb = 256 and scale_group = K is the per-row-scale format.
 * Constraints: K % 32 == 0, K <= 30000 (x is staged in LDS, else
 * KQ_EUNSUPPORTED), scale_group == K or a power of two >= 32 dividing K,
 * rows_per_cb >= 1, 1 <= batch <= 16. C and S are finite: an infinite codeword or
 * scale gives NaN also where no x multiplies it (K is padded with zeros of x).
 *
 * Replaces: gemv_vq_wide (v5) vq-gemv/src/kernels.metal:337-380, encoded by
 *   addVQ vq-gemv/src/main.mm:266-286,308-312.
 * ------------------------------------------------------------------------ */
kq_status kq_vq_gemv(const uint8_t* IDX, const uint16_t* C, const uint16_t* S,
                     const uint16_t* X, void* Y, kq_dtype y_dtype,
                     uint32_t M, uint32_t K, uint32_t rows_per_cb, uint32_t scale_group,
                     uint32_t batch, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * VQ quantiser: a dense weight matrix into the format kq_vq_gemv reads
 *
 * W: [M][K] of w_dtype (KQ_F32, KQ_F16 or KQ_BF16; finite values).
 * Out: IDX u8 [M][K/2], C fp16 [ceil(M/rows_per_cb)][256][2] (one codebook
 * per block of rows_per_cb rows; rows_per_cb >= M is the reference's one
 * codebook per matrix), S fp16 [M][K/scale_group] (per-group abs-max;
 * scale_group = 32 is the reference format, = K one scale per row).
 * Per block: Lloyd's k-means with 256 codewords on the pairs normalised by
 * their group's scale -- all of the block's pairs, or `sample` of them drawn
 * with replacement when there are more -- 256 initial centroids drawn from
 * that sample, `iters` iterations, then every pair to its nearest centroid.
 * A codeword is fp16 of the mean of its points, rounded once (from the double,
 * not through the fp32 centroid that the searches use).
 * The draws are seeded (splitmix64 of seed, block and draw number) and the
 * cluster sums are exact integer sums, so the output is a function of the
 * arguments (the same on every run and device).
 * Constraints: K % 32 == 0; scale_group == K or a power of two >= 32
 * dividing K; 1 <= sample <= 2^24; iters <= 1000; K <= 2^18,
 * min(rows_per_cb, M) * K / 2 < 2^32 and ceil(M / rows_per_cb) <= 65535
 * (else KQ_EUNSUPPORTED).
 * ws: kq_vq_quantize_workspace_size bytes, 256-byte aligned (the scales,
 * the sample, the centroids and their sums); 0 means invalid arguments.
 * Launches: 4 + 2 * iters (3 + 2 * iters where IDX and the sample have no
 * room for the cells' candidate lists). IDX is scratch memory meanwhile.
 *
 * Replaces: quantize_matrix / _kmeans vq-gemv/quant/pq_quantize.py:28-83
 *   (reference defaults: iters 25, sample 200000, scale_group 32,
 *   rows_per_cb = M).
 * ------------------------------------------------------------------------ */
size_t kq_vq_quantize_workspace_size(uint32_t M, uint32_t K, uint32_t rows_per_cb,
                                     uint32_t scale_group, uint32_t sample);
kq_status kq_vq_quantize(const void* W, kq_dtype w_dtype, uint32_t M, uint32_t K,
                         uint32_t rows_per_cb, uint32_t scale_group, uint32_t iters,
                         uint32_t sample, uint64_t seed, uint8_t* IDX, uint16_t* C, uint16_t* S,
                         void* ws, size_t ws_bytes, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * MoE decode block (gpt-oss expert-blob format)
 *
 * pool: n_experts blobs of `blob` bytes. Within a blob, projection p (gate,
 * up, down) starts at off_p; within a projection, W (uint32 [rows][cols/8]),
 * S and B (bf16 [rows][cols/64]) and BI (bf16 [rows], output bias) start at
 * sub_w / sub_s / sub_b / sub_bi. gate and up are [inter][hidden], down is
 * [hidden][inter]. Group size is 64.
 * Mirrors MoEParams moe-fused/src/kernels.metal:22-35 and the blob constants
 * moe-fused/src/main.mm:23-25 (derived fields are computed, not passed).
 * ------------------------------------------------------------------------ */
typedef struct kq_moe_desc {
    uint32_t hidden, inter, n_experts, top_k;
    uint64_t blob;
    uint64_t off_gate, off_up, off_down;
    uint64_t sub_w, sub_s, sub_b, sub_bi;
} kq_moe_desc;

/* Fills the gpt-oss-120b values: hidden = inter = 2880, 128 experts, top-4,
 * blob 14,024,704 B, offsets as in moe-fused/src/main.mm:23-25. */
void kq_moe_default_desc(kq_moe_desc* d);

/* Bytes of workspace the MoE entry points need for `batch` tokens: the router
 * logits, a completion counter, the one-launch block's grid-barrier word, the
 * routing plan (distinct experts and their token slots) that the block's
 * gate/up and down kernels read, and the per-slot down products (from as many
 * tokens as the shape gives: 6 at the gpt-oss-120b shapes). A new workspace must be zeroed once with
 * kq_moe_workspace_init (a kernel, not a memset, so it can sit in a captured
 * graph) before its first use; every call leaves it ready for the next.
 * Calls sharing one workspace must be stream-ordered. The uint32 at byte
 * KQ_MOE_WS_ERR_OFFSET stays 0 unless a one-launch block's barrier wait gave
 * up (all of its workgroups were not resident together, e.g. beside other
 * work on the GPU): that call's outputs are then invalid, and the word stays
 * set until the workspace is initialised again. The standalone gate_up and
 * down derive the plan from idx and accept a NULL workspace. */
#define KQ_MOE_WS_ERR_OFFSET 128
size_t kq_moe_workspace_size(const kq_moe_desc* d, uint32_t batch);
kq_status kq_moe_workspace_init(void* ws, size_t bytes, kq_stream_t stream);

/* Reads the workspace's error word into *err after the work already on
 * `stream` (this call synchronises the stream, the one entry point that
 * does); with `clear` non-zero a set word is reset to 0 by a kernel on
 * `stream` before the call returns. *err != 0 means a one-launch block on
 * this workspace gave up waiting and its outputs are invalid. ws_bytes must
 * cover the workspace head (at least 256 bytes). No counterpart in the
 * reference, whose Metal command buffers report a failed dispatch through
 * their status (int4-gemv/src/main.mm:109-113). */
kq_status kq_moe_workspace_error(void* ws, size_t ws_bytes, uint32_t* err, int clear,
                                 kq_stream_t stream);

/* Router logits (fp32 accumulation) for every token, top_k by repeated
 * argmax (strictly greater wins, so the lowest index wins ties), softmax over
 * the selected logits. idx: uint32 [batch][top_k] in descending-logit order;
 * wgt: fp32 [batch][top_k]. If X is fp32, xh (fp16 [batch][hidden]) receives
 * half(X) for the projections; xh may be NULL when X is fp16.
 * R: [n_experts][hidden] of r_dtype (KQ_F16 or KQ_F32).
 * Replaces: router_topk moe-fused/src/kernels.metal:121-163 (encoded at
 *   moe-fused/src/main.mm:178-185); batch > 1 is new. */
kq_status kq_moe_router_topk(const void* R, kq_dtype r_dtype, const void* X, kq_dtype x_dtype,
                             uint32_t batch, const kq_moe_desc* d,
                             uint32_t* idx, float* wgt, uint16_t* xh,
                             void* ws, size_t ws_bytes, kq_stream_t stream);

/* H[b][k][m] = fp16( swiglu(gate_e(xh_b)[m] + BIg[m], up_e(xh_b)[m] + BIu[m]) )
 * for e = idx[b][k], with swiglu(g, u) = min(g,7)*sigmoid(1.702*min(g,7)) *
 * (clamp(u,-7,7) + 1). Each selected expert's rows are read once for all the
 * tokens that chose it. H: fp16 [batch][top_k][inter].
 * Replaces: fused_gate_up_swiglu moe-fused/src/kernels.metal:177-215
 *   (encoded at moe-fused/src/main.mm:187-194). */
kq_status kq_moe_gate_up_swiglu(const uint8_t* pool, const kq_moe_desc* d,
                                const uint32_t* idx, const uint16_t* xh, uint16_t* H,
                                uint32_t batch, void* ws, size_t ws_bytes, kq_stream_t stream);

/* Y[b][m] = sum_k wgt[b][k] * (down_e(H[b][k])[m] + BId[m]), e = idx[b][k],
 * summed in k order. Y: [batch][hidden] of y_dtype (KQ_F32 or KQ_F16).
 * A workspace is optional; where one is given the call may write it, at any
 * batch (the per-slot products), so calls that share one must be stream-ordered.
 * Replaces: fused_down_combine moe-fused/src/kernels.metal:224-265
 *   (encoded at moe-fused/src/main.mm:196-204). */
kq_status kq_moe_down_combine(const uint8_t* pool, const kq_moe_desc* d,
                              const uint32_t* idx, const float* wgt, const uint16_t* H,
                              void* Y, kq_dtype y_dtype, uint32_t batch,
                              void* ws, size_t ws_bytes, kq_stream_t stream);

/* The three passes back to back on one stream (encodeFused,
 * moe-fused/src/main.mm:176-206): three launches; where the slots' h vectors
 * don't fit one workgroup (from 6 tokens at the gpt-oss-120b shapes) down writes
 * per-slot products to the workspace and a fourth, small launch sums them in
 * slot order. idx, wgt, xh (if X is fp32) and H are caller-provided
 * outputs/intermediates of the sizes above. */
kq_status kq_moe_block(const uint8_t* pool, const kq_moe_desc* d,
                       const void* R, kq_dtype r_dtype, const void* X, kq_dtype x_dtype,
                       uint32_t batch, uint32_t* idx, float* wgt, uint16_t* xh, uint16_t* H,
                       void* Y, kq_dtype y_dtype, void* ws, size_t ws_bytes,
                       kq_stream_t stream);

/* kq_moe_block with the launch structure chosen (bit-identical results on
 * every path). KQ_MOE_PATH_AUTO and KQ_MOE_PATH_LAUNCHES: what kq_moe_block
 * does, the three passes of encodeFused (moe-fused/src/main.mm:176-206).
 * KQ_MOE_PATH_ONE: one token, the whole block in one launch of one
 * workgroup per CU (router logits exchanged through tagged device-coherent
 * stores, h through one grid-wide barrier); inside a graph 0.3-0.6 us a
 * block faster than three launches (about 20.7 against 21.3 us at the
 * gpt-oss-120b shape), two launches fewer for eager callers. It stays an
 * option rather than the default for its residency demand. Every workgroup must
 * be resident at once: the path is refused (KQ_EUNSUPPORTED) when the
 * occupancy query says otherwise, and a wait that still gives up (the GPU
 * shared with other work) sets the workspace's error word (see
 * kq_moe_workspace_size). KQ_EUNSUPPORTED too unless batch is 1, hidden and
 * inter need the same number of 1024-element steps, and each wave's down
 * rows fit its registers (ceil(ceil(hidden / (2 x CUs)) / floor(8 / top_k))
 * <= 4, 2 when hidden > 3072). A PATH_ONE call needs every CU to itself:
 * it must not overlap any other work on the device, another PATH_ONE call
 * on another stream included (kq_moe_workspace_error reads the error word
 * a give-up sets). New: the reference always encodes three passes.
 * KQ_MOE_PATH_ATOMIC: the reference's atomic sum(h) block
 * (fused_gate_up_swiglu_at and fused_down_combine_at,
 * moe-fused/src/kernels.metal:400-487; encodeFused with atomicVar,
 * moe-fused/src/main.mm:176-206): three launches, the router zeroing a
 * workspace array of sum(h) per slot and 32-element chunk, gate/up adding
 * every h value to it (as a float, before its fp16 rounding) with a
 * device-scope atomic, down reading the sums instead of summing h. The sums'
 * order is not fixed, so y may differ in the last bits from call to call;
 * idx, wgt and h are those of the other paths. KQ_EUNSUPPORTED unless batch
 * <= 2 and the streaming kernels take the shapes (the block's default form
 * there). */
#define KQ_MOE_PATH_AUTO 0
#define KQ_MOE_PATH_LAUNCHES 1
#define KQ_MOE_PATH_ONE 2
#define KQ_MOE_PATH_ATOMIC 3
kq_status kq_moe_block_path(const uint8_t* pool, const kq_moe_desc* d,
                            const void* R, kq_dtype r_dtype, const void* X, kq_dtype x_dtype,
                            uint32_t batch, uint32_t* idx, float* wgt, uint16_t* xh, uint16_t* H,
                            void* Y, kq_dtype y_dtype, void* ws, size_t ws_bytes, int path,
                            kq_stream_t stream);

/* kq_moe_block without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). It has no counterpart in the reference.
 * The workspace is a fixed array of KQ_MOE_NOALLOC_WS_BYTES in libkq's own
 * device memory, one per GPU, held until the process ends; the call
 * allocates nothing. A (desc, batch) whose kq_moe_workspace_size exceeds
 * KQ_MOE_NOALLOC_WS_BYTES returns KQ_EWORKSPACE (gpt-oss-120b shapes fit up
 * to 16 tokens). The first call on a GPU looks the array's address up
 * (hipGetSymbolAddress) and enqueues nothing else: the array starts as zeros
 * (static storage), so a first call made under stream capture records only
 * the block's own kernels. Every call on one GPU shares that GPU's
 * array: calls that overlap on one GPU (different streams, or different
 * host threads, without ordering between them) race and must not be made.
 * Otherwise the same arguments, results and launches as kq_moe_block. */
#define KQ_MOE_NOALLOC_WS_BYTES (1u << 20)
kq_status kq_moe_block_noalloc(const uint8_t* pool, const kq_moe_desc* d,
                               const void* R, kq_dtype r_dtype, const void* X, kq_dtype x_dtype,
                               uint32_t batch, uint32_t* idx, float* wgt, uint16_t* xh,
                               uint16_t* H, void* Y, kq_dtype y_dtype, kq_stream_t stream);

/* The same block with one operation per launch, one token: router logits,
 * top-k, softmax, then per slot gate GEMV, up GEMV, SwiGLU, and per slot
 * down GEMV, weighted accumulate -- 3 + 5 * top_k launches (23 at top-4),
 * every intermediate through `ws`. It exists to measure what the
 * three-launch block saves. Same arguments and results as kq_moe_block at
 * batch 1 (other batches: KQ_EUNSUPPORTED); ws needs
 * kq_moe_unfused_workspace_size bytes, 256-byte aligned, and no
 * initialisation. n_launches (may be NULL) receives the number of kernel
 * launches made.
 * Replaces: encodeUnfused moe-fused/src/main.mm:208-284 and its kernels
 *   u_router .. u_axpy moe-fused/src/kernels.metal:284-392 (the reference's
 *   28 launches include five x-sum passes that this GEMV does in-kernel). */
size_t kq_moe_unfused_workspace_size(const kq_moe_desc* d);
kq_status kq_moe_block_unfused(const uint8_t* pool, const kq_moe_desc* d,
                               const void* R, kq_dtype r_dtype, const void* X, kq_dtype x_dtype,
                               uint32_t batch, uint32_t* idx, float* wgt, uint16_t* xh,
                               uint16_t* H, void* Y, kq_dtype y_dtype, void* ws, size_t ws_bytes,
                               uint32_t* n_launches, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * 8-bit key/value cache, and the attention that reads it
 *
 * A paged cache: n_pages pages of `page` tokens of every head. A sequence is a
 * row of page ids; its token p is token p % page of its page p / page.
 *
 *   k     : codes [n_pages][heads][page][head_dim]
 *   v     : codes [n_pages][heads][page / 16][head_dim][16] -- the 16 tokens of
 *           a column lie together, as the product with the probabilities
 *           takes them
 *   k_exp, v_exp : uint8 [n_pages][heads][page / block], a byte for each block
 *           of `block` tokens and head: a code c of the block stands for
 *           c * 2^(byte - 127). kq_kv_write keeps byte - 127 within [-64, 121]
 *           (KQ_KV_I8) or [-64, 119] (KQ_KV_E4M3).
 *
 * A code is an int8 (KQ_KV_I8) or an OCP e4m3 (KQ_KV_E4M3). Powers of two as
 * scales: every product with one is exact, so the codes do not depend on how
 * they are computed, and a block that tokens are appended to one by one is
 * rarely scaled anew (a running maximum would be, 3.4 times on average over 16
 * tokens, and cost each older token half a step every time).
 *
 * Constraints: head_dim 64, 96, 128, 192 or 256 (else KQ_EUNSUPPORTED); block a
 * power of two from 16 to 256; page a power of two from block to 4096; 1 <=
 * heads <= 1024; k and v 16-byte aligned. Offsets are 64-bit: the cache may be
 * of any size.
 * No counterpart in the reference, which has no attention.
 * ------------------------------------------------------------------------ */
typedef enum kq_kv_type { KQ_KV_I8 = 0, KQ_KV_E4M3 = 1 } kq_kv_type;

typedef struct kq_kv_cache {
    void* k;
    void* v;
    uint8_t* k_exp;
    uint8_t* v_exp;
    uint32_t type; /* kq_kv_type */
    uint32_t n_pages, page, block, heads, head_dim;
} kq_kv_cache;

/* The sequences of a call and their newest tokens, the rows of q, k, v and o:
 * sequence i has rows q_start[i] .. q_start[i + 1] - 1, or with q_start NULL the
 * max_q rows from i * max_q on. They are the last of its kv_len[i] tokens:
 * kv_len counts them, in kq_kv_write too.
 *
 * pages   : int32 [n_seq][max_pages] page ids; those behind a sequence's last
 *           token may be anything
 * kv_len  : int32 [n_seq], 0 <= kv_len[i] <= max_len
 * q_start : int32 [n_seq + 1], ascending, q_start[n_seq] <= n_rows; or NULL
 * max_q   : at least the most rows of a sequence;  n_rows: the rows of the
 *           arrays (more than the sequences have: the rest is left as it was;
 *           0: the call does nothing)
 * max_len : at least the longest kv_len; both bounds shape the launch
 *
 * pages, kv_len and q_start are device memory and cannot be checked on the
 * host. The kernels stay in bounds whatever they hold: lengths are cut to
 * max_len and max_pages * page, rows to max_q and n_rows, and the tokens of a
 * page id outside [0, n_pages) are left out -- not written, not attended to,
 * read as zeros.
 * Constraints: 1 <= n_seq <= 65535; max_q, max_pages, max_len >= 1; max_len, n_rows
 * < 2^31 - 2^16; q_start NULL: n_seq * max_q <= n_rows. KQ_EUNSUPPORTED where the
 * bounds ask for more than a launch can have, 2^24 workgroups:
 *   kq_kv_write, kq_kv_read: (max_q / block + 2) * ceil(heads / 2), block 16 in kq_kv_read
 *   kq_kv_attn, with rows = max_q * q_heads / heads: n_seq * heads, rounded up to
 *     a multiple of 8, for each 32 rows (each 16 where rows <= 16 or head_dim is
 *     192 or 256) if rows <= 64; beyond, n_seq * heads for each 128 rows (two for
 *     each 256 where head_dim is 96 or 128 and rows > 128)
 * and in kq_kv_attn for n_seq * max_q * q_heads of 2^31 - 2^16. */
typedef struct kq_kv_batch {
    const int32_t* pages;
    const int32_t* kv_len;
    const int32_t* q_start;
    uint32_t n_seq, max_pages, max_q, n_rows, max_len;
} kq_kv_batch;

/* The rows of a tensor [n_rows][heads][head_dim]: element strides of a row and of a
 * head; head_dim is contiguous. Strides are non-negative multiples of 8 (that of
 * a single row or head is not looked at), the pointer 16-byte aligned (a slice
 * of a fused projection's output is). Where a call writes them, no two rows or
 * heads share elements (else KQ_EINVAL), nor two of the call's tensors. */
typedef struct kq_kv_rows {
    void* p;
    int64_t row, head;
} kq_kv_rows;

/* Writes the newest tokens' keys and values K, V (dtype KQ_F16 or KQ_BF16).
 * Per block and head: a = the largest |x| of the block's new values, e = the
 * smallest integer within the type's range with a <= 127 * 2^e (448 * 2^e), at
 * least the block's present one where it holds older tokens of the sequence;
 * codes are x * 2^-e rounded to nearest even, saturated. Where an older block's
 * e grows its codes are rounded anew from their present values. Infinities
 * become the largest code (and do not count in a), NaN zero: what is written
 * is finite. Nothing but those blocks' new and re-rounded codes and exponents
 * changes. One launch. A page that the call writes must belong to one
 * sequence of it (pages of a shared prefix are only read). */
kq_status kq_kv_write(const kq_kv_cache* cache, const kq_kv_batch* batch, const kq_kv_rows* K,
                      const kq_kv_rows* V, kq_dtype dtype, kq_stream_t stream);

/* Reads the newest tokens of each sequence -- q_start of whole lengths: the whole
 * sequences -- into K, V (dtype KQ_F16, KQ_BF16 or KQ_F32): code * 2^e rounded to
 * nearest even; values beyond the type's largest finite one become that. Rows
 * at negative positions (more rows than tokens) are left as they were. */
kq_status kq_kv_read(const kq_kv_cache* cache, const kq_kv_batch* batch, const kq_kv_rows* K,
                     const kq_kv_rows* V, kq_dtype dtype, kq_stream_t stream);

/* Attention of each row over its sequence's tokens in the cache. Query head h
 * reads head h / (q_heads / heads). Row j of a sequence's n is at position
 * pos = kv_len - n + j and sees tokens p with
 *   causal:     p <= pos, and with window > 0 also p > pos - window
 *   not causal: every p < kv_len (window must be 0).
 *   O = sum_p exp(s_p) v_p / L,  L = sum_p exp(s_p) + exp(sinks[h]),
 *   s_p = scale * (q . k_p);  lse = log L
 * sinks: float [q_heads], or NULL for none. lse: float [n_rows][q_heads], or
 * NULL. A row that sees nothing gets zeros (lse: the sink, or -inf). Rows of
 * no sequence are left as they were. Q and O have q_heads heads, of dtype KQ_F16
 * or KQ_BF16; O may not overlap Q.
 * Scores, softmax and sums are fp32. The products run in fp16 on exact
 * codes: bf16 queries are scaled to fp16 by a power of two for each row, which
 * keeps every bit down to 2^-28 of the row's largest; probabilities are
 * rounded to fp16 (subnormal from 2^-25 of the row's largest down; smaller
 * than 2^-36 of it they are lost, in O alone).
 * A cache from elsewhere holds no NaN codes (e4m3 0x7F, 0xFF) below kv_len, or
 * rows of that sequence and head may be NaN; behind it any bytes do. The
 * exponents of a sequence and head's V, of all its blocks below kv_len, differ
 * by 100 at most, wherever in 0 .. 255 they lie.
 * ws: kq_kv_attn_workspace_size bytes (enough for any window), 256-byte
 * aligned, no initialisation and nothing kept in it between calls: the partial
 * results of sequences that are split among workgroups. Calls that share one must be
 * stream-ordered. 0 from kq_kv_attn_workspace_size means invalid arguments.
 * q_heads: a multiple of cache->heads, at most 64 times as many. Results do
 * not change from run to run (no atomics).
 * A batch whose max_q * q_heads / heads is over 64 runs the kernel for many rows
 * throughout. Sequences of few rows over long contexts are slow in it: give them
 * a call of their own (KQ_OK either way; slices of one batch's arrays do). */
typedef struct kq_kv_attn_desc {
    uint32_t q_heads;
    float scale;
    uint32_t causal, window;
    const float* sinks;
} kq_kv_attn_desc;
size_t kq_kv_attn_workspace_size(const kq_kv_cache* cache, const kq_kv_batch* batch,
                                 uint32_t q_heads);
kq_status kq_kv_attn(const kq_kv_cache* cache, const kq_kv_batch* batch, const kq_kv_attn_desc* d,
                     const kq_kv_rows* Q, const kq_kv_rows* O, kq_dtype dtype, float* lse,
                     void* ws, size_t ws_bytes, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * Rotary positions
 *
 * Pairs (a, b) of a head's first `rot` columns are turned by the angle t = pos *
 * inv_freq[i], i the pair:
 *   y_a = A (x_a cos t - x_b sin t),  y_b = A (x_b cos t + x_a sin t)
 * with (a, b) = (i, i + rot / 2) (KQ_ROPE_HALVES) or (2i, 2i + 1) (KQ_ROPE_PAIRS), A
 * the amplitude. Columns from rot on stay as they are. `inverse` turns the other
 * way, times A again: the gradient of x, given that of y.
 * Angles, their cosines and sines and the products are 64-bit, so that far
 * positions keep their angle (|t| < 2^32); y is rounded to 32 bits, then to its type.
 *
 * inv_freq  : float [rot / 2], device memory, finite (kq_rope_freqs makes them)
 * rot       : even, 2 <= rot <= head_dim
 * amplitude : finite
 * No counterpart in the reference, which has no attention.
 * ------------------------------------------------------------------------ */
typedef enum kq_rope_layout { KQ_ROPE_HALVES = 0, KQ_ROPE_PAIRS = 1 } kq_rope_layout;
typedef struct kq_rope_desc {
    const float* inv_freq;
    uint32_t rot;
    uint32_t layout; /* kq_rope_layout */
    double amplitude;
    uint32_t inverse;
} kq_rope_desc;

/* Frequencies f_i = base^(-2i / rot) and their forms for contexts longer than a
 * model was trained on (`original` tokens, stretched by `factor`), and the
 * amplitude that goes with them (1 but for KQ_ROPE_YARN):
 *   KQ_ROPE_PLAIN   f_i
 *   KQ_ROPE_LINEAR  f_i / factor
 *   KQ_ROPE_NTK     base * factor^(rot / (rot - 2)) for base
 *   KQ_ROPE_BANDS   turns n_i = original f_i / 2 pi in the original context: f_i where n_i >
 *                   high, f_i / factor where n_i < low, in between the mean of the two,
 *                   (n_i - low) / (high - low) of the former
 *   KQ_ROPE_YARN    f_i (1 - r) + f_i / factor r, r_i = (i - from) / (to - from) within [0, 1], from =
 *                   floor(c(high)), to = ceil(c(low)), both within [0, rot - 1] (to + 0.001
 *                   where they are the same), c(n) = rot ln(original / (2 pi n)) / (2 ln base);
 *                   amplitude 0.1 ln(factor) + 1
 * Host memory, computed in 64 bits; no GPU call. base > 1 (NTK: rot > 2), factor >= 1, 0 < low <
 * high, original > 0 where they are used, all finite. */
typedef enum kq_rope_kind {
    KQ_ROPE_PLAIN = 0,
    KQ_ROPE_LINEAR = 1,
    KQ_ROPE_NTK = 2,
    KQ_ROPE_BANDS = 3,
    KQ_ROPE_YARN = 4
} kq_rope_kind;
typedef struct kq_rope_scaling {
    uint32_t kind; /* kq_rope_kind */
    uint32_t rot;
    double base, factor, low, high, original;
} kq_rope_scaling;
kq_status kq_rope_freqs(const kq_rope_scaling* s, float* inv_freq, double* amplitude);

/* Y = X turned, rows x heads x head_dim of dtype KQ_F16, KQ_BF16 or KQ_F32, row i at
 * position pos[i] (int32 [n_rows], device memory; any values). Y may be X (the same
 * address and strides), and overlaps it in no other way. A slice of a fused projection that holds the
 * queries' and then the keys' heads is turned in one call. head_dim a multiple of 8,
 * at most 512, heads <= 65535; the strides as kq_kv_rows has them. n_rows 0: the call does nothing.
 * One launch. rot a multiple of 16 takes whole vectors, 64 / (rot / 16) heads of a row a wave, and twice that
 * beyond 1024 rows; others go value by value, one head a wave, and beyond 1024 rows all of a row.
 * KQ_EUNSUPPORTED where these are more than 4 * (2^24 - 1) waves. */
kq_status kq_rope(const kq_rope_desc* d, const int32_t* pos, const kq_kv_rows* X, const kq_kv_rows* Y,
                  uint32_t n_rows, uint32_t heads, uint32_t head_dim, kq_dtype dtype,
                  kq_stream_t stream);

/* kq_kv_write with the rotation on the way: the cache's keys are those that kq_rope
 * leaves, rounded to their type as it rounds them (bit for bit what kq_rope and
 * kq_kv_write leave one after the other), the values as in kq_kv_write. K itself is not
 * changed. With Q (q_heads heads) its rows of the batch are turned into Qo too (which
 * may be Q); Q NULL: none, Qo and q_heads are not looked at.
 * pos: int32 [n_rows], device memory, the position of each row (of a tree: kq_kv_tree's);
 * NULL: a row's place in its sequence, kv_len - n + j.
 * rot a multiple of 16 (else KQ_EUNSUPPORTED: kq_rope first); q_heads <= 65535. One launch;
 * KQ_EUNSUPPORTED too where kq_kv_write's workgroups and max_q * ceil(q_heads / 4) / 4 + 1
 * more for the queries are over its bound. */
kq_status kq_kv_write_rope(const kq_kv_cache* cache, const kq_kv_batch* batch,
                           const kq_rope_desc* d, const int32_t* pos, const kq_kv_rows* Q,
                           const kq_kv_rows* Qo, uint32_t q_heads, const kq_kv_rows* K,
                           const kq_kv_rows* V, kq_dtype dtype, kq_stream_t stream);

/* ------------------------------------------------------------------------
 * Trees of drafted tokens
 *
 * A sequence's rows of a step as a tree: row 0 is the last token that is certain,
 * rows 1 .. n - 1 are drafted, and row j continues row parent[j] < j. Their keys
 * and values stand in the cache one after the other, as kq_kv_write puts them.
 * No counterpart in the reference.
 *
 * kq_kv_tree: what the step's calls take of a tree, once for all layers.
 * parent : int32 [n_rows], of each row the number of its parent among its
 *          sequence's rows; one that is not in 0 .. j - 1 makes row j a root
 * mask   : uint32 [n_rows][words], written: bit t of row j says that the row sees
 *          its sequence's row t: itself and the rows it continues; with
 *          window > 0 the nearest `window` of them alone. words >= max_q / 32, rounded up
 * pos    : int32 [n_rows] or NULL, written: kv_len - n + the row's depth
 * Rows of no sequence are left as they were. max_q <= 1024 (else KQ_EUNSUPPORTED). The
 * batch's pages are not read (lengths are cut to max_len alone). One launch. */
kq_status kq_kv_tree(const kq_kv_batch* batch, const int32_t* parent, uint32_t* mask,
                     uint32_t words, int32_t* pos, uint32_t window, kq_stream_t stream);

/* kq_kv_attn of a tree's rows: a row sees the tokens of its sequence before the
 * batch's rows -- with window > 0 those behind position pos - window -- and of the batch's
 * rows of its sequence those whose bit is set in its mask, whatever they are (a mask of
 * nothing is one, too). Everything else is kq_kv_attn's: sums and roundings (probabilities and
 * queries as fp16 in the products), sinks, lse, rows that see nothing. d->causal is not looked at. Limits of a launch: kq_kv_attn's, n_seq * heads rounded up
 * to a multiple of 8; where max_q * (q_heads / heads) > 64, for each 128 of those rows (of 96 or 128 columns, where they are more
 * than 128: two for each 256).
 * pos: int32 [n_rows], the rows' positions, below 2^31 - 2^16 and at least that of their
 * sequence's first row (else they count as that); read with window > 0 alone, else NULL will do.
 * words * 32 >= max_q, max_q <= 1024 (else KQ_EUNSUPPORTED).
 * ws: kq_kv_attn_tree_workspace_size bytes (up to some 70 MB while max_q * (q_heads / heads) is 32768 at most,
 * and some 140 beyond, of heads of 256), otherwise as kq_kv_attn's. */
typedef struct kq_kv_nodes {
    const uint32_t* mask;
    const int32_t* pos;
    uint32_t words;
} kq_kv_nodes;
size_t kq_kv_attn_tree_workspace_size(const kq_kv_cache* cache, const kq_kv_batch* batch,
                                      uint32_t q_heads);
kq_status kq_kv_attn_tree(const kq_kv_cache* cache, const kq_kv_batch* batch,
                          const kq_kv_attn_desc* d, const kq_kv_nodes* nodes, const kq_kv_rows* Q,
                          const kq_kv_rows* O, kq_dtype dtype, float* lse, void* ws,
                          size_t ws_bytes, kq_stream_t stream);

/* Which drafted tokens are kept, and the token behind them, so that what comes out
 * is distributed as the target's own draws are. From row 0 on: with P the target's
 * probabilities after the row, S = 1, the rows that continue it are tried in order,
 *   row c of token x, drawn from Q: kept if u[c] S Q(x) < P(x); if not,
 *   P becomes max(P - S Q, 0) and S its sum
 *   (a token picked outright: Q(x) = 1, and P(x) becomes 0, S less by what it was)
 * and the way goes on from the one that is kept. Where none is, the last token is
 * the first whose sum of P up to it is over u[row 0] times P's whole sum (if that is
 * 0: the first of the largest probability of the row). All of it is 64-bit.
 *
 * p      : float [n_rows][vocab], row stride p_row: after each row, adding up to 1
 * q      : float [n_q][vocab], row stride q_row, or NULL: every token is picked outright
 * q_index: int32 [n_rows] or NULL: the row of q that a row's token was drawn from; outside
 *          [0, n_q): picked outright. NULL: the row's own (n_q >= n_rows)
 * token  : int32 [n_rows] (a row 0's is not looked at); outside [0, vocab): never kept
 * parent : int32 [n_rows] or NULL: each row continues the one before. Rows whose
 *          parent is not in 0 .. j - 1 are never reached
 * u      : float [n_rows], in [0, 1)
 * start  : int32 [n_seq + 1], ascending, or NULL: max_q rows each
 * Probabilities that are negative or not finite count as 0. 64-bit sums of many are taken
 * in one order, whatever the run.
 * Written: keep int32 [n_seq][max_q], the kept rows' numbers (row 0 first), n_keep int32
 * [n_seq], how many (0: the sequence has no rows), out int32 [n_seq][max_q], n_keep
 * tokens: those of the kept rows but row 0, then the last one. Behind them keep
 * and out are -1. No two written arrays, and none that is read, overlap.
 * max_q <= 1024, vocab < 2^31 - 2^16 (else KQ_EUNSUPPORTED); 1 <= n_seq <= 65535.
 * ws: kq_draft_verify_workspace_size bytes, 256-byte aligned, no initialisation and nothing
 * kept in it; calls that share one must be stream-ordered. */
typedef struct kq_draft {
    const float* p;
    const float* q;
    int64_t p_row, q_row;
    const int32_t *q_index, *token, *parent, *start;
    const float* u;
    uint32_t n_seq, max_q, n_rows, n_q, vocab;
} kq_draft;
size_t kq_draft_verify_workspace_size(uint32_t n_seq, uint32_t max_q, uint32_t vocab);
kq_status kq_draft_verify(const kq_draft* d, int32_t* keep, int32_t* n_keep, int32_t* out, void* ws,
                          size_t ws_bytes, kq_stream_t stream);

/* Moves the kept rows of each sequence together: row keep[i][j] of sequence i's newest
 * tokens goes to the place of its row j, j < n_keep[i]. keep: int32 [n_seq][max_q],
 * ascending (so that keep[i][j] >= j); n_keep: int32 [n_seq], cut to max_q and the
 * sequence's rows. An entry that is less than its j, not more than the one before it, or no row, ends
 * the list there. The sequence then holds kv_len - n + n_keep tokens, which
 * is the caller's to set; what is behind them may be overwritten by the next step.
 * Codes are moved as they are where the two blocks' exponents are the same. A
 * block that rows are moved into takes the largest exponent of its own and of those
 * they come from; all its tokens below kv_len go by it, rounded to nearest even
 * where it grows. Tokens of a page id outside [0, n_pages) are read as zeros, of the
 * smallest exponent, and not written. A page that the call writes must belong to one sequence of it.
 * max_q <= 1024 (else KQ_EUNSUPPORTED). One launch. */
kq_status kq_kv_keep(const kq_kv_cache* cache, const kq_kv_batch* batch, const int32_t* keep,
                     const int32_t* n_keep, kq_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KQ_H */
