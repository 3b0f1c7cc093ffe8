// kq_kv_cache.hip -- writing the 8-bit key/value cache and reading it back
// (kq_kv_write, kq_kv_read; the layout and the rule of the scales: kq.h).
#include "kq_internal.h"
#include "kq_kv_write_kernel.h"

namespace kq {
namespace kv {
namespace {

template <int D, int TYPE, int BF>
__global__ __launch_bounds__(256) void kv_write_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups) {
    write_block<D, TYPE, BF, -1>(c, b, K, V, groups, blockIdx.x, Turn{}, nullptr);
}

// F: the type of the rows.
template <int F>
__device__ __forceinline__ float saturate(float y) {
    const float top = F == KQ_F16 ? 65504.0f : F == KQ_BF16 ? 0x1.FEp127f : 3.402823466e38f;
    return y != y ? y : fminf(fmaxf(y, -top), top);
}
// Two, four, eight values to consecutive elements.
template <int F>
__device__ __forceinline__ void put2(uint8_t* to, const float (&y)[2]) {
    if constexpr (F == KQ_F32) *reinterpret_cast<float2*>(to) = make_float2(y[0], y[1]);
    else *reinterpret_cast<uint32_t*>(to) = pair16<F>(y[0], y[1]);
}
template <int F>
__device__ __forceinline__ void put4(uint8_t* to, const float (&y)[4]) {
    if constexpr (F == KQ_F32) *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
    else *reinterpret_cast<u32x2*>(to) = u32x2{pair16<F>(y[0], y[1]), pair16<F>(y[2], y[3])};
}

template <int F>
__device__ __forceinline__ void put8(uint8_t* to, const float (&y)[8]) {
    if constexpr (F == KQ_F32) {
        *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<f32x4*>(to + 16) = f32x4{y[4], y[5], y[6], y[7]};
    } else {
        *reinterpret_cast<u32x4*>(to) = u32x4{pair16<F>(y[0], y[1]), pair16<F>(y[2], y[3]), pair16<F>(y[4], y[5]), pair16<F>(y[6], y[7])};
    }
}

// One wave reads SPAN tokens (16 or 64, an aligned span of the sequence) of one head's K or V. What bounds it is
// the writes: 131k tokens of 8 heads of 128, e4m3 to fp16, 167 us for 805 MB, 4.8 TB/s, where a copy of that
// size reaches 4.9.
template <int D, int TYPE, int F, int SPAN>
__global__ __launch_bounds__(256) void kv_read_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups) {
    const int lane = threadIdx.x & 63;
    const uint32_t job = (blockIdx.x % groups) * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (job >= 2 * c.heads) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int first = s.len - s.n, first0 = max(first, 0);
    const uint32_t t0u = ((uint32_t)first0 / SPAN + blockIdx.x / groups) * SPAN;  // unsigned, as in kv_write_k
    if (s.n == 0 || t0u >= (uint32_t)s.len) return;
    const int t0 = (int)t0u;
    const int lo = max(first0 - t0, 0), hi = min(s.len - t0, SPAN);
    const int32_t* const table = b.pages + (uint64_t)blockIdx.y * b.max_pages;
    const Rows& R = is_v ? V : K;
    constexpr int kSize = F == KQ_F32 ? 4 : 2;
    uint8_t* const out = static_cast<uint8_t*>(R.p) +
                         ((int64_t)(s.row0 + t0 - first) * R.row + (int64_t)h * R.head) * kSize;
    const int64_t pitch = R.row * kSize;
    // its 16-token blocks: where their codes are, and their exponents; no page: zeros of anything
    constexpr int N = SPAN / 16, C = N == 1 ? 2 : 4;  // columns of 16 values a lane
    constexpr int kNone = -1;
    const uint8_t* from[N];
    int exps[N];  // bytes
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = min(t0 + 16 * i, s.len - 1), page = page_of(c, table, t);
        from[i] = (is_v ? c.v : c.k) + code_offset(c, D, max(page, 0), h, t);
        exps[i] = (is_v ? c.v_exp : c.k_exp)[exp_offset(c, max(page, 0), h, t)];
        if (page < 0) exps[i] = kNone;
    }
    // not times 2^(e - 127), which is no normal float at bytes 0 and 255
    auto value = [&](uint32_t byte, int e) {
        return e == kNone ? 0.0f : saturate<F>(__builtin_ldexpf(Code<TYPE>::value(byte), e - 127));
    };
    if (!is_v) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (16 * n + 16 <= lo || 16 * n >= hi) continue;
            u32x2 w[D / 32];
#pragma unroll
            for (int j = 0; j < D / 32; ++j) w[j] = *reinterpret_cast<const u32x2*>(from[n] + (lane + 64 * j) * 8);
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const int i = lane + 64 * j, t = 16 * n + i / (D / 8);  // 8 columns of token t
                float y[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = value(w[j][k / 4] >> k % 4 * 8 & 0xFF, exps[n]);
                if (t >= lo && t < hi) put8<F>(out + t * pitch + i % (D / 8) * 8 * kSize, y);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < (N * D / C + 63) / 64; ++j) {
        const int i = lane + 64 * j, n = i / (D / C), t = n * 16, d = i % (D / C) * C;  // C columns of block n
        if (t + 16 <= lo || t >= hi) continue;  // hi <= SPAN: past the last block too
        int e = exps[0];
        const uint8_t* at = from[0];
#pragma unroll
        for (int k = 1; k < N; ++k) {
            e = n == k ? exps[k] : e;
            at = n == k ? from[k] : at;
        }
        at += d * 16;
        u32x4 w[C];
#pragma unroll
        for (int k = 0; k < C; ++k) w[k] = *reinterpret_cast<const u32x4*>(at + k * 16);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            float y[C];
#pragma unroll
            for (int k = 0; k < C; ++k) y[k] = value(w[k][q / 4] >> q % 4 * 8 & 0xFF, e);
            if (t + q < lo || t + q >= hi) continue;
            if constexpr (C == 4) put4<F>(out + (t + q) * pitch + d * kSize, y);
            else put2<F>(out + (t + q) * pitch + d * kSize, y);
        }
    }
}

// blockIdx.x = the block (write) or span (read), counted from the sequence's first newest token's, x the groups
// of four waves of its heads; .y = the sequence.

template <int D, int TYPE>
hipError_t write_d(const Cache& c, const Batch& b, const Rows& K, const Rows& V, bool bf, dim3 grid, uint32_t groups,
                   hipStream_t s) {
    if (bf) kv_write_k<D, TYPE, 1><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    else kv_write_k<D, TYPE, 0><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    return hipGetLastError();
}

// Workgroups of 16 tokens a wave beyond which 64 a wave are the faster: fewer workgroups then find nothing in ragged batches,
// and two heads of 64 fill a wave's loads better. A wave of the widest heads, or one that writes fp32, has enough to do with
// 16. Graph replays in us, 16 and 64 tokens a wave; 8 heads, int8 to bf16 and lengths spread by their logarithm unless said:
//   64 wide   one of 70001 (e4m3 to fp16) 67, 56 (17508 workgroups); 64 of 10-4000 57, 43 (64512); 200 of 10-900 51, 54 (46400);
//             one of 9001 18, 18 (2260)
//   96        64 of 10-8000 112, 97 (128512); 64 of 10-4000 63, 66 (64512)
//   128       64 of 10-8000 129, 109 (128512); 64 of 10-4000 73, 71 (64512); 200 of 10-900 66, 86 (46400)
//   192, 256  64 of 10-8000 170, 159 and 201, 208; 64 of 10-4000 97, 103 and 116, 132
//   to fp32   64 wide: 64 of 10-8000 119, 104, of 10-4000 68, 73; 128 wide: 177, 203 and 102, 133
constexpr uint64_t kNeverWide = ~0ull;
constexpr uint64_t wide_beyond(uint32_t D, kq_dtype f) {
    if (D == 64) return f == KQ_F32 ? 65536 : 16384;
    return D <= 128 && f != KQ_F32 ? 65536 : kNeverWide;
}

template <int D, int TYPE, kq_dtype F>
hipError_t read_f(const Cache& c, const Batch& b, const Rows& K, const Rows& V, hipStream_t s) {
    const uint32_t groups = (2 * c.heads + 3) / 4;
    const uint32_t narrow = spans(b.max_q, 16) * groups;
    if constexpr (wide_beyond(D, F) != kNeverWide)
        if ((uint64_t)narrow * b.n_seq > wide_beyond(D, F)) {
            kv_read_k<D, TYPE, F, 64><<<dim3(spans(b.max_q, 64) * groups, b.n_seq), 256, 0, s>>>(c, b, K, V, groups);
            return hipGetLastError();
        }
    kv_read_k<D, TYPE, F, 16><<<dim3(narrow, b.n_seq), 256, 0, s>>>(c, b, K, V, groups);
    return hipGetLastError();
}

}  // namespace
}  // namespace kv

hipError_t launch_kv_write(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Rows& K,
                           const kv::Rows& V, bool bf, hipStream_t s) {
    const uint32_t groups = (2 * c.heads + 3) / 4;
    const dim3 grid(kv::spans(b.max_q, 1u << c.block_log2) * groups, b.n_seq);
    return kv::by_dim(D, type, [&](auto d, auto t) {
        return kv::write_d<decltype(d)::value, decltype(t)::value>(c, b, K, V, bf, grid, groups, s);
    });
}

hipError_t launch_kv_read(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Rows& K,
                          const kv::Rows& V, kq_dtype f, hipStream_t s) {
    return kv::by_dim(D, type, [&](auto d, auto t) {
        constexpr int N = decltype(d)::value, T = decltype(t)::value;
        return f == KQ_F16    ? kv::read_f<N, T, KQ_F16>(c, b, K, V, s)
               : f == KQ_BF16 ? kv::read_f<N, T, KQ_BF16>(c, b, K, V, s)
                              : kv::read_f<N, T, KQ_F32>(c, b, K, V, s);
    });
}

}  // namespace kq
