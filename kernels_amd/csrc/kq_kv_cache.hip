// kq_kv_cache.hip -- writing the 8-bit key/value cache and reading it back
// (kq_kv_write, kq_kv_read; the layout and the rule of the scales: kq.h).
#include "kq_internal.h"
#include "kq_kv_device.h"

namespace kq {
namespace kv {
namespace {

// Magnitude bits of both halves of a pair, 0 for infinities and NaN: for finite
// values they order as the magnitudes do.
template <int BF>
__device__ __forceinline__ uint32_t finite_max(uint32_t pair, uint32_t m) {
    const uint32_t top = BF ? 0x7F80u : 0x7C00u;
    const uint32_t a = pair & 0x7FFFu, b = pair >> 16 & 0x7FFFu;
    m = max(m, a < top ? a : 0u);
    return max(m, b < top ? b : 0u);
}

// One wave writes one block of one head's K or V: the largest new magnitude
// over the wave, the exponent, then the codes.
template <int D, int TYPE, int BF>
__global__ __launch_bounds__(256) void kv_write_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups) {
    const uint32_t lane = threadIdx.x & 63, job = (blockIdx.x % groups) * 4 + (threadIdx.x >> 6);
    if (job >= 2 * c.heads) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int first = s.len - s.n, first0 = max(first, 0), B = 1 << c.block_log2;
    const int t0 = ((first0 >> c.block_log2) + (int)(blockIdx.x / groups)) << c.block_log2;
    if (s.n == 0 || t0 >= s.len) return;
    const int page = page_of(c, b.pages + (uint64_t)blockIdx.y * b.max_pages, t0);
    if (page < 0) return;
    const int lo = max(first0 - t0, 0), hi = min(s.len - t0, B);  // the block's new tokens
    uint8_t* const codes = (is_v ? c.v : c.k) + code_offset(c, D, page, h, t0);
    uint8_t* const ep = (is_v ? c.v_exp : c.k_exp) + exp_offset(c, page, h, t0);
    const Rows& R = is_v ? V : K;
    const uint16_t* const x = static_cast<const uint16_t*>(R.p) + (int64_t)(s.row0 + t0 - first) * R.row +
                              (int64_t)h * R.head;  // token t0's values
    // 8 values a lane and step
    uint32_t m = 0;
    for (int i = lo * (D / 8) + (int)lane; i < hi * (D / 8); i += 64) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(x + (int64_t)(i / (D / 8)) * R.row + i % (D / 8) * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = finite_max<BF>(v[j], m);
    }
    m = wave_max(m);
    int e = block_exponent<TYPE>(elem<BF>(m));
    float keep = 1.0f;  // what older codes are multiplied by
    bool grew = false;
    if (lo > 0) {
        const int was = (int)*ep - 127;
        grew = e > was;
        e = max(e, was);
        keep = pow2f(max(was - e, -126));
    }
    // a foreign cache may hold any byte: stay within pow2f's range
    const float scale = pow2f(min(max(-e, -126), 127));
    if (lane == 0) *ep = (uint8_t)(e + 127);
    if (!is_v) {
        for (int i = (grew ? 0 : lo * (D / 8)) + (int)lane; i < hi * (D / 8); i += 64) {
            const int t = i / (D / 8);
            u32x2* const at = reinterpret_cast<u32x2*>(codes + (uint32_t)i * 8);
            u32x2 out;
            if (t < lo) {
                const u32x2 old = *at;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float y[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) y[q] = to_range<TYPE>(Code<TYPE>::value(old[j] >> 8 * q & 0xFF), keep);
                    out[j] = Code<TYPE>::code2(y[0], y[1]) | Code<TYPE>::code2(y[2], y[3]) << 16;
                }
            } else {
                const u32x4 v = *reinterpret_cast<const u32x4*>(x + (int64_t)t * R.row + i % (D / 8) * 8);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    out[j] = Code<TYPE>::code2(to_range<TYPE>(elem<BF>(v[2 * j] & 0xFFFF), scale),
                                               to_range<TYPE>(elem<BF>(v[2 * j] >> 16), scale)) |
                             Code<TYPE>::code2(to_range<TYPE>(elem<BF>(v[2 * j + 1] & 0xFFFF), scale),
                                               to_range<TYPE>(elem<BF>(v[2 * j + 1] >> 16), scale)) << 16;
            }
            *at = out;
        }
        return;
    }
    // V: two columns of 16 tokens a lane and step, 32 contiguous bytes
    for (int i = (int)lane; i < (B >> 4) * (D / 2); i += 64) {
        const int sub = i / (D / 2) * 16, d = i % (D / 2) * 2;
        if (sub >= hi || (sub + 16 <= lo && !grew)) continue;
        u32x4* const at = reinterpret_cast<u32x4*>(codes + (uint32_t)sub * D + d * 16);
        u32x4 col[2] = {};
        if (lo > sub || hi < sub + 16) {
            col[0] = at[0];
            col[1] = at[1];
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const uint32_t sh = t % 4 * 8;
            uint32_t n0, n1;
            if (sub + t >= hi) continue;
            if (sub + t < lo) {
                if (!grew) continue;
                n0 = Code<TYPE>::code(to_range<TYPE>(Code<TYPE>::value(col[0][t / 4] >> sh & 0xFF), keep));
                n1 = Code<TYPE>::code(to_range<TYPE>(Code<TYPE>::value(col[1][t / 4] >> sh & 0xFF), keep));
            } else {
                const uint32_t v = *reinterpret_cast<const uint32_t*>(x + (int64_t)(sub + t) * R.row + d);
                n0 = Code<TYPE>::code(to_range<TYPE>(elem<BF>(v & 0xFFFF), scale));
                n1 = Code<TYPE>::code(to_range<TYPE>(elem<BF>(v >> 16), scale));
            }
            col[0][t / 4] = (col[0][t / 4] & ~(0xFFu << sh)) | n0 << sh;
            col[1][t / 4] = (col[1][t / 4] & ~(0xFFu << sh)) | n1 << sh;
        }
        at[0] = col[0];
        at[1] = col[1];
    }
}

// F: the type of the rows. Eight values to eight consecutive elements, two to two.
template <int F>
__device__ __forceinline__ float saturate(float y) {
    const float top = F == KQ_F16 ? 65504.0f : F == KQ_BF16 ? 0x1.FEp127f : 3.402823466e38f;
    return y != y ? y : fminf(fmaxf(y, -top), top);
}

// One wave reads 16 tokens (an aligned 16 of the sequence) of one head's K or V.
template <int D, int TYPE, int F>
__global__ __launch_bounds__(256) void kv_read_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups) {
    const uint32_t lane = threadIdx.x & 63, job = (blockIdx.x % groups) * 4 + (threadIdx.x >> 6);
    if (job >= 2 * c.heads) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int first = s.len - s.n, first0 = max(first, 0);
    const int t0 = ((first0 >> 4) + (int)(blockIdx.x / groups)) << 4;
    if (s.n == 0 || t0 >= s.len) return;
    const int lo = max(first0 - t0, 0), hi = min(s.len - t0, 16);
    const int page = page_of(c, b.pages + (uint64_t)blockIdx.y * b.max_pages, t0);
    const Rows& R = is_v ? V : K;
    constexpr int kSize = F == KQ_F32 ? 4 : 2;
    uint8_t* const out = static_cast<uint8_t*>(R.p) +
                         ((int64_t)(s.row0 + t0 - first) * R.row + (int64_t)h * R.head) * kSize;
    const int64_t pitch = R.row * kSize;
    const uint64_t off = page < 0 ? 0 : code_offset(c, D, page, h, t0);
    const uint8_t* const codes = (is_v ? c.v : c.k) + off;
    float scale = 0.0f;
    if (page >= 0) {
        const int e = (int)(is_v ? c.v_exp : c.k_exp)[exp_offset(c, page, h, t0)] - 127;
        scale = pow2f(max(e, -126));
    }
    if (!is_v) {
        for (int i = lo * (D / 4) + (int)lane; i < hi * (D / 4); i += 64) {
            const uint32_t w = page < 0 ? 0u : *reinterpret_cast<const uint32_t*>(codes + (uint32_t)i * 4);
            float y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = saturate<F>(Code<TYPE>::value(w >> 8 * q & 0xFF) * scale);
            uint8_t* const to = out + (i / (D / 4)) * pitch + i % (D / 4) * 4 * kSize;
            if constexpr (F == KQ_F32) *reinterpret_cast<f32x4*>(to) = f32x4{y[0], y[1], y[2], y[3]};
            else *reinterpret_cast<u32x2*>(to) = u32x2{pair16<F>(y[0], y[1]), pair16<F>(y[2], y[3])};
        }
        return;
    }
    for (int i = (int)lane; i < D / 2; i += 64) {
        u32x4 col[2] = {};
        if (page >= 0) {
            col[0] = *reinterpret_cast<const u32x4*>(codes + i * 32);
            col[1] = *reinterpret_cast<const u32x4*>(codes + i * 32 + 16);
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            if (t < lo || t >= hi) continue;
            const float y0 = saturate<F>(Code<TYPE>::value(col[0][t / 4] >> t % 4 * 8 & 0xFF) * scale);
            const float y1 = saturate<F>(Code<TYPE>::value(col[1][t / 4] >> t % 4 * 8 & 0xFF) * scale);
            uint8_t* const to = out + t * pitch + i * 2 * kSize;
            if constexpr (F == KQ_F32) *reinterpret_cast<float2*>(to) = make_float2(y0, y1);
            else *reinterpret_cast<uint32_t*>(to) = pair16<F>(y0, y1);
        }
    }
}

template <int D, int TYPE>
hipError_t write_d(const Cache& c, const Batch& b, const Rows& K, const Rows& V, bool bf, dim3 grid, uint32_t groups,
                   hipStream_t s) {
    if (bf) kv_write_k<D, TYPE, 1><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    else kv_write_k<D, TYPE, 0><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    return hipGetLastError();
}

template <int D, int TYPE>
hipError_t read_d(const Cache& c, const Batch& b, const Rows& K, const Rows& V, kq_dtype f, dim3 grid, uint32_t groups,
                  hipStream_t s) {
    if (f == KQ_F16) kv_read_k<D, TYPE, KQ_F16><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    else if (f == KQ_BF16) kv_read_k<D, TYPE, KQ_BF16><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    else kv_read_k<D, TYPE, KQ_F32><<<grid, 256, 0, s>>>(c, b, K, V, groups);
    return hipGetLastError();
}

}  // namespace
}  // namespace kv

// The launches of one wave a block: blockIdx.x = the block counted from the
// sequence's first new one x the groups of four waves of its heads, .y = the sequence.
hipError_t launch_kv_write(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Rows& K,
                           const kv::Rows& V, bool bf, hipStream_t s) {
    const uint32_t blocks = ((b.max_q - 1) >> c.block_log2) + 1 + (b.max_q > 1), groups = (2 * c.heads + 3) / 4;
    const dim3 grid(blocks * groups, b.n_seq);
    return kv::by_dim(D, type, [&](auto d, auto t) {
        return kv::write_d<decltype(d)::value, decltype(t)::value>(c, b, K, V, bf, grid, groups, s);
    });
}

hipError_t launch_kv_read(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Rows& K,
                          const kv::Rows& V, kq_dtype f, hipStream_t s) {
    const uint32_t blocks = ((b.max_q - 1) >> 4) + 1 + (b.max_q > 1), groups = (2 * c.heads + 3) / 4;
    const dim3 grid(blocks * groups, b.n_seq);
    return kv::by_dim(D, type, [&](auto d, auto t) {
        return kv::read_d<decltype(d)::value, decltype(t)::value>(c, b, K, V, f, grid, groups, s);
    });
}

}  // namespace kq
