// kq_kv_cache.hip -- writing the 8-bit key/value cache and reading it back
// (kq_kv_write, kq_kv_read; the layout and the rule of the scales: kq.h).
#include "kq_internal.h"
#include "kq_kv_device.h"

namespace kq {
namespace kv {
namespace {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Magnitude bits of both halves of pairs order as the magnitudes do; from kInf on they are no finite value's.
template <int BF>
constexpr uint32_t kInf = BF ? 0x7F80u : 0x7C00u;
__device__ __forceinline__ uint32_t pair_max(uint32_t pair, uint32_t m) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, pair & 0x7FFF7FFFu),
                                                                  __builtin_bit_cast(u16x2, m)));
}
// The larger half, and the same of finite values alone.
__device__ __forceinline__ uint32_t half_max(uint32_t m) { return max(m & 0xFFFFu, m >> 16); }
template <int BF>
__device__ __forceinline__ uint32_t finite_max(uint32_t pair, uint32_t m) {
    const uint32_t a = pair & 0x7FFFu, b = pair >> 16 & 0x7FFFu;
    return max(m, max(a < kInf<BF> ? a : 0u, b < kInf<BF> ? b : 0u));
}

// Four codes of a dword anew: the values they stand for times `keep`, rounded.
template <int TYPE>
__device__ __forceinline__ uint32_t rounded_anew(uint32_t w, float keep) {
    float y[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) y[q] = to_range<TYPE>(Code<TYPE>::value(w >> 8 * q & 0xFF), keep);
    return Code<TYPE>::code2(y[0], y[1]) | Code<TYPE>::code2(y[2], y[3]) << 16;
}
// Codes of four values times `scale`. PLAIN: all are finite and within the codes' range as they are.
// int8: adding 1.5 * 2^23 rounds to nearest even and leaves the integer's low byte in the sum's.
template <int TYPE, bool PLAIN>
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float scale) {
    if constexpr (!PLAIN) {
        return Code<TYPE>::code2(to_range<TYPE>(a, scale), to_range<TYPE>(b, scale)) |
               Code<TYPE>::code2(to_range<TYPE>(c, scale), to_range<TYPE>(d, scale)) << 16;
    } else if constexpr (TYPE == KQ_KV_I8) {
        auto low = [&](float x) { return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, scale, 12582912.0f)); };
        return __builtin_amdgcn_perm(low(b), low(a), 0x0C0C0400u) | __builtin_amdgcn_perm(low(d), low(c), 0x04000C0Cu);
    } else {
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * scale, b * scale, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * scale, d * scale, w, true);
    }
}

// One wave writes one block of one head's K or V: the largest new magnitude over the wave, the
// exponent, then the codes. Blocks of 16 tokens stay in registers in between (bf16 prefill of 13k
// tokens, 8 heads of 128: 28-35 us for 82 MB with a second read, 21-27 without); larger ones are read
// twice, 16 tokens at a time, the second time from a cache.
template <int D, int TYPE, int BF>
__global__ __launch_bounds__(256) void kv_write_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups) {
    const int lane = threadIdx.x & 63;
    const uint32_t job = (blockIdx.x % groups) * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (job >= 2 * c.heads) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int first = s.len - s.n, first0 = max(first, 0), B = 1 << c.block_log2;
    // unsigned: blocks behind a sequence of nearly 2^31 tokens pass 31 bits
    const uint32_t t0u = (((uint32_t)first0 >> c.block_log2) + blockIdx.x / groups) << c.block_log2;
    if (s.n == 0 || t0u >= (uint32_t)s.len) return;
    const int t0 = (int)t0u;
    const int page = page_of(c, b.pages + (uint64_t)blockIdx.y * b.max_pages, t0);
    const int lo = max(first0 - t0, 0), hi = min(s.len - t0, B);  // the block's new tokens
    const Rows& R = is_v ? V : K;
    const uint16_t* const x = static_cast<const uint16_t*>(R.p) + (int64_t)(s.row0 + t0 - first) * R.row +
                              (int64_t)h * R.head;  // token t0's values

    // 16 tokens in registers. K: 8 columns of a token a piece. V: two columns of 16 tokens, or of 8
    // where that fills the wave.
    constexpr int NK = D / 32, H = D == 64 ? 2 : 1, TL = 16 / H, NV = (D / 2 * H + 63) / 64;
    u32x4 xk[NK];
    uint32_t xv[NV][TL];
    // (inlined by force: of functions of their own, which the compiler makes of the two at 192 and 256 wide, the
    // values' registers go through memory: five prompts of 331 to 5001 tokens, 8 heads of 256, written and
    // read 143 us so, 64 inlined)
    auto load = [&](int sub) __attribute__((always_inline)) {
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                const int i = lane + 64 * j, t = sub + i / (D / 8);
                xk[j] = t >= lo && t < hi ? *reinterpret_cast<const u32x4*>(x + (int64_t)t * R.row + i % (D / 8) * 8) : u32x4{};
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < TL; ++q) {
                    const int i = lane + 64 * j, t = sub + i / (D / 2) * TL + q;
                    const bool there = t >= lo && t < hi && (NV * 64 == D / 2 * H || i < D / 2 * H);
                    xv[j][q] = there ? *reinterpret_cast<const uint32_t*>(x + (int64_t)t * R.row + i % (D / 2) * 2) : 0u;
                }
        }
    };
    load(lo & ~15);  // on its way while the page id is
    if (page < 0) return;
    uint8_t* const codes = (is_v ? c.v : c.k) + code_offset(c, D, page, h, t0);
    uint8_t* const ep = (is_v ? c.v_exp : c.k_exp) + exp_offset(c, page, h, t0);
    const int was = lo > 0 ? (int)*ep - 127 : -127;
    uint32_t m = 0;
    for (int sub = lo & ~15; sub < hi; sub += 16) {
        if (sub > lo) load(sub);
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = pair_max(xk[j][q], m);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < TL; ++q) m = pair_max(xv[j][q], m);
        }
    }
    m = wave_max(half_max(m));
    const bool finite = m < kInf<BF>;
    if (!finite) {  // once more, without infinities and NaN
        m = 0;
        for (int sub = lo & ~15; sub < hi; sub += 16) {
            if (B > 16) load(sub);
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) m = finite_max<BF>(xk[j][q], m);
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int q = 0; q < TL; ++q) m = finite_max<BF>(xv[j][q], m);
            }
        }
        m = wave_max(m);
    }
    const int wanted = block_exponent<TYPE>(elem<BF>(m));
    const int e = max(wanted, was);
    const bool grew = lo > 0 && wanted > was;
    const float keep = pow2f(max(was - e, -126));  // what older codes are multiplied by
    // e >= kMinExp; up to 128 where a cache from elsewhere holds such a byte: a subnormal scale, exact too
    const float scale = __builtin_ldexpf(1.0f, -e);
    if (lane == 0) *ep = (uint8_t)(e + 127);
    auto write = [&](auto plain) __attribute__((always_inline)) {
        constexpr bool P = decltype(plain)::value;
        for (int sub = grew ? 0 : lo & ~15; sub < hi; sub += 16) {
            if (B > 16) load(sub);
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    const int i = lane + 64 * j, t = sub + i / (D / 8);
                    u32x2* const at = reinterpret_cast<u32x2*>(codes + (uint32_t)(sub * D + i * 8));
                    if (t >= lo && t < hi) {
                        const u32x4 v = xk[j];
                        u32x2 w;
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            w[q] = four_codes<TYPE, P>(elem<BF>(v[2 * q] & 0xFFFF), elem<BF>(v[2 * q] >> 16),
                                                       elem<BF>(v[2 * q + 1] & 0xFFFF), elem<BF>(v[2 * q + 1] >> 16), scale);
                        *at = w;
                    } else if (t < lo && grew) {
                        const u32x2 old = *at;
                        *at = u32x2{rounded_anew<TYPE>(old.x, keep), rounded_anew<TYPE>(old.y, keep)};
                    }
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = lane + 64 * j, t = sub + i / (D / 2) * TL;
                if (NV * 64 != D / 2 * H && i >= D / 2 * H) continue;
                uint32_t* const at = reinterpret_cast<uint32_t*>(codes + (uint32_t)(sub * D + i % (D / 2) * 32 + i / (D / 2) * TL));
                const bool part = t < lo || t + TL > hi;  // older tokens, or none, among them
                uint32_t out[2][TL / 4];
#pragma unroll
                for (int w = 0; w < TL / 4; ++w) {
                    const uint32_t* const v = xv[j] + 4 * w;
                    uint32_t col[2] = {four_codes<TYPE, P>(elem<BF>(v[0] & 0xFFFF), elem<BF>(v[1] & 0xFFFF), elem<BF>(v[2] & 0xFFFF),
                                                           elem<BF>(v[3] & 0xFFFF), scale),
                                       four_codes<TYPE, P>(elem<BF>(v[0] >> 16), elem<BF>(v[1] >> 16), elem<BF>(v[2] >> 16),
                                                           elem<BF>(v[3] >> 16), scale)};
                    if (part) {
                        // bytes of older tokens stay, or are rounded anew; those behind the last stay
                        uint32_t fresh = 0, older = 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            fresh |= t + 4 * w + q >= lo && t + 4 * w + q < hi ? 0xFFu << 8 * q : 0u;
                            older |= t + 4 * w + q < lo ? 0xFFu << 8 * q : 0u;
                        }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            uint32_t old = at[4 * n + w];
                            if (grew) old = (rounded_anew<TYPE>(old, keep) & older) | (old & ~older);
                            col[n] = (col[n] & fresh) | (old & ~fresh);
                        }
                    }
                    out[0][w] = col[0];
                    out[1][w] = col[1];
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    if constexpr (TL == 16) *reinterpret_cast<u32x4*>(at + 4 * n) = u32x4{out[n][0], out[n][1], out[n][2], out[n][3]};
                    else *reinterpret_cast<u32x2*>(at + 4 * n) = u32x2{out[n][0], out[n][1]};
            }
        }
    };
    // at the range's end a finite value may still exceed the largest code
    if (finite && e < Code<TYPE>::kMaxExp) write(Int<1>());
    else write(Int<0>());
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
uint32_t spans(uint32_t max_q, uint32_t tokens) { return (max_q - 1) / tokens + 1 + (max_q > 1); }

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
