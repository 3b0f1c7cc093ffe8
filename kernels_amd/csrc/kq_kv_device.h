// kq_kv_device.h -- what the kernels of the 8-bit key/value cache share: the
// sequences of a call, the places of tokens, codes and their conversions.
#pragma once
#include "kq_device.h"
#include "kq_internal.h"

namespace kq {
namespace kv {

// Sequence i of a call: `len` tokens in the cache, the last n of them in rows
// row0 .. row0 + n - 1. Whatever the arrays hold, rows and tokens are in bounds.
struct Seq {
    int len, row0, n;
};
__device__ __forceinline__ Seq sequence(const Batch& b, uint32_t page_log2, uint32_t i) {
    Seq s;
    const uint64_t room = (uint64_t)b.max_pages << page_log2;
    const int most = (int)(room < b.max_len ? room : b.max_len), rows = (int)b.n_rows, max_q = (int)b.max_q;
    if (b.q_start) {
        // asked for together: one way to memory, not three
        const int len = b.kv_len[i], from = b.q_start[i], to = b.q_start[i + 1];
        s.len = min(max(len, 0), most);
        s.row0 = min(max(from, 0), rows);
        s.n = min(min(max(to, s.row0), rows) - s.row0, max_q);
    } else {
        s.len = min(max(b.kv_len[i], 0), most);
        s.row0 = (int)i * max_q;
        s.n = max_q;
    }
    return s;
}

// Page of token t of a sequence whose table row is `row`; -1 where the id is no page.
__device__ __forceinline__ int page_of(const Cache& c, const int32_t* row, int t) {
    const int p = row[t >> c.page_log2];
    return (uint32_t)p < c.n_pages ? p : -1;
}

// Offset of a 16-token block's codes (in K and in V alike) and of a token's
// exponent: `t` is any token of the block.
__device__ __forceinline__ uint64_t code_offset(const Cache& c, uint32_t D, int page, uint32_t h, int t) {
    const uint32_t in = (uint32_t)t & ((1u << c.page_log2) - 1) & ~15u;
    return ((((uint64_t)page * c.heads + h) << c.page_log2) + in) * D;
}
__device__ __forceinline__ uint64_t exp_offset(const Cache& c, int page, uint32_t h, int t) {
    const uint32_t in = (uint32_t)t & ((1u << c.page_log2) - 1);
    return (((uint64_t)page * c.heads + h) << (c.page_log2 - c.block_log2)) + (in >> c.block_log2);
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2f(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

constexpr int kMinExp = -64;
template <int TYPE>
struct Code;

template <>
struct Code<KQ_KV_I8> {
    static constexpr float kLargest = 127.0f;
    static constexpr int kMaxExp = 121;
    // The smallest e with a <= 127 * 2^e: a = 1.f * 2^E lies in [64, 128) * 2^(E - 6), and from
    // 127 * 2^(E - 6) (mantissa 0x7E0000) on only just above its end.
    static __device__ __forceinline__ int exponent(float a) {
        const uint32_t u = __builtin_bit_cast(uint32_t, a);
        return (int)(u >> 23) - 127 - 6 + ((u & 0x7FFFFFu) > 0x7E0000u);
    }
    static __device__ __forceinline__ float value(uint32_t byte) { return (float)(int8_t)byte; }
    // Code of y, |y| <= 127.
    static __device__ __forceinline__ uint32_t code(float y) { return (uint32_t)(int)__builtin_rintf(y) & 0xFFu; }
    static __device__ __forceinline__ uint32_t code2(float a, float b) { return code(a) | code(b) << 8; }
};

template <>
struct Code<KQ_KV_E4M3> {
    static constexpr float kLargest = 448.0f;
    static constexpr int kMaxExp = 119;
    // a <= 448 * 2^e = 1.75 * 2^(e + 8): mantissa of 1.75 is 0x600000.
    static __device__ __forceinline__ int exponent(float a) {
        const uint32_t u = __builtin_bit_cast(uint32_t, a);
        return (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    }
    static __device__ __forceinline__ float value(uint32_t byte) {
        return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
    }
    static __device__ __forceinline__ uint32_t code2(float a, float b) {
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xFFFFu;
    }
    static __device__ __forceinline__ uint32_t code(float y) { return code2(y, 0.0f) & 0xFFu; }
};

// The exponent of a block whose largest finite magnitude is a (a subnormal a
// falls below the range whatever its bits say: kMinExp).
template <int TYPE>
__device__ __forceinline__ int block_exponent(float a) {
    return min(max(Code<TYPE>::exponent(a), kMinExp), Code<TYPE>::kMaxExp);
}

// x * scale to its type's range; NaN gives 0.
template <int TYPE>
__device__ __forceinline__ float to_range(float x, float scale) {
    const float y = fminf(fmaxf(x * scale, -Code<TYPE>::kLargest), Code<TYPE>::kLargest);
    return x == x ? y : 0.0f;
}

// Four codes (one dword) as two fp16 pairs, exact. int8: c + 128 in the low byte of
// 0x64xx is 1024 + 128 + c, and an exact packed subtraction takes the 1152 off.
template <int TYPE>
__device__ __forceinline__ void codes_f16(uint32_t w, f16x2& lo, f16x2& hi) {
    if constexpr (TYPE == KQ_KV_I8) {
        const uint32_t u = w ^ 0x80808080u;
        const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    } else {
        lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
        hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true));
    }
}
// Eight codes as an MFMA operand.
template <int TYPE>
__device__ __forceinline__ f16x8 codes_f16x8(uint32_t a, uint32_t b) {
    f16x2 p0, p1, p2, p3;
    codes_f16<TYPE>(a, p0, p1);
    codes_f16<TYPE>(b, p2, p3);
    return f16x8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// 16-bit element of x, fp16 or bf16.
template <int BF>
__device__ __forceinline__ float elem(uint32_t bits) {
    return BF ? bf2f((uint16_t)bits) : h2f((uint16_t)bits);
}
// Two values as a pair of 16-bit elements, rounded to nearest even.
template <int BF>
__device__ __forceinline__ uint32_t pair16(float a, float b) {
    if constexpr (BF) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    } else {
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
    }
}

// Largest of a value over the wave / over lanes l, l ^ 16, l ^ 32, l ^ 48, in every lane.
__device__ __forceinline__ uint32_t across_rows_max(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));
    return across_rows_max(v);
}

}  // namespace kv
}  // namespace kq
