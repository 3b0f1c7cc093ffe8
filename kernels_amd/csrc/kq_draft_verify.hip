// kq_draft_verify.hip -- drafted tokens against the target's probabilities (kq_draft_verify): which
// rows are kept, and the token behind them.
//
// The way down a sequence's rows takes a few probabilities of each: all of them are read at once, then
// the way is found in LDS. Its end is a draw from one row of probabilities, less what was turned down there:
//   P(x) = max(.. max(p(x) - S_1 Q_1(x), 0) .. - S_k Q_k(x), 0), and 0 where x was picked outright,
// which needs the row's sum: workgroups add up kChunk places each, in 64 bits, and a second launch finds the
// chunk and the place in it. A sum is wanted in the middle too where a token drawn from a Q was turned
// down and another continues the same row (trees with Q alone): a workgroup per sequence walks those first. Elsewhere
// every chunk's workgroup finds the way for itself, which takes less than a launch between.
//
// One tree of 60 rows, without Q, over 128256 tokens: 5.8 + 7.1 us, latencies one behind the other (lengths and parents,
// probabilities, the way, the row; then sums, their prefix, the chunk, its prefix). 64 chains of 5 rows with Q: 16.5 +
// 8.8 us for 66 MB, 4 TB/s in the first: each workgroup finds the way before it asks for its 16 KB of P and of Q. Trees with Q are
// far from what their bytes take: of 16 rows that share their parents' Q, 46 us in the walk for one sequence, 197 for 16 and 423 for 64, then
// 13 to 23. A workgroup sums a row up alone for each sibling behind one that was turned down, from P and all the Q so far, a value at a time for
// each thread.
#include <algorithm>

#include "kq_device.h"
#include "kq_internal.h"

namespace kq {
namespace draft {
namespace {

// Sixteen places a thread: 256 workgroups for eight rows of 128k tokens, and few enough sums for one workgroup to join.
constexpr uint32_t kChunk = 4096;

// What the way's end leaves to the draw: its row (-1: the sequence has none), the tokens that were
// picked outright and turned down there, the rows of q that others were drawn from, and how many are kept.
struct End {
    int row, n_out, n_q, count;
    double u;  // the sequence's number for it
};
// A sequence's part of the workspace: End, then the three lists, then the chunks' sums.
struct Places {
    size_t out, rows, mass, sums, size;
};
__host__ __device__ inline Places places(uint32_t max_q, uint32_t chunks) {
    Places p;
    p.out = sizeof(End);
    p.rows = p.out + 4 * (size_t)max_q;
    p.mass = (p.rows + 4 * (size_t)max_q + 7) / 8 * 8;
    p.sums = p.mass + 8 * (size_t)max_q;
    p.size = (p.sums + 8 * (size_t)chunks + 15) / 16 * 16;
    return p;
}

// A sequence's rows: n of them from row0 on, in bounds whatever start holds.
struct Seq {
    int row0, n;
};
__device__ __forceinline__ Seq sequence(const kq_draft& d, uint32_t i) {
    if (!d.start) return {(int)(i * d.max_q), (int)d.max_q};
    const int rows = (int)d.n_rows, from = min(max(d.start[i], 0), rows), to = min(max(d.start[i + 1], from), rows);
    return {from, min(to - from, (int)d.max_q)};
}

// A probability: what is negative or not finite counts as 0.
__device__ __forceinline__ double prob(float p) { return p > 0.0f && p < __builtin_inff() ? (double)p : 0.0; }

// A sequence's rows in LDS, max_q of each (and the lists of what was turned down at the present row).
struct Rows {
    double *p, *q, *mass;  // P(x) and Q(x) of the row's token; S of the lists
    int *parent, *token, *q_row, *out, *rows;
    float* u;
};
__host__ __device__ inline size_t rows_bytes(uint32_t max_q) { return (size_t)max_q * (3 * 8 + 6 * 4); }
__device__ __forceinline__ Rows rows_in(char* lds, uint32_t max_q) {
    Rows r;
    r.p = reinterpret_cast<double*>(lds);
    r.q = r.p + max_q;
    r.mass = r.q + max_q;
    r.parent = reinterpret_cast<int*>(r.mass + max_q);
    r.token = r.parent + max_q;
    r.q_row = r.token + max_q;
    r.out = r.q_row + max_q;
    r.rows = r.out + max_q;
    r.u = reinterpret_cast<float*>(r.rows + max_q);
    return r;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}
// Of all T threads, in every one; lds: T / 64 doubles.
template <int T>
__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double sum = lds[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) sum += lds[i];
    return sum;
}

// The way of a sequence, the same in every thread of the workgroup: lists in r.out, r.rows and r.mass. `writer`
// writes keep and out but for the last token. SUMS: sums in the middle are computed (scratch: T / 64 doubles).
template <int T, bool SUMS>
__device__ __forceinline__ End walk(const kq_draft& d, uint32_t i, const Rows& r, double* scratch, bool writer, int32_t* keep,
                                    int32_t* n_keep, int32_t* out) {
    const Seq s = sequence(d, i);
    const int tid = threadIdx.x, lane = tid & 63;
    keep += (uint64_t)i * d.max_q;
    out += (uint64_t)i * d.max_q;
    for (int j = tid; j < s.n; j += T) {
        const int row = s.row0 + j, x = d.token[row];
        int parent = d.parent ? d.parent[row] : j - 1;
        parent = parent < j ? parent : -1;
        int from = !d.q ? -1 : d.q_index ? d.q_index[row] : row;
        from = (uint32_t)from < d.n_q ? from : -1;
        const bool real = (uint32_t)x < d.vocab && parent >= 0;
        r.parent[j] = parent;
        r.token[j] = x;
        r.q_row[j] = from;
        r.u[j] = d.u[row];
        r.p[j] = real ? prob(d.p[(int64_t)(s.row0 + parent) * d.p_row + x]) : 0.0;
        r.q[j] = from < 0 ? 1.0 : real ? prob(d.q[(int64_t)from * d.q_row + x]) : 0.0;
    }
    __syncthreads();
    End e = {s.n ? s.row0 : -1, 0, 0, s.n ? 1 : 0, s.n ? (double)r.u[0] : 0.0};
    if (writer && tid == 0 && s.n) keep[0] = 0;
    int at = 0, last = 0;  // the present row, and the latest one tried there
    double mass = 1.0;
    bool stale = false;  // mass is to be summed up anew
    while (true) {
        // the next row that continues `at`
        int j = -1;
        for (int base = (last + 1) & ~63; base < s.n; base += 64) {
            const int k = base + lane;
            const uint64_t hit = __ballot(k > last && k < s.n && r.parent[min(k, s.n - 1)] == at);
            if (hit) {
                j = base + __ffsll((unsigned long long)hit) - 1;
                break;
            }
        }
        if (j < 0) break;
        last = j;
        if constexpr (SUMS)
            if (stale) {
                const float* const p = d.p + (int64_t)e.row * d.p_row;
                double sum = 0.0;
                for (uint32_t x = tid; x < d.vocab; x += T) {
                    double v = prob(p[x]);
                    for (int k = 0; k < e.n_q; ++k) v = fmax(v - r.mass[k] * prob(d.q[(int64_t)r.rows[k] * d.q_row + x]), 0.0);
                    for (int k = 0; k < e.n_out; ++k) v = (uint32_t)r.out[k] == x ? 0.0 : v;
                    sum += v;
                }
                mass = block_sum<T>(sum, scratch);
                stale = false;
            }
        // P(x) of its token by now
        const int x = r.token[j], from = r.q_row[j];
        double there = r.p[j];
        for (int k = 0; k < e.n_out; ++k) there = r.out[k] == x ? 0.0 : there;
        if (there > 0.0)
            for (int k = 0; k < e.n_q; ++k) there = fmax(there - r.mass[k] * prob(d.q[(int64_t)r.rows[k] * d.q_row + x]), 0.0);
        if ((double)r.u[j] * mass * r.q[j] < there) {
            at = last = j;
            if (writer && tid == 0) {
                keep[e.count] = j;
                out[e.count - 1] = x;
            }
            e = {s.row0 + j, 0, 0, e.count + 1, e.u};
            mass = 1.0;
            stale = false;
            continue;
        }
        __syncthreads();  // the lists are read no more
        if (from < 0) {
            if (tid == 0) r.out[e.n_out] = x;
            ++e.n_out;
            mass -= there;
        } else {
            if (tid == 0) {
                r.rows[e.n_q] = from;
                r.mass[e.n_q] = mass;
            }
            ++e.n_q;
            stale = true;
        }
        __syncthreads();
    }
    if (writer) {
        if (tid == 0) n_keep[i] = e.count;
        for (int k = e.count + tid; k < (int)d.max_q; k += T) keep[k] = out[k] = -1;
    }
    return e;
}

// The lists into the workspace, or out of it.
template <int T>
__device__ __forceinline__ void put_end(char* ws, const Places& at, const End& e, const Rows& r) {
    if (threadIdx.x == 0) *reinterpret_cast<End*>(ws) = e;
    for (int k = threadIdx.x; k < e.n_out; k += T) reinterpret_cast<int*>(ws + at.out)[k] = r.out[k];
    for (int k = threadIdx.x; k < e.n_q; k += T) {
        reinterpret_cast<int*>(ws + at.rows)[k] = r.rows[k];
        reinterpret_cast<double*>(ws + at.mass)[k] = r.mass[k];
    }
}
template <int T>
__device__ __forceinline__ End get_end(const char* ws, const Places& at, const Rows& r) {
    const End e = *reinterpret_cast<const End*>(ws);
    for (int k = threadIdx.x; k < e.n_out; k += T) r.out[k] = reinterpret_cast<const int*>(ws + at.out)[k];
    for (int k = threadIdx.x; k < e.n_q; k += T) {
        r.rows[k] = reinterpret_cast<const int*>(ws + at.rows)[k];
        r.mass[k] = reinterpret_cast<const double*>(ws + at.mass)[k];
    }
    return e;
}

// Trees with Q: a workgroup per sequence.
constexpr int kWalk = 1024;
__global__ __launch_bounds__(kWalk) void verify_walk_k(kq_draft d, int32_t* keep, int32_t* n_keep, int32_t* out, char* ws, Places at) {
    extern __shared__ __attribute__((aligned(16))) char row_lds[];
    __shared__ double scratch[kWalk / 64];
    const Rows r = rows_in(row_lds, d.max_q);
    const End e = walk<kWalk, true>(d, blockIdx.x, r, scratch, true, keep, n_keep, out);
    put_end<kWalk>(ws + at.size * blockIdx.x, at, e, r);
}

// Places of a chunk that were picked outright, a bit each.
__device__ __forceinline__ void mark_outright(uint32_t* bits, const Rows& r, const End& e, uint32_t c0) {
    for (int k = threadIdx.x; k < (int)kChunk / 32; k += 256) bits[k] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < e.n_out; k += 256) {
        const uint32_t x = (uint32_t)r.out[k] - c0;
        if (x < kChunk) atomicOr(&bits[x / 32], 1u << x % 32);
    }
    __syncthreads();
}

// Rows of probabilities are aligned to a value.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f32x4 load4(const float* row, uint32_t x, uint32_t vocab) {
    f32x4 v = {0, 0, 0, 0};
    if (x + 4 <= vocab) {
        v = *reinterpret_cast<const f32x4u*>(row + x);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (x + k < vocab) v[k] = row[x + k];
    }
    return v;
}
// P of the sixteen places of a thread, four by four: place(k) is the first of the k-th four.
template <class Place>
__device__ __forceinline__ void sixteen(const kq_draft& d, const End& e, const Rows& r, const uint32_t* bits, uint32_t c0, Place place,
                                        double (&v)[16]) {
    const float* const p = d.p + (int64_t)e.row * d.p_row;
    const float* const q0 = d.q + (int64_t)(e.n_q ? r.rows[0] : 0) * d.q_row;
    f32x4 a[4], b[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = load4(p, c0 + place(k), d.vocab);
    if (e.n_q) {  // on their way together
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = load4(q0, c0 + place(k), d.vocab);
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = prob(a[k / 4][k % 4]);
    if (e.n_q) {
        const double mass = r.mass[0];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = fmax(v[k] - mass * prob(b[k / 4][k % 4]), 0.0);
    }
    for (int i = 1; i < e.n_q; ++i) {
        const float* const q = d.q + (int64_t)r.rows[i] * d.q_row;
        const double mass = r.mass[i];
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = load4(q, c0 + place(k), d.vocab);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = fmax(v[k] - mass * prob(b[k / 4][k % 4]), 0.0);
    }
    if (e.n_out) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t x = place(k), gone = bits[x / 32] >> x % 32;
#pragma unroll
            for (int n = 0; n < 4; ++n) v[4 * k + n] = gone >> n & 1 ? 0.0 : v[4 * k + n];
        }
    }
}

// The sum of one chunk (blockIdx.x) of a sequence's last row (.y). WALKED: the way's end is in the workspace;
// else each workgroup walks for itself, and a sequence's first one writes what it found.
template <bool WALKED>
__global__ __launch_bounds__(256) void verify_sums_k(kq_draft d, int32_t* keep, int32_t* n_keep, int32_t* out, char* ws, Places at) {
    extern __shared__ __attribute__((aligned(16))) char row_lds[];
    __shared__ double scratch[4];
    __shared__ uint32_t bits[kChunk / 32];
    const Rows r = rows_in(row_lds, d.max_q);
    ws += at.size * blockIdx.y;
    End e;
    if constexpr (WALKED) {
        e = get_end<256>(ws, at, r);
    } else {
        e = walk<256, false>(d, blockIdx.y, r, scratch, blockIdx.x == 0, keep, n_keep, out);
        if (blockIdx.x == 0) put_end<256>(ws, at, e, r);
    }
    if (e.row < 0) return;
    const uint32_t c0 = blockIdx.x * kChunk;
    mark_outright(bits, r, e, c0);
    double v[16];
    sixteen(d, e, r, bits, c0, [](int k) { return (uint32_t)(k * 256 + threadIdx.x) * 4; }, v);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += v[k];
    sum = block_sum<256>(sum, scratch);
    if (threadIdx.x == 0) reinterpret_cast<double*>(ws + at.sums)[blockIdx.x] = sum;
}

// Sums up to and with each of 256 threads; lds: 4 doubles.
__device__ __forceinline__ double block_prefix(double v, double* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += lds[w];
    return before + v;
}

// A workgroup per sequence draws the last token: among the chunks' sums, then within the chunk.
__global__ __launch_bounds__(256) void verify_draw_k(kq_draft d, int32_t* out, const char* ws, Places at, uint32_t chunks) {
    extern __shared__ __attribute__((aligned(16))) char row_lds[];
    __shared__ double scratch[4], ends[256], before_chunk;
    __shared__ uint32_t bits[kChunk / 32], chunk;
    __shared__ int found;
    const Rows r = rows_in(row_lds, d.max_q);
    const int tid = threadIdx.x;
    ws += at.size * blockIdx.x;
    const double* const sums = reinterpret_cast<const double*>(ws + at.sums);
    const uint32_t each = (chunks + 255) / 256, mine = min(tid * each, chunks), end = min(mine + each, chunks);
    // on their way together with the rest (of a sequence without rows: whatever stands there)
    double part = 0.0;
    for (uint32_t c = mine; c < end; ++c) part += sums[c];
    const End e = get_end<256>(ws, at, r);
    if (e.row < 0) return;
    const double u = e.u;
    ends[tid] = block_prefix(part, scratch);
    if (tid == 0) found = -1;
    __syncthreads();
    const double total = ends[255];
    int32_t* const to = out + (uint64_t)blockIdx.x * d.max_q + e.count - 1;
    if (!(total > 0.0)) {  // nothing is left: the first of the row's largest
        const float* const p = d.p + (int64_t)e.row * d.p_row;
        double best = -1.0;
        uint32_t where = 0;
        for (uint32_t x = tid; x < d.vocab; x += 256) {
            const double v = prob(p[x]);
            if (v > best) best = v, where = x;
        }
        __shared__ uint32_t places_of[256];
        __syncthreads();
        ends[tid] = best;
        places_of[tid] = where;
        __syncthreads();
        if (tid == 0) {
            for (int k = 1; k < 256; ++k)
                if (ends[k] > best || (ends[k] == best && places_of[k] < where)) best = ends[k], where = places_of[k];
            *to = (int)where;
        }
        return;
    }
    // the last thread with a part whose sums begin at the aim or below: for an aim within the sums, the one that
    // passes it. (The first part begins at 0, and a chunk's at the aim at most: there is always one.)
    const double aim = fmax(u * total, 0.0), start = tid ? ends[tid - 1] : 0.0;
    if (part > 0.0 && start <= aim) atomicMax(&found, tid);
    __syncthreads();
    if (tid == found) {
        double up = start;
        uint32_t c = mine, hit = mine;
        for (; c < end; ++c) {
            const double v = sums[c];
            if (v > 0.0) hit = c, before_chunk = up;
            up += v;
            if (v > 0.0 && up > aim) break;
        }
        chunk = hit;
    }
    __syncthreads();
    const uint32_t c0 = chunk * kChunk;
    const double before = before_chunk;
    if (tid == 0) found = -1;  // read by all before the last barrier but one
    mark_outright(bits, r, e, c0);
    double v[16];
    sixteen(d, e, r, bits, c0, [](int k) { return (uint32_t)threadIdx.x * 16 + 4 * k; }, v);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += v[k];
    ends[tid] = block_prefix(sum, scratch);
    __syncthreads();
    const double from = before + (tid ? ends[tid - 1] : 0.0);
    if (sum > 0.0 && from <= aim) atomicMax(&found, tid);
    __syncthreads();
    if (tid == found) {
        double up = from;
        int hit = 0;
        bool passed = false;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (!passed && v[k] > 0.0) hit = k;
            up += v[k];
            passed = passed || (v[k] > 0.0 && up > aim);
        }
        *to = (int)(c0 + tid * 16 + hit);
    }
}

uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }

}  // namespace
}  // namespace draft

size_t draft_verify_ws_bytes(uint32_t n_seq, uint32_t max_q, uint32_t vocab) {
    return (n_seq * draft::places(max_q, draft::chunks_of(vocab)).size + 255) / 256 * 256;
}

hipError_t launch_draft_verify(const kq_draft& d, int32_t* keep, int32_t* n_keep, int32_t* out, void* ws, hipStream_t s) {
    const uint32_t chunks = draft::chunks_of(d.vocab);
    const draft::Places at = draft::places(d.max_q, chunks);
    const size_t lds = draft::rows_bytes(d.max_q);
    char* const w = static_cast<char*>(ws);
    const dim3 grid(chunks, d.n_seq);
    if (d.q && d.parent) {
        draft::verify_walk_k<<<d.n_seq, draft::kWalk, lds, s>>>(d, keep, n_keep, out, w, at);
        draft::verify_sums_k<true><<<grid, 256, lds, s>>>(d, keep, n_keep, out, w, at);
    } else {
        draft::verify_sums_k<false><<<grid, 256, lds, s>>>(d, keep, n_keep, out, w, at);
    }
    draft::verify_draw_k<<<d.n_seq, 256, lds, s>>>(d, out, w, at, chunks);
    return hipGetLastError();
}

}  // namespace kq
