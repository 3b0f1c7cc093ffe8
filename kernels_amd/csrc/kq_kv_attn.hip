// kq_kv_attn.hip -- attention over the 8-bit key/value cache (kq_kv_attn): which
// kernel a call runs, and its launch plan.
#include <algorithm>

#include "kq_kv_attn_kernel.h"

namespace kq {
namespace kv {
namespace {

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Tokens that `rows` rows of a sequence and head see at most, from a multiple of 64 on. Rows of a tree may each see all of them.
uint64_t longest_span(const Batch& b, uint64_t rows, uint32_t window, bool tree) {
    if (tree) rows = b.max_q;
    return window ? std::min<uint64_t>(b.max_len, (uint64_t)window + rows - 1 + kTile - 1) : b.max_len;
}

// Few rows: up to 64, in tiles of 16 or 32. The workgroups of a group read the same codes, which one
// L2 keeps for all of them.
bool few(const Batch& b, uint32_t group) { return (uint64_t)b.max_q * group <= 64; }

// Their groups: all that the device holds at once (two workgroups a compute unit: three were slower, 80 us
// against 64 for 64 sequences of 2486 tokens of 8 heads of 128), or one for each 256 tokens where
// there is less. Where there are enough of them each takes a part of one row of work, for the beginning of
// another costs it about as long as 384 tokens 128 wide do; in equal shares the beginning of a row is priced
// (64 ragged sequences: 94 us without, 73 with). One for each row of work where those are short: up to
// 1024 tokens instead of parts, which a second launch joins (one sequence of 300 tokens 8.2 us a call, in parts
// 11.0; 1000: 11.2, 11.3; 1500: 14.2, 11.4), up to 2048 instead of shares (73 sequences of 100 to 1795
// tokens, 16 heads of 64: 30 us, in shares 34; 48 of 200 to 2500, 8 heads of 128: 40 us, in shares
// 35). So too where the sequences are too many to add up their lengths in each workgroup.
FewPlan few_plan(const Cache& c, const Batch& b, uint32_t D, uint32_t group, uint32_t window, bool tree) {
    FewPlan p = {};
    const uint32_t start = 768 / D;
    const uint32_t q_rows = b.max_q * group;
    p.sixteens = q_rows <= 16 ? 1 : few_sixteens(D);
    p.tiles = (uint32_t)ceil_div(q_rows, 16 * p.sixteens);
    const uint64_t longest = longest_span(b, q_rows, window, tree), rounds = ceil_div(longest, kRound);
    const uint64_t rows = (uint64_t)b.n_seq * c.heads, fit = (uint64_t)cu_count() * few_waves(D) / p.tiles;
    p.groups = (uint32_t)std::min<uint64_t>(fit, rows * rounds);
    p.mode = 2 * rows <= p.groups ? FewPlan::kParts : FewPlan::kShares;
    if (rounds <= (p.mode == FewPlan::kShares ? 8 : 4) || b.n_seq > kScan || b.n_seq * (ceil_div(b.max_len, kTile) + start) >= 0x7FFFFFFF) {
        p.mode = FewPlan::kRows;
        p.groups = (uint32_t)rows;
        return p;
    }
    p.start = p.mode == FewPlan::kShares && rows * rounds >= 4 * fit ? start : 0;
    p.by_row = rows <= p.groups;
    p.cuts = p.by_row ? (uint32_t)rows : p.groups;
    return p;
}
// Descriptors and slots.
size_t few_ws_bytes(const FewPlan& p, uint32_t D) {
    return p.mode == FewPlan::kRows ? 0 : (size_t)p.groups * (sizeof(Cut) + 2 * p.tiles * 16 * p.sixteens * (D + kRowSum) * 4);
}

uint64_t row_splits_wanted(const Cache& c, const Batch& b, const RowPlan& p) {
    return ceil_div((uint64_t)cu_count() * (p.rows == 256 ? 1 : 2), (uint64_t)b.n_seq * p.tiles * c.heads);
}
RowPlan row_plan(const Cache& c, const Batch& b, uint32_t D, uint32_t group, uint32_t window) {
    RowPlan p;
    const uint64_t rows = (uint64_t)b.max_q * group;
    p.rows = rows <= 128 ? 128 : row_most(D);
    p.tiles = (uint32_t)ceil_div(rows, p.rows);
    const uint64_t longest = longest_span(b, p.rows, window, false);
    p.chunk = (uint32_t)std::max<uint64_t>(ceil_div(ceil_div(longest, row_splits_wanted(c, b, p)), kTile) * kTile, kRound);
    p.splits = (uint32_t)ceil_div(longest, p.chunk);
    return p;
}
size_t row_ws_bytes(const Cache& c, const Batch& b, const RowPlan& p, uint64_t splits, uint32_t D) {
    return splits > 1 ? (size_t)b.n_seq * splits * p.tiles * c.heads * p.rows * (D + kRowSum) * 4 : 0;
}

// Many rows of trees: shares and parts as for few rows, of whole units of 64 tokens, among the workgroups that the
// device holds at once. A cut costs more than with few rows, for its 128 or 256 rows' sums are written and read again (256 rows
// of 128 columns: 135 KB): one workgroup for each row of work up to 2048 tokens instead of shares (64 heads over 8 of 128,
// 20-30 rows a sequence; 64 sequences of 1024: 106 us, in shares 134; 32 of 2048: 96, 126; 40 of 256 to 2048: 106, 98;
// 24 of 512 to 4096: 144, 97; 48 of 4096: 287, 272), up to 192 instead of parts (one sequence of 128: 14.0, in parts 15.9;
// 192: 16.2, 16.0; 256: 18.4, 16.2; 1024: 43.9, 22.0). A row's beginning is priced as 5 units of 64 tokens (measured on one batch
// alone, 16 sequences of 300 to 12000 tokens and 33 to 64 rows: 203 us, priced as 2: 213, as 8: 209, as 14: 220). One
// long sequence was faster in splits by the host's bounds, which kq_kv_attn's rows have (60 rows over 131071 tokens: 166 us, in
// shares 176, for a cause not known); that batch took 359 in them.
FewPlan tree_plan(const Cache& c, const Batch& b, uint32_t D, uint32_t group, uint32_t window) {
    FewPlan p = {};
    const uint64_t q_rows = (uint64_t)b.max_q * group;
    const uint32_t tile = q_rows <= 128 ? 128 : row_most(D);
    p.sixteens = tile / 16;
    p.tiles = (uint32_t)ceil_div(q_rows, tile);
    const uint64_t rounds = ceil_div(longest_span(b, q_rows, window, true), kTile);
    const uint64_t rows = (uint64_t)b.n_seq * c.heads, at_once = (uint64_t)cu_count() * (tile == 256 || D >= 192 ? 1 : 2);
    const uint64_t fit = std::max<uint64_t>(at_once / p.tiles, 1);
    p.groups = (uint32_t)std::min<uint64_t>(fit, rows * rounds);
    p.mode = 2 * rows <= p.groups ? FewPlan::kParts : FewPlan::kShares;
    constexpr uint32_t start = 5;
    if (rounds <= (p.mode == FewPlan::kShares ? 32 : 3) || b.n_seq > kScan || b.n_seq * (ceil_div(b.max_len, kTile) + start) >= 0x7FFFFFFF) {
        p.mode = FewPlan::kRows;
        p.groups = (uint32_t)rows;
        return p;
    }
    p.start = p.mode == FewPlan::kShares && rows * rounds >= 4 * fit ? start : 0;
    p.by_row = rows <= p.groups;
    p.cuts = p.by_row ? (uint32_t)rows : p.groups;
    return p;
}

size_t ws_need(const Cache& c, const Batch& b, uint32_t D, uint32_t group, uint32_t window, bool tree) {
    if (few(b, group)) return few_ws_bytes(few_plan(c, b, D, group, window, tree), D);
    if (tree) return few_ws_bytes(tree_plan(c, b, D, group, window), D);
    const RowPlan p = row_plan(c, b, D, group, window);
    return row_ws_bytes(c, b, p, p.splits, D);
}

// Without a window there are the most groups, and shares or parts wherever there are some with one. Splits
// are not as orderly: no window makes more than are wanted, nor of less than a round.
size_t ws_bytes(const Cache& c, const Batch& b, uint32_t D, uint32_t group, bool tree) {
    size_t n = ws_need(c, b, D, group, 0, tree);
    if (!few(b, group) && !tree) {
        const RowPlan p = row_plan(c, b, D, group, 0);
        n = row_ws_bytes(c, b, p, std::min(row_splits_wanted(c, b, p), ceil_div(b.max_len, kRound)), D);
    }
    return n > 256 ? (n + 255) / 256 * 256 : 256;
}

bool fits(const Cache& c, const Batch& b, uint32_t D, uint32_t group, bool tree) {
    if ((uint64_t)b.n_seq * b.max_q * c.heads * group >= 0x7FFF0000ull) return false;
    // Shares, parts and splits are made of few rows of work, and are few.
    const uint64_t rows = (uint64_t)b.n_seq * c.heads;
    if (few(b, group)) return (rows + 7) / 8 * 8 * few_plan(c, b, D, group, 0, tree).tiles <= kMostGroups;
    // of 512 threads count as two
    if (tree) {
        const FewPlan p = tree_plan(c, b, D, group, 0);
        return (rows + 7) / 8 * 8 * p.tiles * (p.sixteens / 8) <= kMostGroups;
    }
    const RowPlan p = row_plan(c, b, D, group, 0);
    return rows * p.tiles * (p.rows / 128) <= kMostGroups;
}

}  // namespace
}  // namespace kv

size_t kv_attn_ws_need(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group, uint32_t window) {
    return kv::ws_need(c, b, D, group, window, false);
}
size_t kv_attn_ws_bytes(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) { return kv::ws_bytes(c, b, D, group, false); }
bool kv_attn_fits(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) { return kv::fits(c, b, D, group, false); }
size_t kv_tree_ws_need(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group, uint32_t window) {
    return kv::ws_need(c, b, D, group, window, true);
}
size_t kv_tree_ws_bytes(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) { return kv::ws_bytes(c, b, D, group, true); }
bool kv_tree_fits(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) { return kv::fits(c, b, D, group, true); }

hipError_t launch_kv_attn(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Attn& a,
                          const kv::Rows& Q, const kv::Rows& O, bool bf, void* ws, hipStream_t s) {
    float* const w = static_cast<float*>(ws);
    return kv::by_dim(D, type, [&](auto d, auto) {
        constexpr int N = decltype(d)::value;
        if (a.mask)
            return kv::few(b, a.group)
                       ? kv::TreeKernels<N>::few(type, c, b, a, kv::few_plan(c, b, D, a.group, a.window, true), Q, O, bf, w, s)
                       : kv::TreeKernels<N>::rows(type, c, b, a, kv::tree_plan(c, b, D, a.group, a.window), Q, O, bf, w, s);
        return kv::few(b, a.group)
                   ? kv::AttnKernels<N>::few(type, c, b, a, kv::few_plan(c, b, D, a.group, a.window, false), Q, O, bf, w, s)
                   : kv::AttnKernels<N>::rows(type, c, b, a, kv::row_plan(c, b, D, a.group, a.window), Q, O, bf, w, s);
    });
}

}  // namespace kq
