// Blocks of query rows of the windowed attention kernels: which sequence, KV
// head and rows a workgroup has, and which pages those rows see.
//
// Row rho of a sequence is query head offset rho % r of its new token rho / r
// (r query heads share a KV head), so the rows of a block cover neighbouring
// positions and read nearly the same tokens.  A row at position p sees
// tokens t <= p with t > p - window or t < sinks; a block's pages are those of
// its sinks that lie before its window, then its window's, one list of
// `pages` entries.
#pragma once
#include "token_device.hpp"

namespace dh {
namespace {

struct RowBlock {
    Sequence seq;
    int rho0, nrows;      // first row, rows (0: the block does not exist)
    int kv_head;
    int pmin, pmax;       // positions of the first and the last row
    int sink_pages;       // list entries before the window's
    int window_page;      // the window's first page of the table
    int pages;            // entries of the list
    bool zero;            // rows of a refused or unused sequence: zeros
};

// Block `unit` of `kRows` rows (a power of two, 1 << SHIFT), KV head kv_head.
template <int SHIFT>
__device__ __forceinline__ RowBlock find_rows(const WindowArgs& a, uint64_t unit, int kv_head) {
    RowBlock k{};
    k.kv_head = kv_head;
    uint32_t u;
    if (a.t.q_indptr) {
        k.seq = find_sequence(a.t, unit, a.r, SHIFT, 1, u);
    } else {
        const uint32_t per = (a.r + (1u << SHIFT) - 1) >> SHIFT;
        if (unit >= uint64_t(a.t.batch) * per) return k;
        const uint32_t b = per == 1 ? uint32_t(unit) : uint32_t(unit) / per;
        u = uint32_t(unit) - b * per;
        k.seq = uniform_sequence(load_sequence(a.t, b));
    }
    const int64_t rows = int64_t(k.seq.nrows) * a.r, rho0 = int64_t(u) << SHIFT;
    if (rho0 >= rows) return k;
    k.rho0 = int(rho0);
    k.nrows = int(min(int64_t(1) << SHIFT, rows - rho0));
    k.zero = !k.seq.ok || k.seq.n == 0;
    if (k.zero) return k;
    const int first = k.seq.len - k.seq.n;
    k.pmin = first + int(a.by_r(k.rho0));
    k.pmax = first + int(a.by_r(k.rho0 + k.nrows - 1));
    const int lo = a.window ? max(0, k.pmin - a.window + 1) : 0;
    k.window_page = lo >> 4;
    k.sink_pages = a.window ? min((min(a.sinks, k.pmax + 1) + 15) >> 4, k.window_page) : 0;
    k.pages = k.sink_pages + (k.pmax >> 4) + 1 - k.window_page;
    return k;
}

// The same, told to the compiler as wave-uniform once more: the fields merge
// over find_rows' early returns, after which it holds them in vector registers
// and masks execution where a scalar branch will do.
__device__ __forceinline__ RowBlock uniform_block(const RowBlock& x) {
    RowBlock k;
    k.seq = uniform_sequence(x.seq);
    k.rho0 = uniform(x.rho0);
    k.nrows = uniform(x.nrows);
    k.kv_head = uniform(x.kv_head);
    k.pmin = uniform(x.pmin);
    k.pmax = uniform(x.pmax);
    k.sink_pages = uniform(x.sink_pages);
    k.window_page = uniform(x.window_page);
    k.pages = uniform(x.pages);
    k.zero = uniform(x.zero ? 1 : 0) != 0;
    return k;
}

// The block, and the part of its page list, of a workgroup of a wide kernel: KV
// heads fastest (neighbouring pages' planes), then parts, then blocks.
struct BlockPart {
    uint32_t unit;
    int head, split, parts;
    uint32_t place;         // the block's in the tail (0 where there is none)
};

// TAIL: the call may have one (a.tail).
template <bool TAIL>
__device__ __forceinline__ BlockPart block_part(const WindowArgs& a) {
    uint32_t x = blockIdx.x, split = 0, parts = a.splits, place = 0;
    if (TAIL && x >= a.tail) {
        place = a.by_tail(x - a.tail);
        parts = a.tail_parts;
        split = x - a.tail - place * parts;
        x = a.tail + place;
    }
    const uint32_t x0 = a.by_hkv(x), unit = a.by_splits(x0);
    return {unit, uniform(int(x - x0 * a.hkv)), uniform(int(split + x0 - unit * a.splits)), uniform(int(parts)), place};
}

// Entries of a part of the list.
template <bool TAIL>
__device__ __forceinline__ int part_pages(const WindowArgs& a, const BlockPart& b, int pages) {
    const uint32_t n = uint32_t(pages) + uint32_t(b.parts) - 1;
    return uniform(int(TAIL && blockIdx.x >= a.tail ? a.by_tail(n) : a.by_splits(n)));
}

// Where row i of the block (of `rows`), row `at` of the call, keeps its state.
template <bool TAIL>
__device__ __forceinline__ uint64_t state_slot(const WindowArgs& a, const BlockPart& b, int rows, int i, uint64_t at,
                                               int head) {
    const uint64_t row = TAIL && blockIdx.x >= a.tail ? uint64_t(b.place) * rows + i : at * a.hq + head;
    return row * b.parts + b.split;
}

// Page of the table that list entry j stands for.
__device__ __forceinline__ int list_page(const RowBlock& k, int j) {
    return j < k.sink_pages ? j : k.window_page + j - k.sink_pages;
}

// Row rho's offset (in rows of q / out) and query head.
__device__ __forceinline__ void row_place(const WindowArgs& a, const RowBlock& k, int rho, int& token, int& head) {
    token = int(a.by_r(rho));
    const int j = rho - token * int(a.r);
    head = a.tiled ? k.kv_head + j * int(a.hkv) : k.kv_head * int(a.r) + j;
}

// FP8 blocks: V's scale v goes into the weights, as log2 v beside the score, so
// that the reference a row's weights are kept near is that of weight times
// scale: 16-bit weights then keep their precision whatever the scale.  Below
// 2^-64, the least that an append writes, a scale counts as that (a page nobody
// wrote may hold zero).  The row's sum takes the scales out again, 2^(s - m) up
// to 2^(64 + 8) a token and down to 2^-119 for the largest scales: it is counted
// in units of 2^-32, which keeps either end within f32.
constexpr float kSumUnitLog2 = 32.f, kSumUnit = 0x1p-32f;
__device__ __forceinline__ float value_log2(float v) { return __builtin_amdgcn_logf(fmaxf(v, 0x1p-64f)); }

// Zero rows of a refused or unused sequence.
typedef uint32_t word16 __attribute__((ext_vector_type(4)));
template <int D, uint32_t QT>
__device__ __forceinline__ void zero_rows(const WindowArgs& a, const RowBlock& k) {
    constexpr int EB = QT == DH_DTYPE_F32 ? 4 : 2, W = D * EB / 16;      // 16-byte words a row
    for (int i = threadIdx.x; i < k.nrows * W; i += blockDim.x) {
        int token, head;
        row_place(a, k, k.rho0 + i / W, token, head);
        reinterpret_cast<word16*>(a.out + (uint64_t(k.seq.row0) + token) * a.out_stride + uint64_t(head) * D * EB)[i % W] =
            word16{0u, 0u, 0u, 0u};
    }
}

// Blocks of 1 << shift rows the call may need (find_rows' numbering).
inline uint64_t row_blocks(const WindowArgs& a, int shift) {
    if (!a.t.q_indptr) return uint64_t(a.t.batch) * ((a.r + (1u << shift) - 1) >> shift);
    return (uint64_t(a.t.rows) * a.r >> shift) + a.t.batch;
}

// Workgroups of a wide kernel.
inline uint64_t wide_workgroups(const WindowArgs& a, int shift) {
    const uint64_t n = row_blocks(a, shift) * a.hkv;
    return a.tail == kNoTail ? n * a.splits : a.tail + (n - a.tail) * a.tail_parts;
}

}  // namespace
}  // namespace dh
