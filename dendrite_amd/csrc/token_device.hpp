// Device tables of the token operators (dh_token_tables) as their kernels
// read them: which sequence a unit of work belongs to, what that sequence
// holds, and whether its entries can be trusted.
//
// Units are handed out without a prefix sum over the sequences.  A sequence
// of n rows takes at most ((n * mul) >> shift) + pad units; with f(b) =
// ((q_indptr[b] * mul) >> shift) + pad * b, f(b + 1) - f(b) is at least that, so
// unit u is number u - f(b) of the largest b with f(b) <= u, and the units
// past a sequence's last exit.  f is searched with 64 samples a round (one
// load each for up to 64 sequences, two for 4 096).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dh_device.hpp"

namespace dh {
namespace {

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// What sequence b holds.  ok: its entries are in order (dh_token_tables);
// rows_ok: its rows at least are (row0 .. row0 + nrows inside the call's).
struct Sequence {
    int page0;       // first entry of its table
    int len;         // tokens
    int row0, nrows; // rows of the call that are its own
    int n;           // new tokens (0 for an unused row)
    bool ok, rows_ok;
};

// Sequence b from its table entries p0 .. p1, length, and rows r0 .. r1.
__device__ __forceinline__ Sequence make_sequence(const TokenTables& t, int p0, int p1, int len, int r0, int r1) {
    Sequence s;
    s.page0 = p0;
    s.len = len;
    s.row0 = r0;
    s.rows_ok = r0 >= 0 && r1 >= r0 && uint32_t(r1) <= t.rows;
    s.nrows = s.rows_ok ? r1 - r0 : 0;
    s.n = t.q_indptr ? s.nrows : (len > 0 ? 1 : 0);
    s.ok = s.rows_ok && p0 >= 0 && p1 >= p0 && uint32_t(p1) <= t.num_indices && len >= 0 &&
           uint32_t(len) <= t.max_kv_len && (int64_t(len) + kPageSize - 1) / kPageSize <= p1 - p0 && s.n <= len;
    return s;
}

__device__ __forceinline__ Sequence load_sequence(const TokenTables& t, uint32_t b) {
    const int r0 = t.q_indptr ? t.q_indptr[b] : int(b), r1 = t.q_indptr ? t.q_indptr[b + 1] : int(b) + 1;
    return make_sequence(t, t.indptr[b], t.indptr[b + 1], t.kv_len[b], r0, r1);
}

__device__ __forceinline__ Sequence uniform_sequence(const Sequence& x) {
    Sequence s;
    s.page0 = uniform(x.page0);
    s.len = uniform(x.len);
    s.row0 = uniform(x.row0);
    s.nrows = uniform(x.nrows);
    s.n = uniform(x.n);
    s.ok = uniform(x.ok ? 1 : 0) != 0;
    s.rows_ok = uniform(x.rows_ok ? 1 : 0) != 0;
    return s;
}

// Sequence of unit u and u's number in it.  Every lane of the wave calls it.
// The last of its levels brings what the sequence holds along: a small call's
// time is its dependent loads.
__device__ __forceinline__ Sequence find_sequence(const TokenTables& t, uint64_t u, uint32_t mul, uint32_t shift,
                                                  uint32_t pad, uint32_t& unit) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, n = t.batch;      // the answer is in [lo, lo + n)
    auto number = [&](uint32_t b, int q) { return (uint64_t(uint32_t(q)) * mul >> shift) + uint64_t(pad) * b; };
    while (n > 64) {
        const uint32_t step = (n + 63) / 64, b = min(lo + lane * step, t.batch - 1);
        const uint64_t m = __ballot(lane * step < n && number(b, t.q_indptr[b]) <= u);
        lo += uint32_t(m ? 63 - __builtin_clzll(m) : 0) * step;
        n = min(step, t.batch - lo);
    }
    const uint32_t b = min(lo + lane, t.batch - 1);
    const int r0 = t.q_indptr[b], r1 = t.q_indptr[b + 1], p0 = t.indptr[b], p1 = t.indptr[b + 1], len = t.kv_len[b];
    const uint64_t m = __ballot(lane < n && number(b, r0) <= u);
    const int at = uniform(m ? 63 - __builtin_clzll(m) : 0);
    auto pick = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
    const Sequence s = make_sequence(t, pick(p0), pick(p1), pick(len), pick(r0), pick(r1));
    const uint64_t base = number(uint32_t(uniform(int(lo))) + at, pick(r0));
    unit = uint32_t(uniform(int(u >= base && u - base < 0xFFFFFFFFull ? uint32_t(u - base) : 0xFFFFFFFFu)));
    return uniform_sequence(s);
}

// Whether a sequence that falls to this thread is refused: workgroup w of the
// launch looks at sequences w * blockDim.x + tid (its last ones at the batch's
// last), so a launch of at least batch / blockDim.x workgroups looks at all,
// whichever units find them.  A value, to be reported once other loads are
// under way.
__device__ __forceinline__ bool sees_refused(const TokenTables& t, uint32_t wg) {
    const uint64_t first = uint64_t(wg) * blockDim.x;
    if (first >= t.batch) return false;
    return !load_sequence(t, uint32_t(min(first + threadIdx.x, uint64_t(t.batch - 1)))).ok;
}

__device__ __forceinline__ void report(bool refused, int32_t* status) {
    if (refused && status) *status = DH_EINVAL;
}

// A table entry as a page of the pool: -1 where it is outside it.
__device__ __forceinline__ int checked_page(int id, uint32_t num_pages, int32_t* status) {
    if (uint32_t(id) < num_pages) return id;
    if (id != int(DH_INVALID_PAGE) && status) *status = DH_EINVAL;
    return -1;
}

}  // namespace
}  // namespace dh
