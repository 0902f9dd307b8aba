// Windowed attention of few query rows a sequence, from device tables: single
// tokens and short chunks (dh_attend_window), and the merge of split work.
//
// A workgroup of 4, 8 or 16 waves has one block of 16 rows (one MFMA tile) of
// one KV head and one of `splits` equal parts of the block's page list; each
// wave takes its share of the part, a pair of pages (32 tokens) at a time, with
// the loads of the next pair in flight behind the math of the current one:
//   s = scale q K^T, m' = max(m, max s), O = O 2^(m - m') + 2^(s - m') V,
//   L = L 2^(m - m') + sum 2^(s - m')   (s in log2 units)
// with S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32 (16x16x4 for
// f32), operands straight from global memory (attend_device.hpp's layout).
// The waves' states are joined in LDS; with several parts each workgroup
// writes (O, m, L) in f32 and a merge kernel joins them.
//
// Every page is read once per block.  Large batches are bound by those bytes (64
// sequences under a window of 4096, bf16, 32 heads of 128: 152 us, 6.1 TB/s; 256
// in FP8 under 1024 + 64, 64 heads: 101 us, 5.1; one token over 100 000, f16, 16
// heads of 256: 38 us, 5.3), blocks of several tokens by 8-bit conversion (32
// sequences of 3 to 9 tokens in MXFP8, 16 heads of 256: 42 us), small calls by
// their dependent loads (one f32 token under a window of 256: 9.1 us).
#include "attend_device.hpp"
#include "window_device.hpp"

namespace dh {
namespace {

// Whether the lanes' shares of a page's V make whole lines of its rows (8 or 16
// bytes each): only then can V be loaded without leaving lines behind, since
// parts of lines would be fetched again.
template <int D, uint32_t KVF>
constexpr bool kWholeLines = D / 16 * (PageRaw<D, KVF>::FP8 ? 1 : 2) == 8 || D / 16 * (PageRaw<D, KVF>::FP8 ? 1 : 2) == 16;

// A page's V as load_page_v has it, in loads that leave no line behind.
template <int D, uint32_t KVF>
__device__ __forceinline__ void load_v_once(PageRaw<D, KVF>& r, const AttendArgs& kv, uint32_t page, uint32_t head, int g,
                                            int c) {
    using R = PageRaw<D, KVF>;
    constexpr int EB = R::FP8 ? 1 : 2, W = R::EPL * EB / 4;
    typedef uint32_t words __attribute__((ext_vector_type(W)));
    const uint8_t* p = kv.kv + plane_offset(page, 1, head, kv.hkv, D, EB) + (4 * g * D + c * R::EPL) * EB;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        const words v = __builtin_nontemporal_load(reinterpret_cast<const words*>(p + j * D * EB));
        #pragma unroll
        for (int w = 0; w < W; ++w) r.v[j][w] = v[w];
    }
    if constexpr (KVF == KVF_MX) {
        const uint8_t* s = reinterpret_cast<const uint8_t*>(kv.scales) +
                           ((uint64_t(page) * 2 + 1) * kv.hkv + head) * uint64_t(kPageSize) * R::G;
        #pragma unroll
        for (int j = 0; j < 4; ++j) r.vsc[j] = s[(4 * g + j) * R::G + c * R::EPL / 32];
    }
}

// The page ids of a wave's part of the list, kNarrowWavePages at most, in
// registers (lane l holds entries l, l + 64, ...): -1 for an entry outside the
// pool, whose tokens nobody sees.
struct WavePages {
    int id[kNarrowWavePages / 64];
    int j0, n;      // first list entry, entries

    // Part `part` of a.splits NW.
    template <int NW>
    __device__ __forceinline__ void load(const WindowArgs& a, const RowBlock& k, int part) {
        int per = uniform(int(a.by_splits(uint32_t(k.pages) + a.splits * NW - 1) / NW));
        per += per & 1;
        j0 = min(part * per, k.pages);
        n = min(min(per, k.pages - j0), int(kNarrowWavePages));
        const int lane = threadIdx.x & 63;
        #pragma unroll
        for (int i = 0; i < int(kNarrowWavePages / 64); ++i) {
            const int j = lane + 64 * i;
            id[i] = -1;
            if (j < n) id[i] = checked_page(a.t.indices[k.seq.page0 + list_page(k, j0 + j)], a.page_limit, a.status);
        }
    }
    __device__ __forceinline__ int at(int j) const {
        int r = -1;
        #pragma unroll
        for (int i = 0; i < int(kNarrowWavePages / 64); ++i)
            if ((j >> 6) == i) r = __builtin_amdgcn_readlane(id[i], j & 63);
        return j < n ? r : -1;
    }
};

// Tokens of a page (base token t0) that one row at position p sees.
struct Sight {
    int p, lo, sinks;     // t <= p and (t >= lo or t < sinks)
    __device__ __forceinline__ bool sees(int t) const { return t <= p && (t >= lo || t < sinks); }
};

__device__ __forceinline__ int window_lo(const WindowArgs& a, int p) { return a.window ? p - a.window + 1 : 0; }

// Whether every row of a block sees all of a page / any row sees any of it.
__device__ __forceinline__ bool all_see(const WindowArgs& a, int pmin, int pmax, int t0) {
    return t0 + 15 <= pmin && (t0 >= window_lo(a, pmax) || t0 + 15 < a.sinks);
}

// Joins the states of the workgroup's waves and writes the block's rows:
// to out, or as one part's state to the workspace.  Lane (g, c) holds
// O[row c][(4g + i) * EPL + e] = O[e][i], L its row's sum (already over the
// four lanes of the row) and m the row's reference.
template <int D, uint32_t QT, int NW>
__device__ __forceinline__ void join_waves(const WindowArgs& a, const RowBlock& k, int split, float m, float L,
                                           const f4 (&O)[D / 16], float* lds) {
    constexpr int EPL = D / 16, RS = D + 4;          // padded row
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
    float* o = lds + wave * 16 * RS;
    float* ml = lds + NW * 16 * RS;              // [wave][16][2]
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        #pragma unroll
        for (int e = 0; e < EPL; e += 4)
            *reinterpret_cast<f4*>(o + c * RS + (4 * g + i) * EPL + e) = f4{O[e][i], O[e + 1][i], O[e + 2][i], O[e + 3][i]};
    if (g == 0) {
        ml[(wave * 16 + c) * 2] = m;
        ml[(wave * 16 + c) * 2 + 1] = L;
    }
    __syncthreads();
    const int row = tid >> 4, d0 = (tid & 15) * EPL;
    if (tid >= 256 || row >= k.nrows) return;
    float mx = kNegInf;
    #pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, ml[(w * 16 + row) * 2]);
    float x[EPL], sum = 0.f;
    #pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = 0.f;
    #pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float mw = ml[(w * 16 + row) * 2];
        const float al = mw == kNegInf ? 0.f : fast_exp2(mw - mx);
        sum += al * ml[(w * 16 + row) * 2 + 1];
        const f4* p = reinterpret_cast<const f4*>(lds + (w * 16 + row) * RS + d0);
        #pragma unroll
        for (int e = 0; e < EPL; e += 4) {
            const f4 v = p[e / 4];
            #pragma unroll
            for (int i = 0; i < 4; ++i) x[e + i] += al * v[i];
        }
    }
    int token, head;
    row_place(a, k, k.rho0 + row, token, head);
    const uint64_t at = uint64_t(k.seq.row0) + token;
    if (a.splits > 1) {
        const uint64_t slot = (at * a.hq + head) * a.splits + split;
        f4* p = reinterpret_cast<f4*>(a.ws_o + slot * D + d0);
        #pragma unroll
        for (int e = 0; e < EPL; e += 4) p[e / 4] = f4{x[e], x[e + 1], x[e + 2], x[e + 3]};
        if ((tid & 15) == 0) *reinterpret_cast<f2*>(a.ws_ml + slot * 2) = f2{mx, sum};
        return;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    if constexpr (QT == DH_DTYPE_F32) {
        f4* p = reinterpret_cast<f4*>(a.out + at * a.out_stride + (uint64_t(head) * D + d0) * 4);
        #pragma unroll
        for (int e = 0; e < EPL; e += 4) p[e / 4] = f4{x[e] * inv, x[e + 1] * inv, x[e + 2] * inv, x[e + 3] * inv};
    } else {
        uint32_t w[EPL / 2];
        #pragma unroll
        for (int e = 0; e < EPL; e += 2) w[e / 2] = pack2(x[e] * inv, x[e + 1] * inv, QT == DH_DTYPE_F16);
        store_u32s<EPL / 2>(reinterpret_cast<uint16_t*>(a.out + at * a.out_stride) + uint64_t(head) * D + d0, w);
    }
}

// The block of a workgroup: KV heads fastest (neighbouring pages' planes),
// then parts, then blocks.
template <int SHIFT>
__device__ __forceinline__ RowBlock workgroup_rows(const WindowArgs& a, int& split) {
    const bool refused = sees_refused(a.t, blockIdx.x);
    const uint32_t x = a.by_hkv(blockIdx.x);
    const int head = uniform(int(blockIdx.x - x * a.hkv));
    const uint32_t unit = a.by_splits(x);
    split = uniform(int(x - unit * a.splits));
    const RowBlock k = uniform_block(find_rows<SHIFT>(a, unit, head));
    report(refused, a.status);
    return k;
}

// Waves a SIMD the registers are to leave room for.  8-bit pages are converted a
// block of dims at a time, as the products take them, and need few: whole
// operands (64 sequences of 5000 tokens in MXFP8, 64 heads of 128: 129 us
// against 126, 40 of 2000: 45 against 39; 32 verifying 6 tokens, 16 heads of
// 256, window 2001: 61 against 49) leave room for one wave less, at 256 dims for
// one only.
template <int D, bool CODES>
constexpr int kNarrowPerSimd = !CODES ? 1 : D == 256 ? 2 : D == 128 ? 3 : 4;

template <int D, uint32_t KVF, bool F16, int NW, bool ONCE>
__global__ __launch_bounds__(64 * NW, (kNarrowPerSimd<D, PageRaw<D, KVF>::FP8>)) void window_narrow_kernel(WindowArgs a) {
    using R = PageRaw<D, KVF>;
    constexpr int KB = D / 32, EPL = D / 16;
    constexpr uint32_t QT = F16 ? DH_DTYPE_F16 : DH_DTYPE_BF16;
    __shared__ __attribute__((aligned(16))) float lds[NW * 16 * (D + 4) + NW * 32];
    int split;
    const RowBlock k = workgroup_rows<4>(a, split);
    if (k.nrows == 0) return;
    if (k.zero) {
        if (split == 0 && a.splits == 1) zero_rows<D, QT>(a, k);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), g = lane >> 4, c = lane & 15;
    WavePages pages;
    pages.load<NW>(a, k, split * NW + wave);

    // Query rows as B operands: lane (g, c) holds row c.
    const int rho = k.rho0 + min(c, k.nrows - 1);
    int token, head;
    row_place(a, k, rho, token, head);
    uint32_t qB[1][KB][4];
    {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q + (uint64_t(k.seq.row0) + token) * a.q_stride) +
                             uint64_t(head) * D;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            load_dwords<4>(qB[0][kb], qp + (R::FP8 ? 64 * (kb >> 1) + 16 * g + 8 * (kb & 1) : kb * 32 + 8 * g));
            #pragma unroll
            for (int i = 0; i < 4; ++i) qB[0][kb][i] ^= a.q_sign;
        }
    }
    Sight row;
    row.p = k.seq.len - k.seq.n + token;
    row.lo = window_lo(a, row.p);
    row.sinks = a.sinks;
    const Sight any{k.pmax, window_lo(a, k.pmin), a.sinks};    // what some row of the block sees

    float m = kNegInf, l = 0.f;
    f4 O[EPL];
    #pragma unroll
    for (int e = 0; e < EPL; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    AttendArgs kv{};
    kv.kv = a.kv;
    kv.scales = a.scales;
    kv.hkv = a.hkv;
    const float* bsc = reinterpret_cast<const float*>(a.scales);

    R pr[2];
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
    auto load_k = [&](int pair) {
        #pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int id = pages.at(2 * pair + q);
            const uint32_t pg = uint32_t(max(id, 0));
            load_page_k<D, KVF>(pr[q], kv, pg, k.kv_head, g, c);
            if constexpr (KVF == KVF_FP8) ks[q] = id < 0 ? 1.f : bsc[(uint64_t(pg) * 2 + 0) * a.hkv + k.kv_head];
        }
    };
    auto load_values = [&](int pair) {
        #pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int id = pages.at(2 * pair + q);
            const uint32_t pg = uint32_t(max(id, 0));
            if constexpr (ONCE) load_v_once<D, KVF>(pr[q], kv, pg, k.kv_head, g, c);
            else load_page_v<D, KVF>(pr[q], kv, pg, k.kv_head, g, c);
            if constexpr (KVF == KVF_FP8) vs[q] = id < 0 ? 1.f : bsc[(uint64_t(pg) * 2 + 1) * a.hkv + k.kv_head];
        }
    };
    const int npairs = (pages.n + 1) >> 1;
    if (npairs > 0) {
        load_k(0);
        load_values(0);
    }
    #pragma unroll 1
    for (int pi = 0; pi < npairs; ++pi) {
        // 8-bit pages are loaded past the list's end too (page 0): a load on some
        // paths only makes every wait for others stricter (64 sequences of 5000
        // tokens in MXFP8, 64 heads of 128: 132 us, and 144 with the branch).
        // 16-bit pages lose more by those extra loads (32 sequences of 3 new
        // tokens, 32 heads of 64, window 2001: 32 us, and 30 with the branch).
        const bool refill = R::FP8 || pi + 1 < npairs;
        int t0[2];
        bool ok[2], full = true;
        #pragma unroll
        for (int q = 0; q < 2; ++q) {
            ok[q] = pages.at(2 * pi + q) >= 0;
            t0[q] = 16 * list_page(k, pages.j0 + 2 * pi + q);
            full = full && ok[q] && all_see(a, k.pmin, k.pmax, t0[q]);
        }
        f4 s[1][2];
        if constexpr (R::FP8) {
            s[0][0] = s[0][1] = f4{0.f, 0.f, 0.f, 0.f};
            #pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                #pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float sc = KVF == KVF_MX ? e8m0_to_float(pr[q].ksc[kb]) : 1.f;
                    uint32_t op[4];
                    e4m3x4_cvt<F16>(pr[q].k[kb][0], sc, op[0], op[1]);
                    e4m3x4_cvt<F16>(pr[q].k[kb][1], sc, op[2], op[3]);
                    s[0][q] = mma16<F16>(op, qB[0][kb], s[0][q]);
                }
        } else {
            uint32_t kop[2][KB][4];
            k_operand<D, KVF, F16>(pr[0], kop[0]);
            k_operand<D, KVF, F16>(pr[1], kop[1]);
            pair_scores<D, F16, 1, 1>(kop[0], kop[1], qB, s);
        }
        // A scale of zero (a page nobody wrote) must not meet a masked -inf.
        const float f0 = KVF == KVF_FP8 ? fmaxf(a.scale_log2 * ks[0], 1e-30f) : a.scale_log2;
        const float f1 = KVF == KVF_FP8 ? fmaxf(a.scale_log2 * ks[1], 1e-30f) : a.scale_log2;
        const float v0 = KVF == KVF_FP8 ? value_log2(vs[0]) : 0.f, v1 = KVF == KVF_FP8 ? value_log2(vs[1]) : 0.f;
        if (refill) load_k(pi + 1);
        // V of tokens nobody sees: their weights are zero, but what lies there
        // need not be a number.
        if (!full) {
            #pragma unroll
            for (int q = 0; q < 2; ++q)
                #pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool keep = ok[q] && any.sees(t0[q] + 4 * g + j);
                    #pragma unroll
                    for (int w = 0; w < R::VW; ++w) pr[q].v[j][w] = keep ? pr[q].v[j][w] : 0u;
                    if constexpr (KVF == KVF_MX) pr[q].vsc[j] = keep ? pr[q].vsc[j] : 127u;
                }
        }
        float x[8];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = s[0][0][i];
            x[4 + i] = s[0][1][i];
        }
        if (!full) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(ok[0] && row.sees(t0[0] + 4 * g + i))) x[i] = kNegInf;
                if (!(ok[1] && row.sees(t0[1] + 4 * g + i))) x[4 + i] = kNegInf;
            }
        }
        const float r0 = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), r1 = fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]));
        const float lm = KVF == KVF_FP8 ? fmaxf(__builtin_fmaf(r0, f0, v0), __builtin_fmaf(r1, f1, v1)) : fmaxf(r0 * f0, r1 * f1);
        // The reference moves only when a score passes it by 8 (2^8 at most
        // then), so the accumulators are seldom rescaled.
        if (__ballot(lm > m + 8.f)) {
            const float mx = rowgroup_max(lm);
            const float mnew = mx > m + 8.f ? mx : m;
            const float alpha = m == kNegInf ? 0.f : fast_exp2(m - mnew);
            m = mnew;
            l *= alpha;
            #pragma unroll
            for (int e = 0; e < EPL; ++e) O[e] *= alpha;
        }
        const float nm = m == kNegInf ? 0.f : -m;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = fast_exp2(__builtin_fmaf(x[i], f0, nm + v0));
            x[4 + i] = fast_exp2(__builtin_fmaf(x[4 + i], f1, nm + v1));
        }
        // Each weight as two 16-bit numbers, the second the first one's rounding
        // error: alone, the first's errors (2^-9 relative in bf16, 2^-12 in f16)
        // are in the output as large as its own rounding, whatever the number of
        // tokens.  The sum is of the weights before that, in f32.  A wave waits
        // for its pages: the second products cost it 1 %.
        uint32_t hi[4], lo[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = pack2(x[2 * i], x[2 * i + 1], F16);
            lo[i] = pack2(x[2 * i] - unpack_lo(hi[i], F16), x[2 * i + 1] - unpack_hi(hi[i], F16), F16);
        }
        const float l0 = (x[0] + x[1]) + (x[2] + x[3]), l1 = (x[4] + x[5]) + (x[6] + x[7]);
        if constexpr (KVF == KVF_FP8)
            l = __builtin_fmaf(l0, fast_exp2(kSumUnitLog2 - v0), __builtin_fmaf(l1, fast_exp2(kSumUnitLog2 - v1), l));
        else
            l += l0 + l1;
        // O^T += V^T P^T of dims e, given its dword w of tokens (q, j)
        auto product = [&](int e, auto&& w) __attribute__((always_inline)) {
            const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
            const uint32_t vA[4] = {__builtin_amdgcn_perm(w(0, 1), w(0, 0), sel), __builtin_amdgcn_perm(w(0, 3), w(0, 2), sel),
                                    __builtin_amdgcn_perm(w(1, 1), w(1, 0), sel), __builtin_amdgcn_perm(w(1, 3), w(1, 2), sel)};
            O[e] = mma16<F16>(vA, hi, O[e]);
            O[e] = mma16<F16>(vA, lo, O[e]);
        };
        if constexpr (R::FP8) {
            #pragma unroll
            for (int i = 0; i < R::VW; ++i) {      // four dims
                uint32_t op[2][4][2];
                #pragma unroll
                for (int q = 0; q < 2; ++q)
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        e4m3x4_cvt<F16>(pr[q].v[j][i], KVF == KVF_MX ? e8m0_to_float(pr[q].vsc[j]) : 1.f, op[q][j][0],
                                        op[q][j][1]);
                #pragma unroll
                for (int e = 0; e < 4; ++e)
                    product(4 * i + e, [&](int q, int j) __attribute__((always_inline)) { return op[q][j][e >> 1]; });
            }
        } else {
            #pragma unroll
            for (int e = 0; e < EPL; ++e)
                product(e, [&](int q, int j) __attribute__((always_inline)) { return pr[q].v[j][e >> 1]; });
        }
        if (refill) load_values(pi + 1);
    }
    join_waves<D, QT, NW>(a, k, split, m, rowgroup_sum(l) * (KVF == KVF_FP8 ? kSumUnit : 1.f), O, lds);
}

// f32 queries and cache: one page a step on v_mfma_f32_16x16x4_f32, which bounds
// chunks (1024 tokens x 32 heads of 128 over 2000: 488 us, 86 TFLOP/s; a large
// library product reaches 153); few rows are bound by their pages' bytes.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW) void window_narrow32_kernel(WindowArgs a) {
    constexpr int KQ = D / 4, EPL = D / 16;
    __shared__ __attribute__((aligned(16))) float lds[NW * 16 * (D + 4) + NW * 32];
    int split;
    const RowBlock k = workgroup_rows<4>(a, split);
    if (k.nrows == 0) return;
    if (k.zero) {
        if (split == 0 && a.splits == 1) zero_rows<D, DH_DTYPE_F32>(a, k);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), g = lane >> 4, c = lane & 15;
    WavePages pages;
    pages.load<NW>(a, k, split * NW + wave);
    const int rho = k.rho0 + min(c, k.nrows - 1);
    int token, head;
    row_place(a, k, rho, token, head);
    float qv[KQ];
    load_dwords<KQ>(reinterpret_cast<uint32_t*>(qv),
                    a.q + (uint64_t(k.seq.row0) + token) * a.q_stride + (uint64_t(head) * D + g * KQ) * 4);
    #pragma unroll
    for (int i = 0; i < KQ; ++i) qv[i] = __uint_as_float(__float_as_uint(qv[i]) ^ a.q_sign);
    Sight row;
    row.p = k.seq.len - k.seq.n + token;
    row.lo = window_lo(a, row.p);
    row.sinks = a.sinks;
    const Sight any{k.pmax, window_lo(a, k.pmin), a.sinks};
    float m = kNegInf, l = 0.f;
    f4 O[EPL];
    #pragma unroll
    for (int e = 0; e < EPL; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    float kb[KQ], vb[4][EPL];
    // One wave a SIMD (256 dims) has nothing to do while K lands: it is loaded
    // as soon as the scores are done, past the list's end too (page 0; 1024
    // tokens x 16 heads over 2000: 474 us, and 535 at the step's end).  More waves
    // do not gain by it (256 tokens x 32 heads of 128: 119 us, and 115).
    constexpr bool EARLY = D == 256;
    auto load_k = [&](int j) {
        const uint8_t* kp = a.kv + plane_offset(uint32_t(max(pages.at(j), 0)), 0, k.kv_head, a.hkv, D, 4);
        load_dwords<KQ>(reinterpret_cast<uint32_t*>(kb), kp + (c * D + g * KQ) * 4);
    };
    auto load_v = [&](int j) {
        const uint8_t* vp = a.kv + plane_offset(uint32_t(max(pages.at(j), 0)), 1, k.kv_head, a.hkv, D, 4);
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            load_dwords<EPL>(reinterpret_cast<uint32_t*>(vb[i]), vp + ((4 * g + i) * D + c * EPL) * 4);
    };
    if (pages.n > 0) {
        load_k(0);
        load_v(0);
    }
    #pragma unroll 1
    for (int j = 0; j < pages.n; ++j) {
        const bool ok = pages.at(j) >= 0;
        const int t0 = 16 * list_page(k, pages.j0 + j);
        f4 s = {0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int i = 0; i < KQ; ++i) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kb[i], qv[i], s, 0, 0, 0);
        if constexpr (EARLY) load_k(j + 1);
        float x[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = s[i] * a.scale_log2;
        if (!(ok && all_see(a, k.pmin, k.pmax, t0))) {
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!(ok && row.sees(t0 + 4 * g + i))) x[i] = kNegInf;
                const bool keep = ok && any.sees(t0 + 4 * g + i);
                #pragma unroll
                for (int e = 0; e < EPL; ++e) vb[i][e] = keep ? vb[i][e] : 0.f;
            }
        }
        // (the reference moves as in the 16-bit kernel)
        const float lm = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        if (__ballot(lm > m + 8.f)) {
            const float mx = rowgroup_max(lm);
            const float mnew = mx > m + 8.f ? mx : m;
            const float alpha = m == kNegInf ? 0.f : fast_exp2(m - mnew);
            m = mnew;
            l *= alpha;
            #pragma unroll
            for (int e = 0; e < EPL; ++e) O[e] *= alpha;
        }
        const float ref = m == kNegInf ? 0.f : m;
        #pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = fast_exp2(x[i] - ref);
        l += (x[0] + x[1]) + (x[2] + x[3]);
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            #pragma unroll
            for (int e = 0; e < EPL; ++e) O[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[i][e], x[i], O[e], 0, 0, 0);
        if (EARLY || j + 1 < pages.n) {
            if constexpr (!EARLY) load_k(j + 1);
            load_v(j + 1);
        }
    }
    join_waves<D, DH_DTYPE_F32, NW>(a, k, split, m, rowgroup_sum(l), O, lds);
}

// Writes elements 4 col .. 4 col + 3 of a merged row.
template <int D, uint32_t QT>
__device__ __forceinline__ void write_merged(const WindowArgs& a, uint64_t at, int head, int col, f4 x, float sum) {
    const f4 o = x * (sum > 0.f ? 1.f / sum : 0.f);
    uint8_t* dst = a.out + at * a.out_stride;
    if constexpr (QT == DH_DTYPE_F32)
        *reinterpret_cast<f4*>(dst + (uint64_t(head) * D + 4 * col) * 4) = o;
    else
        *reinterpret_cast<u32x2*>(dst + (uint64_t(head) * D + 4 * col) * 2) =
            u32x2{pack2(o[0], o[1], QT == DH_DTYPE_F16), pack2(o[2], o[3], QT == DH_DTYPE_F16)};
}

// Joins the `parts` states from `slot` on (kMergeFew at most): elements 4 col ..
// of row `at`, head `head`.
template <int D, uint32_t QT>
__device__ __forceinline__ void merge_few(const WindowArgs& a, uint64_t slot, int parts, uint64_t at, int head, int col) {
    const f2* ml = reinterpret_cast<const f2*>(a.ws_ml) + slot;
    const f4* o = reinterpret_cast<const f4*>(a.ws_o + slot * D) + col;
    float mx = kNegInf, sum = 0.f;
    for (int s = 0; s < parts; ++s) mx = fmaxf(mx, ml[s][0]);
    f4 x = {0.f, 0.f, 0.f, 0.f};
    #pragma unroll 4
    for (int s = 0; s < parts; ++s) {
        const f2 v = ml[s];
        const float al = v[0] == kNegInf ? 0.f : fast_exp2(v[0] - mx);
        sum += al * v[1];
        x += o[s * (D / 4)] * al;
    }
    write_merged<D, QT>(a, at, head, col, x, sum);
}

// Joins a few parts of split work, a block of 16 rows a workgroup: D / 4 lanes
// take a row, four elements each.  Bound by the states' bytes.
template <int D, uint32_t QT>
__global__ __launch_bounds__(256) void window_merge_few_kernel(WindowArgs a) {
    constexpr int LPP = D / 4, G = 256 / LPP;
    const uint32_t unit = a.by_hkv(blockIdx.x);
    const RowBlock k = find_rows<4>(a, unit, int(blockIdx.x - unit * a.hkv));
    #pragma unroll 1
    for (int row = threadIdx.x / LPP; row < k.nrows; row += G) {
        int token, head;
        row_place(a, k, k.rho0 + row, token, head);
        const uint64_t at = uint64_t(k.seq.row0) + token;
        merge_few<D, QT>(a, (at * a.hq + head) * a.splits, k.zero ? 0 : int(a.splits), at, head, threadIdx.x % LPP);
    }
}

// The same for the blocks of a.tail on, 16 rows of a block a workgroup.
template <int D, uint32_t QT, int SHIFT>
__global__ __launch_bounds__(256) void window_merge_tail_kernel(WindowArgs a) {
    constexpr int LPP = D / 4, G = 256 / LPP, R16 = (1 << SHIFT) / 16;
    const uint32_t place = blockIdx.x / R16, x = a.tail + place, unit = a.by_hkv(x);
    const RowBlock k = find_rows<SHIFT>(a, unit, int(x - unit * a.hkv));
    const int row0 = int(blockIdx.x % R16) * 16;
    #pragma unroll 1
    for (int row = row0 + threadIdx.x / LPP; row < min(k.nrows, row0 + 16); row += G) {
        int token, head;
        row_place(a, k, k.rho0 + row, token, head);
        merge_few<D, QT>(a, ((uint64_t(place) << SHIFT) + row) * a.tail_parts, k.zero ? 0 : int(a.tail_parts),
                         uint64_t(k.seq.row0) + token, head, threadIdx.x % LPP);
    }
}

// Joins many parts of split work, COLS columns of a row a workgroup: COLS / 4
// lanes take a part's (four elements each), the workgroup's lane groups every so
// many parts; their sums are added in LDS in a fixed order.  Whole rows and 256
// threads; beyond kMergeMany parts, of few rows, 64 columns and 1024 threads have
// all loads in flight at once (16 rows of 256 dims in 256 parts: 5.8 us, and
// 10.2 by whole rows; 3840 rows of 128 in a dozen: 15 by 64 columns, and 9.9).
template <int D, uint32_t QT, int COLS, int NT>
__global__ __launch_bounds__(NT) void window_merge_kernel(WindowArgs a) {
    constexpr int CB = D / COLS, LPP = COLS / 4, G = NT / LPP;
    __shared__ float red[NT / 64];
    __shared__ __attribute__((aligned(16))) f4 acc[G][LPP];
    __shared__ float sums[G];
    const uint32_t x0 = blockIdx.x / (16 * CB), unit = a.by_hkv(x0);
    const int row = int(blockIdx.x / CB & 15), cb = int(blockIdx.x % CB);
    const RowBlock k = find_rows<4>(a, unit, int(x0 - unit * a.hkv));
    if (row >= k.nrows) return;
    const int tid = threadIdx.x;
    int token, head;
    row_place(a, k, k.rho0 + row, token, head);
    const uint64_t at = uint64_t(k.seq.row0) + token, slot = (at * a.hq + head) * a.splits;
    const f2* ml = reinterpret_cast<const f2*>(a.ws_ml) + slot;
    const int splits = k.zero ? 0 : int(a.splits);
    float mx = kNegInf;
    for (int s = tid; s < splits; s += NT) mx = fmaxf(mx, ml[s][0]);
    #pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = red[0];
    #pragma unroll
    for (int i = 1; i < NT / 64; ++i) mx = fmaxf(mx, red[i]);
    const int grp = tid / LPP, col = cb * LPP + tid % LPP;
    f4 x = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
    #pragma unroll 4
    for (int s = grp; s < splits; s += G) {
        const f2 v = ml[s];
        const float al = v[0] == kNegInf ? 0.f : fast_exp2(v[0] - mx);
        sum += al * v[1];
        x += reinterpret_cast<const f4*>(a.ws_o + (slot + s) * D)[col] * al;
    }
    acc[grp][tid % LPP] = x;
    if (tid % LPP == 0) sums[grp] = sum;
    __syncthreads();
    if (tid >= LPP) return;
    x = acc[0][tid];
    sum = sums[0];
    #pragma unroll
    for (int g = 1; g < G; ++g) {
        x += acc[g][tid];
        sum += sums[g];
    }
    write_merged<D, QT>(a, at, head, col, x, sum);
}

template <int D, uint32_t KVF, bool F16, int NW>
hipError_t launch_narrow_f(const WindowArgs& a, dim3 grid, hipStream_t s) {
    if constexpr (kWholeLines<D, KVF>) {
        if (a.once) {
            hipLaunchKernelGGL((window_narrow_kernel<D, KVF, F16, NW, true>), grid, dim3(64 * NW), 0, s, a);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((window_narrow_kernel<D, KVF, F16, NW, false>), grid, dim3(64 * NW), 0, s, a);
    return hipGetLastError();
}

template <int D, int NW>
hipError_t launch_narrow_w(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, dim3 grid, hipStream_t s) {
    const bool bf16 = q_dtype == DH_DTYPE_BF16, f16 = q_dtype == DH_DTYPE_F16;
    if (bf16 && fmt == KVF_FP8) return launch_narrow_f<D, KVF_FP8, false, NW>(a, grid, s);
    if (f16 && fmt == KVF_FP8) return launch_narrow_f<D, KVF_FP8, true, NW>(a, grid, s);
    if (bf16 && fmt == KVF_MX) return launch_narrow_f<D, KVF_MX, false, NW>(a, grid, s);
    if (f16 && fmt == KVF_MX) return launch_narrow_f<D, KVF_MX, true, NW>(a, grid, s);
    if constexpr (NW <= int(narrow_waves(D, false))) {
        if (bf16 && fmt == KVF_BF16) return launch_narrow_f<D, KVF_BF16, false, NW>(a, grid, s);
        if (f16 && fmt == KVF_F16) return launch_narrow_f<D, KVF_F16, true, NW>(a, grid, s);
        if (q_dtype == DH_DTYPE_F32 && fmt == KVF_F32) {
            hipLaunchKernelGGL((window_narrow32_kernel<D, NW>), grid, dim3(64 * NW), 0, s, a);
            return hipGetLastError();
        }
    }
    return hipErrorInvalidValue;
}

template <int D>
hipError_t launch_narrow_d(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, uint32_t waves, dim3 grid, hipStream_t s) {
    if constexpr (narrow_waves(D, true) >= 16) {
        if (waves == 16) return launch_narrow_w<D, 16>(a, q_dtype, fmt, grid, s);
    }
    if (waves == 8) return launch_narrow_w<D, 8>(a, q_dtype, fmt, grid, s);
    return waves == kWaves ? launch_narrow_w<D, kWaves>(a, q_dtype, fmt, grid, s) : hipErrorInvalidValue;
}

template <int D, uint32_t QT>
void launch_merge_q(const WindowArgs& a, uint32_t blocks, hipStream_t s) {
    if (a.splits <= kMergeFew)
        hipLaunchKernelGGL((window_merge_few_kernel<D, QT>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.splits <= kMergeMany)
        hipLaunchKernelGGL((window_merge_kernel<D, QT, D, 256>), dim3(blocks * 16), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((window_merge_kernel<D, QT, 64, 1024>), dim3(blocks * (16 * (D / 64))), dim3(1024), 0, s, a);
}

template <int D>
hipError_t launch_merge_w(const WindowArgs& a, uint32_t q_dtype, uint32_t blocks, hipStream_t s) {
    switch (q_dtype) {
        case DH_DTYPE_F16: launch_merge_q<D, DH_DTYPE_F16>(a, blocks, s); break;
        case DH_DTYPE_BF16: launch_merge_q<D, DH_DTYPE_BF16>(a, blocks, s); break;
        default: launch_merge_q<D, DH_DTYPE_F32>(a, blocks, s); break;
    }
    return hipGetLastError();
}

}  // namespace

int launch_window_narrow(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, uint32_t d, uint32_t waves,
                         void* stream) {
    const uint64_t blocks = row_blocks(a, 4) * a.splits * a.hkv;
    if (blocks > 0x7FFFFFFFull) return hipErrorInvalidValue;
    const dim3 grid{uint32_t(blocks)};
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (d) {
        case 64: return launch_narrow_d<64>(a, q_dtype, fmt, waves, grid, s);
        case 128: return launch_narrow_d<128>(a, q_dtype, fmt, waves, grid, s);
        case 256: return launch_narrow_d<256>(a, q_dtype, fmt, waves, grid, s);
        default: return hipErrorInvalidValue;
    }
}

int launch_window_merge(const WindowArgs& a, uint32_t q_dtype, uint32_t d, void* stream) {
    const uint64_t blocks = row_blocks(a, 4) * a.hkv;
    if (blocks > 0x1FFFFFFull) return hipErrorInvalidValue;
    const uint32_t grid = uint32_t(blocks);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (d) {
        case 64: return launch_merge_w<64>(a, q_dtype, grid, s);
        case 128: return launch_merge_w<128>(a, q_dtype, grid, s);
        case 256: return launch_merge_w<256>(a, q_dtype, grid, s);
        default: return hipErrorInvalidValue;
    }
}

namespace {
template <int D, int SHIFT>
hipError_t launch_merge_tail_s(const WindowArgs& a, uint32_t q_dtype, uint32_t blocks, hipStream_t s) {
    const dim3 grid(blocks << (SHIFT - 4));
    if (q_dtype == DH_DTYPE_F16)
        hipLaunchKernelGGL((window_merge_tail_kernel<D, DH_DTYPE_F16, SHIFT>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((window_merge_tail_kernel<D, DH_DTYPE_BF16, SHIFT>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}
}  // namespace

int launch_window_merge_tail(const WindowArgs& a, uint32_t q_dtype, uint32_t d, uint32_t blocks, uint32_t rows,
                             void* stream) {
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (d == 64 && rows == 256) return launch_merge_tail_s<64, 8>(a, q_dtype, blocks, s);
    if (d == 128 && rows == 128) return launch_merge_tail_s<128, 7>(a, q_dtype, blocks, s);
    if (d == 256 && rows == 128) return launch_merge_tail_s<256, 7>(a, q_dtype, blocks, s);
    return hipErrorInvalidValue;
}

}  // namespace dh
