// Windowed attention of many query rows a sequence, from device tables: chunks
// of prompts (dh_attend_window), 16-bit queries.
//
// A workgroup has a block of rows (32 a wave) of one KV head and walks the
// block's page list TK tokens at a time.  The tile's K and V go from the
// pages through registers (8-bit codes become 16-bit there) into LDS, two
// tiles deep: while the waves compute on one, the next is written and the
// loads of the one after are in flight; one barrier a tile.  On
// v_mfma_f32_32x32x16, lane l = 32 h + c, row c of the wave's tile:
//   S^T = K Q^T:  A = K, lane holds token c, dims 8h..8h+7 of a 16-dim step
//                 (ds_read_b128); B = Q^T from registers.  The lane gets the
//                 scores of row c for tokens 8 (i / 4) + 4 h + i % 4, i < 16.
//   O^T += V^T P^T: the B operand of 16 tokens is 8 of those scores after
//                 exp2, as they lie; A = V^T by two transposing LDS reads
//                 (ds_read_b64_tr_b16) of the same tokens' rows.
// so probabilities never leave registers and a row's maximum and sum need one
// exchange between two lanes.  16-byte chunk j of tile row t is at chunk
// j ^ swz(t): both reads then touch every bank once.
//
// E4M3 codes are exact in bf16 and f16; a block scale multiplies the scores (K)
// and the probabilities (V), MXFP8's power of two the code as it is converted.
#include "attend_device.hpp"
#include "window_device.hpp"

namespace dh {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <int D>
struct WideCfg {
    static constexpr int ROWS = int(wide_rows(D)), NW = ROWS / 32, THREADS = NW * 64;
    static constexpr int SHIFT = ROWS == 256 ? 8 : 7;
    static constexpr int TK = D == 64 ? 64 : 32;       // tokens a tile
    static constexpr int NP = TK / kPageSize;          // pages a tile
    static constexpr int RB = 2 * D, CH = RB / 16;     // row bytes, 16-byte chunks
    static constexpr int PLANE = TK * RB, TILE = 2 * PLANE;
    static constexpr int RING = D == 128 ? 4 : 3;      // tiles in LDS
};

// Chunk swizzle of a tile row.  K reads take 16 rows at one chunk, V reads 4
// rows x 4 chunks: the two low bits of the row move the four-chunk group.
template <int D>
__device__ __forceinline__ int wide_swz(int row) {
    if constexpr (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
}

template <bool F16>
__device__ __forceinline__ f16v mma32(u32x4 a, u32x4 b, f16v c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
}

// One tile on its way from the pages to LDS: this thread's 16-byte words of
// its K and V rows (8-bit ones make two chunks each).  Word i is STEP rows
// after word i - 1, so all of a thread's words have one column; a wave's word
// lies in one page.
template <int D, uint32_t KVF>
struct TileStage {
    using C = WideCfg<D>;
    static constexpr bool FP8 = KVF == KVF_FP8 || KVF == KVF_MX;
    static constexpr int EB = FP8 ? 1 : 2;
    static constexpr int WPR = D * EB / 16;              // words a row
    static constexpr int STEP = C::THREADS / WPR;        // rows
    static constexpr int N = 2 * C::TK / STEP;
    static_assert(2 * C::TK % STEP == 0 && 64 / WPR <= kPageSize && (STEP % 16 == 0 || STEP == 8), "words of a tile");
    u32x4 w[N];
    uint32_t sc[KVF == KVF_MX ? N : 1];
    int limit[N];        // tokens of the word's page that the sequence holds, where not `whole`
    bool whole;          // all of every page

    // Row of word i in its plane, K or V (0 / 1), and page of the tile; the
    // last two are a wave's.
    static __device__ __forceinline__ int row(int i, int tid) {
        return STEP > C::TK ? tid / WPR % C::TK : tid / WPR + i * STEP % C::TK;
    }
    static __device__ __forceinline__ int plane(int i, int tid) {
        return STEP > C::TK ? uniform(tid / WPR / C::TK) : i * STEP / C::TK;
    }
    static __device__ __forceinline__ int page(int i, int tid) { return uniform(row(i, tid) >> 4); }

    // idv: lane l holds the id of the tile's page l % NP (-1: none); all_whole:
    // every page is one of the pool and all its tokens the sequence's.
    __device__ __forceinline__ void load(const WindowArgs& a, const RowBlock& k, int idv, int j, bool all_whole, int tid) {
        const int r = tid / WPR & (STEP == 8 ? 7 : 15), col = tid % WPR;
        const uint32_t off = r * (D * EB) + col * 16, soff = r * (D / 32) + col / 2;
        whole = all_whole;
        auto word = [&](int i, int id) {
            const uint32_t blk = plane(i, tid) * a.hkv + k.kv_head;
            const int more = STEP == 8 ? (i & 1) * 8 : 0;        // rows past `r` in the page
            const uint8_t* p = a.kv + uint64_t(uint32_t(id)) * (2 * a.hkv * kPageSize * D * EB) +
                               (blk * (kPageSize * D * EB) + more * (D * EB));
            w[i] = *reinterpret_cast<const u32x4*>(p + off);
            if constexpr (KVF == KVF_MX)
                sc[i] = (a.scales + uint64_t(uint32_t(id)) * (2 * a.hkv * kPageSize * D / 32) +
                         (blk * (kPageSize * D / 32) + more * (D / 32)))[soff];
        };
        if (all_whole) {
            #pragma unroll
            for (int i = 0; i < N; ++i) word(i, __builtin_amdgcn_readlane(idv, page(i, tid)));
        } else {
            #pragma unroll
            for (int i = 0; i < N; ++i) {
                const int pg = page(i, tid), id = __builtin_amdgcn_readlane(idv, pg);
                limit[i] = id < 0 ? 0 : min(k.seq.len - 16 * list_page(k, j + pg), 16);
                word(i, max(id, 0));
            }
        }
    }

    template <bool F16>
    __device__ __forceinline__ void store(uint8_t* tile, int tid) {
        const int col = tid % WPR;
        if (!whole) {      // slots past the sequence's end, entries outside the pool: zeros
            asm volatile("");
            #pragma unroll
            for (int i = 0; i < N; ++i) {
                const bool keep = (row(i, tid) & 15) < limit[i];
                #pragma unroll
                for (int e = 0; e < 4; ++e) w[i][e] = keep ? w[i][e] : 0u;
                if constexpr (KVF == KVF_MX) sc[i] = keep ? sc[i] : 127u;
            }
        }
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row(i, tid), swz = wide_swz<D>(r);
            uint8_t* p = tile + plane(i, tid) * C::PLANE + r * C::RB;
            if constexpr (!FP8) {
                *reinterpret_cast<u32x4*>(p + ((col ^ swz) << 4)) = w[i];
            } else {
                const float s = KVF == KVF_MX ? e8m0_to_float(sc[i]) : 1.f;
                uint32_t o[8];
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = w[i][e];
                    e4m3x4_cvt<F16>(x, s, o[2 * e], o[2 * e + 1]);
                }
                *reinterpret_cast<u32x4*>(p + (((2 * col) ^ swz) << 4)) = u32x4{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<u32x4*>(p + (((2 * col + 1) ^ swz) << 4)) = u32x4{o[4], o[5], o[6], o[7]};
            }
        }
    }
};

__device__ __forceinline__ float pair_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float pair_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// What a wave keeps of its 32 rows (lane l = 32 h + c: row c).
template <int D>
struct WideRows {
    float m, L;            // reference (log2 units), this lane's share of the sum
    f16v O[D / 32];        // [32 e + 8 (i / 4) + 4 h + i % 4] = O[e][i]
};

// The lane's LDS read addresses in a tile at byte offset 0: K rows of token c
// (16-dim step kb), V rows of the transposing reads (tokens 4 h + .. of the
// first or second half of a page, 32-dim block e).
template <int D>
struct WideReads {
    uint32_t k[D / 16], v[2][D / 32];

    __device__ __forceinline__ WideReads(uint32_t base, int h, int c) {
        using C = WideCfg<D>;
        #pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) k[kb] = base + c * C::RB + (((2 * kb + h) ^ wide_swz<D>(c)) << 4);
        #pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = 8 * half + 4 * h + ((c & 15) >> 2), col = 2 * (c >> 4) + ((c & 3) >> 1);
            #pragma unroll
            for (int e = 0; e < D / 32; ++e)
                v[half][e] = base + C::PLANE + row * C::RB + (((4 * e + col) ^ wide_swz<D>(row)) << 4) + ((c & 1) << 3);
        }
        // Opaque from here: else `base` is split off again and added to the
        // tile's offset, an addition for every read instead of an immediate.
        #pragma unroll
        for (int kb = 0; kb < D / 16; ++kb) asm volatile("" : "+v"(k[kb]));
        #pragma unroll
        for (int e = 0; e < D / 32; ++e) asm volatile("" : "+v"(v[0][e]), "+v"(v[1][e]));
    }
};

// K operands of the 32 tokens at byte offset `at`.
template <int D>
__device__ __forceinline__ void wide_k(const WideReads<D>& r, uint32_t at, u32x4 (&kw)[D / 16]) {
    #pragma unroll
    for (int kb = 0; kb < D / 16; ++kb) kw[kb] = *reinterpret_cast<const lds_u32x4*>(uintptr_t(r.k[kb] + at));
}

template <int D, bool F16>
__device__ __forceinline__ f16v wide_scores(const u32x4 (&kw)[D / 16], const u32x4 (&q)[D / 16]) {
    f16v s;
    #pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
    #pragma unroll
    for (int kb = 0; kb < D / 16; ++kb) s = mma32<F16>(kw[kb], q[kb], s);
    return s;
}

// V operands of the 32 tokens at byte offset `at`, and O += V^T P^T.
template <int D>
__device__ __forceinline__ void wide_v(const WideReads<D>& r, uint32_t at, u32x4 (&vw)[2][D / 32]) {
    using C = WideCfg<D>;
    #pragma unroll
    for (int g = 0; g < 2; ++g)
        #pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)uintptr_t(r.v[0][e] + at + g * 16 * C::RB)));
            const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)uintptr_t(r.v[1][e] + at + g * 16 * C::RB)));
            vw[g][e] = u32x4{a[0], a[1], b[0], b[1]};
        }
}

template <int D, bool F16>
__device__ __forceinline__ void wide_values(const u32x4 (&vw)[2][D / 32], const u32x4 (&pk)[2], f16v (&O)[D / 32]) {
    #pragma unroll
    for (int g = 0; g < 2; ++g)
        #pragma unroll
        for (int e = 0; e < D / 32; ++e) O[e] = mma32<F16>(vw[g][e], pk[g], O[e]);
}

// Largest scaled score of the lane's 16 (page factors f).
__device__ __forceinline__ float wide_max(const f16v& s, float f0, float f1) {
    float a = s[0], b = s[8];
    #pragma unroll
    for (int i = 1; i < 8; ++i) {
        a = fmaxf(a, s[i]);
        b = fmaxf(b, s[8 + i]);
    }
    return fmaxf(a * f0, b * f1);
}

// Moves the reference of the rows that a score passes by 8.
template <int D>
__device__ __forceinline__ void wide_rescale(WideRows<D>& w, float lm) {
    const float mx = pair_max(lm);
    const float mnew = mx > w.m + 8.f ? mx : w.m;
    const float alpha = w.m == kNegInf ? 0.f : fast_exp2(w.m - mnew);
    w.m = mnew;
    w.L *= alpha;
    #pragma unroll
    for (int e = 0; e < D / 32; ++e) w.O[e] *= alpha;
}

// Sum of the two weights packed in w, added to c.
template <bool F16>
__device__ __forceinline__ float add2(uint32_t w, float c) {
    if constexpr (F16)
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
    else
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, w), s16x2{0x3F80, 0x3F80}, c, false);
}

// Weights of 32 tokens as the B operand, V's block scales v0 / v1 on them.  The
// row's sum is of the weights as V gets them, but for the block scales.
template <uint32_t KVF, bool F16>
__device__ __forceinline__ void wide_weights(const f16v& s, float f0, float f1, float v0, float v1, float m, float& L,
                                             u32x4 (&pk)[2]) {
    const float nm = m == kNegInf ? 0.f : -m;
    #pragma unroll
    for (int g = 0; g < 2; ++g) {
        float x[8];
        #pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = fast_exp2(__builtin_fmaf(s[8 * g + i], g ? f1 : f0, nm));
            if constexpr (KVF == KVF_FP8) {
                L += x[i];
                x[i] *= g ? v1 : v0;
            }
        }
        uint32_t w[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack2(x[2 * i], x[2 * i + 1], F16);
            if constexpr (KVF != KVF_FP8) L = add2<F16>(w[i], L);
        }
        pk[g] = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// Masks the scores of list entries j, j + 1 that the lane's row (position p)
// does not see; false if no row of the wave (wmin .. wmax) sees any of them.
__device__ __forceinline__ bool wide_mask(f16v& s, const WindowArgs& a, const RowBlock& k, const int* ids, int j0, int n,
                                          int j, int wmin, int wmax, int p, int h) {
    int t0[2];
    bool some = false;
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool ok = j + i < n && uniform(ids[j + i]) >= 0;
        t0[i] = ok ? 16 * list_page(k, j0 + j + i) : 0x7FFFFF00;      // nobody sees that
        some = some || (t0[i] <= wmax && (!a.window || t0[i] + 15 > wmin - a.window || t0[i] < a.sinks));
    }
    if (!some) return false;
    #pragma unroll
    for (int g = 0; g < 2; ++g) {
        // bit t of see: the row sees token t0 + t
        auto below = [](int x) { return (1u << min(max(x, 0), 16)) - 1u; };
        uint32_t see = below(p - t0[g] + 1);
        if (a.window) see &= ~below(p - a.window + 1 - t0[g]) | below(a.sinks - t0[g]);
        see >>= 4 * h;
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!((see >> (8 * (i / 4) + i % 4)) & 1u)) s[8 * g + i] = kNegInf;
    }
    return true;
}

template <int D, uint32_t KVF, bool F16>
__global__ __launch_bounds__(WideCfg<D>::THREADS, D == 256 ? 1 : 2) void window_wide_kernel(WindowArgs a) {
    using C = WideCfg<D>;
    constexpr int NP = C::NP, SUB = C::TK / 32, EB = D / 32, KB = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[C::RING * C::TILE];
    __shared__ int ids[kWideMaxPages + (C::RING + 2) * NP];        // (read ahead)
    __shared__ __attribute__((aligned(16))) f2 scl[KVF == KVF_FP8 ? kWideMaxPages + 2 * NP : 1];
    report_bad_tables(a.t, a.status, blockIdx.x);
    const uint32_t x0 = blockIdx.x / a.hkv;
    const uint32_t unit = x0 / a.splits;
    const int split = uniform(int(x0 - unit * a.splits));
    const RowBlock k = uniform_block(find_rows<C::SHIFT>(a, unit, int(blockIdx.x - x0 * a.hkv)));
    if (k.nrows == 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5, c = lane & 31;
    if (k.zero) {
        if (a.splits > 1) return;      // the merge writes them
        for (int i = tid; i < k.nrows * (D / 8); i += C::THREADS) {
            int token, head;
            row_place(a, k, k.rho0 + i / (D / 8), token, head);
            reinterpret_cast<u32x4*>(a.out + (uint64_t(k.seq.row0) + token) * a.out_stride +
                                     uint64_t(head) * D * 2)[i % (D / 8)] = u32x4{0u, 0u, 0u, 0u};
        }
        return;
    }
    // This workgroup's part of the page list, whole tiles.
    int per = uniform((k.pages + int(a.splits) - 1) / int(a.splits));
    per = (per + NP - 1) / NP * NP;
    const int j0 = min(split * per, k.pages), n = min(min(per, k.pages - j0), int(kWideMaxPages));
    const int ntiles = (n + NP - 1) / NP;
    int bad = 0;
    for (int j = tid; j < (ntiles + C::RING + 1) * NP; j += C::THREADS) {
        int id = -1;
        if (j < n) {
            id = checked_page(a.t.indices[k.seq.page0 + list_page(k, j0 + j)], a.page_limit, a.status);
            bad |= id < 0 ? 1 : 0;
        }
        ids[j] = id;
        if constexpr (KVF == KVF_FP8) {
            if (j < ntiles * NP + 2 * NP) {
                f2 s = {1.f, 1.f};
                if (id >= 0) {
                    const float* p = reinterpret_cast<const float*>(a.scales) + uint64_t(id) * 2 * a.hkv + k.kv_head;
                    s = f2{p[0], p[a.hkv]};
                }
                // a scale of zero (a page nobody wrote) must not meet a masked -inf
                scl[j] = f2{fmaxf(a.scale_log2 * s[0], 1e-30f), s[1]};
            }
        }
    }

    // The lane's row, and the positions of the wave's rows.
    const int wrow = wave * 32;
    const bool live = wrow + c < k.nrows;
    int token, head;
    row_place(a, k, k.rho0 + min(wrow + c, k.nrows - 1), token, head);
    const int first = k.seq.len - k.seq.n, p = first + token;
    const int wmin = uniform(first + (k.rho0 + min(wrow, k.nrows - 1)) / int(a.r));
    const int wmax = uniform(first + (k.rho0 + min(wrow + 31, k.nrows - 1)) / int(a.r));
    u32x4 q[KB];
    {
        const uint8_t* qp = a.q + (uint64_t(k.seq.row0) + token) * a.q_stride + uint64_t(head) * D * 2 + 16 * h;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) q[kb] = *reinterpret_cast<const u32x4*>(qp + 32 * kb) ^ a.q_sign;
    }
    WideRows<D> w;
    w.m = kNegInf;
    w.L = 0.f;
    #pragma unroll
    for (int e = 0; e < EB; ++e)
        #pragma unroll
        for (int i = 0; i < 16; ++i) w.O[e][i] = 0.f;
    const uint32_t lds0 = uint32_t(uniform(int(uint32_t(reinterpret_cast<uintptr_t>(tiles)))));
    const WideReads<D> rd(lds0, h, c);

    // Entries all of whose tokens every row of the wave sees (between its
    // window's ends), and entries that are whole pages of the pool: what
    // needs no mask, tested by two comparisons a step.
    const bool holes = uniform(__syncthreads_or(bad)) != 0;
    int seen0 = 0, seen1 = 0, whole1 = 0;
    if (!holes) {
        const int lo = a.window ? max(wmax - a.window + 1, 0) : 0;
        seen0 = k.sink_pages + max(((lo + 15) >> 4) - k.window_page, 0) - j0;
        seen1 = k.sink_pages + ((wmin + 1) >> 4) - k.window_page - j0;
        whole1 = min(n, k.sink_pages + (k.seq.len >> 4) - k.window_page - j0);
    }
    seen0 = uniform(seen0);
    seen1 = uniform(min(seen1, n));
    whole1 = uniform(whole1);
    // Two or more tiles in LDS, another on its way in registers; the page ids
    // of the one after that in idv (a lane's page l % NP).
    constexpr int R = C::RING;
    TileStage<D, KVF> stage;
    const int l = lane % NP;
    if (ntiles > 0) {
        #pragma unroll
        for (int i = 0; i < R - 1; ++i) {
            stage.load(a, k, ids[i * NP + l], j0 + i * NP, (i + 1) * NP <= whole1, tid);
            stage.template store<F16>(tiles + i * C::TILE, tid);
        }
        stage.load(a, k, ids[(R - 1) * NP + l], j0 + (R - 1) * NP, R * NP <= whole1, tid);
    }
    int idv = ids[R * NP + l];
    __syncthreads();
    // Scores run one sub-tile (32 tokens) ahead: their products are
    // independent of the softmax of the current ones.
    f16v s;
    {
        u32x4 kw[KB];
        wide_k<D>(rd, 0, kw);
        s = wide_scores<D, F16>(kw, q);
    }
    // Unrolled over the ring, so that a tile's place is an immediate offset.
    #pragma unroll 1
    for (int base = 0; base < ntiles; base += R) {
        static_for<0, R>([&](auto J) {
            constexpr int slot = decltype(J)::value;
            const int tile = base + slot;
            if (tile >= ntiles) return;
            // The tile before is done with (the barrier below): its place
            // takes the one R - 1 ahead.
            if (tile + R - 1 < ntiles) {
                stage.template store<F16>(tiles + (slot + R - 1) % R * C::TILE, tid);
                if (tile + R < ntiles) {
                    stage.load(a, k, idv, j0 + (tile + R) * NP, (tile + R + 1) * NP <= whole1, tid);
                    idv = ids[(tile + R + 1) * NP + l];
                }
            }
            static_for<0, SUB>([&](auto U) {
                constexpr int u = decltype(U)::value;
                constexpr uint32_t at = slot * C::TILE + u * 32 * C::RB;
                constexpr uint32_t ahead = u + 1 < SUB ? at + 32 * C::RB : (slot + 1) % R * C::TILE;
                const int j = tile * NP + 2 * u;
                bool some = true;
                if (j < seen0 || j + 2 > seen1) some = wide_mask(s, a, k, ids, j0, n, j, wmin, wmax, p, h);
                u32x4 kw[KB];
                if (some) {
                    float f0 = a.scale_log2, f1 = a.scale_log2, v0 = 1.f, v1 = 1.f;
                    if constexpr (KVF == KVF_FP8) {
                        const f4 x = *reinterpret_cast<const f4*>(scl + j);
                        f0 = x[0];
                        v0 = x[1];
                        f1 = x[2];
                        v1 = x[3];
                    }
                    const float lm = wide_max(s, f0, f1);
                    if (__ballot(lm > w.m + 8.f)) wide_rescale<D>(w, lm);
                    // In this order: K of the next sub-tile on its way, the
                    // weights meanwhile, the next scores with V's reads
                    // between them, then V's products.
                    __builtin_amdgcn_sched_barrier(0);
                    wide_k<D>(rd, ahead, kw);
                    __builtin_amdgcn_sched_barrier(0);
                    u32x4 pk[2], vw[2][EB];
                    wide_weights<KVF, F16>(s, f0, f1, v0, v1, w.m, w.L, pk);
                    __builtin_amdgcn_sched_barrier(0);
                    s = wide_scores<D, F16>(kw, q);
                    wide_v<D>(rd, at, vw);
                    #pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // two LDS reads
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    wide_values<D, F16>(vw, pk, w.O);
                } else {
                    wide_k<D>(rd, ahead, kw);
                    s = wide_scores<D, F16>(kw, q);
                }
            });
            __syncthreads();
        });
    }
    const float sum = pair_sum(w.L);
    if (!live) return;
    const uint64_t at = uint64_t(k.seq.row0) + token;
    if (a.splits > 1) {
        const uint64_t slot = (at * a.hq + head) * a.splits + split;
        #pragma unroll
        for (int e = 0; e < EB; ++e)
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f4*>(a.ws_o + slot * D + 32 * e + 8 * i + 4 * h) =
                    f4{w.O[e][4 * i], w.O[e][4 * i + 1], w.O[e][4 * i + 2], w.O[e][4 * i + 3]};
        if (h == 0) *reinterpret_cast<f2*>(a.ws_ml + slot * 2) = f2{w.m, sum};
        return;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    uint8_t* o = a.out + at * a.out_stride + uint64_t(head) * D * 2;
    #pragma unroll
    for (int e = 0; e < EB; ++e)
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x2*>(o + 2 * (32 * e + 8 * i + 4 * h)) =
                u32x2{pack2(w.O[e][4 * i] * inv, w.O[e][4 * i + 1] * inv, F16),
                      pack2(w.O[e][4 * i + 2] * inv, w.O[e][4 * i + 3] * inv, F16)};
}

template <int D>
hipError_t launch_wide_d(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, hipStream_t s) {
    const uint64_t blocks = row_blocks(a, WideCfg<D>::SHIFT) * a.splits * a.hkv;
    if (blocks > 0x7FFFFFFFull) return hipErrorInvalidValue;
    const dim3 grid{uint32_t(blocks)}, block(WideCfg<D>::THREADS);
    if (q_dtype == DH_DTYPE_BF16 && fmt == KVF_BF16)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_BF16, false>), grid, block, 0, s, a);
    else if (q_dtype == DH_DTYPE_F16 && fmt == KVF_F16)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_F16, true>), grid, block, 0, s, a);
    else if (q_dtype == DH_DTYPE_BF16 && fmt == KVF_FP8)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_FP8, false>), grid, block, 0, s, a);
    else if (q_dtype == DH_DTYPE_F16 && fmt == KVF_FP8)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_FP8, true>), grid, block, 0, s, a);
    else if (q_dtype == DH_DTYPE_BF16 && fmt == KVF_MX)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_MX, false>), grid, block, 0, s, a);
    else if (q_dtype == DH_DTYPE_F16 && fmt == KVF_MX)
        hipLaunchKernelGGL((window_wide_kernel<D, KVF_MX, true>), grid, block, 0, s, a);
    else
        return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

int launch_window_wide(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, uint32_t d, void* stream) {
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (d) {
        case 64: return launch_wide_d<64>(a, q_dtype, fmt, s);
        case 128: return launch_wide_d<128>(a, q_dtype, fmt, s);
        case 256: return launch_wide_d<256>(a, q_dtype, fmt, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dh
