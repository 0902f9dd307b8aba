// Windowed attention of many query rows a sequence over 8-bit caches, and over
// 16-bit ones of heads of 256 dims, from device tables: chunks of prompts
// (dh_attend_window).
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
// exchange between two lanes.  LDS rows are padded: both reads then touch
// every bank once, from one address register.
//
// E4M3 codes are exact in bf16 and f16; a block scale multiplies the scores (K)
// and the probabilities (V), MXFP8's power of two the code as it is converted.
//
// Bound by the matrix cores and, for 8-bit codes, by the vector instructions of
// their conversion beside them: 4096 tokens x 64 heads of 128 dims over a window
// of 2048 and 128 first tokens in FP8 take 351 us, 0.81 PFLOP/s (16-bit caches
// in window_ring.hip: 294).  128 rows a workgroup and two workgroups a CU beat
// 256 rows and one (three chunks of 300 to 900 tokens over 5000: 232 us
// against 278; 202 since the last round of few blocks is split).
#include "attend_device.hpp"
#include "window_device.hpp"

namespace dh {
namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

template <int D>
struct WideCfg {
    static constexpr int ROWS = int(wide_rows(D)), NW = 4, THREADS = NW * 64;
    static constexpr int RT = ROWS / (32 * NW);        // row tiles of 32 a wave
    static constexpr int SHIFT = ROWS == 256 ? 8 : 7;
    static constexpr int TK = 32, NP = TK / kPageSize; // tokens, pages a tile
    // Row strides in LDS.  A K read takes 16 bytes of 16 rows at a time, a V
    // read 64 bytes of 4: these strides put either on 64 different banks, and
    // one register addresses all of a tile's reads.
    static constexpr int CH = D / 8;                   // 16-byte words a row
    static constexpr int KS = 2 * D + 16, VS = D == 64 ? 192 : 2 * D + 64;
    static constexpr int VOFF = TK * KS, TILE = VOFF + TK * VS;
    static constexpr int RING = 4;                     // tiles in LDS
    static constexpr int AHEAD = D == 256 ? 1 : 2;     // tiles on their way in registers
    static constexpr bool ACC = D == 256;              // one wave a SIMD: O in the accumulation registers
};

template <bool F16>
__device__ __forceinline__ f16v mma32(u32x4 a, u32x4 b, f16v c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
}

// A wave-uniform address of global memory, in scalar registers.
typedef const __attribute__((address_space(1))) uint8_t* global_ptr;
__device__ __forceinline__ global_ptr uniform_ptr(const uint8_t* p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = uint32_t(uniform(int(uint32_t(x)))), hi = uint32_t(uniform(int(uint32_t(x >> 32))));
    return reinterpret_cast<global_ptr>(hi << 32 | lo);
}

// One tile on its way from the pages to LDS: this thread's 16-byte words of
// its K and V rows (8-bit ones make two words each).  Word i is STEP rows after
// word i - 1, so all of a thread's words have one column; a wave's word lies
// in one page.  Entries outside the pool read page 0: nobody sees them.
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

    // Row of word i in its plane, K or V (0 / 1), and page of the tile; the
    // last two are a wave's.
    static __device__ __forceinline__ int row(int i, int tid) {
        return STEP > C::TK ? tid / WPR % C::TK : tid / WPR + i * STEP % C::TK;
    }
    static __device__ __forceinline__ int plane(int i, int tid) {
        return STEP > C::TK ? uniform(tid / WPR / C::TK) : i * STEP / C::TK;
    }
    static __device__ __forceinline__ int page(int i, int tid) { return uniform(row(i, tid) >> 4); }

    // idv: lane l holds the id of the tile's page l % NP (-1: none).
    __device__ __forceinline__ void load(const WindowArgs& a, const RowBlock& k, int idv, int tid) {
        const int r = tid / WPR & (STEP == 8 ? 7 : 15), col = tid % WPR;
        const uint32_t off = r * (D * EB) + col * 16, soff = r * (D / 32) + col / 2;
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t id = uint32_t(max(__builtin_amdgcn_readlane(idv, page(i, tid)), 0));
            const uint32_t blk = plane(i, tid) * a.hkv + k.kv_head;
            const int more = STEP == 8 ? (i & 1) * 8 : 0;        // rows past `r` in the page
            // (the page's address kept apart, in scalar registers: else the
            // thread's part is added to the pool's once, and the page's as a
            // vector)
            const global_ptr p = uniform_ptr(a.kv + uint64_t(id) * (2 * a.hkv * kPageSize * D * EB) +
                                             (blk * (kPageSize * D * EB) + more * (D * EB)));
            w[i] = *reinterpret_cast<const __attribute__((address_space(1))) u32x4*>(p + off);
            if constexpr (KVF == KVF_MX) {
                const global_ptr s = uniform_ptr(a.scales + uint64_t(id) * (2 * a.hkv * kPageSize * D / 32) +
                                                 (blk * (kPageSize * D / 32) + more * (D / 32)));
                sc[i] = s[soff];
            }
        }
    }

    template <bool F16>
    __device__ __forceinline__ void store(uint8_t* tile, int tid) const {
        const int col = tid % WPR;
        #pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row(i, tid), pl = plane(i, tid);
            uint8_t* p = tile + (pl ? C::VOFF + r * C::VS : r * C::KS);
            if constexpr (!FP8) {
                *reinterpret_cast<u32x4*>(p + (col << 4)) = w[i];
            } else {
                const float s = KVF == KVF_MX ? e8m0_to_float(sc[i]) : 1.f;
                uint32_t o[8];
                #pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = w[i][e];
                    e4m3x4_cvt<F16>(x, s, o[2 * e], o[2 * e + 1]);
                }
                *reinterpret_cast<u32x4*>(p + (col << 5)) = u32x4{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<u32x4*>(p + (col << 5) + 16) = u32x4{o[4], o[5], o[6], o[7]};
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

// What a wave keeps of a tile of 32 rows (lane l = 32 h + c: row c).
template <int D>
struct WideRows {
    float m, L;            // reference (log2 units), this lane's share of the sum
    f16v O[D / 32];        // [32 e + 8 (i / 4) + 4 h + i % 4] = O[e][i]
};

// The lane's LDS read addresses in the tile at byte offset 0 of the ring: K
// row of token c, V rows of the transposing reads (tokens 4 h + ..).
template <int D>
struct WideReads {
    uint32_t k, v;
    __device__ __forceinline__ WideReads(uint32_t base, int h, int c) {
        using C = WideCfg<D>;
        k = base + c * C::KS + 16 * h;
        v = base + C::VOFF + (4 * h + ((c & 15) >> 2)) * C::VS + 32 * (c >> 4) + 8 * (c & 3);
    }
};

// K operands of the 32 tokens of the tile at byte offset `at`.
template <int D>
__device__ __forceinline__ void wide_k(const WideReads<D>& r, uint32_t at, u32x4 (&kw)[D / 16]) {
    const uint32_t p = r.k + at;
    #pragma unroll
    for (int kb = 0; kb < D / 16; ++kb) kw[kb] = *reinterpret_cast<const lds_u32x4*>(uintptr_t(p + 32 * kb));
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

// V operands of its 32 tokens: page g, 32-dim block e.
template <int D>
__device__ __forceinline__ void wide_v(const WideReads<D>& r, uint32_t at, u32x4 (&vw)[2][D / 32]) {
    using C = WideCfg<D>;
    const uint32_t p = r.v + at;
    #pragma unroll
    for (int g = 0; g < 2; ++g)
        #pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)uintptr_t(p + g * 16 * C::VS + 64 * e)));
            const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4*)uintptr_t(p + (g * 16 + 8) * C::VS + 64 * e)));
            vw[g][e] = u32x4{a[0], a[1], b[0], b[1]};
        }
}

// Largest scaled score of the lane's 16, as the reference counts it (the pages'
// factors and log2 V scales fac).
template <uint32_t KVF>
__device__ __forceinline__ float wide_max(const f16v& s, const f4& fac) {
    float a = s[0], b = s[8];
    #pragma unroll
    for (int i = 1; i < 8; ++i) {
        a = fmaxf(a, s[i]);
        b = fmaxf(b, s[8 + i]);
    }
    if constexpr (KVF == KVF_FP8) return fmaxf(__builtin_fmaf(a, fac[0], fac[1]), __builtin_fmaf(b, fac[2], fac[3]));
    return fmaxf(a * fac[0], b * fac[2]);
}

// O *= alpha.  With one wave a SIMD, O lives in the accumulation half of the
// registers, which vector instructions cannot use; said in C++, the compiler
// moves all of O to the other half and back around this seldom taken branch,
// on every step.  The waits: a result of the matrix unit may still be on its
// way to the register read first, and a written one is its next operand.
template <bool ACC>
__device__ __forceinline__ void wide_scale(f16v& O, float alpha) {
    if constexpr (ACC) {
        #pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float x = O[i], y = O[i + 1], z = O[i + 2], v = O[i + 3], t0, t1, t2, t3;
            asm volatile("s_nop %9\n\ts_nop %9\n\t"
                         "v_accvgpr_read_b32 %4, %0\n\tv_accvgpr_read_b32 %5, %1\n\t"
                         "v_accvgpr_read_b32 %6, %2\n\tv_accvgpr_read_b32 %7, %3\n\t"
                         "v_mul_f32 %4, %4, %8\n\tv_mul_f32 %5, %5, %8\n\t"
                         "v_mul_f32 %6, %6, %8\n\tv_mul_f32 %7, %7, %8\n\t"
                         "v_accvgpr_write_b32 %0, %4\n\tv_accvgpr_write_b32 %1, %5\n\t"
                         "v_accvgpr_write_b32 %2, %6\n\tv_accvgpr_write_b32 %3, %7\n\t"
                         "s_nop %10"
                         : "+a"(x), "+a"(y), "+a"(z), "+a"(v), "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
                         : "v"(alpha), "i"(i == 0 ? 15 : 0), "i"(i == 12 ? 7 : 0));
            O[i] = x;
            O[i + 1] = y;
            O[i + 2] = z;
            O[i + 3] = v;
        }
    } else {
        O *= alpha;
    }
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
    for (int e = 0; e < D / 32; ++e) wide_scale<WideCfg<D>::ACC>(w.O[e], alpha);
}

// Sum of the two weights packed in w, added to c.
template <bool F16>
__device__ __forceinline__ float add2(uint32_t w, float c) {
    if constexpr (F16)
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.f, (_Float16)1.f}, c, false);
    else
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(s16x2, w), s16x2{0x3F80, 0x3F80}, c, false);
}

// Weights of 32 tokens as the B operand: 2^(s - m), with V's block scale in the
// exponent.  The row's sum is of the weights as V gets them, in kSumUnit where
// the scales are taken out of it again.
template <uint32_t KVF, bool F16>
__device__ __forceinline__ void wide_weights(const f16v& s, const f4& fac, float m, float& L, u32x4 (&pk)[2]) {
    const float nm = m == kNegInf ? 0.f : -m;
    #pragma unroll
    for (int g = 0; g < 2; ++g) {
        uint32_t w[4];
        float l = KVF == KVF_FP8 ? 0.f : L;
        const float c = KVF == KVF_FP8 ? nm + fac[2 * g + 1] : nm;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = fast_exp2(__builtin_fmaf(s[8 * g + 2 * i], fac[2 * g], c));
            const float x1 = fast_exp2(__builtin_fmaf(s[8 * g + 2 * i + 1], fac[2 * g], c));
            w[i] = pack2(x0, x1, F16);
            l = add2<F16>(w[i], l);
        }
        L = KVF == KVF_FP8 ? __builtin_fmaf(l, fast_exp2(kSumUnitLog2 - fac[2 * g + 1]), L) : l;
        pk[g] = u32x4{w[0], w[1], w[2], w[3]};
    }
}

// Masks the scores of list entries j, j + 1 that the lane's rows (positions p)
// do not see, and zeroes their V rows (in LDS, `v`) past the sequence's end:
// those weights are zero, but what lies there need not be a number.  Every
// wave does so for itself before it reads them.
template <int D, int RT>
__device__ __forceinline__ void wide_mask(f16v (&s)[RT], uint8_t* v, const WindowArgs& a, const RowBlock& k,
                                          const int* ids, int j0, int n, int j, const int (&p)[RT], int lane) {
    using C = WideCfg<D>;
    #pragma unroll
    for (int g = 0; g < 2; ++g) {
        const bool ok = j + g < n && uniform(ids[j + g]) >= 0;
        const int t0 = ok ? 16 * list_page(k, j0 + j + g) : 0x7FFFFF00;      // nobody sees that
        const int held = max(k.seq.len - t0, 0);
        for (int i = held * C::CH + lane; i < kPageSize * C::CH; i += 64)
            *reinterpret_cast<u32x4*>(v + (16 * g + i / C::CH) * C::VS + i % C::CH * 16) = u32x4{0u, 0u, 0u, 0u};
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            // bit t of see: the row sees token t0 + t
            auto below = [](int x) { return (1u << min(max(x, 0), 16)) - 1u; };
            uint32_t see = below(p[rt] - t0 + 1);
            if (a.window) see &= ~below(p[rt] - a.window + 1 - t0) | below(a.sinks - t0);
            see >>= 4 * (lane >> 5);
            #pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!((see >> (8 * (i / 4) + i % 4)) & 1u)) s[rt][8 * g + i] = kNegInf;
        }
    }
}

template <int D, uint32_t KVF, bool F16>
__global__ __launch_bounds__(WideCfg<D>::THREADS, WideCfg<D>::ACC ? 1 : 2) void window_wide_kernel(WindowArgs a) {
    using C = WideCfg<D>;
    constexpr int NP = C::NP, EB = D / 32, KB = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[C::RING * C::TILE];
    __shared__ int ids[kWideMaxPages + (C::RING + C::AHEAD + 2) * NP];        // (read ahead)
    __shared__ __attribute__((aligned(16))) f2 scl[KVF == KVF_FP8 ? kWideMaxPages + 2 * NP : 1];
    const bool refused = sees_refused(a.t, blockIdx.x);
    const BlockPart b = block_part<true>(a);
    const RowBlock k = uniform_block(find_rows<C::SHIFT>(a, b.unit, b.head));
    report(refused, a.status);
    if (k.nrows == 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), h = lane >> 5, c = lane & 31;
    if (k.zero) {
        if (b.parts == 1) zero_rows<D, DH_DTYPE_F16>(a, k);     // (else the merge writes them)
        return;
    }
    // This workgroup's part of the page list, whole tiles.
    int per = part_pages<true>(a, b, k.pages);
    per = (per + NP - 1) / NP * NP;
    const int j0 = min(b.split * per, k.pages), n = min(min(per, k.pages - j0), int(kWideMaxPages));
    const int ntiles = (n + NP - 1) / NP;
    int bad = 0;
    for (int j = tid; j < (ntiles + C::RING + C::AHEAD + 1) * NP; j += C::THREADS) {
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
                scl[j] = f2{fmaxf(a.scale_log2 * s[0], 1e-30f), value_log2(s[1])};
            }
        }
    }

    // The lane's rows (one a tile), and the positions of the wave's rows.
    constexpr int RT = C::RT;
    const int wrow = wave * 32 * RT, first = k.seq.len - k.seq.n;
    int token[RT], head[RT], p[RT];
    u32x4 q[RT][KB];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        row_place(a, k, k.rho0 + min(wrow + 32 * rt + c, k.nrows - 1), token[rt], head[rt]);
        p[rt] = first + token[rt];
        const uint8_t* qp = a.q + (uint64_t(k.seq.row0) + token[rt]) * a.q_stride + uint64_t(head[rt]) * D * 2 + 16 * h;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) q[rt][kb] = *reinterpret_cast<const u32x4*>(qp + 32 * kb) ^ a.q_sign;
    }
    const int wmin = uniform(first + int(a.by_r(k.rho0 + min(wrow, k.nrows - 1))));
    const int wmax = uniform(first + int(a.by_r(k.rho0 + min(wrow + 32 * RT - 1, k.nrows - 1))));
    WideRows<D> w[RT];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        w[rt].m = kNegInf;
        w[rt].L = 0.f;
        #pragma unroll
        for (int e = 0; e < EB; ++e)
            #pragma unroll
            for (int i = 0; i < 16; ++i) w[rt].O[e][i] = 0.f;
    }
    const uint32_t lds0 = uint32_t(uniform(int(uint32_t(reinterpret_cast<uintptr_t>(tiles)))));
    const WideReads<D> rd(lds0, h, c);

    // Entries all of whose tokens every row of the wave sees (between its
    // window's ends, none of them outside the pool): steps on them need no mask.
    const bool holes = uniform(__syncthreads_or(bad)) != 0;
    int seen0 = 0, seen1 = 0;
    if (!holes) {
        const int lo = a.window ? max(wmax - a.window + 1, 0) : 0;
        seen0 = k.sink_pages + max(((lo + 15) >> 4) - k.window_page, 0) - j0;
        seen1 = min(n, k.sink_pages + ((wmin + 1) >> 4) - k.window_page - j0);
    }
    seen0 = uniform(seen0);
    seen1 = uniform(seen1);
    // Three tiles in LDS, AH more on their way in registers; the page ids of
    // the one after those in idv (a lane's page l % NP).
    constexpr int R = C::RING, AH = C::AHEAD;
    TileStage<D, KVF> stage[AH];
    const int l = lane % NP;
    if (ntiles > 0) {
        #pragma unroll
        for (int i = 0; i < 3 + AH; ++i) {
            if (i >= AH) stage[i % AH].template store<F16>(tiles + (i - AH) * C::TILE, tid);
            stage[i % AH].load(a, k, ids[i * NP + l], tid);
        }
    }
    int idv = ids[(3 + AH) * NP + l];
    __syncthreads();
    // Scores run one tile ahead of the softmax, K's reads one more: each
    // step's products need nothing that the step's vector work makes.
    f16v s[RT];
    u32x4 kw[KB];
    wide_k<D>(rd, 0, kw);
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt] = wide_scores<D, F16>(kw, q[rt]);
    wide_k<D>(rd, C::TILE, kw);
    f4 fac = {a.scale_log2, 0.f, a.scale_log2, 0.f};    // the two pages' score factors and log2 of V's scales
    if constexpr (KVF == KVF_FP8) fac = *reinterpret_cast<const f4*>(scl);
    uint32_t cur = 0;                           // byte offset of the tile in the ring
    auto step = [&](auto T, int tile) __attribute__((always_inline)) {
        constexpr int turn = decltype(T)::value;
        const int j = tile * NP;
        if (__builtin_expect(j < seen0 || j + NP > seen1, 0))
            wide_mask<D, RT>(s, tiles + cur + C::VOFF, a, k, ids, j0, n, j, p, lane);
        float lm[RT];
        bool up = false;
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            lm[rt] = wide_max<KVF>(s[rt], fac);
            up = up || lm[rt] > w[rt].m + 8.f;
        }
        if (__builtin_expect(__ballot(up) != 0, 0)) {
            #pragma unroll
            for (int rt = 0; rt < RT; ++rt) wide_rescale<D>(w[rt], lm[rt]);
        }
        __builtin_amdgcn_sched_barrier(0);
        // The next scores with the weights of these between them, and V's
        // reads; then V's products with what else there is to do.
        f16v sn[RT];
        u32x4 pk[RT][2], vw[2][EB];
        wide_v<D>(rd, cur, vw);
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            sn[rt] = wide_scores<D, F16>(kw, q[rt]);
            wide_weights<KVF, F16>(s[rt], fac, w[rt].m, w[rt].L, pk[rt]);
        }
        __builtin_amdgcn_sched_barrier(0);
        wide_k<D>(rd, (cur + 2 * C::TILE) % (R * C::TILE), kw);
        if constexpr (KVF == KVF_FP8) fac = *reinterpret_cast<const f4*>(scl + j + NP);
        // The tile before is done with (the barrier below): its place takes
        // the one three ahead.  Past the list's end too: a load on some paths
        // only would make every wait for the older ones a wait for all.
        stage[(turn + 3) % AH].template store<F16>(tiles + (cur + 3 * C::TILE) % (R * C::TILE), tid);
        stage[(turn + 3) % AH].load(a, k, idv, tid);
        idv = ids[(tile + 4 + AH) * NP + l];
        #pragma unroll
        for (int g = 0; g < 2; ++g)
            #pragma unroll
            for (int e = 0; e < EB; ++e)
                #pragma unroll
                for (int rt = 0; rt < RT; ++rt) w[rt].O[e] = mma32<F16>(vw[g][e], pk[rt][g], w[rt].O[e]);
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt] = sn[rt];
        __syncthreads();
        cur = (cur + C::TILE) % (R * C::TILE);
    };
    #pragma unroll 1
    for (int base = 0; base < ntiles; base += AH) {
        static_for<0, AH>([&](auto T) {
            const int tile = base + decltype(T)::value;
            if (tile >= ntiles) return;
            step(T, tile);
        });
    }
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = pair_sum(w[rt].L) * (KVF == KVF_FP8 ? kSumUnit : 1.f);
        if (wrow + 32 * rt + c >= k.nrows) continue;
        const uint64_t at = uint64_t(k.seq.row0) + token[rt];
        if (b.parts > 1) {
            const uint64_t slot = state_slot<true>(a, b, int(C::ROWS), wrow + 32 * rt + c, at, head[rt]);
            #pragma unroll
            for (int e = 0; e < EB; ++e)
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<f4*>(a.ws_o + slot * D + 32 * e + 8 * i + 4 * h) =
                        f4{w[rt].O[e][4 * i], w[rt].O[e][4 * i + 1], w[rt].O[e][4 * i + 2], w[rt].O[e][4 * i + 3]};
            if (h == 0) *reinterpret_cast<f2*>(a.ws_ml + slot * 2) = f2{w[rt].m, sum};
            continue;
        }
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        uint8_t* o = a.out + at * a.out_stride + uint64_t(head[rt]) * D * 2;
        #pragma unroll
        for (int e = 0; e < EB; ++e)
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u32x2*>(o + 2 * (32 * e + 8 * i + 4 * h)) =
                    u32x2{pack2(w[rt].O[e][4 * i] * inv, w[rt].O[e][4 * i + 1] * inv, F16),
                          pack2(w[rt].O[e][4 * i + 2] * inv, w[rt].O[e][4 * i + 3] * inv, F16)};
    }
}

template <int D>
hipError_t launch_wide_d(const WindowArgs& a, uint32_t q_dtype, uint32_t fmt, hipStream_t s) {
    const uint64_t blocks = wide_workgroups(a, WideCfg<D>::SHIFT);
    if (blocks > 0x7FFFFFFFull) return hipErrorInvalidValue;
    const dim3 grid{uint32_t(blocks)}, block(WideCfg<D>::THREADS);
    if constexpr (D == 256) {      // (smaller heads of 16 bits: window_ring.hip)
        if (q_dtype == DH_DTYPE_BF16 && fmt == KVF_BF16) {
            hipLaunchKernelGGL((window_wide_kernel<D, KVF_BF16, false>), grid, block, 0, s, a);
            return hipGetLastError();
        }
        if (q_dtype == DH_DTYPE_F16 && fmt == KVF_F16) {
            hipLaunchKernelGGL((window_wide_kernel<D, KVF_F16, true>), grid, block, 0, s, a);
            return hipGetLastError();
        }
    }
    if (q_dtype == DH_DTYPE_BF16 && fmt == KVF_FP8)
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
