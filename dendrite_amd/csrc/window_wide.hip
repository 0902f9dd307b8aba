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

template <int D>
struct WideCfg {
    static constexpr int ROWS = int(wide_rows(D)), NW = ROWS / 32, THREADS = NW * 64;
    static constexpr int SHIFT = ROWS == 256 ? 8 : 7;
    static constexpr int TK = D == 256 ? 32 : 64;      // tokens a tile
    static constexpr int NP = TK / kPageSize;          // pages a tile
    static constexpr int RB = 2 * D, CH = RB / 16;     // row bytes, 16-byte chunks
    static constexpr int PLANE = TK * RB, TILE = 2 * PLANE;
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

// One tile on its way from the pages to LDS: this thread's words of it.
template <int D, uint32_t KVF>
struct TileRegs {
    using C = WideCfg<D>;
    static constexpr bool FP8 = KVF == KVF_FP8 || KVF == KVF_MX;
    // words of 16 bytes of K and V rows; 8-bit ones make two chunks each
    static constexpr int WPR = FP8 ? D / 16 : D / 8;
    static constexpr int N = 2 * C::TK * WPR / C::THREADS;
    u32x4 w[N];
    uint32_t sc[KVF == KVF_MX ? N : 1];
    uint32_t keep;         // bit n: word n is a token of the sequence
    static_assert(2 * C::TK * WPR % C::THREADS == 0 && (64 / WPR) * 1 <= kPageSize, "a wave's word is in one page");
};

// Where word n of thread tid lies in the tile.
template <int D, uint32_t KVF>
__device__ __forceinline__ void word_place(int n, int tid, int& plane, int& row, int& col) {
    using T = TileRegs<D, KVF>;
    const int q = tid + n * WideCfg<D>::THREADS;
    plane = q / (WideCfg<D>::TK * T::WPR);
    const int rem = q - plane * (WideCfg<D>::TK * T::WPR);
    row = rem / T::WPR;
    col = rem - row * T::WPR;
}

template <int D, uint32_t KVF>
__device__ __forceinline__ void load_tile(TileRegs<D, KVF>& r, const WindowArgs& a, const RowBlock& k, const int* ids,
                                          int j0, int n, int tile, int tid) {
    using C = WideCfg<D>;
    using T = TileRegs<D, KVF>;
    constexpr int EB = T::FP8 ? 1 : 2;
    r.keep = 0;
    #pragma unroll
    for (int i = 0; i < T::N; ++i) {
        int plane, row, col;
        word_place<D, KVF>(i, tid, plane, row, col);
        const int j = uniform(tile * C::NP + (row >> 4));       // a wave's word is in one page
        const int id = j < n ? uniform(ids[j]) : -1;
        const uint32_t page = uint32_t(max(id, 0));
        const uint64_t blk = (uint64_t(page) * 2 + uniform(plane)) * a.hkv + k.kv_head;
        r.w[i] = *reinterpret_cast<const u32x4*>(a.kv + blk * (kPageSize * D * EB) + ((row & 15) * (D * EB) + col * 16));
        if constexpr (KVF == KVF_MX)
            r.sc[i] = a.scales[blk * (kPageSize * D / 32) + (row & 15) * (D / 32) + col / 2];
        const int t = 16 * list_page(k, j0 + j) + (row & 15);
        r.keep |= (id >= 0 && t < k.seq.len ? 1u : 0u) << i;
    }
}

template <int D, uint32_t KVF, bool F16>
__device__ __forceinline__ void store_tile(const TileRegs<D, KVF>& r, uint8_t* lds, int tid) {
    using C = WideCfg<D>;
    using T = TileRegs<D, KVF>;
    #pragma unroll
    for (int i = 0; i < T::N; ++i) {
        int plane, row, col;
        word_place<D, KVF>(i, tid, plane, row, col);
        uint8_t* p = lds + plane * C::PLANE + row * C::RB;
        const bool keep = (r.keep >> i) & 1;
        const u32x4 w = keep ? r.w[i] : u32x4{0u, 0u, 0u, 0u};
        if constexpr (!T::FP8) {
            *reinterpret_cast<u32x4*>(p + ((col ^ wide_swz<D>(row)) << 4)) = w;
        } else {
            const float sc = KVF == KVF_MX && keep ? e8m0_to_float(r.sc[i]) : 1.f;
            uint32_t o[8];
            #pragma unroll
            for (int e = 0; e < 4; ++e) e4m3x4_cvt<F16>(w[e], sc, o[2 * e], o[2 * e + 1]);
            *reinterpret_cast<u32x4*>(p + (((2 * col) ^ wide_swz<D>(row)) << 4)) = u32x4{o[0], o[1], o[2], o[3]};
            *reinterpret_cast<u32x4*>(p + (((2 * col + 1) ^ wide_swz<D>(row)) << 4)) = u32x4{o[4], o[5], o[6], o[7]};
        }
    }
}

__device__ __forceinline__ float pair_max(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float pair_sum(float x) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

template <int D, uint32_t KVF, bool F16>
__global__ __launch_bounds__(WideCfg<D>::THREADS, D == 256 ? 1 : 2) void window_wide_kernel(WindowArgs a) {
    using C = WideCfg<D>;
    constexpr int TK = C::TK, NP = C::NP, SUB = TK / 32, EB = D / 32, KB = D / 16;
    __shared__ __attribute__((aligned(1024))) uint8_t tiles[2][C::TILE];
    __shared__ int ids[kWideMaxPages];
    report_bad_tables(a.t, a.status, blockIdx.x);
    const uint32_t x0 = blockIdx.x / a.hkv;
    const uint32_t unit = x0 / a.splits;
    const int split = int(x0 - unit * a.splits);
    const RowBlock k = find_rows<C::SHIFT>(a, unit, int(blockIdx.x - x0 * a.hkv));
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
    int per = (k.pages + int(a.splits) - 1) / int(a.splits);
    per = (per + NP - 1) / NP * NP;
    const int j0 = min(split * per, k.pages), n = min(min(per, k.pages - j0), int(kWideMaxPages));
    const int ntiles = (n + NP - 1) / NP;
    for (int j = tid; j < n; j += C::THREADS)
        ids[j] = checked_page(a.t.indices[k.seq.page0 + list_page(k, j0 + j)], a.page_limit, a.status);

    // The lane's row, and what the wave's rows see.
    const int wrow = wave * 32, mine = wrow + c;
    const bool live = mine < k.nrows;
    const int rho = k.rho0 + min(mine, k.nrows - 1);
    int token, head;
    row_place(a, k, rho, token, head);
    const int first = k.seq.len - k.seq.n;
    const int p = first + token, lo = a.window ? p - a.window + 1 : 0;
    const int wmin = first + (k.rho0 + min(wrow, k.nrows - 1)) / int(a.r);
    const int wmax = first + (k.rho0 + min(wrow + 31, k.nrows - 1)) / int(a.r);
    const int wlo_min = a.window ? wmin - a.window + 1 : 0, wlo_max = a.window ? wmax - a.window + 1 : 0;
    u32x4 q[KB];
    {
        const uint8_t* qp = a.q + (uint64_t(k.seq.row0) + token) * a.q_stride + uint64_t(head) * D * 2 + 16 * h;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) q[kb] = *reinterpret_cast<const u32x4*>(qp + 32 * kb) ^ a.q_sign;
    }
    float m = kNegInf, L = 0.f;
    f16v O[EB];
    #pragma unroll
    for (int e = 0; e < EB; ++e)
        #pragma unroll
        for (int i = 0; i < 16; ++i) O[e][i] = 0.f;

    TileRegs<D, KVF> stage;
    __syncthreads();
    if (ntiles > 0) {
        load_tile<D, KVF>(stage, a, k, ids, j0, n, 0, tid);
        store_tile<D, KVF, F16>(stage, tiles[0], tid);
        if (ntiles > 1) load_tile<D, KVF>(stage, a, k, ids, j0, n, 1, tid);
    }
    // LDS byte offsets of the lane's K and V reads inside a plane.
    const uint32_t kbase = c * C::RB, ksw = wide_swz<D>(c);
    const int vrow = 4 * h + ((c & 15) >> 2);
    const uint32_t vcol = 2 * (c >> 4) + ((c & 3) >> 1), vhalf = (c & 1) << 3;

    #pragma unroll 1
    for (int tile = 0; tile < ntiles; ++tile) {
        __syncthreads();       // the tile is in; the other buffer is free
        uint8_t* cur = tiles[tile & 1];
        // Pages of the tile: masked, or wholly in sight of every row.
        int t0[NP];
        float ks[NP], vs[NP];
        bool full = true, some = false;
        #pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int j = tile * NP + i;
            const int id = j < n ? uniform(ids[j]) : -1;
            t0[i] = id >= 0 ? 16 * list_page(k, j0 + j) : 0x7FFFFF00;
            full = full && t0[i] + 15 <= wmin && (t0[i] >= wlo_max || t0[i] + 15 < a.sinks);
            some = some || (t0[i] <= wmax && (t0[i] + 15 >= wlo_min || t0[i] < a.sinks));
            ks[i] = vs[i] = 1.f;
            if constexpr (KVF == KVF_FP8) {
                const float* s = reinterpret_cast<const float*>(a.scales) + uint64_t(max(id, 0)) * 2 * a.hkv + k.kv_head;
                ks[i] = id < 0 ? 1.f : s[0];
                vs[i] = id < 0 ? 1.f : s[a.hkv];
            }
        }
        if (tile + 1 < ntiles) {
            store_tile<D, KVF, F16>(stage, tiles[(tile + 1) & 1], tid);
            if (tile + 2 < ntiles) load_tile<D, KVF>(stage, a, k, ids, j0, n, tile + 2, tid);
        }
        if (!some) continue;
        f16v s[SUB];
        #pragma unroll
        for (int u = 0; u < SUB; ++u) {
            #pragma unroll
            for (int i = 0; i < 16; ++i) s[u][i] = 0.f;
            #pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const u32x4 kw = *reinterpret_cast<const u32x4*>(cur + u * 32 * C::RB + kbase + (((2 * kb + h) ^ ksw) << 4));
                s[u] = mma32<F16>(kw, q[kb], s[u]);
            }
        }
        if (!full) {
            #pragma unroll
            for (int u = 0; u < SUB; ++u)
                #pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int t = t0[2 * u + i / 8] + 8 * ((i / 4) & 1) + 4 * h + i % 4;
                    if (!(t <= p && (t >= lo || t < a.sinks))) s[u][i] = kNegInf;
                }
        }
        float f[NP], lm = kNegInf;
        #pragma unroll
        for (int g = 0; g < NP; ++g) {
            f[g] = KVF == KVF_FP8 ? fmaxf(a.scale_log2 * ks[g], 1e-30f) : a.scale_log2;
            float x = s[g / 2][8 * (g & 1)];
            #pragma unroll
            for (int i = 1; i < 8; ++i) x = fmaxf(x, s[g / 2][8 * (g & 1) + i]);
            lm = fmaxf(lm, x * f[g]);
        }
        // The reference moves only when a score passes it by 8.
        if (__ballot(lm > m + 8.f)) {
            const float mx = pair_max(lm);
            const float mnew = mx > m + 8.f ? mx : m;
            const float alpha = m == kNegInf ? 0.f : fast_exp2(m - mnew);
            m = mnew;
            L *= alpha;
            #pragma unroll
            for (int e = 0; e < EB; ++e) O[e] *= alpha;
        }
        const float nm = m == kNegInf ? 0.f : -m;
        u32x4 pk[2 * SUB];
        #pragma unroll
        for (int g = 0; g < NP; ++g) {
            float x[8];
            #pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = fast_exp2(__builtin_fmaf(s[g / 2][8 * (g & 1) + i], f[g], nm));
                L += x[i];
                if constexpr (KVF == KVF_FP8) x[i] *= vs[g];
            }
            pk[g] = u32x4{pack2(x[0], x[1], F16), pack2(x[2], x[3], F16), pack2(x[4], x[5], F16), pack2(x[6], x[7], F16)};
        }
        #pragma unroll
        for (int g = 0; g < NP; ++g) {
            #pragma unroll
            for (int e = 0; e < EB; ++e) {
                u32x4 vw;
                #pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = 16 * g + 8 * half + vrow;
                    const uint32_t at = C::PLANE + row * C::RB + (((4 * e + vcol) ^ wide_swz<D>(row)) << 4) + vhalf;
                    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(cur + at));
                    const u32x2 vv = __builtin_bit_cast(u32x2, v);
                    vw[2 * half] = vv[0];
                    vw[2 * half + 1] = vv[1];
                }
                O[e] = mma32<F16>(vw, pk[g], O[e]);
            }
        }
    }
    const float sum = pair_sum(L);
    if (!live) return;
    const uint64_t at = uint64_t(k.seq.row0) + token;
    if (a.splits > 1) {
        const uint64_t slot = (at * a.hq + head) * a.splits + split;
        #pragma unroll
        for (int e = 0; e < EB; ++e)
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<f4*>(a.ws_o + slot * D + 32 * e + 8 * i + 4 * h) =
                    f4{O[e][4 * i], O[e][4 * i + 1], O[e][4 * i + 2], O[e][4 * i + 3]};
        if (h == 0) *reinterpret_cast<f2*>(a.ws_ml + slot * 2) = f2{m, sum};
        return;
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    uint8_t* o = a.out + at * a.out_stride + uint64_t(head) * D * 2;
    #pragma unroll
    for (int e = 0; e < EB; ++e)
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x2*>(o + 2 * (32 * e + 8 * i + 4 * h)) =
                u32x2{pack2(O[e][4 * i] * inv, O[e][4 * i + 1] * inv, F16),
                      pack2(O[e][4 * i + 2] * inv, O[e][4 * i + 3] * inv, F16)};
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
