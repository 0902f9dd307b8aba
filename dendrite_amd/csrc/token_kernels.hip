// Token-wise cache writes and reads from device tables: the new tokens' K / V
// quantised into their sequences' pages (dh_pool_append_tokens, the device half
// of ReferenceBackend::append_kv, crates/dendrite-core/src/attention/
// backend.rs:285-301, for a batch) and the inverse (dh_pool_read_tokens).
//
// One wave per (page a sequence's new tokens touch, K|V, KV head): a block of
// up to 16 rows of D elements.  Lane l holds 8 consecutive elements (a 16-byte
// word of 16-bit rows) of rows l / (D / 8) + k * 512 / D, so a load or store
// instruction covers whole rows in order and a 32-element MX group lies in four
// neighbouring lanes.
//
// Long calls are bound by their bytes (six prompts of 301 to 2500 tokens into
// MXFP8, 8 heads of 128: 15 us, 4.0 TB/s; four prefixes of 2000 to 9000 read back
// from FP8: 23 us, 6.3 TB/s), a decode step's by its dependent loads: search,
// sequence, page, scale (256 tokens into FP8 pages: 7.7 us; 601 tokens read back
// 3.4).  Rows are loaded beside the page id that says where they go.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "token_device.hpp"

namespace dh {
namespace {

typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef uint32_t w2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

// DH_DTYPE_* and the unscaled DH_KV_* formats have the same numbers.
constexpr uint32_t kF16 = 0, kBF16 = 1, kF32 = 2, kFP8 = 3, kMX = 4;
constexpr float kScaleFloor = 0x1p-64f;   // least block scale of a written FP8 block

// Eight elements of type T from / to a 16-byte aligned address.
template <uint32_t T>
__device__ __forceinline__ void load8(const uint8_t* p, float (&x)[8]) {
    if constexpr (T == kF32) {
        const w4 a = reinterpret_cast<const w4*>(p)[0], b = reinterpret_cast<const w4*>(p)[1];
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(a[i]);
            x[4 + i] = __uint_as_float(b[i]);
        }
    } else {
        const w4 a = *reinterpret_cast<const w4*>(p);
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = a[i];     // a bit_cast of the vector's element itself reads element 0
            if constexpr (T == kBF16) {
                x[2 * i] = __uint_as_float(w << 16);
                x[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
            } else {
                const h2 v = __builtin_bit_cast(h2, w);
                x[2 * i] = float(v[0]);
                x[2 * i + 1] = float(v[1]);
            }
        }
    }
}

// One store of a row that the call writes out (ROW: past the caches, which a
// long read would only push other lines out of: four prefixes of 2000 to 9000
// tokens from FP8 in 23 us, 6.3 TB/s, and 34 through them), or into a page, which
// attention reads next.
template <bool ROW, class V>
__device__ __forceinline__ void put(V* p, V x) {
    if constexpr (ROW) __builtin_nontemporal_store(x, p);
    else *p = x;
}

template <uint32_t T, bool ROW>
__device__ __forceinline__ void store8(uint8_t* p, const float (&x)[8]) {
    if constexpr (T == kF32) {
        #pragma unroll
        for (int j = 0; j < 2; ++j)
            put<ROW>(reinterpret_cast<w4*>(p) + j, w4{__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]),
                                                      __float_as_uint(x[4 * j + 2]), __float_as_uint(x[4 * j + 3])});
    } else {
        w4 o;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (T == kBF16) o[i] = __builtin_bit_cast(uint32_t, b2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
            else o[i] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        }
        put<ROW>(reinterpret_cast<w4*>(p), o);
    }
}

// E4M3 codes of eight values, round to nearest even, saturated at +-448 (the
// comparisons let a NaN through: its code is NaN).
__device__ __forceinline__ w2 encode8(const float (&y)[8]) {
    auto cl = [](float v) { return v > 448.f ? 448.f : (v < -448.f ? -448.f : v); };
    w2 o;
    #pragma unroll
    for (int j = 0; j < 2; ++j) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(y[4 * j]), cl(y[4 * j + 1]), 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(cl(y[4 * j + 2]), cl(y[4 * j + 3]), w, true);
        o[j] = uint32_t(w);
    }
    return o;
}

__device__ __forceinline__ void decode8(w2 c, float (&x)[8]) {
    #pragma unroll
    for (int j = 0; j < 2; ++j) {
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j]), false);
        const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j]), true);
        x[4 * j] = lo[0];
        x[4 * j + 1] = lo[1];
        x[4 * j + 2] = hi[0];
        x[4 * j + 3] = hi[1];
    }
}

// Largest finite magnitude of eight elements.
__device__ __forceinline__ float amax8(const float (&x)[8]) {
    float a = 0.f;
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = fabsf(x[i]);
        a = fmaxf(a, v < __builtin_inff() ? v : 0.f);
    }
    return a;
}

__device__ __forceinline__ float wave_max(float x) {
    #pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// Times a block's scale s has to be doubled for amax > limit = 448 s: the
// least k with amax <= limit 2^k, from both as [0.5, 1) times a power of two.
__device__ __forceinline__ int doublings(float amax, float limit) {
    return __builtin_amdgcn_frexp_expf(amax) - __builtin_amdgcn_frexp_expf(limit) +
           (__builtin_amdgcn_frexp_mantf(amax) > __builtin_amdgcn_frexp_mantf(limit) ? 1 : 0);
}

// A wave's block: slots [lo, hi) of table entry `entry` of its sequence are
// the call's, slot t being row row0 + t.
struct Block {
    int entry, lo, hi;
    int64_t row0;
    uint32_t plane, head;
    bool any;
};

__device__ __forceinline__ Block find_block(const TokenCopyArgs& a) {
    Block k{};
    const uint32_t per = 2 * a.hkv;
    const uint32_t item = blockIdx.x * 4 + uint32_t(uniform(threadIdx.x >> 6));
    const uint32_t unit = a.by_planes(item), ph = item - unit * per;
    k.plane = ph >= a.hkv ? 1u : 0u;
    k.head = ph - k.plane * a.hkv;
    uint32_t u = 0;
    Sequence s;
    if (a.t.q_indptr) {
        s = find_sequence(a.t, unit, 1, 4, 2, u);
    } else {
        if (unit >= a.t.batch) return k;
        s = uniform_sequence(load_sequence(a.t, unit));
    }
    if (!s.ok || s.n == 0) return k;
    const int first = s.len - s.n, last_page = (s.len - 1) >> 4;
    if (u > uint32_t(last_page - (first >> 4))) return k;
    const int page = (first >> 4) + int(u);
    k.entry = s.page0 + page;
    k.lo = max(first - 16 * page, 0);
    k.hi = min(s.len - 16 * page, 16);
    k.row0 = int64_t(s.row0) + 16 * int64_t(page) - first;
    k.any = true;
    return k;
}

template <int D, uint32_t SRC, uint32_t FMT>
__global__ __launch_bounds__(256) void append_tokens_kernel(TokenCopyArgs a) {
    constexpr int LPR = D / 8, RPI = 64 / LPR, NI = kPageSize / RPI;   // lanes a row, rows a step, steps
    constexpr uint32_t EB = SRC == kF32 ? 4 : 2;
    const bool refused = sees_refused(a.t, blockIdx.x);
    const Block k = find_block(a);
    report(refused, a.status);
    if (!k.any) return;
    const int lane = threadIdx.x & 63, cd = lane % LPR, lr = lane / LPR;
    const int id = uniform(a.t.indices[k.entry]);
    // The rows do not depend on the page: both loads go out together.
    const uint8_t* src = (k.plane ? a.v : a.k) + (uint64_t(k.head) * D + 8 * cd) * EB;
    const uint64_t stride = k.plane ? a.v_stride : a.k_stride;
    float x[NI][8];
    #pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int t = i * RPI + lr;
        if (t >= k.lo && t < k.hi) {
            load8<SRC>(src + uint64_t(k.row0 + t) * stride, x[i]);
        } else {
            #pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        }
    }
    const int page = checked_page(id, a.num_pages, a.status);
    if (page < 0) return;
    const uint64_t blk = (uint64_t(page) * 2 + k.plane) * a.hkv + k.head;
    if constexpr (FMT == kFP8) {
        float* sp = reinterpret_cast<float*>(a.scales) + blk;
        uint8_t* dst = a.data + blk * (kPageSize * D) + 8 * cd;
        const float old = k.lo > 0 ? *sp : 0.f;
        float amax = 0.f;
        #pragma unroll
        for (int i = 0; i < NI; ++i) amax = fmaxf(amax, amax8(x[i]));
        amax = wave_max(amax);
        float sc;
        if (old > 0.f && old < __builtin_inff()) {
            sc = old;
            if (amax > 448.f * old) {
                // Powers of two: an earlier code loses nothing unless it
                // becomes subnormal, however often its block grows.
                const int n = doublings(amax, 448.f * old);
                sc = __builtin_amdgcn_ldexpf(old, n);
                #pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int t = i * RPI + lr;
                    if (t < k.lo) {
                        float y[8];
                        w2* p = reinterpret_cast<w2*>(dst + t * D);
                        decode8(*p, y);
                        #pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_ldexpf(y[e], -n);
                        *p = encode8(y);
                    }
                }
            }
        } else {
            sc = fmaxf(amax / 448.f, kScaleFloor);
        }
        #pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = i * RPI + lr;
            if (t >= k.lo && t < k.hi) {
                #pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = x[i][e] / sc;
                *reinterpret_cast<w2*>(dst + t * D) = encode8(x[i]);
            }
        }
        if (lane == 0) *sp = sc;
    } else if constexpr (FMT == kMX) {
        uint8_t* dst = a.data + blk * (kPageSize * D) + 8 * cd;
        uint8_t* sp = a.scales + blk * (kPageSize * D / 32) + cd / 4;
        #pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = i * RPI + lr;
            float m = amax8(x[i]);
            m = fmaxf(m, __shfl_xor(m, 1, 64));
            m = fmaxf(m, __shfl_xor(m, 2, 64));
            // floor(log2 amax) - 8 (E4M3's largest exponent), within E8M0
            const int e0 = m > 0.f ? min(127, max(-127, __builtin_amdgcn_frexp_expf(m) - 9)) : -127;
            if (t >= k.lo && t < k.hi) {
                #pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = __builtin_amdgcn_ldexpf(x[i][e], -e0);
                *reinterpret_cast<w2*>(dst + t * D) = encode8(x[i]);
                if ((cd & 3) == 0) sp[t * (D / 32)] = uint8_t(e0 + 127);
            }
        }
    } else {
        constexpr int DB = FMT == kF32 ? 4 : 2;
        uint8_t* dst = a.data + (blk * (kPageSize * D) + 8 * cd) * DB;
        #pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int t = i * RPI + lr;
            if (t >= k.lo && t < k.hi) store8<FMT, false>(dst + t * (D * DB), x[i]);
        }
    }
}

template <int D, uint32_t DST, uint32_t FMT>
__global__ __launch_bounds__(256) void read_tokens_kernel(TokenCopyArgs a) {
    constexpr int LPR = D / 8, RPI = 64 / LPR, NI = kPageSize / RPI;
    constexpr uint32_t EB = DST == kF32 ? 4 : 2;
    constexpr bool CODES = FMT == kFP8 || FMT == kMX;
    constexpr int SB = CODES ? 1 : (FMT == kF32 ? 4 : 2);
    const bool refused = sees_refused(a.t, blockIdx.x);
    const Block k = find_block(a);
    report(refused, a.status);
    if (!k.any) return;
    const int lane = threadIdx.x & 63, cd = lane % LPR, lr = lane / LPR;
    const int page = checked_page(uniform(a.t.indices[k.entry]), a.num_pages, a.status);
    uint8_t* dst = (k.plane ? a.v : a.k) + (uint64_t(k.head) * D + 8 * cd) * EB;
    const uint64_t stride = k.plane ? a.v_stride : a.k_stride;
    const uint64_t blk = (uint64_t(max(page, 0)) * 2 + k.plane) * a.hkv + k.head;
    const uint8_t* src = a.data + (blk * (kPageSize * D) + 8 * cd) * SB;
    float x[NI][8];
    float sc = 1.f;
    if constexpr (FMT == kFP8) sc = reinterpret_cast<const float*>(a.scales)[blk];
    #pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int t = i * RPI + lr;
        #pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
        if (page >= 0 && t >= k.lo && t < k.hi) {
            if constexpr (CODES) {
                decode8(*reinterpret_cast<const w2*>(src + t * D), x[i]);
                if constexpr (FMT == kMX) {
                    const uint32_t e0 = a.scales[(blk * kPageSize + t) * (D / 32) + cd / 4];
                    #pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[i][e] = e0 == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(x[i][e], int(e0) - 127);
                } else {
                    #pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][e] *= sc;
                }
            } else {
                load8<FMT>(src + t * (D * SB), x[i]);
            }
        }
    }
    #pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int t = i * RPI + lr;
        if (t >= k.lo && t < k.hi) store8<DST, true>(dst + uint64_t(k.row0 + t) * stride, x[i]);
    }
}

// Units a call may need: one a sequence, or the bound find_sequence counts by
// (16 rows a page, and a sequence touches at most two pages more than n / 16).
uint64_t token_units(const TokenTables& t) {
    return t.q_indptr ? (uint64_t(t.rows) >> 4) + 2 * uint64_t(t.batch) : t.batch;
}

template <bool APPEND, int D, uint32_t ROW, uint32_t FMT>
hipError_t launch_one(const TokenCopyArgs& a, hipStream_t s) {
    const uint64_t blocks = (token_units(a.t) * 2 * a.hkv + 3) / 4;
    if (blocks > 0x1FFFFFFFull) return hipErrorInvalidValue;     // four items a workgroup in 31 bits
    if constexpr (APPEND)
        hipLaunchKernelGGL((append_tokens_kernel<D, ROW, FMT>), dim3(uint32_t(blocks)), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((read_tokens_kernel<D, ROW, FMT>), dim3(uint32_t(blocks)), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <bool APPEND, int D, uint32_t ROW>
hipError_t launch_fmt(const TokenCopyArgs& a, uint32_t fmt, hipStream_t s) {
    switch (fmt) {
        case kF16: return launch_one<APPEND, D, ROW, kF16>(a, s);
        case kBF16: return launch_one<APPEND, D, ROW, kBF16>(a, s);
        case kF32: return launch_one<APPEND, D, ROW, kF32>(a, s);
        case kFP8: return launch_one<APPEND, D, ROW, kFP8>(a, s);
        case kMX: return launch_one<APPEND, D, ROW, kMX>(a, s);
        default: return hipErrorInvalidValue;
    }
}

template <bool APPEND, int D>
hipError_t launch_row(const TokenCopyArgs& a, uint32_t row, uint32_t fmt, hipStream_t s) {
    switch (row) {
        case kF16: return launch_fmt<APPEND, D, kF16>(a, fmt, s);
        case kBF16: return launch_fmt<APPEND, D, kBF16>(a, fmt, s);
        case kF32: return launch_fmt<APPEND, D, kF32>(a, fmt, s);
        default: return hipErrorInvalidValue;
    }
}

template <bool APPEND>
hipError_t launch_d(const TokenCopyArgs& a, uint32_t row, uint32_t fmt, uint32_t d, void* stream) {
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (d) {
        case 64: return launch_row<APPEND, 64>(a, row, fmt, s);
        case 128: return launch_row<APPEND, 128>(a, row, fmt, s);
        case 256: return launch_row<APPEND, 256>(a, row, fmt, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

int launch_append_tokens(const TokenCopyArgs& a, uint32_t src_dtype, uint32_t fmt, uint32_t d, void* stream) {
    return launch_d<true>(a, src_dtype, fmt, d, stream);
}

int launch_read_tokens(const TokenCopyArgs& a, uint32_t dst_dtype, uint32_t fmt, uint32_t d, void* stream) {
    return launch_d<false>(a, dst_dtype, fmt, d, stream);
}

}  // namespace dh
