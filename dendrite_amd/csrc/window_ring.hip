// Windowed attention of many query rows a sequence over 16-bit caches of heads
// of 64 or 128 dims, from device tables: chunks of prompts (dh_attend_window).
//
// A workgroup of four waves has 128 rows (two tiles of 16 a wave) of one KV
// head and walks the block's page list two pages (32 tokens) a step.  Pages go
// straight from memory into an LDS ring of four pairs (global_load_lds), so
// that no register or vector instruction is spent on them; a step computes the
// scores of the next pair and finishes this one:
//   S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32, lane l = 16 g + c
//   holding row c of its tiles, probabilities in registers throughout
// (attend_device.hpp has the layout and the reads).  What a row does not see is
// masked in the steps at its window's ends only: the others are known by their
// place in the list, and the mask stands apart from the one copy of the step
// (two copies, masked and not, took 208 registers more than there are).
//
// Bound by the matrix cores' clock: 4096 tokens over 8192, 32 heads of 128 dims,
// window 4096, run at 1.08 to 1.15 PFLOP/s (240 to 255 us, bf16; the matrix unit
// busy 55 % of the cycles), as a large library product does (1.08).  Pages staged
// through registers instead (window_wide.hip) 340 us; one workgroup a CU, which
// two copies of the step allow, 560.  Heads of 64: three workgroups a CU (168
// registers) 92 us at 4096 tokens x 32 heads over 2048 and 35 at 12 prompts of
// 500, two 96 and 40; short windows' blocks are bound by their start (12 prompts,
// window 256: 52 us, 16 % busy).
#include "attend_device.hpp"
#include "window_device.hpp"

namespace dh {
namespace {

// Masks the scores of list entries j, j + 1 that the lane's rows (positions p)
// do not see, and zeroes their V rows (in LDS, slot `v` of the pair) past the
// sequence's end: those weights are zero, but what lies there need not be a
// number.  Every wave does so for itself before it reads them.
template <int D, int RT>
__device__ __forceinline__ void mask_pair(f4 (&s)[RT][2], uint8_t* v, const WindowArgs& a, const RowBlock& k,
                                          const int* ids, int j0, int n, int j, const int (&p)[RT], int lane) {
    using C = DmaCfg<D>;
    #pragma unroll
    for (int q = 0; q < 2; ++q) {
        const bool ok = j + q < n && uniform(ids[j + q]) >= 0;
        const int t0 = ok ? 16 * list_page(k, j0 + j + q) : 0x7FFFFF00;      // nobody sees that
        const int held = max(k.seq.len - t0, 0);
        for (int i = held * C::RB + 16 * lane; i < C::PLANE; i += 1024)
            *reinterpret_cast<u32x4*>(v + q * C::PAGE + C::PLANE + i) = u32x4{0u, 0u, 0u, 0u};
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            // bit t of see: the row sees token t0 + t
            auto below = [](int y) { return (1u << min(max(y, 0), 16)) - 1u; };
            uint32_t see = below(p[rt] - t0 + 1);
            if (a.window) see &= ~below(p[rt] - a.window + 1 - t0) | below(a.sinks - t0);
            see >>= 4 * (lane >> 4);
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(see >> i & 1u)) s[rt][q][i] = kNegInf;
        }
    }
}

// Largest raw score of the lane's eight.
__device__ __forceinline__ float pair_max8(const f4 (&x)[2]) {
    const float a = fmaxf(fmaxf(x[0][0], x[0][1]), x[0][2]);
    const float b = fmaxf(fmaxf(a, x[0][3]), x[1][0]);
    const float c = fmaxf(fmaxf(b, x[1][1]), x[1][2]);
    return fmaxf(c, x[1][3]);
}

// One step of the pair loop (dma_step's order): the reference check of the
// pair whose scores are in sc, then K of the next pair, the probabilities
// while it lands, the next scores with V's reads between them, V's products.
template <int D, bool F16, bool NEXT>
__device__ __forceinline__ void window_step(uint32_t vs, uint32_t ks, const LdsBases<D>& lb,
                                            const u32x4 (&qB)[DmaCfg<D>::RT][D / 32], f4 (&sc)[DmaCfg<D>::RT][2],
                                            RowMax<DmaCfg<D>::RT>& rm, f4 (&L)[DmaCfg<D>::RT],
                                            f4 (&O)[DmaCfg<D>::RT][D / 16], float f, float finv) {
    constexpr int RT = DmaCfg<D>::RT, KB = D / 32;
    bool need = false;
    float lm[RT];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        lm[rt] = pair_max8(sc[rt]);
        need |= lm[rt] > rm.thr[rt];
    }
    if (__builtin_expect(__ballot(need) != 0, 0)) dma_rescale<D, RT, F16>(lm, rm, L, O, f, finv);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 kop[2][KB];
    if constexpr (NEXT) dma_k_operands<D>(ks, lb, kop);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 pB[RT];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        // a row that has seen nothing yet: its scores are -inf, its weights 0
        const float m = rm.m[rt] == kNegInf ? 0.f : rm.m[rt];
        pB[rt] = dma_probs<F16>(sc[rt], f, f, m, L[rt]);
    }
    __builtin_amdgcn_sched_barrier(0);
    u32x4 vop[D / 16];
    dma_v_operands<D>(vs, lb, vop);
    if constexpr (NEXT) {
        dma_score_mma<D, F16, RT>(kop, qB, sc);
        constexpr int NM = RT * 2 * KB, NV = D / 8;   // score MFMAs, V reads
        #pragma unroll
        for (int i = 0; i < (NM > NV ? NM : NV); ++i) {
            if (i < NV) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // one LDS read
            if (i < NM) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // one MFMA
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    #pragma unroll
    for (int e = 0; e < D / 16; ++e) {
        #pragma unroll
        for (int rt = 0; rt < RT; ++rt) O[rt][e] = mma16v<F16>(vop[e], pB[rt], O[rt][e]);
    }
}

template <int D, bool F16>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void window_ring_kernel(WindowArgs a) {
    using C = DmaCfg<D>;
    constexpr int RT = C::RT, KB = D / 32;
    constexpr uint32_t P = C::NP, SLOT = 2 * C::PAGE;
    static_assert(kRingRows == RT * kWaves * kTileRows, "rows a block");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[C::RING];
    __shared__ int ids[kRingMaxPages + 2 * (P + 1)];
    const bool refused = sees_refused(a.t, blockIdx.x);
    const BlockPart b = block_part<D != 64>(a);
    const RowBlock k = uniform_block(find_rows<kRingShift>(a, b.unit, b.head));
    report(refused, a.status);
    if (k.nrows == 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), g = lane >> 4, c = lane & 15;
    if (k.zero) {
        if (b.parts == 1) zero_rows<D, DH_DTYPE_F16>(a, k);     // (else the merge writes them)
        return;
    }
    // This workgroup's part of the page list, whole pairs.
    int per = part_pages<D != 64>(a, b, k.pages);
    per += per & 1;
    const int j0 = min(b.split * per, k.pages), n = min(min(per, k.pages - j0), int(kRingMaxPages));
    const uint32_t npairs = uint32_t(n + 1) >> 1;
    int bad = 0;
    for (int j = tid; j < n + 2 * int(P + 1); j += 256) {
        int id = -1;
        if (j < n) {
            id = checked_page(a.t.indices[k.seq.page0 + list_page(k, j0 + j)], a.page_limit, a.status);
            bad |= id < 0 ? 1 : 0;
        }
        ids[j] = id;
    }
    // The lane's rows (one a tile) and their queries.
    const int first = k.seq.len - k.seq.n;
    int token[RT], head[RT], p[RT];
    u32x4 qB[RT][KB];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        row_place(a, k, k.rho0 + min((rt * kWaves + wave) * kTileRows + c, k.nrows - 1), token[rt], head[rt]);
        p[rt] = first + token[rt];
        const uint8_t* qp = a.q + (uint64_t(k.seq.row0) + token[rt]) * a.q_stride + uint64_t(head[rt]) * D * 2 + 16 * g;
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) qB[rt][kb] = *reinterpret_cast<const u32x4*>(qp + 64 * kb) ^ a.q_sign;
    }
    // Entries all of whose tokens every row of the wave sees: no mask needed.
    const bool holes = uniform(__syncthreads_or(bad)) != 0;
    int seen0 = 0, seen1 = 0;
    if (!holes) {
        const int last = k.nrows - 1;
        const int wmin = first + int(a.by_r(k.rho0 + min(wave * kTileRows, last)));
        const int wmax = first + int(a.by_r(k.rho0 + min(((RT - 1) * kWaves + wave) * kTileRows + kTileRows - 1, last)));
        const int lo = a.window ? max(wmax - a.window + 1, 0) : 0;
        seen0 = k.sink_pages + max(((lo + 15) >> 4) - k.window_page, 0) - j0;
        seen1 = min(n, k.sink_pages + ((wmin + 1) >> 4) - k.window_page - j0);
    }
    seen0 = uniform(seen0);
    seen1 = uniform(seen1);

    RowMax<RT> rm;
    f4 L[RT], O[RT][D / 16];
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        rm.m[rt] = kNegInf;
        rm.thr[rt] = kNegInf;
        L[rt] = f4{0.f, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int e = 0; e < D / 16; ++e) O[rt][e] = f4{0.f, 0.f, 0.f, 0.f};
    }
    const float f = a.scale_log2, finv = 1.f / f;
    AttendArgs kv{};
    kv.kv = a.kv;
    DmaSrc src;
    src.page_stride = uint64_t(2) * a.hkv * C::PLANE;
    #pragma unroll
    for (int u = 0; u < C::DPP; ++u) {
        const int b = (wave * C::DPP + u) * 1024 + 16 * lane;
        const int plane = b / C::PLANE, rem = b - plane * C::PLANE;
        const int row = rem / C::RB, pos = (rem - row * C::RB) >> 4;
        src.loff[u] = uint32_t((plane * a.hkv + k.kv_head) * C::PLANE + row * C::RB + (pos ^ chunk_swz<D>(row)) * 16);
    }
    const uint32_t ring_lds = uint32_t(uniform(int(uint32_t(reinterpret_cast<uintptr_t>(ring)))));
    const LdsBases<D> lb = lds_bases<D>(ring_lds, g, c);
    // Entry j of the part as a page to load: one outside the pool, or past the
    // list's end, loads page 0, which nobody sees.
    auto page = [&](int j) { return uint32_t(max(uniform(ids[j]), 0)); };
    // Every load the compiler issued (queries, page ids) has landed before the
    // ring's start, so that no wait of its own drains the ring.
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        #pragma unroll
        for (int kb = 0; kb < KB; ++kb) asm volatile("" : "+v"(qB[rt][kb]));
    __builtin_amdgcn_s_waitcnt(0x0070);
    compiler_fence();
    if (npairs > 0) {
        const uint32_t pro = min(P - 1, npairs);
        #pragma unroll 1
        for (uint32_t q = 0; q < pro; ++q) dma_pair_pages<D>(kv, page(2 * q), page(2 * q + 1), src, ring_lds, q, wave);
        f4 sc[RT][2];
        wait_vmcnt((pro - 1) * C::PER_PAIR);   // pair 0 has landed
        block_barrier();
        dma_scores<D, F16, RT>(0, lb, qB, sc);
        int nid0 = ids[2 * (P - 1)], nid1 = ids[2 * (P - 1) + 1];
        // Pair pi sits in slot pi % P; the steps are unrolled over the slots, so
        // that every LDS read takes its slot as an immediate offset.  After
        // step pi's barrier the slot of pair pi - 1 is free and takes pair
        // pi + P - 1.  The last pair runs apart: it has no next one.
        const uint32_t nmain = npairs - 1;
        #pragma unroll 1
        for (uint32_t p0 = 0; p0 < nmain; p0 += P) {
            static_for<0, int(P)>([&](auto J) {
                constexpr uint32_t s = decltype(J)::value;
                const uint32_t pi = p0 + s;
                if (pi >= nmain) return;
                asm volatile(".p2align 3");
                if (pi + P - 1 <= npairs) wait_vmcnt_const<(P - 3) * C::PER_PAIR>();   // pair pi + 1 has landed
                else wait_vmcnt((npairs - pi - 2) * C::PER_PAIR);
                block_barrier();
                if (pi + P - 1 < npairs)
                    dma_pair_pages<D>(kv, uint32_t(max(uniform(nid0), 0)), uint32_t(max(uniform(nid1), 0)), src, ring_lds,
                                      (s + P - 1) % P, wave);
                nid0 = ids[2 * (pi + P)];
                nid1 = ids[2 * (pi + P) + 1];
                const int j = int(2 * pi);
                if (__builtin_expect(j < seen0 || j + 2 > seen1, 0))
                    mask_pair<D, RT>(sc, ring + s * SLOT, a, k, ids, j0, n, j, p, lane);
                window_step<D, F16, true>(s * SLOT, ((s + 1) % P) * SLOT, lb, qB, sc, rm, L, O, f, finv);
            });
        }
        mask_pair<D, RT>(sc, ring + (nmain % P) * SLOT, a, k, ids, j0, n, int(2 * nmain), p, lane);
        window_step<D, F16, false>((nmain % P) * SLOT, 0, lb, qB, sc, rm, L, O, f, finv);
    }
    #pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if ((rt * kWaves + wave) * kTileRows + c >= k.nrows) continue;
        const uint64_t at = uint64_t(k.seq.row0) + token[rt];
        const float sum = L[rt][0];
        if (b.parts > 1) {
            const uint64_t slot = state_slot<D != 64>(a, b, int(kRingRows), (rt * kWaves + wave) * kTileRows + c, at, head[rt]);
            #pragma unroll
            for (int e = 0; e < D / 16; ++e) *reinterpret_cast<f4*>(a.ws_o + slot * D + 16 * e + 4 * g) = O[rt][e];
            if (g == 0) *reinterpret_cast<f2*>(a.ws_ml + slot * 2) = f2{rm.m[rt], sum};
            continue;
        }
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        uint8_t* o = a.out + at * a.out_stride + uint64_t(head[rt]) * D * 2;
        #pragma unroll
        for (int e = 0; e < D / 16; ++e) {
            const f4 v = O[rt][e] * inv;
            *reinterpret_cast<u32x2*>(o + 2 * (16 * e + 4 * g)) = u32x2{pack2(v[0], v[1], F16), pack2(v[2], v[3], F16)};
        }
    }
}

template <int D>
hipError_t launch_ring_d(const WindowArgs& a, uint32_t q_dtype, hipStream_t s) {
    const uint64_t blocks = wide_workgroups(a, kRingShift);
    if (blocks > 0x7FFFFFFFull) return hipErrorInvalidValue;
    const dim3 grid{uint32_t(blocks)}, block(256);
    if (q_dtype == DH_DTYPE_BF16)
        hipLaunchKernelGGL((window_ring_kernel<D, false>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((window_ring_kernel<D, true>), grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace

int launch_window_ring(const WindowArgs& a, uint32_t q_dtype, uint32_t d, void* stream) {
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    switch (d) {
        case 64: return launch_ring_d<64>(a, q_dtype, s);
        case 128: return launch_ring_d<128>(a, q_dtype, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace dh
