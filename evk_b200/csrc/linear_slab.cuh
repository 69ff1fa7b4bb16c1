// linear_slab.cuh — the kernel behind the products of linear.cu that are too
// small to fill the SM pairs: decode steps, short prompts, weight gradients
// of narrow layers.
//
// The tile is transposed: accumulator rows (TMEM lanes) are 128 columns of
// the output, accumulator columns are MR of its rows, D[n, m] = sum_k W[k, n]
// x[m, k].  With one row of x the weight is then the MMA's 128-row operand
// and nothing is multiplied by padding but 16 columns; the bound is reading
// W.  K is split over the CTAs of a cluster, so that a few column slabs still
// keep every SM loading: each CTA copies its fp32 partial to its (now idle)
// ring, and after a cluster barrier the CTAs share out the output and add the
// partials in rank order over distributed shared memory.  A fixed order, and
// no scratch in global memory that two calls could share.
//
// Warp 0 feeds 64-deep k-blocks by TMA, warp 1 issues tcgen05.mma, warps 2-5
// read the accumulator, and all warps run the epilogue on eight consecutive
// columns at a time.  A gated slab holds 64 gate columns and the 64 up
// columns of the same hidden units.
#pragma once

#include "linear.cuh"
#include "sm100.cuh"

namespace evkcu {
namespace slabk {

using namespace sm100;

constexpr int COLS = 128;
constexpr int BK = 64;
constexpr int W_BYTES = COLS * BK * 2;
constexpr int LD = COLS + 4;  // floats per staged output row
constexpr int THREADS = 192;
constexpr uint32_t kTimeout = 0x601;

// The ring holds about 100 KB (MR = 16, two CTAs per SM) or 190 KB: a block
// takes about 1.5 us from its request to its use, and an SM has to pull
// 44 GB/s to read W at the HBM rate.
template <int MR>
struct Cfg {
    static constexpr int X_BYTES = MR * BK * 2;
    static constexpr int STAGE = W_BYTES + X_BYTES;
    static constexpr int STAGES = MR == 64 ? 8 : 6;
    static constexpr int PER_SM = MR == 16 ? 2 : 1;
    static constexpr int SMEM = STAGES * STAGE + 1024 /*align*/ + 256 /*barriers*/;
    static constexpr int TMEM = MR < 32 ? 32 : MR;
    static_assert(STAGES * STAGE >= MR * LD * 4, "the staged accumulator must fit in the ring");
    static_assert(PER_SM * (SMEM + 1024) <= 228 * 1024, "CTAs per SM");
};

// Four floats at a shared-memory address of any CTA of the cluster.
__device__ __forceinline__ void ld4_cluster(uint32_t addr, float* f) {
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                 : "r"(addr)
                 : "memory");
}

// grid (slabs, row tiles, splits), cluster (1, 1, splits).  early: W blocks
// requested before the earlier kernels are waited for (only where no kernel
// still running may write W).  trigger: the next kernel may start early.
template <typename T, int MR, bool X_MN, bool W_MN, class Epi>
__global__ void __launch_bounds__(THREADS, Cfg<MR>::PER_SM)
    slab_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, Epi epi, uint32_t M,
                uint32_t N, uint32_t K, uint32_t kb_per_cta, uint32_t idesc, int early, int trigger,
                unsigned int* err) {
    using C = Cfg<MR>;
    constexpr int STAGES = C::STAGES;
    constexpr uint32_t OUT = Epi::kGated ? COLS / 2 : COLS;  // output columns of a slab
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sX = smem + STAGES * W_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* accum = empty + STAGES;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(accum + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t n0 = blockIdx.x * OUT, m0 = blockIdx.y * MR, split = blockIdx.z, splits = gridDim.z;
    const uint32_t kb0 = split * kb_per_cta, nkb = min(kb_per_cta, (K + BK - 1) / BK - kb0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(accum, 1);
        *s_abort = 0;
        fence_barrier_init();
        prefetch_tmap(&tmX);
        prefetch_tmap(&tmW);
    }
    if (warp == 1) {
        tmem_alloc(s_tmem, C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    uint32_t issued = 0;  // k-blocks requested (thread 0)

    // All lanes run these loops and one is elected for the asynchronous
    // instructions (see linear_pair.cuh).
    if (warp == 0) {
        const bool leader = elect_one();
        auto load_w = [&](uint32_t i, int s) {
            const int k0 = (int)((kb0 + i) * BK);
            uint8_t* w = sW + s * W_BYTES;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int nb = (int)(n0 + (Epi::kGated ? N : 64u) * (uint32_t)j);
                if (W_MN) tma_load_3d(w + j * 8192, &tmW, &full[s], nb, k0, 0);
                else tma_load_3d(w + j * 8192, &tmW, &full[s], k0, nb, 0);
            }
        };
        auto load_x = [&](uint32_t i, int s) {
            const int k0 = (int)((kb0 + i) * BK);
            uint8_t* x = sX + s * C::X_BYTES;
            if (X_MN) {
#pragma unroll
                for (int j = 0; j < MR / 64; ++j) tma_load_3d(x + j * 8192, &tmX, &full[s], (int)m0 + 64 * j, k0, 0);
            } else {
                tma_load_3d(x, &tmX, &full[s], k0, (int)m0, 0);
            }
        };
        const uint32_t ahead = early ? min(nkb, (uint32_t)STAGES) : 0u;
        for (uint32_t i = 0; i < ahead; ++i)
            if (leader) {
                mbar_arrive_expect_tx(&full[i], C::STAGE);
                load_w(i, (int)i);
            }
        // Only now may dependents start: whatever they request early, the
        // kernels before this one have finished.
        pdl_wait();
        if (trigger) pdl_trigger();
        int s = 0;
        uint32_t ph = 1;
        for (; issued < nkb; ++issued) {
            if (issued >= ahead && !mbar_wait(&empty[s], ph, s_abort, err, kTimeout)) break;
            if (leader) {
                if (issued >= ahead) {
                    mbar_arrive_expect_tx(&full[s], C::STAGE);
                    load_w(issued, s);
                }
                load_x(issued, s);
            }
            if (++s == STAGES) s = 0, ph ^= 1;
        }
        // The last releases of the slots have arrived before the CTA leaves.
        bool ok = issued == nkb;
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; ok && i < issued; ++i)
            ok = mbar_wait(&empty[i % STAGES], (i / STAGES) & 1, s_abort, err, kTimeout);
    } else if (warp == 1) {
        const bool leader = elect_one();
        bool ok = true;
        int s = 0;
        uint32_t ph = 0;
        for (uint32_t i = 0; i < nkb; ++i) {
            if (!mbar_wait(&full[s], ph, s_abort, err, kTimeout)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = smem_u32(sW + s * W_BYTES), b = smem_u32(sX + s * C::X_BYTES);
            const uint64_t ad = W_MN ? make_sw128_desc(a, 8192, 1024) : make_sw128_desc(a, 16, 1024);
            const uint64_t bd = X_MN ? make_sw128_desc(b, 8192, 1024) : make_sw128_desc(b, 16, 1024);
            if (leader) {
                // the next 16 of K: 2048 bytes on (MN-major) or 32, in units of 16
#pragma unroll
                for (int k = 0; k < BK / 16; ++k)
                    mma_f16_ss(tmem, ad + (W_MN ? 128 : 2) * k, bd + (X_MN ? 128 : 2) * k, idesc, (i | k) != 0);
                mma_commit(&empty[s]);
            }
            if (++s == STAGES) s = 0, ph ^= 1;
        }
        if (ok && leader) mma_commit(accum);
    }
    float* stage = reinterpret_cast<float*>(smem);
    if (warp >= 2) {
        const int q = warp & 3;  // TMEM lane quarter: output columns 32 q + lane
        const bool ok = __shfl_sync(0xffffffffu,
                                    lane == 0 ? (int)mbar_wait_sleep(accum, 0, s_abort, err, kTimeout) : 0, 0) != 0;
        __syncwarp();  // a shuffle orders no memory: what lane 0 waited for, the others may read after this
        tc_fence_after();
        if (ok) {
            float* col = stage + q * 32 + lane;
            const uint32_t live = min((uint32_t)MR, M - m0);
#pragma unroll 1
            for (uint32_t c = 0; c < live; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + c, r);
                tmem_wait_ld();
#pragma unroll
                for (int m = 0; m < 16; ++m) col[(c + m) * LD] = __uint_as_float(r[m]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
    // A wait gave up: the copies in flight land before the CTA leaves.
    if (*s_abort && threadIdx.x == 0)
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
            mbar_drain(&full[i % STAGES], (i / STAGES) & 1);
    pdl_wait();  // before the epilogue reads or writes what earlier kernels may
    if (splits > 1) cluster_sync_all();
    // This CTA's share of the tile's rows, summed in place: nobody else reads
    // these rows of its own partial.  A warp reads 512 consecutive bytes of
    // each peer (16 of every 32 took twice as long), eight loads in flight.
    const uint32_t rows = min((uint32_t)MR, M - m0), share = (rows + splits - 1) / splits;
    const uint32_t r0 = split * share, r1 = min(rows, r0 + share);
    if (splits > 1 && !*s_abort) {
        constexpr uint32_t Q = COLS / 4;  // 16-byte pieces of a row
        const uint32_t base = smem_u32(stage), n = r1 > r0 ? (r1 - r0) * Q : 0;
        for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 2 * THREADS) {
            float sum[2][4] = {};
            // without a second piece the first again: any other is being written by its own thread
            const uint32_t i1 = i0 + THREADS < n ? i0 + THREADS : i0;
            const uint32_t at[2] = {base + ((r0 + i0 / Q) * LD + i0 % Q * 4) * 4,
                                    base + ((r0 + i1 / Q) * LD + i1 % Q * 4) * 4};
            for (uint32_t p0 = 0; p0 < splits; p0 += 4) {  // in rank order
                float t[4][2][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (p0 + j >= splits) continue;
#pragma unroll
                    for (int k = 0; k < 2; ++k) ld4_cluster(map_shared_rank_u32(at[k], p0 + j), t[j][k]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (p0 + j >= splits) continue;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum[k][e] += t[j][k][e];
                }
            }
            float* dst = stage + (r0 + i0 / Q) * LD + i0 % Q * 4;
            *reinterpret_cast<float4*>(dst) = make_float4(sum[0][0], sum[0][1], sum[0][2], sum[0][3]);
            if (i0 + THREADS < n) {
                dst = stage + (r0 + i1 / Q) * LD + i1 % Q * 4;
                *reinterpret_cast<float4*>(dst) = make_float4(sum[1][0], sum[1][1], sum[1][2], sum[1][3]);
            }
        }
        __syncthreads();
    }
    if (!*s_abort) {
#pragma unroll 2
        for (uint32_t v = r0 * (OUT / 8) + threadIdx.x; v < r1 * (OUT / 8); v += THREADS) {
            const uint32_t r = v / (OUT / 8), c = (v % (OUT / 8)) * 8;
            const float* src = stage + r * LD + c;
            float f[8], g[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = src[e], g[e] = Epi::kGated ? src[64 + e] : 0.0f;
            if (n0 + c < N) epi(m0 + r, n0 + c, f, g);
        }
    }
    if (splits > 1) cluster_sync_relaxed();  // no CTA leaves while its partial is read
}

}  // namespace slabk
}  // namespace evkcu
