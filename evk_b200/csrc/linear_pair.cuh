// linear_pair.cuh — the paired-SM kernel behind the large products of
// linear.cu: persistent, one cluster of two CTAs on neighbouring SMs per
// 256 x 256 tile of accumulators at a time.
//
// CTA rank r of the pair loads A rows [m0 + 128 r, +128) and 128 rows (or
// columns) of B; rank 0 issues tcgen05.mma.cta_group::2 (M 256, N 256, K 16)
// on both CTAs' operands, and each CTA's TMEM receives its 128 rows.  In a
// gated product rank 0 loads the gate columns [n0, +128) and rank 1 the up
// columns [F + n0, +128), so each CTA ends with both halves of 128 hidden
// units of its rows, and the pair needs no exchange.
//
// Roles (320 threads per CTA): warp 0 TMA producer, warp 1 MMA issue (rank
// 0) into one of two 256-column accumulators, warps 2-9 epilogue: two groups
// of four warps take alternate 32-column chunks, so one group's TMA traffic
// (residual or saved pre-activations in, up to three outputs out, 128 x 32
// boxes in the 64-byte swizzle) overlaps the other's arithmetic, and both
// overlap the next tile's MMAs.  One group alone would need longer than a
// mainloop of K = 512.  No load is multicast.  All waits are bounded.
#pragma once

#include "linear.cuh"
#include "sm100.cuh"

namespace evkcu {
namespace pairk {

using namespace sm100;

constexpr int ROWS = 128;  // rows of A and of B per CTA
constexpr int BK = 64;
constexpr int OP_BYTES = ROWS * BK * 2;
constexpr int STAGE_BYTES = 2 * OP_BYTES;
constexpr int STAGES = 5;
constexpr int BOX_BYTES = ROWS * 64;  // 128 rows x 32 columns
constexpr int GROUP_BOXES = 4;
constexpr int SMEM = STAGES * STAGE_BYTES + 2 * GROUP_BOXES * BOX_BYTES + 1024 + 256;
constexpr int THREADS = 320;
constexpr uint32_t kTimeout = 0x602;
static_assert(SMEM + 64 <= 232448, "shared memory above the per-CTA limit");

struct Maps {
    CUtensorMap a, b, in0, in1, out0, out1, out2;
};

struct Tile {
    uint32_t m0, n0;
};
// Groups of 8 row tiles, row tile fastest: the pairs in flight share a few B
// column tiles and one group's A rows in L2.
__device__ __forceinline__ Tile tile_at(uint32_t t, uint32_t mt, uint32_t nt, uint32_t cols) {
    constexpr uint32_t G = 8;
    const uint32_t per_group = G * nt, first = t / per_group * G, in = t % per_group;
    const uint32_t gm = min(G, mt - first);
    return Tile{(first + in % gm) * 256, in / gm * cols};
}

// 16-byte chunk c (of 4) of row r in a box of 64-byte rows, 64-byte swizzle.
__device__ __forceinline__ Vec8* box_at(uint8_t* box, uint32_t r, uint32_t c) {
    return reinterpret_cast<Vec8*>(box + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// The epilogues of linear.cuh on staged boxes.  kIn / kOut: boxes loaded and
// stored per chunk; inputs lie in boxes 0 and 1 and are replaced in place.
template <typename T>
struct StagedLinear {
    static constexpr bool kGated = false;
    static constexpr int kBoxes = 2;
    const T* bias;
    uint32_t N;
    int act, has_res, has_pre;
    __device__ __forceinline__ int inputs() const { return has_res ? 1 : 0; }
    __device__ __forceinline__ bool stores(int i) const { return i == 0 || (i == 1 && has_pre); }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t c, uint32_t col, float (&f)[8],
                                          float (&)[8]) const {
        float t[8];
        if (bias && col < N) {
            unpack8<T>(ld_vec8(bias + col), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += t[e];
        }
        if (has_pre) st_shared_vec8(box_at(set + BOX_BYTES, r, c), pack8<T>(f));
        act8(f, act);
        Vec8* p = box_at(set, r, c);
        if (has_res) {
            unpack8<T>(ld_shared_vec8(p), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += t[e];
        }
        st_shared_vec8(p, pack8<T>(f));
    }
};

template <typename T>
struct StagedGated {
    static constexpr bool kGated = true;
    static constexpr int kBoxes = 3;
    int act, has_pre;
    __device__ __forceinline__ int inputs() const { return 0; }
    __device__ __forceinline__ bool stores(int i) const { return i == 0 || has_pre; }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t c, uint32_t, float (&g)[8],
                                          float (&u)[8]) const {
        if (has_pre) {
            st_shared_vec8(box_at(set + BOX_BYTES, r, c), pack8<T>(g));
            st_shared_vec8(box_at(set + 2 * BOX_BYTES, r, c), pack8<T>(u));
        }
        act8(g, act);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= u[e];
        st_shared_vec8(box_at(set, r, c), pack8<T>(g));
    }
};

template <typename T>
struct StagedGatedBwd {
    static constexpr bool kGated = false;
    static constexpr int kBoxes = 3;
    int act, has_h;
    __device__ __forceinline__ int inputs() const { return 2; }
    __device__ __forceinline__ bool stores(int i) const { return i < 2 || has_h; }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t c, uint32_t, float (&dh)[8],
                                          float (&)[8]) const {
        Vec8 *pg = box_at(set, r, c), *pu = box_at(set + BOX_BYTES, r, c);
        float g[8], u[8], dg[8], du[8], h[8];
        unpack8<T>(ld_shared_vec8(pg), g);
        unpack8<T>(ld_shared_vec8(pu), u);
        gated_bwd8(dh, g, u, dg, du, h, act);
        st_shared_vec8(pg, pack8<T>(dg));
        st_shared_vec8(pu, pack8<T>(du));
        if (has_h) st_shared_vec8(box_at(set + 2 * BOX_BYTES, r, c), pack8<T>(h));
    }
};

template <typename T, bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    pair_kernel(const __grid_constant__ Maps maps, const Epi epi, uint32_t M, uint32_t N, uint32_t K, uint32_t idesc,
                unsigned int* err) {
    constexpr uint32_t COLS = Epi::kGated ? 128 : 256;  // output columns of a tile
    constexpr uint32_t SETS = Epi::kBoxes <= GROUP_BOXES / 2 ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * OP_BYTES;
    uint8_t* boxes = smem + STAGES * STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(boxes + 2 * GROUP_BOXES * BOX_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;  // [2] accumulator complete
    uint64_t* tempty = tfull + 2;      // [2] accumulator read by both CTAs (rank 0's: 16 arrivals)
    uint64_t* inbar = tempty + 2;      // [2 groups][2 sets] input boxes loaded
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(inbar + 4);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const uint32_t rank = cluster_ctarank(), pair = cluster_id_x(), npairs = cluster_count_x();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t mt = (M + 255) / 256, nt = (N + COLS - 1) / COLS, total = mt * nt;
    const uint32_t num_kb = (K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 16);
            mbar_init(&inbar[2 * b], 1);
            mbar_init(&inbar[2 * b + 1], 1);
        }
        *s_abort = 0;
        fence_barrier_init();
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        prefetch_tmap(&maps.out0);
    }
    if (warp == 1) {
        tmem_alloc_pair(s_tmem, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // both CTAs' barriers exist before any remote arrive or load
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    uint32_t issued = 0;  // stages requested (thread 0)

    if (warp == 0) {
        if (lane == 0) {
            bool ok = true;
            for (uint32_t t = pair; ok && t < total; t += npairs) {
                const Tile tl = tile_at(t, mt, nt, COLS);
                const int am = (int)(tl.m0 + ROWS * rank), bn = (int)(tl.n0 + (Epi::kGated ? N : ROWS) * rank);
                for (uint32_t kb = 0; kb < num_kb; ++kb, ++issued) {
                    const int s = (int)(issued % STAGES);
                    if (!mbar_wait_cluster(&empty[s], ((issued / STAGES) & 1) ^ 1, s_abort, err, kTimeout)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * STAGE_BYTES);
                    const uint32_t fb = map_shared_rank(&full[s], 0);
                    const int k0 = (int)(kb * BK);
                    uint8_t *a = sA + s * OP_BYTES, *b = sB + s * OP_BYTES;
                    if (!A_MN) {
                        tma_load_3d_pair(a, &maps.a, fb, k0, am, 0);
                    } else {
                        tma_load_3d_pair(a, &maps.a, fb, am, k0, 0);
                        tma_load_3d_pair(a + 8192, &maps.a, fb, am + 64, k0, 0);
                    }
                    if (!B_MN) {
                        tma_load_3d_pair(b, &maps.b, fb, k0, bn, 0);
                    } else {
                        tma_load_3d_pair(b, &maps.b, fb, bn, k0, 0);
                        tma_load_3d_pair(b + 8192, &maps.b, fb, bn + 64, k0, 0);
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && lane == 0) {
            uint32_t it = 0, j = 0;
            bool ok = true;
            for (uint32_t t = pair; ok && t < total; t += npairs, ++j) {
                const uint32_t buf = j & 1;
                if (!mbar_wait_cluster(&tempty[buf], ((j >> 1) & 1) ^ 1, s_abort, err, kTimeout)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * 256;
                for (uint32_t kb = 0; kb < num_kb; ++kb, ++it) {
                    const int s = (int)(it % STAGES);
                    if (!mbar_wait(&full[s], (it / STAGES) & 1, s_abort, err, kTimeout)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(sA + s * OP_BYTES), b = smem_u32(sB + s * OP_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) {
                        const uint64_t ad =
                            A_MN ? make_sw128_desc(a + k * 2048, 8192, 1024) : make_sw128_desc(a + k * 32, 16, 1024);
                        const uint64_t bd =
                            B_MN ? make_sw128_desc(b + k * 2048, 8192, 1024) : make_sw128_desc(b + k * 32, 16, 1024);
                        mma_f16_ss_pair(d, ad, bd, idesc, (kb | k) != 0);
                    }
                    mma_commit_pair_mask(&empty[s], 3);  // the slot is free in both CTAs
                }
                if (ok) mma_commit_pair_mask(&tfull[buf], 3);
            }
        }
    } else {
        const uint32_t grp = (uint32_t)(warp - 2) >> 2;
        const int q = warp & 3;             // TMEM lane quarter of this warp
        const uint32_t rr = q * 32 + lane;  // row within the CTA's 128
        const bool leader = warp == 2 + 4 * (int)grp && lane == 0;
        uint8_t* gbox = boxes + grp * GROUP_BOXES * BOX_BYTES;
        uint64_t* gbar = inbar + 2 * grp;
        const int nin = epi.inputs();
        uint32_t j = 0, nchunk = 0;
        // After a wait that gave up the group runs on without waiting or
        // storing, so that its named barriers keep meeting all four warps.
        bool live = true;
        for (uint32_t t = pair; t < total; t += npairs, ++j) {
            const Tile tl = tile_at(t, mt, nt, COLS);
            const uint32_t buf = j & 1, row0 = tl.m0 + ROWS * rank;
            // Requests the inputs of the group's i-th chunk of this tile,
            // once the set's previous stores have been read.
            auto request = [&](uint32_t i, uint32_t n) {
                if (!leader || !live) return;
                tma_store_wait_read<SETS - 1>();
                if (nin) {
                    uint8_t* set = gbox + (n % SETS) * (GROUP_BOXES / SETS) * BOX_BYTES;
                    uint64_t* bar = gbar + n % SETS;
                    const int col = (int)(tl.n0 + 32 * (2 * i + grp));
                    mbar_arrive_expect_tx(bar, (uint32_t)(nin * BOX_BYTES));
                    tma_load_3d(set, &maps.in0, bar, col, (int)row0, 0);
                    if (nin == 2) tma_load_3d(set + BOX_BYTES, &maps.in1, bar, col, (int)row0, 0);
                }
            };
            request(0, nchunk);
            int got = 0;
            if (lane == 0 && live) got = (int)mbar_wait_cluster(&tfull[buf], (j >> 1) & 1, s_abort, err, kTimeout);
            const bool was = live;
            live = __shfl_sync(0xffffffffu, got, 0) != 0;
            if (was && !live && leader && nin) mbar_drain(gbar + nchunk % SETS, (nchunk / SETS) & 1);
            tc_fence_after();
#pragma unroll 1
            for (uint32_t i = 0; i < COLS / 64; ++i, ++nchunk) {
                const uint32_t c = 2 * i + grp, col0 = tl.n0 + 32 * c;
                uint8_t* set = gbox + (nchunk % SETS) * (GROUP_BOXES / SETS) * BOX_BYTES;
                uint32_t r0[32], r1[32];
                const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16) + buf * 256 + c * 32;
                tmem_ld32(ta, r0);
                if (Epi::kGated) tmem_ld32(ta + 128, r1);
                if (i > 0) request(i, nchunk);
                tmem_wait_ld();
                if (i == COLS / 64 - 1) {  // the group's part of the accumulator is in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (rank == 0) mbar_arrive(&tempty[buf]);
                        else mbar_arrive_remote(map_shared_rank(&tempty[buf], 0));
                    }
                }
                if (nin) {
                    got = 0;
                    if (lane == 0 && live)
                        got = (int)mbar_wait(gbar + nchunk % SETS, (nchunk / SETS) & 1, s_abort, err, kTimeout);
                    const bool before = live;
                    live = __shfl_sync(0xffffffffu, got, 0) != 0;
                    if (before && !live && leader) mbar_drain(gbar + nchunk % SETS, (nchunk / SETS) & 1);
                } else {
                    named_barrier(1 + grp, 128);  // the leader has seen the set free
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float f[8], u[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        f[e] = __uint_as_float(r0[g * 8 + e]);
                        u[e] = Epi::kGated ? __uint_as_float(r1[g * 8 + e]) : 0.0f;
                    }
                    epi.apply(set, rr, g, col0 + 8 * g, f, u);
                }
                fence_proxy_async_smem();
                named_barrier(1 + grp, 128);
                if (leader && live) {
                    if (row0 < M && col0 < N) {
                        if (epi.stores(0)) tma_store_3d(&maps.out0, set, (int)col0, (int)row0, 0);
                        if (epi.stores(1)) tma_store_3d(&maps.out1, set + BOX_BYTES, (int)col0, (int)row0, 0);
                        if (Epi::kBoxes > 2 && epi.stores(2))
                            tma_store_3d(&maps.out2, set + 2 * BOX_BYTES, (int)col0, (int)row0, 0);
                    }
                    tma_store_commit();
                }
            }
        }
        if (leader) tma_store_wait_all();
        tc_fence_before();
    }
    __syncthreads();
    // A wait gave up: the copies in flight land before either CTA leaves.
    if (*s_abort && rank == 0 && threadIdx.x == 0)
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
            mbar_drain(&full[i % STAGES], (i / STAGES) & 1);
    cluster_sync_all();  // no CTA leaves while its pair may still touch its memory
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

}  // namespace pairk
}  // namespace evkcu
