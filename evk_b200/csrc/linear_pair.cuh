// linear_pair.cuh — the paired-SM kernel behind the large products of
// linear.cu: persistent, one cluster of two CTAs on neighbouring SMs per
// 256 x 2 NB tile of accumulators at a time (NB = 128, or 64 where that
// fills the SM pairs better).
//
// CTA rank r of the pair loads A rows [m0 + 128 r, +128) and NB rows (or
// columns) of B; rank 0 issues tcgen05.mma.cta_group::2 (M 256, N 2 NB, K 16)
// on both CTAs' operands, and each CTA's TMEM receives its 128 rows.  In a
// gated product rank 0 loads the gate columns [n0, +NB) and rank 1 the up
// columns [F + n0, +NB), so each CTA ends with both halves of NB hidden
// units of its rows, and the pair needs no exchange.
//
// Roles (320 threads per CTA): warp 0 TMA producer, warp 1 MMA issue (rank
// 0) into one of two accumulators, so that an epilogue overlaps the next
// tile's MMAs, and warps 2-9 epilogue.  Each epilogue warp works alone on 32
// rows x 32 columns at a time (its TMEM lane quarter, alternate chunks with
// the other warp of that quarter) through two or four 2 KB boxes of its own:
// inputs (residual, saved pre-activations) arrive and outputs leave by TMA in
// the 64-byte swizzle, inputs one chunk ahead where the boxes allow, and only
// warp barriers order them.
// Groups of four warps sharing boxes behind named barriers were no faster, and
// a warp that gave up waiting would have left the others in the barrier.
// No load is multicast.  All waits are bounded.
#pragma once

#include "linear.cuh"
#include "sm100.cuh"

namespace evkcu {
namespace pairk {

using namespace sm100;

constexpr int ROWS = 128;  // rows of A per CTA
constexpr int BK = 64;     // one 128-byte swizzle row of K
constexpr int BOX_BYTES = 32 * 64;  // 32 rows x 32 columns
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 320;
constexpr uint32_t kTimeout = 0x602;

// A stage holds SUB blocks of 64 of K behind one barrier.  The round of the
// MMA warp (wait, issue, commit) takes about 430 clocks, more than the 256 of
// a block's MMAs at NB = 64, hence two blocks a stage there (512 at NB = 128).
// The ring has to cover the 1,500 to 2,000 clocks from a stage's release to
// the next use of it: 160 KB hold that at NB = 128, 192 KB at NB = 64.
template <int NB>
struct Cfg {
    static constexpr int SUB = NB == 128 ? 1 : 2;
    static constexpr int A_SUB = ROWS * BK * 2, B_SUB = NB * BK * 2;
    static constexpr int A_BYTES = SUB * A_SUB, B_BYTES = SUB * B_SUB;
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGES = NB == 128 ? 5 : 4;
    static constexpr int WARP_BOXES = NB == 128 ? 4 : 2;
    static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * WARP_BOXES * BOX_BYTES + 1024 + 512;
    static_assert(SMEM + 64 <= 232448, "shared memory above the per-CTA limit");
};

struct Maps {
    CUtensorMap a, b, in0, in1, out0, out1;
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

// The epilogues of linear.cuh on staged boxes, 32 columns of a lane's row at a
// time: box 0 (and 1) of a set hold the inputs, are replaced in place and
// stored as out0 (and out1).  boxes(): boxes a chunk needs, 1 or 2; inputs():
// how many of them are loaded first.  A third output goes straight to memory,
// 64 bytes of a row per lane.
template <typename T>
__device__ __forceinline__ Vec8 pack_at(const float (&f)[32], int g) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = f[g * 8 + e];
    return pack8<T>(t);
}
template <typename T>
__device__ __forceinline__ void add_at(float (&f)[32], int g, const Vec8& v) {
    float t[8];
    unpack8<T>(v, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[g * 8 + e] += t[e];
}

template <typename T>
struct StagedLinear {
    static constexpr bool kGated = false;
    const T* bias;
    uint32_t N;
    int act, has_res, has_pre;
    __device__ __forceinline__ int inputs() const { return has_res ? 1 : 0; }
    __device__ __forceinline__ int boxes() const { return has_pre ? 2 : 1; }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t, bool, uint32_t col, float (&f)[32],
                                          float (&)[32]) const {
        if (bias) {
            Vec8 b[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) b[g] = ld_vec8(bias + min(col + 8 * g, N - 8));  // past N: not stored
#pragma unroll
            for (int g = 0; g < 4; ++g) add_at<T>(f, g, b[g]);
        }
        if (has_pre) {
#pragma unroll
            for (int g = 0; g < 4; ++g) st_shared_vec8(box_at(set + BOX_BYTES, r, g), pack_at<T>(f, g));
        }
        act_all(f, act);
        if (has_res) {
#pragma unroll
            for (int g = 0; g < 4; ++g) add_at<T>(f, g, ld_shared_vec8(box_at(set, r, g)));
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) st_shared_vec8(box_at(set, r, g), pack_at<T>(f, g));
    }
};

// boxes: h alone, or g and u with h stored directly
template <typename T>
struct StagedGated {
    static constexpr bool kGated = true;
    T* h;
    uint32_t F;
    int act, has_pre;
    __device__ __forceinline__ int inputs() const { return 0; }
    __device__ __forceinline__ int boxes() const { return has_pre ? 2 : 1; }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t row, bool row_ok, uint32_t col,
                                          float (&f)[32], float (&u)[32]) const {
        if (has_pre) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                st_shared_vec8(box_at(set, r, g), pack_at<T>(f, g));
                st_shared_vec8(box_at(set + BOX_BYTES, r, g), pack_at<T>(u, g));
            }
        }
        act_all(f, act);
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] *= u[e];
        if (!has_pre) {
#pragma unroll
            for (int g = 0; g < 4; ++g) st_shared_vec8(box_at(set, r, g), pack_at<T>(f, g));
        } else if (row_ok) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (col + 8 * g < F) st_vec8(h + (uint64_t)row * F + col + 8 * g, pack_at<T>(f, g));
        }
    }
};

// boxes: g -> dg and u -> du; h stored directly
template <typename T>
struct StagedGatedBwd {
    static constexpr bool kGated = false;
    T* h;
    uint32_t F;
    int act;
    __device__ __forceinline__ int inputs() const { return 2; }
    __device__ __forceinline__ int boxes() const { return 2; }
    template <int ACT>
    __device__ __forceinline__ void apply_of(uint8_t* set, uint32_t r, uint32_t row, bool row_ok, uint32_t col,
                                             const float (&f)[32]) const {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            Vec8 *pg = box_at(set, r, c), *pu = box_at(set + BOX_BYTES, r, c);
            float dh[8], g[8], u[8], dg[8], du[8], hh[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) dh[e] = f[c * 8 + e];
            unpack8<T>(ld_shared_vec8(pg), g);
            unpack8<T>(ld_shared_vec8(pu), u);
            gated_bwd8_of<ACT>(dh, g, u, dg, du, hh);
            st_shared_vec8(pg, pack8<T>(dg));
            st_shared_vec8(pu, pack8<T>(du));
            if (h && row_ok && col + 8 * c < F) st_vec8(h + (uint64_t)row * F + col + 8 * c, pack8<T>(hh));
        }
    }
    __device__ __forceinline__ void apply(uint8_t* set, uint32_t r, uint32_t row, bool row_ok, uint32_t col,
                                          float (&f)[32], float (&)[32]) const {
        if (act == EVKCU_ACT_SILU) apply_of<EVKCU_ACT_SILU>(set, r, row, row_ok, col, f);
        else if (act == EVKCU_ACT_GELU) apply_of<EVKCU_ACT_GELU>(set, r, row, row_ok, col, f);
        else if (act == EVKCU_ACT_RELU) apply_of<EVKCU_ACT_RELU>(set, r, row, row_ok, col, f);
        else apply_of<EVKCU_ACT_NONE>(set, r, row, row_ok, col, f);
    }
};

template <typename T, int NB, bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    pair_kernel(const __grid_constant__ Maps maps, const Epi epi, uint32_t M, uint32_t N, uint32_t K, uint32_t idesc,
                int trigger, unsigned int* err) {
    using C = Cfg<NB>;
    constexpr int STAGES = C::STAGES, SUB = C::SUB, WARP_BOXES = C::WARP_BOXES;
    constexpr uint32_t COLS = Epi::kGated ? NB : 2 * NB;  // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * C::A_BYTES;
    uint8_t* boxes = smem + STAGES * C::STAGE_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(boxes + EPI_WARPS * WARP_BOXES * BOX_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;  // [2] accumulator complete
    uint64_t* tempty = tfull + 2;      // [2] accumulator read by both CTAs (rank 0's: 16 arrivals)
    uint64_t* inbar = tempty + 2;      // [warp][set] input boxes loaded
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(inbar + EPI_WARPS * WARP_BOXES);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const uint32_t rank = cluster_ctarank(), pair = cluster_id_x(), npairs = cluster_count_x();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t mt = (M + 255) / 256, nt = (N + COLS - 1) / COLS, total = mt * nt;
    const uint32_t num_kb = (K + SUB * BK - 1) / (SUB * BK);  // a block past K is zeros

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 16);
        }
        for (int b = 0; b < EPI_WARPS * WARP_BOXES; ++b) mbar_init(&inbar[b], 1);
        *s_abort = 0;
        fence_barrier_init();
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.b);
        prefetch_tmap(&maps.out0);
    }
    if (warp == 1) {
        tmem_alloc_pair(s_tmem, 4 * NB);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_relaxed();  // both CTAs' barriers exist before any remote arrive or load
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    uint32_t issued = 0;  // stages requested (thread 0)
    pdl_wait();  // the prologue above may overlap the kernel before
    if (trigger && threadIdx.x == 0) pdl_trigger();

    // Producer and MMA warps run their loops with all lanes and elect one for
    // the asynchronous instructions only: with a single lane in the loop its
    // addresses and descriptors are no longer warp-uniform, and issuing a
    // k-block took 610 clocks against the 512 of its MMAs (NB = 128).
    if (warp == 0) {
        const bool leader = elect_one();
        const uint32_t fb0 = map_shared_rank(full, 0);
        bool ok = true;
        int s = 0;
        uint32_t ph = 1;
        for (uint32_t t = pair; ok && t < total; t += npairs) {
            const Tile tl = tile_at(t, mt, nt, COLS);
            const int am = (int)(tl.m0 + ROWS * rank), bn = (int)(tl.n0 + (Epi::kGated ? N : NB) * rank);
            for (uint32_t kb = 0; kb < num_kb; ++kb, ++issued) {
                if (!mbar_wait(&empty[s], ph, s_abort, err, kTimeout)) {
                    ok = false;
                    break;
                }
                const uint32_t fb = fb0 + (uint32_t)s * 8;
                if (leader) {
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE_BYTES);
#pragma unroll
                    for (int h = 0; h < SUB; ++h) {
                        const int k0 = (int)((kb * SUB + h) * BK);
                        uint8_t *a = sA + s * C::A_BYTES + h * C::A_SUB, *b = sB + s * C::B_BYTES + h * C::B_SUB;
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
                            if (NB == 128) tma_load_3d_pair(b + 8192, &maps.b, fb, bn + 64, k0, 0);
                        }
                    }
                }
                if (++s == STAGES) s = 0, ph ^= 1;
            }
        }
        // The last releases of the slots have arrived before the CTA leaves.
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; ok && i < issued; ++i)
            ok = mbar_wait(&empty[i % STAGES], (i / STAGES) & 1, s_abort, err, kTimeout);
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            uint32_t j = 0, ph = 0;
            int s = 0;
            bool ok = true;
            for (uint32_t t = pair; ok && t < total; t += npairs, ++j) {
                const uint32_t buf = j & 1;
                if (!mbar_wait(&tempty[buf], ((j >> 1) & 1) ^ 1, s_abort, err, kTimeout)) break;
                tc_fence_after();
                const uint32_t d = tmem + buf * 2 * NB;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(&full[s], ph, s_abort, err, kTimeout)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(sA + s * C::A_BYTES), b = smem_u32(sB + s * C::B_BYTES);
                    const uint64_t ad = A_MN ? make_sw128_desc(a, 8192, 1024) : make_sw128_desc(a, 16, 1024);
                    const uint64_t bd = B_MN ? make_sw128_desc(b, 8192, 1024) : make_sw128_desc(b, 16, 1024);
                    if (leader) {
                        // the next 16 of K: 2048 bytes on (MN-major) or 32, in units of 16
#pragma unroll
                        for (int k = 0; k < SUB * BK / 16; ++k)
                            mma_f16_ss_pair(d, ad + (k / 4) * (C::A_SUB >> 4) + (A_MN ? 128 : 2) * (k % 4),
                                            bd + (k / 4) * (C::B_SUB >> 4) + (B_MN ? 128 : 2) * (k % 4), idesc,
                                            (kb | k) != 0);
                        mma_commit_pair_mask(&empty[s], 3);  // the slot is free in both CTAs
                    }
                    if (++s == STAGES) s = 0, ph ^= 1;
                }
                if (ok && leader) mma_commit_pair_mask(&tfull[buf], 3);
            }
        }
    } else {
        const uint32_t ew = (uint32_t)(warp - 2), grp = ew >> 2;
        const uint32_t q = (uint32_t)(warp & 3);  // TMEM lane quarter: rows 32 q + lane of the CTA's 128
        uint8_t* wbox = boxes + ew * WARP_BOXES * BOX_BYTES;
        uint64_t* wbar = inbar + ew * WARP_BOXES;
        const int nin = epi.inputs(), nbox = epi.boxes();
        const uint32_t sets = nbox == 1 ? WARP_BOXES : WARP_BOXES / 2;
        constexpr uint32_t CHUNKS = COLS / 64;  // of this warp per tile
        uint32_t j = 0, n = 0;                  // tiles, chunks
        bool live = true;
        for (uint32_t t = pair; live && t < total; t += npairs, ++j) {
            const Tile tl = tile_at(t, mt, nt, COLS);
            const uint32_t buf = j & 1, row0 = tl.m0 + ROWS * rank + 32 * q, row = row0 + lane;
            // Requests the inputs of chunk i of this tile, the warp's k-th,
            // once the stores that last used its set have been read: all but
            // the sets - 2 groups committed since (with one set: all).
            auto request = [&](uint32_t i, uint32_t k) {
                if (lane != 0) return;
                if (WARP_BOXES == 4 && sets == 4) tma_store_wait_read<2>();
                else tma_store_wait_read<0>();
                if (nin) {
                    uint8_t* set = wbox + (k % sets) * (uint32_t)nbox * BOX_BYTES;
                    uint64_t* bar = wbar + k % sets;
                    const int col = (int)(tl.n0 + 32 * (2 * i + grp));
                    mbar_arrive_expect_tx(bar, (uint32_t)(nin * BOX_BYTES));
                    tma_load_3d(set, &maps.in0, bar, col, (int)row0, 0);
                    if (nin == 2) tma_load_3d(set + BOX_BYTES, &maps.in1, bar, col, (int)row0, 0);
                }
            };
            request(0, n);
            int got = 0;
            if (lane == 0) got = (int)mbar_wait(&tfull[buf], (j >> 1) & 1, s_abort, err, kTimeout);
            live = __shfl_sync(0xffffffffu, got, 0) != 0;
            __syncwarp();  // a shuffle orders no memory: what lane 0 waited for, the others may read after this
            if (!live) {
                if (nin && lane == 0) mbar_drain(wbar + n % sets, (n / sets) & 1);
                break;
            }
            tc_fence_after();
#pragma unroll 1
            for (uint32_t i = 0; i < CHUNKS; ++i, ++n) {
                const uint32_t c = 2 * i + grp, col0 = tl.n0 + 32 * c;
                uint8_t* set = wbox + (n % sets) * (uint32_t)nbox * BOX_BYTES;
                uint32_t r0[32], r1[32];
                const uint32_t ta = tmem + ((q * 32) << 16) + buf * 2 * NB + c * 32;
                tmem_ld32(ta, r0);
                if (Epi::kGated) tmem_ld32(ta + NB, r1);
                if (sets == 1) {
                    if (i > 0) request(i, n);
                } else if (i + 1 < CHUNKS) {
                    request(i + 1, n + 1);  // one chunk ahead
                }
                tmem_wait_ld();
                if (i + 1 == CHUNKS) {  // the warp's part of the accumulator is in registers
                    tc_fence_before();
                    __syncwarp();
                    // Only arrivals that a later tile waits for: rank 0 may leave before any other lands.
                    if (lane == 0 && t + 2 * npairs < total) mbar_arrive_relaxed(map_shared_rank(&tempty[buf], 0));
                }
                if (nin) {
                    got = 0;
                    if (lane == 0) got = (int)mbar_wait(wbar + n % sets, (n / sets) & 1, s_abort, err, kTimeout);
                    live = __shfl_sync(0xffffffffu, got, 0) != 0;
                    __syncwarp();  // lane 0 has seen the inputs arrive and the set's other box free
                    if (!live) {
                        if (lane == 0) {
                            mbar_drain(wbar + n % sets, (n / sets) & 1);
                            if (sets > 1 && i + 1 < CHUNKS)
                                mbar_drain(wbar + (n + 1) % sets, ((n + 1) / sets) & 1);
                        }
                        break;
                    }
                } else {
                    __syncwarp();  // lane 0 has seen the set free
                }
                float f[32], u[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    f[e] = __uint_as_float(r0[e]);
                    u[e] = Epi::kGated ? __uint_as_float(r1[e]) : 0.0f;
                }
                epi.apply(set, lane, row, row < M, col0, f, u);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < M && col0 < N) {
                        tma_store_3d(&maps.out0, set, (int)col0, (int)row0, 0);
                        if (nbox == 2) tma_store_3d(&maps.out1, set + BOX_BYTES, (int)col0, (int)row0, 0);
                    }
                    tma_store_commit();
                }
            }
        }
        if (lane == 0) tma_store_wait_all();  // written, not only read, before the CTA counts as done
        tc_fence_before();
    }
    __syncthreads();
    // A wait gave up: the copies in flight land before either CTA leaves.
    if (*s_abort && rank == 0 && threadIdx.x == 0)
        for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
            mbar_drain(&full[i % STAGES], (i / STAGES) & 1);
    cluster_sync_relaxed();  // no CTA leaves while its pair may still touch its memory
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 4 * NB);
    }
}

}  // namespace pairk
}  // namespace evkcu
