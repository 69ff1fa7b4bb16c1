// linear.cu — matrix products with fused epilogues: evkcu_linear
// (bias, activation, residual) and evkcu_gated_ffn (both input projections,
// the activation and the product in one kernel), forward and backward.
//
//   y = act(x W + bias) + residual            [rows, N], x [rows, K]
//     dz = dy act'(z);  dx = dz W^T;  dW = x^T dz;  dbias = sum_rows dz
//   h = act(x Wg) (x Wu);  y = h Wd + residual
//     dh = dy Wd^T (kept in fp32);  dpre = [dh u act'(g) | dh act(g)]
//     dx = dpre [Wg | Wu]^T;  d[Wg | Wu] = x^T dpre;  dWd = h^T dy
//
// Every product runs on tcgen05 with fp32 accumulators and an epilogue of
// linear.cuh.  Transposed operands are MN-major descriptors, never copies.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <string>

#include "linear.cuh"
#include "linear_pair.cuh"
#include "sm100.cuh"

namespace evkcu {
namespace {

using namespace sm100;

constexpr int BM = 128;
constexpr int BK = 64;
constexpr uint32_t kTimeoutTile = 0x601;

// ------------------------------------------------- 128 x BN tile kernel ----
// One CTA per 128 x BN output tile.  Warp 0 feeds 64-deep k-blocks by TMA
// into a ring, warp 1 issues tcgen05.mma into a 128 x BN accumulator; warps
// 2-5 then copy the accumulator to the (now idle) ring as fp32 and all warps
// run the epilogue on eight consecutive columns at a time, so every global
// access of the epilogue is a 16-byte one next to its neighbour lane's.
// B arrives in boxes of 64 of its rows (or columns): a gated tile takes its
// first box from the gate half of the weight and its second from the up
// half, so accumulator columns c and c + 64 belong to the same hidden unit.
template <int BN>
struct TileCfg {
    static constexpr int A_BYTES = BM * BK * 2;
    static constexpr int B_BYTES = BN * BK * 2;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int LD = BN + 4;  // floats per staged row (16-byte rows on different banks)
    static constexpr int SMEM = STAGES * STAGE + 1024 /*align*/ + 256 /*barriers*/;
    static_assert(STAGES * STAGE >= BM * LD * 4, "the staged accumulator must fit in the ring");
};
constexpr int kTileThreads = 192;

template <typename T, int BN, bool A_MN, bool B_MN, class Epi>
__global__ void __launch_bounds__(kTileThreads, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, Epi epi, uint32_t M,
                uint32_t N, uint32_t K, uint32_t up_off, uint32_t idesc, unsigned int* err) {
    using Cfg = TileCfg<BN>;
    constexpr int STAGES = Cfg::STAGES;
    constexpr uint32_t COLS = Epi::kGated ? BN / 2 : BN;  // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* accum = empty + STAGES;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(accum + 1);
    volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t n0 = blockIdx.x * COLS, m0 = blockIdx.y * BM;
    const uint32_t num_kb = (K + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(accum, 1);
        *s_abort = 0;
        fence_barrier_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
    }
    if (warp == 1) {
        tmem_alloc(s_tmem, BN);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;

    uint32_t issued = 0;  // k-blocks requested (thread 0)
    if (warp == 0) {
        if (lane == 0) {
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                const int s = (int)(kb % STAGES);
                if (!mbar_wait(&empty[s], ((kb / STAGES) & 1) ^ 1, s_abort, err, kTimeoutTile)) break;
                mbar_arrive_expect_tx(&full[s], Cfg::STAGE);
                const int k0 = (int)(kb * BK);
                uint8_t* a = sA + s * Cfg::A_BYTES;
                uint8_t* b = sB + s * Cfg::B_BYTES;
                if (!A_MN) {
                    tma_load_3d(a, &tmA, &full[s], k0, (int)m0, 0);
                } else {
                    tma_load_3d(a, &tmA, &full[s], (int)m0, k0, 0);
                    tma_load_3d(a + 8192, &tmA, &full[s], (int)m0 + 64, k0, 0);
                }
#pragma unroll
                for (int j = 0; j < BN / 64; ++j) {
                    const int nb = Epi::kGated ? (int)(n0 + (uint32_t)j * up_off) : (int)n0 + 64 * j;
                    if (!B_MN) tma_load_3d(b + j * 8192, &tmB, &full[s], k0, nb, 0);
                    else tma_load_3d(b + j * 8192, &tmB, &full[s], nb, k0, 0);
                }
                issued = kb + 1;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                const int s = (int)(kb % STAGES);
                if (!mbar_wait(&full[s], (kb / STAGES) & 1, s_abort, err, kTimeoutTile)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a = smem_u32(sA + s * Cfg::A_BYTES);
                const uint32_t b = smem_u32(sB + s * Cfg::B_BYTES);
#pragma unroll
                for (int k = 0; k < BK / 16; ++k) {
                    const uint64_t ad =
                        A_MN ? make_sw128_desc(a + k * 2048, 8192, 1024) : make_sw128_desc(a + k * 32, 16, 1024);
                    const uint64_t bd =
                        B_MN ? make_sw128_desc(b + k * 2048, 8192, 1024) : make_sw128_desc(b + k * 32, 16, 1024);
                    mma_f16_ss(tmem, ad, bd, idesc, (kb | k) != 0);
                }
                mma_commit(&empty[s]);
            }
            if (ok) mma_commit(accum);
        }
    }
    float* stage = reinterpret_cast<float*>(smem);
    if (warp >= 2) {
        const int q = warp & 3;  // TMEM lane quarter of this warp
        const bool ok = __shfl_sync(0xffffffffu,
                                    lane == 0 ? (int)mbar_wait_sleep(accum, 0, s_abort, err, kTimeoutTile) : 0,
                                    0) != 0;
        tc_fence_after();
        if (ok) {
            float* row = stage + (q * 32 + lane) * Cfg::LD;
#pragma unroll 1
            for (int c = 0; c < BN / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c * 32, r);
                tmem_wait_ld();
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    *reinterpret_cast<uint4*>(row + c * 32 + g * 4) =
                        make_uint4(r[4 * g], r[4 * g + 1], r[4 * g + 2], r[4 * g + 3]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, BN);
    }
    if (*s_abort) {
        // A wait gave up: the copies in flight land before the CTA leaves.
        if (threadIdx.x == 0)
            for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
                mbar_drain(&full[i % STAGES], (i / STAGES) & 1);
        return;
    }
    for (uint32_t v = threadIdx.x; v < BM * (COLS / 8); v += kTileThreads) {
        const uint32_t r = v / (COLS / 8), c = (v % (COLS / 8)) * 8;
        if (m0 + r >= M || n0 + c >= N) continue;
        float f[8], g[8];
        const float* src = stage + r * Cfg::LD + c;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = src[e];
        if (Epi::kGated) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = src[64 + e];
        }
        epi(m0 + r, n0 + c, f, g);
    }
}

// A product C[M, N] = A[M, K] . B[K, N] with an epilogue.  a_mn: A is stored
// [K, M]; b_mn: B is stored [K, nb] (else [nb, K]), of which a gated product
// reads columns n and n + N for its output column n (nb = 2 N).
struct Product {
    const void *A, *B;
    uint32_t M, N, K, nb;
    bool b_mn;
    int dtype;
    cudaStream_t st;
};

// Sets a kernel's shared-memory limit once per device.
template <class K>
int allow_smem(K* kern, int bytes, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (state()->device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return EVKCU_OK;
    EVKCU_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return EVKCU_OK;
}

// Operand maps; box_b: rows of a box of B stored [nb, K].
template <bool A_MN, bool B_MN>
int operand_maps(const Product& p, CUtensorMap* ta, CUtensorMap* tb, uint32_t box_b) {
    EVKCU_TRY(A_MN ? make_tmap_3d(ta, p.A, p.M, p.K, 1, p.M, (uint64_t)p.M * p.K, 64, BK, p.dtype)
                   : make_tmap_3d(ta, p.A, p.K, p.M, 1, p.K, (uint64_t)p.M * p.K, BK, BM, p.dtype));
    return B_MN ? make_tmap_3d(tb, p.B, p.nb, p.K, 1, p.nb, (uint64_t)p.nb * p.K, 64, BK, p.dtype)
                : make_tmap_3d(tb, p.B, p.K, p.nb, 1, p.K, (uint64_t)p.nb * p.K, BK, box_b, p.dtype);
}

template <typename T, int BN, bool A_MN, bool B_MN, class Epi>
int launch_tile(const Product& p, const Epi& epi) {
    using Cfg = TileCfg<BN>;
    CUtensorMap ta, tb;
    EVKCU_TRY((operand_maps<A_MN, B_MN>(p, &ta, &tb, 64)));
    auto kern = tile_kernel<T, BN, A_MN, B_MN, Epi>;
    static std::atomic<uint64_t> done{0};
    EVKCU_TRY(allow_smem(kern, Cfg::SMEM, done));
    constexpr uint32_t COLS = Epi::kGated ? BN / 2 : BN;
    const dim3 grid((p.N + COLS - 1) / COLS, (p.M + BM - 1) / BM);
    const uint32_t idesc = make_idesc_f16(BM, BN, p.dtype == EVKCU_BF16 ? 1 : 0, A_MN, B_MN);
    kern<<<grid, kTileThreads, Cfg::SMEM, p.st>>>(ta, tb, epi, p.M, p.N, p.K, p.N, idesc, state()->d_error);
    return after_launch("evkcu_linear(tile)");
}

// The staged form of each epilogue: its boxes' maps (128 rows x 32 columns of
// a [M, N] matrix with rows of `pitch` elements) and parameters.
int box_map(CUtensorMap* m, const void* p, const Product& pr, uint64_t pitch) {
    return make_tmap_3d(m, p, pr.N, pr.M, 1, pitch, pitch * pr.M, 32, 128, pr.dtype, 64);
}
template <typename T>
int stage(const Product& p, const EpiLinear<T>& e, pairk::Maps& m, pairk::StagedLinear<T>& s) {
    s = pairk::StagedLinear<T>{e.bias, e.N, e.act, e.res != nullptr, e.pre != nullptr};
    if (e.res) EVKCU_TRY(box_map(&m.in0, e.res, p, p.N));
    if (e.pre) EVKCU_TRY(box_map(&m.out1, e.pre, p, p.N));
    return box_map(&m.out0, e.y, p, p.N);
}
template <typename T>
int stage(const Product& p, const EpiGated<T>& e, pairk::Maps& m, pairk::StagedGated<T>& s) {
    s = pairk::StagedGated<T>{e.act, e.pre != nullptr};
    if (e.pre) {
        EVKCU_TRY(box_map(&m.out1, e.pre, p, 2 * (uint64_t)p.N));
        EVKCU_TRY(box_map(&m.out2, e.pre + p.N, p, 2 * (uint64_t)p.N));
    }
    return box_map(&m.out0, e.h, p, p.N);
}
template <typename T>
int stage(const Product& p, const EpiGatedBwd<T>& e, pairk::Maps& m, pairk::StagedGatedBwd<T>& s) {
    s = pairk::StagedGatedBwd<T>{e.act, e.h != nullptr};
    const uint64_t pitch = 2 * (uint64_t)p.N;
    EVKCU_TRY(box_map(&m.in0, e.pre, p, pitch));
    EVKCU_TRY(box_map(&m.in1, e.pre + p.N, p, pitch));
    EVKCU_TRY(box_map(&m.out0, e.dpre, p, pitch));
    EVKCU_TRY(box_map(&m.out1, e.dpre + p.N, p, pitch));
    return e.h ? box_map(&m.out2, e.h, p, p.N) : (int)EVKCU_OK;
}
template <class Epi> struct StagedOf;
template <typename T> struct StagedOf<EpiLinear<T>> { using type = pairk::StagedLinear<T>; };
template <typename T> struct StagedOf<EpiGated<T>> { using type = pairk::StagedGated<T>; };
template <typename T> struct StagedOf<EpiGatedBwd<T>> { using type = pairk::StagedGatedBwd<T>; };

template <typename T, bool A_MN, bool B_MN, class Epi>
int launch_pair(const Product& p, const Epi& epi) {
    using S = typename StagedOf<Epi>::type;
    DeviceState* ds = state();
    auto kern = pairk::pair_kernel<T, A_MN, B_MN, S>;
    static std::atomic<uint64_t> done{0};
    EVKCU_TRY(allow_smem(kern, pairk::SMEM, done));
    if (!ds->linear_clusters) {  // equal for every instantiation: one CTA per SM
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (ds->sm_count / 2));
        cfg.blockDim = dim3(pairk::THREADS);
        cfg.dynamicSmemBytes = pairk::SMEM;
        int n = 0;
        EVKCU_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        ds->linear_clusters = std::max(n, 1);
    }
    pairk::Maps maps;
    memset(&maps, 0, sizeof(maps));
    S s;
    EVKCU_TRY((operand_maps<A_MN, B_MN>(p, &maps.a, &maps.b, 128)));
    EVKCU_TRY(stage(p, epi, maps, s));
    constexpr uint64_t COLS = Epi::kGated ? 128 : 256;
    const uint64_t tiles = ((uint64_t)p.M + 255) / 256 * ((p.N + COLS - 1) / COLS);
    EVKCU_CHECK_ARG(tiles <= 0xFFFFFFFFu / 2, EVKCU_BAD_SHAPE, "evkcu_linear: too many output tiles");
    const uint32_t grid = 2 * (uint32_t)std::min<uint64_t>(tiles, (uint64_t)ds->linear_clusters);
    const uint32_t idesc = make_idesc_f16(256, 256, p.dtype == EVKCU_BF16 ? 1 : 0, A_MN, B_MN);
    kern<<<grid, pairk::THREADS, pairk::SMEM, p.st>>>(maps, s, p.M, p.N, p.K, idesc, ds->d_error);
    return after_launch("evkcu_linear(pair)");
}

template <typename T, bool A_MN, bool B_MN, class Epi>
int launch_product(const Product& p, const Epi& epi) {
    constexpr uint64_t COLS = Epi::kGated ? 128 : 256;
    const uint64_t pair_tiles = ((uint64_t)p.M + 255) / 256 * ((p.N + COLS - 1) / COLS);
    if (pair_tiles >= 40) return launch_pair<T, A_MN, B_MN>(p, epi);
    return launch_tile<T, 128, A_MN, B_MN>(p, epi);
}

// A transposed A (weight gradients) always comes with a B stored [K, nb].
template <typename T, bool A_MN, class Epi>
int product(const Product& p, const Epi& epi) {
    if constexpr (!A_MN) {
        if (!p.b_mn) return launch_product<T, false, false>(p, epi);
    }
    return launch_product<T, A_MN, true>(p, epi);
}

// -------------------------------- dz = dy act'(z) and its column sums ----
// A cluster of 8 CTAs owns 64 columns; each CTA takes an eighth of the rows,
// eight columns per thread, and keeps the column sums in registers.  They
// are added across the CTA's 32 row lanes in shared memory, then across the
// cluster in rank order over distributed shared memory: a fixed order and no
// scratch in global memory.
constexpr uint32_t kDactCluster = 8;
constexpr int kDactThreads = 256;

template <typename T>
__global__ void __cluster_dims__(1, kDactCluster, 1) __launch_bounds__(kDactThreads)
    dact_kernel(const T* dy, const T* pre, T* dz, T* dbias, uint32_t rows, uint32_t N, int act, int acc) {
    __shared__ float s_sum[32][64];
    __shared__ float s_col[64];
    const uint32_t cl = threadIdx.x & 7, rl = threadIdx.x >> 3;
    const uint32_t col = blockIdx.x * 64 + cl * 8;
    const uint32_t per = (rows + kDactCluster - 1) / kDactCluster;
    const uint32_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    float sum[8] = {};
    if (col < N) {
#pragma unroll 4
        for (uint32_t r = r0 + rl; r < r1; r += 32) {
            const uint64_t at = (uint64_t)r * N + col;
            float f[8];
            unpack8<T>(ld_vec8(dy + at), f);
            if (act != EVKCU_ACT_NONE) {
                float z[8];
                unpack8<T>(ld_vec8(pre + at), z);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float a, da;
                    act_both(z[e], act, a, da);
                    f[e] *= da;
                }
                st_vec8(dz + at, pack8<T>(f));
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += f[e];
        }
    }
    if (!dbias) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s_sum[rl][cl * 8 + e] = sum[e];
    __syncthreads();
    if (threadIdx.x < 64) {
        float t = 0.0f;
        for (int i = 0; i < 32; ++i) t += s_sum[i][threadIdx.x];
        s_col[threadIdx.x] = t;
    }
    cluster_sync_all();
    const uint32_t c = blockIdx.x * 64 + threadIdx.x;
    if (blockIdx.y == 0 && threadIdx.x < 64 && c < N) {
        float t = acc ? Elem<T>::to_f(dbias[c]) : 0.0f;
        float part = 0.0f;
        for (uint32_t r = 0; r < kDactCluster; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_shared_rank(&s_col[threadIdx.x], r)));
            part += v;
        }
        dbias[c] = Elem<T>::from_f(t + part);
    }
    cluster_sync_all();  // no CTA leaves while rank 0 still reads its sums
}

template <typename T>
int launch_dact(const void* dy, const void* pre, void* dz, void* dbias, uint32_t rows, uint32_t N, int act, int acc,
                cudaStream_t st) {
    dact_kernel<T><<<dim3((N + 63) / 64, kDactCluster), kDactThreads, 0, st>>>((const T*)dy, (const T*)pre, (T*)dz,
                                                                              (T*)dbias, rows, N, act, acc);
    return after_launch("evkcu_linear_backward(dact)");
}

// ---------------------------------------------------------------- checks ----
constexpr uint32_t kMaxDim = 1u << 30;  // TMA coordinates are signed 32-bit

int check_common(const char* op, uint32_t rows, uint32_t a, uint32_t b, int act, uint32_t flags, uint32_t allowed,
                 int dtype) {
    const std::string o(op);
    EVKCU_CHECK_ARG(dtype == EVKCU_F16 || dtype == EVKCU_BF16, EVKCU_BAD_ARG, o + ": unknown dtype");
    EVKCU_CHECK_ARG(act >= EVKCU_ACT_NONE && act <= EVKCU_ACT_SILU, EVKCU_BAD_ARG, o + ": unknown activation");
    EVKCU_CHECK_ARG((flags & ~allowed) == 0, EVKCU_BAD_ARG, o + ": unknown flag");
    EVKCU_CHECK_ARG(a > 0 && b > 0 && a % 8 == 0 && b % 8 == 0, EVKCU_BAD_SHAPE,
                    o + ": feature sizes must be positive multiples of 8");
    EVKCU_CHECK_ARG(rows <= kMaxDim && a <= kMaxDim && b <= kMaxDim, EVKCU_BAD_SHAPE, o + ": size above 2^30");
    return EVKCU_OK;
}

Span in_span(const char* name, const void* p, uint64_t rows, uint64_t cols) { return Span{name, p, rows, cols, cols}; }
Span out_span(const char* name, const void* p, uint64_t rows, uint64_t cols, const char* same = nullptr,
              const char* same2 = nullptr) {
    return Span{name, p, rows, cols, cols, true, same, same2};
}

// y = x W, the plain linear with an optional accumulate (residual = y).
template <typename T>
EpiLinear<T> epi_plain(void* y, uint32_t N, bool acc) {
    return EpiLinear<T>{nullptr, acc ? (const T*)y : nullptr, (T*)y, nullptr, N, EVKCU_ACT_NONE};
}

// dx[rows, K] (+)= dz[rows, N] . W^T, W [K, N] (or [N, K] when nk).
template <typename T>
int grad_input(const void* dz, const void* w, void* dx, uint32_t rows, uint32_t K, uint32_t N, bool nk, bool acc,
               int dtype, cudaStream_t st) {
    return product<T, false>(Product{dz, w, rows, K, N, K, nk, dtype, st}, epi_plain<T>(dx, K, acc));
}
// dW[K, N] (+)= x^T dz (or its transpose [N, K] = dz^T x when nk).
template <typename T>
int grad_weight(const void* x, const void* dz, void* dw, uint32_t rows, uint32_t K, uint32_t N, bool nk, bool acc,
                int dtype, cudaStream_t st) {
    if (nk) return product<T, true>(Product{dz, x, N, K, rows, K, true, dtype, st}, epi_plain<T>(dw, K, acc));
    return product<T, true>(Product{x, dz, K, N, rows, N, true, dtype, st}, epi_plain<T>(dw, N, acc));
}

int zero_grad(void* p, uint64_t elems, bool acc, cudaStream_t st) {
    if (!p || acc) return EVKCU_OK;
    EVKCU_CUDA_TRY(cudaMemsetAsync(p, 0, elems * 2, st));
    return EVKCU_OK;
}

}  // namespace
}  // namespace evkcu

using namespace evkcu;

extern "C" int evkcu_linear(const void* x, const void* w, const void* bias, const void* residual, void* y, void* pre,
                            uint32_t rows, uint32_t K, uint32_t N, int act, uint32_t flags, int dtype, void* stream) {
    const char* op = "evkcu_linear";
    EVKCU_TRY(check_common(op, rows, K, N, act, flags, EVKCU_MM_TRANSPOSE_B, dtype));
    if (rows == 0) return EVKCU_OK;
    EVKCU_TRY(check_ptr(op, "x", x, true));
    EVKCU_TRY(check_ptr(op, "w", w, true));
    EVKCU_TRY(check_ptr(op, "y", y, true));
    EVKCU_TRY(check_ptr(op, "bias", bias, false));
    EVKCU_TRY(check_ptr(op, "residual", residual, false));
    EVKCU_TRY(check_ptr(op, "pre", pre, false));
    EVKCU_TRY(check_spans(op, {in_span("x", x, rows, K), in_span("w", w, K, N), in_span("bias", bias, 1, N),
                               in_span("residual", residual, rows, N), out_span("y", y, rows, N, "residual"),
                               out_span("pre", pre, rows, N)}));
    EVKCU_CHECK_ARG(state(), EVKCU_CUDA_ERROR, "evkcu_linear: no device state");
    const bool nk = flags & EVKCU_MM_TRANSPOSE_B;
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        return product<T, false>(Product{x, w, rows, N, K, N, !nk, dtype, as_stream(stream)},
                                 EpiLinear<T>{(const T*)bias, (const T*)residual, (T*)y, (T*)pre, N, act});
    });
}

extern "C" int evkcu_linear_backward(const void* x, const void* w, const void* pre, const void* dy, void* dpre,
                                     void* dx, void* dw, void* dbias, uint32_t rows, uint32_t K, uint32_t N, int act,
                                     uint32_t flags, int dtype, void* stream) {
    const char* op = "evkcu_linear_backward";
    EVKCU_TRY(check_common(op, rows, K, N, act, flags, EVKCU_MM_TRANSPOSE_B | EVKCU_MM_ACC_C, dtype));
    const bool nk = flags & EVKCU_MM_TRANSPOSE_B, acc = flags & EVKCU_MM_ACC_C;
    cudaStream_t st = as_stream(stream);
    const bool has_act = act != EVKCU_ACT_NONE;
    EVKCU_TRY(check_ptr(op, "dy", dy, rows > 0));
    EVKCU_TRY(check_ptr(op, "x", x, rows > 0 && dw));
    EVKCU_TRY(check_ptr(op, "w", w, rows > 0 && dx));
    EVKCU_TRY(check_ptr(op, "pre", pre, rows > 0 && has_act));
    EVKCU_TRY(check_ptr(op, "dpre", dpre, rows > 0 && has_act));
    EVKCU_TRY(check_ptr(op, "dx", dx, false));
    EVKCU_TRY(check_ptr(op, "dw", dw, false));
    EVKCU_TRY(check_ptr(op, "dbias", dbias, false));
    if (rows == 0) {  // empty sums
        EVKCU_TRY(zero_grad(dw, (uint64_t)K * N, acc, st));
        return zero_grad(dbias, N, acc, st);
    }
    EVKCU_TRY(check_spans(op, {in_span("x", x, rows, K), in_span("w", w, K, N), in_span("pre", pre, rows, N),
                               in_span("dy", dy, rows, N),
                               out_span("dpre", has_act ? dpre : nullptr, rows, N, "pre", "dy"),
                               out_span("dx", dx, rows, K), out_span("dw", dw, K, N), out_span("dbias", dbias, 1, N)}));
    EVKCU_CHECK_ARG(state(), EVKCU_CUDA_ERROR, "evkcu_linear_backward: no device state");
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        if (has_act || dbias) EVKCU_TRY(launch_dact<T>(dy, pre, dpre, dbias, rows, N, act, acc, st));
        const void* dz = has_act ? dpre : dy;
        if (dx) EVKCU_TRY(grad_input<T>(dz, w, dx, rows, K, N, nk, acc, dtype, st));
        if (dw) EVKCU_TRY(grad_weight<T>(x, dz, dw, rows, K, N, nk, acc, dtype, st));
        return (int)EVKCU_OK;
    });
}

extern "C" int evkcu_gated_ffn(const void* x, const void* w_in, const void* w_out, const void* residual, void* y,
                               void* hidden, void* pre, uint32_t rows, uint32_t D, uint32_t F, int act,
                               uint32_t flags, int dtype, void* stream) {
    const char* op = "evkcu_gated_ffn";
    EVKCU_TRY(check_common(op, rows, D, F, act, flags, EVKCU_MM_TRANSPOSE_B, dtype));
    EVKCU_CHECK_ARG(F <= kMaxDim / 2, EVKCU_BAD_SHAPE, "evkcu_gated_ffn: hidden size above 2^29");
    if (rows == 0) return EVKCU_OK;
    EVKCU_TRY(check_ptr(op, "x", x, true));
    EVKCU_TRY(check_ptr(op, "w_in", w_in, true));
    EVKCU_TRY(check_ptr(op, "w_out", w_out, y != nullptr));
    EVKCU_TRY(check_ptr(op, "hidden", hidden, true));
    EVKCU_TRY(check_ptr(op, "y", y, false));
    EVKCU_TRY(check_ptr(op, "residual", residual, false));
    EVKCU_TRY(check_ptr(op, "pre", pre, false));
    EVKCU_TRY(check_spans(op, {in_span("x", x, rows, D), in_span("w_in", w_in, D, 2 * (uint64_t)F),
                               in_span("w_out", w_out, F, D), in_span("residual", residual, rows, D),
                               out_span("y", y, rows, D, "residual"), out_span("hidden", hidden, rows, F),
                               out_span("pre", pre, rows, 2 * (uint64_t)F)}));
    EVKCU_CHECK_ARG(state(), EVKCU_CUDA_ERROR, "evkcu_gated_ffn: no device state");
    const bool nk = flags & EVKCU_MM_TRANSPOSE_B;
    cudaStream_t st = as_stream(stream);
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        EVKCU_TRY((product<T, false>(Product{x, w_in, rows, F, D, 2 * F, !nk, dtype, st},
                                     EpiGated<T>{(T*)hidden, (T*)pre, F, act})));
        if (!y) return (int)EVKCU_OK;
        return product<T, false>(Product{hidden, w_out, rows, D, F, D, !nk, dtype, st},
                                 EpiLinear<T>{nullptr, (const T*)residual, (T*)y, nullptr, D, EVKCU_ACT_NONE});
    });
}

extern "C" int evkcu_gated_ffn_backward(const void* x, const void* w_in, const void* w_out, const void* pre,
                                        const void* dy, void* dpre, void* hidden, void* dx, void* dw_in,
                                        void* dw_out, uint32_t rows, uint32_t D, uint32_t F, int act, uint32_t flags,
                                        int dtype, void* stream) {
    const char* op = "evkcu_gated_ffn_backward";
    EVKCU_TRY(check_common(op, rows, D, F, act, flags, EVKCU_MM_TRANSPOSE_B | EVKCU_MM_ACC_C, dtype));
    EVKCU_CHECK_ARG(F <= kMaxDim / 2, EVKCU_BAD_SHAPE, "evkcu_gated_ffn_backward: hidden size above 2^29");
    const bool nk = flags & EVKCU_MM_TRANSPOSE_B, acc = flags & EVKCU_MM_ACC_C, some = rows > 0;
    cudaStream_t st = as_stream(stream);
    EVKCU_TRY(check_ptr(op, "x", x, some && dw_in));
    EVKCU_TRY(check_ptr(op, "w_in", w_in, some && dx));
    EVKCU_TRY(check_ptr(op, "w_out", w_out, some));
    EVKCU_TRY(check_ptr(op, "pre", pre, some));
    EVKCU_TRY(check_ptr(op, "dy", dy, some));
    EVKCU_TRY(check_ptr(op, "dpre", dpre, some));
    EVKCU_TRY(check_ptr(op, "hidden", hidden, some && dw_out));
    EVKCU_TRY(check_ptr(op, "dx", dx, false));
    EVKCU_TRY(check_ptr(op, "dw_in", dw_in, false));
    EVKCU_TRY(check_ptr(op, "dw_out", dw_out, false));
    if (rows == 0) {  // empty sums
        EVKCU_TRY(zero_grad(dw_in, 2 * (uint64_t)D * F, acc, st));
        return zero_grad(dw_out, (uint64_t)D * F, acc, st);
    }
    EVKCU_TRY(check_spans(op, {in_span("x", x, rows, D), in_span("w_in", w_in, D, 2 * (uint64_t)F),
                               in_span("w_out", w_out, F, D), in_span("pre", pre, rows, 2 * (uint64_t)F),
                               in_span("dy", dy, rows, D), out_span("dpre", dpre, rows, 2 * (uint64_t)F, "pre"),
                               out_span("hidden", dw_out ? hidden : nullptr, rows, F), out_span("dx", dx, rows, D),
                               out_span("dw_in", dw_in, D, 2 * (uint64_t)F), out_span("dw_out", dw_out, F, D)}));
    EVKCU_CHECK_ARG(state(), EVKCU_CUDA_ERROR, "evkcu_gated_ffn_backward: no device state");
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        EVKCU_TRY((product<T, false>(Product{dy, w_out, rows, F, D, F, nk, dtype, st},
                                     EpiGatedBwd<T>{(const T*)pre, (T*)dpre, dw_out ? (T*)hidden : nullptr, F, act})));
        if (dx) EVKCU_TRY(grad_input<T>(dpre, w_in, dx, rows, D, 2 * F, nk, acc, dtype, st));
        if (dw_in) EVKCU_TRY(grad_weight<T>(x, dpre, dw_in, rows, D, 2 * F, nk, acc, dtype, st));
        if (dw_out) EVKCU_TRY(grad_weight<T>(hidden, dy, dw_out, rows, F, D, nk, acc, dtype, st));
        return (int)EVKCU_OK;
    });
}
