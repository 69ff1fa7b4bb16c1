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
// linear.cuh, in the paired-SM kernel (linear_pair.cuh) or the slab kernel
// (linear_slab.cuh).  Transposed operands are MN-major descriptors, never
// copies.
//
// Rounded to the storage type in between: dz, h and dpre, which are operands of
// the next product, and the tensor cores take no wider ones at this rate (two
// halves of a value would double that product).  The error of a result of theirs
// is about sqrt(2) times that of its own rounding: 2-norm against 64 bits in bf16
// 0.0023 to 0.0024 for y of one token and for the gradients, 0.0017 for one
// rounding.  dh and the sums behind dbias are not rounded.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <string>

#include "linear.cuh"
#include "linear_pair.cuh"
#include "linear_slab.cuh"
#include "sm100.cuh"

namespace evkcu {
namespace {

// A product C[M, N] = A[M, K] . B[K, N] with an epilogue.  a_mn: A is stored
// [K, M]; b_mn: B is stored [K, nb] (else [nb, K]), of which a gated product
// reads columns n and n + N for its output column n (nb = 2 N).  early: B is
// an argument of the call and a kernel of the same call runs just before, so
// B may be read while that one ends (linear_slab.cuh).  trigger: another
// kernel of the same call follows and may start while this one ends; the
// caller's next kernel may not, since it need not expect that.
struct Product {
    const void *A, *B;
    uint32_t M, N, K, nb;
    bool b_mn;
    int dtype;
    cudaStream_t st;
    bool early = false;
    bool trigger = false;
};

// Operand maps; box_a, box_b: rows of a box of A stored [M, K] and of B
// stored [nb, K] (otherwise boxes are 64 columns of a K-row).
constexpr uint32_t BK = 64;
template <bool A_MN, bool B_MN>
int operand_maps(const Product& p, CUtensorMap* ta, CUtensorMap* tb, uint32_t box_a, uint32_t box_b) {
    EVKCU_TRY(A_MN ? make_tmap_3d(ta, p.A, p.M, p.K, 1, p.M, (uint64_t)p.M * p.K, 64, BK, p.dtype)
                   : make_tmap_3d(ta, p.A, p.K, p.M, 1, p.K, (uint64_t)p.M * p.K, BK, box_a, p.dtype));
    return B_MN ? make_tmap_3d(tb, p.B, p.nb, p.K, 1, p.nb, (uint64_t)p.nb * p.K, 64, BK, p.dtype)
                : make_tmap_3d(tb, p.B, p.K, p.nb, 1, p.K, (uint64_t)p.nb * p.K, BK, box_b, p.dtype);
}

// Splits of K for `tiles` slab tiles: one CTA per SM where that is possible
// (16 x 14336 x 4096: 4 splits of 32 slabs 20.9 us, 8 23.8), else as many as
// are resident; two k-blocks each at least.  A cluster of 8 packs badly where
// a CTA takes an SM (64 x 8192 x 2048: 4 splits 13.6 us, 8 22.1).
uint32_t slab_splits(int mr, uint64_t tiles, uint32_t kblocks, int sms) {
    const uint64_t sm = (uint64_t)sms, slots = mr == 16 ? 2 * sm : sm;
    const uint64_t most = mr == 16 ? 8 : 4, fit = tiles <= sm / 2 ? sm / tiles : slots / tiles;
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({most, fit, (kblocks + 1) / 2}));
}

template <typename T, int MR, bool A_MN, bool B_MN, class Epi>
int launch_slab(const Product& p, const Epi& epi) {
    using C = slabk::Cfg<MR>;
    CUtensorMap tx, tw;
    EVKCU_TRY((operand_maps<A_MN, B_MN>(p, &tx, &tw, MR, 64)));
    auto kern = slabk::slab_kernel<T, MR, A_MN, B_MN, Epi>;
    static std::atomic<uint64_t> done{0};
    EVKCU_TRY(allow_smem(kern, C::SMEM, done));
    DeviceState* ds = state();
    const uint32_t out = Epi::kGated ? 64 : 128;
    const uint32_t slabs = (p.N + out - 1) / out, tiles = (p.M + MR - 1) / MR, kblocks = (p.K + BK - 1) / BK;
    EVKCU_CHECK_ARG(tiles <= 65535, EVKCU_BAD_SHAPE, "evkcu_linear: too many output tiles");
    const uint32_t want = slab_splits(MR, (uint64_t)slabs * tiles, kblocks, ds->sm_count);
    const uint32_t per = (kblocks + want - 1) / want;
    const uint32_t splits = (kblocks + per - 1) / per;  // none of them empty
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(slabs, tiles, splits);
    cfg.blockDim = dim3(slabk::THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = p.st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = splits;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ds->pdl ? 2 : 1;
    const uint32_t idesc = sm100::make_idesc_f16(128, MR, p.dtype == EVKCU_BF16 ? 1 : 0, B_MN, A_MN);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, tw, epi, p.M, p.N, p.K, per, idesc,
                                             (int)(p.early && ds->pdl), (int)p.trigger, ds->d_error);
    if (e != cudaSuccess) return cuda_fail(e, "evkcu_linear(slab)");
    return after_launch("evkcu_linear(slab)");
}

// The staged form of each epilogue: its boxes' maps (32 rows x 32 columns of
// a [M, N] matrix with rows of `pitch` elements) and parameters.
int box_map(CUtensorMap* m, const void* p, const Product& pr, uint64_t pitch) {
    return make_tmap_3d(m, p, pr.N, pr.M, 1, pitch, pitch * pr.M, 32, 32, pr.dtype, 64);
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
    s = pairk::StagedGated<T>{e.h, e.F, e.act, e.pre != nullptr};
    if (!e.pre) return box_map(&m.out0, e.h, p, p.N);
    EVKCU_TRY(box_map(&m.out0, e.pre, p, 2 * (uint64_t)p.N));
    return box_map(&m.out1, e.pre + p.N, p, 2 * (uint64_t)p.N);
}
template <typename T>
int stage(const Product& p, const EpiGatedBwd<T>& e, pairk::Maps& m, pairk::StagedGatedBwd<T>& s) {
    s = pairk::StagedGatedBwd<T>{e.h, e.F, e.act};
    const uint64_t pitch = 2 * (uint64_t)p.N;
    EVKCU_TRY(box_map(&m.in0, e.pre, p, pitch));
    EVKCU_TRY(box_map(&m.in1, e.pre + p.N, p, pitch));
    EVKCU_TRY(box_map(&m.out0, e.dpre, p, pitch));
    return box_map(&m.out1, e.dpre + p.N, p, pitch);
}
template <class Epi> struct StagedOf;
template <typename T> struct StagedOf<EpiLinear<T>> { using type = pairk::StagedLinear<T>; };
template <typename T> struct StagedOf<EpiGated<T>> { using type = pairk::StagedGated<T>; };
template <typename T> struct StagedOf<EpiGatedBwd<T>> { using type = pairk::StagedGatedBwd<T>; };

template <typename T, int NB, bool A_MN, bool B_MN, class Epi>
int launch_pair(const Product& p, const Epi& epi) {
    using S = typename StagedOf<Epi>::type;
    using C = pairk::Cfg<NB>;
    DeviceState* ds = state();
    auto kern = pairk::pair_kernel<T, NB, A_MN, B_MN, S>;
    static std::atomic<uint64_t> done{0};
    EVKCU_TRY(allow_smem(kern, C::SMEM, done));
    if (!ds->linear_clusters) {  // equal for every instantiation: one CTA per SM
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (ds->sm_count / 2));
        cfg.blockDim = dim3(pairk::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        int n = 0;
        EVKCU_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
        ds->linear_clusters = std::max(n, 1);
    }
    pairk::Maps maps;
    memset(&maps, 0, sizeof(maps));
    S s;
    EVKCU_TRY((operand_maps<A_MN, B_MN>(p, &maps.a, &maps.b, 128, NB)));
    EVKCU_TRY(stage(p, epi, maps, s));
    constexpr uint64_t COLS = Epi::kGated ? NB : 2 * NB;
    const uint64_t tiles = ((uint64_t)p.M + 255) / 256 * ((p.N + COLS - 1) / COLS);
    EVKCU_CHECK_ARG(tiles <= 0xFFFFFFFFu / 2, EVKCU_BAD_SHAPE, "evkcu_linear: too many output tiles");
    const uint32_t grid = 2 * (uint32_t)std::min<uint64_t>(tiles, (uint64_t)ds->linear_clusters);
    const uint32_t idesc = sm100::make_idesc_f16(256, 2 * NB, p.dtype == EVKCU_BF16 ? 1 : 0, A_MN, B_MN);
    return launch_pdl("evkcu_linear(pair)", kern, dim3(grid), dim3(pairk::THREADS), C::SMEM, p.st, maps, s, p.M, p.N,
                      p.K, idesc, (int)p.trigger, ds->d_error);
}

// Which kernel a product takes: the least estimated time.  The estimates are
// a start-and-finish cost plus rounds of tiles times k-blocks, in us (a slab CTA
// works on one tile, so each of its rounds starts and finishes), fitted to
// graph-replayed runs of bf16 products with operands from HBM:
//   M x K x N            pair 128   pair 64   slab 128 / 64   taken
//   4096 x 2048 x 8192     90.4      104.3         -          pair 128
//   2048 x 2048 x 2048     15.7       16.8       26.4         pair 128
//   1024 x 2048 x 2048     15.2       11.1       13.8         pair 64
//    333 x  512 x 1368      7.6        5.8        7.2         pair 64
//    512 x 8192 x 2048     41.8       27.6       23.9         slab 128
//     32 x 4096 x 14336    26.1       30.4       20.3         slab 64
//    512 x 16384 x 512     76.9       47.4       22.2         slab 64
//   2048 x   64 x 8192     13.2       14.3       35.0         pair 128
// Up to 16 rows W is read once and multiplied by little: always the slab.
template <typename T, bool A_MN, bool B_MN, class Epi>
int launch_product(const Product& p, const Epi& epi) {
    const int sms = state()->sm_count;
    const uint32_t per = Epi::kGated ? 2 : 1;  // accumulator columns per output column
    const double kb = (p.K + BK - 1) / BK;
    auto tiles = [&](uint64_t rows, uint64_t cols) {
        return (p.M + rows - 1) / rows * ((p.N * (uint64_t)per + cols - 1) / cols);
    };
    auto pair_us = [&](uint64_t cols, double start, double block, double least) {
        return start + (double)((tiles(256, cols) + sms / 2 - 1) / (sms / 2)) * std::max(block * kb, least);
    };
    auto slab_us = [&](int mr) {
        const uint64_t t = tiles(mr, 128);
        const uint32_t s = slab_splits(mr, t, (uint32_t)kb, sms);
        return (s > 1 ? 2.0 : 0.0) + (double)((t * s + sms - 1) / sms) * (4.6 + 0.27 * std::ceil(kb / s));
    };
    if constexpr (!A_MN) {
        if (p.M <= 16) return launch_slab<T, 16, A_MN, B_MN>(p, epi);
    }
    const double wide = pair_us(256, 5.0, 0.285, 1.8), narrow = pair_us(128, 4.4, 0.18, 1.2);
    const double s64 = slab_us(64), s128 = slab_us(128);
    if (std::min(wide, narrow) <= std::min(s64, s128))
        return wide <= narrow ? launch_pair<T, 128, A_MN, B_MN>(p, epi) : launch_pair<T, 64, A_MN, B_MN>(p, epi);
    return s64 <= s128 ? launch_slab<T, 64, A_MN, B_MN>(p, epi) : launch_slab<T, 128, A_MN, B_MN>(p, epi);
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
// A cluster of 8 CTAs owns 8 L columns; each CTA takes an eighth of the rows,
// L lanes of eight columns a row, U rows of a lane in flight, and keeps the
// column sums in registers.  They are added across the CTA's row lanes in
// shared memory, then across the cluster in rank order over distributed shared
// memory: a fixed order and no scratch in global memory.  dz may be dy or pre:
// every element is read before it is written, by the same thread.  The
// activation is a template parameter: chosen inside, the one-row form held to 32
// registers spilled 16 to 44 bytes (4096 x 8192 SILU: 41.8 us against 37.7).
constexpr uint32_t kDactCluster = 8;
constexpr int kDactThreads = 256;

template <typename T, int L, int U, int ACT>
__global__ void __cluster_dims__(1, kDactCluster, 1) __launch_bounds__(kDactThreads, U == 1 ? 8 : 3)
    dact_kernel(const T* dy, const T* pre, T* dz, T* dbias, uint32_t rows, uint32_t N, int acc, int trigger) {
    constexpr uint32_t RL = kDactThreads / L;  // row lanes
    __shared__ float s_sum[RL][8 * L + 1];
    __shared__ float s_col[8 * L];
    const uint32_t cl = threadIdx.x % L, rl = threadIdx.x / L;
    const uint32_t col = blockIdx.x * (8 * L) + cl * 8;
    const uint32_t per = (rows + kDactCluster - 1) / kDactCluster;
    const uint32_t r0 = blockIdx.y * per, r1 = min(rows, r0 + per);
    float sum[8] = {};
    pdl_wait();
    if (trigger) pdl_trigger();  // the product that follows; it waits for dz
    if (col < N) {
        for (uint32_t r = r0 + rl; r < r1; r += U * RL) {
            Vec8 a[U], z[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // past the end its first row again: others may be writing theirs (dz may be dy or pre)
                const uint32_t row = U == 1 || r + u * RL < r1 ? r + u * RL : r;
                const uint64_t at = (uint64_t)row * N + col;
                a[u] = ld_vec8(dy + at);
                if (ACT != EVKCU_ACT_NONE) z[u] = ld_vec8(pre + at);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + u * RL >= r1) break;
                float f[8];
                unpack8<T>(a[u], f);
                if (ACT != EVKCU_ACT_NONE) {
                    float y[8];
                    unpack8<T>(z[u], y);
                    dact_all(f, y, ACT);
                    st_vec8(dz + (uint64_t)(r + u * RL) * N + col, pack8<T>(f));
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += f[e];
            }
        }
    }
    if (!dbias) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s_sum[rl][cl * 8 + e] = sum[e];
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 8 * L; i += kDactThreads) {
        float t = 0.0f;
        for (uint32_t k = 0; k < RL; ++k) t += s_sum[k][i];
        s_col[i] = t;
    }
    sm100::cluster_sync_all();
    const uint32_t c = blockIdx.x * (8 * L) + threadIdx.x;
    if (blockIdx.y == 0 && threadIdx.x < 8 * L && c < N) {
        float part = 0.0f;
        for (uint32_t r = 0; r < kDactCluster; ++r) {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(v)
                         : "r"(sm100::map_shared_rank(&s_col[threadIdx.x], r))
                         : "memory");
            part += v;
        }
        if (acc) part += Elem<T>::to_f(dbias[c]);
        dbias[c] = Elem<T>::from_f(part);
    }
    sm100::cluster_sync_relaxed();  // no CTA leaves while rank 0 still reads its sums
}

template <typename T, int L, int U>
int launch_dact_of(const void* dy, const void* pre, void* dz, void* dbias, uint32_t rows, uint32_t N, int act, int acc,
                   int trigger, cudaStream_t st) {
    auto go = [&](auto kern) {
        return launch_pdl("evkcu_linear_backward(dact)", kern, dim3((N + 8 * L - 1) / (8 * L), kDactCluster),
                          dim3(kDactThreads), 0, st, (const T*)dy, (const T*)pre, (T*)dz, (T*)dbias, rows, N, acc,
                          trigger);
    };
    switch (act) {
        case EVKCU_ACT_RELU: return go(dact_kernel<T, L, U, EVKCU_ACT_RELU>);
        case EVKCU_ACT_GELU: return go(dact_kernel<T, L, U, EVKCU_ACT_GELU>);
        case EVKCU_ACT_SILU: return go(dact_kernel<T, L, U, EVKCU_ACT_SILU>);
        default: return go(dact_kernel<T, L, U, EVKCU_ACT_NONE>);
    }
}

// One row a lane and eight CTAs an SM hide the memory best where there are
// that many CTAs: 32 columns a cluster (4096 x 8192 GELU: 45 us; 64 columns 49,
// four rows a lane and 64 columns 56), 16 in narrower layers (16384 x 2048: 49 us
// against 57), and four rows a lane where even those are too few (16384 x 512:
// 19 us against 26).  Set at GELU; SILU and RELU, which compute less, take 37,
// 46 and 13 us there, and 64 columns would do in 35 (one row a lane) and, four rows
// a lane, 39 us.
template <typename T>
int launch_dact(const void* dy, const void* pre, void* dz, void* dbias, uint32_t rows, uint32_t N, int act, int acc,
                int trigger, cudaStream_t st) {
    const uint32_t enough = 5 * (uint32_t)state()->sm_count;
    if ((N + 31) / 32 * kDactCluster >= enough)
        return launch_dact_of<T, 4, 1>(dy, pre, dz, dbias, rows, N, act, acc, trigger, st);
    if ((N + 15) / 16 * kDactCluster >= enough)
        return launch_dact_of<T, 2, 1>(dy, pre, dz, dbias, rows, N, act, acc, trigger, st);
    return launch_dact_of<T, 2, 4>(dy, pre, dz, dbias, rows, N, act, acc, trigger, st);
}

// ---------------------------------------------------------------- checks ----
constexpr uint32_t kMaxDim = 1u << 30;  // TMA coordinates are signed 32-bit

int check_common(const char* op, uint32_t rows, uint32_t a, uint32_t b, int act, uint32_t flags, uint32_t allowed,
                 int dtype) {
    EVKCU_CHECK_ARG(dtype == EVKCU_F16 || dtype == EVKCU_BF16, EVKCU_BAD_ARG, std::string(op) + ": unknown dtype");
    EVKCU_CHECK_ARG(act >= EVKCU_ACT_NONE && act <= EVKCU_ACT_SILU, EVKCU_BAD_ARG,
                    std::string(op) + ": unknown activation");
    EVKCU_CHECK_ARG((flags & ~allowed) == 0, EVKCU_BAD_ARG, std::string(op) + ": unknown flag");
    EVKCU_CHECK_ARG(a > 0 && b > 0 && a % 8 == 0 && b % 8 == 0, EVKCU_BAD_SHAPE,
                    std::string(op) + ": feature sizes must be positive multiples of 8");
    EVKCU_CHECK_ARG(rows <= kMaxDim && a <= kMaxDim && b <= kMaxDim, EVKCU_BAD_SHAPE,
                    std::string(op) + ": size above 2^30");
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
               int dtype, cudaStream_t st, bool early, bool trigger) {
    return product<T, false>(Product{dz, w, rows, K, N, K, nk, dtype, st, early, trigger}, epi_plain<T>(dx, K, acc));
}
// dW[K, N] (+)= x^T dz (or its transpose [N, K] = dz^T x when nk).
template <typename T>
int grad_weight(const void* x, const void* dz, void* dw, uint32_t rows, uint32_t K, uint32_t N, bool nk, bool acc,
                int dtype, cudaStream_t st, bool trigger) {
    if (nk)
        return product<T, true>(Product{dz, x, N, K, rows, K, true, dtype, st, false, trigger},
                                epi_plain<T>(dw, K, acc));
    return product<T, true>(Product{x, dz, K, N, rows, N, true, dtype, st, false, trigger}, epi_plain<T>(dw, N, acc));
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
        if (has_act || dbias) EVKCU_TRY(launch_dact<T>(dy, pre, dpre, dbias, rows, N, act, acc, dx || dw, st));
        const void* dz = has_act ? dpre : dy;
        if (dx) EVKCU_TRY(grad_input<T>(dz, w, dx, rows, K, N, nk, acc, dtype, st, has_act || dbias, dw != nullptr));
        if (dw) EVKCU_TRY(grad_weight<T>(x, dz, dw, rows, K, N, nk, acc, dtype, st, false));
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
        EVKCU_TRY((product<T, false>(Product{x, w_in, rows, F, D, 2 * F, !nk, dtype, st, false, y != nullptr},
                                     EpiGated<T>{(T*)hidden, (T*)pre, F, act})));
        if (!y) return (int)EVKCU_OK;
        return product<T, false>(Product{hidden, w_out, rows, D, F, D, !nk, dtype, st, true},
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
        EVKCU_TRY((product<T, false>(Product{dy, w_out, rows, F, D, F, nk, dtype, st, false, dx || dw_in || dw_out},
                                     EpiGatedBwd<T>{(const T*)pre, (T*)dpre, dw_out ? (T*)hidden : nullptr, F, act})));
        if (dx) EVKCU_TRY(grad_input<T>(dpre, w_in, dx, rows, D, 2 * F, nk, acc, dtype, st, true, dw_in || dw_out));
        if (dw_in) EVKCU_TRY(grad_weight<T>(x, dpre, dw_in, rows, D, 2 * F, nk, acc, dtype, st, dw_out != nullptr));
        if (dw_out) EVKCU_TRY(grad_weight<T>(hidden, dy, dw_out, rows, F, D, nk, acc, dtype, st, false));
        return (int)EVKCU_OK;
    });
}
