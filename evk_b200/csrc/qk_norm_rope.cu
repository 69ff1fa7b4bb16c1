// qk_norm_rope.cu — RMSNorm of every query and key head and its position
// rotation in one pass, forward (optionally into a KV cache) and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps);  n = x r;  y = R(pos) (n * gain)
// with R the rotation of rot_dim / 2 pairs by pos * base^(-2 i / rot_dim).
// Backward, from dy and the saved x:
//   t = R^T dy;  dgain += t * n;  dn = t * gain
//   dx = r (dn - n mean(dn * n))
//
// Bound by HBM: each value is read once and written once (backward: read x
// and dy, write dx).  A group of LPH lanes holds one head in registers, eight
// elements (16 bytes) a lane, so the mean is a few shuffles.  A block's G =
// 256 / LPH groups are GH heads x GR rows, and a group takes one head of U
// rows at a time: the gain is loaded once for them and U (backward: 2 U)
// 16-byte loads per lane are in flight.  The angles of a row are computed once
// per block into shared memory, behind the first loads, and serve all heads.
#include <algorithm>
#include <cmath>
#include <string>
#include <type_traits>

#include "linear.cuh"

namespace evkcu {
namespace {

constexpr int kThreads = 256;
// Rows a group takes at a time, and resident blocks per SM.  Forward, 16384
// rows of 32 heads of 128: 57 us; 2 rows and 5 blocks 65, 4 and 3 64, 4 and 5
// 61, 1 and 8 77.  Backward, 8192 rows of 40: 67 us; 2 rows and 3 blocks 75,
// 2 and 4 79.  (41 and 39 us at the copy rate; issue slots are 63 % busy.)
constexpr int kFwdRows = 4, kFwdBlocks = 4, kBwdRows = 4, kBwdBlocks = 2;
constexpr uint32_t kMaxHalf = 128;       // rotation pairs of the largest head (256)
constexpr uint32_t kMaxPartials = 1024;  // gain-gradient partial rows in the workspace

struct QkArgs {
    const void *q, *k, *v, *gq, *gk;
    void *qo, *ko, *vo;
    uint64_t q_pitch, k_pitch, v_pitch, qo_pitch, ko_pitch;
    const int32_t* positions;
    uint32_t rows, S, H, Hk, Dh, rot;
    uint32_t pos_offset, cache_len;
    int half_split, cache;
    float eps, inv_dh;
    uint32_t GH, GR;  // a block's groups: heads x rows (GH GR = G, powers of two)
    uint32_t heads_per_block;
    // backward: gradients of the outputs come through (q, k)-shaped dqo, dko
    const void *dqo, *dko;
    uint64_t dqo_pitch, dko_pitch;
    float* partial;  // [gridDim.x][2][Dh], or null
    // turns per position of pair i: base^(-2 i / rot) / (2 pi), in 64 bits
    double turns[kMaxHalf];
};

__device__ __forceinline__ int32_t position(const QkArgs& a, uint32_t row) {
    return a.positions ? a.positions[row] : (int32_t)(a.pos_offset + row % a.S);
}

// (cos, sin) of pos * base^(-2 i / rot).  The angle is reduced to a fraction
// of a turn in 64 bits: in 32 a position of 10^5 would leave it 0.004 off.
// Within half a turn sin.approx and cos.approx are off by 2^-21 at most.
__device__ __forceinline__ float2 turn_cs(double turns, int32_t pos) {
    const double t = (double)pos * turns;
    const float x = 6.2831853071795865f * (float)(t - rint(t));
    return make_float2(__cosf(x), __sinf(x));
}

// Row pitch of the angles: whole lanes of four pairs, the pairs past rot / 2
// turned by 0 so that a lane need not look where the rotation ends.
__host__ __device__ inline uint32_t angle_pitch(uint32_t rot) { return (rot / 2 + 3) / 4 * 4; }

// The table lies among the kernel's parameters.  Lanes read different entries,
// which the constant cache serves one at a time; by its generic address it
// goes through L1.
__device__ __forceinline__ double turns_at(const QkArgs& a, uint32_t p) {
    double t;
    asm("ld.f64 %0, [%1];" : "=d"(t) : "l"(&a.turns[p]));
    return t;
}

__device__ __forceinline__ void fill_angles(const QkArgs& a, float2* cs, uint32_t row0, uint32_t nrows) {
    const uint32_t pitch = angle_pitch(a.rot);
    for (uint32_t i = threadIdx.x; i < nrows * pitch; i += kThreads) {
        const uint32_t p = i % pitch;
        cs[i] = p < a.rot / 2 ? turn_cs(turns_at(a, p), position(a, row0 + i / pitch)) : make_float2(1.0f, 0.0f);
    }
}

// Rotates the lane's eight elements f (element c * 8 of the head on) by the
// row's angles cs (16-byte aligned rows: see angle_pitch); sgn = -1 is the
// inverse rotation.  All lanes of the warp call it together (half-split pairs
// exchange lanes c and c + rot / 16).
template <int LPH>
__device__ __forceinline__ void rotate8(const QkArgs& a, const float2* cs, uint32_t c, float sgn, float (&f)[8]) {
    if (!a.half_split) {
        if (c * 8 >= a.rot) return;
        const float4* v = reinterpret_cast<const float4*>(cs + c * 4);
        const float4 t0 = v[0], t1 = v[1];
        const float co[4] = {t0.x, t0.z, t1.x, t1.z}, si[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = f[2 * j], y = f[2 * j + 1], s = sgn * si[j];
            f[2 * j] = x * co[j] - y * s;
            f[2 * j + 1] = x * s + y * co[j];
        }
        return;
    }
    const uint32_t hl = a.rot / 16;  // lanes of one half
    const bool lo = c < hl, hi = !lo && c < 2 * hl;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = __shfl_sync(0xffffffffu, f[e], lo ? c + hl : (hi ? c - hl : c), LPH);
    if (!lo && !hi) return;
    const float4* v = reinterpret_cast<const float4*>(cs + (lo ? c : c - hl) * 8);
    const float s0 = lo ? -sgn : sgn;  // low half x cos - y sin, high half y cos + x sin
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 t = v[e];
        f[2 * e] = f[2 * e] * t.x + s0 * o[2 * e] * t.y;
        f[2 * e + 1] = f[2 * e + 1] * t.z + s0 * o[2 * e + 1] * t.w;
    }
}

// Sums over a group's lanes, U of them side by side.
template <int LPH, int U>
__device__ __forceinline__ void group_sums(float (&v)[U]) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o, LPH);
}

template <typename T>
__device__ __forceinline__ Vec8 load8(const void* p, uint64_t at, bool ok) {
    Vec8 z = {{0u, 0u, 0u, 0u}};
    return ok ? ld_vec8(reinterpret_cast<const T*>(p) + at) : z;
}

// The lane's eight gains, or ones.
template <typename T>
__device__ __forceinline__ void load_gain(const void* gain, uint32_t c, bool lane_on, float (&w)[8]) {
    if (gain) {
        unpack8<T>(load8<T>(gain, c * 8, lane_on), w);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.0f;
}

template <typename T, int LPH, int U>
__global__ void __launch_bounds__(kThreads, kFwdBlocks) qk_forward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ __align__(16) float2 s_cs[];  // [GR U][angle_pitch]
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t gh = g % a.GH, gr = g / a.GH, half = angle_pitch(a.rot);
    const uint32_t total = a.H + a.Hk + (a.v ? a.Hk : 0);
    const uint32_t h_end = min(total, (blockIdx.y + 1) * a.heads_per_block);
    const uint32_t R = a.GR * U, row0 = blockIdx.x * R, nrows = min(R, a.rows - row0);
    const bool lane_on = c * 8 < a.Dh;
    bool first = true;
    for (uint32_t h0 = blockIdx.y * a.heads_per_block; h0 < h_end; h0 += a.GH) {
        const uint32_t h = h0 + gh;
        const bool on = h < h_end && lane_on;
        const bool is_q = h < a.H, is_v = h >= a.H + a.Hk;
        const uint32_t hk = is_q ? h : (is_v ? h - a.H - a.Hk : h - a.H);
        const void* src = is_q ? a.q : (is_v ? a.v : a.k);
        const uint64_t pitch = is_q ? a.q_pitch : (is_v ? a.v_pitch : a.k_pitch);
        const uint64_t col = (uint64_t)hk * a.Dh + c * 8;
        Vec8 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t rl = gr + u * a.GR;
            raw[u] = load8<T>(src, (row0 + rl) * pitch + col, on && rl < nrows);
        }
        const void* gain = is_q ? a.gq : a.gk;
        float w[8];
        load_gain<T>(gain, c, lane_on, w);
        if (first) {
            fill_angles(a, s_cs, row0, nrows);
            __syncthreads();
            first = false;
        }
        void* dst = is_q ? a.qo : (is_v ? a.vo : a.ko);
        const uint64_t opitch = is_q ? a.qo_pitch : a.ko_pitch;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t rl = gr + u * a.GR, row = row0 + rl;
            float f[8], ss[1] = {0.0f};
            unpack8<T>(raw[u], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[0] += f[e] * f[e];
            group_sums<LPH, 1>(ss);
            const float r = rsqrtf(ss[0] * a.inv_dh + a.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= r * w[e];
            rotate8<LPH>(a, s_cs + min(rl, nrows - 1) * half, c, 1.0f, f);
            bool st = on && rl < nrows;
            uint64_t at = row;
            if (a.cache && !is_q && st) {
                const int32_t pos = position(a, row);
                st = pos >= 0 && (uint32_t)pos < a.cache_len;  // outside the cache: not stored
                at = (uint64_t)(row / a.S) * a.cache_len + (uint32_t)pos;
            }
            if (st) st_vec8(reinterpret_cast<T*>(dst) + at * opitch + col, is_v ? raw[u] : pack8<T>(f));
        }
    }
}

// Block b walks row tiles b, b + gridDim.x, ...: each lane adds its columns'
// gain gradients over all heads it meets, the block adds its groups in order
// and stores one partial row, and qk_gain_kernel adds the partials in order,
// so the sums do not depend on timing.
template <typename T, int LPH, int U>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) qk_backward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ __align__(16) float2 s_cs[];  // [GR U][angle_pitch]; then the groups' sums [G][2][Dh]
    constexpr uint32_t G = kThreads / LPH;
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t gh = g % a.GH, gr = g / a.GH, half = angle_pitch(a.rot);
    const uint32_t total = a.H + a.Hk, R = a.GR * U;
    const bool lane_on = c * 8 < a.Dh;
    float accq[8] = {}, acck[8] = {};
    if (a.partial) pdl_trigger();  // qk_gain_kernel, which waits for this one to end
    for (uint32_t row0 = blockIdx.x * R; row0 < a.rows; row0 += gridDim.x * R) {
        const uint32_t nrows = min(R, a.rows - row0);
        bool first = true;
        for (uint32_t h0 = 0; h0 < total; h0 += a.GH) {
            const uint32_t h = h0 + gh;
            const bool on = h < total && lane_on, is_q = h < a.H;
            const uint64_t col = (uint64_t)(is_q ? h : h - a.H) * a.Dh + c * 8;
            Vec8 rx[U], rt[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t rl = gr + u * a.GR, row = row0 + rl;
                const bool ld = on && rl < nrows;
                rx[u] = load8<T>(is_q ? a.q : a.k, row * (is_q ? a.q_pitch : a.k_pitch) + col, ld);
                rt[u] = load8<T>(is_q ? a.dqo : a.dko, row * (is_q ? a.dqo_pitch : a.dko_pitch) + col, ld);
            }
            const void* gain = is_q ? a.gq : a.gk;
            float w[8];
            load_gain<T>(gain, c, lane_on, w);
            if (first) {
                __syncthreads();  // the previous tile's angles have been read
                fill_angles(a, s_cs, row0, nrows);
                __syncthreads();
                first = false;
            }
            float x[U][8], t[U][8], ss[U], m[U], acc[8] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                unpack8<T>(rx[u], x[u]);
                unpack8<T>(rt[u], t[u]);
                ss[u] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss[u] += x[u][e] * x[u][e];
            }
            group_sums<LPH, U>(ss);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rotate8<LPH>(a, s_cs + min(gr + u * a.GR, nrows - 1) * half, c, -1.0f, t[u]);
                ss[u] = rsqrtf(ss[u] * a.inv_dh + a.eps);
                m[u] = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[u][e] *= ss[u];  // n
                    acc[e] += t[u][e] * x[u][e];
                    t[u][e] *= w[e];  // dn
                    m[u] += t[u][e] * x[u][e];
                }
            }
            group_sums<LPH, U>(m);
            T* dst = reinterpret_cast<T*>(is_q ? a.qo : a.ko) + col;
            const uint64_t opitch = is_q ? a.qo_pitch : a.ko_pitch;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t rl = gr + u * a.GR;
                m[u] *= a.inv_dh;
#pragma unroll
                for (int e = 0; e < 8; ++e) t[u][e] = ss[u] * (t[u][e] - x[u][e] * m[u]);
                if (on && rl < nrows) st_vec8(dst + (row0 + rl) * opitch, pack8<T>(t[u]));
            }
            if (!a.partial) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (is_q) accq[e] += acc[e];
                else acck[e] += acc[e];
            }
        }
    }
    if (!a.partial) return;
    float* sums = reinterpret_cast<float*>(s_cs);
    __syncthreads();
    if (lane_on) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sums[(g * 2 + 0) * a.Dh + c * 8 + e] = accq[e];
            sums[(g * 2 + 1) * a.Dh + c * 8 + e] = acck[e];
        }
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < 2 * a.Dh; j += kThreads) {
        float s = 0.0f;
        for (uint32_t i = 0; i < G; ++i) s += sums[i * 2 * a.Dh + j];
        a.partial[(uint64_t)blockIdx.x * 2 * a.Dh + j] = s;
    }
}

// dgain (+)= sum of the partial rows: 32 columns a block, 32 row lanes.
template <typename T>
__global__ void __launch_bounds__(1024) qk_gain_kernel(const float* partial, uint32_t n, uint32_t Dh,
                                                       T* dgq, T* dgk, int acc) {
    __shared__ float s[32][33];
    const uint32_t lane = threadIdx.x & 31, rl = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float v = 0.0f;
    pdl_wait();
    for (uint32_t i0 = rl; i0 < n; i0 += 32 * 8) {  // eight loads in flight, added in order
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            t[k] = i0 + 32 * k < n && j < 2 * Dh ? partial[(uint64_t)(i0 + 32 * k) * 2 * Dh + j] : 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) v += t[k];
    }
    s[rl][lane] = v;
    __syncthreads();
    if (rl != 0 || j >= 2 * Dh) return;
    float t = 0.0f;
    for (int i = 0; i < 32; ++i) t += s[i][lane];
    T* dst = j < Dh ? dgq : dgk;
    if (!dst) return;
    dst += j < Dh ? j : j - Dh;
    *dst = Elem<T>::from_f(acc ? Elem<T>::to_f(*dst) + t : t);
}

uint32_t lanes_per_head(uint32_t Dh) { return Dh <= 32 ? 4 : Dh <= 64 ? 8 : Dh <= 128 ? 16 : 32; }

// Calls f with the lanes-per-head constant of head size Dh.
template <class F>
int with_lph(uint32_t Dh, F&& f) {
    switch (lanes_per_head(Dh)) {
        case 4: return f(std::integral_constant<int, 4>());
        case 8: return f(std::integral_constant<int, 8>());
        case 16: return f(std::integral_constant<int, 16>());
        default: return f(std::integral_constant<int, 32>());
    }
}

// Heads x rows of a block's groups: the most heads that leave under a
// sixteenth of the groups without one (40 heads, 16 groups: 8 x 2).
void set_groups(QkArgs& a, uint32_t total) {
    const uint32_t G = kThreads / lanes_per_head(a.Dh);
    for (a.GH = G; a.GH > 1; a.GH /= 2)
        if (total * 16 >= (total + a.GH - 1) / a.GH * a.GH * 15) break;
    a.GR = G / a.GH;
}

bool pitch_ok(uint64_t pitch, uint64_t cols) { return pitch >= cols && pitch % 8 == 0 && pitch <= (1ull << 40); }

int check_desc(const char* name, const evkcu_qk_norm_rope_desc* d, uint32_t allowed, int dtype) {
    const std::string op(name);
    EVKCU_CHECK_ARG(d, EVKCU_BAD_ARG, op + ": descriptor is null");
    EVKCU_CHECK_ARG(dtype == EVKCU_F16 || dtype == EVKCU_BF16, EVKCU_BAD_ARG, op + ": unknown dtype");
    EVKCU_CHECK_ARG((d->flags & ~allowed) == 0, EVKCU_BAD_ARG, op + ": unknown flag");
    EVKCU_CHECK_ARG(d->head_dim >= 8 && d->head_dim <= 256 && d->head_dim % 8 == 0, EVKCU_BAD_SHAPE,
                    op + ": head_dim must be a multiple of 8, 8 to 256");
    const uint32_t step = (d->flags & EVKCU_QK_HALF_SPLIT) ? 16 : 2;
    EVKCU_CHECK_ARG(d->rot_dim <= d->head_dim && (d->rot_dim ? d->rot_dim : d->head_dim) % step == 0, EVKCU_BAD_SHAPE,
                    op + ": rot_dim must be at most head_dim and a multiple of 2 (of 16 for half-split pairs)");
    EVKCU_CHECK_ARG(d->heads > 0 && d->heads <= 65535 && d->kv_heads <= 65535, EVKCU_BAD_SHAPE,
                    op + ": heads must be 1 to 65535, kv_heads at most 65535");
    EVKCU_CHECK_ARG((uint64_t)d->batch * d->seq_len <= (1ull << 30), EVKCU_BAD_SHAPE, op + ": more than 2^30 rows");
    EVKCU_CHECK_ARG(d->positions || (uint64_t)d->pos_offset + d->seq_len <= (1ull << 31), EVKCU_BAD_SHAPE,
                    op + ": positions above 2^31 - 1");
    EVKCU_CHECK_ARG(std::isfinite(d->base) && d->base > 0.0f && d->eps >= 0.0f, EVKCU_BAD_ARG,
                    op + ": base must be positive and eps not negative");
    EVKCU_CHECK_ARG((reinterpret_cast<uintptr_t>(d->positions) & 3u) == 0, EVKCU_BAD_ALIGN,
                    op + ": positions must be 4-byte aligned");
    return EVKCU_OK;
}

int check_tensor(const char* op, const char* name, const void* p, uint64_t pitch, uint64_t cols) {
    EVKCU_TRY(check_ptr(op, name, p, true));
    EVKCU_CHECK_ARG(pitch_ok(pitch, cols), EVKCU_BAD_SHAPE,
                    std::string(op) + ": the row pitch of " + name + " must be a multiple of 8 that holds its row");
    return EVKCU_OK;
}

void fill_args(QkArgs& a, const evkcu_qk_norm_rope_desc* d) {
    a.rows = d->batch * d->seq_len;  // at most 2^30, checked in 64 bits
    a.S = d->seq_len;
    a.H = d->heads;
    a.Hk = d->kv_heads;
    a.Dh = d->head_dim;
    a.rot = d->rot_dim ? d->rot_dim : d->head_dim;
    a.pos_offset = d->pos_offset;
    a.positions = d->positions;
    a.half_split = (d->flags & EVKCU_QK_HALF_SPLIT) ? 1 : 0;
    a.eps = d->eps;
    a.inv_dh = 1.0f / (float)a.Dh;
    // base^(-2 i / rot) by repeated products: 128 roundings of 2^-53 at most.
    const double ratio = std::pow((double)d->base, -2.0 / (double)a.rot);
    double t = 0.15915494309189535;  // 1 / (2 pi)
    for (uint32_t i = 0; i < a.rot / 2; ++i, t *= ratio) a.turns[i] = t;
}

}  // namespace
}  // namespace evkcu

using namespace evkcu;

extern "C" int evkcu_qk_norm_rope(const evkcu_qk_norm_rope_desc* d, const void* q, const void* k, const void* v,
                                  const void* gain_q, const void* gain_k, void* q_out, void* k_out, void* v_out,
                                  int dtype, void* stream) {
    const char* op = "evkcu_qk_norm_rope";
    EVKCU_TRY(check_desc(op, d, EVKCU_QK_HALF_SPLIT | EVKCU_QK_CACHE, dtype));
    const bool cache = d->flags & EVKCU_QK_CACHE;
    EVKCU_CHECK_ARG(!cache || d->cache_len > 0, EVKCU_BAD_SHAPE, std::string(op) + ": cache_len is 0");
    EVKCU_CHECK_ARG((v == nullptr) == (v_out == nullptr), EVKCU_BAD_ARG, std::string(op) + ": v and v_out come together");
    if ((uint64_t)d->batch * d->seq_len == 0) return EVKCU_OK;
    const uint64_t qc = (uint64_t)d->heads * d->head_dim, kc = (uint64_t)d->kv_heads * d->head_dim;
    EVKCU_TRY(check_tensor(op, "q", q, d->q_pitch, qc));
    EVKCU_TRY(check_tensor(op, "q_out", q_out, d->q_out_pitch, qc));
    if (d->kv_heads) {
        EVKCU_TRY(check_tensor(op, "k", k, d->k_pitch, kc));
        EVKCU_TRY(check_tensor(op, "k_out", k_out, d->k_out_pitch, kc));
        if (v) {
            EVKCU_TRY(check_tensor(op, "v", v, d->v_pitch, kc));
            EVKCU_TRY(check_tensor(op, "v_out", v_out, d->k_out_pitch, kc));
        }
    }
    EVKCU_TRY(check_ptr(op, "gain_q", gain_q, false));
    EVKCU_TRY(check_ptr(op, "gain_k", gain_k, false));
    const uint64_t rows = (uint64_t)d->batch * d->seq_len, krows = cache ? (uint64_t)d->batch * d->cache_len : rows;
    EVKCU_TRY(check_spans(op, {Span{"q", q, rows, d->q_pitch, qc}, Span{"k", k, rows, d->k_pitch, kc},
                               Span{"v", v, rows, d->v_pitch, kc}, Span{"gain_q", gain_q, 1, d->head_dim, d->head_dim},
                               Span{"gain_k", gain_k, 1, d->head_dim, d->head_dim},
                               Span{"positions", d->positions, 1, 2 * rows, 2 * rows},
                               Span{"q_out", q_out, rows, d->q_out_pitch, qc, true, "q"},
                               Span{"k_out", k_out, krows, d->k_out_pitch, kc, true, cache ? nullptr : "k"},
                               Span{"v_out", v_out, krows, d->k_out_pitch, kc, true, cache ? nullptr : "v"}}));
    DeviceState* ds = state();
    EVKCU_CHECK_ARG(ds, EVKCU_CUDA_ERROR, std::string(op) + ": no device state");
    QkArgs a = {};
    fill_args(a, d);
    a.q = q, a.k = k, a.v = v, a.gq = gain_q, a.gk = gain_k, a.qo = q_out, a.ko = k_out, a.vo = v_out;
    a.q_pitch = d->q_pitch, a.k_pitch = d->k_pitch, a.v_pitch = d->v_pitch;
    a.qo_pitch = d->q_out_pitch, a.ko_pitch = d->k_out_pitch;
    a.cache = cache;
    a.cache_len = d->cache_len;
    const uint32_t total = a.H + a.Hk + (v ? a.Hk : 0);
    set_groups(a, total);
    // kFwdRows rows a group where that still fills the SMs twice over; otherwise
    // (decode) one row a group and one round of heads a block.
    const uint64_t rounds = (total + a.GH - 1) / a.GH;
    const bool large = ((uint64_t)a.rows + a.GR * kFwdRows - 1) / (a.GR * kFwdRows) >= 2 * (uint64_t)ds->sm_count;
    a.heads_per_block = large ? total : a.GH;
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        return with_lph(a.Dh, [&](auto lph) {
            const uint32_t R = a.GR * (large ? kFwdRows : 1);
            const dim3 grid((a.rows + R - 1) / R, large ? 1 : (uint32_t)rounds);
            const size_t smem = R * angle_pitch(a.rot) * sizeof(float2);  // at most 32 KB
            if (large) qk_forward_kernel<T, lph.value, kFwdRows><<<grid, kThreads, smem, as_stream(stream)>>>(a);
            else qk_forward_kernel<T, lph.value, 1><<<grid, kThreads, smem, as_stream(stream)>>>(a);
            return after_launch("evkcu_qk_norm_rope");
        });
    });
}

extern "C" uint64_t evkcu_qk_norm_rope_workspace(uint32_t head_dim) {
    return (uint64_t)kMaxPartials * 2 * head_dim * sizeof(float);
}

extern "C" int evkcu_qk_norm_rope_backward(const evkcu_qk_norm_rope_desc* d, const void* q, const void* k,
                                           const void* gain_q, const void* gain_k, const void* dq_out,
                                           const void* dk_out, void* dq, void* dk, void* dgain_q, void* dgain_k,
                                           void* workspace, uint64_t workspace_bytes, int dtype, void* stream) {
    const char* op = "evkcu_qk_norm_rope_backward";
    EVKCU_TRY(check_desc(op, d, EVKCU_QK_HALF_SPLIT | EVKCU_QK_ACC_GAIN, dtype));
    const bool acc = d->flags & EVKCU_QK_ACC_GAIN, gains = dgain_q || dgain_k;
    cudaStream_t st = as_stream(stream);
    EVKCU_TRY(check_ptr(op, "gain_q", gain_q, false));
    EVKCU_TRY(check_ptr(op, "gain_k", gain_k, false));
    if ((uint64_t)d->batch * d->seq_len == 0) {  // empty sums
        if (dgain_q && !acc) EVKCU_CUDA_TRY(cudaMemsetAsync(dgain_q, 0, d->head_dim * 2, st));
        if (dgain_k && !acc) EVKCU_CUDA_TRY(cudaMemsetAsync(dgain_k, 0, d->head_dim * 2, st));
        return EVKCU_OK;
    }
    const uint64_t qc = (uint64_t)d->heads * d->head_dim, kc = (uint64_t)d->kv_heads * d->head_dim;
    EVKCU_TRY(check_tensor(op, "q", q, d->q_pitch, qc));
    EVKCU_TRY(check_tensor(op, "dq_out", dq_out, d->q_out_pitch, qc));
    EVKCU_TRY(check_tensor(op, "dq", dq, d->dq_pitch, qc));
    if (d->kv_heads) {
        EVKCU_TRY(check_tensor(op, "k", k, d->k_pitch, kc));
        EVKCU_TRY(check_tensor(op, "dk_out", dk_out, d->k_out_pitch, kc));
        EVKCU_TRY(check_tensor(op, "dk", dk, d->dk_pitch, kc));
    }
    if (gains) {
        EVKCU_CHECK_ARG(workspace && workspace_bytes >= evkcu_qk_norm_rope_workspace(d->head_dim), EVKCU_BAD_ARG,
                        std::string(op) + ": the gain gradients need a workspace of evkcu_qk_norm_rope_workspace bytes");
        EVKCU_CHECK_ARG(aligned16(workspace), EVKCU_BAD_ALIGN, std::string(op) + ": workspace must be 16-byte aligned");
    }
    const uint64_t rows = (uint64_t)d->batch * d->seq_len, dh = d->head_dim, wse = gains ? 4 * kMaxPartials * dh : 0;
    EVKCU_TRY(check_spans(op, {Span{"q", q, rows, d->q_pitch, qc}, Span{"k", k, rows, d->k_pitch, kc},
                               Span{"gain_q", gain_q, 1, dh, dh}, Span{"gain_k", gain_k, 1, dh, dh},
                               Span{"positions", d->positions, 1, 2 * rows, 2 * rows},
                               Span{"dq_out", dq_out, rows, d->q_out_pitch, qc},
                               Span{"dk_out", dk_out, rows, d->k_out_pitch, kc},
                               Span{"dq", dq, rows, d->dq_pitch, qc, true, "dq_out"},
                               Span{"dk", dk, rows, d->dk_pitch, kc, true, "dk_out"},
                               Span{"dgain_q", dgain_q, 1, dh, dh, true}, Span{"dgain_k", dgain_k, 1, dh, dh, true},
                               Span{"workspace", gains ? workspace : nullptr, 1, wse, wse, true}}));
    DeviceState* ds = state();
    EVKCU_CHECK_ARG(ds, EVKCU_CUDA_ERROR, std::string(op) + ": no device state");
    QkArgs a = {};
    fill_args(a, d);
    a.q = q, a.k = k, a.gq = gain_q, a.gk = gain_k, a.dqo = dq_out, a.dko = dk_out, a.qo = dq, a.ko = dk;
    a.q_pitch = d->q_pitch, a.k_pitch = d->k_pitch, a.dqo_pitch = d->q_out_pitch, a.dko_pitch = d->k_out_pitch;
    a.qo_pitch = d->dq_pitch, a.ko_pitch = d->dk_pitch;
    a.partial = gains ? (float*)workspace : nullptr;
    set_groups(a, a.H + a.Hk);
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        return with_lph(a.Dh, [&](auto lph) {
            constexpr uint32_t U = kBwdRows;
            const uint32_t R = a.GR * U, tiles = (a.rows + R - 1) / R;
            const uint32_t grid = std::min({tiles, kMaxPartials, kBwdBlocks * (uint32_t)ds->sm_count});  // resident at once
            const size_t smem = std::max<size_t>(R * angle_pitch(a.rot) * sizeof(float2),
                                                 gains ? (size_t)(kThreads / lph.value) * 2 * a.Dh * sizeof(float) : 0);
            qk_backward_kernel<T, lph.value, U><<<grid, kThreads, smem, st>>>(a);
            EVKCU_TRY(after_launch("evkcu_qk_norm_rope_backward"));
            if (!gains) return (int)EVKCU_OK;
            return launch_pdl("evkcu_qk_norm_rope_backward(gains)", qk_gain_kernel<T>, dim3((2 * a.Dh + 31) / 32),
                              dim3(1024), 0, st, (const float*)a.partial, grid, a.Dh, (T*)dgain_q, (T*)dgain_k,
                              (int)acc);
        });
    });
}
