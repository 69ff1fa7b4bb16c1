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
// elements (16 bytes) a lane, so the mean is a few shuffles.  The angles of a
// row are computed once per block into shared memory and serve all its heads.
#include <algorithm>
#include <cmath>
#include <string>

#include "linear.cuh"

namespace evkcu {
namespace {

constexpr int kThreads = 256;
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
    float eps;
    uint32_t R, heads_per_block;  // rows and heads of a block's tile
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
__device__ __forceinline__ float2 turn_cs(double turns, int32_t pos) {
    const double t = (double)pos * turns;
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    return make_float2(c, s);
}

__device__ __forceinline__ void fill_angles(const QkArgs& a, float2* cs, uint32_t row0, uint32_t nrows) {
    const uint32_t half = a.rot / 2;
    for (uint32_t i = threadIdx.x; i < nrows * half; i += kThreads)
        cs[i] = turn_cs(a.turns[i % half], position(a, row0 + i / half));
}

// Rotates the lane's eight elements f (element c * 8 of the head on) by the
// row's angles; sgn = -1 is the inverse rotation.  All lanes of the warp call
// it together (half-split pairs exchange lanes c and c + rot / 16).
template <int LPH>
__device__ __forceinline__ void rotate8(const QkArgs& a, const float2* cs, uint32_t c, float sgn, float (&f)[8]) {
    if (!a.half_split) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t p = c * 4 + j;
            if (p < a.rot / 2) {
                const float2 t = cs[p];
                const float x = f[2 * j], y = f[2 * j + 1], s = sgn * t.y;
                f[2 * j] = x * t.x - y * s;
                f[2 * j + 1] = x * s + y * t.x;
            }
        }
        return;
    }
    const uint32_t hl = a.rot / 16;  // lanes of one half
    const bool lo = c < hl, hi = !lo && c < 2 * hl;
    const uint32_t partner = lo ? c + hl : (hi ? c - hl : c);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float o = __shfl_sync(0xffffffffu, f[e], partner, LPH);
        if (lo || hi) {
            const float2 t = cs[(lo ? c : c - hl) * 8 + e];
            const float s = sgn * t.y;
            f[e] = lo ? f[e] * t.x - o * s : o * s + f[e] * t.x;
        }
    }
}

template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, LPH);
    return v;
}

template <typename T>
__device__ __forceinline__ Vec8 load8(const void* p, uint64_t at, bool ok) {
    Vec8 z = {{0u, 0u, 0u, 0u}};
    return ok ? ld_vec8(reinterpret_cast<const T*>(p) + at) : z;
}

template <typename T, int LPH>
__global__ void __launch_bounds__(kThreads) qk_forward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ float2 s_cs[];  // [R][rot / 2]
    constexpr uint32_t G = kThreads / LPH;
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t total = a.H + a.Hk + (a.v ? a.Hk : 0);
    const uint32_t h0 = blockIdx.y * a.heads_per_block, nh = min(a.heads_per_block, total - h0);
    const uint32_t row0 = blockIdx.x * a.R, nrows = min(a.R, a.rows - row0);
    fill_angles(a, s_cs, row0, nrows);
    __syncthreads();
    const bool lane_on = c * 8 < a.Dh;
    for (uint32_t i0 = 0; i0 < nrows * nh; i0 += G) {
        const uint32_t i = i0 + g;
        const bool on = i < nrows * nh;
        const uint32_t rl = on ? i / nh : 0, h = h0 + (on ? i % nh : 0), row = row0 + rl;
        const bool is_q = h < a.H, is_v = h >= a.H + a.Hk;
        const uint32_t hk = is_q ? h : (is_v ? h - a.H - a.Hk : h - a.H);
        const void* src = is_q ? a.q : (is_v ? a.v : a.k);
        const uint64_t pitch = is_q ? a.q_pitch : (is_v ? a.v_pitch : a.k_pitch);
        const bool ld = on && lane_on;
        const Vec8 raw = load8<T>(src, row * pitch + (uint64_t)hk * a.Dh + c * 8, ld);
        float f[8];
        unpack8<T>(raw, f);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
        const float r = rsqrtf(group_sum<LPH>(ss) / (float)a.Dh + a.eps);
        const void* gain = is_q ? a.gq : a.gk;
        float w[8];
        if (gain) unpack8<T>(load8<T>(gain, c * 8, lane_on), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = gain ? f[e] * r * w[e] : f[e] * r;
        rotate8<LPH>(a, s_cs + rl * (a.rot / 2), c, 1.0f, f);
        if (!ld) continue;
        const Vec8 out = is_v ? raw : pack8<T>(f);
        if (is_q) {
            st_vec8(reinterpret_cast<T*>(a.qo) + row * a.qo_pitch + (uint64_t)h * a.Dh + c * 8, out);
        } else {
            uint64_t at = row;
            if (a.cache) {
                const int32_t pos = position(a, row);
                if (pos < 0 || (uint32_t)pos >= a.cache_len) continue;  // outside the cache: not stored
                at = (uint64_t)(row / a.S) * a.cache_len + (uint32_t)pos;
            }
            st_vec8(reinterpret_cast<T*>(is_v ? a.vo : a.ko) + at * a.ko_pitch + (uint64_t)hk * a.Dh + c * 8, out);
        }
    }
}

// Block b walks row tiles b, b + gridDim.x, ...: each lane adds its columns'
// gain gradients over all heads it meets, the block adds its groups in order
// and stores one partial row, and qk_gain_kernel adds the partials in order,
// so the sums do not depend on timing.
template <typename T, int LPH>
__global__ void __launch_bounds__(kThreads) qk_backward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ float2 s_cs[];  // [R][rot / 2]; then the groups' sums [G][2][Dh]
    constexpr uint32_t G = kThreads / LPH;
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t total = a.H + a.Hk;
    const bool lane_on = c * 8 < a.Dh;
    float accq[8] = {}, acck[8] = {};
    for (uint32_t row0 = blockIdx.x * a.R; row0 < a.rows; row0 += gridDim.x * a.R) {
        const uint32_t nrows = min(a.R, a.rows - row0);
        __syncthreads();  // the previous tile's angles have been read
        fill_angles(a, s_cs, row0, nrows);
        __syncthreads();
        for (uint32_t i0 = 0; i0 < nrows * total; i0 += G) {
            const uint32_t i = i0 + g;
            const bool on = i < nrows * total;
            const uint32_t rl = on ? i / total : 0, h = on ? i % total : 0, row = row0 + rl;
            const bool is_q = h < a.H;
            const uint32_t hk = is_q ? h : h - a.H;
            const bool ld = on && lane_on;
            const uint64_t col = (uint64_t)hk * a.Dh + c * 8;
            float x[8], t[8];
            unpack8<T>(load8<T>(is_q ? a.q : a.k, row * (is_q ? a.q_pitch : a.k_pitch) + col, ld), x);
            unpack8<T>(load8<T>(is_q ? a.dqo : a.dko, row * (is_q ? a.dqo_pitch : a.dko_pitch) + col, ld), t);
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
            const float r = rsqrtf(group_sum<LPH>(ss) / (float)a.Dh + a.eps);
            rotate8<LPH>(a, s_cs + rl * (a.rot / 2), c, -1.0f, t);
            const void* gain = is_q ? a.gq : a.gk;
            float w[8];
            if (gain) unpack8<T>(load8<T>(gain, c * 8, lane_on), w);
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] *= r;  // n
                const float d = t[e] * x[e];
                if (is_q) accq[e] += d;
                else acck[e] += d;
                t[e] = gain ? t[e] * w[e] : t[e];  // dn
                m += t[e] * x[e];
            }
            m = group_sum<LPH>(m) / (float)a.Dh;
            if (!ld) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = r * (t[e] - x[e] * m);
            T* dst = reinterpret_cast<T*>(is_q ? a.qo : a.ko) + row * (is_q ? a.qo_pitch : a.ko_pitch) + col;
            st_vec8(dst, pack8<T>(t));
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
__global__ void __launch_bounds__(1024) qk_gain_kernel(const float* __restrict__ partial, uint32_t n, uint32_t Dh,
                                                       T* dgq, T* dgk, int acc) {
    __shared__ float s[32][33];
    const uint32_t lane = threadIdx.x & 31, rl = threadIdx.x >> 5, j = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (j < 2 * Dh)
        for (uint32_t i = rl; i < n; i += 32) v += partial[(uint64_t)i * 2 * Dh + j];
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

bool pitch_ok(uint64_t pitch, uint64_t cols) { return pitch >= cols && pitch % 8 == 0 && pitch <= (1ull << 40); }

int check_desc(const std::string& op, const evkcu_qk_norm_rope_desc* d, uint32_t allowed, int dtype) {
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

int check_tensor(const std::string& op, const char* name, const void* p, uint64_t pitch, uint64_t cols) {
    EVKCU_CHECK_ARG(p, EVKCU_BAD_ARG, op + ": " + name + " is null");
    EVKCU_CHECK_ARG(aligned16(p), EVKCU_BAD_ALIGN, op + ": " + name + " must be 16-byte aligned");
    EVKCU_CHECK_ARG(pitch_ok(pitch, cols), EVKCU_BAD_SHAPE,
                    op + ": the row pitch of " + name + " must be a multiple of 8 that holds its row");
    return EVKCU_OK;
}
int check_gain(const std::string& op, const void* p) {
    EVKCU_CHECK_ARG(aligned16(p), EVKCU_BAD_ALIGN, op + ": gains must be 16-byte aligned");
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
    EVKCU_TRY(check_gain(op, gain_q));
    EVKCU_TRY(check_gain(op, gain_k));
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
    a.R = 1;
    a.heads_per_block = total;
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        return with_lph(a.Dh, [&](auto lph) {
            const dim3 grid((a.rows + a.R - 1) / a.R, (total + a.heads_per_block - 1) / a.heads_per_block);
            qk_forward_kernel<T, lph.value>
                <<<grid, kThreads, a.R * (a.rot / 2) * sizeof(float2), as_stream(stream)>>>(a);
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
    EVKCU_TRY(check_gain(op, gain_q));
    EVKCU_TRY(check_gain(op, gain_k));
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
    a.R = 1;
    return EVKCU_DISPATCH_DTYPE(dtype, T, [&] {
        return with_lph(a.Dh, [&](auto lph) {
            const uint32_t tiles = (a.rows + a.R - 1) / a.R;
            const uint32_t grid = std::min({tiles, kMaxPartials, 4u * (uint32_t)ds->sm_count});
            const size_t smem = std::max<size_t>(a.R * (a.rot / 2) * sizeof(float2),
                                                 gains ? (size_t)(kThreads / lph.value) * 2 * a.Dh * sizeof(float) : 0);
            qk_backward_kernel<T, lph.value><<<grid, kThreads, smem, st>>>(a);
            EVKCU_TRY(after_launch("evkcu_qk_norm_rope_backward"));
            if (!gains) return (int)EVKCU_OK;
            qk_gain_kernel<T><<<(2 * a.Dh + 31) / 32, 1024, 0, st>>>(a.partial, grid, a.Dh, (T*)dgain_q, (T*)dgain_k,
                                                                    acc);
            return after_launch("evkcu_qk_norm_rope_backward(gains)");
        });
    });
}
