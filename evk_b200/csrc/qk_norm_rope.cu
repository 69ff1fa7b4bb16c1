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
// and dy, write dx), with the issue slots not far behind.  A group of LPH
// lanes holds one head in registers, two vectors of eight elements a lane, so
// the mean is three shuffles at 128.  A block's G = 256 / LPH groups are GH
// heads x GR rows and walk its rows in rounds; asynchronous copies into the
// thread's own slots of shared memory run ahead of them.  The angles of a row
// are computed once per block into shared memory and serve all heads.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>
#include <type_traits>

#include "linear.cuh"

namespace evkcu {
namespace {

constexpr int kThreads = 256;
// Rows a group takes in a round, rounds of copies ahead, and resident blocks
// per SM.  Forward, 16384 rows of 32 heads of 128 (41 us at the copy rate):
// 51 us; 3 rows 53, 5 rows 52, 2 rows and 2 ahead 59, 4 blocks 58 (spills).
// Backward, 8192 rows of 40 heads (39 us): 57 us; 4 rows 61, 4 ahead 58,
// 2 rows and 3 blocks 76 (spills).  One vector a lane (twice the lanes, a
// shuffle more) took 55 and 63 us, loads through registers 57 and 67.
constexpr int kFwdRows = 4, kFwdAhead = 1, kFwdBlocks = 3, kBwdRows = 1, kBwdAhead = 2, kBwdBlocks = 2;
constexpr int kMaxSmem = 112 * 1024;     // slots and angles of a block
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

// Row pitch of the angles: whole lanes of four pairs, so that each lane's are
// aligned.  What lies past rot / 2 is not used.
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
        if (p < a.rot / 2) cs[i] = turn_cs(turns_at(a, p), position(a, row0 + i / pitch));
    }
}

// One vector of eight elements rotated by four (cos, sin) pairs; TAIL: only its
// first `pairs` pairs.  (Turning the others by 0 would pass an infinity or NaN
// on to its neighbour, as 0 times it.)
template <bool TAIL>
__device__ __forceinline__ void rotate_pairs(const float2* cs, float sgn, float (&f)[8], uint32_t pairs) {
    const float4* v = reinterpret_cast<const float4*>(cs);
    const float4 t0 = v[0], t1 = v[1];
    const float co[4] = {t0.x, t0.z, t1.x, t1.z}, si[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (TAIL && j >= pairs) break;
        const float x = f[2 * j], y = f[2 * j + 1], s = sgn * si[j];
        f[2 * j] = x * co[j] - y * s;
        f[2 * j + 1] = x * s + y * co[j];
    }
}
// f = f cos + o s0 sin over eight (cos, sin) pairs.
__device__ __forceinline__ void rotate_halves(const float2* cs, float s0, const float (&o)[8], float (&f)[8]) {
    const float4* v = reinterpret_cast<const float4*>(cs);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 t = v[e];
        f[2 * e] = f[2 * e] * t.x + s0 * o[2 * e] * t.y;
        f[2 * e + 1] = f[2 * e + 1] * t.z + s0 * o[2 * e + 1] * t.w;
    }
}

// Rotates the lane's two vectors, c and c + LPH of the head's, by the row's
// angles cs (see angle_pitch); sgn = -1 is the inverse rotation.  All lanes of
// the warp call it together: half-split pairs are vectors n and n + hl, the
// lane's own two where hl = LPH, otherwise exchanged.  TAIL: the rotated part ends
// inside a vector (adjacent pairs only).  A template and not a branch: with the
// test in every kernel 16384 rows of 32 heads of 128 took 55 us instead of 53.
template <int LPH, bool TAIL>
__device__ __forceinline__ void rotate(const QkArgs& a, const float2* cs, uint32_t c, float sgn, float (&f)[2][8]) {
    if (!a.half_split) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
            if ((c + v * LPH) * 8 < a.rot)
                rotate_pairs<TAIL>(cs + (c + v * LPH) * 4, sgn, f[v], a.rot / 2 - (c + v * LPH) * 4);
        return;
    }
    const uint32_t hl = a.rot / 16;
    if (hl == LPH) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = f[0][e];
        rotate_halves(cs + c * 8, -sgn, f[1], f[0]);  // low half: x cos - y sin
        rotate_halves(cs + c * 8, sgn, o, f[1]);      // high half: y cos + x sin
        return;
    }
    float o[2][8];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t n = c + v * LPH, at = n < hl ? n + hl : (n < 2 * hl ? n - hl : n);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            o[v][e] = __shfl_sync(0xffffffffu, f[0][e], at % LPH, LPH);
            if (2 * hl > LPH) {  // the pair reaches into the second vectors
                const float p = __shfl_sync(0xffffffffu, f[1][e], at % LPH, LPH);
                if (at >= LPH) o[v][e] = p;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t n = c + v * LPH;
        if (n < 2 * hl) rotate_halves(cs + (n < hl ? n : n - hl) * 8, n < hl ? -sgn : sgn, o[v], f[v]);
    }
}

// Sum over a group's lanes.
template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, LPH);
    return v;
}

// The lane's sixteen gains, or ones.
template <typename T, int LPH>
__device__ __forceinline__ void load_gain(const void* gain, uint32_t c, uint32_t Dh, float (&w)[2][8]) {
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const uint32_t n = c + v * LPH;
        if (gain && n * 8 < Dh) {
            unpack8<T>(ld_vec8(reinterpret_cast<const T*>(gain) + n * 8), w[v]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[v][e] = 1.0f;
        }
    }
}

// Asynchronous 16-byte copies to the thread's own slots in shared memory: the
// loads in flight need no registers, and no thread reads another's slot.
__device__ __forceinline__ void cp16(Vec8* dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
                 "l"(src), "r"(ok ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A block walks row tiles b, b + gridDim.x, ... in rounds of one head of U
// rows a group; the copies of the next LA rounds, running on from one tile
// into the next, are in flight while one is worked on.
template <typename T, int LPH, int U, int LA, bool TAIL>
__global__ void __launch_bounds__(kThreads, U == 1 ? 4 : kFwdBlocks)
    qk_forward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ __align__(16) uint8_t s_raw[];
    Vec8* slot = reinterpret_cast<Vec8*>(s_raw) + threadIdx.x;                     // [LA U][2][kThreads]
    float2* s_cs = reinterpret_cast<float2*>(s_raw + 2 * LA * U * kThreads * 16);  // [GR U][angle_pitch]
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t gh = g % a.GH, gr = g / a.GH, pitch = angle_pitch(a.rot);
    const uint32_t total = a.H + a.Hk + (a.v ? a.Hk : 0);
    const uint32_t h_begin = blockIdx.y * a.heads_per_block, h_end = min(total, h_begin + a.heads_per_block);
    const uint32_t rounds = (h_end - h_begin + a.GH - 1) / a.GH, R = a.GR * U;
    const bool lane0 = c * 8 < a.Dh, lane1 = (c + LPH) * 8 < a.Dh;
    uint32_t next_row0 = blockIdx.x * R, next_round = 0, next_slot = 0;  // what is requested next
    auto request = [&]() {
        if (next_row0 < a.rows) {
            const uint32_t h = h_begin + next_round * a.GH + gh;
            const bool is_q = h < a.H, is_v = h >= a.H + a.Hk;
            const uint32_t hk = is_q ? h : (is_v ? h - a.H - a.Hk : h - a.H);
            const T* src = reinterpret_cast<const T*>(is_q ? a.q : (is_v ? a.v : a.k)) + (uint64_t)hk * a.Dh + c * 8;
            const uint64_t step = is_q ? a.q_pitch : (is_v ? a.v_pitch : a.k_pitch);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t row = next_row0 + gr + u * a.GR;
                const bool ok = h < h_end && row < a.rows;
                const T* p = ok ? src + row * step : reinterpret_cast<const T*>(a.q);
                Vec8* s = slot + (next_slot * U + u) * 2 * kThreads;
                cp16(s, p, ok && lane0);
                cp16(s + kThreads, ok && lane1 ? p + LPH * 8 : p, ok && lane1);
            }
            if (++next_round == rounds) next_round = 0, next_row0 += gridDim.x * R;
            if (++next_slot == LA) next_slot = 0;
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < LA; ++i) request();
    uint32_t cur = 0;
    for (uint32_t row0 = blockIdx.x * R; row0 < a.rows; row0 += gridDim.x * R) {
        const uint32_t nrows = min(R, a.rows - row0);
        if (row0 != blockIdx.x * R) __syncthreads();  // the previous tile's angles have been read
        fill_angles(a, s_cs, row0, nrows);
        __syncthreads();
        for (uint32_t round = 0; round < rounds; ++round) {
            const uint32_t h = h_begin + round * a.GH + gh;
            const bool on = h < h_end, is_q = h < a.H, is_v = h >= a.H + a.Hk;
            const uint32_t hk = is_q ? h : (is_v ? h - a.H - a.Hk : h - a.H);
            float w[2][8];
            load_gain<T, LPH>(is_q ? a.gq : a.gk, c, a.Dh, w);
            T* dst = reinterpret_cast<T*>(is_q ? a.qo : (is_v ? a.vo : a.ko)) + (uint64_t)hk * a.Dh + c * 8;
            const uint64_t opitch = is_q ? a.qo_pitch : a.ko_pitch;
            cp_wait<LA - 1>();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t rl = gr + u * a.GR, row = row0 + rl;
                const Vec8* s = slot + (cur * U + u) * 2 * kThreads;
                const Vec8 raw0 = ld_shared_vec8(s), raw1 = ld_shared_vec8(s + kThreads);
                float f[2][8], ss = 0.0f;
                unpack8<T>(raw0, f[0]);
                unpack8<T>(raw1, f[1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += f[0][e] * f[0][e] + f[1][e] * f[1][e];
                const float r = rsqrtf(group_sum<LPH>(ss) * a.inv_dh + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[0][e] *= r * w[0][e];
                    f[1][e] *= r * w[1][e];
                }
                rotate<LPH, TAIL>(a, s_cs + min(rl, nrows - 1) * pitch, c, 1.0f, f);
                bool st = on && rl < nrows;
                uint64_t at = row;
                if (a.cache && !is_q && st) {
                    const int32_t pos = position(a, row);
                    st = pos >= 0 && (uint32_t)pos < a.cache_len;  // outside the cache: not stored
                    at = (uint64_t)(row / a.S) * a.cache_len + (uint32_t)pos;
                }
                T* p = dst + at * opitch;
                if (st && lane0) st_vec8(p, is_v ? raw0 : pack8<T>(f[0]));
                if (st && lane1) st_vec8(p + LPH * 8, is_v ? raw1 : pack8<T>(f[1]));
            }
            if (++cur == LA) cur = 0;
            request();
        }
    }
}

// The same walk.  Each lane adds its columns' gain gradients over all heads it
// meets, the block adds its groups in order and stores one partial row, and
// qk_gain_kernel adds the partials in order, so the sums do not depend on
// timing.
template <typename T, int LPH, int U, int LA, bool TAIL>
__global__ void __launch_bounds__(kThreads, kBwdBlocks) qk_backward_kernel(const __grid_constant__ QkArgs a) {
    extern __shared__ __align__(16) uint8_t s_raw[];
    Vec8* slot = reinterpret_cast<Vec8*>(s_raw) + threadIdx.x;  // [LA U][x, dy][2][kThreads]
    // [GR U][angle_pitch]; then, over all of it, the groups' sums [G][2][Dh]
    float2* s_cs = reinterpret_cast<float2*>(s_raw + 4 * LA * U * kThreads * 16);
    constexpr uint32_t G = kThreads / LPH;
    const uint32_t c = threadIdx.x % LPH, g = threadIdx.x / LPH;
    const uint32_t gh = g % a.GH, gr = g / a.GH, pitch = angle_pitch(a.rot);
    const uint32_t total = a.H + a.Hk, R = a.GR * U, rounds = (total + a.GH - 1) / a.GH;
    const bool lane0 = c * 8 < a.Dh, lane1 = (c + LPH) * 8 < a.Dh;
    float accq[2][8] = {}, acck[2][8] = {};
    if (a.partial) pdl_trigger();  // qk_gain_kernel, which waits for this one to end
    uint32_t next_row0 = blockIdx.x * R, next_round = 0, next_slot = 0;  // what is requested next
    auto request = [&]() {
        if (next_row0 < a.rows) {
            const uint32_t h = next_round * a.GH + gh;
            const bool is_q = h < a.H;
            const uint64_t col = (uint64_t)(is_q ? h : h - a.H) * a.Dh + c * 8;
            const T* x = reinterpret_cast<const T*>(is_q ? a.q : a.k) + col;
            const T* t = reinterpret_cast<const T*>(is_q ? a.dqo : a.dko) + col;
            const uint64_t xs = is_q ? a.q_pitch : a.k_pitch, ts = is_q ? a.dqo_pitch : a.dko_pitch;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t row = next_row0 + gr + u * a.GR;
                const bool ok = h < total && row < a.rows;
                const T* px = ok ? x + row * xs : reinterpret_cast<const T*>(a.q);
                const T* pt = ok ? t + row * ts : reinterpret_cast<const T*>(a.q);
                Vec8* s = slot + (next_slot * U + u) * 4 * kThreads;
                cp16(s, px, ok && lane0);
                cp16(s + kThreads, ok && lane1 ? px + LPH * 8 : px, ok && lane1);
                cp16(s + 2 * kThreads, pt, ok && lane0);
                cp16(s + 3 * kThreads, ok && lane1 ? pt + LPH * 8 : pt, ok && lane1);
            }
            if (++next_round == rounds) next_round = 0, next_row0 += gridDim.x * R;
            if (++next_slot == LA) next_slot = 0;
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < LA; ++i) request();
    uint32_t cur = 0;
    for (uint32_t row0 = blockIdx.x * R; row0 < a.rows; row0 += gridDim.x * R) {
        const uint32_t nrows = min(R, a.rows - row0);
        if (row0 != blockIdx.x * R) __syncthreads();  // the previous tile's angles have been read
        fill_angles(a, s_cs, row0, nrows);
        __syncthreads();
        for (uint32_t round = 0; round < rounds; ++round) {
            const uint32_t h = round * a.GH + gh;
            const bool on = h < total, is_q = h < a.H;
            float w[2][8], acc[2][8] = {};
            load_gain<T, LPH>(is_q ? a.gq : a.gk, c, a.Dh, w);
            T* dst = reinterpret_cast<T*>(is_q ? a.qo : a.ko) + (uint64_t)(is_q ? h : h - a.H) * a.Dh + c * 8;
            const uint64_t opitch = is_q ? a.qo_pitch : a.ko_pitch;
            cp_wait<LA - 1>();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t rl = gr + u * a.GR;
                const Vec8* s = slot + (cur * U + u) * 4 * kThreads;
                float x[2][8], t[2][8], ss = 0.0f, m = 0.0f;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    unpack8<T>(ld_shared_vec8(s + v * kThreads), x[v]);
                    unpack8<T>(ld_shared_vec8(s + (2 + v) * kThreads), t[v]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss += x[v][e] * x[v][e];
                }
                // A group without a head or row works on zeros: with eps = 0 its r would be infinite.
                const bool live = on && rl < nrows;
                const float ms = group_sum<LPH>(ss) * a.inv_dh + a.eps, r = live ? rsqrtf(ms) : 0.0f;
                rotate<LPH, TAIL>(a, s_cs + min(rl, nrows - 1) * pitch, c, -1.0f, t);
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[v][e] *= r;  // n
                        acc[v][e] += t[v][e] * x[v][e];
                        t[v][e] *= w[v][e];  // dn
                        m += t[v][e] * x[v][e];
                    }
                m = group_sum<LPH>(m) * a.inv_dh;
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[v][e] = r * (t[v][e] - x[v][e] * m);
                T* p = dst + (row0 + rl) * opitch;
                if (live && lane0) st_vec8(p, pack8<T>(t[0]));
                if (live && lane1) st_vec8(p + LPH * 8, pack8<T>(t[1]));
            }
            if (++cur == LA) cur = 0;
            request();
            if (!a.partial) continue;
#pragma unroll
            for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (is_q) accq[v][e] += acc[v][e];
                    else acck[v][e] += acc[v][e];
                }
        }
    }
    if (!a.partial) return;
    cp_wait<0>();
    float* sums = reinterpret_cast<float*>(s_raw);
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        if (v ? !lane1 : !lane0) continue;
        float* p = sums + g * 2 * a.Dh + (c + v * LPH) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = accq[v][e];
            p[a.Dh + e] = acck[v][e];
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

uint32_t lanes_per_head(uint32_t Dh) { return Dh <= 32 ? 2 : Dh <= 64 ? 4 : Dh <= 128 ? 8 : 16; }

// Calls f with the lanes-per-head constant of head size Dh.
template <class F>
int with_lph(uint32_t Dh, F&& f) {
    switch (lanes_per_head(Dh)) {
        case 2: return f(std::integral_constant<int, 2>());
        case 4: return f(std::integral_constant<int, 4>());
        case 8: return f(std::integral_constant<int, 8>());
        default: return f(std::integral_constant<int, 16>());
    }
}

// The same with whether the rotated part ends inside a vector of eight.
template <class F>
int with_layout(const QkArgs& a, F&& f) {
    return with_lph(a.Dh, [&](auto lph) {
        if (a.rot % 8 != 0) return f(lph, std::true_type());
        return f(lph, std::false_type());
    });
}

// Heads x rows of a block's groups: the most heads that leave under a
// sixteenth of the groups without one (40 heads, 32 groups: 8 x 4).
void set_groups(QkArgs& a, uint32_t total) {
    const uint32_t G = kThreads / lanes_per_head(a.Dh);
    for (a.GH = G; a.GH > 1; a.GH /= 2)
        if (total * 16 >= (total + a.GH - 1) / a.GH * a.GH * 15) break;
    a.GR = G / a.GH;
}

bool pitch_ok(uint64_t pitch, uint64_t cols) { return pitch >= cols && pitch % 8 == 0 && pitch <= (1ull << 40); }

int check_desc(const char* op, const evkcu_qk_norm_rope_desc* d, uint32_t allowed, int dtype) {
    EVKCU_CHECK_ARG(d, EVKCU_BAD_ARG, std::string(op) + ": descriptor is null");
    EVKCU_CHECK_ARG(dtype == EVKCU_F16 || dtype == EVKCU_BF16, EVKCU_BAD_ARG, std::string(op) + ": unknown dtype");
    EVKCU_CHECK_ARG((d->flags & ~allowed) == 0, EVKCU_BAD_ARG, std::string(op) + ": unknown flag");
    EVKCU_CHECK_ARG(d->head_dim >= 8 && d->head_dim <= 256 && d->head_dim % 8 == 0, EVKCU_BAD_SHAPE,
                    std::string(op) + ": head_dim must be a multiple of 8, 8 to 256");
    const uint32_t step = (d->flags & EVKCU_QK_HALF_SPLIT) ? 16 : 2;
    EVKCU_CHECK_ARG(d->rot_dim <= d->head_dim && (d->rot_dim ? d->rot_dim : d->head_dim) % step == 0, EVKCU_BAD_SHAPE,
                    std::string(op) +
                        ": rot_dim must be at most head_dim and a multiple of 2 (of 16 for half-split pairs)");
    EVKCU_CHECK_ARG(d->heads > 0 && d->heads <= 65535 && d->kv_heads <= 65535, EVKCU_BAD_SHAPE,
                    std::string(op) + ": heads must be 1 to 65535, kv_heads at most 65535");
    EVKCU_CHECK_ARG((uint64_t)d->batch * d->seq_len <= (1ull << 30), EVKCU_BAD_SHAPE,
                    std::string(op) + ": more than 2^30 rows");
    EVKCU_CHECK_ARG(d->positions || (uint64_t)d->pos_offset + d->seq_len <= (1ull << 31), EVKCU_BAD_SHAPE,
                    std::string(op) + ": positions above 2^31 - 1");
    EVKCU_CHECK_ARG(std::isfinite(d->base) && d->base > 0.0f && d->eps >= 0.0f, EVKCU_BAD_ARG,
                    std::string(op) + ": base must be positive and eps not negative");
    EVKCU_CHECK_ARG((reinterpret_cast<uintptr_t>(d->positions) & 3u) == 0, EVKCU_BAD_ALIGN,
                    std::string(op) + ": positions must be 4-byte aligned");
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
    EVKCU_CHECK_ARG((v == nullptr) == (v_out == nullptr), EVKCU_BAD_ARG,
                    std::string(op) + ": v and v_out come together");
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
        return with_layout(a, [&](auto lph, auto tail) {
            const uint32_t R = a.GR * (large ? kFwdRows : 1), tiles = (a.rows + R - 1) / R;
            const size_t smem = 2 * (large ? kFwdRows * kFwdAhead : 1) * kThreads * 16 +
                                R * angle_pitch(a.rot) * sizeof(float2);
            auto kern = large ? qk_forward_kernel<T, lph.value, kFwdRows, kFwdAhead, tail.value>
                              : qk_forward_kernel<T, lph.value, 1, 1, tail.value>;
            static std::atomic<uint64_t> done[2];
            EVKCU_TRY(allow_smem(kern, kMaxSmem, done[large]));
            const dim3 grid(large ? std::min(tiles, kFwdBlocks * (uint32_t)ds->sm_count) : tiles,
                            large ? 1 : (uint32_t)rounds);
            kern<<<grid, kThreads, smem, as_stream(stream)>>>(a);
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
                        std::string(op) +
                            ": the gain gradients need a workspace of evkcu_qk_norm_rope_workspace bytes");
        EVKCU_CHECK_ARG(aligned16(workspace), EVKCU_BAD_ALIGN, std::string(op) + ": workspace must be 16-byte aligned");
    }
    const uint64_t rows = (uint64_t)d->batch * d->seq_len, dh = d->head_dim;
    const uint64_t wse = gains ? 4 * kMaxPartials * dh : 0;
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
        return with_layout(a, [&](auto lph, auto tail) {
            constexpr uint32_t U = kBwdRows;
            const uint32_t R = a.GR * U, tiles = (a.rows + R - 1) / R;
            // resident at once
            const uint32_t grid = std::min({tiles, kMaxPartials, kBwdBlocks * (uint32_t)ds->sm_count});
            const size_t smem = std::max<size_t>(4 * U * kBwdAhead * kThreads * 16 +
                                                     R * angle_pitch(a.rot) * sizeof(float2),
                                                 gains ? (size_t)(kThreads / lph.value) * 2 * a.Dh * sizeof(float) : 0);
            auto kern = qk_backward_kernel<T, lph.value, U, kBwdAhead, tail.value>;
            static std::atomic<uint64_t> done{0};
            EVKCU_TRY(allow_smem(kern, kMaxSmem, done));
            kern<<<grid, kThreads, smem, st>>>(a);
            EVKCU_TRY(after_launch("evkcu_qk_norm_rope_backward"));
            if (!gains) return (int)EVKCU_OK;
            return launch_pdl("evkcu_qk_norm_rope_backward(gains)", qk_gain_kernel<T>, dim3((2 * a.Dh + 31) / 32),
                              dim3(1024), 0, st, (const float*)a.partial, grid, a.Dh, (T*)dgain_q, (T*)dgain_k,
                              (int)acc);
        });
    });
}
