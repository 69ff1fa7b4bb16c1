// linear.cuh — what the linear / gated feed-forward kernels share: the
// activations and their derivatives, and the epilogues that turn fp32
// accumulators into outputs.
#pragma once

#include <atomic>
#include <initializer_list>
#include <string>

#include "common.cuh"

#define EVKCU_TRY(expr)                 \
    do {                                \
        if (int _r = (expr)) return _r; \
    } while (0)

namespace evkcu {

// ------------------------------------------------------ argument checks ----
// A 2-byte matrix argument: `rows` rows of `cols` elements, `pitch` elements
// apart.  An output may be exactly the buffer of the span named
// `same_as` or `same_as2` (its kernel reads each element before it writes it).
struct Span {
    const char* name;
    const void* p;
    uint64_t rows, pitch, cols;
    bool out = false;
    const char* same_as = nullptr;
    const char* same_as2 = nullptr;
};
inline bool same_name(const char* a, const char* b) {
    while (*a && *a == *b) ++a, ++b;
    return *a == *b;
}

inline bool spans_overlap(const Span& a, const Span& b) {
    if (a.rows == 0 || b.rows == 0 || a.cols == 0 || b.cols == 0) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uint64_t ea = 2 * ((a.rows - 1) * a.pitch + a.cols), eb = 2 * ((b.rows - 1) * b.pitch + b.cols);
    if (pa + ea <= pb || pb + eb <= pa) return false;
    if (a.pitch != b.pitch) return true;
    // Rows of one pitch interleave: column ranges side by side do not meet.
    const uint64_t w = 2 * a.pitch, d = pb >= pa ? (pb - pa) % w : (w - (pa - pb) % w) % w;
    return d < 2 * a.cols || d + 2 * b.cols > w;
}

// Refuses an output that shares memory with another argument.
inline int check_spans(const char* op, std::initializer_list<Span> spans) {
    for (const Span* a = spans.begin(); a != spans.end(); ++a)
        for (const Span* b = spans.begin(); b != spans.end(); ++b) {
            if (a == b || !a->out || !a->p || !b->p || (b->out && b < a)) continue;
            const bool named = (a->same_as && same_name(a->same_as, b->name)) ||
                               (a->same_as2 && same_name(a->same_as2, b->name));
            if (named && a->p == b->p && a->pitch == b->pitch) continue;
            if (spans_overlap(*a, *b))
                return fail(EVKCU_BAD_ARG, std::string(op) + ": " + a->name + " overlaps " + b->name);
        }
    return EVKCU_OK;
}

// Sets a kernel's shared-memory limit once per device.
template <class K>
int allow_smem(K* kern, int bytes, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (state()->device & 63);
    if (done.load(std::memory_order_relaxed) & bit) return EVKCU_OK;
    EVKCU_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return EVKCU_OK;
}

inline int check_ptr(const char* op, const char* name, const void* p, bool required) {
    EVKCU_CHECK_ARG(p || !required, EVKCU_BAD_ARG, std::string(op) + ": " + name + " is null");
    EVKCU_CHECK_ARG(aligned16(p), EVKCU_BAD_ALIGN, std::string(op) + ": " + name + " must be 16-byte aligned");
    return EVKCU_OK;
}

// 1 / (1 + 2^(-z log2 e)) from ex2 and a reciprocal, both sides of the quotient
// scaled by 2^-16: unscaled, the exponential and its reciprocal leave fp32 below
// z = -87, where z sigmoid(z) = -1e-36 is still a normal bf16 value; scaled, only
// past z = -98, where it is below half of bf16's smallest step.  Relative error at
// most (9 + 0.6 |z|) 2^-23: the scaled exponent's rounding (half a step at 16, and
// what log2 e and the product leave), 2 units of ex2 and 1 of the reciprocal.  So
// the activations below are exact to well under a 2-byte rounding.
__device__ __forceinline__ float sigmoid_f(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(z, -1.4426950408889634f, -16.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 0x1p-16f));
    return 0x1p-16f * r;
}

constexpr float kGeluA = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

// tanh-form GELU as z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3): the
// same function as 0.5 z (1 + tanh u), without its cancellation for z < 0
// (tanh.approx there is off by more than half a step of fp16).
__device__ __forceinline__ float act_f(float z, int act) {
    switch (act) {
        case EVKCU_ACT_RELU: return z > 0.0f ? z : (z <= 0.0f ? 0.0f : z);  // NaN stays
        case EVKCU_ACT_GELU: return z * sigmoid_f(kGeluA * (z + kGeluB * z * z * z));
        case EVKCU_ACT_SILU: return z * sigmoid_f(z);
        default: return z;
    }
}

// act(z) and d act / d z together.
__device__ __forceinline__ void act_both(float z, int act, float& a, float& da) {
    switch (act) {
        case EVKCU_ACT_RELU:
            a = z > 0.0f ? z : (z <= 0.0f ? 0.0f : z);
            da = z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
            return;
        case EVKCU_ACT_GELU: {
            const float s = sigmoid_f(kGeluA * (z + kGeluB * z * z * z));
            a = z * s;
            // Past |z| = 30 s is exactly 0 or 1; z^2 may overflow there.
            da = z > 30.0f ? 1.0f
                           : (z < -30.0f ? 0.0f : s + z * s * (1.0f - s) * kGeluA * (1.0f + 3.0f * kGeluB * z * z));
            return;
        }
        case EVKCU_ACT_SILU: {
            const float s = sigmoid_f(z);
            a = z * s;
            da = s + a * (1.0f - s);
            return;
        }
        default: a = z; da = 1.0f;
    }
}

template <int ACT>
__device__ __forceinline__ float dact_of(float z) {
    float a, da;
    act_both(z, ACT, a, da);
    return da;
}

// All values of a chunk at once, the activation chosen outside the loop: a
// branch per value costs more in instruction fetches than the function.
template <int N>
__device__ __forceinline__ void act_all(float (&f)[N], int act) {
    if (act == EVKCU_ACT_NONE) return;
    if (act == EVKCU_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = act_f(f[e], EVKCU_ACT_SILU);
    } else if (act == EVKCU_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = act_f(f[e], EVKCU_ACT_GELU);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = act_f(f[e], EVKCU_ACT_RELU);
    }
}

// f *= act'(z)
template <int N>
__device__ __forceinline__ void dact_all(float (&f)[N], const float (&z)[N], int act) {
    if (act == EVKCU_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= dact_of<EVKCU_ACT_SILU>(z[e]);
    } else if (act == EVKCU_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= dact_of<EVKCU_ACT_GELU>(z[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] *= dact_of<EVKCU_ACT_RELU>(z[e]);
    }
}

// dg = dh u act'(g), du = dh act(g), h = act(g) u
template <int ACT>
__device__ __forceinline__ void gated_bwd8_of(const float (&dh)[8], const float (&g)[8], const float (&u)[8],
                                              float (&dg)[8], float (&du)[8], float (&h)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float a, da;
        act_both(g[e], ACT, a, da);
        dg[e] = dh[e] * u[e] * da;
        du[e] = dh[e] * a;
        h[e] = a * u[e];
    }
}
__device__ __forceinline__ void gated_bwd8(const float (&dh)[8], const float (&g)[8], const float (&u)[8],
                                           float (&dg)[8], float (&du)[8], float (&h)[8], int act) {
    if (act == EVKCU_ACT_SILU) gated_bwd8_of<EVKCU_ACT_SILU>(dh, g, u, dg, du, h);
    else if (act == EVKCU_ACT_GELU) gated_bwd8_of<EVKCU_ACT_GELU>(dh, g, u, dg, du, h);
    else if (act == EVKCU_ACT_RELU) gated_bwd8_of<EVKCU_ACT_RELU>(dh, g, u, dg, du, h);
    else gated_bwd8_of<EVKCU_ACT_NONE>(dh, g, u, dg, du, h);
}

__device__ __forceinline__ Vec8 ld_vec8(const void* p) { return *reinterpret_cast<const Vec8*>(p); }
__device__ __forceinline__ void st_vec8(void* p, const Vec8& v) { *reinterpret_cast<Vec8*>(p) = v; }

// ------------------------------------------------------------- epilogues ----
// Each is called with eight consecutive output columns of one row; col and
// every row pitch are multiples of 8 elements.  A thread reads all it needs
// of those elements before it writes them, so an output may be the buffer of
// the input with the same index (y = residual, dpre = pre).

// z = acc (+ bias); pre = z; y = act(z) (+ residual)
template <typename T>
struct EpiLinear {
    static constexpr bool kGated = false;
    const T* bias;
    const T* res;
    T* y;
    T* pre;
    uint32_t N;
    int act;
    __device__ __forceinline__ void operator()(uint32_t row, uint32_t col, float (&f)[8], float (&)[8]) const {
        const uint64_t at = (uint64_t)row * N + col;
        float t[8];
        if (bias) {
            unpack8<T>(ld_vec8(bias + col), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += t[e];
        }
        if (pre) st_vec8(pre + at, pack8<T>(f));
        act_all(f, act);
        if (res) {
            unpack8<T>(ld_vec8(res + at), t);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += t[e];
        }
        st_vec8(y + at, pack8<T>(f));
    }
};

// pre = [g | u]; h = act(g) u, with g and u unrounded
template <typename T>
struct EpiGated {
    static constexpr bool kGated = true;
    T* h;
    T* pre;
    uint32_t F;
    int act;
    __device__ __forceinline__ void operator()(uint32_t row, uint32_t col, float (&g)[8], float (&u)[8]) const {
        if (pre) {
            T* p = pre + (uint64_t)row * (2 * (uint64_t)F) + col;
            st_vec8(p, pack8<T>(g));
            st_vec8(p + F, pack8<T>(u));
        }
        act_all(g, act);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= u[e];
        st_vec8(h + (uint64_t)row * F + col, pack8<T>(g));
    }
};

// From dh (the accumulator, never rounded) and the saved g, u:
// dpre = [dh u act'(g) | dh act(g)]; h = act(g) u again.
template <typename T>
struct EpiGatedBwd {
    static constexpr bool kGated = false;
    const T* pre;
    T* dpre;
    T* h;
    uint32_t F;
    int act;
    __device__ __forceinline__ void operator()(uint32_t row, uint32_t col, float (&dh)[8], float (&)[8]) const {
        const uint64_t at = (uint64_t)row * (2 * (uint64_t)F) + col;
        float g[8], u[8], dg[8], du[8], hh[8];
        unpack8<T>(ld_vec8(pre + at), g);
        unpack8<T>(ld_vec8(pre + at + F), u);
        gated_bwd8(dh, g, u, dg, du, hh, act);
        st_vec8(dpre + at, pack8<T>(dg));
        st_vec8(dpre + at + F, pack8<T>(du));
        if (h) st_vec8(h + (uint64_t)row * F + col, pack8<T>(hh));
    }
};

}  // namespace evkcu
