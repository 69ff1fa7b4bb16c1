// evk_ai_ext.cpp — the extensions of evk_ai_ext.h over the C ABI, through the
// same shape logic (evk_ai_dispatch.h) and backend table as evk_ai.cpp.
#include "evk_ai_ext.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "evk_ai_dispatch.h"
#include "evkcu.h"

namespace evk_b200 {
const Backend& cpp_backend();  // evk_ai.cpp
}

namespace evk::ai {
namespace {
const evk_b200::Backend& be() { return evk_b200::cpp_backend(); }
int dt(DType d) { return static_cast<int>(d); }
}  // namespace

void matmul_ex(Tensor& a, Tensor& b, Tensor& c, bool ta, bool tb, bool acc, DType d) {
    evk_b200::matmul(be(), a, b, c, ta, tb, acc, dt(d));
}
void add_ex(Tensor& a, Tensor& b, Tensor& c, DType d) { evk_b200::add(be(), a, b, c, dt(d)); }
void gelu_ex(Tensor& in, Tensor& out, DType d) { evk_b200::gelu(be(), in, out, dt(d)); }
void softmax_ex(Tensor& in, Tensor& out, float s, DType d) { evk_b200::softmax(be(), in, out, s, dt(d)); }

void flash_attention_ex(Tensor& q, Tensor& k, Tensor& v, Tensor& o, uint32_t heads, bool causal, float scale,
                        DType d) {
    if (q.shape.rank() != 3 || k.shape.rank() != 3 || heads == 0 || q.shape[2] % heads != 0)
        return be().fail(EVKCU_BAD_SHAPE, "flash_attention_ex: shapes");
    const uint32_t B = q.shape[0], N = q.shape[1], Dh = q.shape[2] / heads;
    if (k.shape[2] % Dh != 0 || k.shape[0] != B || k.shape[1] != N || !evk_b200::same_shape(k, v) ||
        !evk_b200::same_shape(q, o))
        return be().fail(EVKCU_BAD_SHAPE, "flash_attention_ex: incompatible shapes");
    evk_b200::check(be(),
                    be().flash_attention(evk_b200::dptr(q), evk_b200::dptr(k), evk_b200::dptr(v), evk_b200::dmut(o), B,
                                         N, heads, k.shape[2] / Dh, Dh, scale, causal ? EVKCU_ATTN_CAUSAL : 0u, dt(d),
                                         be().stream()),
                    "flash_attention_ex");
}

void single_query_attention(Tensor& q, Tensor& kc, Tensor& vc, Tensor& out, uint32_t heads, uint32_t cur_len,
                            float scale, DType d) {
    if (q.shape.rank() < 2 || kc.shape.rank() != 3 || heads == 0 || q.shape[-1] % heads != 0)
        return be().fail(EVKCU_BAD_SHAPE, "single_query_attention: shapes");
    const uint32_t B = kc.shape[0], max_len = kc.shape[1], Dh = q.shape[-1] / heads;
    if (kc.shape[2] % Dh != 0 || !evk_b200::same_shape(kc, vc) || q.shape.count() != B * heads * Dh ||
        out.shape.count() != q.shape.count() || cur_len > max_len)
        return be().fail(EVKCU_BAD_SHAPE, "single_query_attention: incompatible shapes");
    evk_b200::check(be(),
                    be().single_query_attention(evk_b200::dptr(q), evk_b200::dptr(kc), evk_b200::dptr(vc),
                                                evk_b200::dmut(out), B, heads, kc.shape[2] / Dh, Dh, max_len, cur_len,
                                                scale, dt(d), be().stream()),
                    "single_query_attention");
}

void rope_ex(Tensor& in, Tensor& out, uint32_t B, uint32_t S, uint32_t D, float base, uint32_t head_dim,
             uint32_t pos_offset, DType d) {
    evk_b200::rope(be(), in, out, B, S, D, base, head_dim, pos_offset, dt(d));
}

void rms_norm_ex(Tensor& in, Tensor& out, float eps, Tensor* gamma, DType d) {
    if (gamma && gamma->shape.count() != in.shape[-1]) return be().fail(EVKCU_BAD_SHAPE, "rms_norm_ex: gamma size");
    evk_b200::rms_norm(be(), in, out, eps, gamma ? evk_b200::dptr(*gamma) : nullptr, dt(d));
}

void embed_ex(Tensor& E, Tensor& idx, Tensor& out, uint32_t id_bytes, DType d) {
    if (id_bytes != 2 && id_bytes != 4) return be().fail(EVKCU_BAD_ARG, "embed_ex: id_bytes");
    evk_b200::embed(be(), E, idx, out, id_bytes, dt(d));
}

void greedy_sample_ex(Tensor& logits, Tensor& out, uint32_t position, uint32_t base, uint32_t count, uint32_t id_bytes,
                      DType d) {
    if (id_bytes != 2 && id_bytes != 4) return be().fail(EVKCU_BAD_ARG, "greedy_sample_ex: id_bytes");
    evk_b200::greedy_sample(be(), logits, out, position, base, count, id_bytes, dt(d));
}

// ---- decoder-layer operators around attention -------------------------------
namespace {

using evk_b200::dmut;
using evk_b200::dptr;

const void* opt(Tensor* t) { return t ? dptr(*t) : nullptr; }
void* opt_mut(Tensor* t) { return t ? dmut(*t) : nullptr; }
// Elements of t, 2^32 for all that do not fit 32 bits: Shape::count(), by which
// buffers are allocated, keeps only those.
uint64_t count(Tensor& t) {
    uint64_t n = 1;
    for (uint32_t i = 0; i < t.shape.rank(); ++i) n = std::min(n * t.shape[(int)i], uint64_t(1) << 32);
    return n;
}
bool fits(Tensor& t) { return count(t) >> 32 == 0; }
// Rows of t's last dimension (0 where that is 0).
uint64_t rows_of(Tensor& t) { return t.shape[-1] ? count(t) / t.shape[-1] : 0; }
// Every optional tensor that is given holds n elements.
bool sized(uint64_t n, std::initializer_list<Tensor*> ts) {
    for (Tensor* t : ts)
        if (t && (!fits(*t) || count(*t) != n)) return false;
    return true;
}
bool is_matrix(Tensor& t, uint64_t rows, uint64_t cols, bool transposed) {
    if (t.shape.rank() != 2 || !fits(t)) return false;
    return t.shape[0] == (transposed ? cols : rows) && t.shape[1] == (transposed ? rows : cols);
}

}  // namespace

void linear(Tensor& x, Tensor& w, Tensor& y, Tensor* bias, Tensor* residual, Act act, Tensor* pre, bool transpose_w,
            DType d) {
    const uint64_t K = x.shape[-1], N = y.shape[-1], rows = rows_of(x);
    if (K == 0 || !fits(x) || !is_matrix(w, K, N, transpose_w) || !sized(rows * N, {&y, residual, pre}) ||
        !sized(N, {bias}))
        return be().fail(EVKCU_BAD_SHAPE, "linear: incompatible shapes");
    evk_b200::check(be(),
                    evkcu_linear(dptr(x), dptr(w), opt(bias), opt(residual), dmut(y), opt_mut(pre), (uint32_t)rows,
                                 (uint32_t)K, (uint32_t)N, (int)act, transpose_w ? EVKCU_MM_TRANSPOSE_B : 0u, dt(d),
                                 be().stream()),
                    "linear");
}

void linear_backward(Tensor& x, Tensor& w, Tensor& dy, Tensor* dx, Tensor* dw, Tensor* dbias, Act act, Tensor* pre,
                     Tensor* dpre, bool transpose_w, bool acc, DType d) {
    const uint64_t K = x.shape[-1], N = dy.shape[-1], rows = rows_of(x);
    if (K == 0 || !fits(x) || !is_matrix(w, K, N, transpose_w) || (dw && !is_matrix(*dw, K, N, transpose_w)) ||
        !sized(rows * N, {&dy, pre, dpre}) || !sized(count(x), {dx}) || !sized(N, {dbias}))
        return be().fail(EVKCU_BAD_SHAPE, "linear_backward: incompatible shapes");
    const uint32_t flags = (transpose_w ? EVKCU_MM_TRANSPOSE_B : 0u) | (acc ? EVKCU_MM_ACC_C : 0u);
    evk_b200::check(be(),
                    evkcu_linear_backward(dptr(x), dptr(w), opt(pre), dptr(dy), opt_mut(dpre), opt_mut(dx), opt_mut(dw),
                                          opt_mut(dbias), (uint32_t)rows, (uint32_t)K, (uint32_t)N, (int)act, flags,
                                          dt(d), be().stream()),
                    "linear_backward");
}

void gated_ffn(Tensor& x, Tensor& w_in, Tensor& w_out, Tensor& y, Tensor& hidden, Act act, Tensor* residual,
               Tensor* pre, bool transpose_w, DType d) {
    const uint64_t D = x.shape[-1], F = hidden.shape[-1], rows = rows_of(x);
    if (D == 0 || !fits(x) || !is_matrix(w_in, D, 2 * F, transpose_w) || !is_matrix(w_out, F, D, transpose_w) ||
        !sized(rows * D, {&y, residual}) || !sized(rows * F, {&hidden}) || !sized(2 * rows * F, {pre}))
        return be().fail(EVKCU_BAD_SHAPE, "gated_ffn: incompatible shapes");
    evk_b200::check(be(),
                    evkcu_gated_ffn(dptr(x), dptr(w_in), dptr(w_out), opt(residual), dmut(y), dmut(hidden),
                                    opt_mut(pre), (uint32_t)rows, (uint32_t)D, (uint32_t)F, (int)act,
                                    transpose_w ? EVKCU_MM_TRANSPOSE_B : 0u, dt(d), be().stream()),
                    "gated_ffn");
}

void gated_ffn_backward(Tensor& x, Tensor& w_in, Tensor& w_out, Tensor& pre, Tensor& dy, Tensor& dpre, Tensor& hidden,
                        Tensor* dx, Tensor* dw_in, Tensor* dw_out, Act act, bool transpose_w, bool acc, DType d) {
    const uint64_t D = x.shape[-1], F = hidden.shape[-1], rows = rows_of(x);
    if (D == 0 || !fits(x) || !is_matrix(w_in, D, 2 * F, transpose_w) || !is_matrix(w_out, F, D, transpose_w) ||
        (dw_in && !is_matrix(*dw_in, D, 2 * F, transpose_w)) || (dw_out && !is_matrix(*dw_out, F, D, transpose_w)) ||
        !sized(rows * D, {&dy, dx}) || !sized(rows * F, {&hidden}) || !sized(2 * rows * F, {&pre, &dpre}))
        return be().fail(EVKCU_BAD_SHAPE, "gated_ffn_backward: incompatible shapes");
    const uint32_t flags = (transpose_w ? EVKCU_MM_TRANSPOSE_B : 0u) | (acc ? EVKCU_MM_ACC_C : 0u);
    evk_b200::check(be(),
                    evkcu_gated_ffn_backward(dptr(x), dptr(w_in), dptr(w_out), dptr(pre), dptr(dy), dmut(dpre),
                                             dmut(hidden), opt_mut(dx), opt_mut(dw_in), opt_mut(dw_out),
                                             (uint32_t)rows, (uint32_t)D, (uint32_t)F, (int)act, flags, dt(d),
                                             be().stream()),
                    "gated_ffn_backward");
}

namespace {
// The descriptor of a fused qkv (B, S, (heads + 2 Hkv) Dh) with q (B, S,
// heads Dh); false when the shapes do not fit.
bool qk_desc(evkcu_qk_norm_rope_desc& d, Tensor& qkv, Tensor& q, Tensor& k, Tensor* gain_q, Tensor* gain_k,
             const QkRope& r) {
    if (qkv.shape.rank() != 3 || q.shape.rank() != 3 || k.shape.rank() != 3 || r.heads == 0 ||
        q.shape[2] % r.heads != 0 || q.shape[0] != qkv.shape[0] || q.shape[1] != qkv.shape[1] ||
        k.shape[0] != qkv.shape[0] || qkv.shape[2] != q.shape[2] + 2 * (uint64_t)k.shape[2] || !fits(qkv) ||
        !fits(q) || !fits(k))
        return false;
    const uint32_t Dh = q.shape[2] / r.heads;
    if (Dh == 0 || k.shape[2] % Dh != 0 || !sized(Dh, {gain_q, gain_k})) return false;
    d = {};
    d.batch = qkv.shape[0], d.seq_len = qkv.shape[1], d.heads = r.heads, d.kv_heads = k.shape[2] / Dh;
    d.head_dim = Dh, d.rot_dim = r.rot_dim, d.flags = r.half_split ? EVKCU_QK_HALF_SPLIT : 0u;
    d.pos_offset = r.pos_offset, d.eps = r.eps, d.base = r.base;
    d.q_pitch = d.k_pitch = d.v_pitch = d.dq_pitch = d.dk_pitch = qkv.shape[2];
    d.q_out_pitch = q.shape[2], d.k_out_pitch = k.shape[2];
    return true;
}
template <class P>
P* part(P* base, uint64_t elems) {  // an element offset into 2-byte storage
    return reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(base) + 2 * elems);
}
}  // namespace

void qk_norm_rope(Tensor& qkv, Tensor& q, Tensor& k, Tensor& v, Tensor* gain_q, Tensor* gain_k, const QkRope& rope,
                  bool cached, DType d) {
    evkcu_qk_norm_rope_desc desc;
    if (!qk_desc(desc, qkv, q, k, gain_q, gain_k, rope) || !evk_b200::same_shape(k, v) ||
        (!cached && k.shape[1] != qkv.shape[1]))
        return be().fail(EVKCU_BAD_SHAPE, "qk_norm_rope: incompatible shapes");
    if (cached) {
        desc.flags |= EVKCU_QK_CACHE;
        desc.cache_len = k.shape[1];
    }
    const void* in = dptr(qkv);
    evk_b200::check(be(),
                    evkcu_qk_norm_rope(&desc, in, part(in, q.shape[2]), part(in, q.shape[2] + k.shape[2]), opt(gain_q),
                                       opt(gain_k), dmut(q), dmut(k), dmut(v), dt(d), be().stream()),
                    "qk_norm_rope");
}

void qk_norm_rope_backward(Tensor& qkv, Tensor& dq, Tensor& dk, Tensor& dqkv, Tensor* gain_q, Tensor* gain_k,
                           Tensor* dgain_q, Tensor* dgain_k, Tensor* workspace, const QkRope& rope, DType d) {
    evkcu_qk_norm_rope_desc desc;
    if (!qk_desc(desc, qkv, dq, dk, gain_q, gain_k, rope) || !evk_b200::same_shape(qkv, dqkv) ||
        dk.shape[1] != qkv.shape[1] || !sized(desc.head_dim, {dgain_q, dgain_k}) || (workspace && !fits(*workspace)))
        return be().fail(EVKCU_BAD_SHAPE, "qk_norm_rope_backward: incompatible shapes");
    const void* in = dptr(qkv);
    void* out = dmut(dqkv);
    evk_b200::check(be(),
                    evkcu_qk_norm_rope_backward(&desc, in, part(in, dq.shape[2]), opt(gain_q), opt(gain_k), dptr(dq),
                                                dptr(dk), out, part(out, dq.shape[2]), opt_mut(dgain_q),
                                                opt_mut(dgain_k), opt_mut(workspace),
                                                workspace ? 2 * count(*workspace) : 0, dt(d), be().stream()),
                    "qk_norm_rope_backward");
}

uint64_t qk_norm_rope_workspace(uint32_t head_dim) { return evkcu_qk_norm_rope_workspace(head_dim); }

}  // namespace evk::ai
