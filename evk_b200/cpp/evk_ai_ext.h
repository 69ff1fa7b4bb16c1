// evk_ai_ext.h — additive extensions of the evk::ai operator API for the
// B200 backend.  Nothing here changes a reference signature; each function
// is a new entry point beside its reference counterpart (evk_ai.h:489-615)
// and calls the same C ABI (include/evkcu.h).
//
//   DType            tensors are 2-byte storage; fp16 as in the reference, or
//                    bf16 for the LLM configurations.
//   *_ex             the reference operator plus the parameters it lacks:
//                    grouped-query / causal attention, RoPE per head with a
//                    position offset (decode), RMSNorm with a gain, 32-bit
//                    token ids and counts (vocabularies above 65,535).
//   single_query_attention  host wrapper of the decode-attention shader,
//                    which the reference ships without one
//                    (shaders/single_query_attention.comp:27-71), generalised
//                    to batches, heads and long KV caches.
#pragma once

#include "evk_ai.h"

namespace evk::ai {

enum class DType : int { F16 = 0, BF16 = 1 };

// c = op(a) op(b) (+ c), as matmul (evk_ai.h:495), in the given storage type.
void matmul_ex(Tensor& a, Tensor& b, Tensor& c, bool transpose_a, bool transpose_b, bool acc_c, DType dtype);
void add_ex(Tensor& a, Tensor& b, Tensor& c, DType dtype);
void gelu_ex(Tensor& in, Tensor& out, DType dtype);
void softmax_ex(Tensor& in, Tensor& out, float input_scale, DType dtype);

// Attention O = softmax(Q K^T scale) V with Q, O (B, N, heads * Dh) and K, V
// (B, N, Hkv * Dh), Dh = Q.shape[2] / heads, Hkv = K.shape[2] / Dh (1 is the
// reference's multi-query call; heads is multi-head); causal masks keys
// after the query; scale <= 0 means 1 / sqrt(Dh).
void flash_attention_ex(Tensor& q, Tensor& k, Tensor& v, Tensor& o, uint32_t heads, bool causal, float scale = 0.0f,
                        DType dtype = DType::F16);

// Decode attention for one new query per sequence over a KV cache:
// q, out (B, heads * Dh); kcache, vcache (B, max_len, Hkv * Dh) of which the
// first cur_len positions are used.
void single_query_attention(Tensor& q, Tensor& kcache, Tensor& vcache, Tensor& out, uint32_t heads, uint32_t cur_len,
                            float scale = 0.0f, DType dtype = DType::F16);

// rope (evk_ai.h:587-591) rotating each head_dim slice of the last dimension
// (0 = the whole dimension, as the reference) at positions pos_offset + t.
void rope_ex(Tensor& input, Tensor& out, uint32_t batch_size, uint32_t seq_len, uint32_t embed_dim, float rotary_base,
             uint32_t head_dim, uint32_t pos_offset, DType dtype = DType::F16);

// rms_norm (evk_ai.h:607-610) followed by a per-column gain (gamma: (D), or
// nullptr for none).
void rms_norm_ex(Tensor& input, Tensor& output, float eps, Tensor* gamma, DType dtype = DType::F16);

// embed / greedy_sample with 2- or 4-byte token ids (id_bytes) and 32-bit
// token_base / token_count.  With 4-byte ids, `indices` / `out_tokens` hold
// two 2-byte slots per id.
void embed_ex(Tensor& embeddings, Tensor& indices, Tensor& out, uint32_t id_bytes, DType dtype = DType::F16);
void greedy_sample_ex(Tensor& logits, Tensor& out_tokens, uint32_t position, uint32_t token_base,
                      uint32_t token_count, uint32_t id_bytes, DType dtype = DType::F16);

// ---- decoder-layer operators around attention -------------------------------
// The rules of include/evkcu.h hold (sizes in multiples of 8, which buffers
// may coincide), and a tensor holds less than 2^32 elements; optional tensors are
// pointers, nullptr for none.
enum class Act : int { None = 0, Relu = 1, Gelu = 2, Silu = 3 };

// y = act(x w + bias) + residual over the rows of x's last dimension; w is
// (K, N), or (N, K) with transpose_w.  pre receives x w + bias.
void linear(Tensor& x, Tensor& w, Tensor& y, Tensor* bias, Tensor* residual, Act act, Tensor* pre = nullptr,
            bool transpose_w = false, DType dtype = DType::F16);
// Gradients of linear from dy into those of dx, dw and dbias that are given,
// or added to them with acc.  With an activation, pre is linear's and dpre
// (like pre) receives its gradient.
void linear_backward(Tensor& x, Tensor& w, Tensor& dy, Tensor* dx, Tensor* dw, Tensor* dbias, Act act,
                     Tensor* pre = nullptr, Tensor* dpre = nullptr, bool transpose_w = false, bool acc = false,
                     DType dtype = DType::F16);

// Gated feed-forward block: [g | u] = x w_in, hidden = act(g) u, y = hidden
// w_out + residual; w_in (D, 2 F), w_out (F, D), both transposed with
// transpose_w.  pre (2 F a row) receives [g | u].
void gated_ffn(Tensor& x, Tensor& w_in, Tensor& w_out, Tensor& y, Tensor& hidden, Act act, Tensor* residual = nullptr,
               Tensor* pre = nullptr, bool transpose_w = false, DType dtype = DType::F16);
// Its gradients from dy and the saved pre into those that are given; dpre
// (like pre) receives pre's gradient, hidden is recomputed for dw_out.
void gated_ffn_backward(Tensor& x, Tensor& w_in, Tensor& w_out, Tensor& pre, Tensor& dy, Tensor& dpre, Tensor& hidden,
                        Tensor* dx, Tensor* dw_in, Tensor* dw_out, Act act, bool transpose_w = false,
                        bool acc = false, DType dtype = DType::F16);

// What qk_norm_rope rotates by, and how.
struct QkRope {
    uint32_t heads = 0;
    uint32_t rot_dim = 0;     // rotated part of a head, even; 0 for all of it
    bool half_split = false;  // pairs (i, i + rot_dim / 2) instead of (2 i, 2 i + 1); the
                              // rotated part is then a multiple of 16
    uint32_t pos_offset = 0;  // position of token t of every sequence: pos_offset + t
                              // (positions of each sequence's own: evkcu_qk_norm_rope)
    float eps = 1e-5f, base = 10000.0f;
};

// RMSNorm of every query and key head and its position rotation in one pass:
// qkv (B, S, (heads + 2 Hkv) Dh) is a fused projection's output; q (B, S,
// heads Dh), k and v (B, S, Hkv Dh) receive the queries, the keys and a copy
// of the values.  With cached, k and v are caches (B, cache_len, Hkv Dh)
// written at the tokens' positions.  gain_q, gain_k (Dh) or nullptr.
void qk_norm_rope(Tensor& qkv, Tensor& q, Tensor& k, Tensor& v, Tensor* gain_q, Tensor* gain_k, const QkRope& rope,
                  bool cached = false, DType dtype = DType::F16);
// Its gradients: from dq, dk (as q and k without a cache) into the query and
// key parts of dqkv (its value part is left as it is) and, where given,
// dgain_q and dgain_k, which need a workspace of qk_norm_rope_workspace(Dh) bytes.
void qk_norm_rope_backward(Tensor& qkv, Tensor& dq, Tensor& dk, Tensor& dqkv, Tensor* gain_q, Tensor* gain_k,
                           Tensor* dgain_q, Tensor* dgain_k, Tensor* workspace, const QkRope& rope,
                           DType dtype = DType::F16);
uint64_t qk_norm_rope_workspace(uint32_t head_dim);

}  // namespace evk::ai
