// layer_refusals.cpp — calls of the decoder-layer operators of evk_ai_ext.h
// that have to end in their refusal (a message and an abort, as every failing
// evk::ai call does) before anything reaches a GPU.  The tensors have shapes
// and no memory.  tests/test_layer_ops_refusals.py runs one case a process.
#include <cstdio>
#include <string>

#include "evk_ai_ext.h"

using evk::ai::Act;

static Tensor shaped(const Shape& s) { return Tensor::alias(s, evk::Buffer{}); }

int main(int argc, char** argv) {
    if (argc != 2) return 2;
    const std::string c = argv[1];
    // a last dimension of 0
    if (c == "linear of nothing") {
        Tensor x = shaped({4, 0}), w = shaped({0, 8}), y = shaped({4, 8});
        evk::ai::linear(x, w, y, nullptr, nullptr, Act::None);
    } else if (c == "linear_backward of nothing") {
        Tensor x = shaped({4, 0}), w = shaped({0, 8}), dy = shaped({4, 8}), dw = shaped({0, 8});
        evk::ai::linear_backward(x, w, dy, nullptr, &dw, nullptr, Act::None);
    } else if (c == "gated_ffn of nothing") {
        Tensor x = shaped({4, 0}), wi = shaped({0, 16}), wo = shaped({8, 0}), y = shaped({4, 0}), h = shaped({4, 8});
        evk::ai::gated_ffn(x, wi, wo, y, h, Act::Silu);
    } else if (c == "gated_ffn_backward of nothing") {
        Tensor x = shaped({4, 0}), wi = shaped({0, 16}), wo = shaped({8, 0}), dy = shaped({4, 0}), h = shaped({4, 8});
        Tensor pre = shaped({4, 16}), dpre = shaped({4, 16});
        evk::ai::gated_ffn_backward(x, wi, wo, pre, dy, dpre, h, nullptr, nullptr, nullptr, Act::Silu);
        // 2^32 elements and more, which Shape::count() cuts to their low 32 bits
    } else if (c == "linear past 32 bits") {
        Tensor x = shaped({1u << 29, 16}), w = shaped({16, 8}), y = shaped({1u << 29, 8});
        evk::ai::linear(x, w, y, nullptr, nullptr, Act::None);
    } else if (c == "linear_backward past 32 bits") {
        Tensor x = shaped({1u << 29, 16}), w = shaped({16, 8}), dy = shaped({1u << 29, 8}), dw = shaped({16, 8});
        evk::ai::linear_backward(x, w, dy, nullptr, &dw, nullptr, Act::None);
    } else if (c == "gated_ffn past 32 bits") {
        Tensor x = shaped({1u << 29, 16}), wi = shaped({16, 16}), wo = shaped({8, 16}), y = shaped({1u << 29, 16});
        Tensor h = shaped({1u << 29, 8});
        evk::ai::gated_ffn(x, wi, wo, y, h, Act::Silu);
    } else if (c == "gated_ffn_backward past 32 bits") {
        Tensor x = shaped({1u << 29, 16}), wi = shaped({16, 16}), wo = shaped({8, 16}), dy = shaped({1u << 29, 16});
        Tensor h = shaped({1u << 29, 8}), pre = shaped({1u << 29, 16}), dpre = shaped({1u << 29, 16});
        evk::ai::gated_ffn_backward(x, wi, wo, pre, dy, dpre, h, nullptr, nullptr, nullptr, Act::Silu);
    } else if (c == "qk_norm_rope past 32 bits") {
        Tensor qkv = shaped({1u << 15, 1u << 15, 24}), q = shaped({1u << 15, 1u << 15, 8}), k = shaped(q.shape);
        Tensor v = shaped(q.shape);
        evk::ai::qk_norm_rope(qkv, q, k, v, nullptr, nullptr, {.heads = 1});
    } else if (c == "qk_norm_rope_backward past 32 bits") {
        Tensor qkv = shaped({1u << 15, 1u << 15, 24}), dq = shaped({1u << 15, 1u << 15, 8}), dk = shaped(dq.shape);
        Tensor dqkv = shaped(qkv.shape);
        evk::ai::qk_norm_rope_backward(qkv, dq, dk, dqkv, nullptr, nullptr, nullptr, nullptr, nullptr, {.heads = 1});
    } else {
        return 2;
    }
    std::printf("NOT REFUSED\n");
    return 0;
}
