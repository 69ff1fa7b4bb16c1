// layer_check.cpp — drives the decoder-layer operators of evk_ai_ext.h through
// libevk_ai.so on inputs read from a file and writes their outputs, so
// tests/test_gpu_layer_ops.py can compare them with the C ABI called directly.
// B 2, S 9, heads 4, Hkv 2, Dh 64 (D 256), F 264, bf16, gelu / silu.
// Input file: x (B, S, D), wqkv (D, 512), bqkv, gq, gk, w_in (D, 2 F), w_out
// (F, D), dy (B, S, D).  Output file: qkv | q | k | v | y | pre | dx | dw_in |
// dw_out | dqkv (B, S, 512) | dgq | dgk | dxq | dwqkv | dbqkv | k cache (B, 16, 128).
#include <cstdio>
#include <vector>

#include "evk_ai_ext.h"

using evk::ai::Act;
using evk::ai::DType;

int main(int argc, char** argv) {
    if (argc != 3) return 2;
    FILE* f = std::fopen(argv[1], "rb");
    if (!f) return 2;
    std::vector<uint16_t> in;
    {
        uint16_t buf[4096];
        size_t got;
        while ((got = std::fread(buf, 2, 4096, f)) > 0) in.insert(in.end(), buf, buf + got);
        std::fclose(f);
    }
    if (!evk::InitializeEVK({.applicationName = "layer_check"})) return 2;
    evk::ai::initialize();
    size_t pos = 0;
    std::vector<uint16_t> res;
    auto load = [&](Tensor& t) {
        uint16_t* d = reinterpret_cast<uint16_t*>(t.cpu());
        for (uint32_t i = 0; i < t.shape.count(); ++i) d[i] = in.at(pos++);
        t.cpu_upload();
    };
    auto zero = [&](Tensor& t) {
        uint16_t* d = reinterpret_cast<uint16_t*>(t.cpu());
        for (uint32_t i = 0; i < t.shape.count(); ++i) d[i] = 0;
        t.cpu_upload();
    };
    auto take = [&](Tensor& t) {
        t.cpu_download();
        const uint16_t* d = reinterpret_cast<const uint16_t*>(t.cpu());
        res.insert(res.end(), d, d + t.shape.count());
    };
    const uint32_t B = 2, S = 9, D = 256, F = 264, C = 512, Dh = 64;
    const DType bf = DType::BF16;
    Tensor x({B, S, D}), wqkv({D, C}), bqkv({C}), gq({Dh}), gk({Dh}), wi({D, 2 * F}), wo({F, D}), dy({B, S, D});
    for (Tensor* t : {&x, &wqkv, &bqkv, &gq, &gk, &wi, &wo, &dy}) load(*t);
    Tensor qkv({B, S, C}), q({B, S, D}), k({B, S, 128}), v({B, S, 128}), y({B, S, D}), h({B, S, F});
    Tensor pre({B, S, 2 * F}), dpre({B, S, 2 * F}), dx({B, S, D}), dwi({D, 2 * F}), dwo({F, D}), dqkv({B, S, C});
    Tensor dgq({Dh}), dgk({Dh}), dxq({B, S, D}), dwqkv({D, C}), dbqkv({C}), kc({B, 16, 128}), vc({B, 16, 128});
    Tensor ws({(uint32_t)(evk::ai::qk_norm_rope_workspace(Dh) / 2)});
    zero(dqkv), zero(kc), zero(vc);
    const evk::ai::QkRope rope{.heads = 4, .half_split = true, .pos_offset = 5};
    evk::ai::linear(x, wqkv, qkv, &bqkv, nullptr, Act::None, nullptr, false, bf);
    evk::ai::qk_norm_rope(qkv, q, k, v, &gq, &gk, rope, false, bf);
    evk::ai::qk_norm_rope(qkv, q, kc, vc, &gq, &gk, rope, true, bf);
    evk::ai::gated_ffn(x, wi, wo, y, h, Act::Silu, &x, &pre, false, bf);
    evk::ai::gated_ffn_backward(x, wi, wo, pre, dy, dpre, h, &dx, &dwi, &dwo, Act::Silu, false, false, bf);
    evk::ai::qk_norm_rope_backward(qkv, q, k, dqkv, &gq, &gk, &dgq, &dgk, &ws, rope, bf);
    evk::ai::linear_backward(x, wqkv, dqkv, &dxq, &dwqkv, &dbqkv, Act::None, nullptr, nullptr, false, false, bf);
    for (Tensor* t : {&qkv, &q, &k, &v, &y, &pre, &dx, &dwi, &dwo, &dqkv, &dgq, &dgk, &dxq, &dwqkv, &dbqkv, &kc})
        take(*t);
    evk::ai::SubmitCmd(true);
    FILE* o = std::fopen(argv[2], "wb");
    if (!o || std::fwrite(res.data(), 2, res.size(), o) != res.size()) return 2;
    std::fclose(o);
    evk::ai::shutdown();
    evk::Shutdown();
    std::printf("LAYER_OK\n");
    return 0;
}
