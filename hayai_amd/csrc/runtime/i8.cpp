// Dispatch of the 8-bit path: rows into codes (i8_rows.hip), products of codes (i8_gemm.hip) and
// the choice of the next token (sample.hip).
#include <algorithm>

#include "engine.h"

namespace hh {

const ActType* act_type(int t) {
    static const ActType f32{"f32", 4}, f16{"f16", 2}, bf16{"bf16", 2};
    return t == HH_TYPE_F32 ? &f32 : t == HH_TYPE_F16 ? &f16 : t == HH_TYPE_BF16 ? &bf16 : nullptr;
}

void i8_kernels(std::vector<std::string>& k) {
    for (int t : {HH_TYPE_F32, HH_TYPE_F16, HH_TYPE_BF16}) {
        const std::string ty = act_type(t)->name;
        for (const char* kind : {"plain", "act", "norm"})
            for (const char* v : {"c1", "c2", "loop"}) k.push_back("hh_i8_rows_" + ty + "_" + kind + "_" + v);
        k.push_back("hh_i8_gemm_simple_" + ty);
        k.push_back("hh_sample_simple_" + ty);
    }
}

}  // namespace hh

using namespace hh;

hh_status hh_engine::enqueue_i8_rows(int type, size_t rows, const hh_i8_rows_args& a) {
    const ActType* ty = act_type(type);
    const size_t chunks = (a.cols * ty->bytes + 15) / 16;
    const size_t threads = std::min<size_t>(1024, (chunks + 63) / 64 * 64);
    const char* kind = a.norm ? "norm" : a.b ? "act" : "plain";
    const char* v = chunks <= threads ? "c1" : chunks <= 2 * threads ? "c2" : "loop";
    hipFunction_t f;
    HH_TRY(kernel(std::string("hh_i8_rows_") + ty->name + "_" + kind + "_" + v, &f));
    return launch(f, (uint32_t)rows, (uint32_t)threads, a);
}

hh_status hh_engine::enqueue_i8_gemm(int type, const hh_i8_gemm_args& a) {
    hipFunction_t f;
    HH_TRY(kernel(std::string("hh_i8_gemm_simple_") + act_type(type)->name, &f));
    void* params[] = {const_cast<hh_i8_gemm_args*>(&a)};
    HH_TRY_HIP(hipModuleLaunchKernel(f, (a.m + 63) / 64, (a.t + 63) / 64, 1, 256, 1, 1, 0, stream, params, nullptr),
               "hipModuleLaunchKernel(i8_gemm)");
    return HH_OK;
}

hh_status hh_engine::enqueue_sample(int type, size_t rows, const hh_sample_args& a) {
    hipFunction_t f;
    HH_TRY(kernel(std::string("hh_sample_simple_") + act_type(type)->name, &f));
    return launch(f, (uint32_t)rows, 1024, a);
}
