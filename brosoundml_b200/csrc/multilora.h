// The projection of many requests through one shared weight and each row's own low-rank
// adapter, its backward, and counter-based dropout (include/bsml_decoder.h bsml_multilora_*,
// bsml_dropout_*).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace bsml {

enum DType { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
inline int dtype_size(int dt) { return dt == DT_F32 ? 4 : 2; }

struct MultiLora {
    int dtype = DT_F32;
    int rows = 0, cin = 0, cout = 0, rank = 0, adapters = 0;
    double dropout = 0.0;
    bool zero_padding = false;        // rows with id < -1: zeroed instead of left as they were
    const void* W = nullptr;          // (cout, cin)
    const void* A = nullptr;          // (adapters, rank, cin)
    const void* B = nullptr;          // (adapters, cout, rank)
    const float* scale = nullptr;     // (adapters), nullable: 1
    const int* ids = nullptr;         // (rows)
    const uint64_t* rng = nullptr;    // {seed, offset}, read only with dropout > 0
};

// y = x W^T + bias + B_a h, h = scale_a / (1 - p) A_a (keep * x). h (rows, rank) nullable.
void multilora_forward(const MultiLora& p, const void* x, int64_t ldx, const void* bias, void* y, int64_t ldy,
                       float* h, cudaStream_t st);
// dx = dy W + keep * (g A_a), g = scale_a / (1 - p) B_a^T dy; dA_a = sum g (keep * x)^T;
// dB_a = sum dy h^T. Each output nullable.
void multilora_backward(const MultiLora& p, const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* h,
                        void* dx, int64_t lddx, void* dA, void* dB, cudaStream_t st);
// Gives the current device's scratch that no call uses any more back to it.
void multilora_release_scratch();

// y = residual + keep / (1 - p) * x over (rows, cols); residual nullable, y may be x or residual.
void dropout(int dtype, const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t ldy, int rows,
             int cols, double p, const uint64_t* rng, cudaStream_t st);

}  // namespace bsml
