// qsamp_head.h -- what the host API (qsamp_api.cu) and the output-head
// kernels (qsamp_head.cu) share. Internal; the public C ABI is
// include/qsamp.h.
#ifndef QSAMP_HEAD_H
#define QSAMP_HEAD_H

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/qsamp.h"

namespace qs {

// One cross-entropy call over a head (both directions).
struct HeadCall {
    const uint16_t* hidden;  // bf16 [N][hidden_stride]
    const uint16_t* weight;  // bf16 [V][weight_stride]
    const int32_t* targets;  // [N]
    int N, V, D;
    long long hidden_stride, weight_stride;
    float softcap;
    // forward
    float* loss;
    float* lse_out;
    // backward
    const float* lse;
    const float* grad_loss;
    uint16_t* d_hidden;
    uint16_t* d_weight;
    long long d_hidden_stride, d_weight_stride;
    unsigned char* ws;
    int num_sms;
    int* status;      // mapped host word, written only when a bounded wait ran out
    unsigned long long wait_ns;  // how long a wait may take
    uint32_t* ready;  // the context's kernels whose attributes are set
};

// One 8-bit product: out[m][n] = sum over K blocks of sx sw (x . w).
struct Fp8Call {
    const uint8_t* x;  // e4m3 [M][x_stride]
    const uint8_t* w;  // e4m3 [V][w_stride]
    const float* sx;   // [M][sx_stride]
    const float* sw;   // [ceil(V / 128)][sw_stride]
    void* out;         // [M][out_stride]
    int M, V, K, out_bf16;
    long long x_stride, w_stride, sx_stride, sw_stride, out_stride;
    int num_sms;
    int* status;
    unsigned long long wait_ns;
    uint32_t* ready;
};

constexpr int FP8_BLOCK = 128;

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

}  // namespace qs

extern "C" long long qs_head_loss_ws(int N, int V, int D, int num_sms);
extern "C" long long qs_head_grad_ws(int N, int V, int D, int num_sms);
// Launch counts go to *launches.
extern "C" cudaError_t qs_head_loss(const qs::HeadCall* a, int* launches, cudaStream_t st);
extern "C" cudaError_t qs_head_grad(const qs::HeadCall* a, int* launches, cudaStream_t st);
extern "C" cudaError_t qs_matmul_fp8(const qs::Fp8Call* a, cudaStream_t st);
extern "C" cudaError_t qs_quantize_fp8(const void* x, int dtype, int M, int K, long long x_stride, int block_rows,
                                       uint8_t* q, long long q_stride, float* scale, long long scale_stride,
                                       cudaStream_t st);

#endif
