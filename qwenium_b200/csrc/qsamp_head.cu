// qsamp_head.cu -- the output head's operators: softmax cross entropy of
// hidden rows under a head weight without keeping the logits, its gradients,
// the 8-bit block-scaled product, and the quantiser that feeds it.
//
// First form: one tile routine on the FP32 pipes, 64 x 64 outputs per block,
// for every product; the epilogues hold the operators.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "qsamp_head.h"

namespace qs {
namespace {

constexpr int TM = 64, TN = 64, TK = 16, THREADS = 256;
constexpr int PIECE = 4096;  // vocabulary columns of dz held at once

__device__ __forceinline__ float bf(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ uint16_t to_bf(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
__device__ __forceinline__ float e4m3(uint8_t b) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}

// acc += a[m0 + ..][k0 .. k1) . b[n0 + ..][k0 .. k1); la(m, k) and lb(n, k)
// give 0 outside their operand.
template <typename LA, typename LB>
__device__ void tile_product(float (&acc)[4][4], int m0, int n0, int k0, int k1, LA la, LB lb, float* sa, float* sb) {
    const int t = threadIdx.x, tx = t % 16, ty = t / 16;
    for (int k = k0; k < k1; k += TK) {
        __syncthreads();
        for (int i = t; i < TM * TK; i += THREADS) sa[(i % TK) * TM + i / TK] = k + i % TK < k1 ? la(m0 + i / TK, k + i % TK) : 0.0f;
        for (int i = t; i < TN * TK; i += THREADS) sb[(i % TK) * TN + i / TK] = k + i % TK < k1 ? lb(n0 + i / TK, k + i % TK) : 0.0f;
        __syncthreads();
        for (int q = 0; q < TK; ++q)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) acc[i][j] += sa[q * TM + ty * 4 + i] * sb[q * TN + tx * 4 + j];
    }
    __syncthreads();
}

// Logits tile -> c[64][65].
__device__ void logits_tile(const HeadCall& a, int m0, int v0, float* c, float* sa, float* sb) {
    float acc[4][4] = {};
    tile_product(
        acc, m0, v0, 0, a.D, [&](int m, int k) { return m < a.N ? bf(a.hidden[m * a.hidden_stride + k]) : 0.0f; },
        [&](int v, int k) { return v < a.V ? bf(a.weight[v * a.weight_stride + k]) : 0.0f; }, sa, sb);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            float l = acc[i][j];
            if (a.softcap > 0.0f) l = a.softcap * tanhf(l / a.softcap);
            c[(threadIdx.x / 16 * 4 + i) * 65 + threadIdx.x % 16 * 4 + j] = l;
        }
    __syncthreads();
}

__global__ void __launch_bounds__(THREADS) lse_part_kernel(HeadCall a, float2* part, float* tgt) {
    __shared__ float sa[TM * TK], sb[TN * TK], c[TM * 65];
    const int v0 = blockIdx.x * TN, m0 = blockIdx.y * TM;
    logits_tile(a, m0, v0, c, sa, sb);
    const int m = m0 + threadIdx.x;
    if (threadIdx.x >= TM || m >= a.N) return;
    float mx = -INFINITY, s = 0.0f;
    const int t = a.targets[m];
    for (int j = 0; j < TN && v0 + j < a.V; ++j) mx = fmaxf(mx, c[threadIdx.x * 65 + j]);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    for (int j = 0; j < TN && v0 + j < a.V; ++j) {
        s += expf(c[threadIdx.x * 65 + j] - ref);
        if (v0 + j == t) tgt[m] = c[threadIdx.x * 65 + j];
    }
    part[(long long)blockIdx.x * a.N + m] = make_float2(mx, s);
}

__global__ void lse_join_kernel(HeadCall a, const float2* part, const float* tgt, int parts) {
    const int m = blockIdx.x * blockDim.x + threadIdx.x;
    if (m >= a.N) return;
    float mx = -INFINITY, s = 0.0f;
    for (int p = 0; p < parts; ++p) mx = fmaxf(mx, part[(long long)p * a.N + m].x);
    const float ref = mx == -INFINITY ? 0.0f : mx;
    for (int p = 0; p < parts; ++p) {
        const float2 q = part[(long long)p * a.N + m];
        s += q.y * expf(q.x - ref);
    }
    const float lse = ref + logf(s);
    const int t = a.targets[m];
    a.lse_out[m] = lse;
    a.loss[m] = t < 0 ? 0.0f : t < a.V ? lse - tgt[m] : NAN;
}

__global__ void __launch_bounds__(THREADS) dz_kernel(HeadCall a, uint16_t* dz, int p0, int pw) {
    __shared__ float sa[TM * TK], sb[TN * TK], c[TM * 65];
    const int v0 = p0 + blockIdx.x * TN, m0 = blockIdx.y * TM;
    logits_tile(a, m0, v0, c, sa, sb);
    for (int i = threadIdx.x; i < TM * TN; i += THREADS) {
        const int m = m0 + i / TN, v = v0 + i % TN;
        if (m >= a.N || v >= p0 + pw) continue;
        const int t = a.targets[m];
        const float l = c[i / TN * 65 + i % TN];
        float d = expf(l - a.lse[m]) - (v == t ? 1.0f : 0.0f);
        if (a.softcap > 0.0f) d *= 1.0f - (l / a.softcap) * (l / a.softcap);
        dz[(long long)m * PIECE + v - p0] = to_bf(t >= 0 && t < a.V ? d * a.grad_loss[m] : 0.0f);
    }
}

__global__ void __launch_bounds__(THREADS) dh_kernel(HeadCall a, const uint16_t* dz, float* dh, int p0, int pw) {
    __shared__ float sa[TM * TK], sb[TN * TK];
    const int d0 = blockIdx.x * TN, m0 = blockIdx.y * TM;
    float acc[4][4] = {};
    tile_product(
        acc, m0, d0, 0, pw, [&](int m, int k) { return m < a.N ? bf(dz[(long long)m * PIECE + k]) : 0.0f; },
        [&](int d, int k) { return d < a.D ? bf(a.weight[(p0 + k) * a.weight_stride + d]) : 0.0f; }, sa, sb);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + threadIdx.x / 16 * 4 + i, d = d0 + threadIdx.x % 16 * 4 + j;
            if (m >= a.N || d >= a.D) continue;
            const float s = (p0 ? dh[(long long)m * a.D + d] : 0.0f) + acc[i][j];
            dh[(long long)m * a.D + d] = s;
            if (p0 + pw == a.V) a.d_hidden[m * a.d_hidden_stride + d] = to_bf(s);
        }
}

__global__ void __launch_bounds__(THREADS) dw_kernel(HeadCall a, const uint16_t* dz, int p0, int pw) {
    __shared__ float sa[TM * TK], sb[TN * TK];
    const int d0 = blockIdx.x * TN, v0 = blockIdx.y * TM;
    float acc[4][4] = {};
    tile_product(
        acc, v0, d0, 0, a.N, [&](int v, int k) { return v < pw ? bf(dz[(long long)k * PIECE + v]) : 0.0f; },
        [&](int d, int k) { return d < a.D ? bf(a.hidden[k * a.hidden_stride + d]) : 0.0f; }, sa, sb);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int v = v0 + threadIdx.x / 16 * 4 + i, d = d0 + threadIdx.x % 16 * 4 + j;
            if (v < pw && d < a.D) a.d_weight[(p0 + v) * a.d_weight_stride + d] = to_bf(acc[i][j]);
        }
}

__global__ void __launch_bounds__(THREADS) fp8_kernel(Fp8Call a) {
    __shared__ float sa[TM * TK], sb[TN * TK];
    const int n0 = blockIdx.x * TN, m0 = blockIdx.y * TM;
    float out[4][4] = {};
    for (int k = 0; k < a.K; k += FP8_BLOCK) {
        float acc[4][4] = {};
        tile_product(
            acc, m0, n0, k, min(k + FP8_BLOCK, a.K), [&](int m, int q) { return m < a.M ? e4m3(a.x[m * a.x_stride + q]) : 0.0f; },
            [&](int n, int q) { return n < a.V ? e4m3(a.w[n * a.w_stride + q]) : 0.0f; }, sa, sb);
        for (int i = 0; i < 4; ++i)
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + threadIdx.x / 16 * 4 + i, n = n0 + threadIdx.x % 16 * 4 + j;
                if (m < a.M && n < a.V)
                    out[i][j] += acc[i][j] * (a.sx[m * a.sx_stride + k / FP8_BLOCK] * a.sw[n / FP8_BLOCK * a.sw_stride + k / FP8_BLOCK]);
            }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + threadIdx.x / 16 * 4 + i, n = n0 + threadIdx.x % 16 * 4 + j;
            if (m >= a.M || n >= a.V) continue;
            if (a.out_bf16)
                ((uint16_t*)a.out)[m * a.out_stride + n] = to_bf(out[i][j]);
            else
                ((float*)a.out)[m * a.out_stride + n] = out[i][j];
        }
}

// x / s to the nearest e4m3 value, ties to even, as if rounded once: the
// quotient rounded to 32 bits can only mislead where it lands on the border
// between two e4m3 values, and there the sign of the exact remainder
// x - y s (one fma) says on which side of the border the quotient lies.
__device__ __forceinline__ uint8_t quantize_one(float x, float s) {
    if (x == 0.0f) return 0;
    if (s < 0x1p-64f) {  // keeps the remainder out of the subnormals; both products are exact
        x *= 0x1p80f;
        s *= 0x1p80f;
    }
    float y = __fdiv_rn(x, s);
    const float ay = fabsf(y);
    const float step = ay < 0.015625f ? 0.001953125f : __uint_as_float((__float_as_uint(ay) & 0x7f800000u) - (3u << 23));
    const float h = ay / step;
    if (h - floorf(h) == 0.5f) {
        const float r = fmaf(-y, s, x);
        if (r != 0.0f) y = (r > 0.0f) == (y > 0.0f) ? y * 1.0000002f : y * 0.9999998f;
    }
    return __nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

// One block of 128 threads per quantisation block; thread t holds column t.
__global__ void __launch_bounds__(128) quantize_kernel(const void* x, int bf16, int M, int K, long long x_stride, int rows,
                                                       uint8_t* q, long long q_stride, float* scale, long long scale_stride) {
    __shared__ float red[4];
    const int k = blockIdx.y * FP8_BLOCK + threadIdx.x;
    const long long m0 = (long long)blockIdx.x * rows, m1 = min(m0 + rows, (long long)M);
    float mx = 0.0f;
    bool bad = false;
    auto at = [&](long long m) { return bf16 ? bf(((const uint16_t*)x)[m * x_stride + k]) : ((const float*)x)[m * x_stride + k]; };
    if (k < K)
        for (long long m = m0; m < m1; ++m) {
            const float v = fabsf(at(m));
            bad |= !(v < INFINITY);
            mx = fmaxf(mx, v);
        }
    if (bad) mx = INFINITY;
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float s = mx < INFINITY ? __fdiv_rn(mx, 448.0f) : NAN;
    if (threadIdx.x == 0) scale[blockIdx.x * scale_stride + blockIdx.y] = s;
    if (k < K)
        for (long long m = m0; m < m1; ++m) q[m * q_stride + k] = mx < INFINITY ? quantize_one(at(m), s) : 0x7f;
}

constexpr long long al(long long b) { return (b + 255) / 256 * 256; }

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" long long qs_head_loss_ws(int N, int V, int, int) { return al(8ll * N * ceil_div(V, TN)) + al(4ll * N); }

extern "C" long long qs_head_grad_ws(int N, int, int D, int) { return al(2ll * N * PIECE) + al(4ll * N * D); }

extern "C" cudaError_t qs_head_loss(const HeadCall* a, int* launches, cudaStream_t st) {
    const int parts = (int)ceil_div(a->V, TN);
    float2* part = (float2*)a->ws;
    float* tgt = (float*)(a->ws + al(8ll * a->N * parts));
    lse_part_kernel<<<dim3(parts, (unsigned)ceil_div(a->N, TM)), THREADS, 0, st>>>(*a, part, tgt);
    lse_join_kernel<<<(unsigned)ceil_div(a->N, 128), 128, 0, st>>>(*a, part, tgt, parts);
    *launches = 2;
    return cudaGetLastError();
}

extern "C" cudaError_t qs_head_grad(const HeadCall* a, int* launches, cudaStream_t st) {
    uint16_t* dz = (uint16_t*)a->ws;
    float* dh = (float*)(a->ws + al(2ll * a->N * PIECE));
    *launches = 0;
    const unsigned mt = (unsigned)ceil_div(a->N, TM), dt = (unsigned)ceil_div(a->D, TN);
    for (int p0 = 0; p0 < a->V; p0 += PIECE) {
        const int pw = min(PIECE, a->V - p0);
        if (a->N > 0) {
            dz_kernel<<<dim3((unsigned)ceil_div(pw, TN), mt), THREADS, 0, st>>>(*a, dz, p0, pw);
            dh_kernel<<<dim3(dt, mt), THREADS, 0, st>>>(*a, dz, dh, p0, pw);
            *launches += 2;
        }
        dw_kernel<<<dim3(dt, (unsigned)ceil_div(pw, TM)), THREADS, 0, st>>>(*a, dz, p0, pw);
        *launches += 1;
    }
    return cudaGetLastError();
}

extern "C" cudaError_t qs_matmul_fp8(const Fp8Call* a, cudaStream_t st) {
    fp8_kernel<<<dim3((unsigned)ceil_div(a->V, TN), (unsigned)ceil_div(a->M, TM)), THREADS, 0, st>>>(*a);
    return cudaGetLastError();
}

extern "C" cudaError_t qs_quantize_fp8(const void* x, int dtype, int M, int K, long long x_stride, int block_rows,
                                       uint8_t* q, long long q_stride, float* scale, long long scale_stride,
                                       cudaStream_t st) {
    quantize_kernel<<<dim3((unsigned)ceil_div(M, block_rows), (unsigned)ceil_div(K, FP8_BLOCK)), 128, 0, st>>>(
        x, dtype == QSAMP_BF16, M, K, x_stride, block_rows, q, q_stride, scale, scale_stride);
    return cudaGetLastError();
}
