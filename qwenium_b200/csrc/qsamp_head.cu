// qsamp_head.cu -- the output head's operators: softmax cross entropy of
// hidden rows under a head weight without keeping the logits, its gradients,
// the 8-bit block-scaled product, and the quantiser that feeds it.
//
// Every product runs through one persistent kernel shape, head_kernel: a pair
// of CTAs (two SMs) makes 256 x 256 outputs with tcgen05 (cta_group::2), each
// CTA holding 128 of the rows in its tensor memory, two accumulators of 256
// columns so that one is read while the other is filled. One warp of each CTA
// loads tiles by TMA into a ring of six 32 KB stages, one warp of the leading
// CTA issues the matrix instructions, eight warps run the operator's epilogue
// on the accumulators: a thread owns one row (lane) and 128 columns (half).
// The pair halves what each SM loads per flop: 32 KB per 512 tensor cycles
// instead of 48 KB, which the L2 could not feed to 148 SMs.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "qs_tc.cuh"
#include "qsamp_head.h"

namespace qs {
namespace {

using namespace tc;

constexpr int TILE = 256;             // rows and columns a pair makes
constexpr int STAGES = 6;
constexpr int OPERAND_BYTES = 16384;  // one CTA's half of an operand per stage: 128 rows x 128 bytes
constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
constexpr int EPI_WARPS = 8;
constexpr int THREADS = 32 * (2 + EPI_WARPS);
constexpr int PATCH_PITCH = 33;       // a warp's 32 x 32 patch for stores to unaligned rows
constexpr int PATCH_FLOATS = 32 * PATCH_PITCH;
constexpr float LOG2E = 1.4426950408889634f;

struct Control {
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int gave_up;
};
constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * PATCH_FLOATS * 4 + (int)sizeof(Control);

enum Mode { LSE, DZ, GRAD, FP8 };

// Rows of the left operand are M, of the right one N; jobs are tiles.
struct Params {
    CUtensorMap a, b;    // K contiguous (LSE, DZ, FP8; GRAD: dz for d_hidden)
    CUtensorMap a2, b2;  // GRAD: dz and hidden with K in the rows (d_weight); b: weight with K in the rows
    int m_tiles, n_tiles, k_blocks, jobs;
    int M, N;            // rows of the left and right operand
    int* status;
    // LSE / DZ
    const int32_t* targets;
    float softcap;
    float2* part;        // [2 n_tiles][M] running maximum and sum of a tile's half
    float* target_logit; // [M]
    const float* lse;
    const float* grad;
    uint16_t* dz;        // [M][dz_pitch], columns from n0
    long long dz_pitch;
    int n0;              // DZ, GRAD: first vocabulary column of the piece
    // GRAD: jobs below dh_jobs make d_hidden slabs, the rest d_weight
    int dh_jobs, d_tiles, splits, dh_k_blocks, dw_k_blocks, rows, D;
    float* slabs;        // [splits][rows][D]
    int add;             // slabs hold an earlier piece's sums
    uint16_t* dw;
    long long dw_stride;
    int wide;            // 32-byte stores reach every row of the output
    // FP8
    const float* sx;
    const float* sw;
    long long sx_stride, sw_stride, out_stride;
    void* out;
    int out_bf16;
};

struct Job {
    int m0, n0;      // first row of either operand
    int k0, k_blocks;
    bool second;     // GRAD: a d_weight tile
    int split;
};

// Tiles in groups of eight along M: the pairs at work share few tiles of
// either operand, which then come from L2.
__device__ __forceinline__ void tile_of(int job, int m_tiles, int n_tiles, int& m, int& n) {
    const int group = job / (8 * n_tiles), width = min(8, m_tiles - group * 8);
    const int r = job - group * 8 * n_tiles;
    m = group * 8 + r % width;
    n = r / width;
}

template <int MODE>
__device__ __forceinline__ Job job_of(const Params& p, int job) {
    Job j = {};
    int m, n;
    if (MODE != GRAD) {
        tile_of(job, p.m_tiles, p.n_tiles, m, n);
        j.k_blocks = p.k_blocks;
    } else if (job < p.dh_jobs) {
        const int per = p.dh_jobs / p.splits;
        j.split = job / per;
        tile_of(job % per, p.m_tiles, p.d_tiles, m, n);
        j.k0 = (int)((long long)p.dh_k_blocks * j.split / p.splits);
        j.k_blocks = (int)((long long)p.dh_k_blocks * (j.split + 1) / p.splits) - j.k0;
    } else {
        j.second = true;
        tile_of(job - p.dh_jobs, p.n_tiles, p.d_tiles, m, n);
        j.k_blocks = p.dw_k_blocks;
    }
    j.m0 = m * TILE;
    j.n0 = n * TILE;
    return j;
}

// ---------------------------------------------------------------- epilogues
// One thread's view of a tile: its row, and how to store 32 columns of it.
__device__ __forceinline__ void logits_of(float (&v)[32], float cap) {
    // cap tanh(z / cap) = cap (1 - 2 / (exp(2 z / cap) + 1)): absolute error a
    // few 2^-24 of cap, and the exponential's overflow gives the limit
    if (cap > 0.0f) {
        const float a = 2.0f * LOG2E / cap;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = cap - 2.0f * cap * __fdividef(1.0f, exp2_approx(v[i] * a) + 1.0f);
    }
}

template <int MODE>
struct Epilogue;

// Running maximum and sum over the thread's 128 columns, in one pass: 32
// columns at a time, the sum rescaled when their maximum is larger.
template <>
struct Epilogue<LSE> {
    __device__ static void tile(const Params& p, const Job& j, uint32_t tmem, int row, int half, bool live, int target,
                                float, float) {
        float mx = -INFINITY, sum = 0.0f, found = 0.0f;
        bool has = false;
        const int c0 = j.n0 + half * 128;
#pragma unroll 1
        for (int c = 0; c < 128 && c0 + c < p.N; c += 32) {
            float v[32];
            tmem_load32(tmem + c, v);
            tmem_wait_load(v);
            logits_of(v, p.softcap);
            const int col = c0 + c;
            if (col + 32 > p.N) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (col + i >= p.N) v[i] = -INFINITY;
            }
            float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int i = 4; i < 32; ++i) m4[i % 4] = fmaxf(m4[i % 4], v[i]);
            const float top = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
            const float ref = top == -INFINITY ? 0.0f : top;
            float s4[4] = {sum * exp2_approx((mx - ref) * LOG2E), 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 32; ++i) s4[i % 4] += exp2_approx((v[i] - ref) * LOG2E);
            sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            mx = top;
            if (target >= col && target < col + 32) {
                has = true;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (target == col + i) found = v[i];
            }
        }
        if (live) {
            p.part[(long long)(j.n0 / 128 + half) * p.M + row] = make_float2(mx, sum);
            if (has) p.target_logit[row] = found;
        }
    }
};

// dz = g (exp(l - lse) - [target]) (1 - (l / cap)^2), rounded to bf16: the
// type of the products it goes into. Rows without a gradient are 0.
template <>
struct Epilogue<DZ> {
    __device__ static void tile(const Params& p, const Job& j, uint32_t tmem, int row, int half, bool live, int target,
                                float lse, float g) {
        const bool none = target < 0;
        const float inv = p.softcap > 0.0f ? 1.0f / p.softcap : 0.0f;
        const int c0 = j.n0 + half * 128;
        uint16_t* out = p.dz + row * p.dz_pitch + c0;
#pragma unroll 1
        for (int c = 0; c < 128 && c0 + c < p.N; c += 32) {
            float v[32];
            tmem_load32(tmem + c, v);
            tmem_wait_load(v);
            logits_of(v, p.softcap);
            const int at = target - (p.n0 + c0 + c);
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
                float d[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float l = v[i + q], y = l * inv;
                    d[q] = exp2_approx((l - lse) * LOG2E) - (at == i + q ? 1.0f : 0.0f);
                    d[q] = none ? 0.0f : d[q] * fmaf(-y, y, 1.0f) * g;
                }
                w[i / 2] = pack_bf16(d[0], d[1]);
            }
            if (live) {
                store32(out + c, reinterpret_cast<const uint32_t(&)[8]>(w[0]));
                store32(out + c + 16, reinterpret_cast<const uint32_t(&)[8]>(w[8]));
            }
        }
    }
};

template <>
struct Epilogue<GRAD> {
    __device__ static void tile(const Params& p, const Job& j, uint32_t tmem, int row, int half, bool, int, float, float) {
        const int c0 = j.n0 + half * 128;
        const bool live = row < (j.second ? p.N : p.rows);
#pragma unroll 1
        for (int c = 0; c < 128 && c0 + c < p.D; c += 32) {
            float v[32];
            tmem_load32(tmem + c, v);
            tmem_wait_load(v);
            if (!live) continue;
            const int col = c0 + c;
            if (!j.second) {
                float* out = p.slabs + ((long long)j.split * p.rows + row) * p.D + col;
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (col + i >= p.D) break;
                    if (p.add) {
                        const float4 x = *(const float4*)(out + i), y = *(const float4*)(out + i + 4);
                        v[i] += x.x, v[i + 1] += x.y, v[i + 2] += x.z, v[i + 3] += x.w;
                        v[i + 4] += y.x, v[i + 5] += y.y, v[i + 6] += y.z, v[i + 7] += y.w;
                    }
                    store32(out + i, reinterpret_cast<const uint32_t(&)[8]>(v[i]));
                }
            } else {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
                uint16_t* out = p.dw + (long long)(p.n0 + row) * p.dw_stride + col;
                if (p.wide && col + 32 <= p.D) {
                    store32(out, reinterpret_cast<const uint32_t(&)[8]>(w[0]));
                    store32(out + 16, reinterpret_cast<const uint32_t(&)[8]>(w[8]));
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (col + 8 * i < p.D)
                            *(uint4*)(out + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
            }
        }
    }
};

// 32 columns of the 8-bit product's rows. Rows on 32-byte boundaries: each
// thread stores whole sectors of its own row. Otherwise the warp turns its
// 32 x 32 patch in shared memory and stores one row after the other.
__device__ __forceinline__ void store_product(const Params& p, const float* v, int row, int row0, int col, float* patch) {
    const int lane = threadIdx.x % 32;
    if (p.wide && col + 32 <= p.N) {
        if (row >= p.M) return;
        uint32_t w[8];
        if (p.out_bf16) {
            uint16_t* out = (uint16_t*)p.out + row * p.out_stride + col;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[16 * h + 2 * i], v[16 * h + 2 * i + 1]);
                store32(out + 16 * h, w);
            }
        } else {
            float* out = (float*)p.out + row * p.out_stride + col;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * h + i]);
                store32(out + 8 * h, w);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) patch[lane * PATCH_PITCH + i] = v[i];
    __syncwarp();
    const int rows = min(32, p.M - row0);
    if (col + lane < p.N) {
        for (int r = 0; r < rows; ++r) {
            const float f = patch[r * PATCH_PITCH + lane];
            const long long at = (row0 + r) * p.out_stride + col + lane;
            if (p.out_bf16)
                ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(f);
            else
                ((float*)p.out)[at] = f;
        }
    }
    __syncwarp();
}

// ---------------------------------------------------------------- the kernel
template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) head_kernel(const __grid_constant__ Params p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* patches = (float*)(smem + STAGES * STAGE_BYTES);
    Control* ctl = (Control*)(patches + EPI_WARPS * PATCH_FLOATS);
    const uint32_t stage0 = smem_addr(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cta_rank();
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            bar_init(smem_addr(&ctl->full[s]), 1);
            bar_init(smem_addr(&ctl->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(smem_addr(&ctl->acc_full[b]), 1);
            bar_init(smem_addr(&ctl->acc_empty[b]), 2 * EPI_WARPS);
        }
        ctl->gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&p.a);
        tma_prefetch_map(&p.b);
    }
    if (warp == 1) tmem_alloc(smem_addr(&ctl->tmem), 512);
    __syncwarp();
    fence_before();
    cluster_sync();
    fence_after();
    const uint32_t tmem = ctl->tmem;
    volatile int* gave_up = &ctl->gave_up;

    if (warp == 0 && lane == 0) {
        // loads: this CTA's half of both operands, counted on the leader's barrier
        uint32_t it = 0;
        bool ok = true;
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            for (int kb = 0; kb < j.k_blocks; ++kb, ++it) {
                const uint32_t s = it % STAGES;
                if (!(ok = bar_wait(smem_addr(&ctl->empty[s]), (it / STAGES & 1) ^ 1, gave_up, p.status))) break;
                const uint32_t full = map_to(smem_addr(&ctl->full[s]), 0);
                if (rank == 0) bar_expect(smem_addr(&ctl->full[s]), 2 * STAGE_BYTES);
                const uint32_t da = stage0 + s * STAGE_BYTES, db = da + OPERAND_BYTES;
                const int m = j.m0 + rank * 128, n = j.n0 + rank * 128;
                if (MODE != GRAD) {
                    const int x = kb * (MODE == FP8 ? 128 : 64);
                    tma_load(da, &p.a, x, m, full);
                    tma_load(db, &p.b, x, n, full);
                } else {
                    const int k = (j.k0 + kb) * 64;
                    if (!j.second) {
                        tma_load(da, &p.a, k, m, full);
                        tma_load(db, &p.b, n, p.n0 + k, full);
                        tma_load(db + OPERAND_BYTES / 2, &p.b, n + 64, p.n0 + k, full);
                    } else {
                        tma_load(da, &p.a2, m, k, full);
                        tma_load(da + OPERAND_BYTES / 2, &p.a2, m + 64, k, full);
                        tma_load(db, &p.b2, n, k, full);
                        tma_load(db + OPERAND_BYTES / 2, &p.b2, n + 64, k, full);
                    }
                }
            }
        }
        // the last stages' releases arrive before this CTA may leave
        for (uint32_t back = it < STAGES ? it : STAGES; ok && back > 0; --back, ++it)
            ok = bar_wait(smem_addr(&ctl->empty[it % STAGES]), (it / STAGES & 1) ^ 1, gave_up, p.status);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // matrix instructions: K blocks of 128 bytes, four instructions each
        uint32_t it = 0, acc = 0;
        bool ok = true;
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            const bool mn = MODE == GRAD;
            const uint32_t instr = MODE == FP8 ? instr_e4m3() : instr_bf16(mn && j.second, mn);
            for (int kb = 0; kb < j.k_blocks; ++kb, ++it) {
                if (MODE == FP8 || kb == 0) {
                    if (!(ok = bar_wait(smem_addr(&ctl->acc_empty[acc & 1]), (acc / 2 & 1) ^ 1, gave_up, p.status))) break;
                }
                const uint32_t s = it % STAGES;
                if (!(ok = bar_wait(smem_addr(&ctl->full[s]), it / STAGES & 1, gave_up, p.status))) break;
                fence_after();
                const uint32_t da = stage0 + s * STAGE_BYTES, db = da + OPERAND_BYTES;
                const uint32_t d = tmem + (acc & 1) * TILE;
                // along K: 32 bytes of a row, or 16 rows of 128 bytes
                const uint32_t step_a = mn && j.second ? 2048 : 32, step_b = mn ? 2048 : 32;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint64_t oa = operand(da + q * step_a, OPERAND_BYTES / 2);
                    const uint64_t ob = operand(db + q * step_b, OPERAND_BYTES / 2);
                    if (MODE == FP8)
                        mma_e4m3(d, oa, ob, instr, q > 0);
                    else
                        mma_bf16(d, oa, ob, instr, kb > 0 || q > 0);
                }
                mma_commit(smem_addr(&ctl->empty[s]));
                if (MODE == FP8) mma_commit(smem_addr(&ctl->acc_full[acc++ & 1]));
            }
            if (MODE != FP8 && ok) mma_commit(smem_addr(&ctl->acc_full[acc++ & 1]));
        }
    } else if (warp >= 2) {
        const int quarter = warp % 4, half = (warp - 2) / 4;
        uint32_t acc = 0;
        bool ok = true;
        const uint32_t empty0 = map_to(smem_addr(&ctl->acc_empty[0]), 0), empty1 = map_to(smem_addr(&ctl->acc_empty[1]), 0);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            const int row0 = j.m0 + (int)rank * 128 + quarter * 32, row = row0 + lane;
            if constexpr (MODE != FP8) {
                const int rows = MODE == GRAD ? (j.second ? p.N : p.rows) : p.M;
                const bool live = row < rows;
                int target = -1;
                float lse = 0.0f, g = 0.0f;
                if (MODE == LSE && live) target = p.targets[row];
                if (MODE == DZ && live) {
                    target = p.targets[row];
                    if (target >= p.rows) target = -1;  // DZ: rows holds the vocabulary
                    if (target >= 0) lse = p.lse[row], g = p.grad[row];
                }
                ok = bar_wait(smem_addr(&ctl->acc_full[acc & 1]), acc / 2 & 1, gave_up, p.status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                fence_after();
                if (row0 < rows)
                    Epilogue<MODE>::tile(p, j, tmem + (quarter << 21) + (acc & 1) * TILE + half * 128, row, half, live,
                                         target, lse, g);
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(acc & 1 ? empty1 : empty0);
                ++acc;
            } else {
                // sum over K blocks of the blocks' own sums times their scales,
                // in 128 registers
                float sum[128];
#pragma unroll
                for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
                const bool work = row0 < p.M;
                const int col = j.n0 + half * 128;
                const float* sx = p.sx + (row < p.M ? row : 0) * p.sx_stride;
                const float* sw = p.sw + (col < p.N ? col / 128 : 0) * p.sw_stride;
                float scale = work ? sx[0] * sw[0] : 0.0f;
                for (int kb = 0; kb < j.k_blocks; ++kb, ++acc) {
                    const float now = scale;
                    if (work && kb + 1 < j.k_blocks) scale = sx[kb + 1] * sw[kb + 1];
                    ok = bar_wait(smem_addr(&ctl->acc_full[acc & 1]), acc / 2 & 1, gave_up, p.status);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    fence_after();
                    if (work) {
#pragma unroll
                        for (int c = 0; c < 128; c += 32) {
                            float v[32];
                            tmem_load32(tmem + (quarter << 21) + (acc & 1) * TILE + half * 128 + c, v);
                            tmem_wait_load(v);
#pragma unroll
                            for (int i = 0; i < 32; ++i) sum[c + i] = fmaf(v[i], now, sum[c + i]);
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive_cluster(acc & 1 ? empty1 : empty0);
                }
                if (ok && work) {
#pragma unroll
                    for (int c = 0; c < 128; c += 32)
                        if (col + c < p.N) store_product(p, sum + c, row, row0, col + c, patches + (warp - 2) * PATCH_FLOATS);
                }
            }
        }
    }
    __syncwarp();
    // a role gave up: whatever it had in flight lands while this CTA is here
    if (*gave_up)
        for (int i = 0; i < 20; ++i) __nanosleep(1000000);
    fence_before();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        tmem_free(tmem, 512);
    }
    cluster_sync();
}

// ---------------------------------------------------------------- joins
// lse of a row from its tiles' maxima and sums; 32 rows per block, the tiles
// split over the warps.
__global__ void __launch_bounds__(1024) lse_join_kernel(const float2* part, const float* target_logit, const int32_t* targets,
                                                        int N, int V, int parts, float* loss, float* lse_out) {
    __shared__ float2 red[32][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, row = blockIdx.x * 32 + lane;
    float mx = -INFINITY, sum = 0.0f;
    if (row < N) {
        for (int q = warp; q < parts; q += 32) {
            const float2 x = part[(long long)q * N + row];
            const float top = fmaxf(mx, x.x), ref = top == -INFINITY ? 0.0f : top;
            sum = sum * exp2_approx((mx - ref) * LOG2E) + x.y * exp2_approx((x.x - ref) * LOG2E);
            mx = top;
        }
    }
    red[warp][lane] = make_float2(mx, sum);
    __syncthreads();
    if (warp == 0 && row < N) {
        float top = -INFINITY;
        for (int q = 0; q < 32; ++q) top = fmaxf(top, red[q][lane].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        sum = 0.0f;
        for (int q = 0; q < 32; ++q) sum += red[q][lane].y * exp2_approx((red[q][lane].x - ref) * LOG2E);
        const float lse = ref + logf(sum);
        const int t = targets[row];
        lse_out[row] = lse;
        loss[row] = t < 0 ? 0.0f : t < V ? lse - target_logit[row] : NAN;
    }
}

// d_hidden = the slabs' sum in their order, rounded once; eight columns a thread.
__global__ void __launch_bounds__(256) dh_join_kernel(const float* slabs, int splits, int N, int D, uint16_t* dh,
                                                      long long dh_stride) {
    const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8, n = (long long)N * D;
    if (i >= n) return;
    float v[8] = {};
    for (int s = 0; s < splits; ++s) {
        const float4 x = *(const float4*)(slabs + s * n + i), y = *(const float4*)(slabs + s * n + i + 4);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    const uint4 w = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    *(uint4*)(dh + i / D * dh_stride + i % D) = w;
}

// ---------------------------------------------------------------- quantiser
__device__ __forceinline__ float bf(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

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

// ---------------------------------------------------------------- host
constexpr long long al(long long b) { return (b + 255) / 256 * 256; }

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

cudaError_t encoder(EncodeFn* out) {
    static std::atomic<EncodeFn> known{nullptr};
    EncodeFn fn = known.load(std::memory_order_relaxed);
    if (!fn) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess) return e;
        if (q != cudaDriverEntryPointSuccess || !f) return cudaErrorNotSupported;
        fn = (EncodeFn)f;
        known.store(fn, std::memory_order_relaxed);
    }
    *out = fn;
    return cudaSuccess;
}

// A matrix [rows][cols] of 1- or 2-byte elements in boxes of 128 bytes x
// box_rows; what lies outside reads as 0.
cudaError_t make_map(CUtensorMap* map, const void* base, int esz, long long rows, long long cols, long long stride,
                     int box_rows) {
    EncodeFn fn;
    cudaError_t e = encoder(&fn);
    if (e != cudaSuccess) return e;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride * esz};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / esz), (cuuint32_t)box_rows};
    const cuuint32_t one[2] = {1, 1};
    return fn(map, esz == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)base, dims, strides,
              box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}

template <int MODE>
cudaError_t launch(const Params& p, int num_sms, cudaStream_t st) {
    cudaError_t e = cudaFuncSetAttribute(head_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES);
    if (e != cudaSuccess) return e;
    const int pairs = num_sms / 2 < p.jobs ? num_sms / 2 : p.jobs;
    head_kernel<MODE><<<2 * pairs, THREADS, SMEM_BYTES, st>>>(p);
    return cudaGetLastError();
}

// How the gradients are cut: the vocabulary into equal pieces whose dz takes
// at most DZ_BYTES, and each piece's d_hidden sums into splits along the
// vocabulary, so that a d_hidden tile is at most half of one pair's share of
// the launch (few rows: few tiles with a long sum).
constexpr long long DZ_BYTES = 256ll << 20;
struct GradPlan {
    int piece, pieces, splits;
    long long dz_bytes, slab_bytes;
};
GradPlan grad_plan(int N, int V, int D, int num_sms) {
    GradPlan g;
    const long long most = (DZ_BYTES / 2 / (N > 0 ? N : 1)) / TILE * TILE;
    const long long cap = most < TILE ? TILE : most;
    g.pieces = (int)ceil_div(V, cap);
    g.piece = (int)(ceil_div(ceil_div(V, g.pieces), TILE) * TILE);
    g.pieces = (int)ceil_div(V, g.piece);
    const long long dt = ceil_div(D, TILE), mt = ceil_div(N, TILE), kb = ceil_div(g.piece, 64);
    const long long total = mt * dt * kb + ceil_div(g.piece, TILE) * dt * ceil_div(N, 64);
    long long share = total / (num_sms / 2) / 2;
    share = share < 16 ? 16 : share;
    g.splits = (int)ceil_div(kb, share);
    g.splits = g.splits > 64 ? 64 : g.splits;
    g.dz_bytes = al(2ll * N * g.piece);
    g.slab_bytes = al(4ll * g.splits * N * D);
    return g;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" long long qs_head_loss_ws(int N, int V, int, int) {
    return al(8ll * N * 2 * ceil_div(V, TILE)) + al(4ll * N);
}

extern "C" long long qs_head_grad_ws(int N, int V, int D, int num_sms) {
    const GradPlan g = grad_plan(N, V, D, num_sms);
    return g.dz_bytes + g.slab_bytes;
}

extern "C" cudaError_t qs_head_loss(const HeadCall* a, int* launches, cudaStream_t st) {
    Params p = {};
    cudaError_t e = make_map(&p.a, a->hidden, 2, a->N, a->D, a->hidden_stride, 128);
    if (e == cudaSuccess) e = make_map(&p.b, a->weight, 2, a->V, a->D, a->weight_stride, 128);
    if (e != cudaSuccess) return e;
    p.m_tiles = (int)ceil_div(a->N, TILE);
    p.n_tiles = (int)ceil_div(a->V, TILE);
    p.k_blocks = (int)ceil_div(a->D, 64);
    p.jobs = p.m_tiles * p.n_tiles;
    p.M = a->N;
    p.N = a->V;
    p.status = a->status;
    p.targets = a->targets;
    p.softcap = a->softcap;
    p.part = (float2*)a->ws;
    p.target_logit = (float*)(a->ws + al(8ll * a->N * 2 * p.n_tiles));
    e = launch<LSE>(p, a->num_sms, st);
    if (e != cudaSuccess) return e;
    lse_join_kernel<<<(unsigned)ceil_div(a->N, 32), 1024, 0, st>>>(p.part, p.target_logit, a->targets, a->N, a->V,
                                                                   (int)ceil_div(a->V, 128), a->loss, a->lse_out);
    *launches = 2;
    return cudaGetLastError();
}

extern "C" cudaError_t qs_head_grad(const HeadCall* a, int* launches, cudaStream_t st) {
    *launches = 0;
    if (a->N == 0)
        return cudaMemset2DAsync(a->d_weight, (size_t)a->d_weight_stride * 2, 0, (size_t)a->D * 2, (size_t)a->V, st);
    const GradPlan g = grad_plan(a->N, a->V, a->D, a->num_sms);
    uint16_t* dz = (uint16_t*)a->ws;
    float* slabs = (float*)(a->ws + g.dz_bytes);
    for (int q = 0; q < g.pieces; ++q) {
        const int p0 = q * g.piece, pw = a->V - p0 < g.piece ? a->V - p0 : g.piece;
        Params p = {};
        cudaError_t e = make_map(&p.a, a->hidden, 2, a->N, a->D, a->hidden_stride, 128);
        if (e == cudaSuccess)
            e = make_map(&p.b, a->weight + (long long)p0 * a->weight_stride, 2, pw, a->D, a->weight_stride, 128);
        if (e != cudaSuccess) return e;
        p.m_tiles = (int)ceil_div(a->N, TILE);
        p.n_tiles = (int)ceil_div(pw, TILE);
        p.k_blocks = (int)ceil_div(a->D, 64);
        p.jobs = p.m_tiles * p.n_tiles;
        p.M = a->N;
        p.N = pw;
        p.rows = a->V;
        p.status = a->status;
        p.targets = a->targets;
        p.softcap = a->softcap;
        p.lse = a->lse;
        p.grad = a->grad_loss;
        p.dz = dz;
        p.dz_pitch = g.piece;
        p.n0 = p0;
        e = launch<DZ>(p, a->num_sms, st);
        if (e != cudaSuccess) return e;
        e = make_map(&p.a, dz, 2, a->N, pw, g.piece, 128);
        if (e == cudaSuccess) e = make_map(&p.b, a->weight, 2, a->V, a->D, a->weight_stride, 64);
        if (e == cudaSuccess) e = make_map(&p.a2, dz, 2, a->N, pw, g.piece, 64);
        if (e == cudaSuccess) e = make_map(&p.b2, a->hidden, 2, a->N, a->D, a->hidden_stride, 64);
        if (e != cudaSuccess) return e;
        p.d_tiles = (int)ceil_div(a->D, TILE);
        p.dh_k_blocks = (int)ceil_div(pw, 64);
        // every split has a K block; a short last piece adds to the first slabs
        p.splits = g.splits < p.dh_k_blocks ? g.splits : p.dh_k_blocks;
        p.dw_k_blocks = (int)ceil_div(a->N, 64);
        p.dh_jobs = p.m_tiles * p.d_tiles * p.splits;
        p.jobs = p.dh_jobs + p.n_tiles * p.d_tiles;
        p.rows = a->N;
        p.D = a->D;
        p.slabs = slabs;
        p.add = q > 0;
        p.dw = a->d_weight;
        p.dw_stride = a->d_weight_stride;
        p.wide = (uintptr_t)a->d_weight % 32 == 0 && a->d_weight_stride % 16 == 0;
        e = launch<GRAD>(p, a->num_sms, st);
        if (e != cudaSuccess) return e;
        *launches += 2;
    }
    const long long n = (long long)a->N * a->D / 8;
    dh_join_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, st>>>(slabs, g.splits, a->N, a->D, a->d_hidden, a->d_hidden_stride);
    *launches += 1;
    return cudaGetLastError();
}

extern "C" cudaError_t qs_matmul_fp8(const Fp8Call* a, cudaStream_t st) {
    Params p = {};
    cudaError_t e = make_map(&p.a, a->x, 1, a->M, a->K, a->x_stride, 128);
    if (e == cudaSuccess) e = make_map(&p.b, a->w, 1, a->V, a->K, a->w_stride, 128);
    if (e != cudaSuccess) return e;
    p.m_tiles = (int)ceil_div(a->M, TILE);
    p.n_tiles = (int)ceil_div(a->V, TILE);
    p.k_blocks = (int)ceil_div(a->K, FP8_BLOCK);
    p.jobs = p.m_tiles * p.n_tiles;
    p.M = a->M;
    p.N = a->V;
    p.status = a->status;
    p.sx = a->sx;
    p.sw = a->sw;
    p.sx_stride = a->sx_stride;
    p.sw_stride = a->sw_stride;
    p.out = a->out;
    p.out_stride = a->out_stride;
    p.out_bf16 = a->out_bf16;
    const int esz = a->out_bf16 ? 2 : 4;
    p.wide = (uintptr_t)a->out % 32 == 0 && a->out_stride * esz % 32 == 0;
    return launch<FP8>(p, a->num_sms, st);
}

extern "C" cudaError_t qs_quantize_fp8(const void* x, int dtype, int M, int K, long long x_stride, int block_rows,
                                       uint8_t* q, long long q_stride, float* scale, long long scale_stride,
                                       cudaStream_t st) {
    quantize_kernel<<<dim3((unsigned)ceil_div(M, block_rows), (unsigned)ceil_div(K, FP8_BLOCK)), 128, 0, st>>>(
        x, dtype == QSAMP_BF16, M, K, x_stride, block_rows, q, q_stride, scale, scale_stride);
    return cudaGetLastError();
}
