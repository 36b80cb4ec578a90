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
//
// Measured (4096 x 2048 x 32768, single launches): loss 342 us = 1.61 PFLOP/s,
// tensor pipe 88% active; dz 384 us = 1.43 PFLOP/s, 78%; gradients 710 us = 1.55
// PFLOP/s, 87%. At a depth of 1152, with a soft-cap, the epilogues set the pace
// (45% and 38% in loss and dz). In a loop at 4096 x 2048 x 151936 the 1000 W
// limit does (8.1 ms a step, 1.3 GHz): 90% of cuBLAS's sustained rate over the
// 8 N D V operations, a quarter of them the logits made a second time.
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
constexpr float LOG2E = 1.4426950408889634f;

struct Control {
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem;
    int gave_up;
};
enum Mode { LSE, DZ, GRAD, FP8 };

// DZ and GRAD: a warp's 32 rows of 64 bf16 outputs on their way out.
constexpr int OUT_PATCH = 4096;
__host__ __device__ constexpr int smem_bytes(int mode) {
    return 1024 + STAGES * STAGE_BYTES + (mode == LSE ? 0 : EPI_WARPS * OUT_PATCH) + (int)sizeof(Control);
}
static_assert(smem_bytes(GRAD) <= 232448, "shared memory of a CTA");

// Rows of the left operand are M, of the right one N; jobs are tiles.
struct Params {
    CUtensorMap a, b;    // K contiguous (LSE, DZ; GRAD: dz for d_hidden)
    CUtensorMap a2, b2;  // GRAD: dz and hidden with K in the rows (d_weight); b: weight with K in the rows
    CUtensorMap o;       // the bf16 output: DZ: dz, GRAD: the piece's rows of d_weight
    int m_tiles, n_tiles, k_blocks, jobs;
    int slice;           // K blocks summed in tensor memory before the epilogue takes them
    int M, N;            // rows of the left and right operand
    int* status;
    unsigned long long wait_ns;
    // LSE / DZ
    const int32_t* targets;
    float softcap;
    float2* part;        // [2 n_tiles][M] running maximum and sum of a tile's half
    float* target_logit; // [M]
    const float* lse;
    const float* grad;
    const float* unit;   // DZ, GRAD: what dz is held over (find_unit)
    int n0;              // DZ, GRAD: first vocabulary column of the piece
    // GRAD: jobs below dh_jobs make d_hidden slabs, the rest d_weight
    int dh_jobs, d_tiles, splits, dh_k_blocks, dw_k_blocks, rows, D;
    float* slabs;        // [splits][rows][D]
    int add;             // slabs hold an earlier piece's sums
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

// ---------------------------------------------------------------- packed fp32
// Two floats in one register pair; one instruction does both.
struct Two {
    uint64_t v;
    __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
    __device__ __forceinline__ explicit Two(uint64_t x) : v(x) {}
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two mul2(Two a, Two b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
    return Two(d);
}
__device__ __forceinline__ Two add2(Two a, Two b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
    return Two(d);
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v));
    return Two(d);
}

// ---------------------------------------------------------------- epilogues
// cap tanh(z / cap) = cap (1 - 2 / (exp(2 z / cap) + 1)): the absolute error is
// a few 2^-24 of cap, and the exponential's overflow gives the limit. A cap
// above 64 would lose small logits in that, so there tanh's series to y^9
// serves |z / cap| < 1/4 (it takes 6% of the loss's time, 256 x 2048 x 262144;
// at a cap of 30 the plain form is within 1e-5).
template <int N>
__device__ __forceinline__ void logits_of(float (&v)[N], float cap) {
    if (cap == 0.0f) return;
    const float a = 2.0f * LOG2E / cap, b = -2.0f * cap;
    if (cap <= 64.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = fmaf(b, __fdividef(1.0f, exp2_approx(v[i] * a) + 1.0f), cap);
        return;
    }
    const float inv = 1.0f / cap;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float y = v[i] * inv, y2 = y * y;
        const float series = fmaf(y2, fmaf(y2, fmaf(y2, fmaf(y2, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
        const float whole = fmaf(b, __fdividef(1.0f, exp2_approx(v[i] * a) + 1.0f), cap);
        v[i] = fabsf(y) < 0.25f ? v[i] * series : whole;
    }
}

// Running maximum and sum over the thread's 128 columns, 32 at a time, the
// sum rescaled when their maximum is larger.
__device__ __forceinline__ void softmax_sums(const Params& p, const Job& j, float (&z)[128], int row, int half, bool live,
                                             int target) {
    float mx = -INFINITY, sum = 0.0f, found = 0.0f;
    bool has = false;
    const int c0 = j.n0 + half * 128;
#pragma unroll
    for (int c = 0; c < 128; c += 32) {
        if (c0 + c >= p.N) break;
        float(&v)[32] = reinterpret_cast<float(&)[32]>(z[c]);
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

// 64 bf16 columns of the warp's 32 rows, a row a lane: through the warp's patch
// of shared memory (swizzled in 16-byte pieces as the tensor copy reads it) and
// out as one box. Stored from the lanes themselves a row's bytes would reach
// the L1 as 32 lines an instruction, which for short sums is the kernel's
// time.
__device__ __forceinline__ void store_box(const CUtensorMap* map, const uint32_t (&w)[32], int x, int y, unsigned char* patch) {
    const int lane = threadIdx.x % 32;
    if (lane == 0) tma_store_wait_read();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c)
        *(uint4*)(patch + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) tma_store(map, x, y, smem_addr(patch));
}

// dz = g (exp(l - lse) - [target]) (1 - (l / cap)^2); 0 for rows without a
// gradient. Without a cap (inv_cap 0) the slope is 1 for a logit of -infinity
// too: y is 0 times the lowest finite number there.
__device__ __forceinline__ float dz_of(float l, float lse, float g, float inv_cap, bool hot, bool none) {
    const float y = fmaxf(l, -3.402823466e38f) * inv_cap, d = exp2_approx((l - lse) * LOG2E) - (hot ? 1.0f : 0.0f);
    return none ? 0.0f : d * fmaf(-y, y, 1.0f) * g;
}

// The thread's 128 columns of dz from its logits' products, rounded to bf16, the
// type of the products dz goes into.
__device__ __forceinline__ void dz_tile(const Params& p, const Job& j, float (&z)[128], int row, int half, int target, float lse,
                                        float g, unsigned char* patch) {
    const float inv = p.softcap > 0.0f ? 1.0f / p.softcap : 0.0f;
    const int c0 = j.n0 + half * 128;
#pragma unroll
    for (int c = 0; c < 128; c += 64) {
        if (c0 + c >= p.N) break;
        uint32_t w[32];
#pragma unroll
        for (int q = 0; q < 64; q += 32) {
            float(&v)[32] = reinterpret_cast<float(&)[32]>(z[c + q]);
            logits_of(v, p.softcap);
            const int at = target - (p.n0 + c0 + c + q);
#pragma unroll
            for (int i = 0; i < 32; i += 2)
                w[(q + i) / 2] = pack_bf16(dz_of(v[i], lse, g, inv, at == i, target < 0),
                                           dz_of(v[i + 1], lse, g, inv, at == i + 1, target < 0));
        }
        store_box(&p.o, w, c0 + c, row - (int)(threadIdx.x % 32), patch);
    }
}

// 64 columns of d_weight, from column c.
__device__ __forceinline__ void store_dw(const Params& p, float (&v)[64], int c, int row, float unit, unsigned char* patch) {
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 64; i += 2) w[i / 2] = pack_bf16(v[i] * unit, v[i + 1] * unit);
    store_box(&p.o, w, c, row - (int)(threadIdx.x % 32), patch);
}

// 32 columns of a d_hidden slab, from column c.
__device__ __forceinline__ void store_dh(const Params& p, const Job& j, float (&v)[32], int c, int row) {
    if (row >= p.rows) return;
    float* out = p.slabs + ((long long)j.split * p.rows + row) * p.D + c;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        if (c + i >= p.D) break;
        if (p.add) {
            const float4 x = *(const float4*)(out + i), y = *(const float4*)(out + i + 4);
            v[i] += x.x, v[i + 1] += x.y, v[i + 2] += x.z, v[i + 3] += x.w;
            v[i + 4] += y.x, v[i + 5] += y.y, v[i + 6] += y.z, v[i + 7] += y.w;
        }
        store32(out + i, reinterpret_cast<const uint32_t(&)[8]>(v[i]));
    }
}

// The thread's 128 columns of either gradient, straight from tensor memory.
__device__ __forceinline__ void grad_tile(const Params& p, const Job& j, uint32_t tmem, int row, int half, float unit,
                                          unsigned char* patch) {
    const int c0 = j.n0 + half * 128;
    if (j.second) {
#pragma unroll 1
        for (int c = 0; c < 128 && c0 + c < p.D; c += 64) {
            float v[64];
#pragma unroll
            for (int q = 0; q < 64; q += 32) {
                float(&part)[32] = reinterpret_cast<float(&)[32]>(v[q]);
                tmem_load32(tmem + c + q, part);
                tmem_wait_load(part);
            }
            store_dw(p, v, c0 + c, row, unit, patch);
        }
        return;
    }
#pragma unroll 1
    for (int c = 0; c < 128 && c0 + c < p.D; c += 32) {
        float v[32];
        tmem_load32(tmem + c, v);
        tmem_wait_load(v);
        store_dh(p, j, v, c0 + c, row);
    }
}
// The same from the sum of several slices.
__device__ __forceinline__ void grad_tile(const Params& p, const Job& j, float (&z)[128], int row, int half, float unit,
                                          unsigned char* patch) {
    const int c0 = j.n0 + half * 128;
    if (j.second) {
#pragma unroll
        for (int c = 0; c < 128; c += 64)
            if (c0 + c < p.D) store_dw(p, reinterpret_cast<float(&)[64]>(z[c]), c0 + c, row, unit, patch);
        return;
    }
#pragma unroll
    for (int c = 0; c < 128; c += 32)
        if (c0 + c < p.D) store_dh(p, j, reinterpret_cast<float(&)[32]>(z[c]), c0 + c, row);
}

// ---------------------------------------------------------------- the kernel
// SLICED: an accumulator may hold part of a tile's sums (p.slice K blocks).
template <int MODE, bool SLICED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) head_kernel(const __grid_constant__ Params p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* patches = smem + STAGES * STAGE_BYTES;
    Control* ctl = (Control*)(smem + smem_bytes(MODE) - 1024 - sizeof(Control));
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
    if (warp == 1) tmem_alloc<true>(smem_addr(&ctl->tmem), 512);
    __syncwarp();
    fence_before();
    cluster_sync();
    fence_after();
    const uint32_t tmem = ctl->tmem;
    const Patience patience = {&ctl->gave_up, p.status, p.wait_ns};
    launch_next();
    wait_previous();
    const uint32_t full0 = smem_addr(ctl->full), empty0 = smem_addr(ctl->empty);
    const uint32_t acc_full0 = smem_addr(ctl->acc_full), acc_empty0 = smem_addr(ctl->acc_empty);

    if (warp == 0) {
        // loads: this CTA's half of both operands, counted on the leader's barrier
        Ring<STAGES> at;
        bool ok = true;
        const uint32_t lead_full0 = map_to(full0, 0);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            const int m = j.m0 + rank * 128, n = j.n0 + rank * 128;
            for (int kb = 0; kb < j.k_blocks; ++kb, at.step()) {
                if (!(ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience))) break;
                if (elected()) {
                    const uint32_t full = lead_full0 + 8 * at.slot;
                    if (rank == 0) bar_expect(full0 + 8 * at.slot, 2 * STAGE_BYTES);
                    const uint32_t da = stage0 + at.slot * STAGE_BYTES, db = da + OPERAND_BYTES;
                    if (MODE != GRAD) {
                        const int x = kb * 64;
                        tma_load<true>(da, &p.a, x, m, full);
                        tma_load<true>(db, &p.b, x, n, full);
                    } else {
                        const int k = (j.k0 + kb) * 64;
                        if (!j.second) {
                            tma_load<true>(da, &p.a, k, m, full);
                            tma_load<true>(db, &p.b, n, p.n0 + k, full);
                            tma_load<true>(db + OPERAND_BYTES / 2, &p.b, n + 64, p.n0 + k, full);
                        } else {
                            tma_load<true>(da, &p.a2, m, k, full);
                            tma_load<true>(da + OPERAND_BYTES / 2, &p.a2, m + 64, k, full);
                            tma_load<true>(db, &p.b2, n, k, full);
                            tma_load<true>(db + OPERAND_BYTES / 2, &p.b2, n + 64, k, full);
                        }
                    }
                }
                __syncwarp();
            }
        }
        // the last stages' releases arrive before this CTA may leave (a stage never used passes at once)
        for (int back = 0; ok && back < STAGES; ++back, at.step())
            ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience);
    } else if (warp == 1 && rank == 0) {
        // matrix instructions: K blocks of 128 bytes, four instructions each
        // (a barrier takes some 200 cycles to answer: the next ones are asked
        // while this K block's instructions are issued)
        Ring<STAGES> at;
        Ring<2> acc;
        bool ok = true, full = false, empty = true;
        const uint64_t op0 = operand(stage0, OPERAND_BYTES / 2);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            const bool mn = MODE == GRAD;
            const uint32_t instr = instr_bf16(TILE, TILE, mn && j.second, mn);
            // along K: 32 bytes of a row, or 16 rows of 128 bytes (operands count 16 bytes)
            const uint32_t step_a = (mn && j.second ? 2048 : 32) / 16, step_b = (mn ? 2048 : 32) / 16;
            int left = 0;  // K blocks to the end of the slice
            for (int kb = 0; kb < j.k_blocks; ++kb) {
                const bool first = left == 0;
                if (first) left = min(p.slice, j.k_blocks - kb);
                const bool last = --left == 0;
                if (!__all_sync(0xffffffffu, full) && !(ok = bar_wait_warp<true>(full0 + 8 * at.slot, at.parity, patience)))
                    break;
                if (first && !__all_sync(0xffffffffu, empty) &&
                    !(ok = bar_wait_warp<true>(acc_empty0 + 8 * acc.slot, acc.parity ^ 1, patience)))
                    break;
                const uint32_t slot = at.slot, buf = acc.slot;
                at.step();
                full = bar_test(full0 + 8 * at.slot, at.parity);
                if (last) {
                    acc.step();
                    empty = bar_test(acc_empty0 + 8 * acc.slot, acc.parity ^ 1);
                }
                fence_after();
                if (elected()) {
                    const uint64_t oa = op0 + slot * (STAGE_BYTES / 16), ob = oa + OPERAND_BYTES / 16;
                    const uint32_t d = tmem + buf * TILE;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        mma<true, false>(d, oa + q * step_a, ob + q * step_b, instr, !first || q > 0);
                    mma_commit<true>(empty0 + 8 * slot);
                    if (last) mma_commit<true>(acc_full0 + 8 * buf);
                }
                __syncwarp();
            }
        }
    } else if (warp >= 2) {
        const int quarter = warp % 4, half = (warp - 2) / 4;
        Ring<2> acc;
        bool ok = true;
        const uint32_t lead_empty0 = map_to(acc_empty0, 0);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            const Job j = job_of<MODE>(p, job);
            const int row0 = j.m0 + (int)rank * 128 + quarter * 32, row = row0 + lane;
            const int rows = MODE != GRAD ? p.M : j.second ? p.N : p.rows;
            const bool work = row0 < rows;
            unsigned char* patch = patches + (warp - 2) * OUT_PATCH;
            if constexpr (!SLICED) {
                const float unit = *p.unit;
                ok = bar_wait_warp(acc_full0 + 8 * acc.slot, acc.parity, patience);
                if (!ok) break;
                fence_after();
                if (work) grad_tile(p, j, tmem + (quarter << 21) + acc.slot * TILE + half * 128, row, half, unit, patch);
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(lead_empty0 + 8 * acc.slot);
                acc.step();
                continue;
            }
            int target = -1;
            float lse = 0.0f, g = 0.0f;
            if (MODE == GRAD) g = *p.unit;
            if (MODE != GRAD && row < rows) target = p.targets[row];
            if (MODE == DZ) {
                if (target >= p.rows) target = -1;  // DZ: rows holds the vocabulary
                if (target >= 0) lse = p.lse[row], g = __fdiv_rn(p.grad[row], *p.unit);
            }
            const int slices = (j.k_blocks - 1) / p.slice + 1;
            // the slices' sums added up in 128 registers: tensor memory cuts its
            // sums rather than rounding them (LOGIT_SLICE, GRAD_SLICE)
            float sum[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
            for (int q = 0; q < slices; ++q, acc.step()) {
                ok = bar_wait_warp(acc_full0 + 8 * acc.slot, acc.parity, patience);
                if (!ok) break;
                fence_after();
                if (work) {
#pragma unroll
                    for (int c = 0; c < 128; c += 32) {
                        float v[32];
                        tmem_load32(tmem + (quarter << 21) + acc.slot * TILE + half * 128 + c, v);
                        tmem_wait_load(v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) sum[c + i] += v[i];
                    }
                }
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(lead_empty0 + 8 * acc.slot);
            }
            if (!ok) break;
            if (work) {
                if constexpr (MODE == LSE)
                    softmax_sums(p, j, sum, row, half, row < rows, target);
                else if constexpr (MODE == DZ)
                    dz_tile(p, j, sum, row, half, target, lse, g, patch);
                else
                    grad_tile(p, j, sum, row, half, g, patch);
            }
        }
        // the last boxes leave shared memory, and arrive, before the CTA does
        if (MODE != LSE && lane == 0) tma_store_wait();
    }
    let_land(patience);
    fence_before();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        tmem_free<true>(tmem, 512);
    }
    cluster_sync();
}

// ---------------------------------------------------------------- 8-bit product
// The block-scaled product of many rows. Scales differ from K block to K
// block, so each block's sums leave tensor memory after four instructions and
// are added up in registers: a round trip (instructions, signal, read, signal
// back) per two blocks, which sets the pace: no pipe is full (below), and the
// power limit adds a seventh in a loop. What shortens it: sixteen epilogue
// warps of 64 columns each (four loads and 32 packed fmas a block), accumulators
// handed over in halves of 128 columns, so that one half is read while the other
// is filled, and scales brought to shared memory by asynchronous copies 16 K
// blocks ahead (read from global memory they cost 800 cycles a block).
// Measured: 256 x 4096 x 151936 in 223 us (tensor pipe 36%
// active, 1.00x of the bytes), 255 in a loop at 1.58 GHz; 4096 x 4048 x 16384 in
// 350 us = 1.55 PFLOP/s.
constexpr int WIDE_EPI = 16;
constexpr int WIDE_THREADS = 32 * (2 + WIDE_EPI);
constexpr int CHUNK = 16;   // K blocks of scales copied at once
constexpr int CHUNK_BUFS = 3;
constexpr int PATCH_ROWS = 16, PATCH_PITCH = 9;  // a warp's patch for stores to unaligned rows: 8 columns
struct WideControl {
    uint64_t full[STAGES], empty[STAGES];
    uint64_t acc_full[4], acc_empty[4];  // [buffer][half]
    uint64_t scales_full[CHUNK_BUFS], scales_free[CHUNK_BUFS];
    uint32_t tmem;
    int gave_up;
};
struct WideScales {
    float x[CHUNK][128];  // this CTA's rows
    float w[2][CHUNK];    // the tile's two column blocks
};
constexpr int WIDE_SMEM = 1024 + STAGES * STAGE_BYTES + CHUNK_BUFS * (int)sizeof(WideScales) +
                          WIDE_EPI * PATCH_ROWS * PATCH_PITCH * 4 + (int)sizeof(WideControl);
static_assert(WIDE_SMEM <= 232448, "shared memory of a CTA");

struct WideParams {
    CUtensorMap a, b;
    int m_tiles, n_tiles, k_blocks, jobs, M, V;
    int* status;
    unsigned long long wait_ns;
    const float* sx;
    const float* sw;
    long long sx_stride, sw_stride, out_stride;
    void* out;
    int out_bf16;
    int wide;  // 32-byte stores reach every row of out
};

__device__ __forceinline__ void copy4_async(uint32_t dst, const float* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Copies one chunk of a tile's scales; every epilogue thread takes its part
// and arrives on `bar` when its copies have landed.
__device__ __forceinline__ void copy_scales(const WideParams& p, WideScales* to, uint32_t bar, int job, int rank, int chunk,
                                            int thread) {
    int m, n;
    tile_of(job, p.m_tiles, p.n_tiles, m, n);
    const int k0 = chunk * CHUNK, have = min(CHUNK, p.k_blocks - k0);
    const int kb = thread % CHUNK;
    if (kb < have) {
#pragma unroll
        for (int i = 0; i < 128 * CHUNK / (32 * WIDE_EPI); ++i) {
            const int r = thread / CHUNK + i * (32 * WIDE_EPI / CHUNK), row = min(m * TILE + rank * 128 + r, p.M - 1);
            copy4_async(smem_addr(&to->x[kb][r]), p.sx + row * p.sx_stride + k0 + kb);
        }
        if (thread < 2 * CHUNK) {
            const int block = min(n * 2 + thread / CHUNK, (p.V + 127) / 128 - 1);
            copy4_async(smem_addr(&to->w[thread / CHUNK][kb]), p.sw + block * p.sw_stride + k0 + kb);
        }
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// 64 columns of a row. Rows on 32-byte boundaries: each thread stores whole
// sectors of its own. Otherwise the warp turns patches of 16 rows and 8
// columns in shared memory, and stores four rows' 8 values at a time.
__device__ __forceinline__ void store_row64(const WideParams& p, const float (&v)[64], int row, int row0, int col, float* patch) {
    if (p.wide && col + 64 <= p.V) {
        if (row >= p.M) return;
        uint32_t w[8];
        if (p.out_bf16) {
            uint16_t* out = (uint16_t*)p.out + row * p.out_stride + col;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = pack_bf16(v[16 * h + 2 * i], v[16 * h + 2 * i + 1]);
                store32(out + 16 * h, w);
            }
        } else {
            float* out = (float*)p.out + row * p.out_stride + col;
#pragma unroll
            for (int h = 0; h < 8; ++h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[8 * h + i]);
                store32(out + 8 * h, w);
            }
        }
        return;
    }
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int c = 0; c < 64; c += 8) {
        if (col + c >= p.V) break;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
            if (lane / PATCH_ROWS == part) {
#pragma unroll
                for (int i = 0; i < 8; ++i) patch[lane % PATCH_ROWS * PATCH_PITCH + i] = v[c + i];
            }
            __syncwarp();
#pragma unroll
            for (int r = lane / 8; r < PATCH_ROWS; r += 4) {
                const int at_row = row0 + part * PATCH_ROWS + r, at_col = col + c + lane % 8;
                if (at_row < p.M && at_col < p.V) {
                    const float f = patch[r * PATCH_PITCH + lane % 8];
                    const long long at = at_row * p.out_stride + at_col;
                    if (p.out_bf16)
                        ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(f);
                    else
                        ((float*)p.out)[at] = f;
                }
            }
            __syncwarp();
        }
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WIDE_THREADS, 1) wide_kernel(const __grid_constant__ WideParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    WideScales* scales = (WideScales*)(smem + STAGES * STAGE_BYTES);
    float* patches = (float*)(scales + CHUNK_BUFS);
    WideControl* ctl = (WideControl*)(patches + WIDE_EPI * PATCH_ROWS * PATCH_PITCH);
    const uint32_t stage0 = smem_addr(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cta_rank();
    const int pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    const uint32_t full0 = smem_addr(ctl->full), empty0 = smem_addr(ctl->empty);
    const uint32_t acc_full0 = smem_addr(ctl->acc_full), acc_empty0 = smem_addr(ctl->acc_empty);
    const uint32_t scales_full0 = smem_addr(ctl->scales_full), scales_free0 = smem_addr(ctl->scales_free);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            bar_init(full0 + 8 * s, 1);
            bar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 4; ++b) {
            bar_init(acc_full0 + 8 * b, 1);
            bar_init(acc_empty0 + 8 * b, WIDE_EPI);  // half the epilogue warps of both CTAs
        }
        for (int b = 0; b < CHUNK_BUFS; ++b) {
            bar_init(scales_full0 + 8 * b, 32 * WIDE_EPI);
            bar_init(scales_free0 + 8 * b, WIDE_EPI);
        }
        ctl->gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&p.a);
        tma_prefetch_map(&p.b);
    }
    if (warp == 1) tmem_alloc<true>(smem_addr(&ctl->tmem), 512);
    __syncwarp();
    fence_before();
    cluster_sync();
    fence_after();
    const uint32_t tmem = ctl->tmem;
    const Patience patience = {&ctl->gave_up, p.status, p.wait_ns};

    if (warp == 0) {
        Ring<STAGES> at;
        bool ok = true;
        const uint32_t lead_full0 = map_to(full0, 0);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            int m, n;
            tile_of(job, p.m_tiles, p.n_tiles, m, n);
            for (int kb = 0; kb < p.k_blocks; ++kb, at.step()) {
                if (!(ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience))) break;
                if (elected()) {
                    const uint32_t full = lead_full0 + 8 * at.slot, da = stage0 + at.slot * STAGE_BYTES;
                    if (rank == 0) bar_expect(full0 + 8 * at.slot, 2 * STAGE_BYTES);
                    tma_load<true>(da, &p.a, kb * 128, m * TILE + rank * 128, full);
                    tma_load<true>(da + OPERAND_BYTES, &p.b, kb * 128, n * TILE + rank * 128, full);
                }
                __syncwarp();
            }
        }
        for (int back = 0; ok && back < STAGES; ++back, at.step())
            ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience);
    } else if (warp == 1 && rank == 0) {
        Ring<STAGES> at;
        Ring<2> acc;
        bool ok = true, full = false, empty[2] = {true, true};
        const uint64_t op0 = operand(stage0, 0);
        constexpr uint32_t instr = instr_e4m3(TILE, TILE / 2);
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            for (int kb = 0; ok && kb < p.k_blocks; ++kb) {
                if (!__all_sync(0xffffffffu, full) && !(ok = bar_wait_warp<true>(full0 + 8 * at.slot, at.parity, patience)))
                    break;
                const uint32_t slot = at.slot, buf = acc.slot;
                at.step();
                full = bar_test(full0 + 8 * at.slot, at.parity);
                const uint64_t oa = op0 + slot * (STAGE_BYTES / 16), ob = oa + OPERAND_BYTES / 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!__all_sync(0xffffffffu, empty[h]) &&
                        !(ok = bar_wait_warp<true>(acc_empty0 + 16 * buf + 8 * h, acc.parity ^ 1, patience)))
                        break;
                    fence_after();
                    if (elected()) {
                        // 64 weight rows of either CTA: the half's columns are 64 of each column block
                        const uint64_t obh = ob + h * (64 * 128 / 16);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            mma<true, true>(tmem + buf * TILE + h * (TILE / 2), oa + 2 * q, obh + 2 * q, instr, q > 0);
                        mma_commit<true>(acc_full0 + 16 * buf + 8 * h);
                        if (h == 1) mma_commit<true>(empty0 + 8 * slot);
                    }
                    __syncwarp();
                }
                acc.step();
                empty[0] = bar_test(acc_empty0 + 16 * acc.slot, acc.parity ^ 1);
                empty[1] = bar_test(acc_empty0 + 16 * acc.slot + 8, acc.parity ^ 1);
            }
        }
    } else if (warp >= 2) {
        const int thread = threadIdx.x - 64, e = warp - 2, quarter = warp % 4, half = e / 4 / 2, block = e / 4 % 2;
        const int chunks = (p.k_blocks + CHUNK - 1) / CHUNK;
        Ring<2> acc;
        Ring<CHUNK_BUFS> sc, ahead;  // the chunk in use, and the next to copy
        bool ok = true;
        const uint32_t full = acc_full0 + 8 * half, lead_empty = map_to(acc_empty0 + 8 * half, 0);
        const uint32_t lanes = tmem + (quarter << 21) + half * (TILE / 2) + block * 64;
        if (pair < p.jobs) {
            copy_scales(p, scales + ahead.slot, scales_full0 + 8 * ahead.slot, pair, rank, 0, thread);
            ahead.step();
        }
        for (int job = pair; ok && job < p.jobs; job += pairs) {
            int m, n;
            tile_of(job, p.m_tiles, p.n_tiles, m, n);
            const int row0 = m * TILE + (int)rank * 128 + quarter * 32, row = row0 + lane;
            const int col = n * TILE + block * 128 + half * 64;
            const bool work = row0 < p.M && col < p.V;
            float sum[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) sum[i] = 0.0f;
            for (int c = 0; ok && c < chunks; ++c) {
                const bool more = c + 1 < chunks;
                if (more || job + pairs < p.jobs) {
                    ok = bar_wait_warp(scales_free0 + 8 * ahead.slot, ahead.parity ^ 1, patience);
                    if (!ok) break;
                    copy_scales(p, scales + ahead.slot, scales_full0 + 8 * ahead.slot, more ? job : job + pairs, rank,
                                more ? c + 1 : 0, thread);
                    ahead.step();
                }
                ok = bar_wait_warp(scales_full0 + 8 * sc.slot, sc.parity, patience);
                if (!ok) break;
                const float* xs = &scales[sc.slot].x[0][quarter * 32 + lane];
                const float* ws = scales[sc.slot].w[block];
                const int have = min(CHUNK, p.k_blocks - c * CHUNK);
                for (int kb = 0; kb < have; ++kb, acc.step()) {
                    const float s = xs[kb * 128] * ws[kb];
                    ok = bar_wait_warp(full + 16 * acc.slot, acc.parity, patience);
                    if (!ok) break;
                    fence_after();
                    if (work) {
                        const Two s2(s);
#pragma unroll
                        for (int q = 0; q < 64; q += 16) {
                            float v[16];
                            tmem_load16(lanes + acc.slot * TILE + q, v);
                            tmem_wait_load(v);
#pragma unroll
                            for (int i = 0; i < 16; i += 2)
                                fma2(Two(v[i], v[i + 1]), s2, Two(sum[q + i], sum[q + i + 1])).get(sum[q + i], sum[q + i + 1]);
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive_cluster(lead_empty + 16 * acc.slot);
                }
                __syncwarp();
                if (lane == 0) bar_arrive(scales_free0 + 8 * sc.slot);
                sc.step();
            }
            if (ok && work) store_row64(p, sum, row, row0, col, patches + e * PATCH_ROWS * PATCH_PITCH);
        }
    }
    let_land(patience);
    fence_before();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        tmem_free<true>(tmem, 512);
    }
    cluster_sync();
}

// ---------------------------------------------------------------- few rows
// A decode step's rows (at most 128; 64 for the cross entropy) against the
// whole head: the weight's bytes bound it. Here the weight's rows are the
// lanes: a CTA multiplies 128 of them by COLS hidden rows at once, so that
// the matrix instructions cost COLS columns instead of 256, and tensor memory
// holds 512 / COLS accumulators (up to eight are used), which hides the
// epilogue's round trip behind the weight's loads. Every CTA works alone.
// Measured: 8-bit, 1 x 4096 x 151936 in 105 us = 5.9 TB/s (91% of the copy rate),
// loss of 1 x 2048 x 151936 in 102 us = 6.1 TB/s with its join.
template <int MODE, int COLS>
struct Skinny {
    static constexpr int PART = COLS < 32 ? COLS : 32;  // columns of an epilogue warp: four warps for each 32
    static constexpr int EPI = 4 * (COLS / PART), THREADS = 64 + 32 * EPI;
    static constexpr int A_BYTES = 16384, B_BYTES = COLS * 128, STAGE = A_BYTES + B_BYTES;
    static constexpr int DEPTH = 196608 / STAGE > 10 ? 10 : 196608 / STAGE;
    static constexpr int BUFS = 512 / COLS > 8 ? 8 : 512 / COLS;
    static constexpr int TABLE = 32768;  // bytes of scales, MODE FP8
    static constexpr int SMEM = 1024 + DEPTH * STAGE + TABLE + 256;
};
struct SkinnyControl {
    uint64_t full[10], empty[10], acc_full[8], acc_empty[8];
    uint32_t tmem;
    int gave_up;
};
static_assert(sizeof(SkinnyControl) <= 512, "control block");

struct SkinnyParams {
    CUtensorMap a, b;  // weight (a tile's rows a box) and hidden rows (COLS a box)
    int V, M, k_blocks, slice, jobs;
    int tile;          // weight rows of a tile: at most 128, so that every CTA has the same number of tiles
    int* status;
    unsigned long long wait_ns;
    const int32_t* targets;
    float softcap;
    float2* part;         // LSE: [4 CTAs][M]: a warp's maxima and sums over all its tiles
    float* target_logit;
    const float* lse;     // DZ
    const float* grad;
    uint16_t* dz;         // DZ: [2 M][dz_pitch]: the V vocabulary columns from n0, and below what rounding left
    long long dz_pitch;
    int n0, V_total;
    const float* sx;
    const float* sw;
    long long sx_stride, sw_stride, out_stride;
    void* out;
    int out_bf16;
};

// COLS columns of this warp's lanes from tensor memory, added (times a scale
// per column) to sum.
template <int MODE, int COLS>
__device__ __forceinline__ void take(uint32_t addr, float (&sum)[COLS], const float* sx, float sw) {
#pragma unroll
    for (int c = 0; c < COLS; c += 16) {
        float v[16];
        tmem_load16(addr + c, v);
        tmem_wait_load(v);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            if (MODE == FP8) {
                const ulonglong2 x = *(const ulonglong2*)(sx + c + i);
                fma2(Two(v[i], v[i + 1]), mul2(Two((uint64_t)x.x), Two(sw)), Two(sum[c + i], sum[c + i + 1])).get(sum[c + i], sum[c + i + 1]);
                fma2(Two(v[i + 2], v[i + 3]), mul2(Two((uint64_t)x.y), Two(sw)), Two(sum[c + i + 2], sum[c + i + 3]))
                    .get(sum[c + i + 2], sum[c + i + 3]);
            } else {
#pragma unroll
                for (int q = i; q < i + 4; ++q) sum[c + q] += v[q];
            }
        }
    }
}

template <int MODE, int COLS>
__global__ void __launch_bounds__(Skinny<MODE, COLS>::THREADS, 1) skinny_kernel(const __grid_constant__ SkinnyParams p) {
    using S = Skinny<MODE, COLS>;
    constexpr int PART = S::PART;
    extern __shared__ unsigned char smem_raw[];
    __shared__ SkinnyControl ctl;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* table = (float*)(smem + S::DEPTH * S::STAGE);  // FP8: scales [K block][COLS]; DZ: lse, gradient, target [COLS]
    const uint32_t stage0 = smem_addr(smem);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::DEPTH; ++s) {
            bar_init(smem_addr(&ctl.full[s]), 1);
            bar_init(smem_addr(&ctl.empty[s]), 1);
        }
        for (int b = 0; b < S::BUFS; ++b) {
            bar_init(smem_addr(&ctl.acc_full[b]), 1);
            bar_init(smem_addr(&ctl.acc_empty[b]), S::EPI);
        }
        ctl.gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&p.a);
        tma_prefetch_map(&p.b);
    }
    if (warp == 1) tmem_alloc<false>(smem_addr(&ctl.tmem), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ctl.tmem;
    const Patience patience = {&ctl.gave_up, p.status, p.wait_ns};
    const uint32_t full0 = smem_addr(ctl.full), empty0 = smem_addr(ctl.empty);
    const uint32_t acc_full0 = smem_addr(ctl.acc_full), acc_empty0 = smem_addr(ctl.acc_empty);
    launch_next();
    wait_previous();
    if (warp == 0) {
        Ring<S::DEPTH> at;
        bool ok = true;
        for (int job = blockIdx.x; ok && job < p.jobs; job += gridDim.x) {
            for (int kb = 0; kb < p.k_blocks; ++kb, at.step()) {
                if (!(ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience))) break;
                if (elected()) {
                    const uint32_t full = full0 + 8 * at.slot, da = stage0 + at.slot * S::STAGE;
                    bar_expect(full, p.tile * 128 + S::B_BYTES);
                    const int x = kb * (MODE == FP8 ? 128 : 64);
                    tma_load<false>(da, &p.a, x, job * p.tile, full);
                    tma_load<false>(da + S::A_BYTES, &p.b, x, 0, full);
                }
                __syncwarp();
            }
        }
        for (int back = 0; ok && back < S::DEPTH; ++back, at.step())
            ok = bar_wait_warp(empty0 + 8 * at.slot, at.parity ^ 1, patience);
    } else if (warp == 1) {
        Ring<S::DEPTH> at;
        Ring<S::BUFS> acc;
        bool ok = true, full = false, empty = true;
        const uint64_t op0 = operand(stage0, 0);
        const uint32_t instr = MODE == FP8 ? instr_e4m3(128, COLS) : instr_bf16(128, COLS, false, false);
        for (int job = blockIdx.x; ok && job < p.jobs; job += gridDim.x) {
            int left = 0;  // K blocks to the end of the slice
            for (int kb = 0; kb < p.k_blocks; ++kb) {
                const bool first = left == 0;
                if (first) left = min(p.slice, p.k_blocks - kb);
                const bool last = --left == 0;
                if (!__all_sync(0xffffffffu, full) && !(ok = bar_wait_warp<true>(full0 + 8 * at.slot, at.parity, patience)))
                    break;
                if (first && !__all_sync(0xffffffffu, empty) &&
                    !(ok = bar_wait_warp<true>(acc_empty0 + 8 * acc.slot, acc.parity ^ 1, patience)))
                    break;
                const uint32_t slot = at.slot, buf = acc.slot;
                at.step();
                full = bar_test(full0 + 8 * at.slot, at.parity);
                if (last) {
                    acc.step();
                    empty = bar_test(acc_empty0 + 8 * acc.slot, acc.parity ^ 1);
                }
                fence_after();
                if (elected()) {
                    const uint64_t oa = op0 + slot * (S::STAGE / 16), ob = oa + S::A_BYTES / 16;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        mma<false, MODE == FP8>(tmem + buf * COLS, oa + 2 * q, ob + 2 * q, instr, !first || q > 0);
                    mma_commit<false>(empty0 + 8 * slot);
                    if (last) mma_commit<false>(acc_full0 + 8 * buf);
                }
                __syncwarp();
            }
        }
    } else {
        const int quarter = warp % 4, c0 = (warp - 2) / 4 * PART, mine = p.M - c0;  // rows from c0
        // what the epilogue needs of the rows; the loads are under way meanwhile
        const int thread = threadIdx.x - 64;
        if (MODE == DZ && thread < COLS) {
            const int t = thread < p.M ? p.targets[thread] : -1;
            const bool has = t >= 0 && t < p.V_total;
            table[thread] = has ? p.lse[thread] : 0.0f;
            table[COLS + thread] = has ? p.grad[thread] : 0.0f;
            ((int*)table)[2 * COLS + thread] = has ? t - p.n0 : INT32_MIN;
        }
        if (MODE == FP8) {
            // the rows' scales, K block by K block: every lane reads the same four at a time
            for (int i = thread; i < p.k_blocks * COLS; i += 32 * S::EPI) {
                const int m = i % COLS;
                table[i] = m < p.M ? p.sx[m * p.sx_stride + i / COLS] : 0.0f;
            }
        }
        if (MODE != LSE) asm volatile("bar.sync 1, %0;" ::"n"(32 * S::EPI) : "memory");
        const uint32_t base = tmem + (quarter << 21) + c0;
        const int slices = (p.k_blocks + p.slice - 1) / p.slice;
        Ring<S::BUFS> acc;
        bool ok = true;
        // LSE: each lane's running maximum and sum per row over all its weight rows
        float mx[MODE == LSE ? PART : 1], se[MODE == LSE ? PART : 1];
#pragma unroll
        for (int i = 0; i < (MODE == LSE ? PART : 1); ++i) mx[i] = -3.402823466e38f, se[i] = 0.0f;
        for (int job = blockIdx.x; ok && job < p.jobs; job += gridDim.x) {
            const int v = job * p.tile + quarter * 32 + lane;
            const bool live = quarter * 32 + lane < p.tile && v < p.V;
            // FP8: scales of the one or two blocks of weight rows the tile lies in, 32 K blocks in the lanes
            const int block0 = job * p.tile / FP8_BLOCK, block1 = min(block0 + 1, (p.V - 1) / FP8_BLOCK);
            const bool second = v / FP8_BLOCK > block0;
            float sum[PART], w32 = 0.0f, w32b = 0.0f;
#pragma unroll
            for (int i = 0; i < PART; ++i) sum[i] = 0.0f;
            for (int kb = 0; kb < slices; ++kb, acc.step()) {
                float now = 1.0f;
                if (MODE == FP8) {
                    if (kb % 32 == 0) {
                        const int at = min(kb + lane, slices - 1);
                        w32 = p.sw[block0 * p.sw_stride + at];
                        w32b = p.sw[block1 * p.sw_stride + at];
                    }
                    const float a = __shfl_sync(0xffffffffu, w32, kb % 32), b = __shfl_sync(0xffffffffu, w32b, kb % 32);
                    now = second ? b : a;
                }
                ok = bar_wait_warp(acc_full0 + 8 * acc.slot, acc.parity, patience);
                if (!ok) break;
                fence_after();
                if (mine > 0) take<MODE, PART>(base + acc.slot * COLS, sum, table + kb * COLS + c0, now);
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(acc_empty0 + 8 * acc.slot);
            }
            if (!ok || !live) continue;
            if constexpr (MODE == LSE) {
#pragma unroll
                for (int c = 0; c < PART; c += 16) logits_of(reinterpret_cast<float(&)[16]>(sum[c]), p.softcap);
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    if (i < mine) {
                        // one exponential: the larger of the two terms is 1
                        const float l = sum[i], e = exp2_approx(-fabsf(l - mx[i]) * LOG2E);
                        se[i] = l > mx[i] ? fmaf(se[i], e, 1.0f) : se[i] + e;
                        mx[i] = fmaxf(mx[i], l);
                        if (p.targets[c0 + i] == v) p.target_logit[c0 + i] = l;
                    }
                }
            } else if constexpr (MODE == DZ) {
                const float inv = p.softcap > 0.0f ? 1.0f / p.softcap : 0.0f;
#pragma unroll
                for (int c = 0; c < PART; c += 16) logits_of(reinterpret_cast<float(&)[16]>(sum[c]), p.softcap);
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    if (i < mine) {
                        const int at = ((const int*)table)[2 * COLS + c0 + i];
                        const float d = dz_of(sum[i], table[c0 + i], table[COLS + c0 + i], inv, at == v, at == INT32_MIN);
                        const __nv_bfloat16 high = __float2bfloat16_rn(d);
                        __nv_bfloat16* out = (__nv_bfloat16*)p.dz + (c0 + i) * p.dz_pitch + v;
                        out[0] = high;
                        out[p.M * p.dz_pitch] = __float2bfloat16_rn(d - __bfloat162float(high));
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    if (i < mine) {
                        const long long at = (c0 + i) * p.out_stride + v;
                        if (p.out_bf16)
                            ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(sum[i]);
                        else
                            ((float*)p.out)[at] = sum[i];
                    }
                }
            }
        }
        __syncwarp();
        if constexpr (MODE == LSE) {
#pragma unroll
            for (int i = 0; i < PART; ++i) {
                if (i < mine) {
#pragma unroll
                    for (int o = 16; o; o >>= 1) {
                        const float m2 = __shfl_xor_sync(0xffffffffu, mx[i], o), s2 = __shfl_xor_sync(0xffffffffu, se[i], o);
                        const float top = fmaxf(mx[i], m2);
                        se[i] = se[i] * exp2_approx((mx[i] - top) * LOG2E) + s2 * exp2_approx((m2 - top) * LOG2E);
                        mx[i] = top;
                    }
                    if (lane == 0) p.part[(long long)(blockIdx.x * 4 + quarter) * p.M + c0 + i] = make_float2(mx[i], se[i]);
                }
            }
        }
    }
    let_land(patience);
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_free<false>(tmem, 512);
    }
}

// ---------------------------------------------------------------- joins
// lse of a row from its parts' maxima and sums. A block takes eight rows and
// 128 parts at a time (four a warp), eight such rounds in flight: the sums of
// few rows come in up to two thousand parts, and their latency is the kernel.
__global__ void __launch_bounds__(1024) lse_join_kernel(const float2* part, const float* target_logit, const int32_t* targets,
                                                        int N, int V, int parts, float* loss, float* lse_out) {
    __shared__ float2 red[32][8];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, row = blockIdx.x * 8 + lane % 8;
    float mx = -INFINITY, sum = 0.0f;
    wait_previous();
    for (int q = warp * 4 + lane / 8; q < parts; q += 128 * 8) {
        float2 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = row < N && q + 128 * i < parts ? part[(long long)(q + 128 * i) * N + row] : make_float2(-INFINITY, 0.0f);
        float top = mx;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i].x);
        const float ref = top == -INFINITY ? 0.0f : top;
        sum *= exp2_approx((mx - ref) * LOG2E);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += x[i].y * exp2_approx((x[i].x - ref) * LOG2E);
        mx = top;
    }
#pragma unroll
    for (int o = 8; o < 32; o *= 2) {
        const float m2 = __shfl_xor_sync(0xffffffffu, mx, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        const float top = fmaxf(mx, m2), ref = top == -INFINITY ? 0.0f : top;
        sum = sum * exp2_approx((mx - ref) * LOG2E) + s2 * exp2_approx((m2 - ref) * LOG2E);
        mx = top;
    }
    if (lane < 8) red[warp][lane] = make_float2(mx, sum);
    __syncthreads();
    if (threadIdx.x >= 256) return;
    // eight warps: warp w joins row w's 32 partial sums
    const float2 x = red[lane][warp];
    mx = x.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    sum = x.y * exp2_approx((x.x - ref) * LOG2E);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int r = blockIdx.x * 8 + warp;
    if (lane == 0 && r < N) {
        const float lse = ref + logf(sum);
        const int t = targets[r];
        lse_out[r] = lse;
        loss[r] = t < 0 ? 0.0f : t < V ? lse - target_logit[r] : NAN;
    }
}

// What dz is held over before its rounding: the mantissa, 1 to 2, of the first
// gradient that is a normal number (1 without one). Under a mean over rows all
// gradients are one number g, and a confident row's target has dz = -g: rounded
// to bf16 that would be off by the same up to 2^-8 in every row, which no sum
// averages out. Over its mantissa g is a power of two; the results are
// multiplied by it in 32 bits. Block 0's threads look through the rows 256 at a time.
__device__ __forceinline__ void find_unit(const int32_t* targets, const float* grad, int N, int V, float* unit) {
    __shared__ int first;
    if (threadIdx.x == 0) first = INT32_MAX;
    __syncthreads();
    for (int r0 = 0; r0 < N; r0 += 256) {
        const int r = r0 + (int)threadIdx.x;
        bool has = false;
        if (r < N && targets[r] >= 0 && targets[r] < V) {
            const uint32_t e = __float_as_uint(grad[r]) >> 23 & 255;
            has = e > 0 && e < 255;
        }
        if (has) atomicMin(&first, r);
        if (__syncthreads_or(has)) break;
    }
    if (threadIdx.x == 0)
        *unit = first == INT32_MAX ? 1.0f : __uint_as_float((__float_as_uint(grad[first]) & 0x7fffffu) | 0x3f800000u);
}

// The hidden rows as d_weight's sums take them: zeros where a row has no
// gradient, so that whatever lies there (padding, an infinity, a NaN) does not
// meet its zero dz; parts times one below the other. dz in two parts needs no
// unit: it is 1.
__global__ void __launch_bounds__(256) live_rows_kernel(const uint16_t* hidden, long long stride, const int32_t* targets,
                                                        const float* grad, int N, int D, int V, int parts, uint16_t* out,
                                                        float* unit) {
    const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8, n = (long long)N * D;
    launch_next();
    if (blockIdx.x == 0) find_unit(targets, grad, parts == 1 ? N : 0, V, unit);
    if (i >= n) return;
    const long long row = i / D;
    const int t = targets[row];
    uint4 w = make_uint4(0, 0, 0, 0);
    if (t >= 0 && t < V) w = *(const uint4*)(hidden + row * stride + i % D);
    for (int q = 0; q < parts; ++q) *(uint4*)(out + q * n + i) = w;
}

// d_hidden = the slabs' sum (and the parts' of each) in their order, times the
// unit, rounded once; eight columns a thread.
__global__ void __launch_bounds__(256) dh_join_kernel(const float* slabs, int slices, int N, int D, const float* unit,
                                                      uint16_t* dh, long long dh_stride) {
    const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 8, n = (long long)N * D;
    if (i >= n) return;
    wait_previous();
    float v[8] = {};
    for (int s = 0; s < slices; ++s) {
        const float4 x = *(const float4*)(slabs + s * n + i), y = *(const float4*)(slabs + s * n + i + 4);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
    }
    const float u = *unit;
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] *= u;
    const uint4 w = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    *(uint4*)(dh + i / D * dh_stride + i % D) = w;
}

// ---------------------------------------------------------------- quantiser
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// What quantising by a scale needs: -s, 1 / s (to a step), (2^19 + 1) / s
// and 2^38 / s.
struct Quotient {
    Two minus_s, inv, inv_split;
    float inv_big;
    __device__ __forceinline__ Quotient(float s, float inv)
        : minus_s(-s), inv(inv), inv_split(inv * 524289.0f), inv_big(inv * 0x1p38f) {}
};

// Two values whose rounding to e4m3 is that of the exact quotients x / s. The
// product x inv is off by a few 2^-24, which decides wrongly beside a border
// between two codes (a few per thousand of bf16 activations lie on one to
// 2^-24: their few bits over their block's own largest). So it is first cut
// to h of five bits (Veltkamp's splitting: a sum with 2^19 times itself
// leaves them): every code and every border is such a number. Which side of h
// the quotient lies on is the sign of the remainder x - h s, whose fma is
// exact enough: the remainder is 0 or at least 2^-39 s (29 bits of h s, h from
// 2^-10 up). That sign, made by a saturated fma, moves h by 1.5 2^-16: enough
// to leave the largest border (432, steps of 2^-15), and less than the way
// to a border from the numbers beside the smallest one (2^-10 - 2^-15). A true
// tie stays on its border and rounds to the even code. All of it runs on
// the FMA pipe, two values an instruction, and takes no branch.
__device__ __forceinline__ void round_as_quotients(float& a, float& b, const Quotient& q) {
    const Two x(a, b), g = mul2(x, q.inv_split), minus(-1.0f);
    const Two h = add2(g, fma2(g, minus, mul2(x, q.inv)));
    float ra, rb;
    fma2(h, q.minus_s, x).get(ra, rb);
    const Two side = add2(Two(__saturatef(fmaf(ra, q.inv_big, 0.5f)), __saturatef(fmaf(rb, q.inv_big, 0.5f))), Two(-0.5f));
    fma2(side, Two(3.0f * 0x1p-16f), h).get(a, b);
}

// A quantisation block's scale, the largest magnitude (top, as bits; an
// infinity or a NaN: NaN for all) over 448 rounded once. In the range of
// quantize8: the product with 1/448, corrected by its exact remainder
// (P. Markstein, IBM J. Res. Develop. 34(1), 1990; every mantissa is tested),
// in a quarter of a division's instructions.
constexpr float SMALL_SCALE = 0x1p-60f;
__device__ __forceinline__ float block_scale(uint32_t top) {
    const float t = __uint_as_float(top), r = 1.0f / 448.0f, q = t * r;
    const float s = fmaf(fmaf(-q, 448.0f, t), r, q);
    if (s >= SMALL_SCALE && top < 0x7f800000u) return s;
    return top < 0x7f800000u ? __fdiv_rn(t, 448.0f) : NAN;
}
// 1 / s to a step, for s in that range.
__device__ __forceinline__ float reciprocal(float s) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    return r;
}

__device__ __forceinline__ uint2 quantize8(float (&x)[8], const Quotient& q) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 8; i += 2) round_as_quotients(x[i], x[i + 1], q);
#pragma unroll
    for (int h = 0; h < 2; ++h) w[h] = pack_e4m3(x[4 * h], x[4 * h + 1]) | pack_e4m3(x[4 * h + 2], x[4 * h + 3]) << 16;
    return make_uint2(w[0], w[1]);
}

// Scales whose reciprocals or remainders leave the range, and NaN.
__device__ __forceinline__ uint2 quantize8_small(float (&x)[8], float s) {
    if (s > 0.0f) {  // lifted by an exact power of two
        s *= 0x1p100f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= 0x1p100f;
        return quantize8(x, Quotient(s, reciprocal(s)));
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // 0: a block of zeros, or one whose scale underflowed
        const uint32_t code = s == 0.0f ? (x[i] == 0.0f ? 0u : x[i] < 0.0f ? 0xfeu : 0x7eu) : 0x7fu;
        w[i / 4] |= code << (8 * (i % 4));
    }
    return make_uint2(w[0], w[1]);
}

// Eight neighbouring values of a row as they lie in memory; zeros past K.
template <typename T>
struct Eight {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T* row, int k, int K, bool vec) {
        if (vec && k <= K - 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                const uint4 u = *(const uint4*)((const unsigned char*)(row + k) + 16 * i);
                w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) {
                if (sizeof(T) == 2)
                    w[i / 2] |= (uint32_t)((const uint16_t*)row)[k + i] << (16 * (i % 2));
                else
                    w[i % (2 * sizeof(T))] = ((const uint32_t*)row)[k + i];
            }
    }
    // the largest magnitude, as the bits of a float
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) {
            if (sizeof(T) == 2)
                asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
            else
                m = max(m, w[i] & 0x7fffffffu);
        }
        return sizeof(T) == 2 ? max(m & 0xffff0000u, m << 16) : m;
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = __uint_as_float(sizeof(T) == 4 ? w[i % (2 * sizeof(T))] : i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};

__device__ __forceinline__ void store8(uint8_t* row, int k, int K, bool vec, uint2 w) {
    if (vec && k <= K - 8) {
        *(uint2*)(row + k) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < K) row[k + i] = (uint8_t)((i < 4 ? w.x : w.y) >> (8 * (i % 4)));
    }
}

// Blocks of one row: eight threads a block, sixteen values a thread (two
// pieces, so that a load's lanes are neighbours); a warp takes 512 columns of
// four rows with all their loads in flight. Each value is read once and held
// in registers between the maximum and the quotients (8000 x 8192 bf16 in 38
// us = 5.1 TB/s; neither memory, 49% of its peak, nor issue, 56%, is full: a
// warp's loads and its arithmetic take turns, with three CTAs an SM; the square
// blocks' kernel 151936 x 4096 in 277 us = 6.7 TB/s). FULL: whole blocks and
// whole groups of rows on aligned addresses, without checks per value (which
// would cost registers, and a quarter of the rate). A CTA's warps lie below each
// other, so that the few slower ones at the right edge share CTAs.
constexpr int QROWS = 4, QCOLS = 512;
struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    long long x_stride, q_stride, scale_stride;
    int M, K, x_vec, q_vec;
};
template <typename T, bool FULL>
__device__ __forceinline__ void quantize_rows(const QuantArgs& a, int m0, int k0) {
    const int lane = threadIdx.x % 32, k = k0 + lane / 8 * FP8_BLOCK + lane % 8 * 8;
    const int last = FULL ? INT32_MAX : a.K;
    const T* x = (const T*)a.x + m0 * a.x_stride;
    Eight<T> e[QROWS][2];
#pragma unroll
    for (int r = 0; r < QROWS; ++r) {
        e[r][0].load(x, k, last, FULL || a.x_vec);
        e[r][1].load(x, k + 64, last, FULL || a.x_vec);
        if (FULL || m0 + r + 1 < a.M) x += a.x_stride;
    }
    uint8_t* q = a.q + m0 * a.q_stride;
    float* scale = a.scale + m0 * a.scale_stride + k / FP8_BLOCK;
#pragma unroll
    for (int r = 0; r < QROWS; ++r) {
        uint32_t top = max(e[r][0].top(), e[r][1].top());
#pragma unroll
        for (int o = 4; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = block_scale(top);
        if (FULL || m0 + r < a.M) {
            if (lane % 8 == 0 && (FULL || k < a.K)) *scale = s;
            const Quotient quotient(s, reciprocal(s));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                e[r][h].values(v);
                if (FULL || k + 64 * h < a.K)
                    store8(q, k + 64 * h, last, FULL || a.q_vec, s >= SMALL_SCALE ? quantize8(v, quotient) : quantize8_small(v, s));
            }
        }
        q += a.q_stride;
        scale += a.scale_stride;
    }
}
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
    const int k0 = blockIdx.x * QCOLS;
    for (long long m0 = ((long long)blockIdx.y * 8 + threadIdx.x / 32) * QROWS; m0 < a.M; m0 += (long long)gridDim.y * 8 * QROWS) {
        if (a.x_vec && a.q_vec && m0 + QROWS <= a.M && k0 <= a.K - QCOLS)
            quantize_rows<T, true>(a, (int)m0, k0);
        else
            quantize_rows<T, false>(a, (int)m0, k0);
    }
}

// Blocks of 128 x 128: one CTA each, eight rows' values a thread held in
// registers between the maximum and the quotients.
template <typename T, bool FULL>
__device__ __forceinline__ void quantize_square(const QuantArgs& a, int mb, int kb) {
    __shared__ uint32_t red[8];
    const int m0 = mb * FP8_BLOCK + threadIdx.x / 16, k = kb * FP8_BLOCK + threadIdx.x % 16 * 8;
    const int last = FULL ? INT32_MAX : a.K;
    const T* x = (const T*)a.x + (FULL ? m0 : min(m0, a.M - 1)) * a.x_stride;
    const long long x_step = 16 * a.x_stride, q_step = 16 * a.q_stride;
    Eight<T> e[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        e[r].load(x, k, last, FULL || a.x_vec);
        if (FULL || m0 + 16 * (r + 1) < a.M) x += x_step;
    }
    uint32_t top = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) top = max(top, e[r].top());
    top = __reduce_max_sync(0xffffffffu, top);
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, red[i]);
    const float s = block_scale(top);
    if (threadIdx.x == 0) a.scale[mb * a.scale_stride + kb] = s;
    const Quotient quotient(s, reciprocal(s));
    uint8_t* q = a.q + m0 * a.q_stride;
    const bool small = !(s >= SMALL_SCALE);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        if (FULL || (m0 + 16 * r < a.M && k < a.K)) {
            float v[8];
            e[r].values(v);
            store8(q, k, last, FULL || a.q_vec, small ? quantize8_small(v, s) : quantize8(v, quotient));
        }
        q += q_step;
    }
    __syncthreads();  // red is free for the next block
}
template <typename T>
__global__ void __launch_bounds__(256) quantize_square_kernel(const QuantArgs a) {
    const int kb = blockIdx.x, blocks = (a.M - 1) / FP8_BLOCK + 1;
    for (int mb = blockIdx.y; mb < blocks; mb += gridDim.y) {
        if (a.x_vec && a.q_vec && mb < a.M / FP8_BLOCK && kb < a.K / FP8_BLOCK)
            quantize_square<T, true>(a, mb, kb);
        else
            quantize_square<T, false>(a, mb, kb);
    }
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
// box_rows; what lies outside reads as 0 and is not written.
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

// Lets a kernel use its dynamic shared memory, once per context: `bit` is the
// kernel's in *ready.
template <typename K>
cudaError_t allow_smem(K* kernel, int bytes, int bit, uint32_t* ready) {
    if (*ready >> bit & 1) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) *ready |= 1u << bit;
    return e;
}
// Bits: the pair kernel's modes 0 to 2, the wide kernel 3, the few-row kernel's
// modes times column counts from 4, the pair kernel without slices 31.
constexpr int WIDE_BIT = 3, WHOLE_BIT = 31;
constexpr int skinny_bit(int mode, int cols) { return 4 + mode * 4 + (cols == 16 ? 0 : cols == 32 ? 1 : cols == 64 ? 2 : 3); }
static_assert(skinny_bit(FP8, 128) < WHOLE_BIT, "bits of a word");

// A launch that may begin before the call's previous kernel has ended (the
// kernel calls wait_previous).
template <typename... A, typename... B>
cudaError_t launch_after(void (*kernel)(A...), long long blocks, int threads, int smem, cudaStream_t st, const B&... args) {
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.gridDim = dim3((unsigned)blocks);
    c.blockDim = dim3((unsigned)threads);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = st;
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, args...);
}

template <int MODE, bool SLICED = true>
cudaError_t launch(const Params& p, const HeadCall* a, bool first, cudaStream_t st) {
    constexpr int smem = smem_bytes(MODE);
    const cudaError_t e = allow_smem(head_kernel<MODE, SLICED>, smem, SLICED ? MODE : WHOLE_BIT, a->ready);
    if (e != cudaSuccess) return e;
    const int pairs = a->num_sms / 2 < p.jobs ? a->num_sms / 2 : p.jobs;
    if (!first) return launch_after(head_kernel<MODE, SLICED>, 2 * pairs, THREADS, smem, st, p);
    head_kernel<MODE, SLICED><<<2 * pairs, THREADS, smem, st>>>(p);
    return cudaGetLastError();
}

// The smallest column count that holds the rows, or 0: the pair kernel's.
int skinny_cols(int rows, int most) {
    if (rows > most) return 0;
    for (int c = 16; c < 128; c *= 2)
        if (rows <= c) return c;
    return 128;
}

template <int MODE, int COLS>
cudaError_t launch_skinny(SkinnyParams& p, const void* weight, long long weight_stride, const void* hidden, int esz, long long cols,
                          long long stride, int num_sms, uint32_t* ready, bool first, cudaStream_t st) {
    using S = Skinny<MODE, COLS>;
    // as few tiles a CTA as 128 rows allow, of as few rows as that number allows
    const long long most = ceil_div(p.V, 128ll * num_sms) * num_sms;
    p.tile = (int)ceil_div(p.V, most);
    p.jobs = (int)ceil_div(p.V, p.tile);
    cudaError_t e = make_map(&p.a, weight, esz, p.V, cols, weight_stride, p.tile);
    if (e == cudaSuccess) e = make_map(&p.b, hidden, esz, p.M, cols, stride, COLS);
    if (e == cudaSuccess) e = allow_smem(skinny_kernel<MODE, COLS>, S::SMEM, skinny_bit(MODE, COLS), ready);
    if (e != cudaSuccess) return e;
    const int blocks = num_sms < p.jobs ? num_sms : p.jobs;
    if (!first) return launch_after(skinny_kernel<MODE, COLS>, blocks, S::THREADS, S::SMEM, st, p);
    skinny_kernel<MODE, COLS><<<blocks, S::THREADS, S::SMEM, st>>>(p);
    return cudaGetLastError();
}
template <int MODE>
cudaError_t launch_skinny(int cols, SkinnyParams& p, const void* weight, long long weight_stride, const void* hidden, int esz,
                          long long width, long long stride, int num_sms, uint32_t* ready, bool first, cudaStream_t st) {
    if (cols == 16) return launch_skinny<MODE, 16>(p, weight, weight_stride, hidden, esz, width, stride, num_sms, ready, first, st);
    if (cols == 32) return launch_skinny<MODE, 32>(p, weight, weight_stride, hidden, esz, width, stride, num_sms, ready, first, st);
    if constexpr (MODE == FP8) {
        if (cols == 128) return launch_skinny<MODE, 128>(p, weight, weight_stride, hidden, esz, width, stride, num_sms, ready, first, st);
    }
    return launch_skinny<MODE, 64>(p, weight, weight_stride, hidden, esz, width, stride, num_sms, ready, first, st);
}

// K blocks of 64 whose products are summed in tensor memory before fp32
// registers take the sum. Tensor memory cuts each addition's last bits: the
// lse of random logits comes out low by 0.5e-6 for every K block in a slice
// (0.9e-6, 3.8e-6, 8e-6 measured at 2, 8, 16, whatever D), and a logit of 28
// whose products all have one sign by 4e-4 with all of D 4160 in one slice. The
// gradients take the loss's slices, so that their logits are the loss's to the
// bit: what a row's logits are low by, its lse is too, and exp(l - lse) keeps
// the digits that a confident row's target leaves of exp(l - lse) - 1. (Without
// slices a target of loss 1e-5 had dz -4e-4 at D 4160, -9.6e-4 at D 8192.) Shorter
// slices are free where the weight's bytes bound the kernel; the pair's loss
// takes 2% more at 8 than at 16, 13% at 4; the pair's dz against one slice:
// 509 x 1152 x 50021 76 against 59 us (a step 260 against 245), 4096 x 2048 x
// 151936 1% of a step.
constexpr int LOGIT_SLICE = 8, LOGIT_SKINNY_SLICE = 2;
// The gradients' sums, over the rows (d_weight) and over a split of the
// vocabulary (d_hidden), stay in tensor memory for at most 32768 products. A sum
// of one sign comes out low by 1e-7 of itself per 16 products (1.2e-2 after 2^21
// rows in one slice): 2e-4 here, where the rounding to bf16 is up to 4e-3. Calls
// of no longer sums run the kernel without slices, which at the same sizes takes
// 2% (4096 x 2048 x 151936) to 10% (4 x 2048 x 151936) less.
constexpr int GRAD_SLICE = 512;
// Measured on both sides (V 151936; few-row kernel against the pair's, us):
// loss, D 2048: 1 row 102 / 149, 32 rows 110 / 123, 64 rows 118 / 124, 128
// rows 156 / 126. 8-bit product, K 4096: 1 row 106 / 197, 64 rows 143 / 189,
// 128 rows 180 / 202; 256 rows in two groups 348 / 212.
constexpr int HEAD_SKINNY_ROWS = 64;
constexpr int FP8_SKINNY_ROWS = 128;

// Rows whose partial sums the workspace holds at once; more take several rounds.
constexpr int LSE_ROWS = 16384;

// Partial sums a row's logits come in.
long long lse_parts(bool few, int V, int num_sms) { return few ? 4ll * num_sms : 2 * ceil_div(V, TILE); }

// How the gradients are cut: the vocabulary into equal pieces whose dz takes
// at most DZ_BYTES, and each piece's d_hidden sums into splits along the
// vocabulary. Few rows make few d_hidden tiles with a long sum; the splits are
// the number for which the busiest pair has least to do. Job i runs on pair i
// mod pairs, d_hidden's first: r pairs have one d_hidden job more, and the
// d_weight jobs left over go to the pairs from r on. Every split's slab is read
// and written per piece, so there are at most four jobs a pair of them.
constexpr long long DZ_BYTES = 256ll << 20;  // but at least TILE columns: more above 524288 rows
constexpr int MAX_SPLITS = 32;
struct GradPlan {
    int piece, pieces, splits;
    long long dz_bytes, slab_bytes, rows_bytes;
};
// Few rows (the few-row kernel's) have their dz in two parts, the bf16 value
// and what its rounding left: a row's largest term, its target's, would
// otherwise put its one rounding error on the whole row of d_hidden and of
// d_weight. Their products are bound by the weight's bytes and do not feel
// the second part; with more rows the errors average out.
int grad_parts(int N) { return skinny_cols(N, HEAD_SKINNY_ROWS) ? 2 : 1; }
GradPlan grad_plan(int rows, int V, int D, int num_sms) {
    const int N = rows * grad_parts(rows);
    GradPlan g;
    const long long most = (DZ_BYTES / 2 / (N > 0 ? N : 1)) / TILE * TILE;
    const long long cap = most < TILE ? TILE : most;
    g.pieces = (int)ceil_div(V, cap);
    g.piece = (int)(ceil_div(ceil_div(V, g.pieces), TILE) * TILE);
    g.pieces = (int)ceil_div(V, g.piece);
    const long long dt = ceil_div(D, TILE), tiles = ceil_div(N, TILE) * dt, kb = ceil_div(g.piece, 64), pairs = num_sms / 2;
    // in K blocks; a d_weight tile's epilogue that nothing hides costs about two, a slab's traffic about six
    const long long dw = ceil_div(g.piece, TILE) * dt, dw_cost = ceil_div(N, 64) + 2, dw_each = dw / pairs, dw_left = dw % pairs;
    long long best = INT64_MAX;
    g.splits = 1;
    for (long long s = 1; s == 1 || (s <= MAX_SPLITS && s * 8 <= kb && s * tiles <= 4 * pairs); ++s) {
        const long long cost = ceil_div(kb, s) + 6, each = tiles * s / pairs, r = tiles * s % pairs;
        long long worst = each * cost + (dw_each + (dw_left > 0)) * dw_cost;
        const long long more = r ? (each + 1) * cost + (dw_each + (dw_left > pairs - r)) * dw_cost : 0;
        if (more > worst) worst = more;
        if (worst < best) {
            best = worst;
            g.splits = (int)s;
        }
    }
    g.dz_bytes = al(2ll * N * g.piece);
    g.slab_bytes = al(4ll * g.splits * N * D);
    g.rows_bytes = al(2ll * N * D);
    return g;
}

}  // namespace
}  // namespace qs

using namespace qs;

extern "C" long long qs_head_loss_ws(int N, int V, int, int num_sms) {
    const long long rows = N < LSE_ROWS ? N : LSE_ROWS;
    return al(8 * rows * lse_parts(skinny_cols(N, HEAD_SKINNY_ROWS) != 0, V, num_sms)) + al(4 * rows);
}

extern "C" long long qs_head_grad_ws(int N, int V, int D, int num_sms) {
    const GradPlan g = grad_plan(N, V, D, num_sms);
    return g.dz_bytes + g.slab_bytes + g.rows_bytes + al(sizeof(float));
}

// The loss of at most LSE_ROWS rows. All rounds of a call take the same kernel
// (cols: the few-row one's): a row's bits, which the gradients make again, do
// not depend on its round, and the workspace has one layout.
static cudaError_t loss_round(const HeadCall* a, int cols, bool first, int* launches, cudaStream_t st) {
    float2* part = (float2*)a->ws;
    float* target_logit = (float*)(a->ws + al(8ll * a->N * lse_parts(cols != 0, a->V, a->num_sms)));
    int parts;
    cudaError_t e;
    if (cols) {
        SkinnyParams p = {};
        p.V = a->V;
        p.M = a->N;
        p.k_blocks = (int)ceil_div(a->D, 64);
        p.slice = LOGIT_SKINNY_SLICE;
        p.status = a->status;
        p.wait_ns = a->wait_ns;
        p.targets = a->targets;
        p.softcap = a->softcap;
        p.part = part;
        p.target_logit = target_logit;
        e = launch_skinny<LSE>(cols, p, a->weight, a->weight_stride, a->hidden, 2, a->D, a->hidden_stride, a->num_sms, a->ready, first, st);
        parts = 4 * (a->num_sms < p.jobs ? a->num_sms : p.jobs);
    } else {
        Params p = {};
        e = make_map(&p.a, a->hidden, 2, a->N, a->D, a->hidden_stride, 128);
        if (e == cudaSuccess) e = make_map(&p.b, a->weight, 2, a->V, a->D, a->weight_stride, 128);
        if (e != cudaSuccess) return e;
        p.m_tiles = (int)ceil_div(a->N, TILE);
        p.n_tiles = (int)ceil_div(a->V, TILE);
        p.k_blocks = (int)ceil_div(a->D, 64);
        p.slice = LOGIT_SLICE;
        p.jobs = p.m_tiles * p.n_tiles;
        p.M = a->N;
        p.N = a->V;
        p.status = a->status;
        p.wait_ns = a->wait_ns;
        p.targets = a->targets;
        p.softcap = a->softcap;
        p.part = part;
        p.target_logit = target_logit;
        parts = (int)ceil_div(a->V, 128);
        e = launch<LSE>(p, a, first, st);
    }
    if (e != cudaSuccess) return e;
    *launches += 2;
    return launch_after(lse_join_kernel, ceil_div(a->N, 8), 1024, 0, st, (const float2*)part, (const float*)target_logit,
                        a->targets, a->N, a->V, parts, a->loss, a->lse_out);
}

extern "C" cudaError_t qs_head_loss(const HeadCall* a, int* launches, cudaStream_t st) {
    *launches = 0;
    for (long long r = 0; r < a->N; r += LSE_ROWS) {
        HeadCall part = *a;
        part.hidden += r * a->hidden_stride;
        part.targets += r;
        part.loss += r;
        part.lse_out += r;
        part.N = (int)(a->N - r < LSE_ROWS ? a->N - r : LSE_ROWS);
        const cudaError_t e = loss_round(&part, skinny_cols(a->N, HEAD_SKINNY_ROWS), r == 0, launches, st);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

extern "C" cudaError_t qs_head_grad(const HeadCall* a, int* launches, cudaStream_t st) {
    *launches = 0;
    if (a->N == 0)
        return cudaMemset2DAsync(a->d_weight, (size_t)a->d_weight_stride * 2, 0, (size_t)a->D * 2, (size_t)a->V, st);
    const GradPlan g = grad_plan(a->N, a->V, a->D, a->num_sms);
    uint16_t* dz = (uint16_t*)a->ws;
    float* slabs = (float*)(a->ws + g.dz_bytes);
    uint16_t* rows = (uint16_t*)(a->ws + g.dz_bytes + g.slab_bytes);
    float* unit = (float*)(a->ws + g.dz_bytes + g.slab_bytes + g.rows_bytes);
    const int parts = grad_parts(a->N), R = a->N * parts;
    const long long n = (long long)a->N * a->D / 8;
    live_rows_kernel<<<(unsigned)ceil_div(n, 256), 256, 0, st>>>(a->hidden, a->hidden_stride, a->targets, a->grad_loss, a->N,
                                                                 a->D, a->V, parts, rows, unit);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int cols = skinny_cols(a->N, HEAD_SKINNY_ROWS);
    for (int q = 0; q < g.pieces; ++q) {
        const int p0 = q * g.piece, pw = a->V - p0 < g.piece ? a->V - p0 : g.piece;
        const uint16_t* weight = a->weight + (long long)p0 * a->weight_stride;
        Params p = {};
        p.m_tiles = (int)ceil_div(a->N, TILE);
        p.n_tiles = (int)ceil_div(pw, TILE);
        p.M = a->N;
        p.N = pw;
        p.n0 = p0;
        p.status = a->status;
        p.wait_ns = a->wait_ns;
        p.unit = unit;
        if (cols) {
            SkinnyParams f = {};
            f.V = pw;
            f.V_total = a->V;
            f.n0 = p0;
            f.M = a->N;
            f.k_blocks = (int)ceil_div(a->D, 64);
            f.slice = LOGIT_SKINNY_SLICE;
            f.status = a->status;
            f.wait_ns = a->wait_ns;
            f.targets = a->targets;
            f.softcap = a->softcap;
            f.lse = a->lse;
            f.grad = a->grad_loss;
            f.dz = dz;
            f.dz_pitch = g.piece;
            e = launch_skinny<DZ>(cols, f, weight, a->weight_stride, a->hidden, 2, a->D, a->hidden_stride, a->num_sms, a->ready, false, st);
        } else {
            e = make_map(&p.a, a->hidden, 2, a->N, a->D, a->hidden_stride, 128);
            if (e == cudaSuccess) e = make_map(&p.b, weight, 2, pw, a->D, a->weight_stride, 128);
            if (e == cudaSuccess) e = make_map(&p.o, dz, 2, a->N, g.piece, g.piece, 32);
            if (e != cudaSuccess) return e;
            p.k_blocks = (int)ceil_div(a->D, 64);
            p.slice = LOGIT_SLICE;
            p.jobs = p.m_tiles * p.n_tiles;
            p.rows = a->V;
            p.targets = a->targets;
            p.softcap = a->softcap;
            p.lse = a->lse;
            p.grad = a->grad_loss;
            e = launch<DZ>(p, a, false, st);
        }
        if (e != cudaSuccess) return e;
        p.m_tiles = (int)ceil_div(R, TILE);
        e = make_map(&p.a, dz, 2, R, pw, g.piece, 128);
        if (e == cudaSuccess) e = make_map(&p.b, a->weight, 2, a->V, a->D, a->weight_stride, 64);
        if (e == cudaSuccess) e = make_map(&p.a2, dz, 2, R, pw, g.piece, 64);
        if (e == cudaSuccess) e = make_map(&p.b2, rows, 2, R, a->D, a->D, 64);
        if (e == cudaSuccess)
            e = make_map(&p.o, a->d_weight + (long long)p0 * a->d_weight_stride, 2, pw, a->D, a->d_weight_stride, 32);
        if (e != cudaSuccess) return e;
        p.slice = GRAD_SLICE;
        p.d_tiles = (int)ceil_div(a->D, TILE);
        p.dh_k_blocks = (int)ceil_div(pw, 64);
        // every split has a K block; a short last piece adds to the first slabs
        p.splits = g.splits < p.dh_k_blocks ? g.splits : p.dh_k_blocks;
        p.dw_k_blocks = (int)ceil_div(R, 64);
        p.dh_jobs = p.m_tiles * p.d_tiles * p.splits;
        p.jobs = p.dh_jobs + p.n_tiles * p.d_tiles;
        p.rows = R;
        p.D = a->D;
        p.slabs = slabs;
        p.add = q > 0;
        const bool whole = p.dw_k_blocks <= GRAD_SLICE && ceil_div(p.dh_k_blocks, p.splits) <= GRAD_SLICE;
        e = whole ? launch<GRAD, false>(p, a, false, st) : launch<GRAD>(p, a, false, st);
        if (e != cudaSuccess) return e;
        *launches += 2;
    }
    *launches += 2;
    return launch_after(dh_join_kernel, ceil_div(n, 256), 256, 0, st, (const float*)slabs, g.splits * parts, a->N, a->D,
                        (const float*)unit, a->d_hidden, a->d_hidden_stride);
}

extern "C" cudaError_t qs_matmul_fp8(const Fp8Call* a, cudaStream_t st) {
    const int cols = skinny_cols(a->M, FP8_SKINNY_ROWS);
    const long long blocks = ceil_div(a->K, FP8_BLOCK);
    if (cols && blocks * cols * 4 <= Skinny<FP8, 16>::TABLE) {
        SkinnyParams p = {};
        p.V = a->V;
        p.M = a->M;
        p.k_blocks = (int)blocks;
        p.slice = 1;
        p.status = a->status;
        p.wait_ns = a->wait_ns;
        p.sx = a->sx;
        p.sw = a->sw;
        p.sx_stride = a->sx_stride;
        p.sw_stride = a->sw_stride;
        p.out = a->out;
        p.out_stride = a->out_stride;
        p.out_bf16 = a->out_bf16;
        return launch_skinny<FP8>(cols, p, a->w, a->w_stride, a->x, 1, a->K, a->x_stride, a->num_sms, a->ready, true, st);
    }
    WideParams p = {};
    cudaError_t e = make_map(&p.a, a->x, 1, a->M, a->K, a->x_stride, 128);
    if (e == cudaSuccess) e = make_map(&p.b, a->w, 1, a->V, a->K, a->w_stride, 128);
    if (e == cudaSuccess) e = allow_smem(wide_kernel, WIDE_SMEM, WIDE_BIT, a->ready);
    if (e != cudaSuccess) return e;
    p.m_tiles = (int)ceil_div(a->M, TILE);
    p.n_tiles = (int)ceil_div(a->V, TILE);
    p.k_blocks = (int)blocks;
    p.jobs = p.m_tiles * p.n_tiles;
    p.M = a->M;
    p.V = a->V;
    p.status = a->status;
    p.wait_ns = a->wait_ns;
    p.sx = a->sx;
    p.sw = a->sw;
    p.sx_stride = a->sx_stride;
    p.sw_stride = a->sw_stride;
    p.out = a->out;
    p.out_stride = a->out_stride;
    p.out_bf16 = a->out_bf16;
    const int esz = a->out_bf16 ? 2 : 4;
    p.wide = (uintptr_t)a->out % 32 == 0 && a->out_stride * esz % 32 == 0;
    const int pairs = a->num_sms / 2 < p.jobs ? a->num_sms / 2 : p.jobs;
    wide_kernel<<<2 * pairs, WIDE_THREADS, WIDE_SMEM, st>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t quantize(const QuantArgs& a, int block_rows, cudaStream_t st) {
    const auto grid = [](long long x, long long y) { return dim3((unsigned)x, (unsigned)(y < 65535 ? y : 65535)); };
    if (block_rows == 1)
        quantize_rows_kernel<T><<<grid(ceil_div(a.K, QCOLS), ceil_div(a.M, QROWS * 8)), 256, 0, st>>>(a);
    else
        quantize_square_kernel<T><<<grid(ceil_div(a.K, FP8_BLOCK), ceil_div(a.M, FP8_BLOCK)), 256, 0, st>>>(a);
    return cudaGetLastError();
}

extern "C" cudaError_t qs_quantize_fp8(const void* x, int dtype, int M, int K, long long x_stride, int block_rows,
                                       uint8_t* q, long long q_stride, float* scale, long long scale_stride,
                                       cudaStream_t st) {
    const int esz = dtype == QSAMP_BF16 ? 2 : 4;
    QuantArgs a = {x, q, scale, x_stride, q_stride, scale_stride, M, K, 0, 0};
    a.x_vec = (uintptr_t)x % 16 == 0 && x_stride * esz % 16 == 0;
    a.q_vec = (uintptr_t)q % 8 == 0 && q_stride % 8 == 0;
    return esz == 2 ? quantize<uint16_t>(a, block_rows, st) : quantize<float>(a, block_rows, st);
}
