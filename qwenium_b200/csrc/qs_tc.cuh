// qs_tc.cuh -- sm_100a building blocks of the output-head kernels: barriers
// with bounded waits, tensor copies (TMA), tensor memory and tcgen05 matrix
// instructions for a pair of CTAs. Internal.
#ifndef QS_TC_CUH
#define QS_TC_CUH

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace qs {
namespace tc {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// True in one lane of the converged warp. The loops of the loading and the
// issuing warp run in all lanes and only the instructions themselves in the
// elected one: the loop's values then stay in uniform registers, which is
// where tensor copies and matrix instructions take their operands.
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile(
        "{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The address of this CTA's shared-memory location in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Arrives on a barrier of this CTA.
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Arrives on a barrier of the cluster (an address from map_to). Relaxed: it
// only says that tensor memory has been read into registers (tcgen05.wait::ld
// and the tcgen05 fences order that); a release to the cluster would wait for
// every store the thread has in flight.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Whether the phase is over, without waiting (bar_try may suspend the warp).
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Launches of one call overlap: the next kernel may start its prologue when
// every block of this one has begun to leave or has said launch_next, and
// waits in wait_previous, before its first access to global memory, until this
// one has ended and its writes are visible.
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// How long a role waits for another: a kernel's own copies and matrix
// instructions finish in microseconds. When a wait runs out, *gave_up (shared
// memory of the CTA) and *status (mapped host memory) are set.
struct Patience {
    volatile int* gave_up;
    int* status;
    unsigned long long ns;
    __device__ __forceinline__ void run_out() const {
        *gave_up = 1;
        *(volatile int*)status = 1;
    }
};

// Waits for the barrier's phase. False when the wait ran out, or another role
// of this CTA gave up: the caller leaves its loop. ISSUER (the warp of the matrix
// instructions, on whose progress the others' waits depend): without any time to
// wait, a phase that is not over when it is asked for has run out.
template <bool ISSUER>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Patience& w) {
    if (ISSUER && w.ns == 0) {
        if (bar_test(bar, parity)) return true;
        w.run_out();
        return false;
    }
    // the clock is slow to read: the short waits of a running pipeline end before it is
    for (int spin = 0; spin < 256; ++spin)
        if (bar_try(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    for (uint32_t spin = 1;; ++spin) {
        if (bar_try(bar, parity)) return true;
        if ((spin & 63) == 0) {
            if (*w.gave_up) return false;
            if (now_ns() - t0 > w.ns) {
                w.run_out();
                return false;
            }
        }
    }
}

// The same for a converged warp: the answer is the warp's.
template <bool ISSUER = false>
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, const Patience& w) {
    return __all_sync(0xffffffffu, bar_wait<ISSUER>(bar, parity, w));
}

// Before a CTA leaves: after a role gave up, whatever the CTA had in flight
// (copies, matrix instructions: microseconds) lands while it is here. The clock
// decides, for a sleep may return at once; the count is its own bound.
__device__ __forceinline__ void let_land(const Patience& w) {
    __syncwarp();
    if (*w.gave_up) {
        const unsigned long long t0 = now_ns();
        for (int i = 0; i < 100000 && now_ns() - t0 < 20000000ull; ++i) __nanosleep(1000);
    }
    __syncwarp();
}

// Position in a ring of N barriers: the slot and the parity of its phase,
// stepped rather than divided out (one warp runs these loops, and every
// dependent instruction of them is latency).
template <uint32_t N>
struct Ring {
    uint32_t slot = 0, parity = 0;
    __device__ __forceinline__ void step() {
        const bool wrap = slot == N - 1;
        slot = wrap ? 0 : slot + 1;
        parity ^= wrap;
    }
};

// ---------------------------------------------------------------- tensor copies
// Loads the box at (x, y) into this CTA's shared memory and counts its bytes
// on `bar`: this CTA's, or with PAIR a barrier of either CTA of the pair (an
// address from map_to).
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
            "%3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

// Stores a box from this CTA's shared memory at (x, y); what lies outside the
// matrix is left out. The thread that issued the stores waits for them:
// until their source may be written again, or until they are done.
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, uint32_t src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
                 "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---------------------------------------------------------------- tensor memory
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}

template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: lane i of the warp gets row i.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    __syncwarp();  // the load is the warp's as a whole
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}

// Until tmem_wait_load returns the loaded registers hold nothing; they pass
// through it so that no use is moved ahead of it.
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}

__device__ __forceinline__ void tmem_wait_load(float (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])::
                       "memory");
}

__device__ __forceinline__ void tmem_wait_load(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                   "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                   "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                   "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                   "+f"(v[30]), "+f"(v[31])::"memory");
}

// ---------------------------------------------------------------- matrix instructions
// Shared-memory operand in 128-byte swizzled rows. K contiguous: rows of 128
// bytes (64 bf16 or 128 e4m3 of K), 8-row groups 1024 bytes apart. The other
// dimension contiguous: 64 of its elements per 128-byte row, one row per k,
// 8-k groups 1024 bytes apart, the next 64 elements `lead` bytes on.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// fp32 accumulators of m rows and n columns; bf16 (kind::f16) or e4m3.
__host__ __device__ constexpr uint32_t instr_bf16(int m, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t instr_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

#define QS_MMA(group, kind)                                                                        \
    asm volatile(                                                                                  \
        "{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"                                               \
        "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"(d),        \
        "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)                                             \
        : "memory")
template <bool PAIR, bool E4M3>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
    if (PAIR && E4M3) QS_MMA("2", "f8f6f4");
    if (PAIR && !E4M3) QS_MMA("2", "f16");
    if (!PAIR && E4M3) QS_MMA("1", "f8f6f4");
    if (!PAIR && !E4M3) QS_MMA("1", "f16");
}
#undef QS_MMA

// The barrier (with PAIR the one at this offset of both CTAs) completes when
// the matrix instructions issued so far have.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if (PAIR)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 32 bytes to a 32-byte aligned address.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

}  // namespace tc
}  // namespace qs

#endif
