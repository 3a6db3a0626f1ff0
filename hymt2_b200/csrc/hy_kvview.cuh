// hy_kvview.cuh — what the operators on a paged KV cache share: the checked
// view of a cache, the bounds of a slot's rows and drafted nodes, and the
// sm_100a primitives (mbarriers with bounded waits, TMA boxes, tcgen05) that
// their tensor-core kernels are written in.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/hymt2_cuda.h"
#include "hy_common.cuh"
#include "hy_pages.h"

namespace {
using namespace hyk;

constexpr int kTreeMax = 64;  // nodes of one tree

struct KvView {
    uint16_t *kv;
    const int *pages;
    int layers, npages, kvh, hd, slots, page_max, kvd;
    int tokens;  // of the token arrays
    long long page_stride, layer_stride;  // elements

    // Page of row r of a slot, -1 when there is none.
    __device__ __forceinline__ int page(int slot, int r) const {
        if (r < 0 || (r >> kPageShift) >= page_max) return -1;
        const int p = __ldg(pages + (size_t)slot * page_max + (r >> kPageShift));
        return p < 0 || p >= npages ? -1 : p;
    }
    // Element offset of K row r in page p of a layer (V: + kPageRows * kvd).
    __device__ __forceinline__ long long row(int layer, int p, int r) const {
        return layer * layer_stride + (long long)p * page_stride + (long long)(r & (kPageRows - 1)) * kvd;
    }
};

// Slot s's cached rows and nodes, bounded by its page table, max_nodes and the
// token arrays: nodes of tokens that are not there do not exist.
__device__ __forceinline__ void tree_span(const KvView &v, const int *len, const int *off, int max_nodes, int s, int &L,
                                          int &t0, int &n) {
    const int cap = v.page_max * kPageRows;
    L = min(max(__ldg(len + s), 0), cap);
    t0 = __ldg(off + s);
    const int t1 = min(__ldg(off + s + 1), v.tokens);
    n = t0 >= 0 && t1 > t0 ? min(t1 - t0, max_nodes) : 0;
}

// Waits that gave up (2 s): counted here, read by hyc_kvops_timeouts.
__device__ unsigned g_kv_timeouts;

// ---------------------------------------------------------------- mbarriers and TMA

constexpr unsigned long long kKvWaitNs = 2000000000ull;

__device__ __forceinline__ uint32_t kv_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mb_init(uint64_t *b, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(kv_smem(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mb_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(kv_smem(b)) : "memory");
}
__device__ __forceinline__ void mb_expect(uint64_t *b, unsigned tx) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(kv_smem(b)), "r"(tx) : "memory");
}
__device__ __forceinline__ bool mb_try(uint64_t *b, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(kv_smem(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Waits for a phase for at most 2 s.  A wait that gives up sets the CTA's
// *stop word, after which every wait returns at once: all threads still go
// through the same steps, with whatever data is there, and the kernel ends.
__device__ __forceinline__ void mb_wait(uint64_t *b, unsigned parity, int *stop, unsigned long long limit = kKvWaitNs) {
    if (mb_try(b, parity)) return;
    const unsigned long long t0 = gtimer();
    while (!mb_try(b, parity)) {
        if (*(volatile int *)stop) return;
        if (gtimer() - t0 > limit) {
            *(volatile int *)stop = 1;
            atomicAdd(&g_kv_timeouts, 1u);
            return;
        }
    }
}
// A place in a ring of stages: its stage, and the parity of that stage's use.
// (Counting up: a division by the ring's length a stage cost 0.5 us a tile.)
struct RingPos {
    int st = 0;
    unsigned use = 0;
    __device__ __forceinline__ void next(int stages, int by = 1) {
        st += by;
        if (st >= stages) {
            st -= stages;
            use ^= 1;
        }
    }
};
__device__ __forceinline__ void tma_box(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            kv_smem(dst)),
        "l"(map), "r"(x), "r"(y), "r"(kv_smem(bar))
        : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Barrier of `threads` threads that tells each whether any of them said v.
__device__ __forceinline__ bool bar_or(int id, int threads, bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 q, %3, 0;\n barrier.cta.red.or.pred p, %1, %2, q;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(r)
        : "r"(id), "r"(threads), "r"((uint32_t)v)
        : "memory");
    return r != 0;
}

// ---------------------------------------------------------------- tcgen05

__device__ __forceinline__ void um_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void um_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void um_commit(uint64_t *b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(kv_smem(b)) : "memory");
}
// Instruction descriptor: bf16 x bf16 -> fp32, A K-major, B K-major or (V) MN-major.
__host__ __device__ constexpr uint32_t um_idesc(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// One thread of a converged warp.  The loops that feed the tensor cores and
// the TMA unit run in whole warps with uniform values, and only the
// instructions themselves are this thread's: descriptors then stay in uniform
// registers (a loop of one lane took 70-110 ns a product, more than the
// product itself).
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
    return p != 0;
}
// Shared-memory operand in 128-byte-swizzled rows of 64 bf16, 8-row groups
// 1024 bytes apart: the low word (address, and `lbo`, for MN-major operands
// the bytes between 64-element columns); a step of n bytes adds n / 16 to it.
__device__ __forceinline__ uint32_t um_desc_lo(uint32_t addr, uint32_t lbo) { return ((addr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16); }
constexpr uint32_t kUmDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void um_mma(uint32_t d, uint32_t alo, uint32_t blo, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d),
        "r"(alo), "r"(blo), "r"(idesc), "r"((int)acc), "r"(kUmDescHi)
        : "memory");
}
// A from TMEM (bf16 pairs, one row a lane).
__device__ __forceinline__ void um_mma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d),
        "r"(a), "r"(blo), "r"(idesc), "r"((int)acc), "r"(kUmDescHi)
        : "memory");
}
// 32 lanes x 32 or 16 columns of 32-bit words from, or 16 to, this warp's lane quarter.
__device__ __forceinline__ void um_ld32(uint32_t t, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
          "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
          "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void um_ld16(uint32_t t, float *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void um_st16(uint32_t t, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(t)
        : "memory");
}
// Wait for this thread's tcgen05.ld results; every destination register also
// passes through an empty statement after the wait, so that no use of it can
// move above.
template <int N>
__device__ __forceinline__ void um_wait_ld(float *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void um_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
// bf16 pair, lo in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// x0, x1 -> NT bf16 terms each (packed pairs), every remainder exact in fp32:
// three terms hold all 24 bits of an fp32 number.
template <int NT>
__device__ __forceinline__ void split_bf16(float x0, float x1, uint32_t (&t)[NT]) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
        t[i] = pack_bf16(x0, x1);
        if (i + 1 < NT) {
            x0 -= __uint_as_float(t[i] << 16);
            x1 -= __uint_as_float(t[i] & 0xffff0000u);
        }
    }
}

}  // namespace
