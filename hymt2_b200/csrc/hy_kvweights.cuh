// hy_kvweights.cuh — attention weights accumulated per cached row.
//
// acc[r] += sum over queries j and the group's heads of 2^(x_r log2 e - lse_j
// log2 e), x_r = scale * q_j . k_r, for rows r <= len + j.  The log-sum-exp is
// known, so rows are independent: one pass over K (2 hd bytes a row and KV
// head) with no maximum and no join, and a row's sum stays with one thread.
#pragma once
#include "hy_kvview.cuh"

namespace {

struct WeightArgs {
    KvView v;
    int heads, G, max_q;
    const int *len, *nq, *sel;
    const void *q;
    long long q_ld, q_layer;
    const float *lse;
    long long lse_layer;
    float scale;
    float *acc;
    int acc_rows;
    int block, qbufs, stages;  // query rows of a block (a multiple of 16, <= 128), Q buffers, K stages
};

// Tiles of 128 cached rows in (layer, slot, KV head) order, cut into equal runs.
struct WeightWalk {
    int layer, slot, rem, left, at, L, n, end, T;
    int s_layer, s_slot, s_kvh, s_a, s_b;

    __device__ __forceinline__ static void span(const WeightArgs &a, int s, int &L, int &n, int &end) {
        const int cap = min(a.v.page_max * kPageRows, a.acc_rows);
        L = min(max(__ldg(a.len + s), 0), cap);
        n = min(max(__ldg(a.nq + s), 0), a.max_q);
        end = n > 0 ? min(L + n, cap) : 0;
    }
    __device__ __forceinline__ bool next(const WeightArgs &a) {
        while (left > 0) {
            if (slot >= a.v.slots) {
                slot = 0;
                rem = 0;
                if (++layer >= a.v.layers) return false;
            }
            if (at != slot) {
                span(a, slot, L, n, end);
                T = (end + 127) >> 7;
                at = slot;
            }
            if (rem >= T * a.v.kvh) {
                slot++;
                rem = 0;
                continue;
            }
            s_layer = layer;
            s_slot = slot;
            s_kvh = rem / T;
            s_a = rem % T;
            s_b = min(T, s_a + left);
            left -= s_b - s_a;
            rem += s_b - s_a;
            return true;
        }
        return false;
    }
};

// S^T = K . Q^T on the tensor cores: the cached rows are the 128 lanes of a
// tile, the (query, head) pairs its columns, so a thread sums its row's
// probabilities by itself.  K comes by TMA straight into the K-major operand
// (128-byte swizzled); fp32 queries enter as three bf16 terms.
//   warps 0-3  one cached row a thread: exponentials and sums, acc
//   warp 4     K pages by TMA;  warp 5  MMAs into four S^T tiles
//   warps 6-9  the next column's queries, log-sum-exps and row bounds
// More than 128 (query, head) rows go in blocks of 128 over the same rows,
// whose thread adds one block after the other.
constexpr int kWtThreads = 320;
constexpr int kWtSmem = 222 * 1024;  // of 227 KB: Q buffers and K stages
template <typename T>
__host__ __device__ constexpr int wt_terms() { return sizeof(T) == 4 ? 3 : 1; }

template <typename T, int HD>
__global__ void __launch_bounds__(kWtThreads, 1) cache_weights_tc(const __grid_constant__ WeightArgs a,
                                                                  const __grid_constant__ CUtensorMap map) {
    constexpr int QT = wt_terms<T>(), NH = HD / 64, STB = NH * 16384, kMaxSt = 8, NS = 4;
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[kMaxSt], empty[kMaxSt], sfull[NS], sempty[NS], qfull[2], qempty[2], fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_scan[kWtThreads / 32], s_start[4], s_stop;
    __shared__ __align__(16) float2 s_col[2][128];  // of each query row: lse * log2 e, last row it sees
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, NB = a.block, NST = a.stages;
    const int half_b = NB * 128, term_b = NH * half_b, qbuf_b = QT * term_b;
    uint8_t *sq = (uint8_t *)(((uintptr_t)dsm + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sq + a.qbufs * qbuf_b;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; i++) {
            mb_init(&full[i], 1);
            mb_init(&empty[i], 1);
        }
        for (int i = 0; i < NS; i++) {
            mb_init(&sfull[i], 1);
            mb_init(&sempty[i], 128);
        }
        for (int i = 0; i < 2; i++) {
            mb_init(&qfull[i], 128);
            mb_init(&qempty[i], 129);
        }
        mb_init(&fin, 1);
        s_stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(kv_smem(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        um_fence_before();
    }
    // this CTA's run of tiles
    {
        const int th = threadIdx.x, per = (a.v.slots + kWtThreads - 1) / kWtThreads;
        const int b0 = min(a.v.slots, th * per), b1 = min(a.v.slots, b0 + per);
        int sum = 0;
        for (int s = b0; s < b1; s++) {
            int L, n, end;
            WeightWalk::span(a, s, L, n, end);
            sum += ((end + 127) >> 7) * a.v.kvh;
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        int before = incl - sum, layer_tiles = 0;
        for (int i = 0; i < kWtThreads / 32; i++) {
            if (i < warp) before += s_scan[i];
            layer_tiles += s_scan[i];
        }
        const long long total = (long long)layer_tiles * a.v.layers;
        const int C = (int)((total + gridDim.x - 1) / gridDim.x);
        const long long g0 = (long long)blockIdx.x * C;
        if (th == 0) s_start[3] = (int)max(0LL, min((long long)C, total - g0));
        if (g0 < total) {
            const int in = (int)(g0 % layer_tiles);
            if (in >= before && in < before + sum)
                for (int s = b0; s < b1; s++) {
                    int L, n, end;
                    WeightWalk::span(a, s, L, n, end);
                    const int c = ((end + 127) >> 7) * a.v.kvh;
                    if (in < before + c) {
                        s_start[0] = (int)(g0 / layer_tiles);
                        s_start[1] = s;
                        s_start[2] = in - before;
                        break;
                    }
                    before += c;
                }
        }
        __syncthreads();
    }
    um_fence_after();
    const uint32_t tmem = s_tmem;
    WeightWalk w;
    w.left = s_start[3];
    w.layer = w.left > 0 ? s_start[0] : 0;
    w.slot = w.left > 0 ? s_start[1] : 0;
    w.rem = w.left > 0 ? s_start[2] : 0;
    w.at = -1;
    if (warp == 4) {
        const int yend = a.v.layers * a.v.npages * 2 * kPageRows;
        int pos = 0;
        while (w.next(a)) {
            const int pages = (w.end + kPageRows - 1) / kPageRows;
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB)
                for (int t = w.s_a; t < w.s_b; t++, pos++) {
                    const int j = t * 8 + (lane & 7), st = pos % NST, use = pos / NST;
                    const int pg = j < pages ? __ldg(a.v.pages + (size_t)w.s_slot * a.v.page_max + j) : -1;
                    const int y = pg < 0 || pg >= a.v.npages ? yend : (w.s_layer * a.v.npages + pg) * 2 * kPageRows;
                    if (use > 0) mb_wait(&empty[st], (use - 1) & 1, &s_stop);
                    if (__any_sync(0xffffffffu, *(volatile int *)&s_stop)) {
                        pos--;
                        continue;
                    }
                    if (lane == 0) mb_expect(&full[st], STB);
                    __syncwarp();
                    if (lane < 8) {
#pragma unroll
                        for (int h = 0; h < NH; h++)
                            tma_box(ring + (size_t)st * STB + h * 16384 + lane * 2048, &map, w.s_kvh * HD + h * 64, y, &full[st]);
                    }
                }
        }
        for (int p = max(0, pos - NST); p < pos; p++) {  // copies in flight land before the kernel ends
            int none = 0;
            mb_wait(&full[p % NST], (p / NST) & 1, &none);
        }
    } else if (warp == 5) {
        if (lane == 0) {
            int it = 0, qi = 0;
            while (w.next(a))
                for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                    const int qb = qi % a.qbufs, N = (min(NB, w.n * a.G - q0) + 15) & ~15;
                    const uint32_t id = um_idesc(128, N, false), qa = kv_smem(sq + qb * qbuf_b);
                    mb_wait(&qfull[qb], (qi / a.qbufs) & 1, &s_stop);
                    for (int t = w.s_a; t < w.s_b; t++, it++) {
                        const int st = it % NST, b = it % NS;
                        mb_wait(&full[st], (it / NST) & 1, &s_stop);
                        if (it >= NS) mb_wait(&sempty[b], (it / NS - 1) & 1, &s_stop);
                        um_fence_after();
                        const uint32_t kb = kv_smem(ring + (size_t)st * STB);
#pragma unroll
                        for (int x = QT - 1; x >= 0; x--)  // small terms first
#pragma unroll
                            for (int k = 0; k < HD / 16; k++)
                                um_mma(tmem + b * 128, um_desc(kb + (k >> 2) * 16384 + (k & 3) * 32, 16),
                                       um_desc(qa + x * term_b + (k >> 2) * half_b + (k & 3) * 32, 16), id, !(x == QT - 1 && k == 0));
                        um_commit(&empty[st]);
                        um_commit(&sfull[b]);
                    }
                    um_commit(&qempty[qb]);
                }
            um_commit(&fin);
            int none = 0;
            mb_wait(&fin, 0, &none);
        }
    } else if (warp >= 6) {
        const int wl = warp - 6;
        int qi = 0;
        while (w.next(a))
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                const int qb = qi % a.qbufs, use = qi / a.qbufs, rows = min(NB, w.n * a.G - q0), N = (rows + 15) & ~15;
                if (use > 0) mb_wait(&qempty[qb], (use - 1) & 1, &s_stop);
                uint8_t *dst0 = sq + qb * qbuf_b;
                const int half = HD == 128 ? lane >> 4 : 0, c = (lane & 15) * 4;
#pragma unroll 4
                for (int r = wl; r < N; r += 4) {
                    const int j = (q0 + r) / a.G, head = w.s_kvh * a.G + (q0 + r) % a.G;
                    const int t = r < rows ? __ldg(a.sel + (size_t)w.s_slot * a.max_q + j) : -1;
                    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (t >= 0 && (HD == 128 || lane < 16)) {
                        const T *src = (const T *)a.q + w.s_layer * a.q_layer + t * a.q_ld + (long long)head * HD + half * 64 + c;
                        if constexpr (sizeof(T) == 4) {
                            q = *(const float4 *)src;
                        } else {
                            const uint2 u = *(const uint2 *)src;
                            q = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                                            __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
                        }
                    }
                    if (HD == 128 || lane < 16) {
                        uint32_t lo[QT], hi[QT];
                        split_bf16<QT>(q.x, q.y, lo);
                        split_bf16<QT>(q.z, q.w, hi);
                        uint8_t *dst = dst0 + half * half_b + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | ((c & 4) << 1));
#pragma unroll
                        for (int i = 0; i < QT; i++) *(uint2 *)(dst + i * term_b) = make_uint2(lo[i], hi[i]);
                    }
                    if (lane == 0) {
                        // a query that is left out, or saw nothing (-inf), sees no row
                        const float e = t >= 0 ? a.lse[w.s_layer * a.lse_layer + (long long)t * a.heads + head] : -INFINITY;
                        s_col[qb][r] = make_float2(e * 1.4426950408889634f, __int_as_float(e == -INFINITY ? -1 : w.L + j));
                    }
                }
                fence_async_smem();
                mb_arrive(&qfull[qb]);
            }
    } else {
        const int th = threadIdx.x;
        const float sl2 = a.scale * 1.4426950408889634f;
        int it = 0, qi = 0;
        while (w.next(a)) {
            float *acc = a.acc + (((size_t)w.s_layer * a.v.slots + w.s_slot) * a.v.kvh + w.s_kvh) * a.acc_rows;
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                const int qb = qi % a.qbufs, N = (min(NB, w.n * a.G - q0) + 15) & ~15;
                mb_wait(&qfull[qb], (qi / a.qbufs) & 1, &s_stop);
                for (int t = w.s_a; t < w.s_b; t++, it++) {
                    const int b = it % NS, r = t * 128 + th;
                    float sum = r < w.end && (r < w.L || q0 > 0) ? acc[r] : 0.f;
                    mb_wait(&sfull[b], (it / NS) & 1, &s_stop);
                    um_fence_after();
                    float part[2] = {0.f, 0.f};
                    for (int c = 0; c < N; c += 16) {
                        float x[16];
                        um_ld16(tmem + ((uint32_t)(warp * 32) << 16) + b * 128 + c, x);
                        um_wait_ld<16>(x);
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const float4 e = *(const float4 *)&s_col[qb][c + i];
                            const float p0 = ex2(fmaf(x[i], sl2, -e.x)), p1 = ex2(fmaf(x[i + 1], sl2, -e.z));
                            part[0] += r <= __float_as_int(e.y) ? p0 : 0.f;
                            part[1] += r <= __float_as_int(e.w) ? p1 : 0.f;
                        }
                    }
                    um_fence_before();
                    mb_arrive(&sempty[b]);
                    if (r < w.end) acc[r] = sum + (part[0] + part[1]);
                }
                mb_arrive(&qempty[qb]);
            }
        }
    }
    __syncthreads();
    if (warp == 5) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace
