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
    int lg;                    // log2 G
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

// One row's sum over a block's queries (from query row q0 on) in plain fp32
// arithmetic, in place of one that is not a number: the products split fp32
// queries into bf16 terms, and an infinite key times terms of both signs, or
// times one that is 0, is NaN where the key times the query is not.
template <typename T, int HD>
__device__ __noinline__ float weights_redo(const WeightArgs &a, int layer, int slot, int kvh, int r, int q0, int N, const float *lse,
                                           const int *last, float sl2) {
    const int pg = a.v.page(slot, r);
    const uint16_t *k = a.v.kv + a.v.row(layer, max(pg, 0), r) + kvh * HD;
    float sum = 0.f;
    for (int c = 0; c < N; c++) {
        if (r > last[c]) continue;  // also: past the block's queries, or left out
        const int t = a.sel[(size_t)slot * a.max_q + ((q0 + c) >> a.lg)];
        const T *q = (const T *)a.q + layer * a.q_layer + t * a.q_ld + (long long)(kvh * a.G + ((q0 + c) & (a.G - 1))) * HD;
        float x = 0.f;
        for (int d = 0; d < HD; d++) x = fmaf((float)q[d], pg < 0 ? 0.f : bf16_bits_to_f32(k[d]), x);
        sum += ex2(fmaf(x, sl2, lse[c]));
    }
    return sum;
}

// On a B200, in calls one after the other: 3 fp32 queries over 32 layers x
// 4096 rows, 4 KV heads (139 MB) 32 us, 4.3 TB/s, bound by K's bytes after 6 us
// until the first queries are there; 31 bf16 queries over 16 slots of about
// 4500 rows, 4 layers (316 MB) 76 us, 4.2 TB/s (64 us in short runs, before the
// power limit), 124 columns a row: the exponentials alone would take 33 us, and
// most stalls are waits for tensor memory, 16 columns at a time.  A row whose
// sum is not a number is summed again by weights_redo.
// S^T = K . Q^T on the tensor cores: the cached rows are the 128 lanes of a
// tile, the (query, head) pairs its columns, so a thread sums its row's
// probabilities by itself.  K comes by TMA straight into the K-major operand
// (128-byte swizzled); fp32 queries enter as three bf16 terms.
//   warps 0-15   four groups, one for each of four S^T tiles: a cached row a
//                thread, exponentials and sums, acc (one group took 146 us
//                against 130 with 31 queries, waiting for itself tile by tile)
//   warp 16      K pages by TMA;  warp 17  MMAs
//   warps 18-21  the next column's queries, log-sum-exps and row bounds
// More than 128 (query, head) rows go in blocks of 128 over the same rows,
// whose thread adds one block after the other: a tile's group goes by the tile's
// place in the column, the same for every block.
constexpr int kWtThreads = 22 * 32;
constexpr int kWtSmem = 222 * 1024;  // of 227 KB: Q buffers and K stages
template <typename T>
__host__ __device__ constexpr int wt_terms() { return sizeof(T) == 4 ? 3 : 1; }

template <typename T, int HD>
__global__ void __launch_bounds__(kWtThreads, 1) cache_weights_tc(const __grid_constant__ WeightArgs a,
                                                                  const __grid_constant__ CUtensorMap map) {
    constexpr int QT = wt_terms<T>(), NH = HD / 64, STB = NH * 16384, kMaxSt = 8, NS = 4;  // NS: S^T tiles and row groups
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[kMaxSt], empty[kMaxSt], sfull[NS], sempty[NS], qfull[2], qempty[2], fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_scan[kWtThreads / 32], s_start[4], s_stop;
    __shared__ int s_tok[128];
    __shared__ unsigned s_counts[2];
    __shared__ __align__(16) float s_lse[2][128];  // of each query row: -lse * log2 e,
    __shared__ __align__(16) int s_last[2][128];   // and the last cached row it sees
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, NB = a.block, NST = a.stages;
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
            mb_init(&qempty[i], 128 * NS + 1);
        }
        mb_init(&fin, 1);
        s_stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
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
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    WeightWalk w;
    w.left = s_start[3];
    w.layer = w.left > 0 ? s_start[0] : 0;
    w.slot = w.left > 0 ? s_start[1] : 0;
    w.rem = w.left > 0 ? s_start[2] : 0;
    w.at = -1;
    if (warp == 16) {
        const int yend = a.v.layers * a.v.npages * 2 * kPageRows;
        int pos = 0;
        RingPos at;
        while (w.next(a)) {
            const int pages = (w.end + kPageRows - 1) / kPageRows;
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB)
                for (int t = w.s_a; t < w.s_b; t++, pos++, at.next(NST)) {
                    const int j = t * 8 + (lane & 7), st = at.st;
                    const int pg = j < pages ? __ldg(a.v.pages + (size_t)w.s_slot * a.v.page_max + j) : -1;
                    const int y = pg < 0 || pg >= a.v.npages ? yend : (w.s_layer * a.v.npages + pg) * 2 * kPageRows;
                    mb_wait(&empty[st], at.use ^ 1, &s_stop);  // passes on a stage's first use
                    if (__any_sync(0xffffffffu, *(volatile int *)&s_stop)) {
                        pos--;
                        continue;
                    }
                    int yj[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) yj[i] = __shfl_sync(0xffffffffu, y, i);
                    if (elect()) {
                        mb_expect(&full[st], STB);
#pragma unroll
                        for (int i = 0; i < 8; i++)
#pragma unroll
                            for (int h = 0; h < NH; h++)
                                tma_box(ring + (size_t)st * STB + h * 16384 + i * 2048, &map, w.s_kvh * HD + h * 64, yj[i], &full[st]);
                    }
                    __syncwarp();
                }
        }
        for (int p = max(0, pos - NST); p < pos; p++) {  // copies in flight land before the kernel ends
            int none = 0;
            mb_wait(&full[p % NST], (p / NST) & 1, &none);
        }
    } else if (warp == 17) {
        {
            const uint32_t ring0 = __shfl_sync(0xffffffffu, kv_smem(ring), 0), sq0 = __shfl_sync(0xffffffffu, kv_smem(sq), 0);
            RingPos at;
            int qi = 0, turn = 0, used = 0;  // used: parity of each S^T tile's uses
            while (w.next(a)) {
                for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                    const int qb = qi % a.qbufs, N = (min(NB, w.n * a.G - q0) + 15) & ~15;
                    const uint32_t id = um_idesc(128, N, false), qa = um_desc_lo(sq0 + qb * qbuf_b, 16);
                    mb_wait(&qfull[qb], (qi / a.qbufs) & 1, &s_stop);
                    for (int t = w.s_a; t < w.s_b; t++, at.next(NST)) {
                        const int st = at.st, b = (t - w.s_a + turn) % NS;
                        mb_wait(&full[st], at.use, &s_stop);
                        mb_wait(&sempty[b], ((used >> b) & 1) ^ 1, &s_stop);  // passes on the first use
                        used ^= 1 << b;
                        um_fence_after();
                        const uint32_t kb = um_desc_lo(ring0 + st * STB, 16), s0 = tmem + b * 128;
                        if (elect()) {
#pragma unroll
                            for (int x = QT - 1; x >= 0; x--)  // small terms first
#pragma unroll
                                for (int k = 0; k < HD / 16; k++)
                                    um_mma(s0, kb + ((k >> 2) * 16384 + (k & 3) * 32) / 16,
                                           qa + (x * term_b + (k >> 2) * half_b + (k & 3) * 32) / 16, id, !(x == QT - 1 && k == 0));
                            um_commit(&empty[st]);
                            um_commit(&sfull[b]);
                        }
                        __syncwarp();
                    }
                    if (elect()) um_commit(&qempty[qb]);
                    __syncwarp();
                }
                turn++;
            }
            if (elect()) um_commit(&fin);
            __syncwarp();
            int none = 0;
            mb_wait(&fin, 0, &none);
        }
    } else if (warp >= 18) {
        const int wl = warp - 18;
        int qi = 0;
        while (w.next(a))
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                const int qb = qi % a.qbufs, use = qi / a.qbufs, rows = min(NB, w.n * a.G - q0), N = (rows + 15) & ~15;
                if (use > 0) mb_wait(&qempty[qb], (use - 1) & 1, &s_stop);
                const int th = threadIdx.x - 18 * 32;  // a row's token, log-sum-exp and bound
                if (th < N) {
                    const int j = (q0 + th) >> a.lg, head = w.s_kvh * a.G + ((q0 + th) & (a.G - 1));
                    const int sel = th < rows ? __ldg(a.sel + (size_t)w.s_slot * a.max_q + j) : -1, t = sel < a.v.tokens ? sel : -1;
                    // a query that is left out, or saw nothing (-inf), sees no row
                    const float e = t >= 0 ? a.lse[w.s_layer * a.lse_layer + (long long)t * a.heads + head] : -INFINITY;
                    s_lse[qb][th] = e * -1.4426950408889634f;
                    s_last[qb][th] = e == -INFINITY ? -1 : w.L + j;
                    s_tok[th] = t;
                }
                bar_sync(1, 128);
                if (wl == 0) {
                    unsigned ok = 0;
                    for (int i = 0; i < N; i += 32) {  // two groups of 16 a step
                        const unsigned m = __ballot_sync(0xffffffffu, i + lane < N && s_last[qb][i + lane] >= 0);
                        ok |= ((m & 0xffffu) == 0xffffu ? 1u : 0u) << (i >> 4) | (m >> 16 == 0xffffu ? 2u : 0u) << (i >> 4);
                    }
                    if (lane == 0) s_counts[qb] = ok;
                }
                uint8_t *dst0 = sq + qb * qbuf_b;
                if constexpr (sizeof(T) == 2) {
                    // bf16 rows as they are, 16 bytes a copy, all in flight
                    constexpr int CH = HD / 8;
                    const T *src0 = (const T *)a.q + w.s_layer * a.q_layer + (long long)w.s_kvh * a.G * HD;
                    for (int e = th; e < N * CH; e += 128) {
                        const int r = e / CH, c = e % CH, t = s_tok[r];
                        const uint32_t dst = kv_smem(dst0 + (c >> 3) * half_b + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst),
                                     "l"(src0 + (t >= 0 ? t * a.q_ld + ((q0 + r) & (a.G - 1)) * HD + c * 8 : 0)), "r"(t >= 0 ? 16 : 0)
                                     : "memory");
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                } else {
                    const int half = HD == 128 ? lane >> 4 : 0, c = (lane & 15) * 4;
                    const T *src0 = (const T *)a.q + w.s_layer * a.q_layer + (long long)w.s_kvh * a.G * HD + half * 64 + c;
                    constexpr int B = 4;
                    for (int r0 = wl; r0 < N; r0 += 4 * B) {  // a warp to a row, four rows in flight (eight: 74 -> 95 us at 31 queries)
                        float4 q[B];
#pragma unroll
                        for (int i = 0; i < B; i++) {
                            const int r = r0 + 4 * i, t = r < N ? s_tok[r] : -1;
                            q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (t >= 0 && (HD == 128 || lane < 16)) {
                                const T *src = src0 + t * a.q_ld + ((q0 + r) & (a.G - 1)) * HD;
                                q[i] = *(const float4 *)src;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < B; i++) {
                            const int r = r0 + 4 * i;
                            if (r < N && (HD == 128 || lane < 16)) {
                                uint32_t lo[QT], hi[QT];
                                split_bf16<QT>(q[i].x, q[i].y, lo);
                                split_bf16<QT>(q[i].z, q[i].w, hi);
                                uint8_t *dst = dst0 + half * half_b + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | ((c & 4) << 1));
#pragma unroll
                                for (int x = 0; x < QT; x++) *(uint2 *)(dst + x * term_b) = make_uint2(lo[x], hi[x]);
                            }
                        }
                    }
                }
                bar_sync(1, 128);  // s_tok is free again
                fence_async_smem();
                mb_arrive(&qfull[qb]);
            }
    } else {
        const int th = threadIdx.x & 127, group = warp >> 2;
        const float sl2 = a.scale * 1.4426950408889634f;
        int uses = 0, qi = 0, turn = 0;
        while (w.next(a)) {
            float *acc = a.acc + (((size_t)w.s_layer * a.v.slots + w.s_slot) * a.v.kvh + w.s_kvh) * a.acc_rows;
            for (int q0 = 0; q0 < w.n * a.G; q0 += NB, qi++) {
                const int qb = qi % a.qbufs, N = (min(NB, w.n * a.G - q0) + 15) & ~15;
                mb_wait(&qfull[qb], (qi / a.qbufs) & 1, &s_stop);
                const unsigned counts = s_counts[qb];  // bit c: all of queries 16 c .. 16 c + 15 count
                for (int t = w.s_a + (group - turn % NS + NS) % NS; t < w.s_b; t += NS, uses++) {
                    const int r = t * 128 + th;
                    float sum = r < w.end && (r < w.L || q0 > 0) ? acc[r] : 0.f;
                    mb_wait(&sfull[group], uses & 1, &s_stop);
                    um_fence_after();
                    float2 part[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    const bool open = t * 128 + 127 <= w.L;  // all rows of the tile are seen by all queries that count
                    for (int c = 0; c < N; c += 16) {
                        float x[16];
                        um_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + group * 128 + c, x);
                        um_wait_ld<16>(x);
                        float2 p[8];
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const float4 e = *(const float4 *)&s_lse[qb][c + i];
                            const float2 y0 = fma2(make_float2(x[i], x[i + 1]), make_float2(sl2, sl2), make_float2(e.x, e.y));
                            const float2 y1 = fma2(make_float2(x[i + 2], x[i + 3]), make_float2(sl2, sl2), make_float2(e.z, e.w));
                            p[i / 2] = make_float2(ex2(y0.x), ex2(y0.y));
                            p[i / 2 + 1] = make_float2(ex2(y1.x), ex2(y1.y));
                        }
                        if (!open || !((counts >> (c >> 4)) & 1)) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const int4 e = *(const int4 *)&s_last[qb][c + i];
                                if (r > e.x) p[i / 2].x = 0.f;
                                if (r > e.y) p[i / 2].y = 0.f;
                                if (r > e.z) p[i / 2 + 1].x = 0.f;
                                if (r > e.w) p[i / 2 + 1].y = 0.f;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; i++) part[i & 1] = add2(part[i & 1], p[i]);
                    }
                    um_fence_before();
                    mb_arrive(&sempty[group]);
                    if (r < w.end) {
                        float add = (part[0].x + part[0].y) + (part[1].x + part[1].y);
                        if (add != add) add = weights_redo<T, HD>(a, w.s_layer, w.s_slot, w.s_kvh, r, q0, N, s_lse[qb], s_last[qb], sl2);
                        acc[r] = sum + add;
                    }
                }
                mb_arrive(&qempty[qb]);
            }
            turn++;
        }
    }
    __syncthreads();
    if (warp == 17) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace
