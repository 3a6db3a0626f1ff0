// hy_kvtree.cuh — attention of drafted token trees over a paged KV cache.
//
// x_r = scale * q . k_r over the rows r that a node sees (its slot's cached
// rows, its ancestors' and its own), out = sum_r softmax(x)_r v_r, lse = log
// sum_r exp(x_r).  The query heads of a group share K and V, so the rows of
// one problem are the (node, head) pairs of a slot and KV head: 4 hd bytes of
// cache a row r against 4 hd flops for each of them.
#pragma once
#include "hy_kvview.cuh"

namespace {

struct TreeArgs {
    KvView v;
    int layer, heads, G, max_nodes;
    const int *len, *off, *parent;
    const void *q;
    long long q_ld;
    float scale;
    void *out;
    long long out_ld;
    float *lse;
    // split columns: the pieces' (max, sum) and unnormalised outputs, and for
    // each range the column that starts in it and goes on in the next one as
    // {slot, KV head, first tile, tiles per range}; slot < 0: none
    int4 *roots;
    float2 *part_ml;
    float *part_o;
    int lg;  // log2 G
    int ranges, row_blocks, min_tiles;
};

__device__ __forceinline__ void st_row4(float *p, float a, float b, float c, float d) { *(float4 *)p = make_float4(a, b, c, d); }
__device__ __forceinline__ void st_row4(__nv_bfloat16 *p, float a, float b, float c, float d) {
    *(uint2 *)p = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}
__device__ __forceinline__ float4 ld_row4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ float4 ld_row4(const __nv_bfloat16 *p) {
    const uint2 u = *(const uint2 *)p;
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

// Work is cut into tiles of TK cached rows of one (slot, KV head) column, in
// slot order, and into `ranges` runs of equal length, one per CTA (and row
// block): every SM gets the same share whatever the lengths are.  A column
// that ends up in several ranges leaves (max, sum, out) pieces which
// tree_merge joins.
template <int TK>
struct TreeWalk {
    int slot, rem, left, g, g0;       // next tile: slot, index within the slot's tiles; tiles left; global index, first
    int L, t0, n, T, at;              // the slot whose numbers are loaded
    // the segment: tiles a .. b - 1 of column (slot, kvh)
    int s_slot, s_kvh, s_a, s_b, s_g;

    __device__ __forceinline__ static int tiles(int L, int n, int cap) { return n > 0 ? (min(L + n, cap) + TK - 1) / TK : 0; }
    __device__ __forceinline__ bool next(const TreeArgs &a, int first_node) {
        while (left > 0) {
            if (slot >= a.v.slots) return false;
            if (at != slot) {
                tree_span(a.v, a.len, a.off, a.max_nodes, slot, L, t0, n);
                T = tiles(L, n, a.v.page_max * kPageRows);
                at = slot;
            }
            if (rem >= T * a.v.kvh) {
                slot++;
                rem = 0;
                continue;
            }
            s_slot = slot;
            s_kvh = rem / T;
            s_a = rem % T;
            s_b = min(T, s_a + left);
            s_g = g;
            const int c = s_b - s_a;
            left -= c;
            rem += c;
            g += c;
            if (first_node < n) return true;
        }
        return false;
    }
};

// The walk's start for this CTA's range.  Every thread takes a run of slots;
// s_scan holds blockDim.x / 32 + 2 ints of scratch, s_start 4.
template <int TK>
__device__ __forceinline__ void tree_plan(const TreeArgs &a, int range, int *s_scan, int *s_start) {
    const int th = threadIdx.x, nth = blockDim.x, lane = th & 31, w = th >> 5, cap = a.v.page_max * kPageRows;
    const int per = (a.v.slots + nth - 1) / nth, b0 = min(a.v.slots, th * per), b1 = min(a.v.slots, b0 + per);
    int sum = 0;
    for (int s = b0; s < b1; s++) {
        int L, t0, n;
        tree_span(a.v, a.len, a.off, a.max_nodes, s, L, t0, n);
        sum += TreeWalk<TK>::tiles(L, n, cap) * a.v.kvh;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[w] = incl;
    __syncthreads();
    int before = incl - sum, total = 0;
    for (int i = 0; i < (nth >> 5); i++) {
        if (i < w) before += s_scan[i];
        total += s_scan[i];
    }
    const int C = max((total + a.ranges - 1) / a.ranges, a.min_tiles), g0 = range * C;
    if (th == 0) {
        s_start[2] = max(0, min(C, total - g0));  // tiles of this range
        s_start[3] = C;
    }
    if (g0 >= before && g0 < before + sum) {
        for (int s = b0; s < b1; s++) {
            int L, t0, n;
            tree_span(a.v, a.len, a.off, a.max_nodes, s, L, t0, n);
            const int c = TreeWalk<TK>::tiles(L, n, cap) * a.v.kvh;
            if (g0 < before + c) {
                s_start[0] = s;
                s_start[1] = g0 - before;
                break;
            }
            before += c;
        }
    }
    __syncthreads();
}

template <int TK>
__device__ __forceinline__ TreeWalk<TK> tree_walk(const int *s_start, int range) {
    TreeWalk<TK> w;
    w.left = s_start[2];
    w.slot = w.left > 0 ? s_start[0] : 0;
    w.rem = w.left > 0 ? s_start[1] : 0;
    w.g = w.g0 = range * s_start[3];
    w.at = -1;
    return w;
}

// Ancestor masks of a slot's nodes (bit j of s_mask[i]: node i sees node j),
// by pointer doubling: after round k a node knows its next 2^k ancestors.
// Called by NT threads (NT >= 64) that share named barrier `bar`.
template <int NT>
__device__ __forceinline__ void tree_masks(const TreeArgs &a, int t0, int n, int th, int bar, int8_t *s_up,
                                           unsigned long long *s_mask) {
    bar_sync(bar, NT);  // the masks of the segment before are no longer read
    int up = -1;
    unsigned long long m = 0;
    if (th < kTreeMax) {
        const int p = th < n ? __ldg(a.parent + t0 + th) : -2;
        s_up[th] = (int8_t)(p == -2 ? -2 : p < 0 || p >= th ? -1 : p);
    }
    bar_sync(bar, NT);
    if (th < kTreeMax) {
        const int p = s_up[th];
        if (p != -2) {
            m = 1ull << th;
            if (p >= 0 && s_up[p] != -2) up = p;
        }
    }
    bar_sync(bar, NT);
#pragma unroll 1
    for (int k = 0; k < 6; k++) {
        if (th < kTreeMax) {
            s_up[th] = (int8_t)up;
            s_mask[th] = m;
        }
        bar_sync(bar, NT);
        if (th < kTreeMax && up >= 0) {
            m |= s_mask[up];
            up = s_up[up];
        }
        bar_sync(bar, NT);
    }
    if (th < kTreeMax) s_mask[th] = m;
    bar_sync(bar, NT);
}

// p_r v_r of drafted rows whose V is not finite (in dims d0 .. d0 + HD / 2 -
// 1), for one (node, head): the matrix product leaves such rows out, and the
// nodes that see them add them here, in the order of the rows.
template <typename T, int HD>
__device__ __noinline__ void tree_add_bad(const TreeArgs &a, int slot, int kvh, int L, int t, int head, int d0,
                                          unsigned long long bad, float sl2, float m, float *o) {
    while (bad) {
        const int j = __ffsll((long long)bad) - 1;
        bad &= bad - 1;
        const int pg = a.v.page(slot, L + j);
        if (pg < 0) continue;
        const uint16_t *k = a.v.kv + a.v.row(a.layer, pg, L + j) + kvh * HD, *v = k + kPageRows * a.v.kvd;
        const T *q = (const T *)a.q + (long long)t * a.q_ld + (long long)head * HD;
        float x = 0.f;
        for (int d = 0; d < HD; d += 4) {
            const float4 qq = ld_row4(q + d);
            x = fmaf(qq.x, bf16_bits_to_f32(k[d]), x);
            x = fmaf(qq.y, bf16_bits_to_f32(k[d + 1]), x);
            x = fmaf(qq.z, bf16_bits_to_f32(k[d + 2]), x);
            x = fmaf(qq.w, bf16_bits_to_f32(k[d + 3]), x);
        }
        const float p = ex2((a.scale < 0.f ? -x : x) * sl2 - m);
        for (int d = 0; d < HD / 2; d++) o[d] = fmaf(p, bf16_bits_to_f32(v[d0 + d]), o[d]);
    }
}

// ---------------------------------------------------------------- wide trees: tcgen05
//
// One CTA takes up to 128 (node, head) rows, the lanes of a tensor-memory
// tile, against tiles of 128 cached rows:
//   warp 8     streams K and V pages by TMA into a ring of stages, 128-byte
//              swizzled: K rows are the K-major B operand of Q . K^T, V rows
//              the MN-major B operand of P . V, so nothing is transposed
//   warp 9     issues S = Q . K^T (two S tiles, so that the next
//              one runs while this one's softmax does) and O += P . V
//   warps 0-7  half a row's tile a thread: S from tensor memory, running
//              maximum and sum, P back over S as the A operand in tensor
//              memory (with four warps and a whole row a thread, the softmax
//              took 2.7 us a tile, twice what its rows take from memory)
// fp32 queries enter the bf16 products as three bf16 terms (all 24 bits), and
// so does P for fp32 outputs: K and V are bf16 already, and every sum is
// fp32.  For bf16 outputs P has two terms (16 bits): one would add an error
// as large as the output's own rounding.  The maximum that P is taken
// against moves only when it would grow by over 2^8, which rescales O; sums
// and outputs stay exact under it, as the same one divides out at the end.
constexpr int kTtK = 128;       // cached rows of a tile
constexpr int kTtThreads = 320, kTtSoft = 256;

template <typename T>
__host__ __device__ constexpr int tt_qterms() { return sizeof(T) == 4 ? 3 : 1; }
template <typename T>
__host__ __device__ constexpr int tt_pterms() { return sizeof(T) == 4 ? 3 : 2; }
template <int HD>
__host__ __device__ constexpr int tt_stage() { return (HD / 64) * 128 * 128; }
template <typename T, int HD>
__host__ __device__ constexpr int tt_qbytes() { return tt_qterms<T>() * tt_stage<HD>(); }
template <typename T, int HD>
__host__ __device__ constexpr int tt_stages() {
    const int s = (224 * 1024 - tt_qbytes<T, HD>()) / tt_stage<HD>();
    return s > 8 ? 8 : s;
}
// Beside it the kernel has at most 2 KB of static shared memory.
template <typename T, int HD>
__host__ __device__ constexpr size_t tt_smem() { return (size_t)tt_qbytes<T, HD>() + (size_t)tt_stages<T, HD>() * tt_stage<HD>() + 1024; }

// Tensor memory columns: S / P of tiles 2i and 2i + 1 (P's third term apart), O.
constexpr uint32_t kTtS = 0, kTtO = 256, kTtX = 384;

template <typename T, int HD>
__global__ void __launch_bounds__(kTtThreads, 1) tree_attn_tc(const __grid_constant__ TreeArgs a,
                                                              const __grid_constant__ CUtensorMap map) {
    constexpr int QT = tt_qterms<T>(), PT = tt_pterms<T>(), NH = HD / 64, NST = tt_stages<T, HD>(), STB = tt_stage<HD>();
    static_assert(NST >= 4, "K and V of two tiles in flight");
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[NST], empty[NST], sfull[2], pfull[2], odone[2], qfull, ofree, fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_scan[kTtThreads / 32], s_start[4];
    __shared__ int8_t s_up[kTreeMax];
    __shared__ unsigned long long s_mask[kTreeMax], s_bad[2][2];
    __shared__ float s_half[2][128];
    __shared__ int s_stop;
    uint8_t *sq = (uint8_t *)(((uintptr_t)dsm + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sq + tt_qbytes<T, HD>();
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rb = blockIdx.x % a.row_blocks, range = blockIdx.x / a.row_blocks;
    const int NB = 128 / a.G, node0 = rb * NB;  // nodes of a row block
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < NST; i++) {
            mb_init(&full[i], 1);
            mb_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mb_init(&sfull[i], 1);
            mb_init(&pfull[i], kTtSoft);
            mb_init(&odone[i], 1);
            s_bad[i][0] = s_bad[i][1] = 0;
        }
        mb_init(&qfull, kTtSoft);
        mb_init(&ofree, kTtSoft);
        mb_init(&fin, 1);
        s_stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(kv_smem(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        um_fence_before();
    }
    pdl_wait();
    tree_plan<kTtK>(a, range, s_scan, s_start);
    um_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    TreeWalk<kTtK> w = tree_walk<kTtK>(s_start, range);
    const int cap = a.v.page_max * kPageRows;
    const bool range_root = rb == 0 && threadIdx.x == 0;  // the thread that notes the range's split column
    if (range_root) a.roots[range] = make_int4(-1, 0, 0, 0);
    if (warp == 8) {
        // eight pages a tile, K then V; a page that does not exist is read past
        // the end of the map, which fills zeros
        const int y0 = a.layer * a.v.npages * 2 * kPageRows, yend = a.v.layers * a.v.npages * 2 * kPageRows;
        int pos = 0;
        while (w.next(a, node0)) {
            const int pages = (min(w.L + w.n, cap) + kPageRows - 1) / kPageRows;
            for (int t = w.s_a; t < w.s_b; t++) {
                const int j = t * (kTtK / kPageRows) + (lane & 7);
                int pg = j < pages ? __ldg(a.v.pages + (size_t)w.s_slot * a.v.page_max + j) : -1;
                const int y = pg < 0 || pg >= a.v.npages ? yend : y0 + pg * 2 * kPageRows;
                for (int kv = 0; kv < 2; kv++, pos++) {
                    const int st = pos % NST, use = pos / NST;
                    if (use > 0) mb_wait(&empty[st], (use - 1) & 1, &s_stop);
                    if (__any_sync(0xffffffffu, *(volatile int *)&s_stop)) break;
                    int yj[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) yj[i] = __shfl_sync(0xffffffffu, y == yend ? yend : y + kv * kPageRows, i);
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
        }
        // copies in flight land before the kernel ends, also after a wait gave up
        for (int p = max(0, pos - NST); p < pos; p++) {
            int none = 0;  // never set: the wait itself is bounded
            mb_wait(&full[p % NST], (p / NST) & 1, &none);
        }
    } else if (warp == 9) {
        {
            constexpr uint32_t iqk = um_idesc(128, kTtK, false), ipv = um_idesc(128, HD, true);
            const uint32_t ring0 = __shfl_sync(0xffffffffu, kv_smem(ring), 0), q0 = um_desc_lo(__shfl_sync(0xffffffffu, kv_smem(sq), 0), 16);
            int it = 0, seg = 0;  // tiles and segments done
            // O += P(i) . V(i); the segment's first one overwrites O
            auto pv = [&](int i, bool first) {
                const int pos = 2 * i + 1, st = pos % NST;
                mb_wait(&pfull[i & 1], (i >> 1) & 1, &s_stop);
                mb_wait(&full[st], (pos / NST) & 1, &s_stop);
                if (first && seg > 0) mb_wait(&ofree, (seg - 1) & 1, &s_stop);
                um_fence_after();
                const uint32_t vb = um_desc_lo(ring0 + st * STB, 16384), p0 = tmem + kTtS + (i & 1) * 128, px = tmem + kTtX + (i & 1) * 64;
                if (elect()) {
#pragma unroll
                    for (int x = PT - 1; x >= 0; x--)  // small terms first
#pragma unroll
                        for (int k = 0; k < kTtK / 16; k++)
                            um_mma_ts(tmem + kTtO, (x == 2 ? px : p0 + x * 64) + k * 8, vb + k * (2048 / 16), ipv,
                                      x == PT - 1 && k == 0 ? !first : true);
                    um_commit(&empty[st]);
                    um_commit(&odone[i & 1]);
                }
                __syncwarp();
            };
            while (w.next(a, node0)) {
                for (int t = w.s_a; t < w.s_b; t++, it++) {
                    const int pos = 2 * it, st = pos % NST;
                    if (t == w.s_a) mb_wait(&qfull, seg & 1, &s_stop);
                    mb_wait(&full[st], (pos / NST) & 1, &s_stop);
                    um_fence_after();
                    const uint32_t kb = um_desc_lo(ring0 + st * STB, 16), s0 = tmem + kTtS + (it & 1) * 128;
                    if (elect()) {
#pragma unroll
                        for (int x = QT - 1; x >= 0; x--)
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) {
                                const uint32_t at = ((k >> 2) * 16384 + (k & 3) * 32) / 16;
                                um_mma(s0, q0 + x * (STB / 16) + at, kb + at, iqk, !(x == QT - 1 && k == 0));
                            }
                        um_commit(&empty[st]);
                        um_commit(&sfull[it & 1]);
                    }
                    __syncwarp();
                    if (t > w.s_a) pv(it - 1, t - 1 == w.s_a);
                }
                pv(it - 1, w.s_b - 1 == w.s_a);
                seg++;
            }
            if (elect()) um_commit(&fin);
            __syncwarp();
            int none = 0;
            mb_wait(&fin, 0, &none);
        }
    } else {
        const int th = threadIdx.x & 127, h = warp >> 2;  // row, and half of its keys and dims
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float sl2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
        int it = 0, seg = 0, last_slot = -1;
        // the segment's Q into shared memory, a warp to a row, four in flight
        auto load_q = [&](const TreeWalk<kTtK> &x) {
            const int rows = min(NB, x.n - node0) << a.lg;
            const int half = HD == 128 ? lane >> 4 : 0, c = (lane & 15) * 4;  // dims half * 64 + c ..
            const bool on = HD == 128 || lane < 16;
            const T *src = (const T *)a.q + (long long)(x.t0 + node0) * a.q_ld + (long long)x.s_kvh * a.G * HD + half * 64 + c;
            for (int r0 = warp; r0 < rows; r0 += 32) {
                float4 q[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + 8 * i;
                    q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (on && r < rows) q[i] = ld_row4(src + (long long)(r >> a.lg) * a.q_ld + (r & (a.G - 1)) * HD);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + 8 * i;
                    if (!on || r >= rows) continue;
                    if (a.scale < 0.f) q[i] = make_float4(-q[i].x, -q[i].y, -q[i].z, -q[i].w);
                    uint32_t lo[QT], hi[QT];
                    split_bf16<QT>(q[i].x, q[i].y, lo);
                    split_bf16<QT>(q[i].z, q[i].w, hi);
                    uint8_t *dst = sq + half * 16384 + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | ((c & 4) << 1));
#pragma unroll
                    for (int k = 0; k < QT; k++) *(uint2 *)(dst + k * STB) = make_uint2(lo[k], hi[k]);
                }
            }
            fence_async_smem();
            mb_arrive(&qfull);
        };
        bool have = w.next(a, node0);
        if (have) load_q(w);
        while (have) {
            const TreeWalk<kTtK> cur = w;
            if (cur.s_slot != last_slot) {
                tree_masks<kTtSoft>(a, cur.t0, cur.n, threadIdx.x, 1, s_up, s_mask);
                last_slot = cur.s_slot;
            }
            const int rows = min(NB, cur.n - node0) << a.lg, end = min(cur.L + cur.n, cap);
            const bool active = (warp & 3) * 32 < rows;
            const int node = node0 + (th >> a.lg);
            unsigned long long mask = th < rows ? s_mask[node] : 0;
            const bool live = mask != 0;  // not a padding node
            if (end - cur.L < 64) mask &= (1ull << max(0, end - cur.L)) - 1;
            float m = -INFINITY, l = 0.f;
            for (int t = cur.s_a; t < cur.s_b; t++, it++) {
                const int b = it & 1, r0 = t * kTtK;
                const bool tail = r0 + kTtK > cur.L, first = t == cur.s_a;
                mb_wait(&sfull[b], (it >> 1) & 1, &s_stop);
                um_fence_after();
                const uint32_t sp = tmem + lanes + kTtS + b * 128, px = tmem + lanes + kTtX + b * 64;
                float s[64], my = -INFINITY;
                if (active) {
#pragma unroll
                    for (int c = 0; c < 2; c++) um_ld32(sp + h * 64 + c * 32, s + c * 32);
                    um_wait_ld<64>(s);
                    if (tail || !live) {
                        // bits of this half's rows that the node sees
                        const int c = cur.L - r0 - h * 64;  // cached rows among them
                        unsigned long long see = 0;
                        if (live) see = c >= 64 ? ~0ull : c > 0 ? ((1ull << c) - 1) | (mask << c) : -c >= 64 ? 0 : mask >> -c;
#pragma unroll
                        for (int i = 0; i < 64; i++)
                            if (!((see >> i) & 1)) s[i] = -INFINITY;
                    }
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int i = 4; i < 64; i++) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
                    my = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
                }
                // both halves have read S, and whether any row's maximum moves
                if (bar_or(2, kTtSoft, active && (first || my > m + 8.f))) {
                    s_half[h][th] = my;
                    bar_sync(1, kTtSoft);
                    const float tm = fmaxf(my, s_half[h ^ 1][th]);
                    if (first) {
                        m = tm;
                    } else {
                        const float mn = tm > m + 8.f ? tm : m, f = m == -INFINITY ? 1.f : ex2(m - mn);
                        const bool moved = mn > m;
                        m = mn;
                        l *= f;
                        if (active && __any_sync(0xffffffffu, moved)) {
                            mb_wait(&odone[(it - 1) & 1], ((it - 1) >> 1) & 1, &s_stop);
                            um_fence_after();
#pragma unroll
                            for (int c = 0; c < HD / 64; c++) {
                                const uint32_t at = tmem + lanes + kTtO + h * (HD / 2) + c * 32;
                                float o[32];
                                um_ld32(at, o);
                                um_wait_ld<32>(o);
#pragma unroll
                                for (int i = 0; i < 32; i++) o[i] *= f;
                                um_st32(at, o);
                            }
                            um_wait_st();
                        }
                    }
                }
                if (active) {
                    const float mr = m == -INFINITY ? 0.f : m;
                    float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t p[PT][16];
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float p0 = ex2(fmaf(s[c * 32 + 2 * i], sl2, -mr)), p1 = ex2(fmaf(s[c * 32 + 2 * i + 1], sl2, -mr));
                            ls[i & 3] += p0 + p1;
                            uint32_t x[PT];
                            split_bf16<PT>(p0, p1, x);
#pragma unroll
                            for (int k = 0; k < PT; k++) p[k][i] = x[k];
                        }
                        um_st16(sp + h * 32 + c * 16, p[0]);
                        um_st16(sp + 64 + h * 32 + c * 16, p[1]);
                        if constexpr (PT == 3) um_st16(px + h * 32 + c * 16, p[PT - 1]);
                    }
                    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
                    um_wait_st();
                }
                if (tail) {
                    // V rows that no node sees become zeros (a product with a
                    // probability of 0 must be 0), and so do halves of drafted
                    // rows that are not finite, which the nodes that see them
                    // add at the end
                    const int pos = 2 * it + 1, st = pos % NST, r = r0 + th;
                    mb_wait(&full[st], (pos / NST) & 1, &s_stop);
                    if (r >= cur.L) {
                        uint8_t *vr = ring + (size_t)st * STB + (HD == 128 ? h * 16384 : 0) + th * 128;
                        const int c0 = HD == 128 ? 0 : h * 4;  // its 16-byte chunks
                        bool bad = false;
                        if (r < end)
                            for (int i = 0; i < HD / 16; i++) {
                                const uint4 u = *(const uint4 *)(vr + (((c0 + i) ^ (th & 7)) << 4));
                                const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    bad |= (x[k] & 0x7f80u) == 0x7f80u || (x[k] & 0x7f800000u) == 0x7f800000u;
                            }
                        if (bad) atomicOr(&s_bad[seg & 1][h], 1ull << (r - cur.L));
                        if (bad || r >= end)
                            for (int i = 0; i < HD / 16; i++) *(uint4 *)(vr + (((c0 + i) ^ (th & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                }
                um_fence_before();
                mb_arrive(&pfull[b]);
            }
            // every S of the segment is done, so the next one's Q may go in
            // while the last P . V runs
            have = w.next(a, node0);
            if (have) load_q(w);
            s_half[h][th] = l;
            bar_sync(1, kTtSoft);  // and s_bad is complete
            l = h ? s_half[0][th] + l : l + s_half[1][th];
            const unsigned long long bad = s_bad[seg & 1][h] & mask;
            if (th == 0) s_bad[(seg + 1) & 1][h] = 0;
            const bool whole = cur.s_a == 0 && cur.s_b == cur.T;
            mb_wait(&odone[(it - 1) & 1], ((it - 1) >> 1) & 1, &s_stop);
            um_fence_after();
            if (active) {
                constexpr int W = HD / 2;
                float o[W];
#pragma unroll
                for (int c = 0; c < W / 32; c++) um_ld32(tmem + lanes + kTtO + h * W + c * 32, o + c * 32);
                um_wait_ld<W>(o);
                um_fence_before();
                mb_arrive(&ofree);
                if (th < rows) {
                    const int tok = cur.t0 + node, head = cur.s_kvh * a.G + (th & (a.G - 1));
                    if (bad && l > 0.f) {
                        float x[W];  // its address is taken: o stays in registers
#pragma unroll
                        for (int d = 0; d < W; d++) x[d] = o[d];
                        tree_add_bad<T, HD>(a, cur.s_slot, cur.s_kvh, cur.L, tok, head, h * W, bad, sl2, m, x);
#pragma unroll
                        for (int d = 0; d < W; d++) o[d] = x[d];
                    }
                    if (whole) {
                        const float inv = l == 0.f ? 0.f : 1.0f / l;
                        T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + h * W;
#pragma unroll
                        for (int d = 0; d < W; d += 4) st_row4(dst + d, o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
                        if (a.lse && h == 0)
                            a.lse[(long long)tok * a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                    } else {
                        const int piece = (2 * range + (cur.s_g != cur.g0)) * a.row_blocks + rb;
                        if (h == 0) a.part_ml[(size_t)piece * 128 + th] = make_float2(m, l);
                        float *po = a.part_o + (size_t)piece * 128 * HD + h * W * 128 + th * 8;
#pragma unroll
                        for (int d = 0; d < W; d += 8) {
                            *(float4 *)(po + d * 128) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
                            *(float4 *)(po + d * 128 + 4) = make_float4(o[d + 4], o[d + 5], o[d + 6], o[d + 7]);
                        }
                    }
                }
            } else {
                mb_arrive(&ofree);
            }
            if (range_root && cur.s_a == 0 && !whole) a.roots[range] = make_int4(cur.s_slot, cur.s_kvh, cur.s_g, s_start[3]);
            bar_sync(1, kTtSoft);
            seg++;
        }
    }
    __syncthreads();
    if (warp == 9) {
        um_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// grid (ranges, blocks of rows): joins the pieces of the column that starts in
// a range and goes on in the next: M = max m_i, out = sum 2^(m_i - M) o_i / sum
// 2^(m_i - M) l_i.  Four warps to a (node, head) row, each every fourth piece,
// hd / 32 dims a lane, joined in a fixed order.
constexpr int kMergeRows = 4, kMergeThreads = kMergeRows * 128;
template <typename T, int HD, int TK>
__global__ void __launch_bounds__(kMergeThreads) tree_merge(const __grid_constant__ TreeArgs a) {
    constexpr int D = HD / 32;
    __shared__ float s_o[kMergeRows][4][HD], s_s[kMergeRows][4];
    pdl_wait();
    const int4 root = a.roots[blockIdx.x];
    if (root.x < 0) return;
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 7, part = (threadIdx.x >> 5) & 3;
    int L, t0, n;
    tree_span(a.v, a.len, a.off, a.max_nodes, root.x, L, t0, n);
    const int T_ = TreeWalk<TK>::tiles(L, n, a.v.page_max * kPageRows), C = root.w;
    const int p0 = root.z / C, p1 = (root.z + T_ - 1) / C, rows = n * a.G;
    for (int r0 = blockIdx.y * kMergeRows; r0 < rows; r0 += gridDim.y * kMergeRows) {
        const int r = r0 + row, node = r / a.G, rb = r >> 7, lr = r & 127;
        const auto piece = [&](int p) { return (size_t)((2 * p + (p * C < root.z)) * a.row_blocks + rb); };
        float M = -INFINITY, S = 0.f, o[D];
#pragma unroll
        for (int d = 0; d < D; d++) o[d] = 0.f;
        const int d0 = lane * D;
        if (r < rows) {
            for (int p = p0 + lane; p <= p1; p += 32) {
                const float2 ml = a.part_ml[piece(p) * 128 + lr];
                if (ml.y != 0.f) M = fmaxf(M, ml.x);
            }
            M = warp_max(M);
#pragma unroll 4
            for (int p = p0 + part; p <= p1; p += 4) {
                const size_t pc = piece(p);
                const float2 ml = a.part_ml[pc * 128 + lr];
                const float *po = a.part_o + pc * 128 * HD + (d0 >> 3) * 1024 + lr * 8 + (d0 & 7);
                float v[D];
                if constexpr (D == 4) {
                    const float4 x = *(const float4 *)po;
                    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
                } else {
                    const float2 x = *(const float2 *)po;
                    v[0] = x.x, v[1] = x.y;
                }
                const float f = ml.y == 0.f ? 0.f : ex2(ml.x - M);  // 0: nothing seen in this piece
                S = fmaf(ml.y, f, S);
#pragma unroll
                for (int d = 0; d < D; d++) o[d] = fmaf(v[d], f, o[d]);
            }
        }
#pragma unroll
        for (int d = 0; d < D; d++) s_o[row][part][d0 + d] = o[d];
        if (lane == 0) s_s[row][part] = S;
        __syncthreads();
        if (part == 0 && r < rows) {
            S = (s_s[row][0] + s_s[row][1]) + (s_s[row][2] + s_s[row][3]);
            const float inv = S == 0.f ? 0.f : 1.0f / S;
#pragma unroll
            for (int d = 0; d < D; d++)
                o[d] = ((s_o[row][0][d0 + d] + s_o[row][1][d0 + d]) + (s_o[row][2][d0 + d] + s_o[row][3][d0 + d])) * inv;
            const int tok = t0 + node, head = root.y * a.G + r % a.G;
            T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + d0;
            if constexpr (D == 4) st_row4(dst, o[0], o[1], o[2], o[3]);
            else if constexpr (sizeof(T) == 4) *(float2 *)dst = make_float2(o[0], o[1]);
            else *(uint32_t *)dst = pack_bf16(o[0], o[1]);
            if (a.lse && lane == 0) a.lse[(long long)tok * a.heads + head] = S == 0.f ? -INFINITY : (M + log2f(S)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

}  // namespace
