// hy_kvtree.cuh — attention of drafted token trees over a paged KV cache.
//
// x_r = scale * q . k_r over the rows r that a node sees (its slot's cached
// rows, its ancestors' and its own), out = sum_r softmax(x)_r v_r, lse = log
// sum_r exp(x_r).  The query heads of a group share K and V, so the rows of
// one problem are the (node, head) pairs of a slot and KV head: 4 hd bytes of
// cache a row r against 4 hd flops for each of them.
#pragma once
#include <cfloat>
#include <cmath>

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
    // each range the column whose first tile it has and which goes on in the next
    // one as {slot, KV head, first place, places per range}; slot < 0: none
    int4 *roots;
    float2 *part_ml;
    float *part_o;
    int lg;      // log2 G
    bool out32;  // every output row is 32-byte aligned
    bool whole;  // narrow form: whole columns to each range
    int ranges, row_blocks;
};

__device__ __forceinline__ void st_row4(float *p, float a, float b, float c, float d) { *(float4 *)p = make_float4(a, b, c, d); }
__device__ __forceinline__ void st_row4(__nv_bfloat16 *p, float a, float b, float c, float d) {
    *(uint2 *)p = make_uint2(pack_bf16(a, b), pack_bf16(c, d));
}
// Eight values of a row, 32 (bf16: 16) bytes a lane; fp32 rows that are only
// 16-byte aligned (wide false) take two stores.
__device__ __forceinline__ void st_row8(float *p, const float *v, float f, bool wide) {
    if (wide) {
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0] * f), "f"(v[1] * f), "f"(v[2] * f),
                     "f"(v[3] * f), "f"(v[4] * f), "f"(v[5] * f), "f"(v[6] * f), "f"(v[7] * f)
                     : "memory");
    } else {
        st_row4(p, v[0] * f, v[1] * f, v[2] * f, v[3] * f);
        st_row4(p + 4, v[4] * f, v[5] * f, v[6] * f, v[7] * f);
    }
}
__device__ __forceinline__ void st_row8(__nv_bfloat16 *p, const float *v, float f, bool) {
    *(uint4 *)p = make_uint4(pack_bf16(v[0] * f, v[1] * f), pack_bf16(v[2] * f, v[3] * f), pack_bf16(v[4] * f, v[5] * f),
                             pack_bf16(v[6] * f, v[7] * f));
}
__device__ __forceinline__ float4 ld_row4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ float4 ld_row4(const __nv_bfloat16 *p) {
    const uint2 u = *(const uint2 *)p;
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}

// Work is cut into tiles of TK cached rows of one (slot, KV head) column, in
// slot order, and into `ranges` runs of equal cost, one per CTA: every SM gets
// the same share whatever the lengths are.  Starting a column costs about as
// much as tree_lead tiles, which stand before it in the count and hold no work
// (without them CTAs with three short columns ended last: 74 -> 61 us at 32
// slots of 300 to 3000 rows, the one case that three was chosen by; in the narrow form, where several CTAs share an
// SM, one or two places took 49.5 us against 47.5 at 256 slots).  A column that ends up in several ranges leaves
// (max, sum, out) pieces which tree_merge joins.
template <int TK>
__host__ __device__ constexpr int tree_lead() { return TK == 128 ? 3 : 0; }

template <int TK>
struct TreeWalk {
    static constexpr int LEAD = tree_lead<TK>();
    int slot, rem, left, g, g0;       // next place: slot, index within the slot's; places left; global index, first
    int L, t0, n, T, at;              // the slot whose numbers are loaded
    // the segment: tiles a .. b - 1 of column (slot, kvh), which starts at place s_c; the segment's own at s_g
    int s_slot, s_kvh, s_a, s_b, s_g, s_c;

    __device__ __forceinline__ static int tiles(int L, int n, int cap) { return n > 0 ? (min(L + n, cap) + TK - 1) / TK : 0; }
    __device__ __forceinline__ static int places(int L, int n, int cap) {
        const int t = tiles(L, n, cap);
        return t > 0 ? t + LEAD : 0;
    }
    // Whole columns instead (a.whole): range r takes columns r, r + ranges, ..., g being the next one.
    __device__ __forceinline__ bool next_whole(const TreeArgs &a) {
        while (g < a.v.slots * a.v.kvh) {
            s_slot = g / a.v.kvh;
            s_kvh = g - s_slot * a.v.kvh;
            g += a.ranges;
            tree_span(a.v, a.len, a.off, a.max_nodes, s_slot, L, t0, n);
            T = tiles(L, n, a.v.page_max * kPageRows);
            s_a = 0;
            s_b = T;
            if (T > 0) return true;
        }
        return false;
    }
    __device__ __forceinline__ bool next(const TreeArgs &a, int first_node) {
        while (left > 0) {
            if (slot >= a.v.slots) return false;
            if (at != slot) {
                tree_span(a.v, a.len, a.off, a.max_nodes, slot, L, t0, n);
                T = tiles(L, n, a.v.page_max * kPageRows);
                at = slot;
            }
            const int V = T + LEAD;
            if (T == 0 || rem >= V * a.v.kvh) {
                slot++;
                rem = 0;
                continue;
            }
            const int kvh = rem / V, x = rem - kvh * V, c = min(V - x, left);
            s_slot = slot;
            s_kvh = kvh;
            s_a = max(0, x - LEAD);
            s_b = max(0, x + c - LEAD);
            s_g = g;
            s_c = g - x;
            left -= c;
            rem += c;
            g += c;
            if (first_node < n && s_b > s_a) return true;
        }
        return false;
    }
};

// The walks' starts for NR ranges from `range` on.  Every thread takes a run of
// slots; s_scan holds blockDim.x / 32 ints of scratch, s_start 4 for each range.
template <int TK, int NR>
__device__ __forceinline__ void tree_plan(const TreeArgs &a, int range, int *s_scan, int *s_start) {
    const int th = threadIdx.x, nth = blockDim.x, lane = th & 31, w = th >> 5, cap = a.v.page_max * kPageRows;
    const int per = (a.v.slots + nth - 1) / nth, b0 = min(a.v.slots, th * per), b1 = min(a.v.slots, b0 + per);
    int sum = 0;
    for (int s = b0; s < b1; s++) {
        int L, t0, n;
        tree_span(a.v, a.len, a.off, a.max_nodes, s, L, t0, n);
        sum += TreeWalk<TK>::places(L, n, cap) * a.v.kvh;
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
    const int C = max((total + a.ranges - 1) / a.ranges, 1);
    if (th < NR) {
        const long long g0 = (long long)(range + th) * C;
        s_start[4 * th + 2] = (int)max(0LL, min((long long)C, total - g0));  // places of this range
        s_start[4 * th + 3] = C;
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const long long g0 = (long long)(range + i) * C;
        if (g0 < before || g0 >= before + sum) continue;
        int at = before;
        for (int s = b0; s < b1; s++) {
            int L, t0, n;
            tree_span(a.v, a.len, a.off, a.max_nodes, s, L, t0, n);
            const int c = TreeWalk<TK>::places(L, n, cap) * a.v.kvh;
            if (g0 < at + c) {
                s_start[4 * i] = s;
                s_start[4 * i + 1] = (int)g0 - at;
                break;
            }
            at += c;
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
    w.g = w.g0 = w.left > 0 ? range * s_start[3] : 0;
    w.at = -1;
    return w;
}

// A node's parent as the walk below takes it: -2 padding, -1 none.
__device__ __forceinline__ int tree_parent(const TreeArgs &a, int t0, int n, int i) {
    const int p = i < n ? __ldg(a.parent + t0 + i) : -2;
    return p == -2 ? -2 : p < 0 || p >= i ? -1 : p;
}
// One segment of a walk, as the softmax warps share it.
struct TreeSeg {
    int have, slot, kvh, a, b, c, piece, L, t0, n, T;
};
// Bits of the nodes that node i sees: itself and its ancestors up to the root
// or to a padding node.  Parents lie below their nodes, so the walk ends.
__device__ __forceinline__ unsigned long long tree_mask(const int8_t *s_up, int i) {
    unsigned long long m = 0;
    for (int p = i; p >= 0 && s_up[p] != -2; p = s_up[p]) m |= 1ull << p;
    return m;
}

// The factor 2^x of a part that holds something: never 0, so that an infinite
// V keeps its sign where its probability is too small for fp32.
__device__ __forceinline__ float ex2_part(float x) {
    const float f = ex2(x);
    return f < FLT_MIN ? FLT_MIN : f;
}

// The factor of a part whose maximum is x in a join whose maximum is M (both may be +inf).
__device__ __forceinline__ float join_part(float x, float M) {
    const float f = ex2_part(x - M);
    return x == M ? 1.f : f;
}

// Query rows (of the narrow form) to be done again: those with odd outputs, and
// those whose nodes see a drafted row that was left out of the product.
__device__ __noinline__ unsigned tree_again(const int8_t *s_up, int rows, int lg, unsigned odd, unsigned long long bad) {
    unsigned again = 0;
    for (int row = 0; row < rows; row++) {
        const unsigned long long see = tree_mask(s_up, row >> lg);
        if (see && (((odd >> row) & 1) || (see & bad))) again |= 1u << row;
    }
    return again;
}

// One (node, head) row over the rows r0 .. r1 - 1 that its node sees (mask: of
// the drafted ones), by a whole warp in plain fp32 arithmetic, in place of a
// row whose sum or output is not finite or which sees a V that is not.  The
// products split fp32 numbers into bf16 terms, and infinity times a term that
// is 0 or of the other sign is NaN where infinity times the number is not.
// Scores of -inf drop their rows; with one of +inf or NaN the output is NaN.
// The result goes to the output (ml null) or to a piece, dim d of which stands
// at po[d / 8 * step + d % 8].
template <typename T, int HD>
__device__ __noinline__ void tree_redo(const TreeArgs &a, int slot, int kvh, int L, unsigned long long mask, int r0, int r1, int tok,
                                       int head, float sl2, float2 *ml, float *po, int step) {
    constexpr int D = HD / 32, B = 8;  // dims of a lane; rows at a time, all of one page
    const int lane = threadIdx.x & 31, d0 = lane * D;
    float q[D], o[D], m = -INFINITY, l = 0.f;
    bool nan = false;
#pragma unroll
    for (int d = 0; d < D; d++) {
        q[d] = (float)((const T *)a.q)[(long long)tok * a.q_ld + (long long)head * HD + d0 + d];
        if (a.scale < 0.f) q[d] = -q[d];
        o[d] = 0.f;
    }
    const uint16_t *base = a.v.kv + a.layer * a.v.layer_stride + kvh * HD + d0;
    for (int r = r0; r < r1; r += B) {  // r0 is a multiple of a tile
        const int pg = a.v.page(slot, r);
        const uint16_t *row = base + a.v.row(0, max(pg, 0), r);
        uint32_t k[B][D / 2], v[B][D / 2];  // pairs of dims
#pragma unroll
        for (int i = 0; i < B; i++)
#pragma unroll
            for (int d = 0; d < D / 2; d++) {
                const bool on = pg >= 0 && r + i < r1;
                k[i][d] = on ? *(const uint32_t *)(row + i * a.v.kvd + 2 * d) : 0u;
                v[i][d] = on ? *(const uint32_t *)(row + (kPageRows + i) * a.v.kvd + 2 * d) : 0u;
            }
        float x[B], mn = m;
#pragma unroll
        for (int i = 0; i < B; i++) {
            x[i] = 0.f;
#pragma unroll
            for (int d = 0; d < D; d++) x[i] = fmaf(q[d], __uint_as_float(d & 1 ? k[i][d / 2] & 0xffff0000u : k[i][d / 2] << 16), x[i]);
        }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1)
#pragma unroll
            for (int i = 0; i < B; i++) x[i] += __shfl_xor_sync(0xffffffffu, x[i], w);
#pragma unroll
        for (int i = 0; i < B; i++) {
            const bool see = r + i < r1 && (r + i < L || ((mask >> (r + i - L)) & 1));
            x[i] = see ? x[i] * sl2 : -INFINITY;
            nan |= x[i] != x[i];
            mn = fmaxf(mn, x[i]);
        }
        const float f = m == mn ? 1.f : m == -INFINITY ? 0.f : ex2_part(m - mn);
        m = mn;
        l *= f;
#pragma unroll
        for (int d = 0; d < D; d++) o[d] *= f;
#pragma unroll
        for (int i = 0; i < B; i++) {
            if (x[i] == -INFINITY) continue;
            const float p = ex2_part(x[i] - m);
            l += p;
#pragma unroll
            for (int d = 0; d < D; d++) o[d] = fmaf(p, __uint_as_float(d & 1 ? v[i][d / 2] & 0xffff0000u : v[i][d / 2] << 16), o[d]);
        }
    }
    if (m == INFINITY && !nan) l = 1.f;  // lse = +inf
    if (ml) {
        if (lane == 0) *ml = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < D; d++) po[(d0 + d) / 8 * step + (d0 + d) % 8] = o[d];
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + d0;
#pragma unroll
    for (int d = 0; d < D; d++) dst[d] = (T)(o[d] * inv);
    if (a.lse && lane == 0) a.lse[(long long)tok * a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
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
// as large as the output's own rounding.  The tensor cores cut, not round,
// what they add to an fp32 accumulator: over n products the sum falls short by
// about n 2^-26 of itself (1.8e-5 over 125 tiles).  So O leaves tensor memory
// for registers after every tile (fp32 outputs; every 32nd for bf16 ones),
// where sums round, and the small terms of a tile go first, while its sum is
// small (for 3 % of the time).  The maximum that P is taken against moves only
// when it would grow by over 2^8, which rescales O; sums and outputs stay exact
// under it, as the same one divides out at the end.
//
// On a B200, in calls one after the other: 30 nodes over 32 slots of 300 to
// 3000 rows, fp32 (120 rows a tile, 127 MB, 38 GFLOP in three terms) 64 us: the
// products take 1.9 us a tile at the tensor cores' full rate, 22 us in all, the
// rest is the start, two or three changes of column a CTA (about 6 us each) and
// the join.  64 nodes over 12 slots of 11500 to 16500 rows, bf16: 174 us, of
// which this kernel is 152 by itself: 71 tiles a CTA, 2.1 us each, where the
// products of a tile take 1.1.  A tile's softmax overlaps only the next Q . K^T,
// so the tensor cores wait for it; each K and V tile is read by two CTAs at one
// time (rows 0-127 and 128-255 of the tree), once from memory.
//
// Infinities and NaN: rows whose sum or output is not finite are done again by
// tree_redo.  The look for them is one pass over a segment's outputs (no
// difference in any of these times).
constexpr int kTtK = 128;       // cached rows of a tile
constexpr int kTtThreads = 384, kTtSoft = 256;
// Registers of a softmax thread and of the others: 256 * 216 + 128 * 72 = 384 * 168, what the block is launched with.
constexpr int kTtRegsSoft = 216, kTtRegsFeed = 72;
// Tiles that O adds up in tensor memory before it goes to registers.
template <typename T>
__host__ __device__ constexpr int tt_flush() { return sizeof(T) == 4 ? 1 : 32; }

template <typename T>
__host__ __device__ constexpr int tt_qterms() { return sizeof(T) == 4 ? 3 : 1; }
template <typename T>
__host__ __device__ constexpr int tt_pterms() { return sizeof(T) == 4 ? 3 : 2; }
template <int HD>
__host__ __device__ constexpr int tt_stage() { return (HD / 64) * 128 * 128; }
// Shared memory: the Q terms of 64 or 128 rows (a product reads 128 rows from
// there on, whatever lies behind, and the rows past the last are not used),
// then K / V stages.  Beside it the kernel has at most 2 KB of static shared memory.
constexpr int kTtSmem = 224 * 1024, kTtMaxSt = 8;
template <typename T, int HD>
__host__ __device__ constexpr int tt_qbytes(int qrows) { return tt_qterms<T>() * (HD / 64) * qrows * 128; }
template <typename T, int HD>
__host__ __device__ constexpr int tt_stages(int qrows) {
    const int s = (kTtSmem - ((tt_qbytes<T, HD>(qrows) + 1023) & ~1023)) / tt_stage<HD>();
    return s > kTtMaxSt ? kTtMaxSt : s;
}

// Tensor memory columns: S / P of tiles 2i and 2i + 1 (P's third term apart), O.
constexpr uint32_t kTtS = 0, kTtO = 256, kTtX = 384;

template <typename T, int HD, int QR>
__global__ void __launch_bounds__(kTtThreads, 1) tree_attn_tc(const __grid_constant__ TreeArgs a,
                                                              const __grid_constant__ CUtensorMap map) {
    constexpr int QT = tt_qterms<T>(), PT = tt_pterms<T>(), NH = HD / 64, STB = tt_stage<HD>();
    constexpr int NST = tt_stages<T, HD>(QR), QH = QR * 128, QTB = NH * QH;  // stages; bytes of a term's half, and of a term
    static_assert(NST >= 4, "K and V of two tiles in flight");
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[NST], empty[NST], sfull[2], pfull[2], odone[2], qfull, ofree, fin;
    __shared__ uint32_t s_tmem;
    __shared__ int s_scan[kTtThreads / 32], s_start[4];
    __shared__ int8_t s_up[kTreeMax];
    __shared__ unsigned long long s_bad[2][2];
    __shared__ float s_half[2][128];
    __shared__ int s_stop, s_fresh[2];  // s_fresh: P . V of this tile starts O anew
    __shared__ TreeSeg s_seg[2];
    __shared__ TreeWalk<kTtK> s_walk;  // the softmax warps' walk: in registers it would cost them spills
    uint8_t *sq = (uint8_t *)(((uintptr_t)dsm + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sq + ((QT * QTB + 1023) & ~1023);
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
    tree_plan<kTtK, 1>(a, range, s_scan, s_start);
    um_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    TreeWalk<kTtK> w = tree_walk<kTtK>(s_start, range);
    const int cap = a.v.page_max * kPageRows;
    const bool range_root = rb == 0 && threadIdx.x == 0;  // the thread that notes the range's split column
    if (range_root) a.roots[range] = make_int4(-1, 0, 0, 0);
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTtRegsFeed));
        if (warp == 8) {
            // eight pages a tile, K then V; a page that does not exist is read past
            // the end of the map, which fills zeros
            const int y0 = a.layer * a.v.npages * 2 * kPageRows, yend = a.v.layers * a.v.npages * 2 * kPageRows;
            int pos = 0;
            RingPos at;
            while (w.next(a, node0)) {
                const int pages = (min(w.L + w.n, cap) + kPageRows - 1) / kPageRows;
                // the segment's queries towards L2: the softmax warps load them when
                // the segment before has used its own
                for (int i = lane; i < (min(NB, w.n - node0) << a.lg) * (HD * (int)sizeof(T) / 128); i += 32) {
                    const int e = i * (128 / (int)sizeof(T)), r = e / HD;
                    const T *q = (const T *)a.q + (long long)(w.t0 + node0 + (r >> a.lg)) * a.q_ld +
                                 (long long)(w.s_kvh * a.G + (r & (a.G - 1))) * HD + e % HD;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
                }
                for (int t = w.s_a; t < w.s_b; t++) {
                    const int j = t * (kTtK / kPageRows) + (lane & 7);
                    const int pg = j < pages ? __ldg(a.v.pages + (size_t)w.s_slot * a.v.page_max + j) : -1;
                    const int y = pg < 0 || pg >= a.v.npages ? yend : y0 + pg * 2 * kPageRows;
                    for (int kv = 0; kv < 2; kv++, pos++, at.next(NST)) {
                        const int st = at.st;
                        mb_wait(&empty[st], at.use ^ 1, &s_stop);  // passes on a stage's first use
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
                RingPos at_k, at_v;   // K and V of the next tiles
                at_v.next(NST);
                // O += P(i) . V(i), or O = ...; the segment's first one also waits for the last segment's O to be read
                auto pv = [&](int i, bool first) {
                    const int st = at_v.st;
                    mb_wait(&pfull[i & 1], (i >> 1) & 1, &s_stop);
                    mb_wait(&full[st], at_v.use, &s_stop);
                    at_v.next(NST, 2);
                    if (first && seg > 0) mb_wait(&ofree, (seg - 1) & 1, &s_stop);
                    um_fence_after();
                    const bool fresh = s_fresh[i & 1];
                    const uint32_t vb = um_desc_lo(ring0 + st * STB, 16384), p0 = tmem + kTtS + (i & 1) * 128, px = tmem + kTtX + (i & 1) * 64;
                    if (elect()) {
#pragma unroll
                        for (int x = PT - 1; x >= 0; x--)  // small terms first
#pragma unroll
                            for (int k = 0; k < kTtK / 16; k++)
                                um_mma_ts(tmem + kTtO, (x == 2 ? px : p0 + x * 64) + k * 8, vb + k * (2048 / 16), ipv,
                                          x == PT - 1 && k == 0 ? !fresh : true);
                        um_commit(&empty[st]);
                        um_commit(&odone[i & 1]);
                    }
                    __syncwarp();
                };
                while (w.next(a, node0)) {
                    for (int t = w.s_a; t < w.s_b; t++, it++) {
                        const int st = at_k.st;
                        if (t == w.s_a) mb_wait(&qfull, seg & 1, &s_stop);
                        mb_wait(&full[st], at_k.use, &s_stop);
                        at_k.next(NST, 2);
                        um_fence_after();
                        const uint32_t kb = um_desc_lo(ring0 + st * STB, 16), s0 = tmem + kTtS + (it & 1) * 128;
                        if (elect()) {
#pragma unroll
                            for (int x = QT - 1; x >= 0; x--)
#pragma unroll
                                for (int k = 0; k < HD / 16; k++) {
                                    um_mma(s0, q0 + (x * QTB + (k >> 2) * QH + (k & 3) * 32) / 16, kb + ((k >> 2) * 16384 + (k & 3) * 32) / 16, iqk,
                                           !(x == QT - 1 && k == 0));
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
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTtRegsSoft));
        const int th = threadIdx.x & 127, h = warp >> 2;  // row, and half of its keys and dims
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float sl2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
        int it = 0, seg = 0;
        int up = -1;
        // the segment's Q into shared memory, a warp to a row, eight or sixteen in flight,
        // and its nodes' parents on their way
        auto load_q = [&](const TreeSeg &x) {
            const int rows = min(NB, x.n - node0) << a.lg;
            if (threadIdx.x < kTreeMax) up = tree_parent(a, x.t0, x.n, threadIdx.x);
            const int half = HD == 128 ? lane >> 4 : 0, c = (lane & 15) * 4;  // dims half * 64 + c ..
            const bool on = HD == 128 || lane < 16;
            const T *src = (const T *)a.q + (long long)(x.t0 + node0) * a.q_ld + (long long)x.kvh * a.G * HD + half * 64 + c;
            // (fp32: all sixteen of a warp's rows at once took 77 us against 73 at 32 x 30 nodes)
            constexpr int B = sizeof(T) == 4 ? 8 : 16;
            for (int r0 = warp; r0 < rows; r0 += 8 * B) {
                float4 q[B];
#pragma unroll
                for (int i = 0; i < B; i++) {
                    const int r = r0 + 8 * i;
                    q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (on && r < rows) q[i] = ld_row4(src + (long long)(r >> a.lg) * a.q_ld + (r & (a.G - 1)) * HD);
                }
#pragma unroll
                for (int i = 0; i < B; i++) {
                    const int r = r0 + 8 * i;
                    if (!on || r >= rows) continue;
                    if (a.scale < 0.f) q[i] = make_float4(-q[i].x, -q[i].y, -q[i].z, -q[i].w);
                    uint32_t lo[QT], hi[QT];
                    split_bf16<QT>(q[i].x, q[i].y, lo);
                    split_bf16<QT>(q[i].z, q[i].w, hi);
                    uint8_t *dst = sq + half * QH + r * 128 + ((((c >> 3) ^ (r & 7)) << 4) | ((c & 4) << 1));
#pragma unroll
                    for (int k = 0; k < QT; k++) *(uint2 *)(dst + k * QTB) = make_uint2(lo[k], hi[k]);
                }
            }
            fence_async_smem();
            mb_arrive(&qfull);
        };
        // one thread takes the walk a segment ahead
        auto advance = [&](TreeSeg &x) {
            TreeWalk<kTtK> v = s_walk;
            x.have = v.next(a, node0);
            x.slot = v.s_slot;
            x.kvh = v.s_kvh;
            x.a = v.s_a;
            x.b = v.s_b;
            x.c = v.s_c;
            x.piece = v.s_g != v.g0;
            x.L = v.L;
            x.t0 = v.t0;
            x.n = v.n;
            x.T = v.T;
            s_walk = v;
        };
        if (threadIdx.x == 0) {
            s_walk = w;
            advance(s_seg[0]);
        }
        bar_sync(1, kTtSoft);
        if (s_seg[0].have) load_q(s_seg[0]);
        while (s_seg[seg & 1].have) {
            const TreeSeg &cur = s_seg[seg & 1];
            if (threadIdx.x < kTreeMax) s_up[threadIdx.x] = (int8_t)up;
            bar_sync(1, kTtSoft);
            if (threadIdx.x == 0) advance(s_seg[(seg + 1) & 1]);
            const int L = cur.L, t1 = cur.b, rows = min(NB, cur.n - node0) << a.lg, end = min(L + cur.n, cap);
            const bool active = (warp & 3) * 32 < rows;
            const int node = node0 + (th >> a.lg);
            unsigned long long mask = th < rows ? tree_mask(s_up, node) : 0;
            const bool live = mask != 0;  // not a padding node
            if (end - L < 64) mask &= (1ull << max(0, end - L)) - 1;
            constexpr int W = HD / 2;
            float m = -INFINITY, l = 0.f, o[W];
#pragma unroll
            for (int d = 0; d < W; d++) o[d] = 0.f;
            // O of the tiles so far, once their last product is done, into o
            auto flush = [&]() {
                mb_wait(&odone[(it - 1) & 1], ((it - 1) >> 1) & 1, &s_stop);
                um_fence_after();
                if (active) {
#pragma unroll
                    for (int c = 0; c < W / 32; c++) {
                        float x[32];
                        um_ld32(tmem + lanes + kTtO + h * W + c * 32, x);
                        um_wait_ld<32>(x);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[c * 32 + i] += x[i];
                    }
                }
            };
            int since = 0;  // tiles in O that o does not have
            bool first = true;
            for (int t = cur.a; t < t1; t++, it++, first = false) {
                const int b = it & 1, r0 = t * kTtK;
                const bool tail = r0 + kTtK > L;
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
                        const int c = L - r0 - h * 64;  // cached rows among them
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
                        m = mn;
                        l *= f;
                        flush();
                        since = 0;
#pragma unroll
                        for (int d = 0; d < W; d++) o[d] *= f;
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
                if (since == tt_flush<T>()) {
                    flush();
                    since = 0;
                }
                if (threadIdx.x == 0) s_fresh[b] = since == 0;
                since++;
                if (tail) {
                    // V rows that no node sees become zeros (a product with a
                    // probability of 0 must be 0), and so do halves of drafted
                    // rows that are not finite: the nodes that see them are
                    // done again at the end
                    const int pos = 2 * it + 1, st = pos % NST, r = r0 + th;
                    mb_wait(&full[st], (pos / NST) & 1, &s_stop);
                    if (r >= L) {
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
                        if (bad) atomicOr(&s_bad[seg & 1][h], 1ull << (r - L));
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
            if (s_seg[(seg + 1) & 1].have) load_q(s_seg[(seg + 1) & 1]);
            flush();
            um_fence_before();
            mb_arrive(&ofree);
            float odd = 0.f;  // not 0: an output is not finite
#pragma unroll
            for (int d = 0; d < W; d++) odd = fmaf(o[d], 0.f, odd);
            if (odd != 0.f) l = NAN;
            // the halves' sums, each in the word that this thread itself read the
            // other half's last maximum from (the word of its own maximum may
            // still be read by the other half, which no barrier has held since)
            s_half[h ^ 1][th] = l;
            bar_sync(1, kTtSoft);  // and s_bad is complete
            l = h ? s_half[1][th] + l : l + s_half[0][th];
            const unsigned long long bad = (s_bad[seg & 1][0] | s_bad[seg & 1][1]) & mask;
            if (th == 0) s_bad[(seg + 1) & 1][h] = 0;
            const bool whole = cur.a == 0 && t1 == cur.T;
            if (active) {
                const int piece = (2 * range + cur.piece) * a.row_blocks + rb;
                const bool redo = th < rows && live && (l != l || bad);
                // a node that saw nothing: its products with the cached rows are
                // zeros only where those rows are finite
                if (l == 0.f || !live)
#pragma unroll
                    for (int d = 0; d < W; d++) o[d] = 0.f;
                if (!live) l = 0.f;
                if (th < rows && !redo) {
                    const int tok = cur.t0 + node, head = cur.kvh * a.G + (th & (a.G - 1));
                    if (whole) {
                        const float inv = l == 0.f ? 0.f : 1.0f / l;
                        T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + h * W;
#pragma unroll
                        for (int d = 0; d < W; d += 8) st_row8(dst + d, o + d, inv, a.out32);
                        if (a.lse && h == 0)
                            a.lse[(long long)tok * a.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
                    } else {
                        if (h == 0) a.part_ml[(size_t)piece * 128 + th] = make_float2(m, l);
                        float *po = a.part_o + (size_t)piece * 128 * HD + h * W * 128 + th * 8;
#pragma unroll
                        for (int d = 0; d < W; d += 8) st_row8(po + d * 128, o + d, 1.f, true);
                    }
                }
                // rare: the two halves' warps, which agree on the rows, take every other one
                for (unsigned who = __ballot_sync(0xffffffffu, redo) & (h ? 0xaaaaaaaau : 0x55555555u); who; who &= who - 1) {
                    const int row = (warp & 3) * 32 + __ffs(who) - 1, nd = node0 + (row >> a.lg);
                    tree_redo<T, HD>(a, cur.slot, cur.kvh, L, tree_mask(s_up, nd), cur.a * kTtK, min(t1 * kTtK, end), cur.t0 + nd,
                                     cur.kvh * a.G + (row & (a.G - 1)), sl2, whole ? nullptr : a.part_ml + (size_t)piece * 128 + row,
                                     a.part_o + (size_t)piece * 128 * HD + row * 8, 1024);
                }
            }
            if (range_root && cur.a == 0 && !whole) a.roots[range] = make_int4(cur.slot, cur.kvh, cur.c, s_start[3]);
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

// ---------------------------------------------------------------- narrow trees: mma.sync
//
// Up to 32 (node, head) rows, as single tokens and small drafts have, where a
// 128-row tensor-memory tile would run nearly empty and its set-up would not
// pay: small CTAs, several to an SM, that hide one another's waits.  Tiles of
// 64 cached rows; S^T = K Q^T and O^T = V^T P^T with the cached rows (and
// dims) as the 16-row operand and the query rows as the 8-column one, so NT
// tiles of 8 columns waste little on 4 or 20 rows.  Warp w takes the 16 keys
// of the tile's page w, then hd / 4 dims of O^T over all keys: the output needs
// no join between warps, and P^T crosses between them as operand fragments (by
// 8x8 transposes in registers, then shared memory).  K's next tile is copied
// while this one's V is multiplied, and V's while the next scores are made: one
// buffer each, and three CTAs an SM (two buffers and two CTAs: 45 -> 56 us at
// 256 slots of about 120 rows and 5 nodes).  The terms of fp32 queries and
// probabilities and the lagging maximum are those of the wide form.
//
// 256 slots of 70 to 176 rows x 5 nodes, fp32 (81 MB): 47 us, bound by
// instruction issue and its latencies (38 % of the slots with three CTAs an SM;
// a tile takes a CTA 3.5 us, 2.2 of them in the products); one node over 55
// rows: 8 us of kernel time.
constexpr int kTnWarps = 4, kTnThreads = kTnWarps * 32, kTnK = 64;

template <typename T, int HD, int NT>
__host__ __device__ constexpr int tn_qbytes() { return tt_qterms<T>() * (HD / 16) * NT * 256; }
template <typename T, int HD, int NT>
__host__ __device__ constexpr size_t tn_smem() {
    return (size_t)2 * kTnK * HD * 2 + tn_qbytes<T, HD, NT>() + (size_t)tt_pterms<T>() * 4 * NT * 256;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(p)
                 : "memory");
}
__device__ __forceinline__ uint32_t mat_t(uint32_t x) {  // 8x8 transpose of bf16 pairs across the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kTnThreads, 3) tree_attn_mma(const __grid_constant__ TreeArgs a) {
    constexpr int QT = tt_qterms<T>(), PT = tt_pterms<T>(), CH = HD / 8, KS = HD / 16, MT = HD / 64, ROW = HD * 2;
    constexpr int RPI = kTnThreads / CH, NI = kTnK / RPI;  // rows a copy step covers, steps a tile
    extern __shared__ __align__(128) uint8_t dsm[];
    __shared__ int s_scan[kTnWarps], s_start[4];
    __shared__ int8_t s_up[kTreeMax];
    __shared__ float s_mx[kTnWarps][NT * 8];
    __shared__ unsigned s_odd;  // rows with outputs that are not finite
    __shared__ unsigned long long s_bad, s_mask[NT * 8];  // s_mask: what a query row's node sees of its tree
    uint8_t *bk = dsm, *bv = dsm + kTnK * ROW;
    uint2 *qf = (uint2 *)(bv + kTnK * ROW);    // Q fragments [term][16 dims][8 rows][lane]
    uint2 *pf = qf + QT * KS * NT * 32;        // P fragments [term][page][8 rows][lane]
    const int th = threadIdx.x, warp = th >> 5, lane = th & 31, g = lane >> 2, tq = lane & 3, range = blockIdx.x;
    pdl_trigger();
    pdl_wait();
    TreeWalk<kTnK> wi;
    if (a.whole) {
        wi.g = range;
    } else {
        tree_plan<kTnK, 1>(a, range, s_scan, s_start);
        wi = tree_walk<kTnK>(s_start, range);
        if (th == 0) a.roots[range] = make_int4(-1, 0, 0, 0);
    }
    if (th == 0) {  // first used after the barriers of the first tile
        s_bad = 0;
        s_odd = 0;
    }
    const auto step = [&](TreeWalk<kTnK> &w) { return a.whole ? w.next_whole(a) : w.next(a, 0); };
    const int cap = a.v.page_max * kPageRows;
    const float sl2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);
    TreeWalk<kTnK> wc = wi;
    bool more = step(wi);
    int it = more ? wi.s_a : 0;  // the tile to copy next, of column wi
    const uint16_t *src[kTnK / kPageRows];  // its pages' K rows of this thread (first row and chunk), null: no page
    const int cc = th % CH, cr = th / CH;   // this thread's chunk of a row, and its first row of a copy step's
    auto pages = [&]() {
        const int p0 = it * (kTnK / kPageRows), n = (min(wi.L + wi.n, cap) + kPageRows - 1) / kPageRows;
        const uint16_t *base = a.v.kv + a.layer * a.v.layer_stride + (long long)cr * a.v.kvd + wi.s_kvh * HD + cc * 8;
#pragma unroll
        for (int i = 0; i < kTnK / kPageRows; i++) {
            const int pg = more && p0 + i < n ? __ldg(a.v.pages + (size_t)wi.s_slot * a.v.page_max + p0 + i) : -1;
            src[i] = pg >= 0 && pg < a.v.npages ? base + (long long)pg * a.v.page_stride : nullptr;
        }
    };
    // K (kv = 0) or V rows of that tile; rows that do not exist become zeros
    auto copy = [&](int kv) {
        if (more) {
            const int end = min(wi.L + wi.n, cap) - it * kTnK, off = kv * kPageRows * a.v.kvd;
            const uint32_t dst = kv_smem(kv ? bv : bk) + cr * ROW + ((cc ^ (cr & 7)) << 4);
#pragma unroll
            for (int i = 0; i < NI; i++) {  // rows cr + i * RPI: RPI is 8 or 16, so the swizzle stays
                const uint16_t *pg = src[(i * RPI) / kPageRows];
                const bool ok = pg && cr + i * RPI < end;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * RPI * ROW),
                             "l"(ok ? pg + off + (i * RPI % kPageRows) * a.v.kvd : a.v.kv), "r"(ok ? 16 : 0)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pages();
    copy(0);
    copy(1);
    while (step(wc)) {
        const int rows = wc.n << a.lg, end = min(wc.L + wc.n, cap);
        // parents, and the queries as B fragments: lane (g, t) holds row g, dims 2t, 2t + 1, 2t + 8, 2t + 9 of 16
        if (th < kTreeMax) s_up[th] = (int8_t)tree_parent(a, wc.t0, wc.n, th);
        unsigned dead = 0;  // bit 2 nt + j: this lane's row is a padding node's
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + 2 * tq + j;
                if (row < rows && __ldg(a.parent + wc.t0 + (row >> a.lg)) == -2) dead |= 1u << (2 * nt + j);
            }
        {
            const T *q0 = (const T *)a.q + (long long)wc.t0 * a.q_ld + (long long)wc.s_kvh * a.G * HD + 2 * tq;
            const float sg = a.scale < 0.f ? -1.f : 1.f;
            constexpr int NF = KS * NT / kTnWarps;
            float2 x[NF][2];
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int k = (f * kTnWarps + warp) / NT, nt = (f * kTnWarps + warp) % NT, r = nt * 8 + g;
                const T *q = q0 + (long long)(r >> a.lg) * a.q_ld + (r & (a.G - 1)) * HD + k * 16;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    x[f][h] = make_float2(0.f, 0.f);
                    if (r < rows) {
                        if constexpr (sizeof(T) == 4) {
                            x[f][h] = *(const float2 *)(q + h * 8);
                        } else {
                            const uint32_t u = *(const uint32_t *)(q + h * 8);
                            x[f][h] = make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
                        }
                    }
                }
            }
#pragma unroll
            for (int f = 0; f < NF; f++) {
                uint32_t b0[QT], b1[QT];
                split_bf16<QT>(x[f][0].x * sg, x[f][0].y * sg, b0);
                split_bf16<QT>(x[f][1].x * sg, x[f][1].y * sg, b1);
#pragma unroll
                for (int i = 0; i < QT; i++) qf[(i * KS * NT + f * kTnWarps + warp) * 32 + lane] = make_uint2(b0[i], b1[i]);
            }
        }
        // O^T: o[mt][nt] = {(dim g, row 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)} of 16 dims x 8 rows
        float o[MT][NT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o[mt][nt][0] = o[mt][nt][1] = o[mt][nt][2] = o[mt][nt][3] = 0.f;
        }
        for (int t = wc.s_a; t < wc.s_b; t++) {
            const int r0 = t * kTnK;
            const bool tail = r0 + kTnK > wc.L;
            if (++it == wi.s_b) {  // the copies' next tile, and its pages on their way
                more = step(wi);
                it = wi.s_a;
            }
            pages();
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // K, Q and the parents are there
            if (tail && th < NT * 8) s_mask[th] = th < rows ? tree_mask(s_up, th >> a.lg) : 0;  // read past the next barrier
            // the small terms in a sum of their own: an accumulator is cut, not
            // rounded, with every product added, so it should take few
            float s[NT][4], s1[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
                s1[nt][0] = s1[nt][1] = s1[nt][2] = s1[nt][3] = 0.f;
            }
            if (r0 + warp * 16 < end) {
                const int kr = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
                const uint32_t sk = kv_smem(bk) + kr * ROW;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t ka[4];
                    ldm4(ka, sk + (((2 * k + (lane >> 4)) ^ (kr & 7)) << 4));
#pragma unroll
                    for (int i = QT - 1; i >= 0; i--)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint2 b = qf[((i * KS + k) * NT + nt) * 32 + lane];
                            mma_16816(i ? s1[nt] : s[nt], ka, b.x, b.y);
                        }
                }
            }
            if (tail) __syncthreads();  // s_mask
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    unsigned see = (dead >> (2 * nt + j)) & 1 ? 0u : 0xffffu;  // of the page's 16 rows
                    if (tail) {
                        const unsigned long long mk = s_mask[nt * 8 + 2 * tq + j];
                        const int c = wc.L - r0 - warp * 16;  // cached rows among them
                        const unsigned own = c >= 16 ? 0xffffu : c > 0 ? ((1u << c) - 1) | (unsigned)(mk << c) : -c < 64 ? (unsigned)(mk >> -c) : 0u;
                        see &= own & (end - r0 - warp * 16 >= 16 ? 0xffffu : end - r0 - warp * 16 > 0 ? (1u << (end - r0 - warp * 16)) - 1 : 0u);
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float x = (s[nt][2 * h + j] + s1[nt][2 * h + j]) * sl2;
                        if (!((see >> (g + h * 8)) & 1)) x = -INFINITY;
                        s[nt][2 * h + j] = x;
                        grow |= x > m[nt][j] + 8.f;
                    }
                }
            if (bar_or(1, kTnThreads, grow)) {  // K has been read by all; does any maximum move?
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float x = fmaxf(s[nt][j], s[nt][2 + j]);
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                        if (g == 0) s_mx[warp][nt * 8 + 2 * tq + j] = x;
                    }
                __syncthreads();
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int row = nt * 8 + 2 * tq + j;
                        const float x = fmaxf(fmaxf(s_mx[0][row], s_mx[1][row]), fmaxf(s_mx[2][row], s_mx[3][row]));
                        const float mn = x > m[nt][j] + 8.f ? x : m[nt][j], f = m[nt][j] == -INFINITY ? 1.f : ex2(m[nt][j] - mn);
                        m[nt][j] = mn;
                        l[nt][j] *= f;
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            o[mt][nt][j] *= f;
                            o[mt][nt][2 + j] *= f;
                        }
                    }
            }
            copy(0);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] = ex2(s[nt][j] - (m[nt][j & 1] == -INFINITY ? 0.f : m[nt][j & 1]));
                l[nt][0] += p[0] + p[2];
                l[nt][1] += p[1] + p[3];
                uint32_t x[PT], y[PT];
                split_bf16<PT>(p[0], p[1], x);
                split_bf16<PT>(p[2], p[3], y);
#pragma unroll
                for (int i = 0; i < PT; i++) pf[((i * 4 + warp) * NT + nt) * 32 + lane] = make_uint2(mat_t(x[i]), mat_t(y[i]));
            }
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncthreads();  // P and V are there
            if (tail) {
                // drafted rows whose V is not finite become zeros; the nodes
                // that see them are done again at the end
                for (int r = max(wc.L - r0, 0) + warp; r < min(end - r0, kTnK); r += kTnWarps) {
                    bool x = false;
                    uint4 *p = (uint4 *)(bv + r * ROW + (lane % CH) * 16);
                    if (lane < CH) {
                        const uint4 u = *p;
                        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                        for (int k = 0; k < 4; k++) x |= (w[k] & 0x7f80u) == 0x7f80u || (w[k] & 0x7f800000u) == 0x7f800000u;
                    }
                    if (__any_sync(0xffffffffu, x)) {
                        if (lane < CH) *p = make_uint4(0, 0, 0, 0);
                        if (lane == 0) atomicOr(&s_bad, 1ull << (r0 + r - wc.L));
                    }
                }
                __syncthreads();
            }
            const int vr = (lane & 7) + (lane >> 4) * 8;
            const uint32_t sv = kv_smem(bv) + vr * ROW;
            // the tile's sum by itself, small terms first, then added to O: sums
            // in registers round, the products' accumulators cut
            float u[MT][NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++) u[mt][nt][0] = u[mt][nt][1] = u[mt][nt][2] = u[mt][nt][3] = 0.f;
#pragma unroll
            for (int i = PT - 1; i >= 0; i--)
#pragma unroll
                for (int ks = 0; ks < kTnK / 16; ks++) {
                    if (r0 + ks * 16 >= end) break;
                    uint32_t va[MT][4];
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
                        ldm4t(va[mt], sv + ks * 16 * ROW + (((2 * (warp * MT + mt) + ((lane >> 3) & 1)) ^ (vr & 7)) << 4));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const uint2 b = pf[((i * 4 + ks) * NT + nt) * 32 + lane];
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) mma_16816(u[mt][nt], va[mt], b.x, b.y);
                    }
                }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[mt][nt][j] += u[mt][nt][j];
            __syncthreads();  // P and V have been read
            copy(1);
        }
        // the rows' sums: a warp's lanes, then the four warps; and which outputs
        // are not finite (with a sum that is not, all are not)
        unsigned odd = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], w);
                if (g == 0) s_mx[warp][nt * 8 + 2 * tq + j] = l[nt][j];
                float x = 0.f;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) x = fmaf(o[mt][nt][j], 0.f, fmaf(o[mt][nt][2 + j], 0.f, x));
                odd |= (x != 0.f ? 1u : 0u) << (nt * 8 + j);
            }
        if (odd) atomicOr(&s_odd, odd << (2 * tq));
        __syncthreads();
        unsigned again = 0;  // rare
        if (s_odd || s_bad) again = tree_again(s_up, rows, a.lg, s_odd, s_bad);
        const bool whole = wc.s_a == 0 && wc.s_b == wc.T;
        const size_t piece = (size_t)2 * range + (wc.s_g != wc.g0);
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + 2 * tq + j;
                if (row >= rows || ((again >> row) & 1)) continue;
                const int tok = wc.t0 + (row >> a.lg), head = wc.s_kvh * a.G + (row & (a.G - 1));
                const float L = (s_mx[0][row] + s_mx[1][row]) + (s_mx[2][row] + s_mx[3][row]);
                if (L == 0.f)  // a node that saw nothing: 0 times a cached row is not 0 where that is not finite
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) o[mt][nt][j] = o[mt][nt][2 + j] = 0.f;
                if (whole) {
                    const float inv = L == 0.f ? 0.f : 1.0f / L;
                    T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + warp * MT * 16 + g;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        dst[mt * 16] = (T)(o[mt][nt][j] * inv);
                        dst[mt * 16 + 8] = (T)(o[mt][nt][2 + j] * inv);
                    }
                    if (a.lse && g == 0 && warp == 0)
                        a.lse[(long long)tok * a.heads + head] = L == 0.f ? -INFINITY : (m[nt][j] + log2f(L)) * 0.6931471805599453f;
                } else {
                    float *dst = a.part_o + (piece * (NT * 8) + row) * HD + warp * MT * 16 + g;
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        dst[mt * 16] = o[mt][nt][j];
                        dst[mt * 16 + 8] = o[mt][nt][2 + j];
                    }
                    if (g == 0 && warp == 0) a.part_ml[piece * (NT * 8) + row] = make_float2(m[nt][j], L);
                }
            }
        for (int row = warp; again >> row; row += kTnWarps) {
            if (!((again >> row) & 1)) continue;
            const size_t at = piece * (NT * 8) + row;
            tree_redo<T, HD>(a, wc.s_slot, wc.s_kvh, wc.L, tree_mask(s_up, row >> a.lg), wc.s_a * kTnK, min(wc.s_b * kTnK, end),
                             wc.t0 + (row >> a.lg), wc.s_kvh * a.G + (row & (a.G - 1)), sl2, whole ? nullptr : a.part_ml + at,
                             a.part_o + at * HD, 8);
        }
        if (th == 0 && wc.s_a == 0 && !whole) a.roots[range] = make_int4(wc.s_slot, wc.s_kvh, wc.s_c, s_start[3]);
        __syncthreads();
        if (th == 0) {
            s_bad = 0;
            s_odd = 0;
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------- joining the pieces
//
// For the columns that start in one range and go on in the next: M = max m_i,
// out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i over the pieces.  A work list
// over all such columns' (node, head) rows; 1, 2, 4 or 8 warps take a row, as
// many as keep the grid busy (few rows have many pieces), every so many-th
// piece each, hd / 32 dims a lane, joined in a fixed order.  Pieces of the
// narrow form are `rows_per` rows of HD values; those of the wide one (rows_per
// = 0) [8 dims][128 rows][8].
constexpr int kMergeThreads = 256;
template <typename T, int HD, int TK>
__global__ void __launch_bounds__(kMergeThreads) tree_merge(const __grid_constant__ TreeArgs a, int rows_per) {
    constexpr int D = HD / 32, W = kMergeThreads / 32;
    __shared__ int s_scan[W];
    __shared__ float s_part[W][HD], s_m[W], s_l[W];
    __shared__ int4 s_col[W], s_at[W];  // a row's {slot, KV head, first place, places per range}, {row, first token, tiles, -}
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // rows of the columns that start in this thread's ranges (one column a range at most)
    int sum = 0, total = 0;
    const int per = (a.ranges + kMergeThreads - 1) / kMergeThreads, b0 = min(a.ranges, (int)threadIdx.x * per), b1 = min(a.ranges, b0 + per);
    const auto count = [&](const int4 &root, int &t0, int &tiles) {
        if (root.x < 0) return 0;
        int L, n;
        tree_span(a.v, a.len, a.off, a.max_nodes, root.x, L, t0, n);
        tiles = TreeWalk<TK>::tiles(L, n, a.v.page_max * kPageRows);
        return n * a.G;
    };
    for (int i = b0; i < b1; i++) {
        int t0, tiles;
        sum += count(a.roots[i], t0, tiles);
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int i = 0; i < W; i++) {
        if (i < warp) before += s_scan[i];
        total += s_scan[i];
    }
    int wpr = W;  // warps of a row
    while (wpr > 1 && total * wpr > (int)gridDim.x * W) wpr >>= 1;
    const int RPC = W / wpr, mine = warp / wpr, part = warp % wpr;
    for (int row0 = blockIdx.x * RPC; row0 < total; row0 += gridDim.x * RPC) {
        // the CTA's next rows: whoever's ranges hold one says so
        if (before < row0 + RPC && before + sum > row0) {
            int at = before;
            for (int i = b0; i < b1; i++) {
                const int4 root = a.roots[i];
                int t0 = 0, tiles = 0;
                const int c = count(root, t0, tiles);
                for (int x = max(at, row0); x < min(at + c, row0 + RPC); x++) {
                    s_col[x - row0] = root;
                    s_at[x - row0] = make_int4(x - at, t0, tiles, 0);
                }
                at += c;
            }
        }
        __syncthreads();
        const bool on = row0 + mine < total;
        float M = -INFINITY, S = 0.f, o[D];
#pragma unroll
        for (int d = 0; d < D; d++) o[d] = 0.f;
        const int d0 = lane * D;
        if (on) {
            const int4 root = s_col[mine], me = s_at[mine];
            const int r = me.x, C = root.w, lead = tree_lead<TK>();
            const int p0 = (root.z + lead) / C + part, p1 = (root.z + lead + me.z - 1) / C;
            constexpr int B = 4;
            for (int q0 = p0; q0 <= p1; q0 += B * wpr) {  // four pieces in flight
                float v[B][D];
                float2 ml[B];
#pragma unroll
                for (int i = 0; i < B; i++) {
                    ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int d = 0; d < D; d++) v[i][d] = 0.f;
                    const int p = q0 + i * wpr;
                    if (p > p1) continue;
                    const size_t pc = ((size_t)2 * p + (p * C < root.z)) * a.row_blocks + (rows_per ? 0 : r >> 7);
                    ml[i] = a.part_ml[rows_per ? pc * rows_per + r : pc * 128 + (r & 127)];
                    const float *po = a.part_o + (rows_per ? (pc * rows_per + r) * HD + d0
                                                           : pc * 128 * HD + (d0 >> 3) * 1024 + (r & 127) * 8 + (d0 & 7));
                    if constexpr (D == 4) {
                        const float4 x = *(const float4 *)po;
                        v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
                    } else {
                        const float2 x = *(const float2 *)po;
                        v[i][0] = x.x, v[i][1] = x.y;
                    }
                }
                float mn = M;
#pragma unroll
                for (int i = 0; i < B; i++)
                    if (ml[i].y != 0.f) mn = fmaxf(mn, ml[i].x);
                const float old = M == -INFINITY ? 0.f : join_part(M, mn);
                M = mn;
                S *= old;
#pragma unroll
                for (int d = 0; d < D; d++) o[d] *= old;
#pragma unroll
                for (int i = 0; i < B; i++) {
                    const float e = join_part(ml[i].x, M), f = ml[i].y == 0.f ? 0.f : e;  // 0: nothing seen in this piece
                    S = fmaf(ml[i].y, f, S);
#pragma unroll
                    for (int d = 0; d < D; d++) o[d] = fmaf(v[i][d], f, o[d]);
                }
            }
        }
        if (wpr > 1) {
            if (lane == 0) {
                s_m[warp] = M;
                s_l[warp] = S;
            }
#pragma unroll
            for (int d = 0; d < D; d++) s_part[warp][d0 + d] = o[d];
            __syncthreads();
            if (part == 0) {
                for (int i = 1; i < wpr; i++) M = fmaxf(M, s_m[warp + i]);
                S = 0.f;
#pragma unroll
                for (int d = 0; d < D; d++) o[d] = 0.f;
                for (int i = 0; i < wpr; i++) {
                    const float l = s_l[warp + i], e = join_part(s_m[warp + i], M), f = l == 0.f ? 0.f : e;
                    S = fmaf(l, f, S);
#pragma unroll
                    for (int d = 0; d < D; d++) o[d] = fmaf(s_part[warp + i][d0 + d], f, o[d]);
                }
            }
        }
        if (on && part == 0) {
            const int4 root = s_col[mine], me = s_at[mine];
            const int r = me.x;
            const float inv = S == 0.f ? 0.f : 1.0f / S;
            const int tok = me.y + r / a.G, head = root.y * a.G + r % a.G;
            T *dst = (T *)a.out + (long long)tok * a.out_ld + (long long)head * HD + d0;
            if constexpr (D == 4) st_row4(dst, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            else if constexpr (sizeof(T) == 4) *(float2 *)dst = make_float2(o[0] * inv, o[1] * inv);
            else *(uint32_t *)dst = pack_bf16(o[0] * inv, o[1] * inv);
            if (a.lse && lane == 0) a.lse[(long long)tok * a.heads + head] = S == 0.f ? -INFINITY : (M + log2f(S)) * 0.6931471805599453f;
        }
        __syncthreads();
    }
}

}  // namespace
