// hy_kvops.cu — operators on a paged bf16 KV cache: attention of drafted token
// trees, acceptance of a drafted path, attention weights accumulated per
// cached row, and eviction by them (include/hymt2_cuda.h states each).
//
// No counterpart in the reference: it decodes one token per step
// (src/model.c:943-954) over a cache that only grows (:804-808).  The cache
// is the batch engine's, [layer][page][K | V][16][kvdim]; row r of a slot is
// row r % 16 of page pages[slot][r / 16].
#undef HYK_TRACE  // the measurement build's timelines belong to the decode kernels
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "../../include/hymt2_cuda.h"
#include "hy_kvtree.cuh"
#include "hy_kvview.cuh"
#include "hy_kvweights.cuh"

namespace {

int op_fail(char *err, int cap, int code, const char *msg) {
    if (err && cap > 0) snprintf(err, (size_t)cap, "%s", msg);
    return code;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The checked view; false with a message when the geometry is not served.
bool make_view(const hyc_kv_view *v, KvView &o, const char **why) {
    *why = nullptr;
    if (!v || !v->kv || !v->pages) *why = "null cache view";
    else if (v->layers < 1 || v->npages < 1 || v->kv_heads < 1 || v->slots < 1 || v->page_max < 1)
        *why = "empty cache view";
    else if (v->hdim != 64 && v->hdim != 128) *why = "hdim must be 64 or 128";
    else if (!aligned16(v->kv)) *why = "the cache must be 16-byte aligned";
    else if (v->page_max > (1 << 26) || v->kv_heads > 65535 || v->layers > 65535) *why = "cache view too large";
    else if ((long long)v->layers * v->npages * 2 * kPageRows > 0x7fffffffLL ||
             (double)v->layers * v->slots * v->kv_heads * (v->page_max / 4 + 4) > 2147483647.0)
        *why = "cache view too large";
    if (*why) return false;
    o.kv = v->kv;
    o.pages = v->pages;
    o.layers = v->layers;
    o.npages = v->npages;
    o.kvh = v->kv_heads;
    o.hd = v->hdim;
    o.slots = v->slots;
    o.page_max = v->page_max;
    o.tokens = INT_MAX;
    o.kvd = v->kv_heads * v->hdim;
    o.page_stride = 2LL * kPageRows * o.kvd;
    o.layer_stride = o.npages * o.page_stride;
    return true;
}

int lg2(int G) { return G == 1 ? 0 : G == 2 ? 1 : G == 4 ? 2 : 3; }

// Rows (nodes x heads of a group) up to which a tree takes the narrow form
// (its own limit: four 8-row columns of registers; at 20 rows over 256 short
// slots it took 53 us where the wide form took 67; over one slot of 16000 rows
// it takes 37 us for 32 rows where the wide form takes 28 for 36), and its most
// CTAs an SM.
constexpr int kNarrowRows = 32, kNarrowCtas = 3;

bool group_ok(int heads, int kvh, int &G) {
    if (heads < 1 || heads % kvh) return false;
    G = heads / kvh;
    return G == 1 || G == 2 || G == 4 || G == 8;
}

// ---------------------------------------------------------------- tensor maps and kernel attributes

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The whole pool as rows of kvd elements, read in boxes of 64 elements x one
// page's 16 rows, 128-byte swizzled.
bool page_map(const KvView &v, CUtensorMap *map) {
    static EncodeTiled encode = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult st;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &st) == cudaSuccess &&
            st == cudaDriverEntryPointSuccess)
            encode = (EncodeTiled)f;
    });
    if (!encode) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)v.kvd, (cuuint64_t)v.layers * v.npages * 2 * kPageRows}, strides[1] = {(cuuint64_t)v.kvd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)kPageRows}, el[2] = {1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, v.kv, dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, typename F>
bool raise_narrow(F raise) {
    return raise((const void *)tree_attn_mma<T, HD, 1>, tn_smem<T, HD, 1>()) && raise((const void *)tree_attn_mma<T, HD, 2>, tn_smem<T, HD, 2>()) &&
           raise((const void *)tree_attn_mma<T, HD, 3>, tn_smem<T, HD, 3>()) && raise((const void *)tree_attn_mma<T, HD, 4>, tn_smem<T, HD, 4>());
}

template <typename T, int HD, typename F>
bool raise_wide(F raise) {
    return raise((const void *)tree_attn_tc<T, HD, 64>, kTtSmem + 1024) && raise((const void *)tree_attn_tc<T, HD, 128>, kTtSmem + 1024);
}

// SMs of the current device, with the kernels' shared-memory limits raised on
// its first use; 0 when there is no usable device.
int device_sms() {
    constexpr int kMax = 128;
    static std::mutex mu;
    static int sms[kMax];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMax) return 0;
    std::lock_guard<std::mutex> lock(mu);
    if (sms[dev]) return sms[dev];
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 0;
    const auto raise = [](const void *k, size_t b) {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)b) == cudaSuccess;
    };
    if (!raise_wide<float, 64>(raise) || !raise_wide<float, 128>(raise) || !raise_wide<__nv_bfloat16, 64>(raise) ||
        !raise_wide<__nv_bfloat16, 128>(raise) ||
        !raise_narrow<float, 64>(raise) || !raise_narrow<float, 128>(raise) || !raise_narrow<__nv_bfloat16, 64>(raise) ||
        !raise_narrow<__nv_bfloat16, 128>(raise) ||
        !raise((const void *)cache_weights_tc<float, 64>, kWtSmem + 1024) ||
        !raise((const void *)cache_weights_tc<float, 128>, kWtSmem + 1024) ||
        !raise((const void *)cache_weights_tc<__nv_bfloat16, 64>, kWtSmem + 1024) ||
        !raise((const void *)cache_weights_tc<__nv_bfloat16, 128>, kWtSmem + 1024))
        return 0;
    return sms[dev] = n;
}

// ---------------------------------------------------------------- tree commit

struct CommitArgs {
    KvView v;
    int max_nodes;
    const int *len, *off, *parent, *tokens, *next, *forced;
    int *len_out, *naccept, *path, *bonus;
};

// grid (slots, layers).  Warp 0 walks the tree (the next node is the lowest
// one whose parent and token match: two ballots per accepted node); then
// thread c owns 16 bytes of a K or V row and moves the path's rows in order.
// Row j of the path comes from row path[j] >= j, so a row is read before
// anything is written over it.  CTAs of layer 0 write the outcome.
// Bound by latency: a few dependent loads, then one row after the other (32
// layers x 128 slots 10 us, one slot 6 us of kernel time).
__global__ void __launch_bounds__(128) tree_commit(const __grid_constant__ CommitArgs a) {
    __shared__ int s_path[kTreeMax], s_n, s_last;
    const int s = blockIdx.x, layer = blockIdx.y, lane = threadIdx.x & 31;
    int L, t0, n;
    tree_span(a.v, a.len, a.off, a.max_nodes, s, L, t0, n);
    if (threadIdx.x < 32) {
        int par[2], tok[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int i = lane + 32 * h;
            par[h] = i < n ? a.parent[t0 + i] : -3;
            tok[h] = i < n ? a.tokens[t0 + i] : 0;
        }
        int cnt = 0, cur = 0;
        if (n > 0 && a.forced && a.forced[s]) {
            for (int i = lane; i < n; i += 32) s_path[i] = i;
            cnt = n;
            cur = n - 1;
        } else if (n > 0) {
            for (;;) {
                if (lane == 0) s_path[cnt] = cur;
                cnt++;
                const int want = a.next[t0 + cur];
                const unsigned lo = __ballot_sync(0xffffffffu, par[0] == cur && lane > cur && tok[0] == want);
                const unsigned hi = __ballot_sync(0xffffffffu, par[1] == cur && lane + 32 > cur && tok[1] == want);
                if (!lo && !hi) break;
                cur = lo ? __ffs(lo) - 1 : 31 + __ffs(hi);
            }
        }
        if (lane == 0) {
            s_n = cnt;
            s_last = cur;
        }
    }
    __syncthreads();
    const int cnt = s_n;
    if (layer == 0) {
        for (int i = threadIdx.x; i < a.max_nodes; i += blockDim.x)
            a.path[(size_t)s * a.max_nodes + i] = i < cnt ? t0 + s_path[i] : -1;
        if (threadIdx.x == 0) {
            a.len_out[s] = L + cnt;
            a.naccept[s] = cnt;
            a.bonus[s] = n > 0 ? a.next[t0 + s_last] : -1;
        }
    }
    const int chunks = a.v.kvd / 8;  // of a row
    for (int c = threadIdx.x; c < 2 * chunks; c += blockDim.x) {
        uint16_t *base = a.v.kv + (c >= chunks ? (long long)kPageRows * a.v.kvd + (c - chunks) * 8 : (long long)c * 8);
        for (int j = 0; j < cnt; j++) {
            const int i = s_path[j];
            if (i == j) continue;
            const int sp = a.v.page(s, L + i), dp = a.v.page(s, L + j);
            if (dp < 0) continue;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (sp >= 0) x = *(const uint4 *)(base + a.v.row(layer, sp, L + i));
            *(uint4 *)(base + a.v.row(layer, dp, L + j)) = x;
        }
    }
}

// ---------------------------------------------------------------- eviction

struct EvictArgs {
    KvView v, d;
    const int *len;
    const float *acc;
    int acc_rows, budget, sinks, recent;
    int *len_out, *kept;
    float *acc_out;
};

constexpr int kSelThreads = 512;  // a quarter of the select's bins

// Order-preserving key of an accumulated weight: NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// grid (layers * slots * kv heads): the kept rows of one cache column, in
// order.  A radix select over the candidates' 32-bit keys finds the lightest
// kept key T and how many rows equal to T stay; one ordered pass then writes
// the rows that are forced, above T, or among those.  Three passes of 11, 11
// and 10 bits: the first one's bins hold the sign, the exponent and two more
// bits, so that weights of a few magnitudes spread over many bins (by bytes,
// nearly all fell into three, and their shared-memory additions into one
// another).  A warp whose keys all fall into one bin adds them once.  768
// columns of up to 6100 rows take 38 us, 128 of 4096 rows 12 us: passes over
// rows that the L1 holds, one latency after the other.
constexpr int kSelBins = 2048;
__global__ void __launch_bounds__(kSelThreads) evict_select(const __grid_constant__ EvictArgs a) {
    __shared__ unsigned hist[kSelBins], wsum[2][kSelThreads / 32];
    __shared__ unsigned s_prefix, s_need;
    pdl_trigger();
    const int idx = blockIdx.x, kvh = idx % a.v.kvh, s = (idx / a.v.kvh) % a.v.slots, layer = idx / (a.v.kvh * a.v.slots);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = min(min(max(a.len[s], 0), a.acc_rows), a.v.page_max * kPageRows);
    const float *acc = a.acc + (size_t)idx * a.acc_rows;
    int *kept = a.kept + (size_t)idx * a.budget;
    float *acc_out = a.acc_out + (size_t)idx * a.budget;
    if (layer == 0 && kvh == 0 && threadIdx.x == 0) a.len_out[s] = min(n, a.budget);
    for (int j = threadIdx.x + min(n, a.budget); j < a.budget; j += kSelThreads) {
        kept[j] = -1;
        acc_out[j] = 0.f;
    }
    if (n <= a.budget) {
        for (int j = threadIdx.x; j < n; j += kSelThreads) {
            kept[j] = j;
            acc_out[j] = acc[j];
        }
        return;
    }
    const int c0 = a.sinks, c1 = n - a.recent, want = a.budget - a.sinks - a.recent;  // want < c1 - c0
    if (threadIdx.x == 0) {
        s_prefix = 0;
        s_need = want;
    }
    for (int pass = 0; pass < 3 && want > 0; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const unsigned bins = pass == 2 ? 1024 : 2048;
        for (int i = threadIdx.x; i < kSelBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        const unsigned prefix = s_prefix, need = s_need, above = pass == 0 ? 0u : pass == 1 ? ~0u << 21 : ~0u << 10;
        for (int r0 = c0; r0 < c1; r0 += 4 * kSelThreads) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = r0 + i * kSelThreads + threadIdx.x;
                v[i] = r < c1 ? acc[r] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t k = weight_key(v[i]);
                const bool in = r0 + i * kSelThreads + (int)threadIdx.x < c1 && (k & above) == prefix;
                const unsigned bin = (k >> shift) & (bins - 1), who = __ballot_sync(0xffffffffu, in);
                if (!who) continue;
                const unsigned first = __shfl_sync(0xffffffffu, bin, __ffs(who) - 1);
                if (__all_sync(0xffffffffu, !in || bin == first)) {
                    if (lane == 0) atomicAdd(&hist[first], __popc(who));
                } else if (in) {
                    atomicAdd(&hist[bin], 1u);
                }
            }
        }
        __syncthreads();
        // thread t: bins 2047 - 4 t .. 2044 - 4 t, counted from the heaviest
        unsigned c[4], t = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) t += c[i] = hist[kSelBins - 1 - 4 * threadIdx.x - i];
        unsigned incl = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) wsum[0][w] = incl;
        __syncthreads();
        unsigned before = incl - t;
        for (int i = 0; i < w; i++) before += wsum[0][i];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (before < need && need <= before + c[i]) {  // one bin of one thread
                s_prefix = prefix | ((unsigned)(kSelBins - 1 - 4 * threadIdx.x - i) << shift);
                s_need = need - before;
            }
            before += c[i];
        }
        __syncthreads();
    }
    __syncthreads();
    const unsigned T = s_prefix, need = want > 0 ? s_need : 0;
    // thread t owns a run of rows: it counts them, learns how many stand before
    // them, and writes those that stay
    const int run = (n + kSelThreads - 1) / kSelThreads, r0 = min(n, (int)threadIdx.x * run), r1 = min(n, r0 + run);
    const auto kind = [&](int r, float v) {  // 1: stays, 2: tied, 0: goes
        if (r < c0 || r >= c1) return 1;
        if (want == 0) return 0;
        const uint32_t k = weight_key(v);
        return k > T ? 1 : k == T ? 2 : 0;
    };
    unsigned sure = 0, tied = 0;
#pragma unroll 4
    for (int r = r0; r < r1; r++) {
        const int k = kind(r, acc[r]);
        sure += k == 1;
        tied += k == 2;
    }
    unsigned is = sure, it = tied;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, is, o), z = __shfl_up_sync(0xffffffffu, it, o);
        if (lane >= o) {
            is += y;
            it += z;
        }
    }
    if (lane == 31) {
        wsum[0][w] = is;
        wsum[1][w] = it;
    }
    __syncthreads();
    unsigned bs = is - sure, bt = it - tied;  // rows before this run that stay for sure, and tied ones
    for (int i = 0; i < w; i++) {
        bs += wsum[0][i];
        bt += wsum[1][i];
    }
#pragma unroll 4
    for (int r = r0; r < r1; r++) {
        const float v = acc[r];
        const int k = kind(r, v);
        if (k == 1 || (k == 2 && bt < need)) {
            const unsigned j = bs + min(bt, need);
            kept[j] = r;
            acc_out[j] = v;
        }
        bs += k == 1;
        bt += k == 2;
    }
}

// grid (layers * slots * kv heads, row blocks): a warp copies K (lanes 0-15)
// and V (lanes 16-31) of one kept row, 16 bytes a lane (hd 64: 8).  1.15 GB (24
// slots x 8 layers, 1500 rows kept) take 197 us, 5.9 TB/s.  Four rows in flight
// a warp took 274 us with the selection against 239 (the rows' places in memory
// then spread), selection and copy in one kernel 251, the last rows' copy beside
// the selection 282.
constexpr int kGatherRows = 128;
__global__ void __launch_bounds__(256) evict_gather(const __grid_constant__ EvictArgs a) {
    const int idx = blockIdx.x, kvh = idx % a.v.kvh, s = (idx / a.v.kvh) % a.v.slots, layer = idx / (a.v.kvh * a.v.slots);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = min(min(min(max(a.len[s], 0), a.acc_rows), a.v.page_max * kPageRows), a.budget);
    pdl_wait();  // the kept rows
    const int per = a.v.hd / 16;  // elements a lane moves: 8 or 4
    const long long col = (lane >> 4) * (long long)kPageRows * a.v.kvd + kvh * a.v.hd + (lane & 15) * per;
    for (int j = blockIdx.y * kGatherRows + w; j < min(n, (int)(blockIdx.y + 1) * kGatherRows); j += 8) {
        const int r = a.kept[(size_t)idx * a.budget + j];
        const int sp = a.v.page(s, r), dp = a.d.page(s, j);
        if (dp < 0) continue;
        const uint16_t *src = a.v.kv + a.v.row(layer, max(sp, 0), r) + col;
        uint16_t *dst = a.d.kv + a.d.row(layer, dp, j) + col;
        if (per == 8) *(uint4 *)dst = sp < 0 ? make_uint4(0, 0, 0, 0) : *(const uint4 *)src;
        else *(uint2 *)dst = sp < 0 ? make_uint2(0, 0) : *(const uint2 *)src;
    }
}

// In place: grid (layers * slots * kv heads).  Row j comes from row kept[j] >= j,
// so a row may be written once every row up to it has been read: a CTA takes
// its column's rows in order, kMoveRows at a time, reads the next ones while
// these wait for the barrier, and then writes these.  Where rows come from is
// looked up two steps ahead, so that a step waits for one memory access.  With
// the selection 66 us for 128 columns of 4096 -> 1024 rows (39 into another
// cache; 74 without the look ahead, 61 with 128 rows a step) and 304 us for 768
// of up to 6100 -> 1500 (234; 381 with 128 rows a step, one CTA an SM).
constexpr int kMoveWarps = 16, kMoveEach = 4, kMoveRows = kMoveWarps * kMoveEach;
__global__ void __launch_bounds__(kMoveWarps * 32, 2) evict_move(const __grid_constant__ EvictArgs a) {
    const int idx = blockIdx.x, kvh = idx % a.v.kvh, s = (idx / a.v.kvh) % a.v.slots, layer = idx / (a.v.kvh * a.v.slots);
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();  // the kept rows
    if (min(min(max(a.len[s], 0), a.acc_rows), a.v.page_max * kPageRows) <= a.budget) return;
    const int per = a.v.hd / 16;  // elements a lane moves: 8 or 4
    uint16_t *base = a.v.kv + a.v.row(layer, 0, 0) + (lane >> 4) * (long long)kPageRows * a.v.kvd + kvh * a.v.hd + (lane & 15) * per;
    const int *kept = a.kept + (size_t)idx * a.budget;
    // row x of the slot, from the page table: null where there is none
    const auto at = [&](int x) -> uint16_t * {
        const int pg = a.v.page(s, x);
        return pg < 0 ? nullptr : base + a.v.row(0, pg, x);
    };
    const uint16_t *src[kMoveEach];
    const auto find = [&](int j0) {
#pragma unroll
        for (int i = 0; i < kMoveEach; i++) {
            const int j = j0 + i * kMoveWarps + w;
            src[i] = j < a.budget ? at(kept[j]) : nullptr;
        }
    };
    const auto load = [&](uint4 (&v)[kMoveEach]) {
#pragma unroll
        for (int i = 0; i < kMoveEach; i++) {
            v[i] = make_uint4(0, 0, 0, 0);
            if (!src[i]) continue;
            if (per == 8) v[i] = *(const uint4 *)src[i];
            else *(uint2 *)&v[i] = *(const uint2 *)src[i];
        }
    };
    uint4 x[kMoveEach], y[kMoveEach];
    find(0);
    load(x);
    find(kMoveRows);
    for (int j0 = 0; j0 < a.budget; j0 += kMoveRows) {
        load(y);
        find(j0 + 2 * kMoveRows);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMoveEach; i++) {
            const int j = j0 + i * kMoveWarps + w;
            uint16_t *dst = j < a.budget ? at(j) : nullptr;
            if (dst && per == 8) *(uint4 *)dst = x[i];
            else if (dst) *(uint2 *)dst = *(const uint2 *)&x[i];
            x[i] = y[i];
        }
    }
}

// Failure-detection probe: the kernels' wait on a phase that nothing
// completes, for limit_ns.  It gives up, is counted, and the kernel returns.
__global__ void kv_wait_probe(unsigned long long limit_ns) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ int stop;
    if (threadIdx.x == 0) {
        stop = 0;
        mb_init(&bar, 1);
        mb_wait(&bar, 0, &stop, limit_ns);
    }
}

template <typename... KArgs, typename... Args>
cudaError_t go(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, void *stream, bool pdl, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// One tree attention's form and its scratch: the ranges' table, then two
// pieces a range and row block (a range's first and last column may be split).
// Up to 32 (node, head) rows take the narrow form, with a warp to a range.
struct TreeWs {
    bool narrow;
    int ranges, row_blocks, rows;  // rows: of a piece
    size_t ml, o, bytes;
};
TreeWs tree_ws(const KvView &v, int G, int max_nodes, int sms) {
    TreeWs w;
    w.narrow = max_nodes * G <= kNarrowRows;
    w.row_blocks = w.narrow ? 1 : (max_nodes * G + 127) / 128;
    w.rows = w.narrow ? (max_nodes * G + 7) & ~7 : 128;
    w.ranges = w.narrow ? sms * kNarrowCtas : sms / w.row_blocks > 1 ? sms / w.row_blocks : 1;
    const size_t pieces = (size_t)2 * w.ranges * w.row_blocks;
    w.ml = ((size_t)w.ranges * sizeof(int4) + 255) & ~(size_t)255;
    w.o = w.ml + ((pieces * w.rows * sizeof(float2) + 255) & ~(size_t)255);
    w.bytes = w.o + pieces * w.rows * v.hd * sizeof(float);
    return w;
}

int done(cudaError_t e, char *err, int cap) {
    if (e != cudaSuccess) return op_fail(err, cap, -3, cudaGetErrorString(e));
    if (err && cap > 0) err[0] = 0;
    return 0;
}

}  // namespace

extern "C" {

HYC_API int hyc_kvops_timeouts(void) {
    unsigned n = 0;
    return cudaMemcpyFromSymbol(&n, g_kv_timeouts, sizeof n) == cudaSuccess ? (int)n : -1;
}

HYC_API int hyc_kvops_wait_probe(unsigned long long limit_ns) {
    if (limit_ns == 0 || limit_ns > 1000000000ull) return -1;
    kv_wait_probe<<<1, 32>>>(limit_ns);
    return cudaGetLastError() == cudaSuccess && cudaDeviceSynchronize() == cudaSuccess ? 0 : -1;
}

// The count behind the stream's work so far, into pinned memory: for the batch
// engine, which looks at it with every pass's outcome.
int hyk_kvops_timeouts_async(void *stream, unsigned *host) {
    const cudaError_t e = cudaMemcpyFromSymbolAsync(host, g_kv_timeouts, sizeof *host, 0, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
    return e == cudaSuccess ? 0 : -1;
}

HYC_API size_t hyc_tree_attention_ws(const hyc_kv_view *cache, int heads, int max_nodes) {
    KvView v;
    const char *why;
    int G;
    if (!make_view(cache, v, &why) || !group_ok(heads, v.kvh, G) || max_nodes < 1 || max_nodes > kTreeMax) return 0;
    const int sms = device_sms();
    return tree_ws(v, G, max_nodes, sms > 0 ? sms : 148).bytes;
}

HYC_API int hyc_tree_attention_n(void *stream, const hyc_kv_view *cache, int layer, int heads, int max_nodes, int tokens,
                                 const int *d_len, const int *d_off, const int *d_parent, const void *d_q,
                                 long long q_ld, int q_bf16, float scale, void *d_out, long long out_ld, float *d_lse,
                                 void *d_ws, size_t ws_bytes, char *err, int err_cap) {
    TreeArgs a;
    const char *why;
    if (!make_view(cache, a.v, &why)) return op_fail(err, err_cap, -1, why);
    if (tokens < 0) return op_fail(err, err_cap, -1, "tokens must not be negative");
    a.v.tokens = tokens;
    if (!group_ok(heads, a.v.kvh, a.G)) return op_fail(err, err_cap, -1, "heads / kv_heads must be 1, 2, 4 or 8");
    if (layer < 0 || layer >= a.v.layers) return op_fail(err, err_cap, -1, "no such layer");
    if (max_nodes < 1 || max_nodes > kTreeMax) return op_fail(err, err_cap, -1, "max_nodes must be 1 .. 64");
    if (!d_len || !d_off || !d_parent || !d_q || !d_out || !d_ws) return op_fail(err, err_cap, -1, "null argument");
    if (!std::isfinite(scale)) return op_fail(err, err_cap, -1, "scale must be finite");
    const int el = q_bf16 ? 2 : 4;
    if (!aligned16(d_q) || !aligned16(d_out) || ((uintptr_t)d_ws & 255) || (q_ld * el) % 16 || (out_ld * el) % 16 ||
        q_ld < (long long)heads * a.v.hd || out_ld < (long long)heads * a.v.hd)
        return op_fail(err, err_cap, -1, "q and out must be 16-byte aligned with rows of heads * hdim or more, the scratch 256-byte aligned");
    a.layer = layer;
    a.heads = heads;
    a.max_nodes = max_nodes;
    a.len = d_len;
    a.off = d_off;
    a.parent = d_parent;
    a.q = d_q;
    a.q_ld = q_ld;
    a.scale = scale;
    a.out = d_out;
    a.out_ld = out_ld;
    a.lse = d_lse;
    const int sms = device_sms();
    if (sms < 1) return op_fail(err, err_cap, -3, "no usable CUDA device");
    const TreeWs ws = tree_ws(a.v, a.G, max_nodes, sms);
    if (ws_bytes < ws.bytes) return op_fail(err, err_cap, -1, "scratch too small");
    a.out32 = ((uintptr_t)d_out & 31) == 0 && (out_ld * el) % 32 == 0;
    a.roots = (int4 *)d_ws;
    a.lg = lg2(a.G);
    a.part_ml = (float2 *)((char *)d_ws + ws.ml);
    a.part_o = (float *)((char *)d_ws + ws.o);
    a.ranges = ws.ranges;
    a.row_blocks = ws.row_blocks;
    cudaError_t e = cudaErrorInvalidValue;
    const dim3 mgrid(4 * sms);
    if (ws.narrow) {
        // short slots (and columns enough): a column to a CTA, no pieces and no
        // second kernel (256 slots of 192 rows 47.4 -> 45.8 us; one of 64 rows
        // 15.5 -> 13.7, the host's launch); longer slots would leave SMs idle
        const int cap = (a.v.page_max * kPageRows + kTnK - 1) / kTnK;
        a.whole = cap <= 2 || (cap <= 4 && a.v.slots * a.v.kvh >= sms);
        // as many CTAs as an SM holds (ranges are equal shares, so all of them
        // should run at once), by shared memory and the kernel's register bound
#define HY_NT(T_, HD_, NT_)                                                                                             \
    if (ws.rows == 8 * NT_) {                                                                                           \
        a.ranges = sms * std::min(kNarrowCtas, (int)(227 * 1024 / (tn_smem<T_, HD_, NT_>() + 2048)));                             \
        e = go(tree_attn_mma<T_, HD_, NT_>, dim3(a.ranges), dim3(kTnThreads), tn_smem<T_, HD_, NT_>(), stream, false, a); \
        if (e == cudaSuccess && !a.whole)                                                                               \
            e = go(tree_merge<T_, HD_, kTnK>, mgrid, dim3(kMergeThreads), 0, stream, true, a, ws.rows);                 \
    }
#define HY_TREE(T_, HD_) HY_NT(T_, HD_, 1) HY_NT(T_, HD_, 2) HY_NT(T_, HD_, 3) HY_NT(T_, HD_, 4)
        if (q_bf16 && a.v.hd == 64) { HY_TREE(__nv_bfloat16, 64) }
        else if (q_bf16) { HY_TREE(__nv_bfloat16, 128) }
        else if (a.v.hd == 64) { HY_TREE(float, 64) }
        else { HY_TREE(float, 128) }
#undef HY_TREE
#undef HY_NT
        return done(e, err, err_cap);
    }
    CUtensorMap map;
    if (!page_map(a.v, &map)) return op_fail(err, err_cap, -3, "cuTensorMapEncodeTiled failed");
    const dim3 grid(ws.ranges * ws.row_blocks);
#define HY_TREE(T_, HD_)                                                                                                \
    {                                                                                                                   \
        e = max_nodes * a.G <= 64 ? go(tree_attn_tc<T_, HD_, 64>, grid, dim3(kTtThreads), kTtSmem + 1024, stream, false, a, map) \
                                  : go(tree_attn_tc<T_, HD_, 128>, grid, dim3(kTtThreads), kTtSmem + 1024, stream, false, a, map); \
        if (e == cudaSuccess) e = go(tree_merge<T_, HD_, kTtK>, mgrid, dim3(kMergeThreads), 0, stream, true, a, 0);       \
    }
    if (q_bf16) {
        if (a.v.hd == 64) HY_TREE(__nv_bfloat16, 64) else HY_TREE(__nv_bfloat16, 128)
    } else {
        if (a.v.hd == 64) HY_TREE(float, 64) else HY_TREE(float, 128)
    }
#undef HY_TREE
    return done(e, err, err_cap);
}

HYC_API int hyc_tree_attention(void *stream, const hyc_kv_view *cache, int layer, int heads, int max_nodes,
                               const int *d_len, const int *d_off, const int *d_parent, const void *d_q,
                               long long q_ld, int q_bf16, float scale, void *d_out, long long out_ld, float *d_lse,
                               void *d_ws, size_t ws_bytes, char *err, int err_cap) {
    return hyc_tree_attention_n(stream, cache, layer, heads, max_nodes, INT_MAX, d_len, d_off, d_parent, d_q, q_ld, q_bf16,
                                scale, d_out, out_ld, d_lse, d_ws, ws_bytes, err, err_cap);
}

HYC_API int hyc_tree_commit_n(void *stream, const hyc_kv_view *cache, int max_nodes, int tokens, const int *d_len,
                              const int *d_off, const int *d_parent, const int *d_tokens, const int *d_next,
                              const int *d_forced, int *d_len_out, int *d_naccept, int *d_path, int *d_bonus,
                              char *err, int err_cap) {
    CommitArgs a;
    const char *why;
    if (!make_view(cache, a.v, &why)) return op_fail(err, err_cap, -1, why);
    if (tokens < 0) return op_fail(err, err_cap, -1, "tokens must not be negative");
    a.v.tokens = tokens;
    if (max_nodes < 1 || max_nodes > kTreeMax) return op_fail(err, err_cap, -1, "max_nodes must be 1 .. 64");
    if (!d_len || !d_off || !d_parent || !d_tokens || !d_next || !d_len_out || !d_naccept || !d_path || !d_bonus)
        return op_fail(err, err_cap, -1, "null argument");
    if (d_len_out == d_len) return op_fail(err, err_cap, -1, "d_len_out must not be d_len");
    a.max_nodes = max_nodes;
    a.len = d_len;
    a.off = d_off;
    a.parent = d_parent;
    a.tokens = d_tokens;
    a.next = d_next;
    a.forced = d_forced;
    a.len_out = d_len_out;
    a.naccept = d_naccept;
    a.path = d_path;
    a.bonus = d_bonus;
    return done(go(tree_commit, dim3(a.v.slots, a.v.layers), dim3(128), 0, stream, false, a), err, err_cap);
}

HYC_API int hyc_tree_commit(void *stream, const hyc_kv_view *cache, int max_nodes, const int *d_len,
                            const int *d_off, const int *d_parent, const int *d_tokens, const int *d_next,
                            const int *d_forced, int *d_len_out, int *d_naccept, int *d_path, int *d_bonus,
                            char *err, int err_cap) {
    return hyc_tree_commit_n(stream, cache, max_nodes, INT_MAX, d_len, d_off, d_parent, d_tokens, d_next, d_forced, d_len_out,
                             d_naccept, d_path, d_bonus, err, err_cap);
}

HYC_API int hyc_cache_weights_n(void *stream, const hyc_kv_view *cache, int heads, int max_q, int tokens, const int *d_len,
                                const int *d_nq, const int *d_sel, const void *d_q, long long q_ld, long long q_layer,
                                int q_bf16, const float *d_lse, long long lse_layer, float scale, float *d_acc,
                                int acc_rows, char *err, int err_cap) {
    WeightArgs a;
    const char *why;
    if (!make_view(cache, a.v, &why)) return op_fail(err, err_cap, -1, why);
    if (tokens < 0) return op_fail(err, err_cap, -1, "tokens must not be negative");
    a.v.tokens = tokens;
    if (!group_ok(heads, a.v.kvh, a.G)) return op_fail(err, err_cap, -1, "heads / kv_heads must be 1, 2, 4 or 8");
    if (max_q < 1 || max_q > kTreeMax) return op_fail(err, err_cap, -1, "max_q must be 1 .. 64");
    if (!d_len || !d_nq || !d_sel || !d_q || !d_lse || !d_acc || acc_rows < 1)
        return op_fail(err, err_cap, -1, "null argument");
    if (!std::isfinite(scale)) return op_fail(err, err_cap, -1, "scale must be finite");
    const int el = q_bf16 ? 2 : 4;
    if (!aligned16(d_q) || (q_ld * el) % 16 || (q_layer * el) % 16 || q_ld < (long long)heads * a.v.hd)
        return op_fail(err, err_cap, -1, "q must be 16-byte aligned with rows of heads * hdim or more");
    a.heads = heads;
    a.max_q = max_q;
    a.len = d_len;
    a.nq = d_nq;
    a.sel = d_sel;
    a.q = d_q;
    a.q_ld = q_ld;
    a.q_layer = q_layer;
    a.lse = d_lse;
    a.lse_layer = lse_layer;
    a.scale = scale;
    a.acc = d_acc;
    a.acc_rows = acc_rows;
    a.lg = lg2(a.G);
    const int sms = device_sms();
    if (sms < 1) return op_fail(err, err_cap, -3, "no usable CUDA device");
    CUtensorMap map;
    if (!page_map(a.v, &map)) return op_fail(err, err_cap, -3, "cuTensorMapEncodeTiled failed");
    // a second Q buffer where it leaves K four stages or more
    a.block = max_q * a.G < 128 ? (max_q * a.G + 15) & ~15 : 128;
    const int qbytes = (q_bf16 ? 1 : 3) * a.block * a.v.hd * 2, stage = 128 * a.v.hd * 2;
    a.qbufs = (kWtSmem - 2 * qbytes) / stage >= 4 ? 2 : 1;
    a.stages = (kWtSmem - a.qbufs * qbytes) / stage;
    if (a.stages > 8) a.stages = 8;
    const size_t smem = (size_t)a.qbufs * qbytes + (size_t)a.stages * stage + 1024;
    const dim3 grid(sms), block(kWtThreads);
    cudaError_t e;
    if (a.v.hd == 64)
        e = q_bf16 ? go(cache_weights_tc<__nv_bfloat16, 64>, grid, block, smem, stream, false, a, map)
                   : go(cache_weights_tc<float, 64>, grid, block, smem, stream, false, a, map);
    else
        e = q_bf16 ? go(cache_weights_tc<__nv_bfloat16, 128>, grid, block, smem, stream, false, a, map)
                   : go(cache_weights_tc<float, 128>, grid, block, smem, stream, false, a, map);
    return done(e, err, err_cap);
}

HYC_API int hyc_cache_weights(void *stream, const hyc_kv_view *cache, int heads, int max_q, const int *d_len,
                              const int *d_nq, const int *d_sel, const void *d_q, long long q_ld, long long q_layer,
                              int q_bf16, const float *d_lse, long long lse_layer, float scale, float *d_acc,
                              int acc_rows, char *err, int err_cap) {
    return hyc_cache_weights_n(stream, cache, heads, max_q, INT_MAX, d_len, d_nq, d_sel, d_q, q_ld, q_layer, q_bf16, d_lse,
                               lse_layer, scale, d_acc, acc_rows, err, err_cap);
}

HYC_API int hyc_cache_evict(void *stream, const hyc_kv_view *cache, const hyc_kv_view *dst, const int *d_len,
                            const float *d_acc, int acc_rows, int budget, int sinks, int recent, int *d_len_out,
                            int *d_kept, float *d_acc_out, char *err, int err_cap) {
    EvictArgs a;
    const char *why;
    if (!make_view(cache, a.v, &why) || !make_view(dst, a.d, &why)) return op_fail(err, err_cap, -1, why);
    if (a.v.layers != a.d.layers || a.v.slots != a.d.slots || a.v.kvh != a.d.kvh || a.v.hd != a.d.hd)
        return op_fail(err, err_cap, -1, "the two caches must have the same layers, slots and heads");
    if (!d_len || !d_acc || !d_len_out || !d_kept || !d_acc_out) return op_fail(err, err_cap, -1, "null argument");
    if (d_len_out == d_len) return op_fail(err, err_cap, -1, "d_len_out must not be d_len");
    if (budget < 1 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
        return op_fail(err, err_cap, -1, "budget must hold at least sinks + recent rows");
    if ((long long)a.d.page_max * kPageRows < budget)
        return op_fail(err, err_cap, -1, "the destination's page table does not hold budget rows");
    if (acc_rows < 1) return op_fail(err, err_cap, -1, "acc_rows must be positive");
    a.len = d_len;
    a.acc = d_acc;
    a.acc_rows = acc_rows;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.len_out = d_len_out;
    a.kept = d_kept;
    a.acc_out = d_acc_out;
    const long long cols = (long long)a.v.layers * a.v.slots * a.v.kvh;
    if (cols > 0x7fffffff || budget > (1 << 21)) return op_fail(err, err_cap, -1, "cache or budget too large");
    cudaError_t e = go(evict_select, dim3((unsigned)cols), dim3(kSelThreads), 0, stream, false, a);
    const bool same = a.v.kv == a.d.kv && a.v.pages == a.d.pages && a.v.npages == a.d.npages && a.v.page_max == a.d.page_max;
    if (e == cudaSuccess && same) e = go(evict_move, dim3((unsigned)cols), dim3(kMoveWarps * 32), 0, stream, true, a);
    else if (e == cudaSuccess)
        e = go(evict_gather, dim3((unsigned)cols, (budget + kGatherRows - 1) / kGatherRows), dim3(256), 0, stream, true, a);
    return done(e, err, err_cap);
}

}  // extern "C"
