// hy_tree.cuh — speculative decoding over the batch engine, with a bound on
// the cache.  Part of hy_backend.cu's translation unit (it uses HyCtx, Batch
// and the layer loop).
//
// No counterpart in the reference, whose loop feeds one token per step
// (src/model.c:943-954) and lets the cache grow to its context (:804-808).
// A pass feeds every slot a small tree of drafted tokens, node 0 being the
// token its sequence ends with: the projections run over all nodes as over any
// batch, attention lets a node see the slot's cached rows and its ancestors
// (hyc_tree_attention), and the argmax after each node decides which path the
// model would have taken itself (hyc_tree_commit), whose rows stay.  A pass
// thus yields one token or more; the tokens are those of the plain greedy loop
// up to near ties, as projections of other batch sizes and another attention
// sum in another order.  What a pass costs goes by its nodes, through the batch
// engine's per-layer launches: at 256 rows of the 32-layer STQ1_0 model 1.76 ms
// for one node, 3.5 for 4, 8.9 for 16 (GEMVs over groups of tokens), 3.3 for 32
// and 3.4 for 64 (tensor cores), against 0.81 ms a token of the persistent
// kernel: over four accepted tokens a pass in trees of 32 nodes or more are a
// gain, small trees are none.  With weights on, the accepted queries'
// attention probabilities are added up per cached row (hyc_cache_weights), and
// eviction keeps the heaviest rows (hyc_cache_evict): a slot's rows are then
// no longer its positions, so the two are counted apart.

extern "C" int hyk_kvops_timeouts_async(void *stream, unsigned *host);  // hy_kvops.cu

struct TreeState {
    int max_nodes = 0;
    bool weights = false;
    std::vector<int> len, pos;  // rows and next position of each slot
    std::vector<char> fed;      // it has been written from outside since it was opened: len says nothing of its rows
    unsigned gave_up = 0;       // waits of the operators' kernels that had given up before
    // device ints, staged from pinned memory in one copy: len [S] | off [S + 1] |
    // forced [S] | parent [T] | row [T], then the outcome: len_out [S] |
    // accepted [S] | bonus [S] | path [S][max_nodes]; and, on the host alone, the count
    // of waits that have given up
    int *d_int = nullptr, *h_int = nullptr;
    size_t in_ints = 0, ints = 0;
    float *qkv = nullptr, *lse = nullptr, *acc = nullptr;  // [L][T][q | k | v], [L][T][heads], [L][S][kvh][rows]
    void *ws = nullptr;
    size_t ws_bytes = 0;
    int *kept = nullptr;  // eviction: [L][S][kvh][evict_rows], and the kept rows' weights (lazy)
    float *acc2 = nullptr;
    int evict_rows = 0;
    int *d_len() const { return d_int; }
};

int tree_rows(const Batch &b) { return b.page_max * kPageRows; }

void tree_free(Batch *b) {
    TreeState *t = b->tree;
    if (!t) return;
    void *ptrs[] = {t->d_int, t->qkv, t->lse, t->acc, t->ws, t->kept, t->acc2};
    for (void *p : ptrs) cudaFree(p);
    if (t->h_int) cudaFreeHost(t->h_int);
    delete t;
    b->tree = nullptr;
}

hyc_kv_view tree_view(const HyCtx *c, uint16_t *kv) {
    const Batch &b = *c->bat;
    hyc_kv_view v;
    v.kv = kv;
    v.pages = b.d_pages;
    v.layers = c->L;
    v.npages = b.npages;
    v.kv_heads = c->kvh;
    v.hdim = c->hd;
    v.slots = b.slots;
    v.page_max = b.page_max;
    return v;
}

// The count of waits that have given up, with the stream's work done: noted, or
// compared with what it was (an operator that gave up has ended with wrong
// outputs).
bool tree_waits(HyCtx *c, TreeState &t, bool note) {
    unsigned *now = (unsigned *)(t.h_int + t.ints);
    if (hyk_kvops_timeouts_async(c->st, now) != 0) return fail(c, "kvops timeouts", cudaGetLastError());
    CK(c, cudaStreamSynchronize(c->st));
    if (note) t.gave_up = *now;
    if (*now == t.gave_up) return true;
    c->broken = true;
    snprintf(c->err, sizeof c->err, "operators on the KV cache: a wait inside a kernel timed out");
    return false;
}

bool tree_prepare(HyCtx *c, int max_nodes, bool weights) {
    Batch &b = *c->bat;
    REQ(c, max_nodes >= 1 && max_nodes <= 64, "a tree has 1 .. 64 nodes");
    REQ(c, b.max_out >= b.max_tokens || b.max_out >= b.slots * max_nodes, "batch head rows must cover every node of a pass");
    tree_free(&b);
    CK(c, cudaStreamSynchronize(c->st));
    TreeState *t = b.tree = new TreeState();
    const size_t S = (size_t)b.slots, T = (size_t)b.max_tokens;
    t->max_nodes = max_nodes;
    t->weights = weights;
    t->len.assign(S, 0);
    t->pos.assign(S, 0);
    t->fed.assign(S, 0);
    t->in_ints = 3 * S + 1 + 2 * T;
    t->ints = t->in_ints + 3 * S + S * max_nodes;
    CK(c, cudaMalloc(&t->d_int, t->ints * 4));
    CK(c, cudaMallocHost(&t->h_int, (t->ints + 1) * 4));
    if (!tree_waits(c, *t, true)) return false;
    const hyc_kv_view v = tree_view(c, b.kv);
    t->ws_bytes = hyc_tree_attention_ws(&v, c->heads, max_nodes);
    REQ(c, t->ws_bytes > 0, "unsupported head geometry");
    CK(c, cudaMalloc(&t->ws, t->ws_bytes));
    if (weights) {
        const size_t acc = (size_t)c->L * S * c->kvh * tree_rows(b) * 4;
        CK(c, cudaMalloc(&t->qkv, (size_t)c->L * T * (c->qd + 2 * c->kvd) * 4));
        CK(c, cudaMalloc(&t->lse, (size_t)c->L * T * c->heads * 4));
        CK(c, cudaMalloc(&t->acc, acc));
        CK(c, cudaMemsetAsync(t->acc, 0, acc, c->st));
    }
    return true;
}

// The pass's addressing where it is one of drafted trees: rows apart from
// positions, and, with weights, q | k | v of every layer kept for them.
void fwd_tree(HyCtx *c, Fwd &f) {
    const Batch &b = *c->bat;
    const TreeState &t = *b.tree;
    f.tree = true;
    f.tok_row = t.d_int + 3 * b.slots + 1 + b.max_tokens;
    if (t.qkv) {
        f.qkv = t.qkv;
        f.qkv_stride = (size_t)b.max_tokens * (c->qd + 2 * c->kvd);
    }
}

// rope, norms and the rows' store, then the trees' attention of one layer
bool tree_attention(HyCtx *c, const Fwd &f, const AttnArgs &aa, int li, int nt, bool pdl) {
    const Batch &b = *c->bat;
    TreeState &t = *b.tree;
    int warps = aa.heads + aa.kv_heads;
    if (warps > 32) warps = 32;
    const int rgrid = nt < 16 * c->nsm ? nt : 16 * c->nsm;
    const bool stored = c->hd == 128 ? launch(c, rope_norm_store<128>, dim3(rgrid), dim3(warps * 32), 0, pdl, aa)
                                     : launch(c, rope_norm_store<64>, dim3(rgrid), dim3(warps * 32), 0, pdl, aa);
    if (!stored) return false;
    const int S = b.slots;
    const hyc_kv_view v = tree_view(c, f.kv);
    if (hyc_tree_attention_n(c->st, &v, li, c->heads, t.max_nodes, nt, t.d_len(), t.d_int + S, t.d_int + 3 * S + 1, aa.qkv,
                             aa.qkv_ld, 0, aa.scale, aa.ao, aa.qdim, t.lse ? t.lse + (size_t)li * b.max_tokens * c->heads : nullptr,
                             t.ws, t.ws_bytes, c->err, sizeof c->err) != 0) {
        c->broken = true;
        return false;
    }
    c->launches += 2;
    return true;
}

// One pass over every slot's tree; the outcome stays in pinned memory.
bool tree_run(HyCtx *c, const int *tokens, const int *parent, const int *off, const int *forced, int vocab_out) {
    Batch &b = *c->bat;
    TreeState &t = *b.tree;
    const int S = b.slots, T = b.max_tokens, nt = off[S];
    REQ(c, off[0] == 0 && nt >= 1 && nt <= T && nt <= b.max_out, "more nodes than the batch's tokens or head rows");
    int *h_len = t.h_int, *h_off = t.h_int + S, *h_forced = h_off + S + 1, *h_par = h_forced + S, *h_row = h_par + T;
    int *tok = b.h_in, *slot = b.h_in + T, *pos = b.h_in + 2 * T, *rows = b.h_in + 3 * T;
    // all offsets before any of them is used: in between two that hold, one may lie past the arrays
    for (int s = 0; s < S; s++)
        REQ(c, off[s + 1] >= off[s] && off[s + 1] <= nt && off[s + 1] - off[s] <= t.max_nodes,
            "a slot's offsets fall, or its tree has more than max_nodes nodes");
    for (int s = 0; s < S; s++) {
        const int n = off[s + 1] - off[s];
        REQ(c, n == 0 || t.len[s] + n <= b.slot_ctx, "a tree does not fit its slot's context");
        for (int i = 0; i < n; i++) {
            const int k = off[s] + i, p = parent[k];
            REQ(c, i == 0 ? p == -1 : p >= 0 && p < i, "node 0 has parent -1, every other node one below itself");
            REQ(c, !forced || !forced[s] || p == i - 1, "a forced slot's nodes are a chain");
            pos[k] = i == 0 ? t.pos[s] : pos[off[s] + p] + 1;
            REQ(c, pos[k] < c->ctx, "a position is past the prepared context");
            tok[k] = tokens[k];
            slot[k] = s;
            rows[k] = k;
            h_par[k] = p;
            h_row[k] = t.len[s] + i;
        }
        h_len[s] = t.len[s];
        h_off[s] = off[s];
        h_forced[s] = forced ? forced[s] : 0;
    }
    h_off[S] = nt;
    CK(c, cudaMemcpyAsync(t.d_int, t.h_int, (size_t)(3 * S + 1 + nt) * 4, cudaMemcpyHostToDevice, c->st));
    CK(c, cudaMemcpyAsync(t.d_int + 3 * S + 1 + T, h_row, (size_t)nt * 4, cudaMemcpyHostToDevice, c->st));
    if (!batch_upload(c, nt, nt)) return false;
    b.in_tree = true;
    const bool ran = batch_run(c, nt, nt, vocab_out);
    b.in_tree = false;
    if (!ran) return false;
    const hyc_kv_view v = tree_view(c, b.kv);
    int *out = t.d_int + t.in_ints;
    bool ok = hyc_tree_commit_n(c->st, &v, t.max_nodes, nt, t.d_len(), t.d_int + S, t.d_int + 3 * S + 1, b.tok(), b.d_ids,
                                t.d_int + 2 * S + 1, out, out + S, out + 3 * S, out + 2 * S, c->err, sizeof c->err) == 0;
    c->launches++;
    if (ok && t.weights) {
        const int ld = c->qd + 2 * c->kvd;
        ok = hyc_cache_weights_n(c->st, &v, c->heads, t.max_nodes, nt, t.d_len(), out + S, out + 3 * S, t.qkv, ld,
                                 (long long)T * ld, 0, t.lse, (long long)T * c->heads, 1.0f / sqrtf((float)c->hd), t.acc,
                                 tree_rows(b), c->err, sizeof c->err) == 0;
        c->launches++;
    }
    if (!ok) {
        c->broken = true;
        return false;
    }
    CK(c, cudaMemcpyAsync(t.h_int + t.in_ints, out, (t.ints - t.in_ints) * 4, cudaMemcpyDeviceToHost, c->st));
    if (!tree_waits(c, t, false) || !tc_status(c)) return false;
    for (int s = 0; s < S; s++) {
        if (off[s + 1] > off[s]) t.fed[s] = 0;
        t.len[s] = t.h_int[t.in_ints + s];
        t.pos[s] += t.h_int[t.in_ints + S + s];
    }
    return true;
}

bool tree_evict(HyCtx *c, int budget, int sinks, int recent) {
    Batch &b = *c->bat;
    TreeState &t = *b.tree;
    REQ(c, t.weights, "eviction needs accumulated weights (hyc_tree_prepare)");
    REQ(c, budget >= 1 && budget <= tree_rows(b) && sinks >= 0 && recent >= 0 && sinks <= budget - recent,
        "the budget must hold sinks + recent rows and fit a slot");
    const size_t S = (size_t)b.slots, cols = (size_t)c->L * S * c->kvh, R = (size_t)tree_rows(b);
    // a fed slot goes in as one that is within the budget: nothing of it moves
    bool any = false;
    for (size_t s = 0; s < S; s++) {
        any |= t.len[s] > budget && !t.fed[s];
        t.h_int[s] = t.fed[s] ? std::min(t.len[s], budget) : t.len[s];
    }
    if (!any) return true;
    if (t.evict_rows < budget) {
        cudaFree(t.kept);
        cudaFree(t.acc2);
        t.kept = nullptr;
        t.acc2 = nullptr;
        t.evict_rows = 0;
        CK(c, cudaMalloc(&t.kept, cols * budget * 4));
        CK(c, cudaMalloc(&t.acc2, cols * budget * 4));
        t.evict_rows = budget;
    }
    int *out = t.d_int + t.in_ints;
    CK(c, cudaMemcpyAsync(t.d_int, t.h_int, S * 4, cudaMemcpyHostToDevice, c->st));
    const hyc_kv_view v = tree_view(c, b.kv);
    if (hyc_cache_evict(c->st, &v, &v, t.d_len(), t.acc, (int)R, budget, sinks, recent, out, t.kept, t.acc2, c->err,
                        sizeof c->err) != 0) {
        c->broken = true;
        return false;
    }
    c->launches += 2;
    CK(c, cudaMemcpy2DAsync(t.acc, R * 4, t.acc2, (size_t)budget * 4, (size_t)budget * 4, cols, cudaMemcpyDeviceToDevice, c->st));
    CK(c, cudaStreamSynchronize(c->st));
    for (size_t s = 0; s < S; s++)
        if (!t.fed[s]) t.len[s] = std::min(t.len[s], budget);
    return true;
}

void tree_close_all(Batch &b) {
    if (!b.tree) return;
    b.tree->len.assign(b.tree->len.size(), 0);
    b.tree->pos.assign(b.tree->pos.size(), 0);
    b.tree->fed.assign(b.tree->fed.size(), 0);
}

void tree_fed(Batch &b, int slot) {
    if (b.tree) b.tree->fed[(size_t)slot] = 1;
}
