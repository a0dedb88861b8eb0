// Verification of a drafted tree on a model's cache (jl_predict_tree), the
// compaction of the cache to an accepted path (jl_cache_compact) and forks of a
// cache (jl_cache_fork).
//
// The reference verifies a chain (speculative.rs:95-97) and grows each cache on
// its own (model.rs:37-52).  A tree pass appends its nodes behind the cache's
// committed positions, node j at slot len + j, rotated for position len + depth;
// each node attends to the committed positions and to its ancestors.  Forks
// share full pages: KvPool::refs counts the caches that hold a page, and
// cache_reserve gives a cache a page of its own before it writes to a shared one.
#include <algorithm>
#include <cstring>
#include <memory>

#include "jl_internal.h"
#include "kernels.cuh"
#include "ops_host.h"
#include "timeline.cuh"

namespace jl {

jl_status check_device_flag(jl_model* m);
jl_status check_ids(const jl_model* m, const uint32_t* ids, size_t n);

// Device copies of a tree pass's descriptors and the attention's workspace.
struct TreeBuffers {
    struct Desc {
        uint64_t mask[JL_TREE_MAX_NODES][JL_TREE_MAX_NODES / 64];
        int32_t pos[JL_TREE_MAX_NODES], slot[JL_TREE_MAX_NODES], path[JL_TREE_MAX_NODES];
        int32_t start[2], ctx, path_len;
    };
    Desc* dev = nullptr;
    Desc* host = nullptr;  // pinned; every call that uses it ends with a synchronisation
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
};

void tree_buffers_free(TreeBuffers* t) {
    if (!t) return;
    cudaFree(t->dev);
    cudaFreeHost(t->host);
    cudaFree(t->workspace);
    delete t;
}

namespace {

constexpr int MASK_WORDS = JL_TREE_MAX_NODES / 64;

jl_kv_pages pages_of(const jl_model* m, int layer, int layers) {
    const KvView v = kv_view(m, layer);
    jl_kv_pages p{};
    p.k = v.k;
    p.v = v.v;
    p.layer_stride = 2 * m->kv.pages * m->kv.page_elems * m->kv.elem;
    p.layers = layers;
    p.pages = (int)m->kv.pages;
    p.kv_heads = m->kv_heads;
    p.dtype = m->kv.dtype;
    return p;
}

// Made by the first call that needs them.
jl_status tree_buffers(jl_model* m, TreeBuffers** out) {
    if (!m->tree) {
        std::unique_ptr<TreeBuffers, void (*)(TreeBuffers*)> t(new TreeBuffers(), tree_buffers_free);
        jl_tree_attn a{};
        a.pool = pages_of(m, 0, 1);
        a.q_heads = m->q_heads;
        a.dtype = JL_KV_F32;
        a.max_nodes = JL_TREE_MAX_NODES;
        // a smaller tree has fewer tiles and more workers: the largest need is looked for
        for (int n = 1; n <= JL_TREE_MAX_NODES; ++n) {
            size_t bytes = 0;
            a.max_nodes = n;
            JL_TRY(tree::tree_attention_workspace(a, &bytes));
            t->workspace_bytes = std::max(t->workspace_bytes, bytes);
        }
        if (cudaMalloc(&t->dev, sizeof(TreeBuffers::Desc)) != cudaSuccess ||
            cudaMallocHost(&t->host, sizeof(TreeBuffers::Desc)) != cudaSuccess ||
            (t->workspace_bytes && cudaMalloc(&t->workspace, t->workspace_bytes) != cudaSuccess)) {
            cudaGetLastError();
            set_error("cannot allocate %zu bytes for tree passes", t->workspace_bytes + sizeof(TreeBuffers::Desc));
            return JL_ERR_OOM;
        }
        m->tree = t.release();
    }
    *out = m->tree;
    return JL_OK;
}

// Rows 16 k .. of a pass of n rows as a pass of their own: header 1 + k, which
// holds their number.
PassCtx chunk_of(const PassCtx& c, int k, int n) {
    const int rows = std::min(SMALL_M, n - k * SMALL_M);
    PassCtx x{c.m, c.stream, rows, rows};
    x.view = c.m->pass;
    x.view.hdr += 1 + k;
    x.view.head_row += k * SMALL_M;
    x.view.out_ids += k * SMALL_M;
    return x;
}

// One projection of every row: 16 rows at a time on the tensor cores, or as the
// other passes run it.
template <typename Other>
jl_status project_rows(const PassCtx& c, int n, const MxProj& p, int epi, const float* x, int ldx, float* y, int ldy, Other other) {
    if (!p.a) return other();
    for (int k = 0; k * SMALL_M < n; ++k)
        JL_TRY(mx_project(chunk_of(c, k, n), p, epi, 0, x + (size_t)k * SMALL_M * ldx, ldx, nullptr,
                          y + (size_t)k * SMALL_M * ldy, ldy));
    return JL_OK;
}

jl_status record_tree_pass(jl_model* m, const jl_cache* c, const TreeBuffers& t, int n) {
    tl_begin_pass();
    const PassCtx ctx{m, m->stream, n, n};
    const int h = m->hidden, qw = m->q_heads * HEAD, ld = qkv_ld(m);
    jl_norm_rope r{};
    r.rows = n;
    r.q_heads = m->q_heads;
    r.dtype = JL_KV_F32;
    r.qkv = r.q = m->s.qkv;
    r.qkv_ld = r.q_ld = (size_t)ld;
    r.eps = 1e-6f;
    r.rope = (const float*)m->rope;
    r.positions = m->max_positions;
    r.pos = t.dev->pos;
    r.slot = t.dev->slot;
    r.page_table = c->d_pages;
    r.seqs = 1;
    r.max_pages = (int)c->max_pages;
    r.status = m->counters;
    jl_tree_attn a{};
    a.rows = n;
    a.q_heads = m->q_heads;
    a.dtype = JL_KV_F32;
    a.q = m->s.qkv;
    a.q_ld = (size_t)ld;
    a.out = m->s.attn;
    a.out_ld = (size_t)qw;
    a.seqs = 1;
    a.max_nodes = n;
    a.row_start = t.dev->start;
    a.ctx = &t.dev->ctx;
    a.mask = &t.dev->mask[0][0];
    a.mask_words = MASK_WORDS;
    a.page_table = c->d_pages;
    a.max_pages = (int)((c->len + n + PAGE - 1) / PAGE);  // one sequence: the table has one row
    a.workspace = t.workspace;
    a.workspace_bytes = t.workspace_bytes;
    a.status = m->counters;
    JL_TRY(launch_embed(ctx));
    for (int l = 0; l < m->layers; ++l) {
        const LayerW& L = m->lw[l];
        JL_TRY(launch_rmsnorm(ctx, m->s.x, L.in_ln, m->s.xn, false));
        JL_TRY(project_rows(ctx, n, L.mx_qkv, MXE_STORE, m->s.xn, h, m->s.qkv, ld, [&] { return launch_qkv(ctx, L); }));
        r.pool = a.pool = pages_of(m, l, 1);
        r.q_norm = L.q_norm;
        r.k_norm = L.k_norm;
        JL_TRY(qk_norm_rope(r, m->stream));
        JL_TRY(tree::tree_attention(a, m->stream));
        JL_TRY(project_rows(ctx, n, L.mx_o, MXE_ADD, m->s.attn, qw, m->s.x, h, [&] { return launch_o(ctx, L); }));
        JL_TRY(launch_rmsnorm(ctx, m->s.x, L.post_ln, m->s.xn, false));
        JL_TRY(project_rows(ctx, n, L.mx_gateup, MXE_SWIGLU, m->s.xn, h, m->s.act, m->inter, [&] { return launch_gateup(ctx, L); }));
        JL_TRY(project_rows(ctx, n, L.mx_down, MXE_ADD, m->s.act, m->inter, m->s.x, h, [&] { return launch_down(ctx, L); }));
    }
    if (m->bf_head.a) {
        for (int k = 0; k * SMALL_M < n; ++k)
            JL_TRY(mx_head_fused(chunk_of(ctx, k, n), m->bf_head, m->final_norm,
                                 m->s.logits + (size_t)k * SMALL_M * m->vocab, m->vocab));
        return JL_OK;
    }
    JL_TRY(launch_rmsnorm(ctx, m->s.x, m->final_norm, m->s.xh, true));
    JL_TRY(project_rows(ctx, n, m->mx_head, MXE_STORE, m->s.xh, h, m->s.logits, m->vocab, [&] { return launch_head(ctx); }));
    return launch_argmax(ctx);
}

}  // namespace

jl_status predict_tree(jl_model* m, jl_cache* c, const uint32_t* ids, const int32_t* parents, size_t n, uint32_t* out_ids,
                       float* out_logits) {
    const size_t most = std::min<size_t>(JL_TREE_MAX_NODES, (size_t)m->max_rows);
    if (n < 1 || n > most || c->len + n > (size_t)m->max_positions) {
        set_error("a tree has 1..%zu nodes within the context (%zu of %d positions are taken), got %zu", most, c->len,
                  m->max_positions, n);
        return JL_ERR_INVALID_ARG;
    }
    for (size_t i = 0; i < n; ++i)
        if (parents[i] < -1 || parents[i] >= (int32_t)i) {
            set_error("node %zu: its parent must be -1 or an earlier node, got %d", i, parents[i]);
            return JL_ERR_INVALID_ARG;
        }
    JL_TRY(check_ids(m, ids, n));
    JL_CUDA(cudaSetDevice(m->device));
    TreeBuffers* t = nullptr;
    JL_TRY(tree_buffers(m, &t));
    JL_TRY(cache_reserve(c, c->len + n, m->stream));
    c->tree.clear();  // the nodes of an earlier tree are overwritten
    // positions, slots and masks
    TreeBuffers::Desc& d = *t->host;
    for (size_t i = 0; i < n; ++i) {
        const int32_t p = parents[i];
        d.pos[i] = p < 0 ? (int32_t)c->len : d.pos[p] + 1;
        d.slot[i] = (int32_t)(c->len + i);
        for (int w = 0; w < MASK_WORDS; ++w) d.mask[i][w] = p < 0 ? 0 : d.mask[p][w];
        d.mask[i][i / 64] |= 1ull << (i % 64);
    }
    d.start[0] = 0;
    d.start[1] = (int32_t)n;
    d.ctx = (int32_t)c->len;
    StageSlot* sl = nullptr;
    JL_TRY(stage_begin(m, &sl));
    const int chunks = (int)((n + SMALL_M - 1) / SMALL_M);
    static_assert(1 + JL_TREE_MAX_NODES / SMALL_M <= MAX_CHUNKS, "a header for the pass and one for each 16 rows");
    for (int k = 0; k <= chunks; ++k) {
        const int rows = k == 0 ? (int)n : std::min(SMALL_M, (int)n - (k - 1) * SMALL_M);
        sl->hdr[k] = PassHdr{rows, rows, 0, 0};
    }
    for (size_t i = 0; i < n; ++i) {
        sl->row[i] = RowDesc{ids[i], 0, d.pos[i], 0};
        sl->head_row[i] = (int32_t)i;
    }
    sl->page_table[0] = c->d_pages;
    cudaStream_t st = m->stream;
    auto queue = [&]() -> jl_status {
        JL_CUDA(cudaMemcpyAsync(m->pass.hdr, sl->hdr, (1 + chunks) * sizeof(PassHdr), cudaMemcpyHostToDevice, st));
        JL_CUDA(cudaMemcpyAsync(m->pass.row, sl->row, n * sizeof(RowDesc), cudaMemcpyHostToDevice, st));
        JL_CUDA(cudaMemcpyAsync(m->pass.head_row, sl->head_row, n * sizeof(int32_t), cudaMemcpyHostToDevice, st));
        JL_CUDA(cudaMemcpyAsync(m->pass.page_table, sl->page_table, sizeof(int32_t*), cudaMemcpyHostToDevice, st));
        JL_CUDA(cudaMemcpyAsync(t->dev, t->host, sizeof(TreeBuffers::Desc), cudaMemcpyHostToDevice, st));
        JL_TRY(stage_end(m, sl, st));
        JL_TRY(record_tree_pass(m, c, *t, (int)n));
        JL_CUDA(cudaMemcpyAsync(m->host_out, m->pass.out_ids, n * sizeof(uint32_t), cudaMemcpyDeviceToHost, st));
        if (out_logits)
            JL_CUDA(cudaMemcpyAsync(out_logits, m->s.logits, n * m->vocab * sizeof(float), cudaMemcpyDeviceToHost, st));
        return JL_OK;
    };
    // Also after an error: what was queued reads t->host and writes the caller's logits.
    const jl_status rs = queue();
    const cudaError_t done = cudaStreamSynchronize(st);
    JL_TRY(rs);
    JL_CUDA(done);
    JL_TRY(check_device_flag(m));
    memcpy(out_ids, m->host_out, n * sizeof(uint32_t));
    c->tree.assign(parents, parents + n);
    return JL_OK;
}

jl_status cache_compact(jl_cache* c, const uint32_t* path, size_t n) {
    if (n > c->tree.size()) {
        set_error("a path of %zu nodes: the cache's last pass was a tree of %zu", n, c->tree.size());
        return JL_ERR_INVALID_ARG;
    }
    bool moves = false;
    for (size_t i = 0; i < n; ++i) {
        const int32_t want = i ? (int32_t)path[i - 1] : -1;
        if (path[i] >= c->tree.size() || c->tree[path[i]] != want) {
            set_error("path entry %zu (node %u) is no child of the entry before it", i, path[i]);
            return JL_ERR_INVALID_ARG;
        }
        moves |= path[i] != i;
    }
    jl_model* m = c->m;
    if (moves) {
        JL_CUDA(cudaSetDevice(m->device));
        TreeBuffers* t = nullptr;
        JL_TRY(tree_buffers(m, &t));
        TreeBuffers::Desc& d = *t->host;
        std::copy(path, path + n, d.path);
        d.path_len = (int32_t)n;
        d.ctx = (int32_t)c->len;
        JL_CUDA(cudaMemcpyAsync(t->dev, t->host, sizeof d, cudaMemcpyHostToDevice, m->stream));
        jl_kv_compaction k{};
        k.pool = pages_of(m, 0, m->layers);
        k.seqs = 1;
        k.ctx = &t->dev->ctx;
        k.path = t->dev->path;
        k.path_ld = (int)n;
        k.path_len = &t->dev->path_len;
        k.page_table = c->d_pages;
        k.max_pages = (int)c->max_pages;
        k.status = m->counters;
        const jl_status rs = kv_compact(k, m->stream);
        JL_CUDA(cudaStreamSynchronize(m->stream));
        JL_TRY(rs);
        JL_TRY(check_device_flag(m));
    }
    c->len += n;
    c->tree.clear();
    return JL_OK;
}

jl_status cache_fork(jl_cache* c, size_t len, jl_cache** out) {
    jl_model* m = c->m;
    const size_t full = len / PAGE, rest = len % PAGE;
    JL_CUDA(cudaSetDevice(m->device));
    if (rest && m->kv.free_list.empty()) {
        set_error("KV pool exhausted: a fork inside a page needs 1 more page, 0 free (raise kv_pool_tokens)");
        return JL_ERR_OOM;
    }
    jl_cache* f = nullptr;
    JL_TRY(cache_create(m, &f));
    std::unique_ptr<jl_cache, void (*)(jl_cache*)> guard(f, cache_free);
    for (size_t i = 0; i < full; ++i) {
        f->pages.push_back(c->pages[i]);
        ++m->kv.refs[c->pages[i]];
    }
    if (rest) {
        const int32_t src = c->pages[full], rows = (int32_t)rest;
        int32_t dst = 0;
        JL_TRY(page_take(m, &dst));
        f->pages.push_back(dst);
        JL_TRY(kv_copy_pages(pages_of(m, 0, m->layers), &src, &dst, &rows, 1, m->stream));
    }
    std::copy(f->pages.begin(), f->pages.end(), f->h_pages);
    if (!f->pages.empty())
        JL_CUDA(cudaMemcpyAsync(f->d_pages, f->h_pages, f->pages.size() * sizeof(int32_t), cudaMemcpyHostToDevice, m->stream));
    JL_CUDA(cudaStreamSynchronize(m->stream));
    f->len = len;
    *out = guard.release();
    return JL_OK;
}

// A page of its own for the cache, in place of pages[i] that others hold too: its
// first `rows` rows are copied, and the others keep the old page.
jl_status page_unshare(jl_cache* c, size_t i, size_t rows, cudaStream_t stream) {
    jl_model* m = c->m;
    int32_t src = c->pages[i], dst = 0;
    JL_TRY(page_take(m, &dst));
    auto queue = [&]() -> jl_status {
        const int32_t r = (int32_t)rows;
        if (rows) JL_TRY(kv_copy_pages(pages_of(m, 0, m->layers), &src, &dst, &r, 1, stream));
        c->h_pages[i] = dst;
        JL_CUDA(cudaMemcpyAsync(c->d_pages + i, c->h_pages + i, sizeof(int32_t), cudaMemcpyHostToDevice, stream));
        return JL_OK;
    };
    const jl_status rs = queue();
    // After an error the device's table still names the shared page, and so must the cache.
    if (rs != JL_OK) c->h_pages[i] = src;
    c->pages[i] = c->h_pages[i];
    page_release(m, rs == JL_OK ? src : dst);
    return rs;
}

}  // namespace jl
