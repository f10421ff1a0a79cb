// Drafted tokens: the kernels around their attention (lbk_attn_tree.cu).
//
//   embed_tree         rows of the embedding table for the nodes
//   rope_append_tree   queries and keys turned by their node's DEPTH (position pos + number of ancestors), keys and values
//                      appended as bf16 at the node's PLACE (row pos + i)
//   tree_accept        the greedy walk: node 0, then the child whose token is the best one of its parent's row
//   kv_keep_path       the rows of the accepted nodes moved together behind the committed ones, in all layers
//   advance_by         positions moved by the accepted nodes
//   advance_path       the same for the sequences whose path kv_keep_path takes
//
// A decode step of one token is the tree with one node: the same rows of the cache, the same rotation
// (crates/lb-model/src/model.rs:295-303, 334-347). Everything is read from device memory, so a step can be recorded once.
#include "lbk_dense_dev.cuh"
#include "lbk_tree.cuh"

namespace lbk {

namespace {

// One block per node place. A place that is not in use may hold anything as its token (a batch is padded with -1, or with what was there): its row is token 0's, a number that
// the rows of a pass can work with. So is that of a token outside the vocabulary, and the host hears of it. Rows as embed_kernel (lbk_decoder.cu) copies them.
// UNITS: values by four.
template <bool UNITS>
__global__ void embed_tree_kernel(const uint16_t *__restrict__ table, int vocab, const int *__restrict__ tokens, const int *__restrict__ counts, int t, int hidden, float *__restrict__ out,
                                  int *err_word) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int row = blockIdx.x;
    int token = tokens[row];
    if (counts && row % t >= tree_count(counts, row / t, t)) token = 0;
    if (static_cast<unsigned>(token) >= static_cast<unsigned>(vocab)) {
        if (threadIdx.x == 0) atomicExch(err_word, kErrTree);
        token = 0;
    }
    const uint16_t *from = table + static_cast<size_t>(token) * hidden;
    float *to = out + static_cast<size_t>(row) * hidden;
    if (UNITS) {
        for (int i = threadIdx.x; i < hidden >> 2; i += blockDim.x) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(from) + i);
            reinterpret_cast<float4 *>(to)[i] = make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
        }
        return;
    }
    for (int i = threadIdx.x; i < hidden; i += blockDim.x) to[i] = __uint_as_float(static_cast<uint32_t>(from[i]) << 16);
}

// x * cos + other * sin with the rounding of the prompt pass (lbk_decoder.cu): the product with sin rounded, the rest in one step
__device__ __forceinline__ float turned(float x, float c, float other, float s) { return __fmaf_rn(x, c, __fmul_rn(other, s)); }

// One block per node. A thread takes four dimensions of each half of a head at a time, so that loads and stores are 16 bytes, and asks for kItems of them, queries, keys
// and values, before the node's depth is known. Bound by launch and two dependent trips to memory up to some hundred nodes, then by bytes: 16 x 61 nodes of 32 + 8 heads,
// 45 MB, 9.5 us (4.7 TB/s).
// VEC: head_dim is a multiple of 8 and every buffer lies on 16 bytes.
constexpr int kItems = 3;
template <bool VEC>
__global__ void __launch_bounds__(256) rope_append_tree_kernel(float *__restrict__ q, const float *__restrict__ k, const float *__restrict__ v,
                                                               const float *__restrict__ cos_t, const float *__restrict__ sin_t, const int *__restrict__ pos_dev,
                                                               const int *__restrict__ parents, const int *__restrict__ counts, int t, int nh, int kvh, int hd, int cap,
                                                               uint16_t *__restrict__ kcache, uint16_t *__restrict__ vcache, int *err_word) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    __shared__ int s_parent[kTreeNodes];
    const int row = blockIdx.x, seq = row / t, node = row - seq * t, half = hd >> 1, tid = threadIdx.x;
    const int quarter = half >> 2, first = blockIdx.y * blockDim.x * kItems + tid;  // VEC: a head has that many items
    auto ld = [](const float *at) { return *reinterpret_cast<const float4 *>(at); };
    float4 a[kItems], b[kItems], va[kItems], vb[kItems];
    int head[kItems], dim[kItems];
    if (VEC)
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
            const int it = first + e * blockDim.x;
            head[e] = it / quarter;
            dim[e] = (it - head[e] * quarter) * 4;
            if (head[e] >= nh + kvh) continue;
            const float *src = head[e] >= nh ? k + (static_cast<size_t>(row) * kvh + head[e] - nh) * hd : q + (static_cast<size_t>(row) * nh + head[e]) * hd;
            a[e] = ld(src + dim[e]);
            b[e] = ld(src + dim[e] + half);
            if (head[e] >= nh) {
                const float *vv = v + (static_cast<size_t>(row) * kvh + head[e] - nh) * hd;
                va[e] = ld(vv + dim[e]);
                vb[e] = ld(vv + dim[e] + half);
            }
        }
    const int pos = pos_dev[seq], count = tree_count(counts, seq, t);
    bool wrong = false;
    for (int j = tid; j < count; j += blockDim.x) {
        const int p = parents[static_cast<size_t>(seq) * t + j];
        s_parent[j] = p;
        wrong |= p < -1 || p >= j;
    }
    if (__syncthreads_or(wrong)) {
        if (tid == 0) atomicExch(err_word, kErrTree);
        return;
    }
    if (!tree_in_cache(pos, count, cap, err_word) || node >= count) return;
    int depth = 0;
    for (int p = s_parent[node]; p >= 0; p = s_parent[p]) ++depth;  // ends: a parent lies in front of its child
    const float *c = cos_t + static_cast<size_t>(pos + depth) * hd, *s = sin_t + static_cast<size_t>(pos + depth) * hd;
    if (VEC) {
#pragma unroll
        for (int e = 0; e < kItems; ++e) {
            const int h = head[e], i = dim[e];
            if (h >= nh + kvh) continue;
            const float4 c1 = ld(c + i), c2 = ld(c + i + half), s1 = ld(s + i), s2 = ld(s + i + half), x = a[e], y = b[e];
            const float4 lo = make_float4(turned(x.x, c1.x, -y.x, s1.x), turned(x.y, c1.y, -y.y, s1.y), turned(x.z, c1.z, -y.z, s1.z), turned(x.w, c1.w, -y.w, s1.w));
            const float4 hi = make_float4(turned(y.x, c2.x, x.x, s2.x), turned(y.y, c2.y, x.y, s2.y), turned(y.z, c2.z, x.z, s2.z), turned(y.w, c2.w, x.w, s2.w));
            if (h < nh) {
                float *dst = q + (static_cast<size_t>(row) * nh + h) * hd;
                *reinterpret_cast<float4 *>(dst + i) = lo;
                *reinterpret_cast<float4 *>(dst + i + half) = hi;
                continue;
            }
            const size_t slot = ((static_cast<size_t>(seq) * kvh + h - nh) * cap + pos + node) * hd;
            dense::put4(kcache + slot + i, lo);
            dense::put4(kcache + slot + i + half, hi);
            dense::put4(vcache + slot + i, va[e]);
            dense::put4(vcache + slot + i + half, vb[e]);
        }
        return;
    }
    for (int e = tid; e < (nh + kvh) * half; e += blockDim.x) {
        const int hh = e / half, d = e - hh * half;
        if (hh < nh) {
            float *qh = q + (static_cast<size_t>(row) * nh + hh) * hd;
            const float x1 = qh[d], x2 = qh[d + half];
            qh[d] = turned(x1, c[d], -x2, s[d]);
            qh[d + half] = turned(x2, c[d + half], x1, s[d + half]);
        } else {
            const float *kk = k + (static_cast<size_t>(row) * kvh + hh - nh) * hd, *vv = v + (static_cast<size_t>(row) * kvh + hh - nh) * hd;
            const size_t slot = ((static_cast<size_t>(seq) * kvh + hh - nh) * cap + pos + node) * hd;
            const float x1 = kk[d], x2 = kk[d + half];
            kcache[slot + d] = dense::f32_bf16(turned(x1, c[d], -x2, s[d]));
            kcache[slot + d + half] = dense::f32_bf16(turned(x2, c[d + half], x1, s[d + half]));
            vcache[slot + d] = dense::f32_bf16(vv[d]);
            vcache[slot + d + half] = dense::f32_bf16(vv[d + half]);
        }
    }
}

// One block per sequence, a thread a node: every node that fits its parent's best token bids for being what follows it, the lowest wins, and one thread walks along what
// is left: 64 accepted nodes 7.2 -> 3.2 us against a warp that looks at all nodes in every step.
__global__ void __launch_bounds__(kTreeNodes) tree_accept_kernel(const int *__restrict__ tokens, const int *__restrict__ parents, const int *__restrict__ best,
                                                                 const int *__restrict__ counts, int t, int *__restrict__ path, int *__restrict__ count_out,
                                                                 int *__restrict__ next, int *err_word) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    __shared__ int s_best[kTreeNodes], s_follow[kTreeNodes], s_path[kTreeNodes], s_n;
    const int seq = blockIdx.x, i = threadIdx.x, count = tree_count(counts, seq, t);
    const size_t at = static_cast<size_t>(seq) * t;
    const bool mine = i < count;
    const int tok = mine ? tokens[at + i] : 0, par = mine ? parents[at + i] : -1;
    s_best[i] = mine ? best[at + i] : 0;
    s_follow[i] = kTreeNodes;
    if (__syncthreads_or(par < -1 || (mine && par >= i))) {
        if (i == 0) atomicExch(err_word, kErrTree);
        if (i == 0) s_n = 0;
    } else {
        if (par >= 0 && tok == s_best[par]) atomicMin(&s_follow[par], i);
        __syncthreads();
        if (i == 0) {
            int n = 0;
            for (int node = count ? 0 : kTreeNodes; node < kTreeNodes; node = s_follow[node]) s_path[n++] = node;  // ends: what follows lies behind
            s_n = n;
        }
    }
    __syncthreads();
    const int n = s_n;
    if (i < t) path[at + i] = i < n ? s_path[i] : -1;
    if (i == 0) {
        count_out[seq] = n;
        next[seq] = n ? s_best[s_path[n - 1]] : -1;
    }
}

// Whether a path is wrong at place j: it ascends, inside the tree
__device__ __forceinline__ bool path_wrong(const int *__restrict__ path, int j, int t) {
    const int from = path[j];
    return from < j || from >= t || (j > 0 && from <= path[j - 1]);
}

// One block per sequence and kPlanes of its (layer, KV head, keys or values), 16 bytes a thread and row: the accepted nodes of a step are a few rows of 256 bytes
// each, and a block for each plane was launch and waiting (16 sequences, 30 layers of 5 heads, 8 rows, 20 MB: 8.4 -> 5.8 us). Rows move down only (path[j] >= j,
// ascending), so portions in ascending order, each read before it is written, never overwrite a row that is still wanted.
constexpr int kPlanes = 8, kHeld = 8;  // 16-byte units a thread holds
__global__ void __launch_bounds__(128) kv_keep_path_kernel(uint4 *kcache, uint4 *vcache, size_t layer_units, int planes, int heads, int units, int shift, int cap, const int *__restrict__ pos_dev,
                                                           const int *__restrict__ path, const int *__restrict__ counts, int t, int *err_word) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    __shared__ int s_path[kTreeNodes];
    __shared__ uint4 *s_rows[kPlanes];
    __shared__ int s_count, s_pos;
    const int seq = blockIdx.y, tid = threadIdx.x, plane0 = blockIdx.x * kPlanes;
    if (tid == 0) {  // one thread reads, so that all take the same way, whatever happens to the positions meanwhile
        s_count = tree_count(counts, seq, t);
        s_pos = pos_dev[seq];
    }
    __syncthreads();
    const int count = s_count, pos = s_pos;
    if (tid < kPlanes) {
        const int layer = (plane0 + tid) / (2 * heads), rest = plane0 + tid - layer * 2 * heads;
        s_rows[tid] = (rest & 1 ? vcache : kcache) + static_cast<size_t>(layer) * layer_units + ((static_cast<size_t>(seq) * heads + (rest >> 1)) * cap + pos) * units;
    }
    bool wrong = false;
    for (int j = tid; j < count; j += blockDim.x) {
        s_path[j] = path[static_cast<size_t>(seq) * t + j];
        wrong |= path_wrong(path + static_cast<size_t>(seq) * t, j, t);
    }
    if (__syncthreads_or(wrong)) {
        if (tid == 0) atomicExch(err_word, kErrTree);
        return;
    }
    if (!count || !tree_in_cache(pos, s_path[count - 1] + 1, cap, err_word)) return;
    int first = 0;
    while (first < count && s_path[first] == first) ++first;  // these lie where they belong
    const int n = (count - first) * units, all = min(kPlanes, planes - plane0) * n;
    for (int base = 0; base < all; base += kHeld * 128) {
        uint4 held[kHeld], *to[kHeld];
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int i = base + e * 128 + tid;
            if (i >= all) continue;
            int plane = 0;
#pragma unroll
            for (int k = 1; k < kPlanes; ++k) plane += i >= k * n;
            const int in = i - plane * n, j = shift >= 0 ? in >> shift : in / units;
            uint4 *const at = s_rows[plane];
            held[e] = at[static_cast<size_t>(s_path[first + j]) * units + in - j * units];
            to[e] = at + static_cast<size_t>(first) * units + in;
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kHeld; ++e)
            if (base + e * 128 + tid < all) *to[e] = held[e];
        __syncthreads();
    }
}

__global__ void advance_by_kernel(int *pos, const int *__restrict__ count, int n) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    // a position that was refused stays refused (advance_pos_kernel)
    if (i < n && count[i] > 0 && pos[i] < (1 << 30)) pos[i] += min(count[i], kTreeNodes);
}

// A warp a sequence. What kv_keep_path leaves as it was keeps its position too: rows that have not been moved are none of the sequence's.
constexpr int kAdvanceWarps = 4;
__global__ void __launch_bounds__(kAdvanceWarps * 32) advance_path_kernel(int *pos, const int *__restrict__ path, const int *__restrict__ counts, int b, int t, int cap, int *err_word) {
    ptx::pdl_trigger();
    ptx::pdl_wait();
    const int seq = blockIdx.x * kAdvanceWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (seq >= b) return;
    const int count = tree_count(counts, seq, t), *own = path + static_cast<size_t>(seq) * t;
    bool wrong = false;
    for (int j = lane; j < count; j += 32) wrong |= path_wrong(own, j, t);
    wrong = __any_sync(0xffffffffu, wrong);
    if (lane || !count) return;
    const int at = pos[seq];
    if (wrong || at < 0 || at > cap - (own[count - 1] + 1)) atomicExch(err_word, wrong ? kErrTree : kErrPos);
    else pos[seq] = at + count;
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

int lbk_embed_tree_bf16(lbk_ctx *c, const uint16_t *table_dev, size_t vocab, const int32_t *tokens_dev, const int32_t *counts_dev, size_t b, size_t t, size_t hidden, float *out_dev,
                        void *stream) {
    LBK_TREE_PRE("lbk_embed_tree_bf16");
    if (b == 0 || t == 0) return LBK_OK;
    if (!table_dev || !tokens_dev || !out_dev) return fail(LBK_ERR_INVALID, "lbk_embed_tree_bf16: null buffer");
    if (t > LBK_TREE_NODES) return fail(LBK_ERR_UNSUPPORTED, "a tree has at most %d nodes (got %zu)", LBK_TREE_NODES, t);
    if (!vocab || !hidden || vocab > INT32_MAX || hidden > INT32_MAX) return fail(LBK_ERR_SHAPE, "lbk_embed_tree_bf16: %zu rows of %zu values", vocab, hidden);
    if (b * t > INT32_MAX) return fail(LBK_ERR_UNSUPPORTED, "lbk_embed_tree_bf16: more rows than 2^31");
    // units and threads as lbk_embed_bf16 has them
    const bool units = hidden >= 512 && hidden % 4 == 0 && (reinterpret_cast<uintptr_t>(table_dev) & 7) == 0 && (reinterpret_cast<uintptr_t>(out_dev) & 15) == 0;
    const unsigned threads = !units ? 256 : b * t <= 3 * static_cast<size_t>(ctx->sm_count) ? 512 : 128;
    LBK_CUDA(launch_chained(units ? embed_tree_kernel<true> : embed_tree_kernel<false>, dim3(static_cast<unsigned>(b * t)), dim3(threads), 0, st, table_dev, static_cast<int>(vocab), tokens_dev,
                            counts_dev, static_cast<int>(t), static_cast<int>(hidden), out_dev, ctx->err_word));
    ctx->launches++;
    return LBK_OK;
}

int lbk_rope_kv_append_tree(lbk_ctx *c, float *q_dev, const float *k_dev, const float *v_dev, const float *cos_dev, const float *sin_dev, const int32_t *pos_dev,
                            const int32_t *parents_dev, const int32_t *counts_dev, size_t b, size_t t, size_t n_heads, size_t kv_heads, size_t head_dim, size_t cap,
                            uint16_t *kcache_dev, uint16_t *vcache_dev, void *stream) {
    LBK_TREE_PRE("lbk_rope_kv_append_tree");
    if (b == 0 || t == 0) return LBK_OK;
    if (!q_dev || !k_dev || !v_dev || !cos_dev || !sin_dev || !pos_dev || !parents_dev || !kcache_dev || !vcache_dev)
        return fail(LBK_ERR_INVALID, "lbk_rope_kv_append_tree: null buffer");
    if (t > LBK_TREE_NODES) return fail(LBK_ERR_UNSUPPORTED, "a tree has at most %d nodes (got %zu)", LBK_TREE_NODES, t);
    if (!n_heads || !kv_heads || !head_dim || head_dim % 2 || n_heads + kv_heads > (1u << 20) || head_dim > 1024)
        return fail(LBK_ERR_SHAPE, "lbk_rope_kv_append_tree: %zu and %zu heads of %zu (an even number, at most 1024)", n_heads, kv_heads, head_dim);
    if (cap > INT32_MAX || b * t > INT32_MAX) return fail(LBK_ERR_UNSUPPORTED, "lbk_rope_kv_append_tree: more rows than 2^31");
    const uintptr_t all = reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(k_dev) | reinterpret_cast<uintptr_t>(v_dev) | reinterpret_cast<uintptr_t>(cos_dev) |
                          reinterpret_cast<uintptr_t>(sin_dev) | reinterpret_cast<uintptr_t>(kcache_dev) | reinterpret_cast<uintptr_t>(vcache_dev);
    const bool vec = head_dim % 8 == 0 && (all & 15) == 0;
    const size_t items = (n_heads + kv_heads) * head_dim / (vec ? 8 : 2);
    const unsigned threads = items < 256 ? static_cast<unsigned>((items + 31) / 32 * 32) : 256;
    const dim3 grid(static_cast<unsigned>(b * t), static_cast<unsigned>(vec ? (items + kItems * threads - 1) / (kItems * threads) : 1));
    if (grid.y > 65535) return fail(LBK_ERR_UNSUPPORTED, "lbk_rope_kv_append_tree: %zu heads of %zu", n_heads + kv_heads, head_dim);
    LBK_CUDA(launch_chained(vec ? rope_append_tree_kernel<true> : rope_append_tree_kernel<false>, grid, dim3(threads), 0, st, q_dev, k_dev, v_dev, cos_dev, sin_dev, pos_dev, parents_dev,
                            counts_dev, static_cast<int>(t), static_cast<int>(n_heads), static_cast<int>(kv_heads), static_cast<int>(head_dim), static_cast<int>(cap), kcache_dev,
                            vcache_dev, ctx->err_word));
    ctx->launches++;
    return LBK_OK;
}

int lbk_tree_accept(lbk_ctx *c, const int32_t *tokens_dev, const int32_t *parents_dev, const int32_t *best_dev, const int32_t *counts_dev, size_t b, size_t t,
                    int32_t *path_dev, int32_t *count_out_dev, int32_t *next_dev, void *stream) {
    LBK_TREE_PRE("lbk_tree_accept");
    if (b == 0) return LBK_OK;
    if (!tokens_dev || !parents_dev || !best_dev || !path_dev || !count_out_dev || !next_dev) return fail(LBK_ERR_INVALID, "lbk_tree_accept: null buffer");
    if (t == 0 || t > LBK_TREE_NODES) return fail(LBK_ERR_UNSUPPORTED, "a tree has 1 to %d nodes (got %zu)", LBK_TREE_NODES, t);
    if (b > INT32_MAX) return fail(LBK_ERR_UNSUPPORTED, "lbk_tree_accept: more sequences than 2^31");
    LBK_CUDA(launch_chained(tree_accept_kernel, dim3(static_cast<unsigned>(b)), dim3(kTreeNodes), 0, st, tokens_dev, parents_dev, best_dev, counts_dev, static_cast<int>(t), path_dev, count_out_dev,
                            next_dev, ctx->err_word));
    ctx->launches++;
    return LBK_OK;
}

int lbk_kv_keep_path(lbk_ctx *c, uint16_t *kcache_dev, uint16_t *vcache_dev, size_t layers, size_t layer_elems, size_t b, size_t kv_heads, size_t head_dim, size_t cap,
                     const int32_t *pos_dev, const int32_t *path_dev, const int32_t *count_dev, size_t t, void *stream) {
    LBK_TREE_PRE("lbk_kv_keep_path");
    if (b == 0 || layers == 0) return LBK_OK;
    if (!kcache_dev || !vcache_dev || !pos_dev || !path_dev || !count_dev) return fail(LBK_ERR_INVALID, "lbk_kv_keep_path: null buffer");
    if (t == 0 || t > LBK_TREE_NODES) return fail(LBK_ERR_UNSUPPORTED, "a tree has 1 to %d nodes (got %zu)", LBK_TREE_NODES, t);
    if (!kv_heads || !head_dim || head_dim % 8 || layer_elems % 8 || ((reinterpret_cast<uintptr_t>(kcache_dev) | reinterpret_cast<uintptr_t>(vcache_dev)) & 15))
        return fail(LBK_ERR_SHAPE, "lbk_kv_keep_path: head_dim and layer_elems are multiples of 8, the caches lie on 16 bytes");
    if (layers > 1 && layer_elems < b * kv_heads * cap * head_dim) return fail(LBK_ERR_SHAPE, "lbk_kv_keep_path: layers of %zu elements overlap", layer_elems);
    if (cap > INT32_MAX || b > 65535 || layers * kv_heads * 2 > INT32_MAX || head_dim > 8192) return fail(LBK_ERR_UNSUPPORTED, "lbk_kv_keep_path: at most 65535 sequences and 2^31 rows");
    const size_t planes = layers * kv_heads * 2, units = head_dim / 8;
    const int shift = units & (units - 1) ? -1 : static_cast<int>(__builtin_ctzll(units));
    LBK_CUDA(launch_chained(kv_keep_path_kernel, dim3(static_cast<unsigned>((planes + kPlanes - 1) / kPlanes), static_cast<unsigned>(b)), dim3(128), 0, st, reinterpret_cast<uint4 *>(kcache_dev),
                            reinterpret_cast<uint4 *>(vcache_dev), layer_elems / 8, static_cast<int>(planes), static_cast<int>(kv_heads), static_cast<int>(head_dim / 8), shift, static_cast<int>(cap),
                            pos_dev, path_dev, count_dev, static_cast<int>(t), ctx->err_word));
    ctx->launches++;
    return LBK_OK;
}

int lbk_advance_pos_by(lbk_ctx *c, int32_t *pos_dev, const int32_t *count_dev, size_t b, void *stream) {
    LBK_TREE_PRE("lbk_advance_pos_by");
    if (b == 0) return LBK_OK;
    if (!pos_dev || !count_dev) return fail(LBK_ERR_INVALID, "lbk_advance_pos_by: null buffer");
    if (b > INT32_MAX) return fail(LBK_ERR_UNSUPPORTED, "lbk_advance_pos_by: more sequences than 2^31");
    LBK_CUDA(launch_chained(advance_by_kernel, dim3(static_cast<unsigned>((b + 127) / 128)), dim3(128), 0, st, pos_dev, count_dev, static_cast<int>(b)));
    ctx->launches++;
    return LBK_OK;
}

int lbk_advance_pos_path(lbk_ctx *c, int32_t *pos_dev, const int32_t *path_dev, const int32_t *count_dev, size_t b, size_t t, size_t cap, void *stream) {
    LBK_TREE_PRE("lbk_advance_pos_path");
    if (b == 0) return LBK_OK;
    if (!pos_dev || !path_dev || !count_dev) return fail(LBK_ERR_INVALID, "lbk_advance_pos_path: null buffer");
    if (t == 0 || t > LBK_TREE_NODES) return fail(LBK_ERR_UNSUPPORTED, "a tree has 1 to %d nodes (got %zu)", LBK_TREE_NODES, t);
    if (b > INT32_MAX || cap > INT32_MAX) return fail(LBK_ERR_UNSUPPORTED, "lbk_advance_pos_path: more than 2^31 sequences or rows");
    LBK_CUDA(launch_chained(advance_path_kernel, dim3(static_cast<unsigned>((b + kAdvanceWarps - 1) / kAdvanceWarps)), dim3(kAdvanceWarps * 32), 0, st, pos_dev, path_dev, count_dev,
                            static_cast<int>(b), static_cast<int>(t), static_cast<int>(cap), ctx->err_word));
    ctx->launches++;
    return LBK_OK;
}

}  // extern "C"
