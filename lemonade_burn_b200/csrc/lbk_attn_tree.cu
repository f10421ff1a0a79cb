// Attention of drafted tokens: the nodes of a tree over the committed rows of their sequence and their own ancestors.
//
//   o_i = sum_j p_ij V_j,  p_i = softmax_j(scale * q_i . K_j),  j < pos and j = pos + n for n = i and the ancestors of i
//
// The query heads that share a KV head and the nodes of a sequence are the rows of one problem (row = node * group + head of the group), so that
// the cache is read once for all of them. A problem's rows are cut into tiles, its keys into blocks; the (problem, tile, block) units of the whole batch stand in one
// line that is cut evenly among the CTAs, whatever the sequences' lengths (cut_line): a CTA takes neighbouring blocks of a tile, then of the
// next. A tile whose blocks went to one CTA is written out by it; of the others each CTA leaves the unnormalised sum, the maximum
// and the weight of its part in the scratch, and attn_tree_merge_kernel joins them.
//
// f32 queries and probabilities are three bf16 terms each (8 bits a term: an f32 has 24), keys and values are bf16 as they are: every product is exact, and
// what is left are f32 sums. Two terms, as in the decode and prompt kernels, are off by 2^-17 of a query or probability, which was 3 to 6 times
// the error of plain f32 arithmetic. A tensor core cuts its sums off instead of rounding them (2e-8 of a sum for 16 keys), so the products of a block of keys start from
// zero and are added to the row in registers, one rounded addition a block. bf16 queries are exact in one term; their results are rounded to bf16,
// 2^-8 of themselves at most, and so is a probability, whose roundings are of either sign and average out over the keys.
//
// Rows of V that nobody has written may hold anything, and 0 * NaN is NaN: values past the sequence's last node are taken as zeros. Values of OTHER
// branches may be infinite or NaN too; a row that does not see them must not notice. So in the blocks of the nodes values that are no numbers are
// taken as zeros as well, and added at the end to the rows that see them (a weight is never zero in exact arithmetic).
#include <algorithm>

#include "lbk_dense_dev.cuh"
#include "lbk_tcgen05.cuh"
#include "lbk_tree.cuh"

namespace lbk {

namespace {

using dense::bf16_pair;

constexpr int kHd = 128;
constexpr int kMaxSeqs = 256;
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr float kNoMax = -3.0e38f;  // a row that has seen nothing: finite, so that -inf scores less it are no NaN

struct TreeParams {
    CUtensorMap k, v;   // bytes [cache rows][256], boxes of 128 bytes and 64 rows (K of many rows: 128), SWIZZLE_128B
    const void *q;
    void *out;
    long q_pitch, out_pitch;
    const uint16_t *vcache;
    const int *pos, *parents, *counts;
    int b, t, nh, kvh, cap;
    float scale;        // log2(e) * scale: scores in units of log 2
    float *part;        // [CTA][2][tile rows][128]
    float2 *part_ml;    // [CTA][2][tile rows]: maximum, weight
    int workers;        // CTAs of the attention kernel
    unsigned per_group; // 2^32 / heads of a group, rounded up; 0 for one head
    int *err_word;
    __device__ __forceinline__ int node_of(int row) const { return per_group ? static_cast<int>(__umulhi(static_cast<unsigned>(row), per_group)) : row; }
};

__device__ __forceinline__ float ex2(float x) {  // 2^x, the hardware's approximation
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two values at once as bf16 terms: term[i] = bf16(x - the terms in front of it), and with three of them their sum is x
template <int TERMS>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&term)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        term[i] = bf16_pair(x0, x1);
        if (i + 1 < TERMS) {
            x0 -= __uint_as_float(term[i] << 16);
            x1 -= __uint_as_float(term[i] & 0xffff0000u);
        }
    }
}

// two bf16 with zeros in the place of what is no number
__device__ __forceinline__ uint32_t only_numbers(uint32_t x) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu;
    return x;
}

// ---- the line of units ----------------------------------------------------------------------------
struct Line {
    int first[kMaxSeqs + 1];   // units in front of a sequence; [b] is all of them
    int pos[kMaxSeqs], count[kMaxSeqs];
};
// A sequence: kv_heads * tiles problems of `blocks` units each.
__device__ __forceinline__ int line_blocks(const Line &l, int seq, int block_keys) { return (l.pos[seq] + l.count[seq] + block_keys - 1) / block_keys; }
__device__ __forceinline__ int line_tiles(const Line &l, int seq, int group, int rows) { return (l.count[seq] * group + rows - 1) / rows; }

// Fills the line; a sequence outside its cache has no units. All threads of the block. (Loads from L2: the merging kernel comes here in front of its wait.)
template <int ROWS, int KEYS>
__device__ void cut_line(const TreeParams &p, Line &l) {
    const int group = p.nh / p.kvh;
    for (int i = threadIdx.x; i < p.b; i += blockDim.x) {
        const int pos = __ldcg(p.pos + i), count = p.counts ? min(max(__ldcg(p.counts + i), 0), p.t) : p.t;
        const bool fits = pos >= 0 && pos <= p.cap - count;
        if (!fits && blockIdx.x == 0) atomicExch(p.err_word, kErrPos);
        l.pos[i] = pos;
        l.count[i] = fits ? count : 0;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int before = 0;
        for (int i0 = 0; i0 < p.b; i0 += 32) {
            const int i = i0 + threadIdx.x;
            const int mine = i < p.b && l.count[i] ? line_blocks(l, i, KEYS) * line_tiles(l, i, group, ROWS) * p.kvh : 0;
            int sum = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (static_cast<int>(threadIdx.x) >= o) sum += up;
            }
            if (i < p.b) l.first[i] = before + sum - mine;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (threadIdx.x == 0) l.first[p.b] = before;
    }
    __syncthreads();
}
// Worker w takes the units share_begin(w) .. share_begin(w + 1) - 1: `each` of them, one more the first `more` workers.
struct Shares {
    int each, more;
    __device__ __forceinline__ Shares(int units, int workers) : each(units / workers), more(units - units / workers * workers) {}
    __device__ __forceinline__ int begin(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int owner(int u) const { return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each; }
};

struct Segment {
    int seq, kh, tile;     // the problem
    int begin, end;        // its blocks
    int blocks;            // of all there are
};
__device__ __forceinline__ Segment segment_at(const TreeParams &p, const Line &l, int unit, int last, int rows, int keys) {
    Segment s;
    int lo = 0, hi = p.b - 1;   // the last sequence whose units begin at or before this one and that has any
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= unit) lo = mid;
        else hi = mid - 1;
    }
    s.seq = lo;
    s.blocks = line_blocks(l, lo, keys);
    const int tiles = line_tiles(l, lo, p.nh / p.kvh, rows), at = unit - l.first[lo], problem = at / s.blocks;
    s.begin = at - problem * s.blocks;
    s.end = min(s.blocks, s.begin + last - unit);
    s.kh = problem / tiles;
    s.tile = problem - s.kh * tiles;
    return s;
}

// Who sees whom: bit n of mask[i]. A parent that is none counts as -1.
__device__ __forceinline__ void tree_masks(const int *parent, ulonglong2 *mask, int i) {
    unsigned long long lo = 0, hi = 0;
    for (int n = i; n >= 0; n = parent[n]) {
        if (n < 64) lo |= 1ull << n;
        else hi |= 1ull << (n - 64);
    }
    mask[i] = make_ulonglong2(lo, hi);
}
// Parents into shared memory, those that are none as -1, by the first `threads` threads of the block.
__device__ __forceinline__ void load_parents(const TreeParams &p, int *parent, int seq, int count, int threads) {
    for (int i = threadIdx.x; i < count; i += threads) {
        const int up = p.parents[static_cast<size_t>(seq) * p.t + i];
        const bool good = up >= -1 && up < i;
        if (!good) atomicExch(p.err_word, kErrTree);
        parent[i] = good ? up : -1;
    }
}
// Four dimensions of a problem's query row (zeros past the last): f32, or the bits of four bf16 in x and y
template <int TERMS>
__device__ __forceinline__ float4 query(const TreeParams &p, int seq, int kh, int group, int row, int rows_all, int lane) {
    if (row >= rows_all) return make_float4(0.f, 0.f, 0.f, 0.f);
    const int node = p.node_of(row);
    const size_t at = (static_cast<size_t>(seq) * p.t + node) * p.q_pitch + (kh * group + row - node * group) * kHd + lane * 4;
    if (TERMS > 1) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p.q) + at);
    const float2 a = *reinterpret_cast<const float2 *>(static_cast<const uint16_t *>(p.q) + at);
    return make_float4(a.x, a.y, 0.f, 0.f);
}
template <int TERMS>
__device__ __forceinline__ void query_terms(const float4 &a, uint2 (&term)[TERMS]) {
    if (TERMS == 1) {
        term[0] = make_uint2(__float_as_uint(a.x), __float_as_uint(a.y));
        return;
    }
    uint32_t x01[TERMS], x23[TERMS];
    split_pair<TERMS>(a.x, a.y, x01);
    split_pair<TERMS>(a.z, a.w, x23);
#pragma unroll
    for (int x = 0; x < TERMS; ++x) term[x] = make_uint2(x01[x], x23[x]);
}
__device__ __forceinline__ bool sees(const ulonglong2 &m, int n) { return ((n < 64 ? m.x : m.y) >> (n & 63)) & 1; }

// ---- few rows: mma.sync, 16 rows a warp ---------------------------------------------------------------
// Tiles of ROWS = 16 or 32 rows (up to 16 or 32 products of nodes and heads of a group). Every key is 512 bytes from HBM, 22 cycles of an SM at the
// full rate, and some 6 cycles of mma.sync work for 16 rows in three terms: the stream is the bound, and the 128 rows
// of a tcgen05 tile would be padding. Four warps take 16 keys each of a block of 64 for 16 rows; a fifth (ninth) fetches blocks by TMA, kStages deep.
template <int RG>
struct Few {
    static constexpr int kRows = 16 * RG, kWarps = 4 * RG, kThreads = (kWarps + 1) * 32, kKeys = 64;
    static constexpr int kHalf = kKeys * 128, kStage = 4 * kHalf, kStages = 5;
    static constexpr int kQPitch = 272;                               // bytes: eight rows start in eight different bank groups
    static constexpr int kQ0 = kStages * kStage, kQBytes = 3 * kRows * kQPitch;
    static constexpr int kMergePitch = 132;                           // floats
    static constexpr int kMerge0 = kQ0 + kQBytes, kMergeBytes = 2 * kRows * kMergePitch * 4;
    static constexpr int kBars = kMerge0 + kMergeBytes, kSmem = kBars + 2 * kStages * 8 + 1024;
};
struct FewShared {
    Line line;
    int parent[kTreeNodes];
    ulonglong2 mask[kTreeNodes];
    int abort, odd;
};

template <int TERMS, int RG>
__global__ void __launch_bounds__(Few<RG>::kThreads, 1) attn_tree_few_kernel(const __grid_constant__ TreeParams p) {
    using F = Few<RG>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ FewShared sh;
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto full = [&](int s) { return base + F::kBars + s * 8; };
    auto empty = [&](int s) { return base + F::kBars + (F::kStages + s) * 8; };
    volatile int *abort = &sh.abort;
    if (tid == 0) {
        for (int s = 0; s < F::kStages; ++s) {
            ptx::mbar_init(full(s), 1);
            ptx::mbar_init(empty(s), F::kWarps);
        }
        sh.abort = sh.odd = 0;
        ptx::fence_barrier_init();
    }
    ptx::pdl_wait();
    ptx::pdl_trigger();  // behind the wait: what the merging kernel reads in front of its own is settled then
    cut_line<F::kRows, F::kKeys>(p, sh.line);
    const Shares shares(sh.line.first[p.b], p.workers);
    const int u0 = shares.begin(blockIdx.x), u1 = shares.begin(blockIdx.x + 1);
    if (u0 == u1) return;
    const int group = p.nh / p.kvh;
    auto wait = [&](uint32_t bar, uint32_t parity) {
        for (uint32_t i = 0; i < kWaitLimit; ++i) {
            if (ptx::mbar_try_wait(bar, parity)) return true;
            if (*abort) return false;
        }
        *abort = 1;
        return false;
    };

    if (warp == F::kWarps) {
        // ================= TMA producer =================
        if (lane != 0) return;
        int stage = 0, round = 0, sent = 0;
        bool ok = true;
        for (int u = u0; u < u1 && ok;) {
            const Segment s = segment_at(p, sh.line, u, u1, F::kRows, F::kKeys);
            const int row0 = (s.seq * p.kvh + s.kh) * p.cap;
            for (int j = s.begin; j < s.end; ++j, ++sent) {
                if (round > 0 && !wait(empty(stage), (round - 1) & 1)) {
                    ok = false;
                    break;
                }
                const uint32_t at = base + stage * F::kStage;
                ptx::mbar_arrive_expect_tx(full(stage), F::kStage);
                ptx::tma_load_2d(at, &p.k, full(stage), 0, row0 + j * F::kKeys);
                ptx::tma_load_2d(at + F::kHalf, &p.k, full(stage), 128, row0 + j * F::kKeys);
                ptx::tma_load_2d(at + 2 * F::kHalf, &p.v, full(stage), 0, row0 + j * F::kKeys);
                ptx::tma_load_2d(at + 3 * F::kHalf, &p.v, full(stage), 128, row0 + j * F::kKeys);
                if (++stage == F::kStages) {
                    stage = 0;
                    ++round;
                }
            }
            u += s.end - s.begin;
        }
        if (!ok) atomicExch(p.err_word, 5);
        // the copies in flight land before the block may go, whoever has given up
        for (int n = max(0, sent - F::kStages); n < sent; ++n) ptx::mbar_wait(full(n % F::kStages), (n / F::kStages) & 1, kWaitLimit);
        return;
    }

    // ================= the other warps: 16 rows, 16 keys of every block each =================
    const int kg = warp & 3, rg = warp >> 2, g = lane >> 2, tq = lane & 3;
    auto meet = [&]() { ptx::named_barrier(1, F::kWarps * 32); };
    int stage = 0, phase = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
        const Segment s = segment_at(p, sh.line, u, u1, F::kRows, F::kKeys);
        const int pos = sh.line.pos[s.seq], count = sh.line.count[s.seq];
        const int rows_all = count * group, row0 = s.tile * F::kRows;
        const bool nodes = s.end * F::kKeys > pos;  // some of these blocks hold nodes
        // the tile's queries, a row as one load of a warp, all of them asked for before the first is looked at
        float4 qv[F::kRows / F::kWarps];
#pragma unroll
        for (int i = 0; i < F::kRows / F::kWarps; ++i) qv[i] = query<TERMS>(p, s.seq, s.kh, group, row0 + i * F::kWarps + warp, rows_all, lane);
        if (nodes) load_parents(p, sh.parent, s.seq, count, F::kWarps * 32);
#pragma unroll
        for (int i = 0; i < F::kRows / F::kWarps; ++i) {
            uint2 term[TERMS];
            query_terms<TERMS>(qv[i], term);
#pragma unroll
            for (int x = 0; x < TERMS; ++x) *reinterpret_cast<uint2 *>(sm + F::kQ0 + (x * F::kRows + i * F::kWarps + warp) * F::kQPitch + lane * 8) = term[x];
        }
        meet();
        if (nodes)
            for (int i = tid; i < count; i += F::kWarps * 32) tree_masks(sh.parent, sh.mask, i);
        const uint32_t q_at = base + F::kQ0 + (rg * 16 + (lane & 15)) * F::kQPitch + (lane >> 4) * 16;
        if (nodes) meet();
        float o[16][4], m[2] = {kNoMax, kNoMax}, l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < 16; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.0f;
        bool odd = false;  // a value of some node is no number
        for (int j = s.begin; j < s.end; ++j) {
            if (ok) ok = __all_sync(0xffffffffu, wait(full(stage), phase));
            if (ok) {
                const uint32_t ks = base + stage * F::kStage, vs = ks + 2 * F::kHalf;
                const int key0 = j * F::kKeys + kg * 16;
                const bool edge = key0 + 16 > pos;
                // scores: keys 0..7 and 8..15 of the warp's, each term in a sum of its own
                float sc[2][TERMS][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 0; x < TERMS; ++x) sc[h][x][0] = sc[h][x][1] = sc[h][x][2] = sc[h][x][3] = 0.0f;
#pragma unroll
                for (int d2 = 0; d2 < 4; ++d2) {  // 32 dimensions at a time
                    uint32_t kb[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = kg * 16 + h * 8 + (lane & 7), unit = (d2 & 1) * 4 + (lane >> 3);
                        ptx::ldmatrix_x4(kb[h], ks + (d2 >> 1) * F::kHalf + key * 128 + ((unit ^ (key & 7)) << 4));
                    }
#pragma unroll
                    for (int x = 0; x < TERMS; ++x)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            uint32_t qf[4];
                            ptx::ldmatrix_x4(qf, q_at + x * F::kRows * F::kQPitch + (2 * d2 + d) * 32);
#pragma unroll
                            for (int h = 0; h < 2; ++h) ptx::mma_bf16(sc[h][x], qf, kb[h][2 * d], kb[h][2 * d + 1]);
                        }
                }
                float sv[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sv[h][e] = (TERMS > 1 ? sc[h][0][e] + (sc[h][1 % TERMS][e] + sc[h][2 % TERMS][e]) : sc[h][0][e]) * p.scale;
                if (edge) {
                    const int ra = row0 + rg * 16 + g, rb = ra + 8;
                    const ulonglong2 none = make_ulonglong2(0ull, 0ull), ma = ra < rows_all ? sh.mask[p.node_of(ra)] : none, mb = rb < rows_all ? sh.mask[p.node_of(rb)] : none;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + h * 8 + tq * 2 + (e & 1), n = key - pos;
                            if (n >= 0 && (n >= count || !sees(e < 2 ? ma : mb, n))) sv[h][e] = -INFINITY;
                        }
                }
                uint32_t pr[4][TERMS];
                float corr[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // rows g and g + 8
                    const int e = half * 2;
                    float mx = fmaxf(fmaxf(sv[0][e], sv[0][e + 1]), fmaxf(sv[1][e], sv[1][e + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float nm = fmaxf(m[half], mx);
                    corr[half] = ex2(m[half] - nm);
                    m[half] = nm;
                    float sum = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float e0 = ex2(sv[h][e] - nm), e1 = ex2(sv[h][e + 1] - nm);
                        sum += e0 + e1;
                        split_pair<TERMS>(e0, e1, pr[2 * h + half]);
                    }
                    l[half] = l[half] * corr[half] + sum;
                }
                const int key = kg * 16 + (lane & 15);
#pragma unroll
                for (int d2 = 0; d2 < 8; ++d2) {  // 16 dimensions at a time
                    const int unit = (d2 & 3) * 2 + (lane >> 4);
                    uint32_t vb[4];
                    ptx::ldmatrix_x4_trans(vb, vs + (d2 >> 2) * F::kHalf + key * 128 + ((unit ^ (key & 7)) << 4));
                    if (edge) {  // a register: two keys of one dimension
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int n = key0 + (r & 1) * 8 + tq * 2 + e - pos;
                                const bool strange = n >= 0 && ((vb[r] >> (16 * e)) & 0x7f80u) == 0x7f80u;
                                if (strange && n < count) odd = true;
                                if (strange || n >= count) vb[r] &= e ? 0x0000ffffu : 0xffff0000u;
                            }
                    }
                    float add[2][4] = {};
#pragma unroll
                    for (int x = TERMS - 1; x >= 0; --x) {  // the small ones first
                        const uint32_t a[4] = {pr[0][x], pr[1][x], pr[2][x], pr[3][x]};
                        ptx::mma_bf16(add[0], a, vb[0], vb[1]);
                        ptx::mma_bf16(add[1], a, vb[2], vb[3]);
                    }
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[2 * d2 + d][e] = o[2 * d2 + d][e] * corr[e >> 1] + add[d][e];
                }
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(empty(stage));
            }
            if (++stage == F::kStages) {
                stage = 0;
                phase ^= 1;
            }
        }
        if (odd) sh.odd = u + 1;  // read behind the meetings below, written again behind the next segment's first
        // the four warps of a row meet: 2 and 3 hand over to 0 and 1, then 1 to 0
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        }
        float *const place = reinterpret_cast<float *>(sm + F::kMerge0);
#pragma unroll 1
        for (int from = 2; from >= 1; --from) {
            const int slot = from == 2 ? kg & 1 : 0;
            const bool gives = from == 2 ? kg >= 2 : kg == 1, takes = from == 2 ? kg < 2 : kg == 0;
            float *ra = place + (slot * F::kRows + rg * 16 + g) * F::kMergePitch, *rb = ra + 8 * F::kMergePitch;
            if (gives) {
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    *reinterpret_cast<float2 *>(ra + d * 8 + tq * 2) = make_float2(o[d][0], o[d][1]);
                    *reinterpret_cast<float2 *>(rb + d * 8 + tq * 2) = make_float2(o[d][2], o[d][3]);
                }
                if (tq == 0) {
                    *reinterpret_cast<float2 *>(ra + kHd) = make_float2(m[0], l[0]);
                    *reinterpret_cast<float2 *>(rb + kHd) = make_float2(m[1], l[1]);
                }
            }
            meet();
            if (takes) {
                const float2 xa = *reinterpret_cast<const float2 *>(ra + kHd), xb = *reinterpret_cast<const float2 *>(rb + kHd);
                const float na = fmaxf(m[0], xa.x), nb = fmaxf(m[1], xb.x);
                const float wa = ex2(m[0] - na), wb = ex2(m[1] - nb), va = ex2(xa.x - na), vb = ex2(xb.x - nb);
                m[0] = na;
                m[1] = nb;
                l[0] = l[0] * wa + xa.y * va;
                l[1] = l[1] * wb + xb.y * vb;
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                    const float2 ya = *reinterpret_cast<const float2 *>(ra + d * 8 + tq * 2), yb = *reinterpret_cast<const float2 *>(rb + d * 8 + tq * 2);
                    o[d][0] = o[d][0] * wa + ya.x * va;
                    o[d][1] = o[d][1] * wa + ya.y * va;
                    o[d][2] = o[d][2] * wb + yb.x * vb;
                    o[d][3] = o[d][3] * wb + yb.y * vb;
                }
            }
            meet();
        }
        if (kg == 0) {
            const bool fix = nodes && sh.odd == u + 1, whole = s.begin == 0 && s.end == s.blocks;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = rg * 16 + half * 8 + g, row = row0 + r, node = p.node_of(row);
                if (row >= rows_all) continue;
                if (fix) {  // what this row sees that is no number
                    const ulonglong2 mine = sh.mask[node];
                    for (int n = max(0, s.begin * F::kKeys - pos); n < min(count, s.end * F::kKeys - pos); ++n) {
                        if (!sees(mine, n)) continue;
                        const uint16_t *v = p.vcache + (static_cast<size_t>(s.seq * p.kvh + s.kh) * p.cap + pos + n) * kHd + tq * 2;
#pragma unroll
                        for (int d = 0; d < 16; ++d)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if ((v[d * 8 + e] & 0x7f80u) == 0x7f80u) o[d][half * 2 + e] += dense::bf16_f32(v[d * 8 + e]);
                    }
                }
                if (whole) {
                    const float inv = 1.0f / l[half];
                    const size_t at = (static_cast<size_t>(s.seq) * p.t + node) * p.out_pitch + static_cast<size_t>(s.kh * group + row - node * group) * kHd + tq * 2;
#pragma unroll
                    for (int d = 0; d < 16; ++d) {
                        const float x = o[d][half * 2] * inv, y = o[d][half * 2 + 1] * inv;
                        if (TERMS > 1) *reinterpret_cast<float2 *>(static_cast<float *>(p.out) + at + d * 8) = make_float2(x, y);
                        else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p.out) + at + d * 8) = bf16_pair(x, y);
                    }
                } else {
                    const size_t at = (static_cast<size_t>(blockIdx.x) * 2 + (u == u0 ? 0 : 1)) * F::kRows + r;
#pragma unroll
                    for (int d = 0; d < 16; ++d) *reinterpret_cast<float2 *>(p.part + at * kHd + d * 8 + tq * 2) = make_float2(o[d][half * 2], o[d][half * 2 + 1]);
                    if (tq == 0) p.part_ml[at] = make_float2(m[half], l[half]);
                }
            }
        }
        u += s.end - s.begin;
    }
    if (!ok && lane == 0) atomicExch(p.err_word, 5);
}

// ---- many rows: tcgen05, tiles of 128 rows ---------------------------------------------------------------
// Blocks of 128 keys. S = Q K^T: the queries' terms and the K block from shared memory, scores in tensor memory. P V: the probabilities' terms from tensor
// memory, the V block as it lies in the cache (its contraction index, the key, is the strided one: the MN-major operand form), every
// block into zeroed sums, which the softmax warps add to the rows in their registers.
//
//   16 softmax warps four to a quadrant of 32 lanes = rows: warps w, w + 4, .. share rows and take 32 of a block's keys, and of the dimensions, each (eight
//                    warps with 64 took 5900 cycles a block in three terms where the products take 3072: two warps a scheduler do not hide their latencies)
//   K, V producers   a warp each: K blocks of 128 keys are free again after the scores, V in pieces of 64 keys after their product, and one order for
//                    both would have the next K block wait for a piece of V
//   MMA warp         P V of block j - 1, then Q K^T of block j + 1, while the softmax warps work on block j
//
// 512 bytes a key from HBM are 22 cycles of an SM, its products for 128 rows 24 in three terms and 8 in one: f32 is bound by the tensor core, bf16 by
// the stream and by the softmax warps (an exponential per row and key). Padding rows cost nothing but the products: their warps only keep step.
template <int TERMS>
struct Many {
    static constexpr int kRows = 128, kKeys = 128, kHalf = kKeys * 128, kKBytes = 2 * kHalf;
    static constexpr int kPiece = 64, kPieceHalf = kPiece * 128, kPieceBytes = 2 * kPieceHalf;   // V: 64 keys, two halves of 64 dimensions
    static constexpr int kKStages = TERMS == 3 ? 2 : 3, kVStages = TERMS == 3 ? 3 : 5;
    static constexpr int kK0 = TERMS * 2 * kHalf, kV0 = kK0 + kKStages * kKBytes, kBars = kV0 + kVStages * kPieceBytes;
    static constexpr int kPair = kBars + 256, kSmem = kPair + 2 * 4 * kRows * 4 + 1024;
    static constexpr int kSoftWarps = 16, kKWarp = 16, kVWarp = 17, kMmaWarp = 18, kThreads = 20 * 32;
    // Scores (128 columns) and, when all have been read, the probabilities (64 a term) of even blocks in one place, of odd ones in another
    static constexpr uint32_t kPlace = 192, kColO = 384;
};
struct ManyShared {
    Line line;
    int parent[kTreeNodes];
    ulonglong2 mask[kTreeNodes];
    int abort, odd;
    uint32_t tmem;
};
// MN-major SWIZZLE_128B operand: groups of 8 keys 1024 bytes apart (stride byte offset), the halves of 64 dimensions `apart` bytes (leading byte offset)
__device__ __forceinline__ uint64_t desc_mn_sw128(uint32_t addr, uint32_t apart) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | static_cast<uint64_t>(apart >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 |
           static_cast<uint64_t>(2) << 61;
}

template <int TERMS>
__global__ void __launch_bounds__(Many<TERMS>::kThreads, 1) attn_tree_many_kernel(const __grid_constant__ TreeParams p) {
    using M = Many<TERMS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ ManyShared sh;
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kKFull = 0, kKEmpty = 3, kVFull = 6, kVEmpty = 11, kQFull = 16, kPReady = 17, kOFull = 18, kSFull = 19;  // scores: one for even, one for odd blocks
    auto bar = [&](int i) { return base + M::kBars + i * 8; };
    volatile int *abort = &sh.abort;
    if (tid == 0) {
        for (int s = 0; s < M::kKStages; ++s) {
            ptx::mbar_init(bar(kKFull + s), 1);
            ptx::mbar_init(bar(kKEmpty + s), 1);
        }
        for (int s = 0; s < M::kVStages; ++s) {
            ptx::mbar_init(bar(kVFull + s), 1);
            ptx::mbar_init(bar(kVEmpty + s), 1);
        }
        for (int i : {kQFull, kPReady}) ptx::mbar_init(bar(i), M::kSoftWarps);
        for (int i : {kSFull, kSFull + 1, kOFull}) ptx::mbar_init(bar(i), 1);
        sh.abort = sh.odd = 0;
        ptx::fence_barrier_init();
    }
    if (warp == M::kMmaWarp) {
        tc::tmem_alloc(ptx::smem_u32(&sh.tmem), 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    ptx::pdl_wait();
    ptx::pdl_trigger();  // behind the wait: what the merging kernel reads in front of its own is settled then
    cut_line<M::kRows, M::kKeys>(p, sh.line);
    tc::tc_fence_after();
    const uint32_t tmem = *static_cast<volatile uint32_t *>(&sh.tmem);
    const Shares shares(sh.line.first[p.b], p.workers);
    const int u0 = shares.begin(blockIdx.x), u1 = shares.begin(blockIdx.x + 1);
    if (u0 == u1) {
        if (warp == M::kMmaWarp) tc::tmem_dealloc(tmem, 512);
        return;
    }
    const int group = p.nh / p.kvh;
    bool ok = true;

    // The launch has 20 warps x 96 registers; 4 x 64 + 16 x 104 are as many.
    if (warp >= M::kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == M::kKWarp || warp == M::kVWarp) {
            // ================= TMA producers =================
            const bool is_k = warp == M::kKWarp;
            const int stages = is_k ? M::kKStages : M::kVStages, full = is_k ? kKFull : kVFull, empty = is_k ? kKEmpty : kVEmpty;
            if (lane == 0) {
                int stage = 0, round = 0, sent = 0;
                for (int u = u0; u < u1 && ok;) {
                    const Segment s = segment_at(p, sh.line, u, u1, M::kRows, M::kKeys);
                    const int row0 = (s.seq * p.kvh + s.kh) * p.cap;
                    for (int i = is_k ? s.begin : 2 * s.begin; i < (is_k ? s.end : 2 * s.end); ++i, ++sent) {
                        if (round > 0 && !tc::wait_bar(bar(empty + stage), (round - 1) & 1, abort)) {
                            ok = false;
                            break;
                        }
                        if (is_k) {
                            const uint32_t at = base + M::kK0 + stage * M::kKBytes;
                            ptx::mbar_arrive_expect_tx(bar(full + stage), M::kKBytes);
                            ptx::tma_load_2d(at, &p.k, bar(full + stage), 0, row0 + i * M::kKeys);
                            ptx::tma_load_2d(at + M::kHalf, &p.k, bar(full + stage), 128, row0 + i * M::kKeys);
                        } else {
                            const uint32_t at = base + M::kV0 + stage * M::kPieceBytes;
                            ptx::mbar_arrive_expect_tx(bar(full + stage), M::kPieceBytes);
                            ptx::tma_load_2d(at, &p.v, bar(full + stage), 0, row0 + i * M::kPiece);
                            ptx::tma_load_2d(at + M::kPieceHalf, &p.v, bar(full + stage), 128, row0 + i * M::kPiece);
                        }
                        if (++stage == stages) {
                            stage = 0;
                            ++round;
                        }
                    }
                    u += s.end - s.begin;
                }
                // the copies in flight land before the block may go, whoever has given up
                for (int n = max(0, sent - stages); n < sent; ++n) ptx::mbar_wait(bar(full + n % stages), (n / stages) & 1, tc::kTcWaitLimit);
            }
        } else if (warp == M::kMmaWarp) {
            // ================= MMA issue: the warp walks, one lane issues =================
            // D f32, A and B bf16, M = 128, N = 128; for P V the B operand is MN-major (bit 16)
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24), idesc_o = idesc_s | (1u << 16);
            const uint64_t q_desc = tc::smem_desc_sw128(base);
            int ks = 0, kphase = 0, vs = 0, vphase = 0, n = 0, seg = 0;  // n: blocks whose scores have been asked for
            auto wait = [&](int i, int parity) {
                if (ok) ok = tc::warp_wait(bar(i), parity, abort);
                return ok;
            };
            auto scores = [&]() {
                if (!wait(kKFull + ks, kphase)) return;
                tc::tc_fence_after();
                if (tc::elect_one()) {
                    const uint64_t k_desc = tc::smem_desc_sw128(base + M::kK0 + ks * M::kKBytes);
#pragma unroll 1
                    for (int x = TERMS - 1; x >= 0; --x)  // the small ones first
#pragma unroll
                        for (int st = 0; st < 8; ++st) {
                            const uint64_t off = static_cast<uint64_t>((st >> 2) * (M::kHalf >> 4) + (st & 3) * 2);
                            tc::umma_f16_ss(tmem + (n & 1) * M::kPlace, q_desc + static_cast<uint64_t>(x * 2 * (M::kHalf >> 4)) + off, k_desc + off, idesc_s, x < TERMS - 1 || st ? 1u : 0u);
                        }
                    tc::umma_commit(bar(kSFull + (n & 1)));
                    tc::umma_commit(bar(kKEmpty + ks));
                }
                __syncwarp();
                ++n;
                if (++ks == M::kKStages) {
                    ks = 0;
                    kphase ^= 1;
                }
            };
            for (int u = u0; u < u1 && ok; ++seg) {
                const Segment s = segment_at(p, sh.line, u, u1, M::kRows, M::kKeys);
                const int blocks = s.end - s.begin;
                if (wait(kQFull, seg & 1)) scores();
                // Products are carried out in the order they are asked for: the scores of block j + 1 go where the probabilities of block j - 1 were read from
                if (ok && blocks > 1) scores();
                for (int j = 0; j < blocks && ok; ++j) {
                    const int done = n - (j + 1 < blocks ? 2 : 1);  // the number, in the whole walk, of block j
                    if (!wait(kPReady, done & 1)) break;
#pragma unroll 1
                    for (int piece = 0; piece < 2; ++piece) {
                        if (!wait(kVFull + vs, vphase)) break;
                        tc::tc_fence_after();
                        if (tc::elect_one()) {
                            const uint64_t v_desc = desc_mn_sw128(base + M::kV0 + vs * M::kPieceBytes, M::kPieceHalf);
#pragma unroll
                            for (int st = 0; st < 4; ++st)  // 16 keys: 8 columns of P, two groups of V
#pragma unroll
                                for (int x = TERMS - 1; x >= 0; --x)
                                    tc::umma_f16_ts(tmem + M::kColO, tmem + (done & 1) * M::kPlace + x * 64 + (piece * 4 + st) * 8, v_desc + static_cast<uint64_t>(st * (2048 >> 4)), idesc_o,
                                                    piece || st || x < TERMS - 1 ? 1u : 0u);
                            tc::umma_commit(bar(kVEmpty + vs));
                            if (piece) tc::umma_commit(bar(kOFull));
                        }
                        __syncwarp();
                        if (++vs == M::kVStages) {
                            vs = 0;
                            vphase ^= 1;
                        }
                    }
                    if (ok && j + 2 < blocks) scores();
                }
                u += blocks;
            }
        }
    } else {
        // ================= softmax =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int quad = warp & 3, part = warp >> 2, r = quad * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        float *const s_quad = reinterpret_cast<float *>(sm + M::kPair);  // [2][4 parts][128 rows]
        auto wait = [&](int i, int parity) {
            if (ok) ok = tc::warp_wait(bar(i), parity, abort);
            return ok;
        };
        auto arrive = [&](int i) {
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(i));
        };
        auto meet = [&]() { ptx::named_barrier(1, M::kSoftWarps * 32); };
        auto quad_sync = [&]() { ptx::named_barrier(2 + quad, 128); };  // the four warps of a quadrant
        int n = 0;  // blocks so far, over all segments
        for (int u = u0; u < u1;) {
            const Segment s = segment_at(p, sh.line, u, u1, M::kRows, M::kKeys);
            const int pos = sh.line.pos[s.seq], count = sh.line.count[s.seq];
            const int rows_all = count * group, row0 = s.tile * M::kRows, row = row0 + r, node = p.node_of(row);
            const bool nodes = s.end * M::kKeys > pos, live = row0 + quad * 32 < rows_all;  // some blocks hold nodes; some row of the warp exists
            meet();  // nobody reads what the last segment left in the queries' place and in the tree's any more
            // the tile's queries, a row as one load of a warp, all of them asked for before the first is looked at; in the K-major SWIZZLE_128B layout
            // (row r of a half at r * 128, its 16-byte units XOR-ed with r & 7)
            float4 qv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) qv[i] = query<TERMS>(p, s.seq, s.kh, group, row0 + warp * 8 + i, rows_all, lane);
            if (nodes) load_parents(p, sh.parent, s.seq, count, M::kSoftWarps * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint2 term[TERMS];
                query_terms<TERMS>(qv[i], term);
                uint8_t *dst = sm + (lane >> 4) * M::kHalf + (warp * 8 + i) * 128 + ((((lane & 15) >> 1) ^ i) << 4) + (lane & 1) * 8;
#pragma unroll
                for (int x = 0; x < TERMS; ++x) *reinterpret_cast<uint2 *>(dst + x * 2 * M::kHalf) = term[x];
            }
            ptx::fence_proxy_async();  // the tensor core reads them through the asynchronous proxy
            arrive(kQFull);
            if (nodes) {
                meet();
                for (int i = tid; i < count; i += M::kSoftWarps * 32) tree_masks(sh.parent, sh.mask, i);
                meet();
            }
            float acc[32], m = kNoMax, l = 0.0f, corr = 0.0f;  // 32 dimensions of the row; corr: what brings acc to the present maximum
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[i] = 0.0f;
            // acc = acc * corr + the products of block n - 1
            auto add_products = [&]() {
                tc::tc_fence_after();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t v[16];
                    tc::tmem_ld16(lanes + M::kColO + part * 32 + c * 16, v);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[c * 16 + i] = acc[c * 16 + i] * corr + __uint_as_float(v[i]);
                }
            };
            for (int j = s.begin; j < s.end; ++j, ++n) {
                uint32_t sv[32];
                const int key0 = j * M::kKeys + part * 32;
                const uint32_t place = lanes + (n & 1) * M::kPlace;
                float step = 0.0f;
                wait(kSFull + (n & 1), n >> 1 & 1);
                if (live) {
                    tc::tc_fence_after();
                    tc::tmem_ld32(place + part * 32, sv);
                    tc::tmem_ld_wait();
                    if (key0 + 32 > pos) {  // some of these keys are nodes, or nothing: bit i of `seen` is key0 + i
                        const ulonglong2 mine = row < rows_all ? sh.mask[node] : make_ulonglong2(0ull, 0ull);
                        const int n0 = key0 - pos;
                        const uint32_t seen = static_cast<uint32_t>(n0 < 0 ? mine.x << -n0 | ((1ull << -n0) - 1) : n0 == 0 ? mine.x : n0 < 64 ? mine.x >> n0 | mine.y << (64 - n0) : n0 < 128 ? mine.y >> (n0 - 64) : 0ull);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!(seen >> i & 1)) sv[i] = 0xff800000u;  // -inf
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(sv[i]));
                    float *quarter = s_quad + (n & 1) * 4 * M::kRows + r;
                    quarter[part * M::kRows] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    quad_sync();  // the row's scores have all been read; the next block but one writes here again, behind the next block's meeting
                    const float all = fmaxf(fmaxf(quarter[0], quarter[M::kRows]), fmaxf(quarter[2 * M::kRows], quarter[3 * M::kRows]));
                    const float nm = fmaxf(m, all * p.scale);
                    step = ex2(m - nm);
                    m = nm;
                    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[TERMS][8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float e0 = ex2(__fmaf_rn(__uint_as_float(sv[c * 16 + 2 * i]), p.scale, -nm)), e1 = ex2(__fmaf_rn(__uint_as_float(sv[c * 16 + 2 * i + 1]), p.scale, -nm));
                            sum0 += e0;
                            sum1 += e1;
                            uint32_t term[TERMS];
                            split_pair<TERMS>(e0, e1, term);
#pragma unroll
                            for (int x = 0; x < TERMS; ++x) w[x][i] = term[x];
                        }
#pragma unroll
                        for (int x = 0; x < TERMS; ++x) tc::tmem_st8(place + x * 64 + part * 16 + c * 8, w[x]);
                    }
                    l = l * step + (sum0 + sum1);
                }
                if (j * M::kKeys + M::kKeys > pos) {  // values past the last node, and values of nodes that are no numbers: a thread 32 dimensions of a row of this warp's piece
                    const int piece = 2 * n + (part >> 1), vs = piece % M::kVStages, quarter = (part & 1) * 2 + (r >> 6), key = r & 63, at = j * M::kKeys + (part >> 1) * 64 + key - pos;
                    if (wait(kVFull + vs, (piece / M::kVStages) & 1) && at >= 0) {
                        uint4 *v = reinterpret_cast<uint4 *>(sm + M::kV0 + vs * M::kPieceBytes + (quarter >> 1) * M::kPieceHalf + key * 128 + (quarter & 1) * 64);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 x = v[i];
                            if (at >= count) {
                                v[i] = make_uint4(0u, 0u, 0u, 0u);
                            } else {
                                const uint4 y = make_uint4(only_numbers(x.x), only_numbers(x.y), only_numbers(x.z), only_numbers(x.w));
                                if (((x.x ^ y.x) | (x.y ^ y.y) | (x.z ^ y.z) | (x.w ^ y.w)) != 0u) {
                                    v[i] = y;
                                    sh.odd = u + 1;  // read behind a meeting below, written again behind the next segment's first
                                }
                            }
                        }
                    }
                    ptx::fence_proxy_async();
                }
                // the products of the block in front are added, then their place is free
                if (j > s.begin) {
                    wait(kOFull, (n - 1) & 1);
                    if (live) add_products();
                }
                corr = step;
                if (live) tc::tmem_st_wait();
                tc::tc_fence_before();
                arrive(kPReady);
            }
            wait(kOFull, (n - 1) & 1);
            if (live) add_products();
            // the row's weight: the four parts of the keys meet
            float *quarter = s_quad + (n & 1) * 4 * M::kRows + r;
            quarter[part * M::kRows] = l;
            meet();
            l = (quarter[0] + quarter[M::kRows]) + (quarter[2 * M::kRows] + quarter[3 * M::kRows]);
            if (nodes && sh.odd == u + 1 && row < rows_all) {  // what this row sees that is no number
                const ulonglong2 mine = sh.mask[node];
                for (int i = max(0, s.begin * M::kKeys - pos); i < min(count, s.end * M::kKeys - pos); ++i) {
                    if (!sees(mine, i)) continue;
                    const uint16_t *v = p.vcache + (static_cast<size_t>(s.seq * p.kvh + s.kh) * p.cap + pos + i) * kHd + part * 32;
#pragma unroll
                    for (int d = 0; d < 32; ++d)
                        if ((v[d] & 0x7f80u) == 0x7f80u) acc[d] += dense::bf16_f32(v[d]);
                }
            }
            // Rows leave through the queries' place, whose products are done, so that a store instruction writes whole sectors: a warp's 32 rows of 16
            // dimensions at a time, 16-byte units XOR-ed with the row.
            const bool whole = s.begin == 0 && s.end == s.blocks;
            if (live && ok) {
                const float inv = whole ? 1.0f / l : 1.0f;
                const size_t part0 = (static_cast<size_t>(blockIdx.x) * 2 + (u == u0 ? 0 : 1)) * M::kRows;
                if (!whole && part == 0 && row < rows_all) p.part_ml[part0 + r] = make_float2(m, l);
                float *own = reinterpret_cast<float *>(sm + warp * 2048);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4 *>(own + lane * 16 + ((i ^ (lane >> 1 & 3)) << 2)) =
                            make_float4(acc[c * 16 + 4 * i] * inv, acc[c * 16 + 4 * i + 1] * inv, acc[c * 16 + 4 * i + 2] * inv, acc[c * 16 + 4 * i + 3] * inv);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = i * 8 + (lane >> 2), at_row = row0 + quad * 32 + rr, at_node = p.node_of(at_row), d = part * 32 + c * 16 + (lane & 3) * 4;
                        if (at_row < rows_all) {
                            const float4 x = *reinterpret_cast<const float4 *>(own + rr * 16 + (((lane & 3) ^ (rr >> 1 & 3)) << 2));
                            const size_t at = (static_cast<size_t>(s.seq) * p.t + at_node) * p.out_pitch + static_cast<size_t>(s.kh * group + at_row - at_node * group) * kHd + d;
                            if (!whole) *reinterpret_cast<float4 *>(p.part + (part0 + quad * 32 + rr) * kHd + d) = x;
                            else if (TERMS > 1) dense::put4(static_cast<float *>(p.out) + at, x);
                            else dense::put4(static_cast<uint16_t *>(p.out) + at, x);
                        }
                    }
                    __syncwarp();
                }
            }
            u += s.end - s.begin;
        }
    }
    if (!ok && lane == 0) atomicExch(p.err_word, 5);
    tc::tc_fence_before();
    __syncthreads();
    if (warp == M::kMmaWarp) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of the tiles that were cut. A block takes some rows of the tile that begins in its worker's share and ends behind it, if there is one: a
// warp a row, four dimensions a lane. Which that is is known before the attention kernel is done.
constexpr int kMergeRows = 16;  // rows a block
template <int TERMS, int ROWS, int KEYS>
__global__ void __launch_bounds__(kMergeRows * 32) attn_tree_merge_kernel(const __grid_constant__ TreeParams p) {
    __shared__ Line line;
    ptx::pdl_trigger();
    cut_line<ROWS, KEYS>(p, line);
    const Shares shares(line.first[p.b], p.workers);
    const int lane = threadIdx.x & 31, r = blockIdx.y * kMergeRows + (threadIdx.x >> 5), group = p.nh / p.kvh, c0 = blockIdx.x;
    const int u0 = shares.begin(c0), u1 = shares.begin(c0 + 1);
    Segment s{};
    int begin = 0, row = 0, parts = 0;
    if (u0 < u1) {
        s = segment_at(p, line, u1 - 1, u1, ROWS, KEYS);  // the last block of the share
        begin = u1 - 1 - s.begin;
        row = s.tile * ROWS + r;
        const int end = begin + s.blocks;
        if (begin >= u0 && end > u1 && row < line.count[s.seq] * group) parts = shares.owner(end - 1) - c0 + 1;  // neighbours that all have a share: this tile goes on in it
    }
    ptx::pdl_wait();  // blocks without a tile too: the next kernel of the stream waits for this one only
    if (!parts) return;
    const int node = p.node_of(row);
    auto place = [&](int i) { return (static_cast<size_t>(c0 + i) * 2 + (i == 0 && u0 < begin ? 1 : 0)) * ROWS + r; };
    float m = kNoMax;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_ml[place(i)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        const float2 ml = p.part_ml[place(i)];
        const float4 x = *reinterpret_cast<const float4 *>(p.part + place(i) * kHd + lane * 4);
        const float w = ex2(ml.x - m);
        l += ml.y * w;
        sum.x += x.x * w;
        sum.y += x.y * w;
        sum.z += x.z * w;
        sum.w += x.w * w;
    }
    const float inv = 1.0f / l;
    const size_t at = (static_cast<size_t>(s.seq) * p.t + node) * p.out_pitch + static_cast<size_t>(s.kh * group + row - node * group) * kHd + lane * 4;
    if (TERMS > 1) dense::put4(static_cast<float *>(p.out) + at, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
    else dense::put4(static_cast<uint16_t *>(p.out) + at, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
}

int attn_tree_init(Ctx *ctx) {
    struct { void (*k)(TreeParams); int smem; } kernels[] = {{attn_tree_few_kernel<1, 1>, Few<1>::kSmem}, {attn_tree_few_kernel<3, 1>, Few<1>::kSmem},
                                                         {attn_tree_few_kernel<1, 2>, Few<2>::kSmem}, {attn_tree_few_kernel<3, 2>, Few<2>::kSmem}, {attn_tree_many_kernel<1>, Many<1>::kSmem}, {attn_tree_many_kernel<3>, Many<3>::kSmem}};
    for (auto &f : kernels) LBK_CUDA(cudaFuncSetAttribute(f.k, cudaFuncAttributeMaxDynamicSharedMemorySize, f.smem));
    return LBK_OK;
}
const InitHook kInitAttnTree(attn_tree_init);

// Rows of a tile for t nodes of `group` heads.
int tile_rows(size_t t, size_t group) { return t * group <= 16 ? 16 : t * group <= 32 ? 32 : 128; }

template <int ROWS, int KEYS>
int launch_tree(Ctx *ctx, int terms, TreeParams &p, void (*one)(TreeParams), void (*three)(TreeParams), int threads, int smem, cudaStream_t st) {
    LBK_CUDA(launch_chained(terms == 3 ? three : one, dim3(static_cast<unsigned>(p.workers)), dim3(threads), static_cast<size_t>(smem), st, p));
    ctx->launches++;
    const dim3 grid(static_cast<unsigned>(p.workers), (std::min(ROWS, p.t * (p.nh / p.kvh)) + kMergeRows - 1) / kMergeRows);
    LBK_CUDA(launch_chained(terms == 3 ? attn_tree_merge_kernel<3, ROWS, KEYS> : attn_tree_merge_kernel<1, ROWS, KEYS>, grid, dim3(kMergeRows * 32), 0, st, p));
    ctx->launches++;
    return LBK_OK;
}

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

size_t lbk_attn_tree_scratch(const lbk_ctx *c, size_t t, size_t n_heads, size_t kv_heads) {
    if (!c || !kv_heads) return 0;
    return static_cast<size_t>(reinterpret_cast<const Ctx *>(c)->sm_count) * 2 * tile_rows(t, n_heads / kv_heads) * (kHd + 2);
}

int lbk_attn_tree(lbk_ctx *c, int compute, const void *q_dev, size_t q_pitch, const uint16_t *kcache_dev, const uint16_t *vcache_dev, const int32_t *pos_dev,
                  const int32_t *parents_dev, const int32_t *counts_dev, size_t b, size_t t, size_t n_heads, size_t kv_heads, size_t head_dim, size_t cap, float scale,
                  float *scratch_dev, void *out_dev, size_t out_pitch, void *stream) {
    LBK_TREE_PRE("lbk_attn_tree");
    if (b == 0 || t == 0) return LBK_OK;
    if (!q_dev || !kcache_dev || !vcache_dev || !pos_dev || !parents_dev || !scratch_dev || !out_dev) return fail(LBK_ERR_INVALID, "lbk_attn_tree: null buffer");
    if (compute != LBK_COMPUTE_BF16 && compute != LBK_COMPUTE_F32) return fail(LBK_ERR_INVALID, "lbk_attn_tree: unknown compute type %d", compute);
    if (t > LBK_TREE_NODES || b > kMaxSeqs) return fail(LBK_ERR_UNSUPPORTED, "lbk_attn_tree: at most %d nodes of %d sequences (got %zu of %zu)", LBK_TREE_NODES, kMaxSeqs, t, b);
    if (head_dim != kHd || !kv_heads || !n_heads || n_heads % kv_heads) return fail(LBK_ERR_SHAPE, "lbk_attn_tree: heads of %d, a multiple of the KV heads", kHd);
    if (!(scale > 0.0f) || scale > 1e30f) return fail(LBK_ERR_INVALID, "lbk_attn_tree: the scale is a positive number");
    const size_t unit = compute == LBK_COMPUTE_F32 ? 4 : 8, width = n_heads * kHd;
    if (q_pitch < width || out_pitch < width || q_pitch % unit || out_pitch % unit) return fail(LBK_ERR_SHAPE, "lbk_attn_tree: rows of %zu values, pitches of %zu and %zu", width, q_pitch, out_pitch);
    if ((reinterpret_cast<uintptr_t>(q_dev) | reinterpret_cast<uintptr_t>(kcache_dev) | reinterpret_cast<uintptr_t>(vcache_dev) | reinterpret_cast<uintptr_t>(scratch_dev) |
         reinterpret_cast<uintptr_t>(out_dev)) & 15)
        return fail(LBK_ERR_SHAPE, "lbk_attn_tree: buffers lie on 16 bytes");
    if (n_heads > 4096 || cap > (1u << 30)) return fail(LBK_ERR_UNSUPPORTED, "lbk_attn_tree: %zu heads, %zu positions", n_heads, cap);
    const size_t rows = b * kv_heads * cap, group = n_heads / kv_heads;
    if (rows > INT32_MAX || b * kv_heads * ((t * group + 15) / 16) * (cap / 64 + 1) > INT32_MAX)
        return fail(LBK_ERR_UNSUPPORTED, "lbk_attn_tree: a cache of %zu rows", rows);
    TreeParams p{};
    p.q = q_dev;
    p.out = out_dev;
    p.q_pitch = static_cast<long>(q_pitch);
    p.out_pitch = static_cast<long>(out_pitch);
    p.vcache = vcache_dev;
    p.pos = pos_dev;
    p.parents = parents_dev;
    p.counts = counts_dev;
    p.b = static_cast<int>(b);
    p.t = static_cast<int>(t);
    p.nh = static_cast<int>(n_heads);
    p.kvh = static_cast<int>(kv_heads);
    p.cap = static_cast<int>(cap);
    p.scale = scale * 1.4426950408889634f;
    p.workers = ctx->sm_count;
    p.per_group = group > 1 ? static_cast<unsigned>((0x100000000ull + group - 1) / group) : 0u;  // exact: rows * heads of a group < 2^32
    p.err_word = ctx->err_word;
    const int tile = tile_rows(t, group), terms = compute == LBK_COMPUTE_F32 ? 3 : 1;
    p.part = scratch_dev;
    p.part_ml = reinterpret_cast<float2 *>(scratch_dev + static_cast<size_t>(p.workers) * 2 * tile * kHd);
    LBK_TRY(encode_bytes_map(&p.k, kcache_dev, 256, rows, 256, 128, tile == 128 ? 128 : 64));
    LBK_TRY(encode_bytes_map(&p.v, vcache_dev, 256, rows, 256, 128, 64));
    if (tile == 16) return launch_tree<16, 64>(ctx, terms, p, attn_tree_few_kernel<1, 1>, attn_tree_few_kernel<3, 1>, Few<1>::kThreads, Few<1>::kSmem, st);
    if (tile == 128) return launch_tree<128, 128>(ctx, terms, p, attn_tree_many_kernel<1>, attn_tree_many_kernel<3>, Many<1>::kThreads, Many<1>::kSmem, st);
    return launch_tree<32, 64>(ctx, terms, p, attn_tree_few_kernel<1, 2>, attn_tree_few_kernel<3, 2>, Few<2>::kThreads, Few<2>::kSmem, st);
}

}  // extern "C"
