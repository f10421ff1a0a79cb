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
// zero and are added to the row in registers, one rounded addition a block. bf16 queries are exact in one term, and their probabilities are two terms, as in
// the decode and prompt kernels: off by 2^-16 of themselves at most, where the result is rounded by 2^-8 of itself. In one term a weight is off by as much as the result's
// rounding, and what that adds to a result does not average out: over many keys of like weights a sum of values of either sign shrinks as its error does (60 nodes of 65000
// keys: 0.0023 of the result against 0.0017 by its rounding alone), and of a few heavy keys whose values cancel the error is any multiple of the result.
//
// Rows of V that nobody has written may hold anything, and 0 * NaN is NaN: values past the sequence's last node are taken as zeros. Values of OTHER
// branches may be infinite or NaN too; a row that does not see them must not notice. So in the blocks of the nodes values that are no numbers are
// taken as zeros as well, and added at the end to the rows that see them (a weight is never zero in exact arithmetic).
#include <algorithm>
#include <type_traits>

#include "lbk_dense_dev.cuh"
#include "lbk_tcgen05.cuh"
#include "lbk_tree.cuh"

namespace lbk {

namespace {

using dense::bf16_pair;

constexpr int kHd = 128;
constexpr int kMaxSeqs = 256;
constexpr float kNoMax = -3.0e38f;  // a row that has seen nothing: finite, so that -inf scores less it are no NaN

struct TreeParams {
    CUtensorMap k, v;   // bytes [cache rows][256], boxes of 128 bytes and 128 rows of K, 64 of V, SWIZZLE_128B
    const void *q;
    void *out;
    long q_pitch, out_pitch;
    const uint16_t *vcache;
    const int *pos, *parents, *counts;
    int b, t, kvh, group, cap;  // group: query heads of a KV head
    float scale;        // log2(e) * scale: scores in units of log 2
    float *part;        // [CTA][2][tile rows][128]
    float2 *part_ml;    // [CTA][2][tile rows]: maximum, weight
    int workers;        // CTAs of the attention kernel
    unsigned per_worker; // 2^32 / workers
    unsigned per_group; // 2^32 / heads of a group, rounded up; 0 for one head
    int *err_word;
    __device__ __forceinline__ int node_of(int row) const { return per_group ? static_cast<int>(__umulhi(static_cast<unsigned>(row), per_group)) : row; }
};

__device__ __forceinline__ float ex2(float x) {  // 2^x, the hardware's approximation
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// bf16 terms of a probability for queries of TERMS
constexpr int weight_terms(int terms) { return terms == 1 ? 2 : terms; }
// Two values at once as bf16 terms: term[i] = bf16(x - the terms in front of it), and with three of them their sum is x
template <int TERMS>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&term)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        term[i] = bf16_pair(x0, x1);
        if (i + 1 < TERMS) {
            const float2 rest = ptx::fma2(make_float2(__uint_as_float(term[i] << 16), __uint_as_float(term[i] & 0xffff0000u)), make_float2(-1.0f, -1.0f), make_float2(x0, x1));
            x0 = rest.x;
            x1 = rest.y;
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
// A sequence has kv_heads * tiles problems of `blocks` units each.
// A sequence's rows: no nodes if it lies outside its cache. (Loads from L2: the merging kernel comes here in front of its wait.)
__device__ __forceinline__ void line_rows(const TreeParams &p, int seq, int &pos, int &count) {
    pos = count = 0;
    if (seq >= p.b) return;
    pos = __ldcg(p.pos + seq);
    count = p.counts ? min(max(__ldcg(p.counts + seq), 0), p.t) : p.t;
    if (pos < 0 || pos > p.cap - count) {
        if (blockIdx.x == 0) atomicExch(p.err_word, kErrPos);
        count = 0;
    }
}
template <int ROWS, int KEYS>
__device__ __forceinline__ int line_units(const TreeParams &p, int pos, int count) {
    return count ? (pos + count + KEYS - 1) / KEYS * ((count * p.group + ROWS - 1) / ROWS) * p.kvh : 0;
}
__device__ __forceinline__ int sum_up_to(int mine, int lane) {  // over the lanes
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, mine, o);
        if (lane >= o) mine += up;
    }
    return mine;
}
// Fills the line. All threads of the block; a warp does it.
template <int ROWS, int KEYS>
__device__ __forceinline__ void cut_line(const TreeParams &p, Line &l) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int before = 0;
        for (int i0 = 0; i0 < p.b; i0 += 32) {
            const int i = i0 + lane;
            int pos, count;
            line_rows(p, i, pos, count);
            const int mine = line_units<ROWS, KEYS>(p, pos, count), sum = sum_up_to(mine, lane);
            if (i < p.b) {
                l.pos[i] = pos;
                l.count[i] = count;
                l.first[i] = before + sum - mine;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) l.first[p.b] = before;
    }
    __syncthreads();
}
// a / b for 0 <= a and 0 < b, whose quotient is below 2^20: the approximate one is off by one at most
__device__ __forceinline__ int quotient(int a, int b) {
    const int q = static_cast<int>(__fdividef(static_cast<float>(a), static_cast<float>(b))), r = a - q * b;
    return q + (r >= b) - (r < 0);
}
// Worker w takes the units share_begin(w) .. share_begin(w + 1) - 1: `each` of them, one more the first `more` workers.
struct Shares {
    int each, more;
    __device__ __forceinline__ Shares(int units, const TreeParams &p) {
        each = static_cast<int>(__umulhi(static_cast<unsigned>(units), p.per_worker));  // or one less
        each += units - each * p.workers >= p.workers;
        more = units - each * p.workers;
    }
    __device__ __forceinline__ int begin(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int owner(int u) const { return u < more * (each + 1) ? u / (each + 1) : more + (u - more * (each + 1)) / each; }
};

struct Segment {
    int seq, kh, tile;     // the problem
    int begin, end;        // its blocks
    int blocks;            // of all there are
    int pos, count;        // of the sequence
};
// The blocks of a problem from `unit` on, which lies `at` units into the sequence; a share ends in front of `last`
__device__ __forceinline__ Segment segment_in(const TreeParams &p, int seq, int pos, int count, int unit, int at, int last, int rows, int keys) {
    Segment s;
    s.seq = seq;
    s.pos = pos;
    s.count = count;
    s.blocks = (pos + count + keys - 1) / keys;
    const int tiles = (count * p.group + rows - 1) / rows, problem = quotient(at, s.blocks);
    s.begin = at - problem * s.blocks;
    s.end = min(s.blocks, s.begin + last - unit);
    s.kh = quotient(problem, tiles);
    s.tile = problem - s.kh * tiles;
    return s;
}
__device__ __forceinline__ Segment segment_at(const TreeParams &p, const Line &l, int unit, int last, int rows, int keys) {
    int lo = 0, hi = p.b - 1;   // the last sequence whose units begin at or before this one and that has any
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= unit) lo = mid;
        else hi = mid - 1;
    }
    return segment_in(p, lo, l.pos[lo], l.count[lo], unit, unit - l.first[lo], last, rows, keys);
}
// A block's units u0 .. u1 - 1, and the first segment of them. Up to 32 sequences every warp finds it by itself from the sequences' rows: in front of the first
// query everything waits for this. Warp 0 leaves the line for the other segments; who looks for those has met it or waited for its queries since.
struct Share {
    int u0, u1, most;   // most: the largest share of all
    Segment first;
};
// Where the walk over a segment's blocks begins, and goes round: block x comes up when x mod `most` units of the share are done, as far as that can be. The tiles of a KV
// head are walked by different CTAs, each from somewhere else; so they come to a block at about the same time, and HBM is asked for it once: 60 nodes of 65000 keys with 8 heads
// of 4, two tiles, read 518 MB where the cache has 266, and 282 so; us of 36 calls behind one another, without / with it 104.9 / 98.7 in bf16, 159.7 / 153.5 in f32. Of one tile the walk is
// straight.
__device__ __forceinline__ int first_block(const Share &share, const Segment &s, int unit, int group, int rows) {
    if (s.count * group <= rows) return s.begin;
    const int ahead = (unit - share.u0 - s.begin) % share.most, at = s.begin + (ahead < 0 ? ahead + share.most : ahead);
    return at < s.end ? at : s.begin;
}
template <int ROWS, int KEYS>
__device__ __forceinline__ Share own_share(const TreeParams &p, Line &l) {
    Share s{};
    if (p.b > 32) {
        cut_line<ROWS, KEYS>(p, l);
        const Shares shares(l.first[p.b], p);
        s.most = shares.each + (shares.more > 0);
        s.u0 = shares.begin(blockIdx.x);
        s.u1 = shares.begin(blockIdx.x + 1);
        if (s.u0 < s.u1) s.first = segment_at(p, l, s.u0, s.u1, ROWS, KEYS);
        return s;
    }
    const int lane = threadIdx.x & 31;
    int pos, count;
    if (threadIdx.x < 32) {  // one warp reads, so that all see the same, whatever happens to the positions meanwhile
        line_rows(p, lane, pos, count);
        l.pos[lane] = pos;
        l.count[lane] = count;
    }
    __syncthreads();
    pos = l.pos[lane];
    count = l.count[lane];
    const int mine = line_units<ROWS, KEYS>(p, pos, count), sum = sum_up_to(mine, lane), first = sum - mine, all = __shfl_sync(0xffffffffu, sum, 31);
    const Shares shares(all, p);
    s.most = shares.each + (shares.more > 0);
    s.u0 = shares.begin(blockIdx.x);
    s.u1 = shares.begin(blockIdx.x + 1);
    const unsigned has = __ballot_sync(0xffffffffu, mine && first <= s.u0);  // the last one of these
    if (s.u0 < s.u1) {
        const int seq = 31 - __clz(has);
        s.first = segment_in(p, seq, __shfl_sync(0xffffffffu, pos, seq), __shfl_sync(0xffffffffu, count, seq), s.u0, s.u0 - __shfl_sync(0xffffffffu, first, seq), s.u1, ROWS, KEYS);
    }
    if (threadIdx.x < 32) {
        if (lane < p.b) l.first[lane] = first;
        if (lane == 0) l.first[p.b] = all;
    }
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

struct CtaShared {
    Line line;
    Segment seg[20];   // a warp's present one: eight registers that the loop over its blocks has no room for
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

// A warp's wait for what is complete already as a rule.
__device__ __forceinline__ bool look_and_wait(uint32_t bar, uint32_t parity, volatile int *abort) {
    if (__all_sync(0xffffffffu, ptx::mbar_test_wait(bar, parity))) return true;
    return tc::warp_wait(bar, parity, abort);
}
// Zeros for values that are no numbers, or for all of `units` 16-byte units; whether there was one that is no number.
__device__ __forceinline__ bool clean_values(uint4 *v, int units, bool all) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < units; ++i) {
        if (all) {
            v[i] = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        const uint4 x = v[i], y = make_uint4(only_numbers(x.x), only_numbers(x.y), only_numbers(x.z), only_numbers(x.w));
        if (((x.x ^ y.x) | (x.y ^ y.y) | (x.z ^ y.z) | (x.w ^ y.w)) == 0u) continue;
        v[i] = y;
        odd = true;
    }
    return odd;
}
constexpr int kQueriesAsked = 8;  // named barrier
// A producer warp of a kernel with layout M: the K blocks, or the V pieces, of a share. full, empty: the first of the stages' barriers.
template <class M>
__device__ __forceinline__ void produce(const TreeParams &p, const Line &line, const Share &share, int rows, bool is_k, uint32_t base, uint32_t full, uint32_t empty, volatile int *abort, bool &ok) {
    // The first queries go first: behind 128 KB of keys and values an SM, which all ask for at the same time, they took 3000 to 6000 cycles
    ptx::named_barrier(kQueriesAsked, M::kSoftWarps * 32 + 64);
    if ((threadIdx.x & 31) != 0) return;
    const int stages = is_k ? M::kKStages : M::kVStages;
    int stage = 0, round = 0, sent = 0;
    Segment s = share.first;
    for (int u = share.u0; u < share.u1 && ok;) {
        const int row0 = (s.seq * p.kvh + s.kh) * p.cap;
        const int begin = M::kGoesRound ? first_block(share, s, u, p.group, rows) : s.begin, per = is_k ? 1 : 2;  // copies a block
        for (int c = 0, i = begin * per; c < (s.end - s.begin) * per; ++c, ++sent, i = i + 1 == s.end * per ? s.begin * per : i + 1) {
            if (round > 0 && !tc::wait_bar(empty + stage * 8, (round - 1) & 1, abort)) {
                ok = false;
                break;
            }
            const uint32_t at = base + (is_k ? M::kK0 + stage * M::kKBytes : M::kV0 + stage * M::kPieceBytes), done = full + stage * 8;
            ptx::mbar_arrive_expect_tx(done, is_k ? M::kKBytes : M::kPieceBytes);
            ptx::tma_load_2d(at, is_k ? &p.k : &p.v, done, 0, row0 + i * (is_k ? M::kKeys : M::kPiece));
            ptx::tma_load_2d(at + (is_k ? M::kHalf : M::kPieceHalf), is_k ? &p.k : &p.v, done, 128, row0 + i * (is_k ? M::kKeys : M::kPiece));
            if (++stage == stages) {
                stage = 0;
                ++round;
            }
        }
        u += s.end - s.begin;
        if (u < share.u1) s = segment_at(p, line, u, share.u1, rows, M::kKeys);
    }
    // the copies in flight land before the block may go, whoever has given up
    for (int n = max(0, sent - stages); n < sent; ++n) ptx::mbar_wait(full + n % stages * 8, (n / stages) & 1, tc::kTcWaitLimit);
}

// ---- few rows: tcgen05 with keys and dimensions in the lanes ------------------------------------------------
// Tiles of 16 and 32 rows. The 128 lanes of an accumulator are a block's keys, S^T = K Q^T, and then the dimensions, O^T = V^T P^T; rows and terms are its columns, so
// that a product costs what the rows need: 512 and 768 cycles of the tensor core for a block of 128 keys and 16 and 32 rows in three terms, where the block's 64 KB are
// 2800 cycles of an SM's share of HBM. The stream is the bound. (mma.sync has 16 x 16 x 8 products at a sixteenth of this rate: 16 rows in three terms took 4600 cycles for
// 128 keys, 32 rows 6400. Tiles of 64 rows, us at 16 sequences of 8100 keys: so 136, bf16 102; tiles of 128 half empty 124 and 81,
// bf16 with weights in one term. Few sequences of 33 to 64 rows were not measured by themselves.)
//
// All terms of the queries are rows of one operand, and so are those of the probabilities, which go through shared memory. A thread has one key and half of the rows:
// a row's maximum is not at hand, and not needed: probabilities are 2^(s - m) with any m that keeps them in range. m is the maximum of the tile's first block, and is moved
// (and the sums with it) when some score is over it by more than kSlack.
//
//   8 softmax warps  warp w and w + 4: the quadrant of 32 lanes w % 4, the first and the second half of the rows
//   K, V producers, MMA warp  as below, but one MMA warp: Q K^T of block j + 1 as soon as the scores of block j have been read, then P V of block j (two warps: 40.1 -> 43.7
//                             us for 6 nodes of 65000 keys)
constexpr float kSlack = 8.0f;  // in units of log 2: probabilities stay below 2^8
template <int TERMS, int ROWS>
struct Turned {
    static constexpr bool kGoesRound = false;  // one tile a problem
    static constexpr int kKeys = 128, kHalf = kKeys * 128, kKBytes = 2 * kHalf;
    static constexpr int kPiece = 64, kPieceHalf = kPiece * 128, kPieceBytes = 2 * kPieceHalf;   // V: 64 keys, two halves of 64 dimensions
    // queries, and probabilities of a block (a place for even, one for odd ones): [2 halves][terms * rows][128 bytes]
    static constexpr int kPTerms = weight_terms(TERMS), kQCols = TERMS * ROWS, kQHalf = kQCols * 128, kQBytes = 2 * kQHalf, kPCols = kPTerms * ROWS, kPHalf = kPCols * 128, kPBytes = 2 * kPHalf;
    static constexpr int kKStages = kPCols > 64 ? 2 : 3, kVStages = kPCols > 64 ? 4 : 5;
    static constexpr int kP0 = kQBytes, kK0 = kP0 + 2 * kPBytes, kV0 = kK0 + kKStages * kKBytes, kBars = kV0 + kVStages * kPieceBytes;
    static constexpr int kMax = kBars + 256, kPart = kMax + ROWS * 4, kSmem = kPart + 4 * ROWS * 4 + 1024;   // the rows' m; [quadrant][row] floats
    static constexpr int kSoftWarps = 8, kKWarp = 8, kVWarp = 9, kMmaWarp = 10, kThreads = 11 * 32;
    static_assert(kVStages >= 2 * 2, "as of Many::kBehind: a warp in block n has added the products of block n - 2");
    static constexpr uint32_t kColO = kPCols <= 32 ? 32 : kPCols <= 64 ? 64 : 128, kTmem = 4 * kColO;  // scores, and from kColO on the products of even and of odd blocks
    static_assert(kSmem + 6 * 1024 <= 232448 && kQCols % 16 == 0 && kPCols % 16 == 0 && kQCols <= kPCols && kPCols <= 128, "shared memory and operand sizes");
};
// v[0] becomes what `join` makes of value lane / (32 / N) of all lanes: half of the values go to the other half of the lanes in every step
template <int N, class Join>
__device__ __forceinline__ void over_lanes(float (&v)[N], int lane, Join join) {
    int o = 16;
#pragma unroll
    for (int n = N / 2; n > 0; n >>= 1, o >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const bool upper = lane & o;
            const float give = upper ? v[i] : v[i + n], keep = upper ? v[i + n] : v[i];
            v[i] = join(keep, __shfl_xor_sync(0xffffffffu, give, o));
        }
#pragma unroll
    for (; o > 0; o >>= 1) v[0] = join(v[0], __shfl_xor_sync(0xffffffffu, v[0], o));
}
__device__ __forceinline__ bool any_of(int id, int count, bool mine) {  // the block's named barrier, with an answer
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %3, 0;\nbarrier.cta.red.or.pred q, %1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"(id), "r"(count), "r"(static_cast<uint32_t>(mine)) : "memory");
    return any != 0;
}

template <int TERMS, int ROWS>
__global__ void __launch_bounds__(Turned<TERMS, ROWS>::kThreads, 1) attn_tree_turned_kernel(const __grid_constant__ TreeParams p) {
    using M = Turned<TERMS, ROWS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ CtaShared sh;
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kKFull = 0, kKEmpty = 3, kVFull = 6, kVEmpty = 11, kQFull = 16, kSFull = 17, kSFree = 18;
    // one for even, one for odd blocks: a warp may be a block ahead of another here, and a barrier's parity tells two neighbouring phases apart, no more
    constexpr int kPReady = 19, kOFull = 21;
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
        for (int i : {kQFull, kSFree, kPReady, kPReady + 1}) ptx::mbar_init(bar(i), M::kSoftWarps);
        for (int i : {kSFull, kOFull, kOFull + 1}) ptx::mbar_init(bar(i), 1);
        sh.abort = sh.odd = 0;
        ptx::fence_barrier_init();
    }
    if (warp == M::kMmaWarp) {
        tc::tmem_alloc(ptx::smem_u32(&sh.tmem), M::kTmem);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *static_cast<volatile uint32_t *>(&sh.tmem);
    ptx::pdl_wait();
    ptx::pdl_trigger();  // behind the wait: what the merging kernel reads in front of its own is settled then
    const Share share = own_share<ROWS, M::kKeys>(p, sh.line);
    const int u0 = share.u0, u1 = share.u1;
    if (u0 == u1) {
        if (warp == M::kMmaWarp) tc::tmem_dealloc(tmem, M::kTmem);
        return;
    }
    const int group = p.group;
    bool ok = true;
    auto wait = [&](int i, int parity) {
        if (ok) ok = look_and_wait(bar(i), parity, abort);
        return ok;
    };

    if (warp == M::kKWarp || warp == M::kVWarp) {
        produce<M>(p, sh.line, share, ROWS, warp == M::kKWarp, base, bar(warp == M::kKWarp ? kKFull : kVFull), bar(warp == M::kKWarp ? kKEmpty : kVEmpty), abort, ok);
    } else if (warp == M::kMmaWarp) {
        // ================= MMA issue: the warp walks, one lane issues =================
        // D f32, A and B bf16, M = 128, N = terms * rows; for O^T A is MN-major (bit 15)
        constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24), idesc_s = idesc | (static_cast<uint32_t>(M::kQCols >> 3) << 17),
                           idesc_o = idesc | (static_cast<uint32_t>(M::kPCols >> 3) << 17) | (1u << 15);
        const uint64_t q_desc = tc::smem_desc_sw128(base), p_desc = tc::smem_desc_sw128(base + M::kP0);
        int ks = 0, kphase = 0, vs = 0, vphase = 0, n = 0, seg = 0;  // n: the block, in the whole walk
        auto scores = [&]() {
            if (!wait(kKFull + ks, kphase)) return;
            tc::tc_fence_after();
            if (tc::elect_one()) {
                const uint64_t k_desc = tc::smem_desc_sw128(base + M::kK0 + ks * M::kKBytes);
#pragma unroll
                for (int st = 0; st < 8; ++st)
                    tc::umma_f16_ss(tmem, k_desc + static_cast<uint64_t>((st >> 2) * (M::kHalf >> 4) + (st & 3) * 2), q_desc + static_cast<uint64_t>((st >> 2) * (M::kQHalf >> 4) + (st & 3) * 2),
                                    idesc_s, st ? 1u : 0u);
                tc::umma_commit(bar(kSFull));
                tc::umma_commit(bar(kKEmpty + ks));
            }
            __syncwarp();
            if (++ks == M::kKStages) {
                ks = 0;
                kphase ^= 1;
            }
        };
        Segment s = share.first;
        for (int u = u0; u < u1 && ok; ++seg) {
            const int blocks = s.end - s.begin;
            if (wait(kQFull, seg & 1)) scores();
            for (int j = 0; j < blocks && ok; ++j, ++n) {
                if (j + 1 < blocks && wait(kSFree, n & 1)) scores();
                if (!wait(kPReady + (n & 1), n >> 1 & 1)) break;
#pragma unroll 1
                for (int piece = 0; piece < 2; ++piece) {
                    if (!wait(kVFull + vs, vphase)) break;
                    tc::tc_fence_after();
                    if (tc::elect_one()) {
                        const uint64_t v_desc = desc_mn_sw128(base + M::kV0 + vs * M::kPieceBytes, M::kPieceHalf);
#pragma unroll
                        for (int st = 0; st < 4; ++st)  // 16 keys: two groups of V
                            tc::umma_f16_ss(tmem + (1 + (n & 1)) * M::kColO, v_desc + static_cast<uint64_t>(st * (2048 >> 4)),
                                            p_desc + static_cast<uint64_t>((n & 1) * (M::kPBytes >> 4) + piece * (M::kPHalf >> 4) + st * 2), idesc_o,
                                            piece || st ? 1u : 0u);
                        tc::umma_commit(bar(kVEmpty + vs));
                        if (piece) tc::umma_commit(bar(kOFull + (n & 1)));
                    }
                    __syncwarp();
                    if (++vs == M::kVStages) {
                        vs = 0;
                        vphase ^= 1;
                    }
                }
            }
            u += blocks;
            if (u < u1) s = segment_at(p, sh.line, u, u1, ROWS, M::kKeys);
        }
    } else {
        // ================= softmax =================
        constexpr int kR = ROWS / 2;  // rows of a thread
        const int quad = warp & 3, hf = warp >> 2, key = quad * 32 + lane, first = hf * kR;  // the key of a block, and the dimension
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + first;
        float *const s_max = reinterpret_cast<float *>(sm + M::kMax) + first, *const s_part = reinterpret_cast<float *>(sm + M::kPart) + first;  // s_part[quadrant * ROWS + row]
        auto arrive = [&](int i) {
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(i));
        };
        auto meet = [&]() { ptx::named_barrier(1, M::kSoftWarps * 32); };
        auto queries_asked = [&]() { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(kQueriesAsked), "r"(M::kSoftWarps * 32 + 64) : "memory"); };
        auto half_meet = [&]() { ptx::named_barrier(2 + hf, 128); };  // the four warps with the same rows
        // where this thread's probabilities go: column `key` of the operand, row n at n * 128, its 16-byte units XOR-ed with n & 7
        uint8_t *const p_at = sm + M::kP0 + (key >> 6) * M::kPHalf + (key & 7) * 2;
        const int p_unit = (key >> 3) & 7;
        int n = 0;  // blocks so far, over all segments
        Segment s = share.first;
        for (int u = u0; u < u1;) {
            const int pos = s.pos, count = s.count, rows_all = count * group, row0 = s.tile * ROWS;
            const bool nodes = s.end * M::kKeys > pos;  // some blocks hold nodes
            meet();  // nobody reads what the last segment left in the tree's place any more
            // the tile's queries, a row as one load of a warp, all of them asked for before the first is looked at
            constexpr int kEach = ROWS / M::kSoftWarps;
            float4 qv[kEach];
#pragma unroll
            for (int i = 0; i < kEach; ++i) qv[i] = query<TERMS>(p, s.seq, s.kh, group, row0 + warp * kEach + i, rows_all, lane);
            if (u == u0) queries_asked();
            if (nodes) load_parents(p, sh.parent, s.seq, count, M::kSoftWarps * 32);
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                uint2 term[TERMS];
                query_terms<TERMS>(qv[i], term);
                const int r = warp * kEach + i;
#pragma unroll
                for (int x = 0; x < TERMS; ++x)
                    *reinterpret_cast<uint2 *>(sm + (lane >> 4) * M::kQHalf + (x * ROWS + r) * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8) = term[x];
            }
            ptx::fence_proxy_async();  // the tensor core reads them through the asynchronous proxy
            arrive(kQFull);
            if (tid < ROWS) reinterpret_cast<float *>(sm + M::kMax)[tid] = kNoMax;
            meet();
            if (nodes) {
                for (int i = tid; i < count; i += M::kSoftWarps * 32) tree_masks(sh.parent, sh.mask, i);
                meet();
            }
            float acc[kR], l[kR];  // of this thread's dimension; of its key of every block
#pragma unroll
            for (int i = 0; i < kR; ++i) acc[i] = l[i] = 0.0f;
            auto for_rows = [&](auto n_terms, uint32_t at, auto &&give) {  // give(row, the terms' sum)
                constexpr int kChunk = kR < 16 ? kR : 16, kN = decltype(n_terms)::value;
#pragma unroll
                for (int c = 0; c < kR; c += kChunk) {
                    uint32_t w[kN][kChunk];
#pragma unroll
                    for (int x = 0; x < kN; ++x) tc::tmem_ld(at + x * ROWS + c, w[x]);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < kChunk; ++i) {
                        float v = __uint_as_float(w[kN - 1][i]);
#pragma unroll
                        for (int x = kN - 2; x >= 0; --x) v += __uint_as_float(w[x][i]);
                        give(c + i, v);
                    }
                }
            };
            auto add_products = [&](int block) {
                wait(kOFull + (block & 1), block >> 1 & 1);
                tc::tc_fence_after();
                for_rows(std::integral_constant<int, M::kPTerms>(), lanes + (1 + (block & 1)) * M::kColO, [&](int i, float v) { acc[i] += v; });
            };
            for (int j = s.begin; j < s.end; ++j, ++n) {
                float sv[kR];
                bool added = j == s.begin;
                wait(kSFull, n & 1);
                tc::tc_fence_after();
                for_rows(std::integral_constant<int, TERMS>(), lanes, [&](int i, float v) { sv[i] = v * p.scale; });
                tc::tc_fence_before();
                arrive(kSFree);
                const int node = j * M::kKeys + key - pos;  // this thread's key
                if (j * M::kKeys + quad * 32 + 32 > pos && node >= 0) {
#pragma unroll
                    for (int i = 0; i < kR; ++i) {
                        const int row = row0 + first + i;
                        if (node >= count || row >= rows_all || !sees(sh.mask[p.node_of(row)], node)) sv[i] = -INFINITY;
                    }
                }
                bool over = false;
#pragma unroll
                for (int i = 0; i < kR; i += 4) {
                    const float4 m = *reinterpret_cast<const float4 *>(s_max + i);
                    over |= sv[i] > m.x + kSlack || sv[i + 1] > m.y + kSlack || sv[i + 2] > m.z + kSlack || sv[i + 3] > m.w + kSlack;
                }
                if (any_of(2 + hf, 128, over)) {  // the rows' maxima move to this block's
                    if (!added) {
                        add_products(n - 1);
                        added = true;
                    }
                    float most[kR];
#pragma unroll
                    for (int i = 0; i < kR; ++i) most[i] = sv[i];
                    over_lanes<kR>(most, lane, [](float a, float b) { return fmaxf(a, b); });
                    if (lane % (32 / kR) == 0) s_part[quad * ROWS + lane / (32 / kR)] = most[0];
                    half_meet();
                    auto moved = [&](int i) { return fmaxf(fmaxf(fmaxf(s_part[i], s_part[ROWS + i]), fmaxf(s_part[2 * ROWS + i], s_part[3 * ROWS + i])), s_max[i]); };
#pragma unroll
                    for (int i = 0; i < kR; ++i) {
                        const float corr = ex2(s_max[i] - moved(i));
                        acc[i] *= corr;
                        l[i] *= corr;
                    }
                    half_meet();
                    if (quad == 0 && lane < kR) s_max[lane] = moved(lane);
                    half_meet();
                }
#pragma unroll
                for (int i = 0; i < kR; i += 4) {
                    const float4 m = *reinterpret_cast<const float4 *>(s_max + i);
                    sv[i] = ex2(sv[i] - m.x);
                    sv[i + 1] = ex2(sv[i + 1] - m.y);
                    sv[i + 2] = ex2(sv[i + 2] - m.z);
                    sv[i + 3] = ex2(sv[i + 3] - m.w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) l[i + e] += sv[i + e];
                }
                // their place is free: the products of the block in front of the last have been added
#pragma unroll
                for (int i = 0; i < kR; i += 2) {
                    uint32_t term[M::kPTerms];
                    split_pair<M::kPTerms>(sv[i], sv[i + 1], term);
#pragma unroll
                    for (int x = 0; x < M::kPTerms; ++x) {
                        const int r = x * ROWS + first + i;
                        *reinterpret_cast<uint16_t *>(p_at + (n & 1) * M::kPBytes + r * 128 + ((p_unit ^ (r & 7)) << 4)) = static_cast<uint16_t>(term[x]);
                        *reinterpret_cast<uint16_t *>(p_at + (n & 1) * M::kPBytes + (r + 1) * 128 + ((p_unit ^ ((r + 1) & 7)) << 4)) = static_cast<uint16_t>(term[x] >> 16);
                    }
                }
                if (j * M::kKeys + M::kKeys > pos) {  // values past the last node, and values of nodes that are no numbers: a thread half a row of this warp's piece
                    const int piece = 2 * n + hf, vs = piece % M::kVStages, at = j * M::kKeys + hf * 64 + (key & 63) - pos;
                    if (wait(kVFull + vs, (piece / M::kVStages) & 1) && at >= 0 &&
                        clean_values(reinterpret_cast<uint4 *>(sm + M::kV0 + vs * M::kPieceBytes + (key >> 6) * M::kPieceHalf + (key & 63) * 128), 8, at >= count))
                        sh.odd = u + 1;  // read behind a meeting below, written again behind the next segment's first
                }
                ptx::fence_proxy_async();
                tc::tc_fence_before();
                arrive(kPReady + (n & 1));
                if (!added) add_products(n - 1);  // while the tensor core works on this block's
            }
            add_products(n - 1);
            // the rows' weights: over the lanes, then the quadrants
            over_lanes<kR>(l, lane, [](float a, float b) { return a + b; });
            if (lane % (32 / kR) == 0) s_part[quad * ROWS + lane / (32 / kR)] = l[0];
            meet();
            if (nodes && sh.odd == u + 1) {  // what a row sees that is no number
                for (int i = max(0, s.begin * M::kKeys - pos); i < min(count, s.end * M::kKeys - pos); ++i) {
                    const uint16_t v = p.vcache[(static_cast<size_t>(s.seq * p.kvh + s.kh) * p.cap + pos + i) * kHd + key];
                    if ((v & 0x7f80u) != 0x7f80u) continue;
#pragma unroll
                    for (int r = 0; r < kR; ++r)
                        if (row0 + first + r < rows_all && sees(sh.mask[p.node_of(row0 + first + r)], i)) acc[r] += dense::bf16_f32(v);
                }
            }
            const bool whole = s.begin == 0 && s.end == s.blocks;
            const int here = rows_all - row0 - first;  // of this thread's rows
            if (ok && here > 0) {
                auto weight = [&](int r) { return (s_part[r] + s_part[ROWS + r]) + (s_part[2 * ROWS + r] + s_part[3 * ROWS + r]); };
                if (whole) {
                    int at_node = p.node_of(row0 + first), g = row0 + first - at_node * group;
                    size_t at = (static_cast<size_t>(s.seq) * p.t + at_node) * p.out_pitch + (s.kh * group + g) * kHd + key;
#pragma unroll
                    for (int r = 0; r < kR; ++r) {
                        const float x = acc[r] * (1.0f / weight(r));
                        if (r < here) dense::put(static_cast<std::conditional_t<(TERMS > 1), float, uint16_t> *>(p.out) + at, x);
                        const bool next = ++g == group;  // the next row is the next head, or the first head of the next node
                        at += next ? p.out_pitch - (group - 1) * kHd : kHd;
                        g = next ? 0 : g;
                    }
                } else {
                    const size_t part0 = (static_cast<size_t>(blockIdx.x) * 2 + (u == u0 ? 0 : 1)) * ROWS + first;
                    float *to = p.part + part0 * kHd + key;
#pragma unroll
                    for (int r = 0; r < kR; ++r)
                        if (r < here) to[r * kHd] = acc[r];
                    if (quad == 0 && lane < min(kR, here)) p.part_ml[part0 + lane] = make_float2(s_max[lane], weight(lane));
                }
            }
            u += s.end - s.begin;
            if (u < u1) s = segment_at(p, sh.line, u, u1, ROWS, M::kKeys);
        }
    }
    if (!ok && lane == 0) atomicExch(p.err_word, 5);
    tc::tc_fence_before();
    __syncthreads();
    if (warp == M::kMmaWarp) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, M::kTmem);
    }
}

// ---- many rows: tcgen05, tiles of 128 rows ---------------------------------------------------------------
// Blocks of 128 keys. S = Q K^T: the queries' terms and the K block from shared memory, scores in tensor memory. P V: the probabilities' terms from tensor
// memory, the V block as it lies in the cache (its contraction index, the key, is the strided one: the MN-major operand form), with f32 queries every
// block into zeroed sums, which the softmax warps add to the rows in their registers.
//
//   16 softmax warps four to a quadrant of 32 lanes = rows: warps w, w + 4, .. share rows and take 32 of a block's keys, and of the dimensions, each (eight
//                    warps with 64 took 5900 cycles a block in three terms where the products take some 3100: two warps a scheduler do not hide their latencies)
//   K, V producers   a warp each: K blocks of 128 keys are free again after the scores, V in pieces of 64 keys after their product, and one order for
//                    both would have the next K block wait for a piece of V
//   MMA warps        one for P V of block j - 1, one for Q K^T of block j + 1, while the softmax warps work on block j
//
// 512 bytes a key from HBM are 22 cycles of an SM, its products for 128 rows 24 in f32 and 12 in bf16: f32 is bound by the tensor core, bf16 by
// the way of a block's scores through the softmax warps and back: 2700 cycles a block of 128 keys, with 1560 of products and 1150 of exponentials; the block's 64 KB are 2600 of
// an SM's share of HBM, half of that where two tiles share them. us of 36 calls behind one another, weights in one term / in two: 60 nodes of 65000 keys 83 / 99, 16 x 64 of 8100
// keys 112 / 131. Padding rows cost nothing but the products: their warps only keep step.
template <int TERMS>
struct Many {
    static constexpr bool kGoesRound = true;
    static constexpr int kRows = 128, kKeys = 128, kHalf = kKeys * 128, kKBytes = 2 * kHalf;
    static constexpr int kPiece = 64, kPieceHalf = kPiece * 128, kPieceBytes = 2 * kPieceHalf;   // V: 64 keys, two halves of 64 dimensions
    static constexpr int kKStages = TERMS == 3 ? 2 : 3, kVStages = TERMS == 3 ? 3 : 5;
    static constexpr int kK0 = TERMS * 2 * kHalf, kV0 = kK0 + kKStages * kKBytes, kBars = kV0 + kVStages * kPieceBytes;
    static constexpr int kPair = kBars + 256, kSmem = kPair + 2 * 4 * kRows * 4 + 1024;
    static constexpr int kSoftWarps = 16, kKWarp = 16, kVWarp = 17, kScoreWarp = 18, kThreads = 20 * 32;  // the last one: products
    // bf16: the products are summed up in tensor memory, over all blocks, and m is moved as for few rows, with the sums, when a score is over it by kSlack. What the tensor
    // core cuts off of a long sum (some 2e-5 at 8000 keys) does not show in a bf16 result, and a block needs no look at the products of the one in front.
    static constexpr bool kStays = TERMS == 1;
    static constexpr int kPTerms = weight_terms(TERMS);
    // Scores (128 columns) and, when all have been read, the probabilities (64 a term) of even blocks in one place, of odd ones in another
    static constexpr uint32_t kPlace = 192, kColO = 384;
    // A wait for a parity tells a phase from the one in front of it, no more. All roles but one wait for every phase of their barriers, or for one that shows that the phase in
    // front is complete. The one: softmax warps wait for a piece of values only where they clean it (clean_values), in block n for 2n and 2n + 1 at most, having
    // waited for the products of block n - kBehind: in f32 by themselves, in bf16 through the scores of block n, which the score warp asks for behind the products of block
    // n - 2. So piece 2 (n - kBehind) + 1 has landed, and the one that lay in 2n + 1's stage in front of it, 2n + 1 - kVStages, must be none later.
    static constexpr int kBehind = kStays ? 2 : 1;
    static_assert(kVStages >= 2 * kBehind, "the phase in front of the one that is waited for is complete");
    static_assert(kPTerms * 64 <= kPlace && 2 * kPlace <= kColO, "tensor memory");
};
template <int TERMS>
__global__ void __launch_bounds__(Many<TERMS>::kThreads, 1) attn_tree_many_kernel(const __grid_constant__ TreeParams p) {
    using M = Many<TERMS>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ CtaShared sh;
    const uint32_t raw = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kKFull = 0, kKEmpty = 3, kVFull = 6, kVEmpty = 11, kQFull = 16;
    constexpr int kPReady = 17, kOFull = 19, kSFull = 21;  // one for even, one for odd blocks: warps may be a block apart
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
        for (int i : {kQFull, kPReady, kPReady + 1}) ptx::mbar_init(bar(i), M::kSoftWarps);
        for (int i : {kSFull, kSFull + 1, kOFull, kOFull + 1}) ptx::mbar_init(bar(i), 1);
        sh.abort = sh.odd = 0;
        ptx::fence_barrier_init();
    }
    if (warp == M::kScoreWarp) {
        tc::tmem_alloc(ptx::smem_u32(&sh.tmem), 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *static_cast<volatile uint32_t *>(&sh.tmem);
    ptx::pdl_wait();
    ptx::pdl_trigger();  // behind the wait: what the merging kernel reads in front of its own is settled then
    const Share share = own_share<M::kRows, M::kKeys>(p, sh.line);
    const int u0 = share.u0, u1 = share.u1;
    if (u0 == u1) {
        if (warp == M::kScoreWarp) tc::tmem_dealloc(tmem, 512);
        return;
    }
    const int group = p.group;
    bool ok = true;

    // The launch has 20 warps x 96 registers; 4 x 64 + 16 x 104 are as many.
    if (warp >= M::kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == M::kKWarp || warp == M::kVWarp) {
            produce<M>(p, sh.line, share, M::kRows, warp == M::kKWarp, base, bar(warp == M::kKWarp ? kKFull : kVFull), bar(warp == M::kKWarp ? kKEmpty : kVEmpty), abort, ok);
        } else {
            // ================= MMA issue, scores by one warp, products by another: the warps walk, one lane of each issues =================
            // A turn of a wait, products and a commit costs a warp some 400 cycles beside its products, in which those of the other go on: one warp for both took 214 us for
            // 16 x 64 nodes of 8100 keys in f32 where these took 207, and 100 where these took 97 for 60 nodes of 65000 in bf16 (36 calls behind one another; weights in one term
            // then, and walks that did not go round)
            // D f32, A and B bf16, M = 128, N = 128; for P V the B operand is MN-major (bit 16)
            constexpr uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24), idesc_o = idesc_s | (1u << 16);
            auto wait = [&](int i, int parity) {
                if (ok) ok = look_and_wait(bar(i), parity, abort);
                return ok;
            };
            const uint64_t q_desc = tc::smem_desc_sw128(base);
            const bool scores = warp == M::kScoreWarp;
            int stage = 0, phase = 0, n = 0, seg = 0;  // of K or of V; n: the block, in the whole walk
            Segment s = share.first;
            for (int u = u0; u < u1 && ok; ++seg) {
                const int blocks = s.end - s.begin;
                if (scores) wait(kQFull, seg & 1);
                for (int j = 0; j < blocks && ok; ++j, ++n) {
                    if (scores) {
                        // the place of this block's scores: the probabilities of the block but one in front of it have been read (the last segment's all)
                        if (!wait(kKFull + stage, phase) || (j >= 2 && !wait(kOFull + (n & 1), (n - 2) >> 1 & 1))) break;
                        tc::tc_fence_after();
                        if (tc::elect_one()) {
                            const uint64_t k_desc = tc::smem_desc_sw128(base + M::kK0 + stage * M::kKBytes);
#pragma unroll 1
                            for (int x = TERMS - 1; x >= 0; --x)  // the small ones first
#pragma unroll
                                for (int st = 0; st < 8; ++st) {
                                    const uint64_t off = static_cast<uint64_t>((st >> 2) * (M::kHalf >> 4) + (st & 3) * 2);
                                    tc::umma_f16_ss(tmem + (n & 1) * M::kPlace, q_desc + static_cast<uint64_t>(x * 2 * (M::kHalf >> 4)) + off, k_desc + off, idesc_s, x < TERMS - 1 || st ? 1u : 0u);
                                }
                            tc::umma_commit(bar(kSFull + (n & 1)));
                            tc::umma_commit(bar(kKEmpty + stage));
                        }
                        __syncwarp();
                        if (++stage == M::kKStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                        continue;
                    }
                    if (!wait(kPReady + (n & 1), n >> 1 & 1)) break;
#pragma unroll 1
                    for (int piece = 0; piece < 2; ++piece) {
                        if (!wait(kVFull + stage, phase)) break;
                        tc::tc_fence_after();
                        if (tc::elect_one()) {
                            const uint64_t v_desc = desc_mn_sw128(base + M::kV0 + stage * M::kPieceBytes, M::kPieceHalf);
#pragma unroll
                            for (int st = 0; st < 4; ++st)  // 16 keys: 8 columns of P, two groups of V
#pragma unroll
                                for (int x = M::kPTerms - 1; x >= 0; --x)
                                    tc::umma_f16_ts(tmem + M::kColO, tmem + (n & 1) * M::kPlace + x * 64 + (piece * 4 + st) * 8, v_desc + static_cast<uint64_t>(st * (2048 >> 4)), idesc_o, piece || st || x < M::kPTerms - 1 || (M::kStays && j) ? 1u : 0u);
                            tc::umma_commit(bar(kVEmpty + stage));
                            if (piece) tc::umma_commit(bar(kOFull + (n & 1)));
                        }
                        __syncwarp();
                        if (++stage == M::kVStages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
                u += blocks;
                if (u < u1) s = segment_at(p, sh.line, u, u1, M::kRows, M::kKeys);
            }
        }
    } else {
        // ================= softmax =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int quad = warp & 3, part = warp >> 2, r = quad * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
        float *const s_quad = reinterpret_cast<float *>(sm + M::kPair);  // [2][4 parts][128 rows]
        auto wait = [&](int i, int parity) {
            if (ok) ok = look_and_wait(bar(i), parity, abort);
            return ok;
        };
        auto arrive = [&](int i) {
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(bar(i));
        };
        auto meet = [&]() { ptx::named_barrier(1, M::kSoftWarps * 32); };
        auto queries_asked = [&]() { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(kQueriesAsked), "r"(M::kSoftWarps * 32 + 64) : "memory"); };
        auto quad_sync = [&]() { ptx::named_barrier(2 + quad, 128); };  // the four warps of a quadrant
        int n = 0;  // blocks so far, over all segments
        if (lane == 0) sh.seg[warp] = share.first;
        __syncwarp();
        for (int u = u0; u < u1;) {
            const Segment s = sh.seg[warp];
            const int pos = s.pos, count = s.count;
            const int rows_all = count * group, row0 = s.tile * M::kRows, row = row0 + r, node = p.node_of(row);
            const bool nodes = s.end * M::kKeys > pos, live = row0 + quad * 32 < rows_all;  // some blocks hold nodes; some row of the warp exists
            meet();  // nobody reads what the last segment left in the queries' place and in the tree's any more
            // the tile's queries, a row as one load of a warp, all of them asked for before the first is looked at; in the K-major SWIZZLE_128B layout
            // (row r of a half at r * 128, its 16-byte units XOR-ed with r & 7)
            float4 qv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) qv[i] = query<TERMS>(p, s.seq, s.kh, group, row0 + warp * 8 + i, rows_all, lane);
            if (u == u0) queries_asked();
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
                    for (int i = 0; i < 16; i += 2) {
                        const float2 x = ptx::fma2(make_float2(acc[c * 16 + i], acc[c * 16 + i + 1]), make_float2(corr, corr), make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
                        acc[c * 16 + i] = x.x;
                        acc[c * 16 + i + 1] = x.y;
                    }
                }
            };
            int j = first_block(share, s, u, group, M::kRows);
            for (int left = s.end - s.begin; left > 0; --left, ++n, j = j + 1 == s.end ? s.begin : j + 1) {
                const bool begun = left < s.end - s.begin;
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
                    for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = ptx::max3(mx[(i >> 1) & 3], __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                    float *quarter = s_quad + (n & 1) * 4 * M::kRows + r;
                    quarter[part * M::kRows] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    quad_sync();  // the row's scores have all been read; the next block but one writes here again, behind the next block's meeting
                    const float all = fmaxf(fmaxf(quarter[0], quarter[M::kRows]), fmaxf(quarter[2 * M::kRows], quarter[3 * M::kRows]));
                    const float top = all * p.scale, nm = M::kStays ? (top > m + kSlack ? top : m) : fmaxf(m, top);
                    step = ex2(m - nm);
                    if (M::kStays && begun && __any_sync(0xffffffffu, nm != m)) {  // the same in the quadrant's four warps
                        wait(kOFull + ((n - 1) & 1), (n - 1) >> 1 & 1);  // the sums are complete and nothing is added before this block's probabilities are there
                        tc::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            uint32_t v[16];
                            tc::tmem_ld16(lanes + M::kColO + part * 32 + c * 16, v);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * step);
                            tc::tmem_st16(lanes + M::kColO + part * 32 + c * 16, v);
                        }
                    }
                    m = nm;
                    float2 sum = make_float2(0.0f, 0.0f);
                    const float2 scale2 = make_float2(p.scale, p.scale), less = make_float2(-nm, -nm);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[M::kPTerms][8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 d = ptx::fma2(make_float2(__uint_as_float(sv[c * 16 + 2 * i]), __uint_as_float(sv[c * 16 + 2 * i + 1])), scale2, less), e = make_float2(ex2(d.x), ex2(d.y));
                            sum = ptx::add2(sum, e);
                            uint32_t term[M::kPTerms];
                            split_pair<M::kPTerms>(e.x, e.y, term);
#pragma unroll
                            for (int x = 0; x < M::kPTerms; ++x) w[x][i] = term[x];
                        }
#pragma unroll
                        for (int x = 0; x < M::kPTerms; ++x) tc::tmem_st8(place + x * 64 + part * 16 + c * 8, w[x]);
                    }
                    l = l * step + (sum.x + sum.y);
                }
                // the products of the block in front are added, then their place is free; the values of that block have landed and been read then
                if (!M::kStays) {
                    if (begun) {
                        wait(kOFull + ((n - 1) & 1), (n - 1) >> 1 & 1);
                        if (live) add_products();
                    }
                    corr = step;
                }
                if (j * M::kKeys + M::kKeys > pos) {  // values past the last node, and values of nodes that are no numbers: a thread 32 dimensions of a row of this warp's piece
                    const int piece = 2 * n + (part >> 1), vs = piece % M::kVStages, quarter = (part & 1) * 2 + (r >> 6), key = r & 63, at = j * M::kKeys + (part >> 1) * 64 + key - pos;
                    if (wait(kVFull + vs, (piece / M::kVStages) & 1) && at >= 0 &&
                        clean_values(reinterpret_cast<uint4 *>(sm + M::kV0 + vs * M::kPieceBytes + (quarter >> 1) * M::kPieceHalf + key * 128 + (quarter & 1) * 64), 4, at >= count))
                        sh.odd = u + 1;  // read behind a meeting below, written again behind the next segment's first
                    ptx::fence_proxy_async();
                }
                if (live) tc::tmem_st_wait();
                tc::tc_fence_before();
                arrive(kPReady + (n & 1));
            }
            wait(kOFull + ((n - 1) & 1), (n - 1) >> 1 & 1);
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
            if (u < u1) {
                const Segment next = segment_at(p, sh.line, u, u1, M::kRows, M::kKeys);
                if (lane == 0) sh.seg[warp] = next;
                __syncwarp();
            }
        }
    }
    if (!ok && lane == 0) atomicExch(p.err_word, 5);
    tc::tc_fence_before();
    __syncthreads();
    if (warp == M::kScoreWarp) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of the tiles that were cut. Every block lists them, a thread a worker: the tile that begins in its share and ends behind it, if there is one. Their rows are
// cut evenly among the warps, a warp a row, or, of few rows, 2, 4 or 8 warps, which take every 2nd, 4th or 8th part of it; four dimensions a lane. (us in f32 against
// eight blocks for each worker, most of which had no tile: 1 x 5 nodes of 4001 keys 16.8 -> 12.8, 1 x 60 of 2000 keys, 16 tiles in 10 parts, 40.7 -> 25.4, 16 x 64 of 300 keys 34.4 -> 29.9.)
constexpr int kMergeWarps = 8, kMergeAtOnce = 4, kMergeBlocks = 4;  // parts on their way; blocks an SM
constexpr int kMaxWorkers = kMergeWarps * 32;
template <int TERMS, int ROWS, int KEYS>
__global__ void __launch_bounds__(kMergeWarps * 32, kMergeBlocks) attn_tree_merge_kernel(const __grid_constant__ TreeParams p) {
    __shared__ Line line;
    __shared__ int s_first[kMaxWorkers];   // rows in front of a worker's tile
    __shared__ int4 s_tile[kMaxWorkers];   // sequence, KV head, tile, parts; negative: the first part is its worker's second
    __shared__ int s_warp[kMergeWarps], s_most[kMergeWarps];
    __shared__ float4 s_sum[kMergeWarps][32];
    __shared__ float2 s_ml[kMergeWarps];
    ptx::pdl_trigger();
    cut_line<ROWS, KEYS>(p, line);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = p.group;
    {
        const Shares shares(line.first[p.b], p);
        const int u0 = shares.begin(tid), u1 = tid < p.workers ? shares.begin(tid + 1) : u0;
        int rows = 0, parts = 0;
        if (u0 < u1) {
            const Segment s = segment_at(p, line, u1 - 1, u1, ROWS, KEYS);  // the last block of the share
            const int begin = u1 - 1 - s.begin, end = begin + s.blocks;
            if (begin >= u0 && end > u1) {
                parts = shares.owner(end - 1) - tid + 1;  // neighbours that all have a share: this tile goes on in it
                rows = min(ROWS, s.count * group - s.tile * ROWS);
                s_tile[tid] = make_int4(s.seq, s.kh, s.tile, u0 < begin ? -parts : parts);
            }
        }
        const int sum = sum_up_to(rows, lane);
        const int most = __reduce_max_sync(0xffffffffu, parts);
        if (lane == 31) {
            s_warp[warp] = sum;
            s_most[warp] = most;
        }
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += s_warp[w];
        s_first[tid] = before + sum - rows;
    }
    int all = 0, most = 0;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
        all += s_warp[w];
        most = max(most, s_most[w]);
    }
    __syncthreads();
    int splits = kMergeWarps;
    while (splits > 1 && (all * splits > static_cast<int>(gridDim.x) * kMergeWarps || splits * kMergeAtOnce >= 2 * most)) splits >>= 1;
    const int split = warp & (splits - 1), each = kMergeWarps / splits;
    auto worker_of = [&](int index) {  // the last one with `index` rows or fewer in front of its tile
        int c = 0;
#pragma unroll
        for (int step = kMaxWorkers / 2; step > 0; step >>= 1)
            if (s_first[c + step] <= index) c += step;
        return c;
    };
    int index = blockIdx.x * each + warp / splits, c0 = worker_of(index);
    ptx::pdl_wait();  // blocks without a row too: the next kernel of the stream waits for this one only
    for (int r0 = blockIdx.x * each; r0 < all; r0 += gridDim.x * each, index += gridDim.x * each, c0 = worker_of(index)) {
        const int r = index - s_first[c0];
        const int4 tile = s_tile[c0];
        const int parts = index < all ? abs(tile.w) : 0;
        // part i is the first of its worker's two, but the tile's own first part is the second where the worker came from another tile
        auto place = [&](int i) { return (static_cast<size_t>(c0 + i) * 2 + (i == 0 && tile.w < 0 ? 1 : 0)) * ROWS + r; };
        float m = kNoMax, l = 0.0f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = split; i0 < parts; i0 += splits * kMergeAtOnce) {
            float2 ml[kMergeAtOnce];
            float4 x[kMergeAtOnce];
            float up = m;
#pragma unroll
            for (int e = 0; e < kMergeAtOnce; ++e) {
                const int i = i0 + e * splits;
                ml[e] = make_float2(kNoMax, 0.0f);
                x[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < parts) {
                    ml[e] = p.part_ml[place(i)];
                    x[e] = *reinterpret_cast<const float4 *>(p.part + place(i) * kHd + lane * 4);
                }
            }
#pragma unroll
            for (int e = 0; e < kMergeAtOnce; ++e) up = fmaxf(up, ml[e].x);
            const float corr = ex2(m - up);
            m = up;
            l *= corr;
            sum = make_float4(sum.x * corr, sum.y * corr, sum.z * corr, sum.w * corr);
#pragma unroll
            for (int e = 0; e < kMergeAtOnce; ++e) {
                const float w = ex2(ml[e].x - m);
                l += ml[e].y * w;
                sum.x += x[e].x * w;
                sum.y += x[e].y * w;
                sum.z += x[e].z * w;
                sum.w += x[e].w * w;
            }
        }
        if (splits > 1) {
            s_sum[warp][lane] = sum;
            if (lane == 0) s_ml[warp] = make_float2(m, l);
            __syncthreads();
            if (!split)
                for (int e = 1; e < splits; ++e) {
                    const float2 ml = s_ml[warp + e];
                    const float4 x = s_sum[warp + e][lane];
                    const float up = fmaxf(m, ml.x), corr = ex2(m - up), w = ex2(ml.x - up);
                    m = up;
                    l = l * corr + ml.y * w;
                    sum = make_float4(sum.x * corr + x.x * w, sum.y * corr + x.y * w, sum.z * corr + x.z * w, sum.w * corr + x.w * w);
                }
            __syncthreads();
        }
        if (split || !parts) continue;
        const int row = tile.z * ROWS + r, node = p.node_of(row);
        const float inv = 1.0f / l;
        const size_t at = (static_cast<size_t>(tile.x) * p.t + node) * p.out_pitch + static_cast<size_t>(tile.y * group + row - node * group) * kHd + lane * 4;
        dense::put4(static_cast<std::conditional_t<(TERMS > 1), float, uint16_t> *>(p.out) + at, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
    }
}

int attn_tree_init(Ctx *ctx) {
    struct { void (*k)(TreeParams); int smem; } kernels[] = {
        {attn_tree_turned_kernel<1, 16>, Turned<1, 16>::kSmem}, {attn_tree_turned_kernel<3, 16>, Turned<3, 16>::kSmem}, {attn_tree_turned_kernel<1, 32>, Turned<1, 32>::kSmem},
        {attn_tree_turned_kernel<3, 32>, Turned<3, 32>::kSmem}, {attn_tree_many_kernel<1>, Many<1>::kSmem},             {attn_tree_many_kernel<3>, Many<3>::kSmem}};
    for (auto &f : kernels) LBK_CUDA(cudaFuncSetAttribute(f.k, cudaFuncAttributeMaxDynamicSharedMemorySize, f.smem));
    return LBK_OK;
}
const InitHook kInitAttnTree(attn_tree_init);

// Rows of a tile for t nodes of `group` heads.
int tile_rows(size_t t, size_t group) { return t * group <= 16 ? 16 : t * group <= 32 ? 32 : 128; }

template <int TERMS, int ROWS>
int launch_tree(Ctx *ctx, TreeParams &p, cudaStream_t st) {
    using T = Turned<TERMS, ROWS <= 32 ? ROWS : 16>;
    using M = Many<TERMS>;
    if (ROWS <= 32) LBK_CUDA(launch_chained(attn_tree_turned_kernel<TERMS, ROWS <= 32 ? ROWS : 16>, dim3(static_cast<unsigned>(p.workers)), dim3(T::kThreads), static_cast<size_t>(T::kSmem), st, p));
    else LBK_CUDA(launch_chained(attn_tree_many_kernel<TERMS>, dim3(static_cast<unsigned>(p.workers)), dim3(M::kThreads), static_cast<size_t>(M::kSmem), st, p));
    ctx->launches++;
    LBK_CUDA(launch_chained(attn_tree_merge_kernel<TERMS, ROWS, 128>, dim3(static_cast<unsigned>(std::min<size_t>(static_cast<size_t>(kMergeBlocks) * ctx->sm_count, static_cast<size_t>(p.b) * p.t * p.kvh * p.group))), dim3(kMergeWarps * 32), 0, st, p));
    ctx->launches++;
    return LBK_OK;
}
template <int TERMS>
int launch_tree(Ctx *ctx, int tile, TreeParams &p, cudaStream_t st) {
    return tile == 16 ? launch_tree<TERMS, 16>(ctx, p, st) : tile == 32 ? launch_tree<TERMS, 32>(ctx, p, st) : launch_tree<TERMS, 128>(ctx, p, st);
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
    p.group = static_cast<int>(group);
    p.kvh = static_cast<int>(kv_heads);
    p.cap = static_cast<int>(cap);
    p.scale = scale * 1.4426950408889634f;
    p.workers = std::min(ctx->sm_count, kMaxWorkers);
    p.per_worker = static_cast<unsigned>(std::min<unsigned long long>((1ull << 32) / static_cast<unsigned>(p.workers), 0xffffffffu));
    p.per_group = group > 1 ? static_cast<unsigned>((0x100000000ull + group - 1) / group) : 0u;  // exact: rows * heads of a group < 2^32
    p.err_word = ctx->err_word;
    const int tile = tile_rows(t, group);
    p.part = scratch_dev;
    p.part_ml = reinterpret_cast<float2 *>(scratch_dev + static_cast<size_t>(p.workers) * 2 * tile * kHd);
    LBK_TRY(encode_bytes_map(&p.k, kcache_dev, 256, rows, 256, 128, 128));
    LBK_TRY(encode_bytes_map(&p.v, vcache_dev, 256, rows, 256, 128, 64));
    return compute == LBK_COMPUTE_F32 ? launch_tree<3>(ctx, tile, p, st) : launch_tree<1>(ctx, tile, p, st);
}

}  // extern "C"
