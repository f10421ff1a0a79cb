// Log probabilities of given tokens, entropy and the best alternatives of rows of logits.
//
//   c = scale * x;  lse = log sum_j exp(c_j);  logprob(token) = c_token - lse;  H = lse - sum_j p_j c_j
//   alternatives: the `top` largest logits, the lower id first among equal ones, with their log probabilities
//
// The reference has the greedy token only (crates/lb-model/src/sample.rs:17-25).
#include <algorithm>
#include <cfloat>

#include "lbk_dense_dev.cuh"
#include "lbk_tree.cuh"

namespace lbk {

namespace {

using dense::get;
template <typename T>
struct Empty {  // sixteen bytes of -inf
    static __device__ __forceinline__ uint4 vector() {
        const unsigned v = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
        return make_uint4(v, v, v, v);
    }
};

struct ScoreParams {
    const void *logits;
    size_t pitch;
    int vocab;
    const int *tokens;
    int given;
    float scale;
    int top;
    float *logprobs, *entropy;
    int *top_ids;
    float *top_logprobs;
};

// A place in the order of the alternatives: larger values first, then lower ids; every NaN in front of every number, as a sort has it. 0 is
// behind every place, kInFront in front of every one: ids are below 2^30, so the lower word has its upper bit clear.
constexpr unsigned kLastId = 0x7fffffffu;
constexpr unsigned long long kInFront = ~0ull;
__device__ __forceinline__ unsigned order_value(float x) {  // the order of numbers as that of whole ones
    const unsigned bits = __float_as_uint(x + 0.0f);         // -0 and 0 are equal
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    return static_cast<unsigned long long>(x != x ? 0xffffffffu : order_value(x)) << 32 | (kLastId - static_cast<unsigned>(id));
}
__device__ __forceinline__ int key_id(unsigned long long key) { return static_cast<int>(kLastId - static_cast<unsigned>(key)); }

// One pass over the row. A thread keeps the maximum m of what it has seen, s = sum e^(c (x - m)) and t = sum e^(c (x - m)) (x - m); entropy = log s - c t / s.
//
// The alternatives come out of the same pass. Eight threads show their maximum, and at least `top` values reach the `top`-th
// largest of the 32 maxima that are shown: what lies below it is none of the alternatives. Values that reach it go to a list in shared memory, a hundred or so of 128256; the
// bound is looked for again after 2, 4, 8, .. trips, without a barrier (what other threads show may be old: a bound all the same). At the end the list is put in
// order. Rows whose list runs over (most values equal, or ascending), or has too few (most of them -inf), and rows with a NaN or +inf are read again, once an
// alternative.
//
// Bytes bound it: 2000 rows of 128256 f32 are 1.03 GB. A row is cut among the CTAs of a cluster where there are fewer rows than the SMs hold CTAs; they
// meet through distributed shared memory.
constexpr int kThreads = 256, kWarps = kThreads / 32, kLoads = 4;  // 16-byte loads of a thread in flight
constexpr int kList = 2048, kOrder = 512;  // keys on the list; how many of them are put in order by comparing all
constexpr int kTop = LBK_LOGPROBS_TOP, kClusterMost = 16;
static_assert(kThreads == 8 * kTop && kClusterMost * kTop <= kOrder && kClusterMost <= 32, "a maximum of eight threads for each alternative");
using Key = unsigned long long;

struct Stats {
    float m, s, t;
};
__device__ __forceinline__ float ex2(float x) {  // 2^x, the hardware's approximation
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The sums of a part, brought to a maximum that is no less; c is log2(e) * scale. A part that is empty stays it.
__device__ __forceinline__ void raise(Stats &a, float m, float c) {
    const float d = a.m - m, r = ex2(d * c);
    a.t = r == 0.0f ? 0.0f : r * (a.t + a.s * d);  // s * d may be -inf then
    a.s *= r;
    a.m = m;
}
__device__ __forceinline__ Stats join_warp(Stats a, float c) {
    raise(a, value_of(__reduce_max_sync(0xffffffffu, order_value(a.m))), c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return a;
}
using ptx::add2;
using ptx::fma2;
using ptx::mul2;
__device__ __forceinline__ void unpack(const uint4 &v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4 &v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// What a thread has seen: its maximum, and the sums brought to it, of every other value each.
struct Seen {
    float m = -FLT_MAX;
    float2 s{0.0f, 0.0f}, t{0.0f, 0.0f};
    __device__ __forceinline__ void reach(float high, float c) {
        if (!(high > m)) return;
        const float d = m - high, r = ex2(d * c);
        t = r == 0.0f ? make_float2(0.0f, 0.0f) : mul2(make_float2(r, r), fma2(s, make_float2(d, d), t));  // s * d may be -inf for the nothing in front
        s = mul2(s, make_float2(r, r));
        m = high;
    }
    __device__ __forceinline__ void add(float2 v, float c) {  // v.x, v.y <= m, or NaN
        const float2 d = add2(v, make_float2(-m, -m)), f = mul2(d, make_float2(c, c)), e = make_float2(ex2(f.x), ex2(f.y));
        s = add2(s, e);
        t = fma2(e, make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), t);  // 0 * -inf is nothing here
    }
    __device__ __forceinline__ Stats stats() const { return {m, s.x + s.y, t.x + t.y}; }
};
// A row as it lies: `lead` values up to the first 16-byte boundary, `vectors` of 16 bytes, the rest.
template <typename T>
struct Row {
    static constexpr int kVec = 16 / sizeof(T);
    const T *x;
    int lead, vectors, odd;  // odd: values that are in no vector
    __device__ __forceinline__ Row(const ScoreParams &p, size_t row) : x(static_cast<const T *>(p.logits) + row * p.pitch) {
        lead = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
        vectors = (p.vocab - lead) / kVec;
        odd = p.vocab - vectors * kVec;
    }
    __device__ __forceinline__ const uint4 *units() const { return reinterpret_cast<const uint4 *>(x + lead); }
    __device__ __forceinline__ int odd_id(int i) const { return i < lead ? i : i + vectors * kVec; }
    __device__ __forceinline__ int id(int vector, int e) const { return lead + vector * kVec + e; }
};
// The results of a row whose statistics are known
struct Results {
    float m, log_s, scale;
    __device__ __forceinline__ Results(const Stats &a, float scale) : m(a.m), log_s(logf(a.s)), scale(scale) {}
    __device__ __forceinline__ float logprob(float v) const { return (0.5f * v - 0.5f * m) * scale * 2.0f - log_s; }  // halves: v - m may be more than f32 has
    __device__ __forceinline__ float entropy(const Stats &a) const { return log_s - a.t / a.s * scale; }
};
__device__ __forceinline__ float key_value(Key key) { return value_of(static_cast<unsigned>(key >> 32)); }
__device__ __forceinline__ Key warp_max(Key key) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    return key;
}
// how many of n keys are larger
__device__ __forceinline__ int rank_of(const Key *keys, int n, Key mine) {
    int rank = 0, i = 0;
    for (; i + 8 <= n; i += 8) {
        ulonglong2 two[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) two[e] = *reinterpret_cast<const ulonglong2 *>(keys + i + 2 * e);
#pragma unroll
        for (int e = 0; e < 4; ++e) rank += (two[e].x > mine) + (two[e].y > mine);
    }
    for (; i < n; ++i) rank += keys[i] > mine;
    return rank;
}
// Of 32 maxima that are shown, the one of rank top - 1, by a warp: a lane finds the rank of one of them; true for the lane that has it
__device__ __forceinline__ bool has_rank(const unsigned *shown, int lane, int top, unsigned &mine) {
    mine = shown[lane];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kTop; i += 4) {
        const uint4 other = *reinterpret_cast<const uint4 *>(shown + i);
        rank += (other.x > mine || (other.x == mine && i < lane)) + (other.y > mine || (other.y == mine && i + 1 < lane)) + (other.z > mine || (other.z == mine && i + 2 < lane)) +
                (other.w > mine || (other.w == mine && i + 3 < lane));
    }
    return rank == top - 1;
}

// ---- short rows: a warp a row ---------------------------------------------------------------------------
// One walk for the sums and the lanes' maxima, one, from L1 and L2, for the values that reach the `top`-th largest of those. No barrier: a block's meetings are some 5 us a
// row, and a warp has nothing of them, but takes longer for what is long. us, a block a row / a warp a row: 883 rows of 182 bf16 15.1 / 4.0, 2000 rows of 2000 f32 20.7 / 11.8, 1356 rows
// of 4721 bf16 19.7 / 16.5, 2000 rows of 5000 f32 26.7 / 22.2, of 8192 33.7 / 36.8; 100 rows of 5000 f32 5.9 / 13.5. So: where there are more rows than the SMs hold
// blocks, up to kShortBytes a row; in any case up to kTinyBytes.
constexpr int kShortWarps = 8, kShortList = 256, kShortBytes = 20480, kTinyBytes = 2048;
template <typename T>
__global__ void __launch_bounds__(kShortWarps * 32) logprobs_short_kernel(const ScoreParams p, int rows) {
    constexpr int kVec = 16 / sizeof(T);
    __shared__ alignas(16) Key s_list[kShortWarps][kShortList];
    __shared__ alignas(16) unsigned s_shown[kShortWarps][kTop];
    __shared__ int s_count[kShortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t row = static_cast<size_t>(blockIdx.x) * (blockDim.x >> 5) + warp;
    ptx::pdl_trigger();
    ptx::pdl_wait();
    if (row >= static_cast<size_t>(rows)) return;
    const Row<T> r(p, row);
    const uint4 *units = r.units();
    const float c = p.scale * 1.4426950408889634f, odd_value = lane < r.odd ? get(r.x + r.odd_id(lane)) : -INFINITY;
    const bool one_given = lane < p.given;
    const int token0 = one_given ? p.tokens[row * p.given + lane] : -1;
    const float given0 = token0 >= 0 && token0 < p.vocab ? get(r.x + token0) : 0.0f;
    if (lane == 0) s_count[warp] = 0;
    Seen seen;
    uint4 raw[kLoads], next[kLoads];
    auto ask = [&](uint4 (&into)[kLoads], int base) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int i = base + u * 32 + lane;
            into[u] = i < r.vectors ? units[i] : Empty<T>::vector();
        }
    };
    ask(next, 0);
    seen.reach(odd_value, c);
    seen.add(make_float2(odd_value, -INFINITY), c);
    for (int base = 0; base < r.vectors; base += 32 * kLoads) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) raw[u] = next[u];
        ask(next, base + 32 * kLoads);  // on their way while these are looked at
        float high = -INFINITY;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < kVec; ++e) high = fmaxf(high, v[e]);
        }
        seen.reach(high, c);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < kVec; e += 2) seen.add(make_float2(v[e], v[e + 1]), c);
        }
    }
    const Stats a = join_warp(seen.stats(), c);
    const Results result(a, p.scale);
    const float none = __uint_as_float(0x7fc00000u);
    if (lane == 0 && p.entropy) p.entropy[row] = result.entropy(a);
    if (one_given) p.logprobs[row * p.given + lane] = token0 >= 0 && token0 < p.vocab ? result.logprob(given0) : none;
    for (int g = lane + 32; g < p.given; g += 32) {
        const int token = p.tokens[row * p.given + g];
        p.logprobs[row * p.given + g] = token >= 0 && token < p.vocab ? result.logprob(get(r.x + token)) : none;
    }
    if (!p.top) return;
    auto put = [&](int place, Key key) {
        p.top_ids[row * p.top + place] = key_id(key);
        p.top_logprobs[row * p.top + place] = result.logprob(key_value(key));
    };
    s_shown[warp][lane] = order_value(seen.m);
    __syncwarp();
    unsigned mine;
    const unsigned who = __ballot_sync(0xffffffffu, has_rank(s_shown[warp], lane, p.top, mine));
    const float floor = fmaxf(-FLT_MAX, value_of(__shfl_sync(0xffffffffu, mine, __ffs(who) - 1)));  // what a value has to reach; -inf never does
    auto list = [&](float v, int id) {
        if (v >= floor) {
            const int at = atomicAdd(&s_count[warp], 1);
            if (at < kShortList) s_list[warp][at] = order_key(v, id);
        }
    };
    list(odd_value, r.odd_id(lane));
#pragma unroll 4
    for (int i = lane; i < r.vectors; i += 32) {
        float v[kVec], high;
        unpack(units[i], v);
        high = v[0];
#pragma unroll
        for (int e = 1; e < kVec; ++e) high = fmaxf(high, v[e]);
        if (!(high < floor)) {
#pragma unroll
            for (int e = 0; e < kVec; ++e) list(v[e], r.id(i, e));
        }
    }
    __syncwarp();
    const int n = s_count[warp];
    if (n <= kShortList && n >= p.top && a.s == a.s && a.s <= FLT_MAX) {
        for (int k = lane; k < n; k += 32) {
            const Key key = s_list[warp][k];
            const int rank = rank_of(s_list[warp], n, key);
            if (rank < p.top) put(rank, key);
        }
        return;
    }
    Key last = kInFront;  // the largest value behind the last one found, `top` times over
    for (int k = 0; k < p.top; ++k) {
        Key best = 0;
        auto look = [&](float v, int id) {
            const Key key = order_key(v, id);
            if (key < last && key > best) best = key;
        };
        for (int i = lane; i < r.vectors; i += 32) {
            float v[kVec];
            unpack(units[i], v);
#pragma unroll
            for (int e = 0; e < kVec; ++e) look(v[e], r.id(i, e));
        }
        if (lane < r.odd) look(odd_value, r.odd_id(lane));
        last = warp_max(best);
        if (lane == 0) put(k, last);
    }
}

// ---- long rows: a block a row, or a cluster -----------------------------------------------------------------
struct alignas(16) RowShared {
    Key list[kList];
    Key best[kOrder];          // the keys that are put in order
    Key gathered[kOrder];      // all CTAs' alternatives
    Key top[kTop];             // this CTA's alternatives, in order
    Key warp_key[kWarps];
    alignas(16) unsigned shown[kTop];  // order_value of eight threads' maxima
    Stats warp_stats[kWarps], stats, cta_stats[kClusterMost];
    float bound;
    int count, kept;
};

// The `top` largest of n keys of the shared memory, in order, into `out`, zeros behind them. n > kOrder: a search for each.
__device__ void put_in_order(const Key *keys, int n, int top, Key *out, Key *warp_key) {
    const int tid = threadIdx.x;
    if (tid < top) out[tid] = 0;
    __syncthreads();
    if (n <= kOrder) {
        for (int k = tid; k < n; k += kThreads) {
            const Key mine = keys[k];
            const int rank = rank_of(keys, n, mine);
            if (rank < top && mine) out[rank] = mine;
        }
        __syncthreads();
        return;
    }
    Key last = kInFront;
    for (int k = 0; k < top && last; ++k) {
        Key best = 0;
        for (int i = tid; i < n; i += kThreads)
            if (keys[i] < last && keys[i] > best) best = keys[i];
        best = warp_max(best);
        if ((tid & 31) == 0) warp_key[tid >> 5] = best;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) best = max(best, warp_key[w]);
        if (tid == 0) out[k] = best;
        last = best;
        __syncthreads();
    }
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t of_cta(const void *p, uint32_t rank) {  // the same place in another CTA of the cluster
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(p)), "r"(rank));
    return a;
}

// ctas: how many share a row, neighbours in the grid and a cluster
template <typename T>
__global__ void __launch_bounds__(kThreads, 3) logprobs_kernel(const ScoreParams p, int ctas) {
    constexpr int kVec = 16 / sizeof(T);
    __shared__ RowShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = ctas > 1 ? cluster_rank() : 0;
    const size_t row = blockIdx.x / ctas;
    const Row<T> r(p, row);
    const T *x = r.x;
    const uint4 *units = r.units();
    const float c = p.scale * 1.4426950408889634f;
    // this CTA's vectors v0 .. v1 - 1; the odd values are the first CTA's
    const int vectors = r.vectors, odd = rank == 0 ? r.odd : 0, lead = r.lead, each = vectors / ctas, more = vectors - each * ctas;
    const int v0 = each * rank + min(static_cast<int>(rank), more), v1 = v0 + each + (static_cast<int>(rank) < more ? 1 : 0);
    if (tid == 0) {
        sh.count = sh.kept = 0;
        sh.bound = -FLT_MAX;  // what a value has to reach to go on the list; -inf never does
    }
    if (ctas > 1) cluster_arrive();
    ptx::pdl_trigger();
    ptx::pdl_wait();

    Seen seen;
    auto show = [&]() {
        float most = seen.m;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if ((tid & 7) == 0) sh.shown[tid >> 3] = order_value(most);
    };
    auto look_up = [&]() {  // one warp
        unsigned mine;
        if (has_rank(sh.shown, lane, p.top, mine)) sh.bound = fmaxf(sh.bound, value_of(mine));
    };
    float floor = -FLT_MAX;
    auto list = [&](float v, int id) {
        if (v >= floor) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.list[at] = order_key(v, id);
        }
    };
    const float odd_value = tid < odd ? get(x + r.odd_id(tid)) : -INFINITY;
    const int odd_id = r.odd_id(tid);
    // the first tokens' values are asked for now
    const bool one_given = rank == 0 && tid < p.given;
    const int token0 = one_given ? p.tokens[row * p.given + tid] : -1;
    const float given0 = token0 >= 0 && token0 < p.vocab ? get(x + token0) : 0.0f;
    uint4 raw[kLoads], next[kLoads];
    auto ask = [&](uint4 (&into)[kLoads], int base) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int i = base + u * kThreads + tid;
            into[u] = i < v1 ? __ldcs(units + i) : Empty<T>::vector();
        }
    };
    ask(next, v0);
    int trip = 0;
    for (int base = v0; base < v1 || trip == 0; base += kThreads * kLoads, ++trip) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) raw[u] = next[u];
        ask(next, base + kThreads * kLoads);  // on their way while these are looked at
        float high = trip == 0 ? odd_value : -INFINITY, vector_high[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
            vector_high[u] = v[0];
#pragma unroll
            for (int e = 1; e < kVec; ++e) vector_high[u] = fmaxf(vector_high[u], v[e]);
            high = fmaxf(high, vector_high[u]);
        }
        seen.reach(high, c);
        if (trip == 0) seen.add(make_float2(odd_value, -INFINITY), c);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < kVec; e += 2) seen.add(make_float2(v[e], v[e + 1]), c);
        }
        if (p.top) {
            if ((trip & (trip + 1)) == 0) {  // after 1, 2, 4, .. trips
                show();
                if (trip == 0) __syncthreads();
                if (warp == 0) look_up();
                if (trip == 0) __syncthreads();
            }
            floor = *static_cast<const volatile float *>(&sh.bound);
            if (high >= floor) {
                if (trip == 0) list(odd_value, odd_id);
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    if (vector_high[u] < floor) continue;
                    float v[kVec];
                    unpack(raw[u], v);
#pragma unroll
                    for (int e = 0; e < kVec; ++e) list(v[e], lead + (base + u * kThreads + tid) * kVec + e);
                }
            }
        }
    }
    if (p.top) show();
    Stats a = join_warp(seen.stats(), c);
    if (lane == 0) sh.warp_stats[warp] = a;
    __syncthreads();
    if (p.top && warp == 1) look_up();
    if (warp == 0) {
        a = join_warp(lane < kWarps ? sh.warp_stats[lane] : Stats{-FLT_MAX, 0.0f, 0.0f}, c);
        if (lane == 0) sh.stats = a;
    }
    if (p.top) {
        __syncthreads();
        const int n = sh.count, here = (v1 - v0) * kVec + odd, want = min(p.top, here);
        const float s = sh.stats.s;
        floor = sh.bound;
        if (n <= kList && n >= want && s == s && s <= FLT_MAX) {
            // what reaches the last bounds
            const Key least = order_key(floor, kLastId);
            for (int i = tid; i < n; i += kThreads)
                if (sh.list[i] >= least) {
                    const int at = atomicAdd(&sh.kept, 1);
                    if (at < kOrder) sh.best[at] = sh.list[i];
                }
            __syncthreads();
            if (sh.kept <= kOrder) put_in_order(sh.best, sh.kept, p.top, sh.top, sh.warp_key);
            else put_in_order(sh.list, n, p.top, sh.top, sh.warp_key);
        } else {
            // the largest value behind the last one found, `top` times over
            if (tid < p.top) sh.top[tid] = 0;
            Key last = kInFront;
            for (int k = 0; k < want; ++k) {
                Key best = 0;
                auto look = [&](float v, int id) {
                    const Key key = order_key(v, id);
                    if (key < last && key > best) best = key;
                };
                for (int i = v0 + tid; i < v1; i += kThreads) {
                    float v[kVec];
                    unpack(units[i], v);
#pragma unroll
                    for (int e = 0; e < kVec; ++e) look(v[e], lead + i * kVec + e);
                }
                if (tid < odd) look(odd_value, odd_id);
                best = warp_max(best);
                if (lane == 0) sh.warp_key[warp] = best;
                __syncthreads();
                for (int w = 0; w < kWarps; ++w) best = max(best, sh.warp_key[w]);
                if (tid == 0) sh.top[k] = best;
                last = best;
                __syncthreads();
            }
        }
    }
    if (ctas > 1) {
        // the first CTA gets every CTA's sums and alternatives into its shared memory
        __syncthreads();
        cluster_wait();  // it has begun
        if (tid < 3) {
            const uint32_t at = of_cta(&sh.cta_stats[rank], 0) + tid * 4;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(reinterpret_cast<const float *>(&sh.stats)[tid]) : "memory");
        }
        if (tid < p.top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(of_cta(sh.gathered + rank * p.top + tid, 0)), "l"(sh.top[tid]) : "memory");
        cluster_arrive();
        cluster_wait();
        if (rank != 0) return;
        a = join_warp(lane < ctas ? sh.cta_stats[lane] : Stats{-FLT_MAX, 0.0f, 0.0f}, c);  // every warp the same
        if (p.top) {
            // a CTA whose last alternative is the largest has `top` that reach it: the others' behind that are none
            const Key least = warp_max(lane < ctas ? sh.gathered[lane * p.top + p.top - 1] : 0);
            if (tid == 0) sh.kept = 0;
            __syncthreads();
            for (int i = tid; i < ctas * p.top; i += kThreads)
                if (sh.gathered[i] && sh.gathered[i] >= least) sh.best[atomicAdd(&sh.kept, 1)] = sh.gathered[i];
            __syncthreads();
            put_in_order(sh.best, sh.kept, p.top, sh.top, sh.warp_key);
        }
    } else {
        __syncthreads();
        a = sh.stats;
    }
    const Results result(a, p.scale);
    if (tid == 0 && p.entropy) p.entropy[row] = result.entropy(a);
    const float none = __uint_as_float(0x7fc00000u);
    if (one_given) p.logprobs[row * p.given + tid] = token0 >= 0 && token0 < p.vocab ? result.logprob(given0) : none;
    for (int g = tid + kThreads; g < p.given; g += kThreads) {
        const int token = p.tokens[row * p.given + g];
        p.logprobs[row * p.given + g] = token >= 0 && token < p.vocab ? result.logprob(get(x + token)) : none;
    }
    if (tid < p.top) {
        p.top_ids[row * p.top + tid] = key_id(sh.top[tid]);
        p.top_logprobs[row * p.top + tid] = result.logprob(key_value(sh.top[tid]));
    }
}

constexpr int kAlone = 100 << 10, kInPairs = 60 << 10;  // with RowShared more than a half, and a third, of an SM's 228 KB
static_assert(sizeof(RowShared) + kAlone > (114 << 10) && sizeof(RowShared) + kInPairs > (76 << 10) && sizeof(RowShared) + kInPairs < (112 << 10), "shared memory");
int logprobs_init(Ctx *) {
    for (void (*k)(ScoreParams, int) : {logprobs_kernel<float>, logprobs_kernel<uint16_t>}) {
        LBK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        LBK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kAlone));
    }
    return LBK_OK;
}
const InitHook kInitLogprobs(logprobs_init);

}  // namespace
}  // namespace lbk

using namespace lbk;

extern "C" {

int lbk_token_logprobs(lbk_ctx *c, int dtype, const void *logits_dev, size_t pitch, size_t rows, size_t vocab, const int32_t *tokens_dev, size_t given, float scale,
                       size_t top, float *logprobs_dev, float *entropy_dev, int32_t *top_ids_dev, float *top_logprobs_dev, void *stream) {
    LBK_TREE_PRE("lbk_token_logprobs");
    if (rows == 0) return LBK_OK;
    if (!logits_dev || (given && (!tokens_dev || !logprobs_dev)) || (top && (!top_ids_dev || !top_logprobs_dev)))
        return fail(LBK_ERR_INVALID, "lbk_token_logprobs: null buffer");
    if (dtype != LBK_DTYPE_F32 && dtype != LBK_DTYPE_BF16) return fail(LBK_ERR_INVALID, "lbk_token_logprobs: unknown type %d", dtype);
    if (vocab == 0 || pitch < vocab || top > vocab) return fail(LBK_ERR_SHAPE, "lbk_token_logprobs: rows of %zu values, %zu apart, %zu alternatives", vocab, pitch, top);
    // inside these, scale * log2(e) is finite, and what lies 1e30 below the largest value has no weight (Seen::add)
    if (!(scale >= 1e-20f && scale <= 1e20f)) return fail(LBK_ERR_INVALID, "lbk_token_logprobs: the scale is a number from 1e-20 to 1e20");
    if (top > LBK_LOGPROBS_TOP || vocab > (1u << 30) || given > (1u << 20) || rows > (1u << 26))
        return fail(LBK_ERR_UNSUPPORTED, "lbk_token_logprobs: at most %d alternatives, 2^30 values and 2^20 tokens a row, 2^26 rows", LBK_LOGPROBS_TOP);
    const ScoreParams p{logits_dev, pitch, static_cast<int>(vocab), tokens_dev, static_cast<int>(given), scale, static_cast<int>(top), logprobs_dev, entropy_dev, top_ids_dev,
                        top_logprobs_dev};
    const size_t size = dtype == LBK_DTYPE_F32 ? 4 : 2;
    if (vocab * size <= (rows > 3 * static_cast<size_t>(ctx->sm_count) ? kShortBytes : kTinyBytes)) {
        const size_t warps = std::min<size_t>(kShortWarps, (rows + ctx->sm_count - 1) / ctx->sm_count);  // few rows: an SM each
        LBK_CUDA(launch_chained(dtype == LBK_DTYPE_F32 ? logprobs_short_kernel<float> : logprobs_short_kernel<uint16_t>, dim3(static_cast<unsigned>((rows + warps - 1) / warps)),
                                dim3(static_cast<unsigned>(warps * 32)), 0, st, p, static_cast<int>(rows)));
        ctx->launches++;
        return LBK_OK;
    }
    // CTAs a row: as many as the SMs hold beside one another, three each, as long as each has 3.5 trips of loads; of up to 64 CTAs half a trip is
    // enough. us at 128256 f32 with 1 / 2 / 4 / 8 / 16: 1 row 16.6 / 12.2 / 9.4 / 7.5 / 6.5, 16 rows 27 / 19 / 14 / 11 / 12, 64 rows 24 / 19 / 14 / 18 / 24, 150 rows 29 / 21 / 26 / 32 / 48,
    // 300 rows 38 / 44 / 49 / 70 / 116.
    const size_t trip = static_cast<size_t>(kThreads) * kLoads * 16 / size;
    unsigned ctas = 1;
    while (ctas < kClusterMost && rows * ctas * 2 <= 3 * static_cast<size_t>(ctx->sm_count) && (vocab >= 7 * trip * ctas || (rows * ctas <= 64 && vocab >= trip * ctas))) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    // No more CTAs to an SM than it takes: a launch that begins beside the last CTAs of the one in front puts as many as fit on the SMs that are free, and the others
    // stay empty. Shared memory that nobody uses keeps them apart: us of 50021 bf16, one alternative, one call behind the other, 120 rows 12.4 -> 8.9, 203 12.6 -> 10.9. (Clusters
    // are placed by the GPC, and find less room so: 16 rows of 128256 f32 9.0 -> 14.4.)
    const size_t each_sm = (rows + ctx->sm_count - 1) / ctx->sm_count;
    cfg.dynamicSmemBytes = ctas > 1 ? 0 : each_sm == 1 ? kAlone : each_sm == 2 ? kInPairs : 0;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    LBK_CUDA(cudaLaunchKernelEx(&cfg, dtype == LBK_DTYPE_F32 ? logprobs_kernel<float> : logprobs_kernel<uint16_t>, p, static_cast<int>(ctas)));
    ctx->launches++;
    return LBK_OK;
}

}  // extern "C"
