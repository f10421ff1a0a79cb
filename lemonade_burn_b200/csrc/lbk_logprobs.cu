// Log probabilities of given tokens, entropy and the best alternatives of rows of logits.
//
//   c = scale * x;  lse = log sum_j exp(c_j);  logprob(token) = c_token - lse;  H = lse - sum_j p_j c_j
//   alternatives: the `top` largest logits, the lower id first among equal ones, with their log probabilities
//
// The reference has the greedy token only (crates/lb-model/src/sample.rs:17-25).
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

// A place in the order of the alternatives: larger values first, then lower ids; every NaN in front of every number, as a sort has it; 0 is
// behind every place.
__device__ __forceinline__ unsigned order_value(float x) {  // the order of numbers as that of whole ones
    const unsigned bits = __float_as_uint(x + 0.0f);         // -0 and 0 are equal
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ unsigned long long order_key(float x, int id) {
    return static_cast<unsigned long long>(x != x ? 0xffffffffu : order_value(x)) << 32 | static_cast<unsigned>(~id);
}
__device__ __forceinline__ int key_id(unsigned long long key) { return static_cast<int>(~static_cast<unsigned>(key)); }

// One pass over the row. A thread keeps the maximum m of what it has seen, s = sum e^(c (x - m)) and t = sum e^(c (x - m)) (x - m); entropy = log s - c t / s.
//
// The alternatives come out of the same pass. A warp's `each`-th largest lane maximum is a bound that `each` of its values reach; the least of the bounds of
// all warps is reached by `top` values (each = top / warps, rounded up), so what lies below it is none of them. Values that reach it go to a list in shared memory, some hundred of
// 128256; bounds rise as the row goes by and are read without a barrier (an old one is a bound too). At the end the list is put in order. Rows whose list runs
// over (most values equal, or ascending), or has too few (most of them -inf), and rows with a NaN or +inf are read again, once an alternative.
//
// Bytes bound it: 2000 rows of 128256 f32 are 1.03 GB. A row is cut among the CTAs of a cluster where there are fewer rows than the SMs hold CTAs; they
// meet through distributed shared memory.
constexpr int kThreads = 512, kWarps = kThreads / 32, kLoads = 4;  // 16-byte loads of a thread in flight
constexpr int kList = 4096;
constexpr int kTop = LBK_LOGPROBS_TOP, kClusterMost = 16;
static_assert(kTop <= 2 * kWarps && kClusterMost * kTop <= kThreads, "two maxima a warp, a key a thread");
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
__device__ __forceinline__ void join(Stats &a, Stats b, float c) {
    const float m = fmaxf(a.m, b.m);
    raise(a, m, c);
    raise(b, m, c);
    a.s += b.s;
    a.t += b.t;
}
__device__ __forceinline__ Stats join_warp(Stats a, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) join(a, Stats{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o), __shfl_xor_sync(0xffffffffu, a.t, o)}, c);
    return a;
}

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

struct RowShared {
    Key list[kList];
    Key best[kThreads];        // the keys that are put in order: some of the list, or all CTAs' alternatives
    Key top[kTop];             // this CTA's alternatives, in order
    Key warp_key[kWarps];
    Stats warp_stats[kWarps], stats;
    float bound[kWarps];
    int count, kept;
};

// The `top` largest of n keys of the shared memory, in order, into `out`, zeros behind them. n > kThreads: a search for each.
__device__ void put_in_order(const Key *keys, int n, int top, Key *out, Key *warp_key) {
    const int tid = threadIdx.x;
    if (tid < top) out[tid] = 0;
    __syncthreads();
    if (n <= kThreads) {
        if (tid < n) {
            const Key mine = keys[tid];
            int rank = 0;
            for (int i = 0; i < n; ++i) rank += keys[i] > mine;
            if (rank < top && mine) out[rank] = mine;
        }
        __syncthreads();
        return;
    }
    Key last = ~0ull;
    for (int k = 0; k < top && last; ++k) {
        Key best = 0;
        for (int i = tid; i < n; i += kThreads)
            if (keys[i] < last && keys[i] > best) best = keys[i];
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
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
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t of_cta(const void *p, uint32_t rank) {  // the same place in another CTA of the cluster
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(ptx::smem_u32(p)), "r"(rank));
    return a;
}

// ctas: how many share a row, neighbours in the grid and a cluster
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const ScoreParams p, int ctas) {
    constexpr int kVec = 16 / sizeof(T);
    __shared__ RowShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = ctas > 1 ? cluster_rank() : 0;
    const size_t row = blockIdx.x / ctas;
    const T *x = static_cast<const T *>(p.logits) + row * p.pitch;
    const float c = p.scale * 1.4426950408889634f;
    // the row: `lead` values up to the first 16-byte boundary, vectors, the rest; this CTA's vectors v0 .. v1 - 1. The odd values are the first CTA's.
    const int lead = min(p.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    const int vectors = (p.vocab - lead) / kVec, odd = rank == 0 ? p.vocab - vectors * kVec : 0;
    const int v0 = static_cast<int>(static_cast<long long>(vectors) * rank / ctas), v1 = static_cast<int>(static_cast<long long>(vectors) * (rank + 1) / ctas);
    const uint4 *units = reinterpret_cast<const uint4 *>(x + lead);
    const int each = (p.top + kWarps - 1) / kWarps;
    if (tid == 0) sh.count = sh.kept = 0;
    ptx::pdl_trigger();
    ptx::pdl_wait();

    Stats a{-FLT_MAX, 0.0f, 0.0f};
    float floor = -FLT_MAX;  // what a value has to reach to go on the list; -inf never does
    auto write_bound = [&]() {
        unsigned mine = order_value(a.m);
        unsigned best = __reduce_max_sync(0xffffffffu, mine);
        if (each > 1) {  // the second largest: without one lane that has the largest
            if (lane == __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1) mine = 0;
            best = __reduce_max_sync(0xffffffffu, mine);
        }
        if (lane == 0) sh.bound[warp] = value_of(best);
    };
    auto read_bound = [&]() { floor = fmaxf(floor, value_of(__reduce_min_sync(0xffffffffu, order_value(static_cast<const volatile float *>(sh.bound)[lane % kWarps])))); };
    auto list = [&](float v, int id) {
        if (v >= floor) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.list[at] = order_key(v, id);
        }
    };
    auto see = [&](float v) {
        const float d = v - a.m, e = ex2(d * c);
        a.s += e;
        a.t += e * fmaxf(d, -1e30f);  // 0 * -inf is nothing here
    };
    const float odd_value = tid < odd ? get(x + (tid < lead ? tid : tid + vectors * kVec)) : -INFINITY;
    const int odd_id = tid < lead ? tid : tid + vectors * kVec;
    int trip = 0;
    for (int base = v0; base < v1 || trip == 0; base += kThreads * kLoads, ++trip) {
        uint4 raw[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            const int i = base + u * kThreads + tid;
            raw[u] = i < v1 ? __ldcs(units + i) : Empty<T>::vector();
        }
        float high = trip == 0 ? odd_value : -INFINITY;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < kVec; ++e) high = fmaxf(high, v[e]);
        }
        if (high > a.m) raise(a, high, c);
        if (trip == 0) see(odd_value);
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            float v[kVec];
            unpack(raw[u], v);
#pragma unroll
            for (int e = 0; e < kVec; ++e) see(v[e]);
        }
        if (p.top) {
            if ((trip & (trip - 1)) == 0) {  // after 1, 2, 4, .. trips' maxima
                write_bound();
                if (trip == 0) __syncthreads();
            }
            read_bound();
            if (high >= floor) {
                if (trip == 0) list(odd_value, odd_id);
#pragma unroll
                for (int u = 0; u < kLoads; ++u) {
                    float v[kVec];
                    unpack(raw[u], v);
#pragma unroll
                    for (int e = 0; e < kVec; ++e) list(v[e], lead + (base + u * kThreads + tid) * kVec + e);
                }
            }
        }
    }
    if (p.top) write_bound();
    a = join_warp(a, c);
    if (lane == 0) sh.warp_stats[warp] = a;
    __syncthreads();
    if (warp == 0) {
        a = join_warp(lane < kWarps ? sh.warp_stats[lane] : Stats{-FLT_MAX, 0.0f, 0.0f}, c);
        if (lane == 0) sh.stats = a;
    }
    if (p.top) {
        read_bound();
        const int n = sh.count, here = (v1 - v0) * kVec + odd, want = min(p.top, here);
        __syncthreads();  // sh.stats
        const float s = sh.stats.s;
        if (n <= kList && n >= want && s == s && s <= FLT_MAX) {
            // what reaches the last bounds
            const Key least = order_key(floor, 0x7fffffff);
            for (int i = tid; i < n; i += kThreads)
                if (sh.list[i] >= least) {
                    const int at = atomicAdd(&sh.kept, 1);
                    if (at < kThreads) sh.best[at] = sh.list[i];
                }
            __syncthreads();
            if (sh.kept <= kThreads) put_in_order(sh.best, sh.kept, p.top, sh.top, sh.warp_key);
            else put_in_order(sh.list, n, p.top, sh.top, sh.warp_key);
        } else {
            // the largest value behind the last one found, `top` times over
            if (tid < p.top) sh.top[tid] = 0;
            Key last = ~0ull;
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
                for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
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
        cluster_meet();  // every CTA's sums and alternatives are in its shared memory
        if (rank == 0) {
            if (warp == 0) {
                Stats b{-FLT_MAX, 0.0f, 0.0f};
                if (lane < ctas) {
                    const uint32_t at = of_cta(&sh.stats, lane);
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.m) : "r"(at));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(at + 4));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.t) : "r"(at + 8));
                }
                b = join_warp(b, c);
                if (lane == 0) sh.warp_stats[0] = b;
            }
            if (p.top && tid < ctas * p.top)
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(sh.best[tid]) : "r"(of_cta(sh.top + tid % p.top, tid / p.top)));
        }
        cluster_meet();  // nobody leaves while its shared memory is read
        if (rank != 0) return;
        if (p.top) {
            // a CTA whose last alternative is the largest has `top` that reach it: the others' behind that are none
            Key least = tid < ctas ? sh.best[tid * p.top + p.top - 1] : 0;
            for (int o = 16; o > 0; o >>= 1) least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
            if (tid == 0) {
                sh.warp_key[0] = least;
                sh.kept = 0;
            }
            __syncthreads();
            least = sh.warp_key[0];
            if (tid < ctas * p.top && sh.best[tid] && sh.best[tid] >= least) sh.list[atomicAdd(&sh.kept, 1)] = sh.best[tid];
            __syncthreads();
            put_in_order(sh.list, sh.kept, p.top, sh.top, sh.warp_key);
        }
        __syncthreads();
        a = sh.warp_stats[0];
    } else {
        __syncthreads();
        a = sh.stats;
    }
    const float log_s = logf(a.s);
    auto logprob = [&](float v) { return (v - a.m) * p.scale - log_s; };
    if (tid == 0 && p.entropy) p.entropy[row] = log_s - a.t / a.s * p.scale;
    for (int g = tid; g < p.given; g += kThreads) {
        const int token = p.tokens[row * p.given + g];
        p.logprobs[row * p.given + g] = token >= 0 && token < p.vocab ? logprob(get(x + token)) : __uint_as_float(0x7fc00000u);
    }
    if (tid < p.top) {
        const int id = key_id(sh.top[tid]);
        p.top_ids[row * p.top + tid] = id;
        p.top_logprobs[row * p.top + tid] = logprob(get(x + id));
    }
}

int logprobs_init(Ctx *) {
    for (void (*k)(ScoreParams, int) : {logprobs_kernel<float>, logprobs_kernel<uint16_t>}) LBK_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
    if (!(scale > 0.0f) || scale > FLT_MAX) return fail(LBK_ERR_INVALID, "lbk_token_logprobs: the scale is a positive number");
    if (top > LBK_LOGPROBS_TOP || vocab > (1u << 30) || given > (1u << 20) || rows > (1u << 26))
        return fail(LBK_ERR_UNSUPPORTED, "lbk_token_logprobs: at most %d alternatives, 2^30 values and 2^20 tokens a row, 2^26 rows", LBK_LOGPROBS_TOP);
    const ScoreParams p{logits_dev, pitch, static_cast<int>(vocab), tokens_dev, static_cast<int>(given), scale, static_cast<int>(top), logprobs_dev, entropy_dev, top_ids_dev,
                        top_logprobs_dev};
    // As many CTAs to a row as the SMs hold beside one another, two each, and half a trip of loads at least for each
    const size_t per_trip = static_cast<size_t>(kThreads) * kLoads * 16 / (dtype == LBK_DTYPE_F32 ? 4 : 2);
    unsigned ctas = 1;
    while (ctas < kClusterMost && rows * ctas * 2 <= 2 * static_cast<size_t>(ctx->sm_count) && vocab >= per_trip * ctas) ctas *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
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
