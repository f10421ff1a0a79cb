// Drafted tokens as trees: what the kernels over them share (lbk_tree.cu, lbk_attn_tree.cu).
//
// A sequence has `t` node places, the first `count` of them in use. parents[i] is the node that node i follows, always one in
// front of it (parents[i] < i), or -1: node i follows the sequence's last committed position. Node i's row of the cache is
// pos + i whatever its depth; what it follows, and sees, are the rows 0 .. pos - 1 and its ancestors'.
#pragma once

#include "lbk_internal.cuh"
#include "lbk_ptx.cuh"

namespace lbk {

constexpr int kTreeNodes = 128;  // node places of a sequence: two 64-bit words hold who sees whom
constexpr int kErrPos = 7, kErrTree = 8;  // device_error_status

// The context's device is current while this lives; the caller's comes back.
struct OnDevice {
    int before = -1;
    cudaError_t status;
    explicit OnDevice(int device) {
        int now = -1;
        status = cudaGetDevice(&now);
        if (status == cudaSuccess && now != device) {
            status = cudaSetDevice(device);
            if (status == cudaSuccess) before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

#define LBK_TREE_PRE(name)                                         \
    if (!c) return fail(LBK_ERR_INVALID, name ": context is null"); \
    Ctx *ctx = reinterpret_cast<Ctx *>(c);                          \
    const OnDevice on_device(ctx->device);                          \
    LBK_CUDA(on_device.status);                                     \
    cudaStream_t st = static_cast<cudaStream_t>(stream)

// count of a sequence, kept inside its node places
__device__ __forceinline__ int tree_count(const int *counts, int seq, int t) { return counts ? min(max(counts[seq], 0), t) : t; }

// Whether a sequence's rows lie in its cache; if not, that is recorded.
__device__ __forceinline__ bool tree_in_cache(int pos, int count, int cap, int *err_word) {
    if (pos >= 0 && pos <= cap - count) return true;
    if (threadIdx.x == 0) atomicExch(err_word, kErrPos);
    return false;
}

}  // namespace lbk
