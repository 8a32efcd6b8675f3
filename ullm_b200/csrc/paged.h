// Internal interface of the operators over a paged key/value cache (paged.cu, tree_attn.cu, tree_attn_tc.cu).
#pragma once

#include "../../include/ullm_cuda.h"
#include "common.cuh"
#include "kernels.h"

#include <stddef.h>
#include <stdint.h>

namespace ullm {

// Element (layer, page, slot, head, d) of K or V, in elements from the base: 64-bit, pools pass 4 G elements.
struct PoolDev {
    uint8_t *k = nullptr, *v = nullptr; // of layer 0
    long long layer_stride = 0, page_stride = 0, slot_stride = 0, head_stride = 0;
    int n_layer = 0, n_pages = 0, page_size = 0, n_kv_head = 0, head_dim = 0, elem_bytes = 0;
};
struct TableDev {
    int *blocks = nullptr, *len = nullptr, *refs = nullptr, *fault = nullptr;
    int n_seq = 0, max_blocks = 0;
    int *work = nullptr;
};

inline size_t dtype_bytes(int dtype) { return dtype == ULLM_DTYPE_F32 ? 4 : 2; }
// Whether every one of these arrays of 32-bit numbers (null: absent) can be read as such.
template <typename... P> bool ints_aligned(const P *...p) { return (((uintptr_t)p | ...) & 3) == 0; }
// A message when the description cannot be used, else null; fills `out`.
const char *pool_check(const ullm_kv_pages *kv, PoolDev *out);

// One attention call as its kernels see it.
struct TreeDev {
    const uint8_t *q;
    uint8_t *out;
    long long q_stride, out_stride; // elements
    const int *cu, *len, *ids, *blocks;
    const uint32_t *mask;
    const uint8_t *k, *v; // this layer's
    long long page_stride, slot_stride, head_stride;
    int n_rows, n_seq, n_kv, group, dim, n_table, max_blocks, n_pages, page_size, mask_words;
    int page_log; // logarithm of the page size, -1 where that is no power of two (then by division: 2 to 4 % of a call in 32 bits)
    float scale_log2; // scale * log2(e): the kernels work with powers of two
    // work area: per CTA one record and two partial results (rows x (dim + 2) floats each)
    int4 *meta;
    float *part;
    int *count; // for kernels that join units themselves: a counter per CTA
};
constexpr int TREE_META = 2; // int4 per CTA

// f32 queries with heads of 64 or 128 values: the tensor cores on values split in two
bool tree_attn_split_supported(int dim);
cudaError_t launch_tree_attn_split(const DeviceInfo &dev, int kv_dtype, const TreeDev &t, bool pdl, cudaStream_t st);
bool tree_attn_tc_supported(const PoolDev &pool, int dtype);
size_t tree_attn_tc_work(int sm_count, int dim);
cudaError_t launch_tree_attn_tc(const DeviceInfo &dev, const PoolDev &pool, int dtype, const TreeDev &t, int *d_status, long long wait_cycles, bool pdl,
                                cudaStream_t st);

// Puts the caller's current device back when a call ends.
struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            cudaGetLastError();
            prev = -1;
        }
        if (prev != device) cudaSetDevice(device);
        else prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

template <typename... KArgs, typename... Args>
cudaError_t launch_kernel(void (*fn)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

} // namespace ullm
