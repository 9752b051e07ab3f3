// kv_cache.cuh -- the paged 8-bit key/value cache as its kernels see it: the
// device views of sam3b200_kv_cache and sam3b200_kv_batch, how a kernel finds
// its sequence, and the host checks shared by the entry points.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/sam3_b200.h"
#include "backend_impl.h"
#include "error_bits.h"

namespace b200 {

// Pages whose largest magnitude is below this store zeros under scale 0, so
// that reciprocals of scales stay finite.
constexpr float kKvSmallest = 7.888609052210118e-31f;  // 2^-100

struct KvView {
    int8_t *codes[2];  // keys, values: [n_pages][heads][1 << page_log2][D]
    float *scale[2];   // [n_pages][heads]
    int n_pages, heads, page_log2, D;
};

struct KvRows {
    const int32_t *table, *row_start, *kv_len;
    int64_t table_width;
    int n_seqs, n_rows, max_rows;
    int64_t max_len;
};

// One sequence of the batch, with its numbers cut to what the buffers hold:
// rows [r0, r0 + n) of the row tensors, len cached tokens.
struct KvSeq {
    int s, r0, n;
    int len;
};

// Checks every sequence against the sizes that the host gave and records
// kErrKvBatch; one block of a launch runs it, the one of the last unit, which
// mostly has nothing else to do.
__device__ __forceinline__ void kv_check(const KvRows &b, int page_log2, bool rows_are_cached, int *err) {
    for (int s = threadIdx.x; s < b.n_seqs; s += blockDim.x) {
        const int64_t r0 = b.row_start[s], r1 = b.row_start[s + 1], len = b.kv_len[s];
        if (r0 < 0 || r1 < r0 || r1 > b.n_rows || r1 - r0 > b.max_rows || len < 0 || len > b.max_len ||
            len > (b.table_width << page_log2) || (rows_are_cached && r1 - r0 > len))
            atomicOr(err, kErrKvBatch);
    }
}

// Work is cut into units of 1 << unit_log2 consecutive items of a sequence
// that has items [row_start[s] m, row_start[s + 1] m).  Sequence s starts at
// unit first(s) = floor(row_start[s] m >> unit_log2) + spare s, which leaves
// it at least floor(n m >> unit_log2) + spare units; the launch has
// first(n_seqs) of them.  The block's threads count the sequences that start
// at or before unit u, each with its numbers already loaded, so that the one
// that is found costs no second trip to memory.  Every thread of the block
// calls this.  False if there is none; `local` is the unit's number within
// the sequence.
__device__ __forceinline__ bool kv_find(const KvRows &b, int64_t u, int m, int unit_log2, int spare, int page_log2, KvSeq &q,
                                        int64_t &local) {
    __shared__ int found[4];
    int before = 0, mine = -1, r0 = 0, r1 = 0, len = 0;
    for (int base = 0; base < b.n_seqs; base += blockDim.x) {
        const int s = base + threadIdx.x;
        int in = 0;
        if (s < b.n_seqs) {
            const int start = b.row_start[s], end = b.row_start[s + 1], n = b.kv_len[s];
            in = ((static_cast<int64_t>(max(start, 0)) * m) >> unit_log2) + static_cast<int64_t>(spare) * s <= u;
            if (in) mine = s, r0 = start, r1 = end, len = n;
        }
        before += __syncthreads_count(in);
    }
    if (before == 0) return false;
    // starts that fall (kErrKvBatch) may leave the last counted number with no thread: nothing is found then
    if (threadIdx.x == 0) found[3] = -1;
    __syncthreads();
    if (mine == before - 1) found[0] = r0, found[1] = r1, found[2] = len, found[3] = mine;
    __syncthreads();
    if (found[3] < 0) return false;
    const int64_t cap = min(b.table_width << page_log2, b.max_len);
    q.s = found[3];
    q.r0 = min(max(found[0], 0), b.n_rows);
    q.n = min(max(found[1], q.r0), b.n_rows) - q.r0;
    q.len = static_cast<int>(min(static_cast<int64_t>(max(found[2], 0)), cap));
    local = u - (((static_cast<int64_t>(max(found[0], 0)) * m) >> unit_log2) + static_cast<int64_t>(spare) * q.s);
    return local >= 0;
}

// The page of tokens [i << page_log2, ...) of sequence s; a bad entry is
// recorded and reads as -1.
__device__ __forceinline__ int kv_page(const KvView &c, const KvRows &b, int s, int64_t i, int *err) {
    const int p = b.table[s * b.table_width + i];
    if (p >= 0 && p < c.n_pages) return p;
    atomicOr(err, kErrKvPage);
    return -1;
}

__device__ __forceinline__ int64_t kv_slab(const KvView &c, int page, int head) {
    return ((static_cast<int64_t>(page) * c.heads + head) << c.page_log2) * c.D;
}

// ---- element types ------------------------------------------------------------

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight consecutive elements; VEC: p is 16-byte aligned.
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    if constexpr (VEC) {
        uint4 raw[sizeof(T) / 2];
        T *e = reinterpret_cast<T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(p)[i] = raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// ---- launches -----------------------------------------------------------------
// The kernels of this family follow one another in a step's few microseconds,
// so a launch lets its blocks be placed as the last blocks of the kernel in
// front of it on the stream leave, without a wait for its memory first
// (programmatic stream serialisation); each kernel begins with that wait, and
// reads and writes nothing before it.  It reads through ordinary loads: the
// read-only ones ask for memory that nobody writes from a kernel's start, which
// here lies before the end of the kernel in front.  A chain of rotary, rotary,
// write, read and attention in small calls: 21.3 us as a graph and 25.6 called
// one by one, against 23.2 and 31.9 with plain launches.  Letting the next
// kernel in when this one starts (launch_dependents) costs the gain again: its
// blocks then sit beside these with another split of shared memory; 23.8 us.
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const Args &...args) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    cudaGetLastError();  // returned here, not left for the next check
    return e;
}

// ---- host ---------------------------------------------------------------------

// Makes `device` current for the scope and restores the caller's device.
struct DeviceScope {
    int prev = -1;
    explicit DeviceScope(int device) {
        if (cudaGetDevice(&prev) != cudaSuccess || prev == device) prev = -1;
        else cudaSetDevice(device);
    }
    ~DeviceScope() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
};

inline int type_bytes(int type) {
    return type == SAM3B200_TYPE_F32 ? 4 : type == SAM3B200_TYPE_F16 || type == SAM3B200_TYPE_BF16 ? 2 : 0;
}

// Rows of [rows][heads][D] elements given by the element strides nb (token,
// head; NULL: packed).  aligned16: every 8-element group starts on 16 bytes.
struct RowTensor {
    int64_t token, head;
    bool aligned16;
};
inline RowTensor row_tensor(const void *p, int type, const int64_t *nb, int64_t heads, int64_t D) {
    RowTensor t{nb ? nb[0] : heads * D, nb ? nb[1] : D, false};
    const int64_t b = type_bytes(type);
    t.aligned16 = reinterpret_cast<uintptr_t>(p) % 16 == 0 && t.token * b % 16 == 0 && t.head * b % 16 == 0;
    return t;
}

// Host check of a row tensor's strides (`written`: no element may lie twice in it).
bool rows_ok(const char *op, const char *what, const RowTensor &t, int64_t rows, int64_t heads, int64_t D, bool written);
// Host checks of a cache and a batch; on failure the message names `op`.
bool kv_views(const char *op, const sam3b200_kv_cache *c, const sam3b200_kv_batch *b, KvView &cv, KvRows &bv);

}  // namespace b200
