// kv4_cache.cu -- writing rows of keys and values into the paged 4-bit cache
// and reading them back.
//
// 32 consecutive dimensions of one token's head share a scale d:
//   top = the finite element of largest magnitude (the positive one of two)
//   d = bf16(top / -8),  code = min(round(x / d), 7) + 8,  value = d (code - 8)
// The quotient is exact, ties go to even, so codes depend on nothing but the
// group's 32 numbers.  d has 8 significant bits and code - 8 at most 3 (or is
// -8), so every value has 11 bits: f16 holds it exactly.
//
// A block takes up to 16 rows of a sequence for some of its slabs (a slab: one
// head's keys, or its values), 8 values a thread and step, four threads a
// group, the tokens of a slab side by side so that their codes leave as one
// run.  Bound by memory: 2 (f16) bytes in and 0.56 out per value, and the other
// way round on reading.
#include <algorithm>

#include "kv_cache.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 256, kRowsLog2 = 4, kRows = 1 << kRowsLog2;

template <typename Ptr>
struct RowsArgs {
    Kv4View c;
    KvRows b;
    Ptr x[2];  // rows of keys and values
    RowTensor xs[2];
    int slabs;  // of a block
    int *err;
};

// Where a block's work lies: items of 8 dimensions, chunk fastest, then row, then slab.
struct Work {
    KvSeq q;
    int first, rows;   // first row within the sequence, rows of this block
    int slab0, slabs;
};

template <typename Args>
__device__ __forceinline__ bool find_work(const Args &a, Work &w) {
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, true, a.err);
    int64_t local;
    if (!kv_find(a.b, blockIdx.x, 1, kRowsLog2, 1, a.c.page_log2, w.q, local)) return false;
    if ((local << kRowsLog2) >= w.q.n || w.q.len < w.q.n) return false;
    w.first = static_cast<int>(local) << kRowsLog2;
    w.rows = min(w.q.n - w.first, kRows);
    w.slab0 = blockIdx.y * a.slabs;
    w.slabs = min(a.slabs, 2 * a.c.heads - w.slab0);
    return true;
}

// The token of row i of the sequence in the cache, counted in tokens of its slab 0; -1 for a bad page.
template <typename Args>
__device__ __forceinline__ int64_t token_at(const Args &a, const Work &w, int i, int head) {
    const int pos = w.q.len - w.q.n + i;
    const int page = kv_page(a.c, a.b, w.q.s, pos >> a.c.page_log2, a.err);
    if (page < 0) return -1;
    return ((static_cast<int64_t>(page) * a.c.heads + head) << a.c.page_log2) + (pos & ((1 << a.c.page_log2) - 1));
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ RowsArgs<const void *> a) {
    wait_for_stream();
    Work w;
    if (!find_work(a, w)) return;
    const int chunk_log2 = a.c.D == 64 ? 3 : 4;
    const int items = (w.slabs * w.rows) << chunk_log2;
    for (int id0 = 0; id0 < items; id0 += kThreads) {  // all lanes: a group's four are neighbours
        const int id = id0 + threadIdx.x, chunk = id & ((1 << chunk_log2) - 1), unit = id >> chunk_log2;
        const bool live = id < items;
        const int slab = w.slab0 + unit / w.rows, row = w.first + unit % w.rows;
        const int which = slab >= a.c.heads, head = slab - which * a.c.heads;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (live) {
            const Raw8<T> raw = raw8<VEC>(static_cast<const T *>(a.x[which]) + (w.q.r0 + static_cast<int64_t>(row)) * a.xs[which].token +
                                          head * a.xs[which].head + chunk * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(raw.v[j]);
        }
        float high = 0.f, low = 0.f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool f = fabsf(v[j]) <= kF32Max;
            finite = finite && f;
            high = fmaxf(high, f ? v[j] : 0.f), low = fminf(low, f ? v[j] : 0.f);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        }
        const float top = high >= -low ? high : low;
        const __nv_bfloat16 held = __float2bfloat16_rn(fabsf(top) < kKvSmallest ? 0.f : -0.125f * top);
        const float d = to_f32(held), s = fabsf(d);
        if (!live) continue;
        const int64_t at = token_at(a, w, row, head);
        if (at < 0) continue;
        uint32_t packed = 0x88888888u;
        if (s > 0.f) {
            const float end = fminf(8.f * s, kF32Max);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (!finite) v[j] = v[j] == v[j] ? fminf(fmaxf(v[j], -end), end) : 0.f;
                if (d < 0.f) v[j] = -v[j];
            }
            int c[8];
            round_quotients(v, s, __frcp_rn(s), c);
            packed = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) packed |= static_cast<uint32_t>(min(c[j] - 0x4b400000, 7) + 8) << (4 * j);
        }
        reinterpret_cast<uint32_t *>(a.c.codes[which])[(at << chunk_log2) + chunk] = packed;
        if ((chunk & 3) == 0) a.c.scale[which][(at << (chunk_log2 - 2)) + (chunk >> 2)] = held;
    }
}

// 8 codes as numbers: 0x4b00000u is 2^23 + u.
__device__ __forceinline__ void widen8(uint32_t w, float d, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        v[j] = __fmul_rn(__fsub_rn(__uint_as_float(((w >> (4 * j)) & 15u) | 0x4b000000u), 8388616.f), d);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ RowsArgs<void *> a) {
    wait_for_stream();
    Work w;
    if (!find_work(a, w)) return;
    const int chunk_log2 = a.c.D == 64 ? 3 : 4;
    const int items = (w.slabs * w.rows) << chunk_log2;
    for (int id = threadIdx.x; id < items; id += kThreads) {
        const int chunk = id & ((1 << chunk_log2) - 1), unit = id >> chunk_log2;
        const int slab = w.slab0 + unit / w.rows, row = w.first + unit % w.rows;
        const int which = slab >= a.c.heads, head = slab - which * a.c.heads;
        const int64_t at = token_at(a, w, row, head);
        uint32_t packed = 0x88888888u;  // a bad page reads as zeros
        float d = 0.f;
        if (at >= 0) {
            packed = reinterpret_cast<const uint32_t *>(a.c.codes[which])[(at << chunk_log2) + chunk];
            d = to_f32(a.c.scale[which][(at << (chunk_log2 - 2)) + (chunk >> 2)]);
        }
        float v[8];
        widen8(packed, d, v);
        store8<VEC>(static_cast<T *>(a.x[which]) + (w.q.r0 + static_cast<int64_t>(row)) * a.xs[which].token + head * a.xs[which].head +
                        chunk * 8,
                    v);
    }
}

// Checks and the launch, which the two directions share.
template <typename Ptr>
int run(const char *op, sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch, int type, Ptr k,
        const int64_t *k_nb, Ptr v, const int64_t *v_nb, bool written, void (*const (&kernels)[3][2])(RowsArgs<Ptr>)) {
    auto *be = reinterpret_cast<Backend *>(h);
    RowsArgs<Ptr> a;
    if (!kv_views(op, cache, batch, a.c, a.b)) return SAM3B200_STATUS_FAILED;
    const int bytes = type_bytes(type);
    if (!k || !v || !bytes || reinterpret_cast<uintptr_t>(k) % bytes || reinterpret_cast<uintptr_t>(v) % bytes) {
        if (!k || !v) set_error("%s: null argument", op);
        else set_error("%s: unsupported type %d (F32=0, F16=1, BF16=30) or unaligned rows", op, type);
        return SAM3B200_STATUS_FAILED;
    }
    a.x[0] = k, a.x[1] = v;
    a.xs[0] = row_tensor(k, type, k_nb, a.c.heads, a.c.D);
    a.xs[1] = row_tensor(v, type, v_nb, a.c.heads, a.c.D);
    if (!rows_ok(op, "k", a.xs[0], a.b.n_rows, a.c.heads, a.c.D, written) || !rows_ok(op, "v", a.xs[1], a.b.n_rows, a.c.heads, a.c.D, written))
        return SAM3B200_STATUS_FAILED;
    if (!be) {
        set_error("%s: null backend", op);
        return SAM3B200_STATUS_FAILED;
    }
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return SAM3B200_STATUS_SUCCESS;
    a.err = be->err;
    DeviceScope dev(be->device);
    // four steps a block where sequences have 16 rows
    const int per_slab = std::min(std::max(a.b.max_rows, 1), kRows) * a.c.D / 8;
    a.slabs = std::min(std::max(4 * kThreads / per_slab, 1), 2 * a.c.heads);
    const dim3 grid((a.b.n_rows >> kRowsLog2) + a.b.n_seqs, (2 * a.c.heads + a.slabs - 1) / a.slabs);
    const int t = type == SAM3B200_TYPE_F32 ? 0 : type == SAM3B200_TYPE_F16 ? 1 : 2;
    const cudaError_t e = launch_after(kernels[t][a.xs[0].aligned16 && a.xs[1].aligned16], grid, kThreads, 0, be->stream, a);
    be->count();
    return cuda_ok(e, op) ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int sam3b200_kv4_write(sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch,
                                  int type, const void *k, const int64_t *k_nb, const void *v, const int64_t *v_nb) {
    return run<const void *>("kv4_write", h, cache, batch, type, k, k_nb, v, v_nb, false,
                             {{kv4_write_kernel<float, false>, kv4_write_kernel<float, true>},
                              {kv4_write_kernel<__half, false>, kv4_write_kernel<__half, true>},
                              {kv4_write_kernel<__nv_bfloat16, false>, kv4_write_kernel<__nv_bfloat16, true>}});
}

extern "C" int sam3b200_kv4_read(sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch,
                                 int type, void *k, const int64_t *k_nb, void *v, const int64_t *v_nb) {
    return run<void *>("kv4_read", h, cache, batch, type, k, k_nb, v, v_nb, true,
                       {{kv4_read_kernel<float, false>, kv4_read_kernel<float, true>},
                        {kv4_read_kernel<__half, false>, kv4_read_kernel<__half, true>},
                        {kv4_read_kernel<__nv_bfloat16, false>, kv4_read_kernel<__nv_bfloat16, true>}});
}
