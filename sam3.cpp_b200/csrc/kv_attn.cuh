// kv_attn.cuh -- attention over the paged caches of 8 and 4 bits: what its
// kernels and entry points share.
#pragma once

#include <cmath>

#include "kv_cache.cuh"

namespace b200 {

template <typename View>
struct KvAttnArgsOf {
    View c;
    KvRows b;
    const void *q;
    void *y;
    RowTensor qs, ys;
    int q_bf16;           // else f16
    int y_type;           // SAM3B200_TYPE_*
    int group;            // query heads of a kv head
    float scale_log2;     // scale * log2(e)
    int causal, window;   // window 0: none
    int splits;           // most parts of a key range (few rows over 4 bits: of all key ranges)
    int chunk;            // least tokens of a part (a multiple of 64, for 256 rows of 128; few rows over 4 bits: steps of
                          // 64 tokens, 0: the kernel's choice)
    int chunk_short, short_range;  // the same for key ranges below short_range
    float *part;          // partial results: see kPartFloats
    unsigned *done;       // parts finished, one counter for each set of parts; 0 between calls
    int *err;
    unsigned *ready;      // host: kernels whose attributes are set on the device
};
using KvAttnArgs = KvAttnArgsOf<KvView>;
using Kv4AttnArgs = KvAttnArgsOf<Kv4View>;

// 2^x scores: P = 2^(t - m + kPUp) with m within kLazy of the running
// maximum, so f16 P reaches 2^(kPUp + kLazy) < 65504 at most, and what falls
// below f16's smallest number is 2^-32 of the largest.  P is rounded to f16
// because the matrix instructions take the codes exactly only as f16: at
// most 2^-11 of a weight, against 2^-8 as bf16; tf32 runs at half the rate.  The sum of the weights takes them unrounded, in f32.
constexpr float kPUp = 7.f, kLazy = 8.f;

// Scale of a value page that holds only zeros, as the softmax weights see it:
// low, so that the other pages' weights keep their bits (scales from 2^-90
// on), and not so low that its own leave the sum beside scales up to 2^20.
constexpr float kZeroScaleLog2 = -80.f;

// The device workspace of a handle: parts of key ranges, each [rows][D + 2] (sums, maximum, weight), of 8 or 16 rows
// (kv_attn_few) or 256 (kv_attn_tc: 1024 parts of head dim 128); one counter a row tile.
constexpr int kMaxParts = 8192;
constexpr int64_t kPartFloats = int64_t(1024) * 256 * (128 + 2);
static_assert(kPartFloats >= int64_t(kMaxParts) * 16 * (128 + 2), "parts of 16 rows");

// Last key that row i of a sequence sees, and the first.
template <typename Args>
__device__ __forceinline__ int kv_last(const Args &a, const KvSeq &q, int i) {
    return a.causal ? q.len - q.n + i : q.len - 1;
}
template <typename Args>
__device__ __forceinline__ int kv_first(const Args &a, int last) {
    return a.window ? max(last - a.window + 1, 0) : 0;
}

// Stores 8 results of one row.
template <typename Args>
__device__ __forceinline__ void kv_store8(const Args &a, int64_t at, const float (&v)[8]) {
    auto put = [&](auto *y) {
        if (a.ys.aligned16) store8<true>(y + at, v);
        else store8<false>(y + at, v);
    };
    if (a.y_type == SAM3B200_TYPE_F32) put(static_cast<float *>(a.y));
    else if (a.y_type == SAM3B200_TYPE_F16) put(static_cast<__half *>(a.y));
    else put(static_cast<__nv_bfloat16 *>(a.y));
}

// A handle: the workspace, and which kernels' attributes are set.
struct KvAttention {
    Backend *be = nullptr;
    unsigned ready = 0;  // kernels whose attributes are set on this handle's device
    float *part = nullptr;
    unsigned *done = nullptr;
};

// Bits of KvAttention::ready: four kernels of few rows and two for many, of each cache.
constexpr unsigned kReadyFew = 0, kReadyFew4 = 8, kReadyTc = 16, kReadyTc4 = 18;

// 8 or 16 rows a block: kv_attn.cu, kv4_attn.cu
cudaError_t kv_attn_few(KvAttnArgs a, int num_sms, cudaStream_t st);
cudaError_t kv_attn_few(Kv4AttnArgs a, int num_sms, cudaStream_t st);
// 256 rows a block: kv_attn_tc.cu
cudaError_t kv_attn_tc(KvAttnArgs a, int num_sms, cudaStream_t st);
cudaError_t kv_attn_tc(Kv4AttnArgs a, int num_sms, cudaStream_t st);

// The checks of a call with either cache, and its arguments; `empty`: there is nothing to do.
template <typename View, typename Cache>
bool kv_attn_args(const char *op, KvAttention *k, const Cache *cache, const sam3b200_kv_batch *batch, int type, const void *q,
                  const int64_t *q_nb, int64_t n_heads, float scale, int causal, int64_t window, int y_type, void *y,
                  const int64_t *y_nb, KvAttnArgsOf<View> &a, bool &empty) {
    if (!kv_views(op, cache, batch, a.c, a.b)) return false;
    if (!q || !y) {
        set_error("%s: null argument", op);
        return false;
    }
    const int yb = type_bytes(y_type);
    if ((type != SAM3B200_TYPE_F16 && type != SAM3B200_TYPE_BF16) || (y_type != type && y_type != SAM3B200_TYPE_F32) ||
        reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(y) % yb) {
        set_error("%s: unsupported types %d -> %d (q F16=1 or BF16=30, y q's type or F32=0) or unaligned data", op, type, y_type);
        return false;
    }
    if (n_heads >= 1 && a.b.n_rows * (n_heads / a.c.heads) > 0x7fffff00) {
        set_error("%s: %d rows of %lld query heads over %d kv heads are too many", op, a.b.n_rows, (long long)n_heads, a.c.heads);
        return false;
    }
    if (n_heads < 1 || n_heads > 65535 || n_heads % a.c.heads != 0) {
        set_error("%s: %lld query heads over %d kv heads (a positive multiple is needed)", op, (long long)n_heads, a.c.heads);
        return false;
    }
    if (!(scale >= 0.f) || !std::isfinite(scale * 1.4426950408889634f) || window < 0 || (window && !causal)) {
        set_error("%s: bad scale %g or window %lld (a window needs the causal mask)", op, scale, (long long)window);
        return false;
    }
    a.q = q, a.y = y;
    a.qs = row_tensor(q, type, q_nb, n_heads, a.c.D);
    a.ys = row_tensor(y, y_type, y_nb, n_heads, a.c.D);
    if (!rows_ok(op, "q", a.qs, a.b.n_rows, n_heads, a.c.D, false) || !rows_ok(op, "y", a.ys, a.b.n_rows, n_heads, a.c.D, true))
        return false;
    if (!k) {
        set_error("%s: null handle", op);
        return false;
    }
    empty = a.b.n_seqs == 0 || a.b.n_rows == 0;
    a.q_bf16 = type == SAM3B200_TYPE_BF16;
    a.y_type = y_type;
    a.group = static_cast<int>(n_heads / a.c.heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    // a window that no length reaches is none; below 2^30 it cannot pass 32 bits where rows are more than tokens
    a.causal = causal != 0, a.window = window < a.b.max_len ? static_cast<int>(window) : 0;
    a.part = k->part, a.done = k->done, a.ready = &k->ready, a.err = k->be->err;
    return true;
}

}  // namespace b200
