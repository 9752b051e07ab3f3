// kv_attn.cuh -- attention over the paged 8-bit cache: what its kernels share.
#pragma once

#include "kv_cache.cuh"

namespace b200 {

struct KvAttnArgs {
    KvView c;
    KvRows b;
    const void *q;
    void *y;
    RowTensor qs, ys;
    int q_bf16;           // else f16
    int y_type;           // SAM3B200_TYPE_*
    int group;            // query heads of a kv head
    float scale_log2;     // scale * log2(e)
    int causal, window;   // window 0: none
    int splits;           // most parts of a key range
    int chunk;            // least tokens of a part (a multiple of 64, for 256 rows of 128)
    int chunk_short, short_range;  // the same for key ranges below short_range
    float *part;          // partial results: see kPartFloats
    unsigned *done;       // parts finished, one counter a unit and kv head; 0 between calls
    int *err;
    unsigned *ready;      // host: kernels whose attributes are set on the device
};

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
__device__ __forceinline__ int kv_last(const KvAttnArgs &a, const KvSeq &q, int i) {
    return a.causal ? q.len - q.n + i : q.len - 1;
}
__device__ __forceinline__ int kv_first(const KvAttnArgs &a, int last) {
    return a.window ? max(last - a.window + 1, 0) : 0;
}

// Stores 8 results of one row.
__device__ __forceinline__ void kv_store8(const KvAttnArgs &a, int64_t at, const float (&v)[8]) {
    auto put = [&](auto *y) {
        if (a.ys.aligned16) store8<true>(y + at, v);
        else store8<false>(y + at, v);
    };
    if (a.y_type == SAM3B200_TYPE_F32) put(static_cast<float *>(a.y));
    else if (a.y_type == SAM3B200_TYPE_F16) put(static_cast<__half *>(a.y));
    else put(static_cast<__nv_bfloat16 *>(a.y));
}

cudaError_t kv_attn_few(KvAttnArgs a, int num_sms, cudaStream_t st);  // kv_attn.cu: 8 or 16 rows a block
cudaError_t kv_attn_tc(KvAttnArgs a, int num_sms, cudaStream_t st);   // kv_attn_tc.cu: 256 rows a block

}  // namespace b200
