// kv_attn_few.cuh -- what the kernels for few query rows a kv head share over
// the caches of 8 and 4 bits: which rows and keys a block has, how its warps'
// partial results and the parts of a key range are joined, and the launch.
#pragma once

#include <algorithm>

#include "kv_attn.cuh"
#include "mma_sync.cuh"

namespace b200 {

constexpr int kWarps = 4;
constexpr int kMaxSplits = 256;  // most parts of a key range

// A block's rows and keys.
struct FewTile {
    KvSeq q;
    unsigned unit;
    int split, n_split;
    int R, row0, i_lo, i_hi;  // rows of the sequence, this tile's first, its first and last token
    int t_begin, t_end;       // this block's part of the tile's keys
};

// Every thread of the block calls this; false if there is nothing to do.
template <int NT, typename Args>
__device__ __forceinline__ bool few_tile(const Args &a, FewTile &t) {
    constexpr int kRows = 8 * NT;
    const int G = a.group;
    t.unit = blockIdx.x / a.splits;
    t.split = blockIdx.x % a.splits;
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, false, a.err);
    int64_t local;
    if (!kv_find(a.b, t.unit, G, NT == 1 ? 3 : 4, 1, a.c.page_log2, t.q, local)) return false;
    t.R = t.q.n * G;  // the host keeps n_rows * G below 2^31
    if (local * kRows >= t.R) return false;
    t.row0 = static_cast<int>(local) * kRows, t.i_lo = t.row0 / G, t.i_hi = (min(t.row0 + kRows, t.R) - 1) / G;

    // the tile's keys, and this block's part of them
    const int k_end = kv_last(a, t.q, t.i_hi) + 1, k_begin = kv_first(a, kv_last(a, t.q, t.i_lo)) & ~15;
    const int range = max(k_end - k_begin, 0);
    const int chunk = max(range < a.short_range ? a.chunk_short : a.chunk, ((range + a.splits - 1) / a.splits + 63) & ~63);
    t.n_split = max((range + chunk - 1) / chunk, 1);
    if (t.split >= t.n_split) return false;
    t.t_begin = k_begin + t.split * chunk, t.t_end = min(t.t_begin + chunk, k_end);
    return true;
}

// The end of a block: its warps' rows (sums in `smem` as [warp][row][F::kRowFloats], dimension d at F::column(d);
// maxima and sums of weights in s_m and s_l) are joined, the parts of the key range by the last block to finish, and
// the rows stored.  Behind a __syncthreads().
template <typename F, int D, typename Args>
__device__ __forceinline__ void few_finish(const Args &a, const FewTile &t, uint8_t *smem, const float (&s_m)[kWarps][F::kRows],
                                           const float (&s_l)[kWarps][F::kRows]) {
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = blockIdx.y, G = a.group;
    const int row0 = t.row0, R = t.R, split = t.split, n_split = t.n_split;
    const unsigned unit = t.unit;
    const KvSeq &q = t.q;
    float *rows = reinterpret_cast<float *>(smem);
    constexpr int kEach = F::kEach, kPer = D / kEach;  // threads a row
    const int row = threadIdx.x / kPer, d0 = threadIdx.x % kPer * kEach;
    const int r = row0 + row;
    const bool live = row < F::kRows && r < R;
    float M = -INFINITY, L = 0.f, sum[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum[i] = 0.f;
    if (live) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][row]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = s_m[w][row] == M ? 1.f : ex2_approx(s_m[w][row] - M);
            L = fmaf(s_l[w][row], f, L);
            const float *from = rows + (w * F::kRows + row) * F::kRowFloats;
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum[i] = fmaf(from[F::column(d0 + i)], f, sum[i]);
        }
    }
    if (n_split > 1) {
        const int64_t group = static_cast<int64_t>(unit) * a.c.heads + kv;
        float *base = a.part + group * a.splits * F::kRows * (D + 2);
        float *ml = base + static_cast<int64_t>(a.splits) * F::kRows * D;
        if (live) {
            float *to = base + (static_cast<int64_t>(split) * F::kRows + row) * D + d0;
#pragma unroll
            for (int i = 0; i < kEach; i += 4)
                *reinterpret_cast<float4 *>(to + i) = make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]);
            if (d0 == 0) *reinterpret_cast<float2 *>(ml + (split * F::kRows + row) * 2) = make_float2(M, L);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            s_last = atomicInc(a.done + group, n_split - 1) == static_cast<unsigned>(n_split - 1);
            __threadfence();
        }
        __syncthreads();
        if (!s_last) return;
        // Join the parts, in a fixed order: a warp takes a row, or with fewer than 4 rows a share of one's parts, its
        // lanes along the dimensions; then the shares are joined.
        const int n_rows = min(R - row0, F::kRows);
        const int shares = n_rows >= 4 ? 1 : n_rows == 1 ? 4 : 2;
        float *share = reinterpret_cast<float *>(smem), *share_ml = share + kWarps * F::kRows * D;
        constexpr int kLanes = D / 4, kStep = 32 / kLanes;  // lanes a row, parts a warp and step
        constexpr int kFlight = 8;                          // loads of a lane on their way at once
        for (int id = warp; id < n_rows * shares; id += kWarps) {
            const int i = id / shares;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY, total = 0.f;
            const float *from = base + static_cast<int64_t>(i) * D + lane % kLanes * 4;
            auto add = [&](float m1, float l1, const float4 &x) {
                const float to = fmaxf(top, m1);
                const float f = top == to ? 1.f : ex2_approx(top - to), f1 = m1 == to ? 1.f : ex2_approx(m1 - to);
                top = to;
                total = total * f + l1 * f1;
                v.x = v.x * f + x.x * f1, v.y = v.y * f + x.y * f1, v.z = v.z * f + x.z * f1, v.w = v.w * f + x.w * f1;
            };
            for (int k0 = (id % shares) * kStep + lane / kLanes; k0 < n_split; k0 += kFlight * shares * kStep) {
                float2 y[kFlight];
                float4 x[kFlight];
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    const int k = k0 + u * shares * kStep;
                    y[u] = make_float2(-INFINITY, 0.f);
                    if (k >= n_split) continue;
                    y[u] = __ldcg(reinterpret_cast<const float2 *>(ml + (k * F::kRows + i) * 2));
                    x[u] = __ldcg(reinterpret_cast<const float4 *>(from + static_cast<int64_t>(k) * F::kRows * D));
                }
#pragma unroll
                for (int u = 0; u < kFlight; ++u)
                    if (k0 + u * shares * kStep < n_split) add(y[u].x, y[u].y, x[u]);
            }
            if constexpr (kStep == 2) {
                const float4 x = make_float4(__shfl_xor_sync(0xffffffffu, v.x, 16), __shfl_xor_sync(0xffffffffu, v.y, 16),
                                             __shfl_xor_sync(0xffffffffu, v.z, 16), __shfl_xor_sync(0xffffffffu, v.w, 16));
                const float m1 = __shfl_xor_sync(0xffffffffu, top, 16), l1 = __shfl_xor_sync(0xffffffffu, total, 16);
                add(m1, l1, x);
            }
            if (lane < kLanes) *reinterpret_cast<float4 *>(share + id * D + lane * 4) = v;
            if (lane == 0) share_ml[2 * id] = top, share_ml[2 * id + 1] = total;
        }
        __syncthreads();
        if (!live) return;
        M = -INFINITY, L = 0.f;
        for (int w = row * shares; w < (row + 1) * shares; ++w) M = fmaxf(M, share_ml[2 * w]);
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum[i] = 0.f;
        for (int w = row * shares; w < (row + 1) * shares; ++w) {
            const float f = share_ml[2 * w] == M ? 1.f : ex2_approx(share_ml[2 * w] - M);
            L = fmaf(share_ml[2 * w + 1], f, L);
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum[i] = fmaf(share[w * D + d0 + i], f, sum[i]);
        }
    }
    if (!live) return;
    const float inv = L == 0.f ? 0.f : 1.f / L;  // a row that sees no key yields zeros
    const int64_t at = (q.r0 + static_cast<int64_t>(r / G)) * a.ys.token + (kv * static_cast<int64_t>(G) + r % G) * a.ys.head + d0;
#pragma unroll
    for (int i = 0; i < kEach; i += 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sum[i + k] * inv;
        kv_store8(a, at + i, v);
    }
}

// The parts of a key range and the launch; `bit`: the kernel's of a.ready.
template <typename F, int NT, typename Args>
cudaError_t few_launch(void (*kernel)(Args), Args &a, unsigned bit, int num_sms, cudaStream_t st) {
    const int64_t units = ((static_cast<int64_t>(a.b.n_rows) * a.group) >> (NT == 1 ? 3 : 4)) + a.b.n_seqs;
    // parts for two waves where there are few sequences and heads, for four where the lengths of many have to even out
    const int64_t wave = F::kBlocks * static_cast<int64_t>(num_sms), groups = units * a.c.heads;
    const int64_t span =
        std::max(a.window ? std::min(a.b.max_len, static_cast<int64_t>(a.window) + a.b.max_rows + 16) : a.b.max_len, int64_t(1));
    int64_t splits = 2 * groups < wave ? (2 * wave + groups - 1) / groups : (4 * wave + groups - 1) / groups;
    // a block's least part: a turn of its warps while the blocks fit in one wave, else 256
    const int64_t least = groups * ((span + F::kTurn - 1) / F::kTurn) <= wave ? F::kTurn : 256;
    splits = std::min(splits, (span + least - 1) / least);
    splits = std::min(splits, std::min(static_cast<int64_t>(kMaxParts) / groups, static_cast<int64_t>(kMaxSplits)));
    splits = std::max(splits, static_cast<int64_t>(1));
    if (units * splits > 0x7fffffff) return cudaErrorInvalidValue;
    a.splits = static_cast<int>(splits);
    a.chunk = static_cast<int>(((span + splits - 1) / splits + 63) & ~int64_t(63));
    // With few sequences one that is far shorter than max_len (a captured step's bound) is cut finer, into all parts.
    a.chunk_short = static_cast<int>(2 * groups < wave ? std::min<int64_t>(least, a.chunk) : a.chunk);
    a.short_range = static_cast<int>(span / 2);
    if (!(*a.ready & (1u << bit))) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        if (e != cudaSuccess) return e;
        *a.ready |= 1u << bit;
    }
    const dim3 grid(static_cast<unsigned>(units * a.splits), a.c.heads);
    return launch_after(kernel, grid, kWarps * 32, F::kSmem, st, a);
}

}  // namespace b200
