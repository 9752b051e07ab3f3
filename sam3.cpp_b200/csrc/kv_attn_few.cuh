// kv_attn_few.cuh -- what the kernels for few query rows a kv head share over
// the caches of 8 and 4 bits: how a block's warps' partial results and the
// parts of a key range are joined.
#pragma once

#include <algorithm>

#include "kv_attn.cuh"
#include "mma_sync.cuh"

namespace b200 {

constexpr int kWarps = 4;

// A block's rows and keys.
struct FewTile {
    KvSeq q;
    int kv;
    int split, n_split;       // which part of the tile's keys this is, of how many
    int64_t slot;             // the tile's first part in the workspace, and its counter
    int R, row0, i_lo, i_hi;  // rows of the sequence, this tile's first, its first and last token
    int t_begin, t_end;       // this block's part of the tile's keys
};

// The end of a block: its warps' rows (sums in `smem` as [warp][row][F::kRowFloats], dimension d at F::column(d);
// maxima and sums of weights in s_m and s_l) are joined, the parts of the key range by the last block to finish, and
// the rows stored.  Behind a __syncthreads().
template <typename F, int D, typename Args>
__device__ __forceinline__ void few_finish(const Args &a, const FewTile &t, uint8_t *smem, const float (&s_m)[kWarps][F::kRows],
                                           const float (&s_l)[kWarps][F::kRows]) {
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = t.kv, G = a.group;
    const int row0 = t.row0, R = t.R, split = t.split, n_split = t.n_split;
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
        float *base = a.part + t.slot * F::kRows * (D + 2);
        float *ml = base + static_cast<int64_t>(n_split) * F::kRows * D;
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
            s_last = atomicInc(a.done + t.slot, n_split - 1) == static_cast<unsigned>(n_split - 1);
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

}  // namespace b200
