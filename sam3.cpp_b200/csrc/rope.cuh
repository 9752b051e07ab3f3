// rope.cuh -- what the kernels that turn heads by their positions share.
#pragma once

#include "kv_cache.cuh"

namespace b200 {

constexpr int kMaxPairs = 128;

struct RopeTable {
    double turns[kMaxPairs];  // w / 2 pi
    uint8_t axis[kMaxPairs];
    int head_dim, pairs, n_axes, neighbours;
};

struct Rope {
    Backend *be;
    RopeTable t;
};

// The turn of pair i for the positions p; sign -1 turns back.
__device__ __forceinline__ void angle(const RopeTable &t, float sign, int i, const int (&p)[4], float &c, float &s) {
    const int ax = t.axis[i];
    const int at = ax == 0 ? p[0] : ax == 1 ? p[1] : ax == 2 ? p[2] : p[3];
    const double turns = at * t.turns[i];
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    s *= sign;
}

__device__ __forceinline__ void positions(const RopeTable &t, const int32_t *pos, int64_t pos_stride, int row, int (&p)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) p[k] = k < t.n_axes ? pos[k * pos_stride + row] : 0;
}

constexpr int kHeadLanes = 8;  // threads that share a row's 8 pairs, over heads

// 8 elements as they come, read past the L1 and soon to be evicted from the L2: nothing is read twice.
template <typename T>
struct Stream8 {
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) raw[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ float operator[](int i) const { return to_f32(reinterpret_cast<const T *>(raw)[i]); }
};

}  // namespace b200
