// rope_norm.cu -- queries and keys normalised for each head and turned by
// their positions, in one pass over them.
//
//   RMS norm:    u = x / sqrt(mean(x^2) + eps) w  (+ b)
//   layer norm:  u = (x - mean(x)) / sqrt(mean((x - mean(x))^2) + eps) w  (+ b)
//   y = u turned as in rope.cu
// over the head_dim elements of a head, in f32, rounded once, to y's type.
//
// Bound by memory (one read, one write), with a chain of shuffles between
// the two: the layout is rope.cu's (a thread has 16 elements of a head, 2 to 16
// threads a head), so the sums of a head are 16 terms in a thread and one
// to four shuffles.  Up to four sets of heads (queries and keys, each with
// its weights) share a launch and the angles of a row.
#include <algorithm>
#include <cmath>

#include "rope.cuh"

namespace b200 {
namespace {

constexpr int kMaxSets = 4;
constexpr float kSumMost = 3e38f;               // sums of squares above this are taken again, of elements
constexpr float kShrink = 8.470329472543003e-22f;  // 2^-70 times as large

struct HeadSet {
    const void *x, *weight, *bias;
    void *y;
    RowTensor xs, ys;
    int end;  // heads of this set and those in front of it
};

struct RopeNormArgs {
    RopeTable t;
    HeadSet set[kMaxSets];
    const int32_t *pos;
    int64_t pos_stride;
    int n_sets, n_rows, heads_each;  // heads that a block walks over
    int w_type;
    float eps;
};

__device__ __forceinline__ float weight_at(const void *w, int type, int i, float none) {
    if (!w) return none;
    if (type == SAM3B200_TYPE_F32) return static_cast<const float *>(w)[i];
    if (type == SAM3B200_TYPE_F16) return to_f32(static_cast<const __half *>(w)[i]);
    return to_f32(static_cast<const __nv_bfloat16 *>(w)[i]);
}

// The N elements of this lane become (x - mean) / sqrt(var + eps) over the elements of its group of lanes (a power of
// two of them); lanes without elements of the head bring zeros and live = false.
template <bool LAYER, int N>
__device__ __forceinline__ void normalise(float (&f)[N], bool live, int lanes, float dim, float eps) {
    auto total = [&](float s) {
        for (int o = lanes >> 1; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    auto squares = [&] {
        if (LAYER) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) s += f[i];
            const float mean = total(s) / dim;
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = live ? f[i] - mean : 0.f;
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(f[i], f[i], s);
        return total(s);
    };
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = f[i];
    float sum = squares();
    if (__any_sync(0xffffffffu, !(sum <= kSumMost))) {  // elements above 2^60 or so
        const float by = sum <= kSumMost ? 1.f : kShrink;
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = x[i] * by;
        sum = squares();
        eps *= by * by;
    }
    const float r = __frsqrt_rn(sum / dim + eps);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] *= r;
}

// Blocks of `rows` rows; 8 pairs, or 16 elements behind the turned ones, of every eighth head a thread (see rope.cu).
// lanes: threads of a head, head_dim / 16 rounded up to a power of two.
template <typename TX, typename TY, bool NEIGHBOURS, bool LAYER>
__global__ void __launch_bounds__(128) rope_norm_kernel(const __grid_constant__ RopeNormArgs a, int rows, int lanes) {
    __shared__ float2 turn[128];
    extern __shared__ __align__(16) float weights[];  // [set][weight, bias][head_dim]
    wait_for_stream();
    const int n = a.t.pairs, D = a.t.head_dim;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows;
    const int part = threadIdx.x & (lanes - 1), lane = threadIdx.x / lanes % kHeadLanes, row_in = threadIdx.x / (lanes * kHeadLanes);
    const int64_t row = row0 + row_in;
    const bool turned = part < n / 8, mine = part < D / 16 && row < a.n_rows;
    int d0, d1;  // first elements of the two groups of 8
    if (NEIGHBOURS || !turned) d0 = part * 16, d1 = d0 + 8;
    else d0 = part * 8, d1 = n + part * 8;
    for (int id = threadIdx.x; id < a.n_sets * D; id += blockDim.x) {
        const int s = id / D, i = id % D;
        weights[2 * s * D + i] = weight_at(a.set[s].weight, a.w_type, i, 1.f);
        weights[(2 * s + 1) * D + i] = weight_at(a.set[s].bias, a.w_type, i, 0.f);
    }
    for (int id = threadIdx.x; id < rows * n; id += blockDim.x) {
        const int64_t r = row0 + id / n;
        if (r >= a.n_rows) break;
        int p[4];
        positions(a.t, a.pos, a.pos_stride, static_cast<int>(r), p);
        angle(a.t, 1.f, id % n, p, turn[id].x, turn[id].y);
    }
    __syncthreads();
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 z = turned && mine ? turn[row_in * n + part * 8 + j] : make_float2(1.f, 0.f);
        c[j] = z.x, s[j] = z.y;
    }
    const int h_begin = blockIdx.y * a.heads_each, h_end = h_begin + a.heads_each;
#pragma unroll 1
    for (int i = 0, first = 0; i < a.n_sets; first = a.set[i].end, ++i) {
        const HeadSet &q = a.set[i];
        const int lo = max(h_begin, first), hi = min(h_end, q.end);
        if (lo >= hi) continue;
        float w[16], b[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            w[j] = mine ? weights[2 * i * D + d0 + j] : 0.f, w[j + 8] = mine ? weights[2 * i * D + d1 + j] : 0.f;
            b[j] = mine ? weights[(2 * i + 1) * D + d0 + j] : 0.f, b[j + 8] = mine ? weights[(2 * i + 1) * D + d1 + j] : 0.f;
        }
        const TX *x = static_cast<const TX *>(q.x) + row * q.xs.token;
        TY *y = static_cast<TY *>(q.y) + row * q.ys.token;
#pragma unroll 1
        for (int h0 = lo; h0 < hi; h0 += kHeadLanes) {  // all lanes, for the shuffles
            const int h = h0 + lane - first;
            const bool live = mine && h0 + lane < hi;
            float f[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = 0.f;
            if (live) {
                Stream8<TX> u, v;
                u.load(x + h * q.xs.head + d0);
                v.load(x + h * q.xs.head + d1);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = u[j], f[j + 8] = v[j];
            }
            normalise<LAYER>(f, live, lanes, static_cast<float>(D), a.eps);
            if (!live) continue;
#pragma unroll
            for (int j = 0; j < 16; ++j) f[j] = fmaf(f[j], w[j], b[j]);
            float lo8[8], hi8[8];
            if (turned) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {  // pair j: elements j and j + 8 of the 16, or 2 j and 2 j + 1
                    const int e0 = NEIGHBOURS ? 2 * j : j, e1 = NEIGHBOURS ? 2 * j + 1 : j + 8;
                    const float x0 = f[e0], x1 = f[e1];
                    f[e0] = x0 * c[j] - x1 * s[j];
                    f[e1] = x1 * c[j] + x0 * s[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) lo8[j] = f[j], hi8[j] = f[j + 8];
            store8<true>(y + h * q.ys.head + d0, lo8);
            store8<true>(y + h * q.ys.head + d1, hi8);
        }
    }
}

// Any head dim, pair count, stride and alignment: a warp a row and share of its heads, one head at a time through
// shared memory, the angles of its row in registers.
template <typename TX, typename TY, bool LAYER>
__global__ void __launch_bounds__(128) rope_norm_any_kernel(const __grid_constant__ RopeNormArgs a) {
    __shared__ float head[4][2 * kMaxPairs];
    wait_for_stream();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = a.t.pairs, D = a.t.head_dim;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + warp;
    if (row >= a.n_rows) return;
    int p[4];
    positions(a.t, a.pos, a.pos_stride, static_cast<int>(row), p);
    float c[kMaxPairs / 32], s[kMaxPairs / 32];
#pragma unroll
    for (int k = 0; k < kMaxPairs / 32; ++k) {
        c[k] = 1.f, s[k] = 0.f;
        if (lane + 32 * k < n) angle(a.t, 1.f, lane + 32 * k, p, c[k], s[k]);
    }
    const int h_begin = blockIdx.y * a.heads_each, h_end = h_begin + a.heads_each;
    for (int i = 0, first = 0; i < a.n_sets; first = a.set[i].end, ++i) {
        const HeadSet &q = a.set[i];
        for (int h = max(h_begin, first) - first; h < min(h_end, q.end) - first; ++h) {
            const TX *x = static_cast<const TX *>(q.x) + row * q.xs.token + h * q.xs.head;
            TY *y = static_cast<TY *>(q.y) + row * q.ys.token + h * q.ys.head;
            float f[8];
            // elements past the head's are zeros, and stay zeros when the mean is taken off: one lane may have both
            const int have = D > lane ? (D - lane + 31) / 32 : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = k < have ? to_f32(x[lane + 32 * k]) : 0.f;
            float by = 1.f, sum;
            for (int turn = 0;; ++turn) {
                float u[8], mean = 0.f;
                if (LAYER) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) mean += f[k] * by;
                    for (int o = 16; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
                    mean /= static_cast<float>(D);
                }
                sum = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    u[k] = k < have ? f[k] * by - mean : 0.f;
                    sum = fmaf(u[k], u[k], sum);
                }
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (sum <= kSumMost || turn == 1) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] = u[k];
                    break;
                }
                by = kShrink;
            }
            const float r = __frsqrt_rn(sum / static_cast<float>(D) + a.eps * by * by);
            __syncwarp();  // the head before is read
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int d = lane + 32 * k;
                if (k < have)
                    head[warp][d] = fmaf(f[k] * r, weight_at(q.weight, a.w_type, d, 1.f), weight_at(q.bias, a.w_type, d, 0.f));
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kMaxPairs / 32; ++k) {
                const int j = lane + 32 * k;
                if (j >= n) continue;
                const int d0 = a.t.neighbours ? 2 * j : j, d1 = a.t.neighbours ? 2 * j + 1 : j + n;
                const float x0 = head[warp][d0], x1 = head[warp][d1];
                y[d0] = from_f32<TY>(x0 * c[k] - x1 * s[k]);
                y[d1] = from_f32<TY>(x1 * c[k] + x0 * s[k]);
            }
            for (int d = 2 * n + lane; d < D; d += 32) y[d] = from_f32<TY>(head[warp][d]);
        }
    }
}

template <typename TX, typename TY, bool LAYER>
cudaError_t launch_rope_norm(RopeNormArgs &a, bool wide, cudaStream_t st, int num_sms) {
    const int n_heads = a.set[a.n_sets - 1].end;
    auto split_heads = [&](int64_t blocks, int64_t want, int step) {  // heads are split over blocks where the rows give fewer than wanted
        const int64_t split = (want + blocks - 1) / blocks;
        a.heads_each = static_cast<int>((n_heads + split - 1) / split + step - 1) / step * step;
        return dim3(static_cast<unsigned>(blocks), (n_heads + a.heads_each - 1) / a.heads_each);
    };
    if (wide) {
        int lanes = 1;
        while (lanes * 16 < a.t.head_dim) lanes *= 2;
        const int rows = std::max(16 / lanes, 1);  // 128 pairs at most
        const int64_t blocks = (static_cast<int64_t>(a.n_rows) + rows - 1) / rows;
        const dim3 grid = split_heads(blocks, num_sms * int64_t(8), kHeadLanes);
        return launch_after(a.t.neighbours ? rope_norm_kernel<TX, TY, true, LAYER> : rope_norm_kernel<TX, TY, false, LAYER>, grid,
                            rows * lanes * kHeadLanes, a.n_sets * 2 * a.t.head_dim * sizeof(float), st, a, rows, lanes);
    }
    const dim3 grid = split_heads((static_cast<int64_t>(a.n_rows) + 3) / 4, num_sms * int64_t(16), 1);
    return launch_after(rope_norm_any_kernel<TX, TY, LAYER>, grid, 128, 0, st, a);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int sam3b200_rope_norm_run(sam3b200_rope *h, const sam3b200_norm_heads *sets, int n_sets, int x_type, int w_type,
                                      int layer, float eps, const int32_t *pos, int64_t pos_stride, int64_t n_rows, int y_type) {
    auto *r = reinterpret_cast<Rope *>(h);
    if (!r || !sets || !pos) {
        set_error("rope_norm: null argument");
        return SAM3B200_STATUS_FAILED;
    }
    const int xb = type_bytes(x_type), yb = type_bytes(y_type), wb = type_bytes(w_type);
    if (!xb || !yb || !wb || reinterpret_cast<uintptr_t>(pos) % 4) {
        set_error("rope_norm: unsupported types %d -> %d, weights %d (F32=0, F16=1, BF16=30) or unaligned positions", x_type, y_type, w_type);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_sets < 1 || n_sets > kMaxSets || !(eps > 0.f) || !std::isfinite(eps)) {
        set_error("rope_norm: %d sets of heads (1 to %d), eps %g (above 0)", n_sets, kMaxSets, eps);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_rows < 0 || n_rows > (1 << 27) || pos_stride < 0 || (r->t.n_axes > 1 && pos_stride < n_rows)) {
        set_error("rope_norm: bad shape: %lld rows, position stride %lld", (long long)n_rows, (long long)pos_stride);
        return SAM3B200_STATUS_FAILED;
    }
    RopeNormArgs a;
    a.t = r->t;
    const int D = a.t.head_dim;
    // 16-byte groups of 8 pairs: whole groups, aligned rows
    bool wide = a.t.pairs % 8 == 0 && D % 16 == 0;
    int64_t heads = 0;
    a.n_sets = 0;
    for (int i = 0; i < n_sets; ++i) {
        const sam3b200_norm_heads &s = sets[i];
        if (s.n_heads < 0 || s.n_heads > 65535) {
            set_error("rope_norm: set %d has %lld heads (0 to 65535)", i, (long long)s.n_heads);
            return SAM3B200_STATUS_FAILED;
        }
        if (s.n_heads == 0) continue;
        if (!s.x || !s.y) {
            set_error("rope_norm: null argument");
            return SAM3B200_STATUS_FAILED;
        }
        if (reinterpret_cast<uintptr_t>(s.x) % xb || reinterpret_cast<uintptr_t>(s.y) % yb || reinterpret_cast<uintptr_t>(s.weight) % wb ||
            reinterpret_cast<uintptr_t>(s.bias) % wb) {
            set_error("rope_norm: unaligned data in set %d", i);
            return SAM3B200_STATUS_FAILED;
        }
        HeadSet &q = a.set[a.n_sets++];
        q.x = s.x, q.y = s.y, q.weight = s.weight, q.bias = s.bias;
        q.xs = row_tensor(s.x, x_type, s.x_nb, s.n_heads, D);
        q.ys = row_tensor(s.y, y_type, s.y_nb, s.n_heads, D);
        if (!rows_ok("rope_norm", "x", q.xs, n_rows, s.n_heads, D, false) || !rows_ok("rope_norm", "y", q.ys, n_rows, s.n_heads, D, true))
            return SAM3B200_STATUS_FAILED;
        if (s.x == s.y && (x_type != y_type || q.xs.token != q.ys.token || q.xs.head != q.ys.head)) {
            set_error("rope_norm: in place, x and y must have one type and the same strides");
            return SAM3B200_STATUS_FAILED;
        }
        heads += s.n_heads;
        q.end = static_cast<int>(heads);
        wide = wide && q.xs.aligned16 && q.ys.aligned16;
    }
    if (n_rows == 0 || heads == 0) return SAM3B200_STATUS_SUCCESS;
    a.pos = pos, a.pos_stride = pos_stride;
    a.n_rows = static_cast<int>(n_rows);
    a.w_type = w_type, a.eps = eps;
    DeviceScope dev(r->be->device);
    auto go = [&](auto tx, auto ty) {
        using TX = decltype(tx);
        using TY = decltype(ty);
        return layer ? launch_rope_norm<TX, TY, true>(a, wide, r->be->stream, r->be->num_sms)
                     : launch_rope_norm<TX, TY, false>(a, wide, r->be->stream, r->be->num_sms);
    };
    auto from = [&](auto tx) {
        return y_type == SAM3B200_TYPE_F32 ? go(tx, float()) : y_type == SAM3B200_TYPE_F16 ? go(tx, __half()) : go(tx, __nv_bfloat16());
    };
    const cudaError_t e = x_type == SAM3B200_TYPE_F32   ? from(float())
                          : x_type == SAM3B200_TYPE_F16 ? from(__half())
                                                        : from(__nv_bfloat16());
    r->be->count();
    return cuda_ok(e, "rope_norm launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
