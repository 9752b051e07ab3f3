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
// Measured: 21037 rows of 32 + 8 heads of 128 in bf16 87.8 us, 4.9 TB/s (the
// rotation alone 77), with 70 % of the issue slots taken: a head costs the sums,
// the shuffles and two conversions an element on top of the turn.  5184 rows of
// 32 heads of 64, f32 to f16, 16.8 us (64 MB; floor 9.8), in 1296 blocks at 5 an
// SM, 1.75 waves: no unit is busy (issue 42 %, DRAM 27 % of its nominal rate),
// so it is the time from a block's first loads to its last stores, with a last
// wave that leaves a quarter of the places empty.  rope_norm_any_kernel, for pairs
// that do not come in eights and unaligned rows: the first with 61 pairs 421 us, the
// second with 31 pairs 93.  (ptxas spills 8 to 20 bytes of the kernels from 16 bits
// to f32, at 7 blocks an SM.)
// Weights kept in registers for arithmetic on pairs: 124 us, for lack of them;
// several row turns a block in place of one: 105.
#include <algorithm>
#include <cmath>

#include "ptx.cuh"
#include "rope.cuh"

namespace b200 {
namespace {

constexpr int kMaxSets = 4;
// Blocks an SM that the registers are cut for (us, a video prompt of 40 heads of 128 in bf16: 6 blocks 92, 7 87.8, 8 90; an
// image of 32 heads of 64, f32 to f16: 4 blocks 19.5, 5 16.8, 6 17.6).
template <typename TX>
constexpr int kBlocks = sizeof(TX) == 2 ? 7 : 5;
constexpr float kEpsLeast = 1.17549435e-38f;
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
    int w_type, layer;
    float eps, inv_dim;
};

__device__ __forceinline__ float weight_at(const void *w, int type, int i, float none) {
    if (!w) return none;
    if (type == SAM3B200_TYPE_F32) return static_cast<const float *>(w)[i];
    if (type == SAM3B200_TYPE_F16) return to_f32(static_cast<const __half *>(w)[i]);
    return to_f32(static_cast<const __nv_bfloat16 *>(w)[i]);
}

// Off by 2^-22 at most, beside the 14 roundings of 2^-24 that a head's sum and its use take: far below half a step of 16-bit
// results (2^-11), and one instruction a head.
__device__ __forceinline__ float rsqrt_approx(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Over the 16 elements of this lane and those of its group of lanes (a power of two of them; `mine`: this one has
// elements of the head): what is taken off each element, and what it is multiplied by, (x - mean) / sqrt(var + eps).
// Where the squares pass f32 the elements become 2^-70 times as large first.
template <bool CENTER>
__device__ __forceinline__ void moments(float (&f)[16], bool mine, int lanes, float inv_dim, float eps, float &mean, float &by) {
    auto total = [&](float s) {
        s = mine ? s : 0.f;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1)
            if (o < lanes) s += __shfl_xor_sync(0xffffffffu, s, o);  // (the block's threads agree)
        return s;
    };
    auto variance = [&] {
        mean = 0.f;
        if (CENTER) {
            float s0 = f[0], s1 = f[1];
#pragma unroll
            for (int i = 2; i < 16; i += 2) fadd2(s0, s1, s0, s1, f[i], f[i + 1]);
            mean = total(s0 + s1) * inv_dim;
        }
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            float d0 = f[i], d1 = f[i + 1];
            if (CENTER) fadd2(d0, d1, d0, d1, -mean, -mean);
            ffma2(s0, s1, d0, d1, d0, d1);
        }
        return total(s0 + s1);
    };
    float sum = variance();
    if (__any_sync(0xffffffffu, !(sum <= kSumMost))) {  // elements above 2^60 or so
        if (!(sum <= kSumMost)) {
#pragma unroll
            for (int i = 0; i < 16; ++i) f[i] *= kShrink;
            eps *= kShrink * kShrink;
        }
        sum = variance();
    }
    by = rsqrt_approx(fmaf(sum, inv_dim, eps));
}

// Blocks of `rows` rows; a thread: 8 pairs, or 16 elements behind the turned ones, of every eighth head (see rope.cu), the
// next head's on their way while one is worked on.  lanes: threads of a head, head_dim / 16 rounded up to a power of two.
// PLAIN: an RMS norm without biases.
template <typename TX, typename TY, bool NEIGHBOURS, bool PLAIN>
__global__ void __launch_bounds__(128, kBlocks<TX>) rope_norm_kernel(const __grid_constant__ RopeNormArgs a, int rows, int lanes) {
    __shared__ __align__(16) float2 turn[128];
    extern __shared__ __align__(16) float weights[];
    wait_for_stream();
    const int n = a.t.pairs, D = a.t.head_dim, lanes_log2 = 31 - __clz(lanes);
    const int part = threadIdx.x & (lanes - 1), lane = (threadIdx.x >> lanes_log2) % kHeadLanes, row_in = threadIdx.x >> lanes_log2 >> 3;
    static_assert(kHeadLanes == 8, "row_in");
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows, row = min(row0 + row_in, static_cast<int64_t>(a.n_rows) - 1);
    const bool turned = part < n / 8, mine = part < D / 16, here = mine && row0 + row_in < a.n_rows;
    int d0, d1;  // first elements of the two groups of 8; threads without any look at the first ones
    if (NEIGHBOURS || !turned) d0 = mine ? part * 16 : 0, d1 = d0 + 8;
    else d0 = part * 8, d1 = n + part * 8;

    const int h_end = min(static_cast<int>(blockIdx.y + 1) * a.heads_each, a.set[a.n_sets - 1].end);
    int h = blockIdx.y * a.heads_each + lane;  // this lane's head, counted over all sets
    // A walk over this lane's heads of x, and another of y: the set, its end, the head's elements, the way to the next head.
    int x_set = -1, x_end = 0, y_set = -1, y_end = 0;
    const TX *x = nullptr;
    TY *y = nullptr;
    int64_t x_step = 0, y_step = 0;
    auto seek = [&](int at, int &set, int &end) {
        int first = 0;
        do {
            ++set;
            first = set ? a.set[set - 1].end : 0;
            end = a.set[set].end;
        } while (at >= end);
        return at - first;
    };
    auto x_seek = [&](int at) {
        const int k = seek(at, x_set, x_end);
        const HeadSet &q = a.set[x_set];
        x = static_cast<const TX *>(q.x) + row * q.xs.token + k * q.xs.head, x_step = kHeadLanes * q.xs.head;
    };
    auto y_seek = [&](int at) {
        const int k = seek(at, y_set, y_end);
        const HeadSet &q = a.set[y_set];
        y = static_cast<TY *>(q.y) + row * q.ys.token + k * q.ys.head, y_step = kHeadLanes * q.ys.head;
    };
    x_seek(min(h, h_end - 1));  // (lanes behind the end look at the last head)
    Stream8<TX> u, v;
    u.load(x + d0);
    v.load(x + d1);
    // weights in the order in which the threads of a head read them, 4 at a time: [set][weight, bias][4 of a thread's 16][thread]
    for (int id = threadIdx.x; id < a.n_sets * D; id += blockDim.x) {
        const int k = id / D, i = id % D;
        const bool half = !NEIGHBOURS && i < 2 * n;
        const int of = half ? i % n / 8 : i / 16, e = half ? i % n % 8 + i / n * 8 : i % 16;
        float *to = weights + ((2 * k * 4 + e / 4) * lanes + of) * 4 + e % 4;
        *to = weight_at(a.set[k].weight, a.w_type, i, 1.f);
        if (!PLAIN) to[16 * lanes] = weight_at(a.set[k].bias, a.w_type, i, 0.f);
    }
    for (int id = threadIdx.x; id < rows * n; id += blockDim.x) {
        const int64_t r = row0 + id / n;
        if (r >= a.n_rows) break;
        int p[4];
        positions(a.t, a.pos, a.pos_stride, static_cast<int>(r), p);
        angle(a.t, 1.f, id % n, p, turn[id].x, turn[id].y);
    }
    __syncthreads();
    // f[j] and f[j + 8] are pair j: of the 16 elements the halves, or the even and the odd ones
    auto place = [](int e) { return NEIGHBOURS ? (e & 1) * 8 + (e >> 1) : e; };
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float4 z = make_float4(1.f, 0.f, 1.f, 0.f);
        if (turned) z = *reinterpret_cast<const float4 *>(&turn[row_in * n + part * 8 + j]);
        c[j] = z.x, s[j] = z.y, c[j + 1] = z.z, s[j + 1] = z.w;
    }
#pragma unroll 1
    for (int k = blockIdx.y * a.heads_each; k < h_end; k += kHeadLanes, h += kHeadLanes) {  // all lanes, for the shuffles
        float f[16], mean = 0.f, by;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[place(j)] = u[j], f[place(j + 8)] = v[j];
        if (h + kHeadLanes < h_end) {
            if (h + kHeadLanes < x_end) x += x_step;
            else x_seek(h + kHeadLanes);
            u.load(x + d0);
            v.load(x + d1);
        }
        if (PLAIN || !a.layer) moments<false>(f, mine, lanes, a.inv_dim, a.eps, mean, by);
        else moments<true>(f, mine, lanes, a.inv_dim, a.eps, mean, by);
        if (!here || h >= h_end) continue;
        if (h < y_end) y += y_step;
        else y_seek(h);
        // (weights stay in shared memory: their registers are worth more as blocks an SM)
        const float *w = weights + (8 * y_set * lanes + part) * 4;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 z = *reinterpret_cast<const float4 *>(w + e * lanes);
            float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!PLAIN) b = *reinterpret_cast<const float4 *>(w + (16 + e) * lanes);
            f[place(e)] = fmaf((f[place(e)] - mean) * by, z.x, b.x), f[place(e + 1)] = fmaf((f[place(e + 1)] - mean) * by, z.y, b.y);
            f[place(e + 2)] = fmaf((f[place(e + 2)] - mean) * by, z.z, b.z), f[place(e + 3)] = fmaf((f[place(e + 3)] - mean) * by, z.w, b.w);
        }
        if (turned) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x0 = f[j], x1 = f[j + 8];
                f[j] = x0 * c[j] - x1 * s[j];
                f[j + 8] = x1 * c[j] + x0 * s[j];
            }
        }
        float lo8[8], hi8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) lo8[j] = f[place(j)], hi8[j] = f[place(j + 8)];
        store8<true>(y + d0, lo8);
        store8<true>(y + d1, hi8);
    }
}

// Any head dim, pair count, stride and alignment: a warp a row and share of its heads, one head at a time through
// shared memory, the angles of its row in registers.
template <typename TX, typename TY>
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
                if (a.layer) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) mean += f[k] * by;
                    for (int o = 16; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
                    mean *= a.inv_dim;
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
            const float r = rsqrt_approx(fmaf(sum, a.inv_dim, a.eps * by * by));
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

template <typename TX, typename TY>
cudaError_t launch_rope_norm(RopeNormArgs &a, bool wide, bool plain, cudaStream_t st, int num_sms) {
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
        const dim3 grid = split_heads((static_cast<int64_t>(a.n_rows) + rows - 1) / rows, num_sms * int64_t(8), kHeadLanes);
        auto *const kernel = plain ? (a.t.neighbours ? rope_norm_kernel<TX, TY, true, true> : rope_norm_kernel<TX, TY, false, true>)
                                   : (a.t.neighbours ? rope_norm_kernel<TX, TY, true, false> : rope_norm_kernel<TX, TY, false, false>);
        return launch_after(kernel, grid, rows * lanes * kHeadLanes, a.n_sets * 2 * 16 * lanes * sizeof(float), st, a, rows, lanes);
    }
    const dim3 grid = split_heads((static_cast<int64_t>(a.n_rows) + 3) / 4, num_sms * int64_t(16), 1);
    return launch_after(rope_norm_any_kernel<TX, TY>, grid, 128, 0, st, a);
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
    if (n_sets < 1 || n_sets > kMaxSets || !(eps >= kEpsLeast) || !std::isfinite(eps)) {
        set_error("rope_norm: %d sets of heads (1 to %d), eps %g (a normal number above 0)", n_sets, kMaxSets, eps);
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
    bool plain = !layer;
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
        wide = wide && q.xs.aligned16 && q.ys.aligned16, plain = plain && !q.bias;
    }
    if (n_rows == 0 || heads == 0) return SAM3B200_STATUS_SUCCESS;
    a.pos = pos, a.pos_stride = pos_stride;
    a.n_rows = static_cast<int>(n_rows);
    a.w_type = w_type, a.layer = layer != 0, a.eps = eps, a.inv_dim = 1.f / D;
    DeviceScope dev(r->be->device);
    auto go = [&](auto tx, auto ty) {
        return launch_rope_norm<decltype(tx), decltype(ty)>(a, wide, plain, r->be->stream, r->be->num_sms);
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
