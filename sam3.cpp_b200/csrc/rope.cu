// rope.cu -- rotary positions with up to four axes (time, height, width, ...)
// for the heads of any [rows][heads][D] tensor.
//
// Pair i of a head is turned by the angle pos[axis(i)][row] w(i):
//   y0 = x0 cos - x1 sin,  y1 = x1 cos + x0 sin,
//   w(i) = base^(-i / n), or base^(-j / n_axis) with the pair's place j in its
//   own axis (`restart`).
// The frequencies come from the host as turns a position, w / 2 pi, in 64
// bits: the product with the position loses its whole turns there (far
// positions would lose the angle in 32 bits) and the remaining half turns go
// to sincospif, good to 2^-23 or so.
//
// Bound by memory (one read, one write).  A block owns a few rows (128
// pairs of cosines and sines, one or so for each of its threads, through
// shared memory); a thread has 8 pairs of a row in registers and walks over
// every eighth head with 16-byte loads.  An angle costs 50 to 100
// instructions, so it is computed once for a row and not by each thread.
// Measured: 21037 rows of 40 heads of 128, bf16, 77 us, 5.6 TB/s; 5184 rows of
// 32 heads of 64, f32 to f16, 12.5 us, 5.1 TB/s; 7 rows of 40 heads 2.3 us.
#include <algorithm>
#include <cmath>
#include <new>

#include "rope.cuh"

namespace b200 {
namespace {

struct RopeArgs {
    RopeTable t;
    const void *x;
    void *y;
    RowTensor xs, ys;
    const int32_t *pos;
    int64_t pos_stride;
    int n_rows, n_heads, heads_each;  // heads a thread walks over
    float sign;
};

// Blocks of `rows` rows; a thread: 8 pairs, or 16 elements behind the turned ones, of every eighth head, one at a time:
// more blocks an SM serve better than more loads a thread (21037 rows of 40 heads of 128, bf16: 80 us, two heads at a
// time 91, the next head's loads ahead 91).
template <typename TX, typename TY, bool NEIGHBOURS>
__global__ void __launch_bounds__(128) rope_kernel(const __grid_constant__ RopeArgs a, int rows) {
    __shared__ float2 turn[128];
    wait_for_stream();
    const int n = a.t.pairs, each = a.t.head_dim / 16;  // parts of a row
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows;
    const int part = threadIdx.x % each, lane = threadIdx.x / each % kHeadLanes, row_in = threadIdx.x / (each * kHeadLanes);
    const int64_t row = row0 + row_in;
    const bool turned = part < n / 8;
    int d0, d1;  // first elements of the two groups of 8
    if (NEIGHBOURS || !turned) d0 = part * 16, d1 = d0 + 8;
    else d0 = part * 8, d1 = n + part * 8;
    int h = blockIdx.y * a.heads_each + lane;
    const int h1 = row < a.n_rows ? min(static_cast<int>(blockIdx.y + 1) * a.heads_each, a.n_heads) : 0;
    const TX *x = static_cast<const TX *>(a.x) + row * a.xs.token;
    TY *y = static_cast<TY *>(a.y) + row * a.ys.token;
    for (int id = threadIdx.x; id < rows * n; id += blockDim.x) {
        const int64_t r = row0 + id / n;
        if (r >= a.n_rows) break;
        int p[4];
        positions(a.t, a.pos, a.pos_stride, static_cast<int>(r), p);
        angle(a.t, a.sign, id % n, p, turn[id].x, turn[id].y);
    }
    __syncthreads();
    float c[8], s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 z = turned ? turn[row_in * n + part * 8 + j] : make_float2(1.f, 0.f);
        c[j] = z.x, s[j] = z.y;
    }
#pragma unroll 1
    while (h < h1) {
        const int at = h;
        Stream8<TX> u, v;
        u.load(x + h * a.xs.head + d0);
        v.load(x + h * a.xs.head + d1);
        float f[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = u[j], g[j] = v[j];
        h += kHeadLanes;
        if (turned) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (NEIGHBOURS) {  // pair j is (f, g)[2j], (f, g)[2j + 1]
                    float &e = j < 4 ? f[2 * j] : g[2 * j - 8], &o = j < 4 ? f[2 * j + 1] : g[2 * j - 7];
                    const float x0 = e, x1 = o;
                    e = x0 * c[j] - x1 * s[j];
                    o = x1 * c[j] + x0 * s[j];
                } else {
                    const float x0 = f[j], x1 = g[j];
                    f[j] = x0 * c[j] - x1 * s[j];
                    g[j] = x1 * c[j] + x0 * s[j];
                }
            }
        }
        store8<true>(y + at * a.ys.head + d0, f);
        store8<true>(y + at * a.ys.head + d1, g);
    }
}

// Any head dim, pair count, stride and alignment: one pair, or one element
// behind the turned ones, a thread.
template <typename TX, typename TY>
__global__ void __launch_bounds__(128) rope_any_kernel(const __grid_constant__ RopeArgs a) {
    wait_for_stream();
    const int n = a.t.pairs, each = a.t.head_dim - n;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
    const int64_t row64 = id / each;
    if (row64 >= a.n_rows) return;
    const int row = static_cast<int>(row64), part = static_cast<int>(id % each);
    const int h0 = blockIdx.y * a.heads_each, h1 = min(h0 + a.heads_each, a.n_heads);
    const TX *x = static_cast<const TX *>(a.x) + row * a.xs.token;
    TY *y = static_cast<TY *>(a.y) + row * a.ys.token;
    if (part >= n) {
        for (int h = h0; h < h1; ++h)
            y[h * a.ys.head + n + part] = from_f32<TY>(to_f32(x[h * a.xs.head + n + part]));
        return;
    }
    int p[4];
    positions(a.t, a.pos, a.pos_stride, row, p);
    float c, s;
    angle(a.t, a.sign, part, p, c, s);
    const int d0 = a.t.neighbours ? 2 * part : part, d1 = a.t.neighbours ? 2 * part + 1 : part + n;
    for (int h = h0; h < h1; ++h) {
        const float x0 = to_f32(x[h * a.xs.head + d0]), x1 = to_f32(x[h * a.xs.head + d1]);
        y[h * a.ys.head + d0] = from_f32<TY>(x0 * c - x1 * s);
        y[h * a.ys.head + d1] = from_f32<TY>(x1 * c + x0 * s);
    }
}

template <typename TX, typename TY>
cudaError_t launch_rope(RopeArgs &a, bool wide, cudaStream_t st, int num_sms) {
    if (wide) {
        const int each = a.t.head_dim / 16, rows = std::max(16 / each, 1);  // 128 pairs at most
        const int64_t blocks = (static_cast<int64_t>(a.n_rows) + rows - 1) / rows;
        // heads are split over blocks only where the rows give fewer than 8 blocks an SM
        const int64_t split = (num_sms * int64_t(8) + blocks - 1) / blocks;
        a.heads_each = static_cast<int>((a.n_heads + split - 1) / split + kHeadLanes - 1) / kHeadLanes * kHeadLanes;
        const dim3 grid(static_cast<unsigned>(blocks), (a.n_heads + a.heads_each - 1) / a.heads_each);
        return launch_after(a.t.neighbours ? rope_kernel<TX, TY, true> : rope_kernel<TX, TY, false>, grid,
                            rows * each * kHeadLanes, 0, st, a, rows);
    }
    // a thread walks over all heads where the rows alone fill the GPU (2048 threads an SM), else over fewer
    const int64_t threads = static_cast<int64_t>(a.n_rows) * (a.t.head_dim - a.t.pairs);
    const int64_t split = (num_sms * int64_t(2048) + threads - 1) / threads;
    a.heads_each = static_cast<int>(split >= a.n_heads ? 1 : (a.n_heads + split - 1) / split);
    const dim3 grid(static_cast<unsigned>((threads + 127) / 128), (a.n_heads + a.heads_each - 1) / a.heads_each);
    return launch_after(rope_any_kernel<TX, TY>, grid, 128, 0, st, a);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" sam3b200_rope *sam3b200_rope_create(sam3b200_backend *h, const sam3b200_rope_hparams *p) {
    if (!h || !p) {
        set_error("rope_create: null argument");
        return nullptr;
    }
    int64_t pairs = 0;
    bool ok = p->head_dim >= 2 && p->head_dim <= 2 * kMaxPairs && p->n_axes >= 1 && p->n_axes <= 4;
    for (int k = 0; ok && k < p->n_axes; ++k) {
        ok = p->sections[k] >= 0;
        pairs += p->sections[k];
    }
    if (!ok || pairs < 1 || 2 * pairs > p->head_dim || !(p->base > 0.0) || !std::isfinite(p->base) ||
        !std::isfinite(p->pos_scale)) {
        set_error("rope_create: bad parameters: head_dim %d (2 to %d), %d axes (1 to 4) of %lld pairs (1 to head_dim / 2), "
                  "base %g, pos_scale %g",
                  p->head_dim, 2 * kMaxPairs, p->n_axes, (long long)pairs, p->base, p->pos_scale);
        return nullptr;
    }
    auto *r = new (std::nothrow) Rope();
    if (!r) {
        set_error("rope_create: out of host memory");
        return nullptr;
    }
    r->be = reinterpret_cast<Backend *>(h);
    RopeTable &t = r->t;
    t.head_dim = p->head_dim, t.pairs = static_cast<int>(pairs), t.n_axes = p->n_axes, t.neighbours = p->neighbours != 0;
    int used[4] = {0, 0, 0, 0}, ax = 0;
    for (int i = 0; i < t.pairs; ++i) {
        while (used[ax] >= p->sections[ax]) ax = (ax + 1) % p->n_axes;
        const double power = p->restart ? static_cast<double>(used[ax]) / p->sections[ax] : static_cast<double>(i) / t.pairs;
        t.turns[i] = p->pos_scale * std::pow(p->base, -power) / 6.283185307179586476925286766559;
        t.axis[i] = static_cast<uint8_t>(ax);
        ++used[ax];
        if (p->deal) ax = (ax + 1) % p->n_axes;
    }
    return reinterpret_cast<sam3b200_rope *>(r);
}

extern "C" void sam3b200_rope_free(sam3b200_rope *h) { delete reinterpret_cast<Rope *>(h); }

extern "C" int sam3b200_rope_run(sam3b200_rope *h, int x_type, const void *x, const int64_t *x_nb, const int32_t *pos,
                                 int64_t pos_stride, int64_t n_rows, int64_t n_heads, int inverse, int y_type, void *y,
                                 const int64_t *y_nb) {
    auto *r = reinterpret_cast<Rope *>(h);
    if (!r || !x || !y || !pos) {
        set_error("rope: null argument");
        return SAM3B200_STATUS_FAILED;
    }
    const int xb = type_bytes(x_type), yb = type_bytes(y_type);
    if (!xb || !yb || reinterpret_cast<uintptr_t>(x) % xb || reinterpret_cast<uintptr_t>(y) % yb ||
        reinterpret_cast<uintptr_t>(pos) % 4) {
        set_error("rope: unsupported types %d -> %d (F32=0, F16=1, BF16=30) or unaligned data", x_type, y_type);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_rows < 0 || n_rows > (1 << 27) || n_heads < 0 || n_heads > 65535 || pos_stride < 0 ||
        (r->t.n_axes > 1 && pos_stride < n_rows)) {
        set_error("rope: bad shape: %lld rows, %lld heads, position stride %lld", (long long)n_rows, (long long)n_heads,
                  (long long)pos_stride);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_rows == 0 || n_heads == 0) return SAM3B200_STATUS_SUCCESS;
    RopeArgs a;
    a.t = r->t;
    a.x = x, a.y = y;
    a.xs = row_tensor(x, x_type, x_nb, n_heads, a.t.head_dim);
    a.ys = row_tensor(y, y_type, y_nb, n_heads, a.t.head_dim);
    if (!rows_ok("rope", "x", a.xs, n_rows, n_heads, a.t.head_dim, false) ||
        !rows_ok("rope", "y", a.ys, n_rows, n_heads, a.t.head_dim, true))
        return SAM3B200_STATUS_FAILED;
    if (x == y && (xb != yb || x_type != y_type || a.xs.token != a.ys.token || a.xs.head != a.ys.head)) {
        set_error("rope: in place, x and y must have one type and the same strides");
        return SAM3B200_STATUS_FAILED;
    }
    a.pos = pos, a.pos_stride = pos_stride;
    a.n_rows = static_cast<int>(n_rows), a.n_heads = static_cast<int>(n_heads);
    a.sign = inverse ? -1.f : 1.f;
    // 16-byte groups of 8 pairs: whole groups, aligned rows
    const bool wide = a.xs.aligned16 && a.ys.aligned16 && a.t.pairs % 8 == 0 && a.t.head_dim % 16 == 0;
    DeviceScope dev(r->be->device);
    auto go = [&](auto tx, auto ty) { return launch_rope<decltype(tx), decltype(ty)>(a, wide, r->be->stream, r->be->num_sms); };
    auto from = [&](auto tx) {
        return y_type == SAM3B200_TYPE_F32 ? go(tx, float()) : y_type == SAM3B200_TYPE_F16 ? go(tx, __half()) : go(tx, __nv_bfloat16());
    };
    const cudaError_t e = x_type == SAM3B200_TYPE_F32   ? from(float())
                          : x_type == SAM3B200_TYPE_F16 ? from(__half())
                                                        : from(__nv_bfloat16());
    r->be->count();
    return cuda_ok(e, "rope launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
