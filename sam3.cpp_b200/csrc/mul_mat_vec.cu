// mul_mat_vec.cu -- MUL_MAT of 1 to 16 rows with Q4_0 / Q4_1 weights, the
// activations as they are.
//
//   y[m][n] = sum over blocks b of d[n][b] (sum_k (code - 8) x[m][k])
//             (+ (mn[n][b] + 8 d[n][b]) (sum_k x[m][k]) for Q4_1)  + bias[n]
//
// Bound by memory: 18 bytes a block of 32 weights, read once.  A tile is 16 rows
// of the weights; W of a block's 8 warps share it, each with every W-th chunk
// of 128 k, which it copies by cp.async into its own ring of shared memory.  The
// products run on mma.m16n8k16 f16 with f32 sums: the codes are its 16-row
// operand (exact in f16), the rows of x its 8 columns, so up to 8 rows cost what
// one does, and the legacy matrix instruction is wide enough for what memory
// delivers.  Word t of each weight row's block (elements 4t ... and 16 + 4t ...)
// comes to a lane by ldmatrix, a nibble and the one 16 bits above it are one
// operand register after a mask and a subtraction, and x is staged in shared
// memory in the same order.  A block's sum is scaled in f32, 4 multiply-adds a
// lane for 16 x 8 results.
// x as f16: F16 as it is; BF16 after a power of two a row that brings the
// largest element to [2^14, 2^15), exact down to 2^-31 of it, and to 2^-39 of it
// below; F32 the same way as a sum of two f16 numbers in two columns (2^-23 of an
// element at most is lost).
// Warps' sums of a tile are added in their order: results repeat bit for bit.
#include <algorithm>
#include <type_traits>

#include "kv4_codes.cuh"
#include "kv_cache.cuh"
#include "mma_sync.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32, kStages = 4;
constexpr int kMaxRows = 16;
constexpr int kCodeBytes = 16 * 64;  // a chunk: 16 rows of 4 blocks
constexpr int kScaleBytes = 16 * 4 * 2;
constexpr int kXBytes = 64 << 10;    // most shared memory for x: with more k, x comes in phases

struct VecArgs {
    const uint8_t *codes, *scales;
    const void *x;
    int64_t ldx, ldy;
    const float *bias;
    void *y;
    int M, N, K, cols;           // cols: columns of x, M or 2 M
    int tiles, chunks, w_log2;   // warps of a tile
    int phase;                   // chunks of x in shared memory at once, a multiple of 8 or all
    int y_type, aligned;         // aligned: four elements of x at once
};

// f16 of v; `rest`: what it leaves (0 of an infinity or NaN).
__device__ __forceinline__ float f16_of(float v, float &rest) {
    const float h = __half2float(__float2half_rn(v));
    rest = fabsf(h) <= 65504.f ? v - h : 0.f;
    return h;
}

template <typename T>
__device__ __forceinline__ void load4(const T *p, bool aligned, float *v) {
    T e[4];
    if (aligned) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(e) = *reinterpret_cast<const uint4 *>(p);
        else *reinterpret_cast<uint2 *>(e) = *reinterpret_cast<const uint2 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
}

// NT: tiles of 8 columns.
template <int NT, bool MINS, typename TX>
__global__ void __launch_bounds__(kThreads, (NT == 1 ? 4 : NT == 2 ? 3 : 2)) mul_mat_vec_kernel(const __grid_constant__ VecArgs a) {
    constexpr int kParts = sizeof(TX) == 4 ? 2 : 1;  // columns of a row
    constexpr bool kScaled = !std::is_same<TX, __half>::value;
    constexpr int kRecord = MINS ? 2 * kScaleBytes : kScaleBytes, kStageBytes = kCodeBytes + kRecord;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_up[kMaxRows], s_down[kMaxRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int W = 1 << a.w_log2, group = warp >> a.w_log2, w_in = warp & (W - 1), groups = kWarps >> a.w_log2;
    const int rounds = (a.tiles + gridDim.x * groups - 1) / (gridDim.x * groups), blocks = a.K / 32;
    float4 *red = reinterpret_cast<float4 *>(smem);                                   // [2][kWarps][NT][32]
    uint8_t *ring = smem + 2 * kWarps * NT * 512 + warp * (kStages * kStageBytes);
    uint4 *xs = reinterpret_cast<uint4 *>(smem + kWarps * (2 * NT * 512 + kStages * kStageBytes));  // [block][column][4]
    float *sums = reinterpret_cast<float *>(xs + a.phase * 4 * a.cols * 4);           // MINS: [block][8 NT]
    auto tile_of = [&](int round) { return (round * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x)) * groups + group; };

    // chunk next_c of tile next_tile into a slot; zeros behind the weights' rows and blocks
    const int put_row = lane >> 2, put_part = lane & 3;
    int next_round = 0, next_c = w_in;
    auto issue = [&](int slot) {
        const int tile = tile_of(next_round);
        if (next_round < rounds && tile < a.tiles) {
            const uint32_t dst = smem_u32(ring + slot * kStageBytes);
            const int b = next_c * 4 + put_part;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = put_row + 8 * k, n = tile * 16 + row;
                const bool there = n < a.N && b < blocks;
                const uint8_t *from = a.codes + (there ? static_cast<int64_t>(n) * (a.K / 2) + b * 16 : 0);
                cp16_or_zero(dst + row * 64 + ((put_part ^ ((row >> 1) & 3)) * 16), from, there);
            }
            if (lane < kRecord / 16)
                cp16(dst + kCodeBytes + lane * 16, a.scales + (static_cast<int64_t>(tile) * a.chunks + next_c) * kRecord + lane * 16);
            next_c += W;
            if (next_c >= a.chunks) next_c = w_in, ++next_round;
        }
        cp_commit();
    };
    // The weights are nobody's output (their upload waits for itself), so their copies need not wait for the stream.
#pragma unroll
    for (int j = 0; j < kStages - 1; ++j) issue(j);
    wait_for_stream();

    if (kScaled) {  // the power of two of each row, from its largest finite element
        for (int m = warp; m < a.M; m += kWarps) {
            const TX *x = static_cast<const TX *>(a.x) + m * a.ldx;
            float top = 0.f;
            for (int k = lane * 4; k < a.K; k += 128) {
                float v[4];
                load4(x + k, a.aligned, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[i]) <= kF32Max ? fabsf(v[i]) : 0.f);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = top > 0.f ? min(268 - ((__float_as_int(top) >> 23) & 0xff), 253) : 127;
            if (lane == 0) s_down[m] = __int_as_float(e << 23), s_up[m] = __int_as_float((254 - e) << 23);
        }
        __syncthreads();
    }
    auto stage_x = [&](int c0) {  // chunks c0 ... of x
        const int n_blocks = min(a.phase, a.chunks - c0) * 4, items = n_blocks * a.M * 4;
        for (int id0 = 0; id0 < items; id0 += kThreads) {  // all lanes: four neighbours share a block
            const int id = id0 + threadIdx.x, t = id & 3, m = (id >> 2) % a.M, b = (id >> 2) / a.M;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            if (id < items && c0 * 4 + b < blocks) {
                const TX *x = static_cast<const TX *>(a.x) + m * a.ldx + (c0 * 4 + b) * 32 + 4 * t;
                load4(x, a.aligned, v);
                load4(x + 16, a.aligned, v + 4);
                if (kScaled) {
                    const float by = s_down[m];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] *= by;
                }
            }
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                float h[8], sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float rest;
                    h[i] = f16_of(v[i], rest);
                    v[i] = rest;
                    sum += h[i];
                }
                const int col = m * kParts + part;
                if (id < items)
                    xs[(b * a.cols + col) * 4 + t] = make_uint4(pack_f16(h[0], h[2]), pack_f16(h[4], h[6]), pack_f16(h[1], h[3]), pack_f16(h[5], h[7]));
                if (MINS) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    if (id < items && t == 0) sums[b * 8 * NT + col] = sum;
                }
            }
        }
        if (MINS)  // columns of no row
            for (int id = threadIdx.x; id < n_blocks * 8 * NT; id += kThreads)
                if (id % (8 * NT) >= a.cols) sums[id] = 0.f;
    };

    const uint32_t get0 = ((lane & 7) + (lane >> 3 & 1) * 8) * 64, get_turn = (lane & 7) >> 1, get_part = lane >> 4;
    int slot = 0, slot_in = kStages - 1;
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
        const int tile = tile_of(round);
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll 1
        for (int p0 = 0; p0 < a.chunks; p0 += a.phase) {
            if (round == 0 || a.phase < a.chunks) {
                if (round || p0) __syncthreads();  // the phase before is read
                stage_x(p0);
                __syncthreads();
            }
            if (tile >= a.tiles) continue;
            const int end = min(p0 + a.phase, a.chunks);
#pragma unroll 1
            for (int ch = p0 + w_in; ch < end; ch += W) {
                cp_wait<kStages - 2>();
                __syncwarp();  // the chunk is there for all lanes, and the one before is read by all
                issue(slot_in);
                const uint8_t *st = ring + slot * kStageBytes;
                const uint32_t st_at = smem_u32(st);
                slot_in = slot;
                slot = slot + 1 == kStages ? 0 : slot + 1;
                const uint2 da = *reinterpret_cast<const uint2 *>(st + kCodeBytes + g * 8), db = *reinterpret_cast<const uint2 *>(st + kCodeBytes + g * 8 + 64);
                uint2 ma = make_uint2(0u, 0u), mb = ma;
                if (MINS) {
                    ma = *reinterpret_cast<const uint2 *>(st + kCodeBytes + kScaleBytes + g * 8);
                    mb = *reinterpret_cast<const uint2 *>(st + kCodeBytes + kScaleBytes + g * 8 + 64);
                }
                auto half_of = [](const uint2 &w, int b) {
                    const uint32_t x = b < 2 ? w.x : w.y;
                    return __half2float(__ushort_as_half(static_cast<uint16_t>(b & 1 ? x >> 16 : x)));
                };
                const uint4 *xb = xs + static_cast<int64_t>(ch - p0) * 4 * a.cols * 4;
                uint32_t w[2][4];  // rows g and g + 8, word c of each block
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t r[4];
                    ldmatrix4<false>(r, st_at + get0 + (((2 * k + get_part) ^ get_turn) * 16));
                    w[0][2 * k] = r[0], w[1][2 * k] = r[1], w[0][2 * k + 1] = r[2], w[1][2 * k + 1] = r[3];
                }
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    uint32_t u[4], v[4];
                    codes4(w[0][b], u);
                    codes4(w[1][b], v);
                    const float d0 = half_of(da, b), d1 = half_of(db, b);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint4 y = make_uint4(0u, 0u, 0u, 0u);
                        if (n * 8 + g < a.cols) y = xb[(b * a.cols + n * 8 + g) * 4 + c];
                        float s[4] = {0.f, 0.f, 0.f, 0.f};
                        mma16816(s, u[0], v[0], u[1], v[1], y.x, y.y);
                        mma16816(s, u[2], v[2], u[3], v[3], y.z, y.w);
                        acc[n][0] = fmaf(s[0], d0, acc[n][0]), acc[n][1] = fmaf(s[1], d0, acc[n][1]);
                        acc[n][2] = fmaf(s[2], d1, acc[n][2]), acc[n][3] = fmaf(s[3], d1, acc[n][3]);
                        if (MINS) {
                            const float2 x = *reinterpret_cast<const float2 *>(sums + ((ch - p0) * 4 + b) * 8 * NT + n * 8 + 2 * c);
                            const float m0 = fmaf(8.f, d0, half_of(ma, b)), m1 = fmaf(8.f, d1, half_of(mb, b));
                            acc[n][0] = fmaf(x.x, m0, acc[n][0]), acc[n][1] = fmaf(x.y, m0, acc[n][1]);
                            acc[n][2] = fmaf(x.x, m1, acc[n][2]), acc[n][3] = fmaf(x.y, m1, acc[n][3]);
                        }
                    }
                }
            }
        }
        if (tile >= a.tiles) continue;
        if (W > 1) {
            // Two buffers in turn: a round's is written again behind the barrier of the round between.
            float4 *to = red + ((round & 1) * kWarps + group * W) * NT * 32;
#pragma unroll
            for (int n = 0; n < NT; ++n) to[(w_in * NT + n) * 32 + lane] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
            asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(W * 32) : "memory");
            if (w_in != (round & (W - 1))) continue;  // the warps take turns to finish a tile
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float4 s = to[n * 32 + lane];
                for (int k = 1; k < W; ++k) {
                    const float4 x = to[(k * NT + n) * 32 + lane];
                    s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
                }
                acc[n][0] = s.x, acc[n][1] = s.y, acc[n][2] = s.z, acc[n][3] = s.w;
            }
        }
        auto store = [&](int m, int n, float v) {
            if (m >= a.M || n >= a.N) return;
            if (kScaled) v *= s_up[m];
            if (a.bias) v += a.bias[n];
            const int64_t at = m * a.ldy + n;
            if (a.y_type == SAM3B200_TYPE_F32) static_cast<float *>(a.y)[at] = v;
            else static_cast<TX *>(a.y)[at] = from_f32<TX>(v);
        };
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int out = tile * 16 + g + 8 * r;
                if (kParts == 2) {
                    store(n * 4 + c, out, acc[n][2 * r] + acc[n][2 * r + 1]);
                } else {
                    store(n * 8 + 2 * c, out, acc[n][2 * r]);
                    store(n * 8 + 2 * c + 1, out, acc[n][2 * r + 1]);
                }
            }
    }
    cp_wait<0>();
}

// ggml blocks -> the scales (Q4_1: and minima) of 16 rows by 4 blocks side by side, zeros behind the weights.
__global__ void vec_scales_kernel(const uint8_t *blocks, int N, int nblk, int mins, int chunks, int64_t records, __half *out) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (id >= records * 64) return;
    const int64_t record = id >> 6;
    const int row = (id >> 2) & 15, b = static_cast<int>(record % chunks) * 4 + (id & 3);
    const int64_t n = record / chunks * 16 + row;
    uint16_t d = 0, m = 0;
    if (n < N && b < nblk) {
        const uint8_t *p = blocks + (n * nblk + b) * (mins ? 20 : 18);
        d = static_cast<uint16_t>(p[0] | p[1] << 8);
        if (mins) m = static_cast<uint16_t>(p[2] | p[3] << 8);
    }
    out[record * (mins ? 128 : 64) + (id & 63)] = __ushort_as_half(d);
    if (mins) out[record * 128 + 64 + (id & 63)] = __ushort_as_half(m);
}

template <int NT, bool MINS, typename TX>
cudaError_t launch(Backend *be, VecArgs &a) {
    constexpr int kRecord = MINS ? 2 * kScaleBytes : kScaleBytes;
    const int per_chunk = 4 * (a.cols * 64 + (MINS ? 8 * NT * 4 : 0));
    a.phase = a.chunks * per_chunk <= kXBytes ? a.chunks : std::max(kXBytes / per_chunk / 8, 1) * 8;
    const int smem = kWarps * (2 * NT * 512 + kStages * (kCodeBytes + kRecord)) + a.phase * per_chunk;
    void (*const kernel)(VecArgs) = mul_mat_vec_kernel<NT, MINS, TX>;
    constexpr int kSmemMost = kWarps * (2 * NT * 512 + kStages * (kCodeBytes + kRecord)) + std::max(kXBytes, 8 * 4 * 8 * NT * (64 + 4));
    static_assert(kSmemMost + 1024 <= 227 << 10, "shared memory");
    constexpr unsigned kBit = 1u << (NT + 4 * MINS + 8 * (sizeof(TX) == 4 ? 0 : std::is_same<TX, __half>::value ? 1 : 2));
    if (!(be->vec_ready & kBit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        if (e != cudaSuccess) return e;
        be->vec_ready |= kBit;
    }
    const int resident = std::min(NT == 1 ? 4 : NT == 2 ? 3 : 2, (227 << 10) / (smem + 1024 + 256));
    // warps a tile: the number that gives the fewest steps of a warp, a tile's end counted as one
    int64_t least = 0x7fffffffffffffff;
    const int64_t fit = static_cast<int64_t>(be->num_sms) * resident;
    for (int lg = 0; lg <= 3 && (1 << lg) <= a.chunks; ++lg) {
        const int64_t tiles_round = fit * (kWarps >> lg);
        const int64_t cost = (a.tiles + tiles_round - 1) / tiles_round * ((a.chunks + (1 << lg) - 1) / (1 << lg) + 1);
        if (cost <= least) least = cost, a.w_log2 = lg;
    }
    const int groups = kWarps >> a.w_log2;
    const int64_t grid = std::min<int64_t>(fit, (a.tiles + groups - 1) / groups);
    return launch_after(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem, be->stream, a);
}

}  // namespace

size_t vec_scale_bytes(int type, int N, int K) {
    return static_cast<size_t>((N + 15) / 16) * ((K + 127) / 128) * (type == SAM3B200_TYPE_Q4_1 ? 256 : 128);
}

cudaError_t pack_vec_scales(int type, const void *blocks, int N, int K, void *out, cudaStream_t s) {
    const int chunks = (K + 127) / 128;
    const int64_t records = static_cast<int64_t>((N + 15) / 16) * chunks;
    vec_scales_kernel<<<static_cast<unsigned>((records * 64 + 255) / 256), 256, 0, s>>>(
        static_cast<const uint8_t *>(blocks), N, K / 32, type == SAM3B200_TYPE_Q4_1, chunks, records, static_cast<__half *>(out));
    return cudaGetLastError();
}

}  // namespace b200

using namespace b200;

extern "C" int sam3b200_mul_mat_vec(sam3b200_backend *h, const sam3b200_weight *wh, int x_type, const void *x, int64_t ldx,
                                    int64_t M, const float *bias, int y_type, void *dst, int64_t ldd) {
    auto *be = reinterpret_cast<Backend *>(h);
    auto *w = reinterpret_cast<const Weight *>(wh);
    if (!be || !w || !x || !dst) {
        set_error("mul_mat_vec: null argument");
        return SAM3B200_STATUS_FAILED;
    }
    if (w->type != SAM3B200_TYPE_Q4_0 && w->type != SAM3B200_TYPE_Q4_1) {
        set_error("mul_mat_vec: unsupported weight type %d (Q4_0=2, Q4_1=3)", w->type);
        return SAM3B200_STATUS_FAILED;
    }
    const int xb = type_bytes(x_type), yb = type_bytes(y_type);
    if (!xb || (y_type != x_type && y_type != SAM3B200_TYPE_F32) || reinterpret_cast<uintptr_t>(x) % xb ||
        reinterpret_cast<uintptr_t>(dst) % yb || reinterpret_cast<uintptr_t>(bias) % 4) {
        set_error("mul_mat_vec: unsupported types %d -> %d (x F32=0, F16=1 or BF16=30, dst x's type or F32) or unaligned data", x_type, y_type);
        return SAM3B200_STATUS_FAILED;
    }
    if (M < 0 || M > kMaxRows || ldx < w->K || ldd < w->N) {
        set_error("mul_mat_vec: bad shape: %lld rows (at most %d; mul_mat takes more), ldx %lld (K %d), ldd %lld (N %d)", (long long)M,
                  kMaxRows, (long long)ldx, w->K, (long long)ldd, w->N);
        return SAM3B200_STATUS_FAILED;
    }
    if (M == 0) return SAM3B200_STATUS_SUCCESS;
    VecArgs a;
    a.codes = static_cast<const uint8_t *>(w->codes), a.scales = static_cast<const uint8_t *>(w->vec_scales);
    a.x = x, a.ldx = ldx, a.ldy = ldd, a.bias = bias, a.y = dst;
    a.M = static_cast<int>(M), a.N = w->N, a.K = w->K;
    a.cols = a.M * (x_type == SAM3B200_TYPE_F32 ? 2 : 1);
    a.tiles = (a.N + 15) / 16, a.chunks = (a.K + 127) / 128;
    a.w_log2 = 0, a.phase = a.chunks;
    a.y_type = y_type;
    a.aligned = reinterpret_cast<uintptr_t>(x) % (4 * xb) == 0 && ldx % 4 == 0;
    DeviceScope dev(be->device);
    auto go = [&](auto t) {
        using TX = decltype(t);
        auto with = [&](auto mins) {
            constexpr bool kMins = decltype(mins)::value;
            if (a.cols <= 8) return launch<1, kMins, TX>(be, a);
            if (a.cols <= 16) return launch<2, kMins, TX>(be, a);
            if constexpr (sizeof(TX) == 4) return launch<4, kMins, TX>(be, a);
            else return cudaErrorInvalidValue;
        };
        return w->type == SAM3B200_TYPE_Q4_1 ? with(std::true_type()) : with(std::false_type());
    };
    const cudaError_t e = x_type == SAM3B200_TYPE_F32 ? go(float()) : x_type == SAM3B200_TYPE_F16 ? go(__half()) : go(__nv_bfloat16());
    be->count();
    return cuda_ok(e, "mul_mat_vec launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
