// mul_mat_vec.cu -- MUL_MAT of 1 to 16 rows with Q4_0 / Q4_1 weights, the
// activations as they are.
//
//   y[m][n] = sum over blocks b of d[n][b] (sum_k (code - 8) x[m][k])  + bias[n]         Q4_0
//   y[m][n] = sum over b of d[n][b] (sum_k code x[m][k]) + mn[n][b] (sum_k x[m][k])  + bias[n]  Q4_1
//
// 18 bytes a block of 32 weights (Q4_1: 20) are read once.  A block of 16
// warps an SM keeps x in shared memory; W of its warps share a tile of 16 or 32
// rows of the weights, each with every W-th chunk of 128 k, which it copies by
// cp.async into its own ring of shared memory.  The products run on mma.m16n8k16
// f16 with f32 sums: the codes are its 16-row operand (exact in f16), the rows of
// x its 8 columns, so up to 8 rows cost what one does, and the legacy matrix
// instruction is wide enough for what memory delivers; widening the codes and
// scaling the sums take 162 instructions a warp for 1 KB of codes (64 % of the issue
// slots).  Measured: 49408 x 4096 Q4_0 by one row of f16 25.1 to 27.6
// us (114 MB, 4.5 to 4.1 TB/s, 70 to 63 % of the copy; 25.8 with blocks cut at whole
// tiles; Q4_1 29.8), 14339 x 4096 Q4_1 by
// 6 rows of bf16 15.8 us, of which the launch, the staging of x and the end are
// some 6; by 8, 9 and 16 rows of bf16 13.8 (Q4_0), 19.8 and 33 (Q4_0 27), by 4, 8 and 16 of f32 15.2, 26 and 55.
// ptxas spills 12 to 40 bytes of the kernels for 9 and more columns with 32 weight
// rows a warp, and of those for 17 and more.  Chunks dealt to the warps of a tile in turn, joined tile by tile, took
// 28.7 us in place of 25.8; scales widened once
// a warp through shared memory, for arithmetic on pairs, 26.6 (Q4_1 17 for 15.2).
// Word t of each weight row's block (elements 4t ... and 16 + 4t ...) comes to a
// lane by ldmatrix, a nibble and the one 16 bits above it are one operand
// register after a mask and a subtraction, and x is staged in the same order.  A
// block's sum is scaled in f32, 4 multiply-adds a lane for 16 x 8 results.
// x as f16: F16 as it is; BF16 after a power of two (see kUsual) that keeps all
// but 2^-26 of a row's largest element; F32 the same way as a sum of two f16 numbers
// in two columns (2^-23 of an element at most is lost, too).
// Warps' sums of a tile are added in their order: results repeat bit for bit.
#include <algorithm>
#include <type_traits>

#include "kv4_codes.cuh"
#include "kv_cache.cuh"
#include "mma_sync.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32;
constexpr int kMaxRows = 16;
constexpr int kSmem = 226 << 10;  // of a block, one an SM

struct VecArgs {
    const uint8_t *codes, *scales;
    const void *x;
    int64_t ldx, ldy;
    const float *bias;
    void *y;
    int M, N, K, cols;           // cols: columns of x, M or 2 M
    int sixteens, chunks;        // of weight rows; of 128 columns
    int phase, w_log2;           // chunks of x in shared memory at once: all, or a multiple of the 1 << w_log2 warps of a tile
    int y_type, aligned;         // aligned: four elements of x at once
};

// NT: tiles of 8 columns; RT: tiles of 16 weight rows that a warp has at once.
template <int NT, int RT, bool MINS>
struct Vec {
    static constexpr int kStages = RT == 1 ? 4 : 3;
    static constexpr int kCodeBytes = 16 * 64;  // a chunk of 16 rows: 4 blocks each
    static constexpr int kScaleBytes = 16 * 4 * 2, kRecord = MINS ? 2 * kScaleBytes : kScaleBytes;
    static constexpr int kStageBytes = RT * (kCodeBytes + kRecord);
    static constexpr int kRed = 2 * kWarps * NT * RT * 512;
    static constexpr int kX = kRed + kWarps * kStages * kStageBytes;  // where x begins
};

// Rows whose largest element lies in [2^-5, 2^9) are multiplied by 2^6, so that their largest has at least f16's 1: what f16
// then loses is at most 2^-26 of it, and no look over the row has to come first (6 rows of 4096 in bf16 by 14339 Q4_0 weight
// rows, in a graph: 15.1 us with the look, 13.5 without; Q4_1 17.1 and 15.0; one row 12.4 and 11.2).
constexpr float kUsual = 64.f, kUsualLeast = 0.03125f, kUsualMost = 512.f;

// The bits of v's magnitude, 0 for an infinity or NaN.
__device__ __forceinline__ unsigned finite_bits(float v) {
    const unsigned bits = __float_as_uint(fabsf(v));
    return bits < 0x7f800000u ? bits : 0u;
}

// Four elements as they come.
template <typename T>
struct alignas(4 * sizeof(T)) Raw4 {
    T v[4];
    __device__ __forceinline__ void load(const T *p, bool aligned) {
        if (aligned) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
            else *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = from_f32<T>(0.f);
    }
};

// The largest of them for eight elements.
__device__ __forceinline__ unsigned finite_bits(const Raw4<float> (&raw)[2]) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, finite_bits(raw[i >> 2].v[i & 3]));
    return top;
}
__device__ __forceinline__ unsigned finite_bits(const Raw4<__half> (&)[2]) { return 0; }
__device__ __forceinline__ unsigned finite_bits(const Raw4<__nv_bfloat16> (&raw)[2]) {
    // pairs: magnitude + 0x80 is a positive 16-bit number if it is finite, else a negative one
    uint32_t top = 0x00800080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = (reinterpret_cast<const uint32_t *>(raw[i >> 1].v)[i & 1] & 0x7fff7fffu) + 0x00800080u;
        asm("max.s16x2 %0, %0, %1;" : "+r"(top) : "r"(w));
    }
    return (max(top >> 16, top & 0xffffu) - 0x80u) << 16;
}

// f16 of v; `rest`: what it leaves (0 of an infinity or NaN).
__device__ __forceinline__ float f16_of(float v, float &rest) {
    const float h = __half2float(__float2half_rn(v));
    rest = fabsf(h) <= 65504.f ? v - h : 0.f;
    return h;
}

// The results of rows of x with infinities and NaN for rows n0 ... n1 - 1 of Q4_1 weights: what these elements' products with
// d code + m add up to, infinite or NaN, whatever the finite elements are.  Called by a block.
template <typename TX>
__device__ __noinline__ void odd_rows(const VecArgs &a, int n0, int n1) {
    for (int id = threadIdx.x; id < (n1 - n0) * a.M; id += kThreads) {
        const int m = id / (n1 - n0), n = n0 + id % (n1 - n0);
        const TX *x = static_cast<const TX *>(a.x) + m * a.ldx;
        const uint8_t *codes = a.codes + static_cast<int64_t>(n) * (a.K / 2);
        const __half *scales = reinterpret_cast<const __half *>(a.scales) + static_cast<int64_t>(n >> 4) * a.chunks * 128 + (n & 15) * 4;
        bool any = false;
        float sum = 0.f;
        for (int k = 0; k < a.K; ++k) {
            const float v = to_f32(x[k]);
            if (fabsf(v) <= kF32Max) continue;
            const int b = k >> 5, code = codes[b * 16 + (k & 15)] >> (k & 16 ? 4 : 0) & 15;
            const __half *d = scales + (b >> 2) * 128 + (b & 3);
            sum += fmaf(to_f32(d[0]), static_cast<float>(code), to_f32(d[64])) * v;  // d code is exact, so the sign and 0 are right
            any = true;
        }
        if (!any) continue;
        if (a.bias) sum += a.bias[n];
        if (a.y_type == SAM3B200_TYPE_F32) static_cast<float *>(a.y)[m * a.ldy + n] = sum;
        else static_cast<TX *>(a.y)[m * a.ldy + n] = from_f32<TX>(sum);
    }
}

template <int NT, int RT, bool MINS, typename TX>
__global__ void __launch_bounds__(kThreads, 1) mul_mat_vec_kernel(const __grid_constant__ VecArgs a) {
    using V = Vec<NT, RT, MINS>;
    constexpr int kStages = V::kStages, kStageBytes = V::kStageBytes;
    constexpr int kParts = sizeof(TX) == 4 ? 2 : 1;  // columns of a row
    constexpr bool kScaled = !std::is_same<TX, __half>::value;
    constexpr int kFlight = 4;  // rows of x that a thread has on their way at once (us, 8 rows of 14336: 2 34.9, 3 31, 4 28, 8 30.7)
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_up[kMaxRows], s_down[kMaxRows];
    __shared__ unsigned s_top[kMaxRows];
    __shared__ uint4 zeros[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int blocks = a.K / 32;
    float4 *red = reinterpret_cast<float4 *>(smem);                          // [kWarps][2][RT][NT][32]
    const uint8_t *ring = smem + V::kRed + warp * (kStages * kStageBytes);
    uint4 *xs = reinterpret_cast<uint4 *>(smem + V::kX);                     // [block][column][4]
    float *sums = reinterpret_cast<float *>(xs + a.phase * 4 * a.cols * 4);  // MINS: [block][8 NT]

    // The steps of a warp, each one chunk of one tile.  Where all of x fits, the block has tiles 0 ... t1 - 1 of 16 RT rows, whose
    // chunks in a row are cut into 16 equal parts, so that a warp begins and ends within a tile but needs no other warp before
    // the end.  Else W warps share a tile, chunk by chunk, and the block takes 16 / W tiles after the other through all of x.
    const bool whole = a.phase >= a.chunks;
    const int W = 1 << a.w_log2, w_in = warp & (W - 1), batch = kWarps >> a.w_log2;
    // Blocks are cut at 16 rows, so that a block's last tile may be half of one.
    const int u0 = static_cast<int>(static_cast<int64_t>(blockIdx.x) * a.sixteens / gridDim.x);
    const int u1 = static_cast<int>((static_cast<int64_t>(blockIdx.x) + 1) * a.sixteens / gridDim.x);
    const int row_end = min(u1 * 16, a.N), t1 = (u1 - u0 + RT - 1) / RT;
    const int total = t1 * a.chunks;
    auto part = [&](int w) { return static_cast<int>(static_cast<int64_t>(w) * total / kWarps); };
    const int first_step = part(warp), n_steps = part(warp + 1) - first_step;
    const int first_tile = whole ? first_step / a.chunks : warp >> a.w_log2, first_chunk = whole ? first_step % a.chunks : w_in;

    // The copies of those steps in their order: a lane's rows of codes and its part of the scales; zeros behind the
    // weights' rows and blocks.
    const int put_row = lane >> 2, put_part = lane & 3;
    const uint32_t ring_at = smem_u32(ring);
    const uint32_t put0 = put_row * 64 + ((put_part ^ ((put_row >> 1) & 3)) * 16);  // row + 8: 512 further
    const int64_t eight = static_cast<int64_t>(a.K / 2) * 8;                        // rows, in bytes
    const int stride = whole ? 1 : W, tile_stride = whole ? 1 : batch;
    int left = whole ? n_steps : first_tile < t1 ? ((t1 - first_tile - 1) / batch + 1) * ((a.chunks - w_in + W - 1) >> a.w_log2) : 0;
    int next_tile = first_tile, next_c = first_chunk;
    const uint8_t *from = nullptr, *from_scales = nullptr;
    auto seek = [&] {
        from = a.codes + static_cast<int64_t>((u0 + next_tile * RT) * 16 + put_row) * (a.K / 2) + (next_c * 4 + put_part) * 16;
        from_scales = a.scales + ((u0 + static_cast<int64_t>(next_tile) * RT) * a.chunks + next_c) * V::kRecord + lane * 16;
    };
    seek();
    auto issue = [&](int slot) {
        if (left > 0) {
            const uint32_t dst = ring_at + slot * kStageBytes;
            const int n = (u0 + next_tile * RT) * 16;
            if (n + 16 * RT <= row_end && next_c * 4 + 4 <= blocks) {
#pragma unroll
                for (int k = 0; k < 2 * RT; ++k) cp16(dst + put0 + k * 512, from + k * eight);
            } else {
#pragma unroll
                for (int k = 0; k < 2 * RT; ++k) {
                    const bool there = n + put_row + 8 * k < row_end && next_c * 4 + put_part < blocks;
                    cp16_or_zero(dst + put0 + k * 512, there ? from + k * eight : a.codes, there);
                }
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const uint32_t to = dst + RT * V::kCodeBytes + r * V::kRecord + lane * 16;
                if (lane < V::kRecord / 16) {
                    if (r == 0 || n + 16 * r < row_end) cp16(to, from_scales + static_cast<int64_t>(r) * a.chunks * V::kRecord);
                    else cp16_or_zero(to, a.scales, false);
                }
            }
            --left;
            from += stride * 64, from_scales += stride * V::kRecord;
            next_c += stride;
            if (next_c >= a.chunks) {
                next_tile += tile_stride;
                next_c = whole ? 0 : w_in;
                seek();
            }
        }
        cp_commit();
    };
    // The weights are nobody's output (their upload waits for itself), so their copies need not wait for the stream.
#pragma unroll
    for (int j = 0; j < kStages - 1; ++j) issue(j);
    wait_for_stream();

    // The power of two of each row, from the bits of its largest finite element.
    auto scale_rows = [&] {
        if (threadIdx.x < a.M) {
            const unsigned top = s_top[threadIdx.x];
            const int e = top ? min(268 - static_cast<int>(top >> 23), 253) : 127;
            s_down[threadIdx.x] = __int_as_float(e << 23), s_up[threadIdx.x] = __int_as_float((254 - e) << 23);
        }
        __syncthreads();
    };
    if (kScaled) {
        if (threadIdx.x < kMaxRows) s_top[threadIdx.x] = 0, s_down[threadIdx.x] = kUsual, s_up[threadIdx.x] = 1.f / kUsual;
        __syncthreads();
        if (!whole) {  // x will come in phases, so its largest elements are looked for first
            for (int m0 = 0; m0 < a.M; m0 += kFlight) {
                const TX *x = static_cast<const TX *>(a.x) + m0 * a.ldx;
                unsigned top[kFlight];
#pragma unroll
                for (int m = 0; m < kFlight; ++m) top[m] = 0;
                for (int k = threadIdx.x * 4; k < a.K; k += kThreads * 4) {
                    Raw4<TX> raw[kFlight];
#pragma unroll
                    for (int m = 0; m < kFlight; ++m) {
                        raw[m].zero();
                        if (m0 + m < a.M) raw[m].load(x + m * a.ldx + k, a.aligned);
                    }
#pragma unroll
                    for (int m = 0; m < kFlight; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top[m] = max(top[m], finite_bits(to_f32(raw[m].v[i])));
                }
#pragma unroll
                for (int m = 0; m < kFlight; ++m) {
                    top[m] = __reduce_max_sync(0xffffffffu, top[m]);
                    if (lane == m && m0 + m < a.M) atomicMax(&s_top[m0 + m], top[m]);
                }
            }
            __syncthreads();
            scale_rows();
        }
    }
    if (threadIdx.x < 4) zeros[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    // Chunks c0 ... of x; `look`: the rows' largest elements are noted.
    auto stage_x = [&](int c0, bool look) {
        const int n_blocks = min(a.phase, a.chunks - c0) * 4, items = n_blocks * 4;
        for (int id0 = 0; id0 < items; id0 += kThreads) {  // all lanes: four neighbours share a block
            const int id = id0 + threadIdx.x, t = id & 3, b = id >> 2;
            const bool there = id < items && c0 * 4 + b < blocks;
            for (int m0 = 0; m0 < a.M; m0 += kFlight) {
                const TX *x = static_cast<const TX *>(a.x) + m0 * a.ldx + c0 * 128 + b * 32 + 4 * t;
                Raw4<TX> raw[kFlight][2];
#pragma unroll
                for (int m = 0; m < kFlight; ++m) {
                    raw[m][0].zero();
                    raw[m][1].zero();
                    if (there && m0 + m < a.M) {
                        raw[m][0].load(x + m * a.ldx, a.aligned);
                        raw[m][1].load(x + m * a.ldx + 16, a.aligned);
                    }
                }
#pragma unroll
                for (int m = 0; m < kFlight; ++m) {
                    if (m0 + m >= a.M) break;
                    const float by = kScaled ? s_down[m0 + m] : 1.f;
                    float v[8];
                    if (kScaled && look) {
                        const unsigned top = __reduce_max_sync(0xffffffffu, finite_bits(raw[m]));
                        if (lane == 0) atomicMax(&s_top[m0 + m], top);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = to_f32(raw[m][i >> 2].v[i & 3]) * by;
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
                        const int col = (m0 + m) * kParts + part;
                        if (id < items)
                            xs[(b * a.cols + col) * 4 + t] =
                                make_uint4(pack_f16(h[0], h[2]), pack_f16(h[4], h[6]), pack_f16(h[1], h[3]), pack_f16(h[5], h[7]));
                        if (MINS) {
                            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                            if (id < items && t == 0) sums[b * 8 * NT + col] = sum;
                        }
                    }
                }
            }
        }
        if (MINS)  // columns of no row
            for (int id = threadIdx.x; id < n_blocks * 8 * NT; id += kThreads)
                if (id % (8 * NT) >= a.cols) sums[id] = 0.f;
    };

    const uint32_t get0 = ((lane & 7) + (lane >> 3 & 1) * 8) * 64 + (((lane >> 4) ^ ((lane & 7) >> 1)) * 16);  // blocks 2, 3: ^ 32
    // where this lane's column of x lies, and its step from block to block: columns of no row read zeros
    uint32_t x_at[NT], x_step[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const bool there = n * 8 + g < a.cols;
        x_at[n] = there ? smem_u32(xs) + ((n * 8 + g) * 4 + c) * 16 : smem_u32(zeros) + c * 16;
        x_step[n] = there ? a.cols * 64 : 0;
    }
    int slot = 0, slot_in = kStages - 1;
    float acc[RT][NT][4];
    // Chunks first, first + by, ... below end (counted from the first one in shared memory) of a tile.
    auto run = [&](int first, int end, int by) {
        uint32_t x_now[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) x_now[n] = x_at[n] + first * 4 * x_step[n];
#pragma unroll 1
        for (int ch = first; ch < end; ch += by) {
            cp_wait<kStages - 2>();
            __syncwarp();  // the chunk is there for all lanes, and the one before is read by all
            issue(slot_in);
            const uint8_t *st = ring + slot * kStageBytes;
            const uint32_t st_at = ring_at + slot * kStageBytes;
            slot_in = slot;
            slot = slot + 1 == kStages ? 0 : slot + 1;
            __half2 d[RT][2][2], mn[RT][2][2];  // rows g and g + 8, blocks 0, 1 and 2, 3
            uint32_t w[RT][2][4];               // rows g and g + 8, word c of each block
#pragma unroll
            for (int r = 0; r < RT; ++r) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *at = st + RT * V::kCodeBytes + r * V::kRecord + (g + 8 * h) * 8;
                    *reinterpret_cast<uint2 *>(d[r][h]) = *reinterpret_cast<const uint2 *>(at);
                    if (MINS) *reinterpret_cast<uint2 *>(mn[r][h]) = *reinterpret_cast<const uint2 *>(at + V::kScaleBytes);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t z[4];
                    ldmatrix4<false>(z, st_at + r * V::kCodeBytes + (get0 ^ (32 * k)));
                    w[r][0][2 * k] = z[0], w[r][1][2 * k] = z[1], w[r][0][2 * k + 1] = z[2], w[r][1][2 * k + 1] = z[3];
                }
            }
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint4 y[NT];
                float2 x[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    y[n] = lds128(x_now[n]);
                    x_now[n] += x_step[n];
                    if (MINS) x[n] = *reinterpret_cast<const float2 *>(sums + (ch * 4 + b) * 8 * NT + n * 8 + 2 * c);
                }
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    uint32_t u[4], v[4];
                    codes4<MINS ? 0 : 8>(w[r][0][b], u);
                    codes4<MINS ? 0 : 8>(w[r][1][b], v);
                    float ds[2], ms[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        ds[h] = b & 1 ? __high2float(d[r][h][b >> 1]) : __low2float(d[r][h][b >> 1]);
                        if (MINS) ms[h] = b & 1 ? __high2float(mn[r][h][b >> 1]) : __low2float(mn[r][h][b >> 1]);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float s[4];
                        mma16816_first(s, u[0], v[0], u[1], v[1], y[n].x, y[n].y);
                        mma16816(s, u[2], v[2], u[3], v[3], y[n].z, y[n].w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            acc[r][n][i] = fmaf(s[i], ds[i >> 1], acc[r][n][i]);
                            if (MINS) acc[r][n][i] = fmaf(i & 1 ? x[n].y : x[n].x, ms[i >> 1], acc[r][n][i]);
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) x_now[n] += (by - 1) * 4 * x_step[n];
        }
    };
    auto clear = [&] {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[r][n][0] = acc[r][n][1] = acc[r][n][2] = acc[r][n][3] = 0.f;
    };
    auto place = [&](int w, int k) { return red + (w * 2 + k) * RT * NT * 32 + lane; };  // warp w's sums, k: of its first tile or its last
    auto put = [&](float4 *to) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n) to[(r * NT + n) * 32] = make_float4(acc[r][n][0], acc[r][n][1], acc[r][n][2], acc[r][n][3]);
    };
    auto add = [&](const float4 *x) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float4 v = x[(r * NT + n) * 32];
                acc[r][n][0] += v.x, acc[r][n][1] += v.y, acc[r][n][2] += v.z, acc[r][n][3] += v.w;
            }
    };
    bool odd = false;  // this thread has a result that is no finite number
    auto store = [&](int m, int n, float v) {
        if (m >= a.M || n >= row_end) return;
        if (kScaled) v *= s_up[m];
        if (MINS) odd = odd || !(fabsf(v) <= kF32Max);
        if (a.bias) v += a.bias[n];
        const int64_t at = m * a.ldy + n;
        if (a.y_type == SAM3B200_TYPE_F32) static_cast<float *>(a.y)[at] = v;
        else static_cast<TX *>(a.y)[at] = from_f32<TX>(v);
    };
    auto finish = [&](int tile) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int out = (u0 + tile * RT + r) * 16 + g + 8 * h;
                    if (kParts == 2) {
                        store(n * 4 + c, out, acc[r][n][2 * h] + acc[r][n][2 * h + 1]);
                    } else {
                        store(n * 8 + 2 * c, out, acc[r][n][2 * h]);
                        store(n * 8 + 2 * c + 1, out, acc[r][n][2 * h + 1]);
                    }
                }
    };

    if (whole) {
        for (bool look = kScaled;; look = false) {  // (one place, so that the code stays small)
            stage_x(0, look);
            __syncthreads();
            if (!look) break;
            bool usual = true;
            for (int m = 0; m < a.M; ++m) usual = usual && s_top[m] < __float_as_uint(kUsualMost) && (s_top[m] >= __float_as_uint(kUsualLeast) || s_top[m] == 0);
            if (usual) break;
            scale_rows();  // rows of another size than usual get a power of two of their own
        }
        int tile = first_tile, ch = first_chunk;
        for (int steps = n_steps; steps > 0; ++tile, ch = 0) {
            const int end = min(ch + steps, a.chunks);
            clear();
            run(ch, end, 1);
            steps -= end - ch;
            if (end - ch == a.chunks) finish(tile);
            else put(place(warp, tile != first_tile));
        }
        __syncthreads();
        for (tile = warp; tile < t1; tile += kWarps) {  // tiles that several warps have parts of
            const int64_t begin = static_cast<int64_t>(tile) * a.chunks;
            const int w0 = static_cast<int>(((begin + 1) * kWarps - 1) / total), w1 = static_cast<int>(((begin + a.chunks) * kWarps - 1) / total);
            if (w0 == w1) continue;
            clear();
            for (int w = w0; w <= w1; ++w)
                if (part(w + 1) > part(w)) add(place(w, tile != part(w) / a.chunks));
            finish(tile);
        }
    } else {
        for (int tile0 = 0; tile0 < t1; tile0 += batch) {
            const int tile = tile0 + (warp >> a.w_log2);
            clear();
            for (int p0 = 0; p0 < a.chunks; p0 += a.phase) {
                if (tile0 || p0) __syncthreads();  // the phase before is read
                stage_x(p0, false);
                __syncthreads();
                if (tile < t1) run(w_in, min(a.phase, a.chunks - p0), W);
            }
            if (W > 1) {
                if (w_in && tile < t1) put(place(warp, 0));
                __syncthreads();
                if (w_in == 0 && tile < t1)
                    for (int w = warp + 1; w < warp + W; ++w) add(place(w, 0));
            }
            if (w_in == 0 && tile < t1) finish(tile);
        }
    }
    cp_wait<0>();
    // An infinity or NaN in a row of x makes all its results infinite or NaN (and no other row's), but d (sum code x) +
    // m (sum x) not those of (d code + m) x: a code of 0 makes NaN of an infinity, and so do unlike signs of d code and m.  So
    // the results are looked at (6 rows by 14339 x 4096 15.75 us for 15.55; a look at x as it is staged: 16.5).
    if (MINS && __syncthreads_or(odd)) odd_rows<TX>(a, u0 * 16, row_end);
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

template <int NT, int RT, bool MINS, typename TX>
cudaError_t launch(Backend *be, VecArgs &a) {
    using V = Vec<NT, RT, MINS>;
    const int tiles = (a.sixteens + RT - 1) / RT;
    const int per_chunk = 4 * (a.cols * 64 + (MINS ? 8 * NT * 4 : 0));
    static_assert((kSmem - V::kX) / (4 * 8 * NT * (64 + (MINS ? 4 : 0))) >= 8, "phases of several chunks");
    const int most = (kSmem - V::kX) / per_chunk;
    const bool phases = a.chunks > most;
    void (*const kernel)(VecArgs) = mul_mat_vec_kernel<NT, RT, MINS, TX>;
    constexpr unsigned kBit = 1u << (((NT == 4 ? 4 : 2 * (NT - 1) + RT - 1) + 5 * MINS) + 10 * (sizeof(TX) == 4 ? 0 : std::is_same<TX, __half>::value ? 1 : 2));
    if (!(be->vec_ready & kBit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
        if (e != cudaSuccess) return e;
        be->vec_ready |= kBit;
    }
    a.w_log2 = 0, a.phase = a.chunks;
    if (phases) {
        // warps a tile: the number that gives the fewest steps of a warp, with x that comes again for every batch of tiles by
        // its instructions
        int64_t least = 0x7fffffffffffffff;
        const int64_t own = ((a.sixteens + be->num_sms - 1) / be->num_sms + RT - 1) / RT;  // tiles of a block
        for (int lg = 0; lg <= 4 && (1 << lg) <= most; ++lg) {
            const int64_t batches = (own * (1 << lg) + kWarps - 1) / kWarps;
            const int64_t cost = batches * ((a.chunks + (1 << lg) - 1) / (1 << lg) + 1 + a.chunks * static_cast<int64_t>(a.cols) / 64);
            if (cost <= least) least = cost, a.w_log2 = lg;
        }
        a.phase = most >> a.w_log2 << a.w_log2;
    }
    const int smem = V::kX + a.phase * per_chunk;
    const int grid = std::min(be->num_sms, tiles);
    return launch_after(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem, be->stream, a);
}

// Tiles of 16 or of 32 rows, where x is read from shared memory once for both halves: by the steps of a warp, one of 32
// counted as 1.8 of 16.  Us for tiles of 16 and of 32, 4096 columns: 49408 weight rows and one of x 27.8 and 25.8; 14339 rows
// of Q4_1 and 6 of x 17.4 and 18.1; 1024 columns by 4096 and one row 6.2 and 6.6.
template <int NT, bool MINS, typename TX>
cudaError_t launch(Backend *be, VecArgs &a) {
    if constexpr (NT < 4) {
        auto steps = [&](int64_t rt) {
            const int64_t tiles = ((a.sixteens + be->num_sms - 1) / be->num_sms + rt - 1) / rt;  // of a block
            return (tiles * a.chunks + kWarps - 1) / kWarps;
        };
        if (18 * steps(2) <= 10 * steps(1)) return launch<NT, 2, MINS, TX>(be, a);
    }
    return launch<NT, 1, MINS, TX>(be, a);
}

// `rows` runs of `bytes`, `step` bytes from one to the next.
struct Runs {
    uintptr_t at;
    int64_t rows, step, bytes;
};
bool overlap(const Runs &a, const Runs &b) {
    auto apart = [](uintptr_t x, int64_t nx, uintptr_t y, int64_t ny) { return x + nx <= y || y + ny <= x; };
    if (apart(a.at, (a.rows - 1) * a.step + a.bytes, b.at, (b.rows - 1) * b.step + b.bytes)) return false;
    for (int64_t i = 0; i < a.rows; ++i)
        for (int64_t j = 0; j < b.rows; ++j)
            if (!apart(a.at + i * a.step, a.bytes, b.at + j * b.step, b.bytes)) return true;
    return false;
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
    // every block reads all of x, at times when others store
    const Runs out{reinterpret_cast<uintptr_t>(dst), M, ldd * yb, static_cast<int64_t>(w->N) * yb};
    if (overlap(out, {reinterpret_cast<uintptr_t>(x), M, ldx * xb, static_cast<int64_t>(w->K) * xb}) ||
        (bias && overlap(out, {reinterpret_cast<uintptr_t>(bias), 1, 0, static_cast<int64_t>(w->N) * 4}))) {
        set_error("mul_mat_vec: dst overlaps x or bias");
        return SAM3B200_STATUS_FAILED;
    }
    VecArgs a;
    a.codes = static_cast<const uint8_t *>(w->codes), a.scales = static_cast<const uint8_t *>(w->vec_scales);
    a.x = x, a.ldx = ldx, a.ldy = ldd, a.bias = bias, a.y = dst;
    a.M = static_cast<int>(M), a.N = w->N, a.K = w->K;
    a.cols = a.M * (x_type == SAM3B200_TYPE_F32 ? 2 : 1);
    a.sixteens = (a.N + 15) / 16, a.chunks = (a.K + 127) / 128;
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
