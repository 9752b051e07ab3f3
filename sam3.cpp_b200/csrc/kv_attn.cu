// kv_attn.cu -- attention over the paged 8-bit cache: the entry points, and
// the kernel for few query rows a kv head.
//
//   y = softmax(scale q K^T + mask) V,   K = ks ck, V = vs cv a page
//
// Products with the codes are exact in f16 (|code| <= 127), so the scales
// stay outside the matrix products.  With t = s ks scale log2(e) + log2(vs)
// for a raw score s, and m the running maximum of t,
//   p = 2^(t - m),   O = sum p cv,   l = sum p / vs,   y = O / l:
// a page's value scale moves into the exponent, p stays in [0, 1] for f16
// whatever the scales are, and no other step sees them.
//
// kv_attn_few: one block of 4 warps per (8 or 16 query rows of a kv head,
// part of the key range).  The rows are the query heads of the group, times
// the sequence's new tokens.  Each warp takes every fourth block of 16 tokens
// (never across a page), copies it by cp.async into its own ring of shared
// memory, and multiplies by mma.m16n8k16 f16 with f32 sums: bound by memory
// (1 byte per code), the legacy matrix instruction is wide enough.  The codes
// are its 16-row operand and the queries its 8 columns: S^T = K Q^T, then
// O^T = V^T P^T, so one token a sequence and up to 8 query heads a kv head
// fill an instruction.  Dimensions are permuted in both products so that a
// lane reads 16 codes of a token at once, and P^T goes from the first
// product's layout to the second's by movmatrix.  The warps' partial results
// are joined through shared memory, the parts' through the workspace by the
// last block to finish.
//
// Measured (32 heads on 8 of 128): 64 sequences of 500 to 8100 tokens 105
// to 115 us, 5 to 4.6 TB/s; 8 heads without groups over 100 and 131 thousand
// tokens 91 to 96 us, 5.2 to 4.9 TB/s; one token over 700 7.8 us, of which 0.8
// find the sequence, 1.5 the pages and queries, 0.5 the part, 3 its join.  No unit is
// full (DRAM 60 to 64 %, issue 45 %): 16 warps an SM wait on their own chains.
// With the queries as the 16-row operand (8 of 16 rows idle, twice the
// registers and softmax work) the first took 138 us and the second 111.
#include <algorithm>
#include <cmath>
#include <new>

#include "kv_attn.cuh"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxSplits = 256;  // most parts of a key range

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// d += a b: a 16 x 16 (rows), b 16 x 8, f16 in, f32 sums.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// An 8 x 8 matrix of f16, a row's pair of columns a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Bytes i and j of w (codes + 128) as f16: 0x64uu is 1024 + u, exactly.
template <int SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
    const uint32_t h = __byte_perm(w, 0x64646464u, SEL);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Four consecutive query elements (d a multiple of 4), as they come, and the j-th of them.
__device__ __forceinline__ uint2 load_q4(const KvAttnArgs &a, int64_t at) {
    const uint16_t *p = static_cast<const uint16_t *>(a.q) + at;
    if (a.qs.aligned16) return *reinterpret_cast<const uint2 *>(p);
    return make_uint2(p[0] | static_cast<uint32_t>(p[1]) << 16, p[2] | static_cast<uint32_t>(p[3]) << 16);
}
__device__ __forceinline__ float q_value(const KvAttnArgs &a, const uint2 &x, int j) {
    const uint32_t w = j < 2 ? x.x : x.y;
    if (a.q_bf16) return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(j & 1 ? w >> 16 : w)));
}

// NT tiles of 8 query rows.
template <int D, int NT>
struct Few {
    static constexpr int kRows = 8 * NT;
    static constexpr int kStages = NT == 1 ? 3 : 4, kBlocks = NT == 1 ? 4 : 3;  // stages of a warp, blocks an SM
    static constexpr int kBlockBytes = 16 * D;                       // codes of 16 tokens
    static constexpr int kStageBytes = 2 * kBlockBytes + 16;         // keys, values, their two scales
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kLane = D / 8;                              // output dimensions of a lane
    static constexpr int kRowFloats = D + 36;                        // a joined row, padded against bank conflicts
    static constexpr int kJoin = kWarps * kRows * kRowFloats * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    static_assert(kSmem >= kWarps * kRows * (D + 2) * 4, "shares of the parts");
    static constexpr int kEach = D * kRows / 128 > 8 ? D * kRows / 128 : 8;  // dimensions of a thread that joins
    // Byte of 16-byte chunk c of token t within a staged block.  The permutation keeps the reads free of bank
    // conflicts: keys (8 lanes: 2 neighbouring tokens, 4 chunks), values (8 lanes: 4 token pairs, 2 chunks).  Where
    // a lane's tokens or chunks differ by a constant the byte differs by a sum or by ^ 64, which the loops below use.
    static __device__ __forceinline__ uint32_t at(int t, int c) {
        if (D == 128) return t * 128 + (c ^ (t & 6) ^ ((t & 1) << 2)) * 16;
        return (t >> 1) * 128 + ((((t & 1) << 2) | c) ^ (t & 6)) * 16;
    }
    static __device__ __forceinline__ int padded(int d) { return d + d / kLane * 4; }
};

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, (Few<D, NT>::kBlocks)) kv_attn_few_kernel(const __grid_constant__ KvAttnArgs a) {
    using F = Few<D, NT>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_m[kWarps][F::kRows], s_l[kWarps][F::kRows];
    __shared__ int s_last;
    wait_for_stream();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int kv = blockIdx.y, G = a.group;
    const unsigned unit = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, false, a.err);
    int64_t local;
    KvSeq q;
    if (!kv_find(a.b, unit, G, NT == 1 ? 3 : 4, 1, a.c.page_log2, q, local)) return;
    const int R = q.n * G;  // the host keeps n_rows * G below 2^31
    if (local * F::kRows >= R) return;
    const int row0 = static_cast<int>(local) * F::kRows, i_lo = row0 / G, i_hi = (min(row0 + F::kRows, R) - 1) / G;

    // the tile's keys, and this block's part of them
    const int k_end = kv_last(a, q, i_hi) + 1, k_begin = kv_first(a, kv_last(a, q, i_lo)) & ~15;
    const int range = max(k_end - k_begin, 0);
    const int chunk = max(range < a.short_range ? a.chunk_short : a.chunk, ((range + a.splits - 1) / a.splits + 63) & ~63);
    const int n_split = max((range + chunk - 1) / chunk, 1);
    if (split >= n_split) return;
    const int t_begin = k_begin + split * chunk, t_end = min(t_begin + chunk, k_end);
    const int n_blocks = t_end > t_begin ? (t_end - t_begin + 15) / 16 : 0;
    const int mine = n_blocks > warp ? (n_blocks - warp + kWarps - 1) / kWarps : 0;  // blocks warp, warp + 4, ...

    // the queries are on their way while the first pages are looked up
    const int rest0 = row0 - i_lo * G;  // row 0 of the tile: token i_lo, head rest0 of the group
    uint2 qraw[NT][D / 16];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int x = rest0 + 8 * n + g, i = i_lo + x / G;
        const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.qs.token + (static_cast<int64_t>(kv) * G + x % G) * a.qs.head;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qraw[n][k] = make_uint2(0u, 0u);
            if (row0 + 8 * n + g < R) qraw[n][k] = load_q4(a, at + (k >> 2) * 64 + c * 16 + (k & 3) * 4);
        }
    }

    uint8_t *ring = smem + warp * F::kStages * F::kStageBytes;
    // this lane's bytes within a stage: the copy of chunk lane (of 32 a step), keys of token g, values of token 2 c
    const uint32_t put0 = F::at(lane / (D / 16), lane % (D / 16)), key0 = F::at(g, c);
    const uint32_t val0 = D == 128 ? F::at(2 * c, g) : F::at(2 * c, g >> 1) + (g & 1) * 8;
    int page_now = 0, page_next = 0;  // lane j: the page of block 32 b + j of this warp, for batches b and b + 1
    auto load_page = [&](int j) -> int {
        if (j >= mine) return 0;
        const int p = kv_page(a.c, a.b, q.s, (t_begin + (j * kWarps + warp) * 16) >> a.c.page_log2, a.err);
        return max(p, 0);
    };
    page_next = load_page(lane);
    auto issue = [&](int j, int slot) {  // block j of this warp into a slot
        if (j < mine) {
            if ((j & 31) == 0) {
                page_now = page_next;
                page_next = load_page(j + 32 + lane);
            }
            const int page = __shfl_sync(0xffffffffu, page_now, j & 31);
            const int tok = t_begin + (j * kWarps + warp) * 16;
            const int64_t at = kv_slab(a.c, page, kv) + static_cast<int64_t>(tok & ((1 << a.c.page_log2) - 1)) * D + lane * 16;
            const uint32_t dst = smem_u32(ring + slot * F::kStageBytes);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < F::kBlockBytes / 512; ++k) {
                    // a step of 4 (D = 128) or 8 tokens
                    const uint32_t to = (D == 128 && (k & 1) ? put0 ^ 64 : put0) + k * 512;
                    cp16(dst + w * F::kBlockBytes + to, a.c.codes[w] + at + k * 512);
                }
            if (lane < 2) cp4(dst + 2 * F::kBlockBytes + lane * 4, a.c.scale[lane] + static_cast<int64_t>(page) * a.c.heads + kv);
        }
        cp_commit();
    };
#pragma unroll
    for (int j = 0; j < F::kStages - 1; ++j) issue(j, j);

    // queries: row 8 n + g, for each 16-wide step the 4 dimensions that go with this lane's codes
    uint32_t qf[NT][D / 16][2];
    float row_c[NT][2];  // for rows 8 n + 2 c, + 1: scale log2(e), and what the power of two below took
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(q_value(a, qraw[n][k], j)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // bf16 rows are brought to [1, 2) by a power of two, which f16 then holds to 2^-25 of the largest
        const int e = a.q_bf16 ? min((__float_as_int(top) >> 23) & 0xff, 253) : 0;
        const float down = e ? __int_as_float((254 - e) << 23) : 1.f, up = a.scale_log2 * (e ? __int_as_float(e << 23) : 1.f);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                qf[n][k][j] = pack_f16(q_value(a, qraw[n][k], 2 * j) * down, q_value(a, qraw[n][k], 2 * j + 1) * down);
#pragma unroll
        for (int j = 0; j < 2; ++j) row_c[n][j] = __shfl_sync(0xffffffffu, up, (2 * c + j) * 4);
    }
    // tokens that some row of the tile does not see
    const int seen_by_all = kv_last(a, q, i_lo), window_end = kv_first(a, kv_last(a, q, i_hi));

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    int slot = 0, slot_in = F::kStages - 1;
    for (int j = 0; j < mine; ++j) {
        cp_wait<F::kStages - 2>();
        __syncwarp();  // block j is there for all lanes, and block j - 1 is read by all
        issue(j + F::kStages - 1, slot_in);
        const uint8_t *st = ring + slot * F::kStageBytes;
        slot_in = slot;
        slot = slot + 1 == F::kStages ? 0 : slot + 1;

        // scores of tokens g (t[n][0], [1]) and g + 8 ([2], [3]) for rows 8 n + 2 c, + 1
        float t[NT][4], t2[NT][4];  // in two chains
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) t[n][k] = t2[n][k] = 0.f;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
            const uint4 lo = *reinterpret_cast<const uint4 *>(st + (h ? key0 ^ 64 : key0));
            const uint4 hi = *reinterpret_cast<const uint4 *>(st + (h ? key0 ^ 64 : key0) + 8 * D);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = (k == 0 ? lo.x : k == 1 ? lo.y : k == 2 ? lo.z : lo.w) ^ 0x80808080u;
                const uint32_t v = (k == 0 ? hi.x : k == 1 ? hi.y : k == 2 ? hi.z : hi.w) ^ 0x80808080u;
                const uint32_t a0 = codes2<0x4140>(u), a1 = codes2<0x4140>(v), a2 = codes2<0x4342>(u), a3 = codes2<0x4342>(v);
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816(k & 1 ? t2[n] : t[n], a0, a1, a2, a3, qf[n][4 * h + k][0], qf[n][4 * h + k][1]);
            }
        }
        const float2 ksvs = *reinterpret_cast<const float2 *>(st + 2 * F::kBlockBytes);
        const float lv = ksvs.y > 0.f ? __log2f(ksvs.y) : kZeroScaleLog2, inv_vs = ex2_approx(-lv);
        const int tok = t_begin + (j * kWarps + warp) * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) t[n][k] = fmaf(t[n][k] + t2[n][k], row_c[n][k & 1] * ksvs.x, lv);
        if (tok + 15 > seen_by_all || tok < window_end) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int last = kv_last(a, q, i_lo + (rest0 + 8 * n + 2 * c + k) / G), first = kv_first(a, last);
                    if (tok + g > last || tok + g < first) t[n][k] = -INFINITY;
                    if (tok + g + 8 > last || tok + g + 8 < first) t[n][k + 2] = -INFINITY;
                }
        }
        bool rise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) rise |= fmaxf(t[n][k], t[n][k + 2]) > m[n][k] + kLazy;
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float top = fmaxf(t[n][k], t[n][k + 2]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float to = fmaxf(m[n][k], top);
                    const float alpha = m[n][k] == to ? 1.f : ex2_approx(m[n][k] - to);
                    m[n][k] = to;
                    l[n][k] *= alpha;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) o[n][i][k] *= alpha, o[n][i][k + 2] *= alpha;
                }
        }
        uint32_t p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float less = m[n][k] == -INFINITY ? 0.f : m[n][k] - kPUp;
                t[n][k] = ex2_approx(t[n][k] - less);
                t[n][k + 2] = ex2_approx(t[n][k + 2] - less);
                l[n][k] = fmaf(t[n][k] + t[n][k + 2], inv_vs, l[n][k]);
            }
            p[n][0] = transposed(pack_f16(t[n][0], t[n][1]));
            p[n][1] = transposed(pack_f16(t[n][2], t[n][3]));
        }

        // values: lane g holds dimensions D / 8 * g ... of tokens 2c, 2c + 1, 8 + 2c, 9 + 2c
        uint32_t w[4][D / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            // the odd token: its own row (D = 128), or the other half of the pair's
            const uint8_t *from = st + F::kBlockBytes + (r & 1 ? (val0 ^ 64) + (D == 128 ? 128 : 0) : val0) + (r >> 1) * 8 * D;
            if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4 *>(from);
                w[r][0] = x.x, w[r][1] = x.y, w[r][2] = x.z, w[r][3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2 *>(from);
                w[r][0] = x.x, w[r][1] = x.y;
            }
        }
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            uint32_t lo[2], hi[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {  // bytes of two tokens side by side
                lo[r] = __byte_perm(w[2 * r][k], w[2 * r + 1][k], 0x5140) ^ 0x80808080u;
                hi[r] = __byte_perm(w[2 * r][k], w[2 * r + 1][k], 0x7362) ^ 0x80808080u;
            }
            // dimensions D / 8 * g + 4 k, + 1 are rows g, g + 8 of one product, + 2, + 3 of the next
            const uint32_t x0 = codes2<0x4140>(lo[0]), x1 = codes2<0x4342>(lo[0]), x2 = codes2<0x4140>(lo[1]), x3 = codes2<0x4342>(lo[1]);
            const uint32_t y0 = codes2<0x4140>(hi[0]), y1 = codes2<0x4342>(hi[0]), y2 = codes2<0x4140>(hi[1]), y3 = codes2<0x4342>(hi[1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma16816(o[n][2 * k], x0, x1, x2, x3, p[n][0], p[n][1]);
                mma16816(o[n][2 * k + 1], y0, y1, y2, y3, p[n][0], p[n][1]);
            }
        }
    }
    cp_wait<0>();
    __syncthreads();  // every warp is done with its ring

    // join the warps
    float *rows = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int row = 8 * n + 2 * c + k;
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], x);
            if (g == 0) s_m[warp][row] = m[n][k], s_l[warp][row] = l[n][k];
            float *to = rows + (warp * F::kRows + row) * F::kRowFloats + F::padded(g * F::kLane);
#pragma unroll
            for (int i = 0; i < D / 16; i += 2)
                *reinterpret_cast<float4 *>(to + 2 * i) = make_float4(o[n][i][k], o[n][i][k + 2], o[n][i + 1][k], o[n][i + 1][k + 2]);
        }
    __syncthreads();
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
            for (int i = 0; i < kEach; ++i) sum[i] = fmaf(from[F::padded(d0 + i)], f, sum[i]);
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

template <int D, int NT>
cudaError_t launch_few(KvAttnArgs &a, int num_sms, cudaStream_t st) {
    using F = Few<D, NT>;
    const int64_t units = ((static_cast<int64_t>(a.b.n_rows) * a.group) >> (NT == 1 ? 3 : 4)) + a.b.n_seqs;
    // parts for two waves where there are few sequences and heads, for four where the lengths of many have to even out
    const int64_t wave = F::kBlocks * static_cast<int64_t>(num_sms), groups = units * a.c.heads;
    const int64_t span =
        std::max(a.window ? std::min(a.b.max_len, static_cast<int64_t>(a.window) + a.b.max_rows + 16) : a.b.max_len, int64_t(1));
    int64_t splits = 2 * groups < wave ? (2 * wave + groups - 1) / groups : (4 * wave + groups - 1) / groups;
    // a block's least part: 64 tokens, one turn of its warps, while the blocks fit in one wave, else 256
    const int64_t least = groups * ((span + 63) / 64) <= wave ? 64 : 256;
    splits = std::min(splits, (span + least - 1) / least);
    splits = std::min(splits, std::min(static_cast<int64_t>(kMaxParts) / groups, static_cast<int64_t>(kMaxSplits)));
    splits = std::max(splits, static_cast<int64_t>(1));
    if (units * splits > 0x7fffffff) return cudaErrorInvalidValue;
    a.splits = static_cast<int>(splits);
    a.chunk = static_cast<int>(((span + splits - 1) / splits + 63) & ~int64_t(63));
    // With few sequences one that is far shorter than max_len (a captured step's bound) is cut finer, into all parts.
    a.chunk_short = static_cast<int>(2 * groups < wave ? std::min<int64_t>(least, a.chunk) : a.chunk);
    a.short_range = static_cast<int>(span / 2);
    if (!(*a.ready & (1 << (2 * NT + (D == 64))))) {
        const cudaError_t e = cudaFuncSetAttribute(kv_attn_few_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        if (e != cudaSuccess) return e;
        *a.ready |= 1 << (2 * NT + (D == 64));
    }
    const dim3 grid(static_cast<unsigned>(units * a.splits), a.c.heads);
    return launch_after(kv_attn_few_kernel<D, NT>, grid, kWarps * 32, F::kSmem, st, a);
}

struct KvAttention {
    Backend *be = nullptr;
    unsigned ready = 0;  // kernels whose attributes are set on this handle's device
    float *part = nullptr;
    unsigned *done = nullptr;
};

}  // namespace

cudaError_t kv_attn_few(KvAttnArgs a, int num_sms, cudaStream_t st) {
    const bool one = static_cast<int64_t>(a.b.max_rows) * a.group <= 8;
    if (a.c.D == 64) return one ? launch_few<64, 1>(a, num_sms, st) : launch_few<64, 2>(a, num_sms, st);
    return one ? launch_few<128, 1>(a, num_sms, st) : launch_few<128, 2>(a, num_sms, st);
}

}  // namespace b200

using namespace b200;

extern "C" sam3b200_kv_attention *sam3b200_kv_attention_create(sam3b200_backend *h) {
    auto *be = reinterpret_cast<Backend *>(h);
    if (!be) {
        set_error("kv_attention_create: null backend");
        return nullptr;
    }
    auto *k = new (std::nothrow) KvAttention();
    if (!k) {
        set_error("kv_attention_create: out of host memory");
        return nullptr;
    }
    k->be = be;
    DeviceScope dev(be->device);
    if (!cuda_ok(cudaMalloc(&k->part, kPartFloats * sizeof(float)), "cudaMalloc(attention workspace)") ||
        !cuda_ok(cudaMalloc(&k->done, kMaxParts * sizeof(unsigned)), "cudaMalloc(attention counters)") ||
        !cuda_ok(cudaMemsetAsync(k->done, 0, kMaxParts * sizeof(unsigned), be->stream), "memset(attention counters)") ||
        !cuda_ok(cudaStreamSynchronize(be->stream), "kv_attention_create sync")) {
        cudaFree(k->part);
        cudaFree(k->done);
        delete k;
        return nullptr;
    }
    return reinterpret_cast<sam3b200_kv_attention *>(k);
}

extern "C" void sam3b200_kv_attention_free(sam3b200_kv_attention *h) {
    auto *k = reinterpret_cast<KvAttention *>(h);
    if (!k) return;
    DeviceScope dev(k->be->device);
    cudaStreamSynchronize(k->be->stream);
    cudaFree(k->part);
    cudaFree(k->done);
    delete k;
}

extern "C" int sam3b200_kv_attention_run(sam3b200_kv_attention *h, const sam3b200_kv_cache *cache,
                                         const sam3b200_kv_batch *batch, int type, const void *q, const int64_t *q_nb,
                                         int64_t n_heads, float scale, int causal, int64_t window, int y_type, void *y,
                                         const int64_t *y_nb) {
    auto *k = reinterpret_cast<KvAttention *>(h);
    KvAttnArgs a;
    if (!kv_views("kv_attention", cache, batch, a.c, a.b)) return SAM3B200_STATUS_FAILED;
    if (!q || !y) {
        set_error("kv_attention: null argument");
        return SAM3B200_STATUS_FAILED;
    }
    const int yb = type_bytes(y_type);
    if ((type != SAM3B200_TYPE_F16 && type != SAM3B200_TYPE_BF16) || (y_type != type && y_type != SAM3B200_TYPE_F32) ||
        reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(y) % yb) {
        set_error("kv_attention: unsupported types %d -> %d (q F16=1 or BF16=30, y q's type or F32=0) or unaligned data", type,
                  y_type);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_heads >= 1 && a.b.n_rows * (n_heads / a.c.heads) > 0x7fffff00) {
        set_error("kv_attention: %d rows of %lld query heads over %d kv heads are too many", a.b.n_rows, (long long)n_heads, a.c.heads);
        return SAM3B200_STATUS_FAILED;
    }
    if (n_heads < 1 || n_heads > 65535 || n_heads % a.c.heads != 0) {
        set_error("kv_attention: %lld query heads over %d kv heads (a positive multiple is needed)", (long long)n_heads, a.c.heads);
        return SAM3B200_STATUS_FAILED;
    }
    if (!(scale >= 0.f) || !std::isfinite(scale * 1.4426950408889634f) || window < 0 || (window && !causal)) {
        set_error("kv_attention: bad scale %g or window %lld (a window needs the causal mask)", scale, (long long)window);
        return SAM3B200_STATUS_FAILED;
    }
    a.q = q, a.y = y;
    a.qs = row_tensor(q, type, q_nb, n_heads, a.c.D);
    a.ys = row_tensor(y, y_type, y_nb, n_heads, a.c.D);
    if (!rows_ok("kv_attention", "q", a.qs, a.b.n_rows, n_heads, a.c.D, false) ||
        !rows_ok("kv_attention", "y", a.ys, a.b.n_rows, n_heads, a.c.D, true))
        return SAM3B200_STATUS_FAILED;
    if (!k) {
        set_error("kv_attention: null handle");
        return SAM3B200_STATUS_FAILED;
    }
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return SAM3B200_STATUS_SUCCESS;
    a.q_bf16 = type == SAM3B200_TYPE_BF16;
    a.y_type = y_type;
    a.group = static_cast<int>(n_heads / a.c.heads);
    a.scale_log2 = scale * 1.4426950408889634f;
    // a window that no length reaches is none; below 2^30 it cannot pass 32 bits where rows are more than tokens
    a.causal = causal != 0, a.window = window < a.b.max_len ? static_cast<int>(window) : 0;
    a.part = k->part, a.done = k->done, a.ready = &k->ready, a.err = k->be->err;
    DeviceScope dev(k->be->device);
    // us in a graph, 8 kv heads, few rows and tc, for one sequence of 8000 tokens, one of 100000, 16 of 4000.  Heads of 128:
    // 16 rows a kv head 28 and 35, 84 and 112, 51 and 67; 32 rows 36 and 35, 113 and 111, 76 and 68; 64 rows 39 and 35, 185
    // and 112, 125 and 89.  Heads of 64: 16 rows 17 and 24, 54 and 88, 36 and 56; 32 rows 23 and 24, 77 and 89, 53 and 57;
    // 64 rows 27 and 24, 121 and 88, 86 and 71
    const bool few = static_cast<int64_t>(a.b.max_rows) * a.group <= 32;
    const cudaError_t e = few ? kv_attn_few(a, k->be->num_sms, k->be->stream) : kv_attn_tc(a, k->be->num_sms, k->be->stream);
    k->be->count();
    return cuda_ok(e, "kv_attention launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
