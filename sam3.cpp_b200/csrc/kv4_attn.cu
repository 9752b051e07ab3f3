// kv4_attn.cu -- attention over the paged 4-bit cache: the entry point, and
// the kernel for few query rows a kv head.
//
//   y = softmax(scale q K^T + mask) V,   K = dk ck, V = dv cv
//
// with a scale for each 32 dimensions of a token.  Products with the codes are
// exact in f16, so the scales stay outside the matrix products:
//   score = sum over groups g of dk(token, g) (sum over g's dimensions of q ck)
//   O(d) = sum over tokens of (p dv(token, g(d))) cv
// The first takes a multiply-add in f32 a token and group behind two 16-wide
// products.  The second takes one softmax weight a group: p dv is rounded to
// f16 (2^-11 of it).  With m the running maximum of t + log2(max over g of
// |dv|), t = score scale log2(e), the weights p = 2^(t - m) stay in f32 and
// p dv stays in [-1, 1] for f16 whatever the scales are; O and the sum of p
// have the same reference, so y = O / l.
//
// The kernel is kv_attn.cu's otherwise: one block of 4 warps per (8 or 16
// query rows of a kv head, part of the key range), blocks of 16 tokens through
// a warp's own ring of shared memory, codes as the 16-row operand.  A lane's
// codes come by ldmatrix: plain for keys, word c of each group of token g (8
// dimensions), and transposed for values, 4 dimensions of tokens 2c and 2c + 1
// side by side, so a nibble and the one 16 bits above it are the pair that the
// instruction wants, in either product, and widening is a mask and a
// subtraction for a pair.
#include <algorithm>
#include <cmath>

#include "kv4_codes.cuh"
#include "kv_attn_few.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The scales of one token, D / 32 bf16 numbers.
template <int G>
__device__ __forceinline__ void scales_of(const uint8_t *from, float (&d)[G]) {
    if constexpr (G == 4) {
        const uint2 w = *reinterpret_cast<const uint2 *>(from);
        d[0] = low_bf16(w.x), d[1] = high_bf16(w.x), d[2] = low_bf16(w.y), d[3] = high_bf16(w.y);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(from);
        d[0] = low_bf16(w), d[1] = high_bf16(w);
    }
}

// Eight consecutive query elements, as they come, and the j-th of them.
__device__ __forceinline__ uint4 load_q8(const Kv4AttnArgs &a, int64_t at) {
    const uint16_t *p = static_cast<const uint16_t *>(a.q) + at;
    if (a.qs.aligned16) return *reinterpret_cast<const uint4 *>(p);
    uint4 r;
    uint16_t *e = reinterpret_cast<uint16_t *>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
    return r;
}
__device__ __forceinline__ float q_value(const Kv4AttnArgs &a, const uint4 &x, int j) {
    const uint32_t w = j < 2 ? x.x : j < 4 ? x.y : j < 6 ? x.z : x.w;
    if (a.q_bf16) return j & 1 ? high_bf16(w) : low_bf16(w);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(j & 1 ? w >> 16 : w)));
}

// NT tiles of 8 query rows.
template <int D, int NT>
struct Few4 {
    static constexpr int kRows = 8 * NT, kGroups = D / 32;
    static constexpr int kStages = 4, kBlocks = NT == 1 ? 4 : 3;   // stages of a warp, blocks an SM
    static constexpr int kCodeBytes = 16 * D / 2;                  // of 16 tokens
    static constexpr int kScaleBytes = 16 * kGroups * 2;
    static constexpr int kScaleAt = 2 * kCodeBytes;
    static constexpr int kStageBytes = 2 * (kCodeBytes + kScaleBytes);
    static constexpr int kRing = kWarps * kStages * kStageBytes;
    static constexpr int kRowFloats = D + 4;                       // a joined row, padded against bank conflicts
    static constexpr int kJoin = kWarps * kRows * kRowFloats * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    static_assert(kSmem >= kWarps * kRows * (D + 2) * 4, "shares of the parts");
    static constexpr int kEach = D * kRows / 128 > 8 ? D * kRows / 128 : 8;  // dimensions of a thread that joins
    // Byte of group c of token t within 16 staged tokens, turned so that 8 consecutive tokens' 16 bytes have different
    // banks.  Token t + 8 lies 8 tokens further.
    static __device__ __forceinline__ uint32_t at(int t, int c) {
        if (D == 128) return t * 64 + (c ^ ((t >> 1) & 3)) * 16;
        return t * 32 + (c ^ ((t >> 2) & 1)) * 16;
    }
    static __device__ __forceinline__ int column(int d) { return d; }
};

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, (Few4<D, NT>::kBlocks)) kv4_attn_few_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using F = Few4<D, NT>;
    constexpr int kGroups = F::kGroups;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_m[kWarps][F::kRows], s_l[kWarps][F::kRows];
    wait_for_stream();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int kv = blockIdx.y, G = a.group;
    FewTile tile;
    if (!few_tile<NT>(a, tile)) return;
    const KvSeq &q = tile.q;
    const int row0 = tile.row0, i_lo = tile.i_lo, i_hi = tile.i_hi, R = tile.R, t_begin = tile.t_begin, t_end = tile.t_end;
    const int n_blocks = t_end > t_begin ? (t_end - t_begin + 15) / 16 : 0;
    const int mine = n_blocks > warp ? (n_blocks - warp + kWarps - 1) / kWarps : 0;  // blocks warp, warp + 4, ...

    // the queries are on their way while the first pages are looked up: row 8 n + g, dimensions 8 c ... of each group
    const int rest0 = row0 - i_lo * G;  // row 0 of the tile: token i_lo, head rest0 of the group
    uint4 qraw[NT][kGroups];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int x = rest0 + 8 * n + g, i = i_lo + x / G;
        const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.qs.token + (static_cast<int64_t>(kv) * G + x % G) * a.qs.head;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            qraw[n][k] = make_uint4(0u, 0u, 0u, 0u);
            if (row0 + 8 * n + g < R) qraw[n][k] = load_q8(a, at + k * 32 + c * 8);
        }
    }

    uint8_t *ring = smem + warp * F::kStages * F::kStageBytes;
    // this lane's bytes within a stage: the copy of chunk lane (of 32 a step), and its row of the matrices that it loads
    const uint32_t put0 = F::at(lane / kGroups, lane % kGroups);
    const uint32_t get0 = D == 128 ? F::at(lane & 7, lane >> 3) : F::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
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
            const int64_t at = ((static_cast<int64_t>(page) * a.c.heads + kv) << a.c.page_log2) + (tok & ((1 << a.c.page_log2) - 1));
            const uint32_t dst = smem_u32(ring + slot * F::kStageBytes);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int k = 0; k < F::kCodeBytes / 512; ++k)  // a step of 8 (D = 128) or 16 tokens
                    cp16(dst + w * F::kCodeBytes + put0 + k * 512, a.c.codes[w] + at * (D / 2) + lane * 16 + k * 512);
            constexpr int kChunks = F::kScaleBytes / 16;
            if (lane < 2 * kChunks) {
                const int w = lane / kChunks, k = lane % kChunks;
                cp16(dst + F::kScaleAt + lane * 16, a.c.scale[w] + at * kGroups + k * 8);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int j = 0; j < F::kStages - 1; ++j) issue(j, j);

    // queries as f16: for a group's two products the pairs of dimensions that codes4 gives
    uint32_t qf[NT][kGroups][4];
    float row_c[NT][2];  // for rows 8 n + 2 c, + 1: scale log2(e), and what the power of two below took
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(q_value(a, qraw[n][k], j)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // bf16 rows are brought to [1, 2) by a power of two, which f16 then holds to 2^-25 of the largest
        const int e = a.q_bf16 ? min((__float_as_int(top) >> 23) & 0xff, 253) : 0;
        const float down = e ? __int_as_float((254 - e) << 23) : 1.f, up = a.scale_log2 * (e ? __int_as_float(e << 23) : 1.f);
#pragma unroll
        for (int k = 0; k < kGroups; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                qf[n][k][j] = pack_f16(q_value(a, qraw[n][k], j) * down, q_value(a, qraw[n][k], j + 4) * down);
#pragma unroll
        for (int j = 0; j < 2; ++j) row_c[n][j] = __shfl_sync(0xffffffffu, up, (2 * c + j) * 4);
    }
    // tokens that some row of the tile does not see, and those that none sees (they need not hold numbers)
    const int seen_by_all = kv_last(a, q, i_lo), window_end = kv_first(a, kv_last(a, q, i_hi)), first_any = kv_first(a, seen_by_all);

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
        const uint32_t st_at = smem_u32(st);
        slot_in = slot;
        slot = slot + 1 == F::kStages ? 0 : slot + 1;
        const int tok = t_begin + (j * kWarps + warp) * 16;

        // scores of tokens g (t[n][0], [1]) and g + 8 ([2], [3]) for rows 8 n + 2 c, + 1
        float t[NT][4];
        {
            uint32_t w[2][kGroups];  // word c of each group of tokens g and g + 8
            uint32_t r[4];
            ldmatrix4<false>(r, st_at + get0);
            if constexpr (D == 128) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[0][k] = r[k];
                ldmatrix4<false>(r, st_at + get0 + 8 * 64);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[1][k] = r[k];
            } else {
                w[0][0] = r[0], w[0][1] = r[1], w[1][0] = r[2], w[1][1] = r[3];
            }
            float d0[kGroups], d1[kGroups];
            scales_of<kGroups>(st + F::kScaleAt + g * (2 * kGroups), d0);
            scales_of<kGroups>(st + F::kScaleAt + (g + 8) * (2 * kGroups), d1);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                uint32_t u[4], v[4];
                codes4(w[0][k], u);
                codes4(w[1][k], v);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float s[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(s, u[0], v[0], u[1], v[1], qf[n][k][0], qf[n][k][1]);
                    mma16816(s, u[2], v[2], u[3], v[3], qf[n][k][2], qf[n][k][3]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float d = i < 2 ? d0[k] : d1[k];
                        t[n][i] = k ? fmaf(s[i], d, t[n][i]) : s[i] * d;
                    }
                }
            }
        }
        float d0[kGroups], d1[kGroups];  // the values' scales of tokens g and g + 8
        scales_of<kGroups>(st + F::kScaleAt + F::kScaleBytes + g * (2 * kGroups), d0);
        scales_of<kGroups>(st + F::kScaleAt + F::kScaleBytes + (g + 8) * (2 * kGroups), d1);
        if (tok + 15 >= t_end || tok < first_any) {
            const bool out0 = tok + g >= t_end || tok + g < first_any, out1 = tok + g + 8 >= t_end || tok + g + 8 < first_any;
#pragma unroll
            for (int k = 0; k < kGroups; ++k) d0[k] = out0 ? 0.f : d0[k], d1[k] = out1 ? 0.f : d1[k];
        }
        float top0 = 0.f, top1 = 0.f;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) top0 = fmaxf(top0, fabsf(d0[k])), top1 = fmaxf(top1, fabsf(d1[k]));
        const float lv0 = fmaxf(__log2f(top0), kZeroScaleLog2), lv1 = fmaxf(__log2f(top1), kZeroScaleLog2);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) t[n][k] *= row_c[n][k & 1];
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
            for (int k = 0; k < 2; ++k) rise |= fmaxf(t[n][k] + lv0, t[n][k + 2] + lv1) > m[n][k] + kLazy;
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float top = fmaxf(t[n][k] + lv0, t[n][k + 2] + lv1);
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
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float less = m[n][k] == -INFINITY ? 0.f : m[n][k] - kPUp;
                t[n][k] = ex2_approx(t[n][k] - less);
                t[n][k + 2] = ex2_approx(t[n][k + 2] - less);
                l[n][k] += t[n][k] + t[n][k + 2];
            }

        // values: of each group 4 dimensions (4 g ...) of tokens 2c, 2c + 1 and of 8 + 2c, 9 + 2c
        uint32_t w[2][kGroups];
        {
            uint32_t r[4];
            ldmatrix4<true>(r, st_at + F::kCodeBytes + get0);
            if constexpr (D == 128) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[0][k] = r[k];
                ldmatrix4<true>(r, st_at + F::kCodeBytes + get0 + 8 * 64);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[1][k] = r[k];
            } else {
                w[0][0] = r[0], w[0][1] = r[1], w[1][0] = r[2], w[1][1] = r[3];
            }
        }
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            uint32_t u[4], v[4];
            codes4(w[0][k], u);
            codes4(w[1][k], v);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t p0 = transposed(pack_f16(t[n][0] * d0[k], t[n][1] * d0[k]));
                const uint32_t p1 = transposed(pack_f16(t[n][2] * d1[k], t[n][3] * d1[k]));
                // dimensions 4 g, + 1 of the group are rows g, g + 8 of one product, + 2, + 3 of the next
                mma16816(o[n][2 * k], u[0], u[1], v[0], v[1], p0, p1);
                mma16816(o[n][2 * k + 1], u[2], u[3], v[2], v[3], p0, p1);
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
            float *to = rows + (warp * F::kRows + row) * F::kRowFloats + 4 * g;
#pragma unroll
            for (int i = 0; i < D / 16; i += 2)
                *reinterpret_cast<float4 *>(to + 16 * i) = make_float4(o[n][i][k], o[n][i][k + 2], o[n][i + 1][k], o[n][i + 1][k + 2]);
        }
    __syncthreads();
    few_finish<F, D>(a, tile, smem, s_m, s_l);
}

template <int D, int NT>
cudaError_t launch(Kv4AttnArgs &a, int num_sms, cudaStream_t st) {
    return few_launch<Few4<D, NT>, NT>(kv4_attn_few_kernel<D, NT>, a, kReadyFew4 + 2 * (NT - 1) + (D == 64), num_sms, st);
}

}  // namespace

cudaError_t kv_attn_few(Kv4AttnArgs a, int num_sms, cudaStream_t st) {
    const bool one = static_cast<int64_t>(a.b.max_rows) * a.group <= 8;
    if (a.c.D == 64) return one ? launch<64, 1>(a, num_sms, st) : launch<64, 2>(a, num_sms, st);
    return one ? launch<128, 1>(a, num_sms, st) : launch<128, 2>(a, num_sms, st);
}

}  // namespace b200

using namespace b200;

extern "C" int sam3b200_kv4_attention_run(sam3b200_kv_attention *h, const sam3b200_kv4_cache *cache,
                                          const sam3b200_kv_batch *batch, int type, const void *q, const int64_t *q_nb,
                                          int64_t n_heads, float scale, int causal, int64_t window, int y_type, void *y,
                                          const int64_t *y_nb) {
    auto *k = reinterpret_cast<KvAttention *>(h);
    Kv4AttnArgs a;
    bool empty;
    if (!kv_attn_args("kv4_attention", k, cache, batch, type, q, q_nb, n_heads, scale, causal, window, y_type, y, y_nb, a, empty))
        return SAM3B200_STATUS_FAILED;
    if (empty) return SAM3B200_STATUS_SUCCESS;
    DeviceScope dev(k->be->device);
    const bool few = static_cast<int64_t>(a.b.max_rows) * a.group <= 32;
    const cudaError_t e = few ? kv_attn_few(a, k->be->num_sms, k->be->stream) : kv_attn_tc(a, k->be->num_sms, k->be->stream);
    k->be->count();
    return cuda_ok(e, "kv4_attention launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
