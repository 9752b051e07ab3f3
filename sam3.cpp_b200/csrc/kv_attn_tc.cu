// kv_attn_tc.cu -- attention over the paged 8-bit cache for many query rows a
// kv head (prompts, parts of prompts, cross attention), on the
// 5th-generation tensor cores.
//
// A block owns 256 query rows of one kv head (the group's query heads times
// tokens) as two tiles of 128 and streams the keys in tiles of 128 tokens.
//   warps 0-7:  softmax, one thread a row; warps 0-3 tile 0, 4-7 tile 1;
//   warps 8-11: read the keys' codes (16 bytes a lane straight from the
//               pages, the next tile's in registers meanwhile) and write them
//               as f16, exactly, into 128-byte-swizzled shared memory, and
//               each 16 tokens' scales beside them;
//   warps 12-15: the same for the values;
//   warp 16:    issues the MMAs (17-19 only give their registers away): S_t(j) = Q_t K_j^T, and once softmax t has
//               written its weights over S_t(j), O_t += P_t(j) V_j and
//               S_t(j + 1).  One tile's products run under the other's
//               softmax.
// Keys and values have one layout, [token][64 dimensions] rows of 128 bytes:
// keys are the K-major B operand of the first product, values the N-major B
// operand of the second, so neither is transposed.
// The running maximum is of t = s ks scale log2(e) + log2(vs) (see
// kv_attn.cu), so the scales of 16 tokens enter as one multiply-add in front
// of the exponential.  O stays in tensor memory; it is rescaled only where a
// row's maximum rose by more than kLazy.
// Tensor memory (512 columns): S_t, and P_t over it, at 128 t; O_t at 256 + D t.
#include "kv_attn.cuh"
#include "ptx.cuh"

namespace b200 {
namespace {

enum { TERR_Q = 1 << 8, TERR_K = 1 << 9, TERR_V = 1 << 10, TERR_FREE = 1 << 11, TERR_S = 1 << 12, TERR_P = 1 << 13 };

// Registers a thread after the split: a block starts with 96 for each of its
// five warpgroups, and the shares may not add up to more.
constexpr int kRegsStart = 96, kRegsSoftmax = 144, kRegsCodes = 72, kRegsMma = 48;
static_assert(2 * kRegsSoftmax + 2 * kRegsCodes + kRegsMma <= 5 * kRegsStart, "register shares");

template <int REGS>
__device__ __forceinline__ void take_regs() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void give_regs() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

template <int D>
struct Tc {
    static constexpr int kRows = 256, kKeys = 128;
    static constexpr int kThreads = 20 * 32;
    static constexpr int kHalf = kKeys * 128;             // 64 dimensions of 128 rows
    static constexpr int kTile = kHalf * (D / 64);        // f16 tile of 128 rows
    static constexpr int kQ = 0, kK = 2 * kTile, kV = 4 * kTile, kScales = 6 * kTile;
    static constexpr int kScaleSlots = 4;                 // see sc_full
    static constexpr int kBars = kScales + kScaleSlots * 8 * 16;
    static constexpr int kSmem = kBars + 256 + 1024;      // + alignment
};

__device__ __forceinline__ uint32_t f16_codes(uint32_t w, uint32_t sel) {
    const uint32_t h = __byte_perm(w, 0x64646464u, sel);
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), bias);
    return *reinterpret_cast<const uint32_t *>(&r);
}

// 16 codes of one token as 16 f16 (two swizzled 16-byte chunks).  chunk: the
// token's 16-code chunk, dimensions 16 chunk ...
__device__ __forceinline__ void put_codes(uint8_t *tile, int half_bytes, int token, int chunk, const uint4 &x) {
    const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
    uint4 lo, hi;
    lo = make_uint4(f16_codes(w[0], 0x4140), f16_codes(w[0], 0x4342), f16_codes(w[1], 0x4140), f16_codes(w[1], 0x4342));
    hi = make_uint4(f16_codes(w[2], 0x4140), f16_codes(w[2], 0x4342), f16_codes(w[3], 0x4140), f16_codes(w[3], 0x4342));
    uint8_t *row = tile + (chunk >> 2) * half_bytes + token * 128;
    const int c0 = (2 * (chunk & 3)) ^ (token & 7);
    // lanes of the second half write their upper chunk first: the 8 lanes of a row meet 8 different banks groups
    const bool swap = chunk & 4;
    *reinterpret_cast<uint4 *>(row + (swap ? c0 ^ 1 : c0) * 16) = swap ? hi : lo;
    *reinterpret_cast<uint4 *>(row + (swap ? c0 : c0 ^ 1) * 16) = swap ? lo : hi;
}

// B operand descriptor, N-major, 128-byte swizzle: rows of one k and 64 n;
// 8 k at the stride offset (1024), the next 64 n at the leading offset.
__device__ __forceinline__ uint64_t sw128_nmajor_desc(uint32_t smem_addr, uint32_t next_n) {
    return (sw128_kmajor_desc(smem_addr) & ~(static_cast<uint64_t>(0x3FFF) << 16)) |
           (static_cast<uint64_t>(next_n >> 4) << 16);
}

// Waits for a tcgen05.ld of 16 columns; the registers pass through, so that no use of them moves in front.
__device__ __forceinline__ void wait_ld16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// The softmax constants of 16 tokens: ks scale log2(e), log2(vs), 1 / vs.
struct Scales {
    float k, lv, inv_v, pad;
};

template <int D>
__global__ void __launch_bounds__(Tc<D>::kThreads, 1) kv_attn_tc_kernel(const __grid_constant__ KvAttnArgs a) {
    using C = Tc<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + C::kBars);
    uint64_t *k_full = q_full + 1;       // [2] keys of tile j in slot j % 2
    uint64_t *v_full = k_full + 2;       // [2]
    uint64_t *pair_free = v_full + 2;    // [2] pair p = keys p and values p - 1: read by all their MMAs
    uint64_t *s_full = pair_free + 2;    // [2 tiles] phase j: S_t(j) and O_t up to j - 1 are in tensor memory
    uint64_t *p_full = s_full + 2;       // [2 tiles] phase j: P_t(j) is
    // Scales of tile j, in slot j % 4: written again at tile j + 4, which waits for P_t(j + 1), so a slow softmax
    // warp never sees its phase pass by (keys may run two tiles ahead of it: it must not wait on k_full).
    uint64_t *sc_full = p_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sc_full + C::kScaleSlots);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv = blockIdx.x % a.c.heads, G = a.group;
    if (blockIdx.x == 0) kv_check(a.b, a.c.page_log2, false, a.err);
    int64_t local;
    const int s = kv_find(a.b, (gridDim.x - 1 - blockIdx.x) / a.c.heads, G, 8, 1, local);  // late rows, with the most keys, first
    if (s < 0) return;
    const KvSeq q = kv_seq(a.b, s, a.c.page_log2);
    const int64_t R = static_cast<int64_t>(q.n) * G, row0 = local * C::kRows;
    if (row0 >= R) return;
    const int i_lo = static_cast<int>(row0 / G), i_hi = static_cast<int>((min(row0 + C::kRows, R) - 1) / G);
    const int k_end = kv_last(a, q, i_hi) + 1, k_begin = kv_first(a, kv_last(a, q, i_lo)) & ~15;
    const int ntiles = k_end > k_begin ? (k_end - k_begin + C::kKeys - 1) / C::kKeys : 0;
    const int nq = R - row0 > 128 ? 2 : 1;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4 * nq);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&v_full[i], 4);
            mbar_init(&pair_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < C::kScaleSlots; ++i) mbar_init(&sc_full[i], 1);
        fence_mbar_init();
    }
    if (warp == 16) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8 && warp < 16) {
        // ---- codes -> f16 ----
        give_regs<kRegsCodes>();
        const int which = (warp - 8) >> 2, w = warp & 3;  // keys or values
        constexpr int kChunks = D / 16, kPer = C::kKeys * kChunks / 128;  // 16-code chunks a token, a thread
        constexpr int kTokens = 128 / kChunks;                            // tokens a step of all 128 threads
        const int token0 = (w * 32 + lane) / kChunks, chunk = lane % kChunks;
        const int8_t *codes = a.c.codes[which] + static_cast<int64_t>(token0 & 15) * D + chunk * 16;
        const bool scaling = which == 0 && w == 0 && lane < 8;  // lane g: the scales of tokens 16 g ...
        uint4 x[kPer];
        float ks = 0.f, vs = 0.f;
        // lane g & 7: the page of tokens 16 g ... of tile j, -1 behind the end
        auto page_of = [&](int j) -> int {
            const int tok = k_begin + j * C::kKeys + (lane & 7) * 16;
            if (j >= ntiles || tok >= k_end) return -1;
            return max(kv_page(a.c, a.b, s, tok >> a.c.page_log2, a.err), 0);
        };
        auto fetch = [&](int j, int page) {
            const int in_page = (k_begin + j * C::kKeys + (lane & 7) * 16) & ((1 << a.c.page_log2) - 1);
            const int64_t at = page < 0 ? -1 : kv_slab(a.c, page, kv) + static_cast<int64_t>(in_page) * D;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int64_t from = __shfl_sync(0xffffffffu, at, (i * kTokens + token0) >> 4);
                x[i] = make_uint4(0u, 0u, 0u, 0u);
                if (from >= 0) x[i] = __ldg(reinterpret_cast<const uint4 *>(codes + from));
            }
            if (scaling) {
                const int64_t h = static_cast<int64_t>(max(page, 0)) * a.c.heads + kv;
                ks = page < 0 ? 0.f : a.c.scale[0][h];
                vs = page < 0 ? 0.f : a.c.scale[1][h];
            }
        };
        // Pair p of the pipeline is keys p and values p - 1: keys j reuse the slot of pair j - 2, values j that
        // of pair j - 1 (values 1 wait without need, so that no phase is left out).  Pages are looked up two tiles ahead, codes and scales one.
        uint64_t *full = which == 0 ? k_full : v_full;
        uint8_t *slots = smem + (which == 0 ? C::kK : C::kV);
        int page_next = page_of(1);
        fetch(0, page_of(0));
        for (int j = 0; j < ntiles; ++j) {
            const int page_then = page_of(j + 2), pair = j - 2 + which;
            if (pair >= 0 && !__all_sync(0xffffffffu, mbar_wait(&pair_free[pair & 1], (pair >> 1) & 1, a.err, TERR_FREE))) break;
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                put_codes(slots + (j & 1) * C::kTile, C::kHalf, i * kTokens + token0, chunk, x[i]);
            if (scaling) {
                Scales v{ks * a.scale_log2, vs > 0.f ? __log2f(vs) : kZeroScaleLog2, 0.f, 0.f};
                v.inv_v = ex2_approx(-v.lv);
                reinterpret_cast<Scales *>(smem + C::kScales)[(j % C::kScaleSlots) * 8 + lane] = v;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[j & 1]);
            if (lane == 0 && which == 0 && w == 0) mbar_arrive(&sc_full[j % C::kScaleSlots]);
            fetch(j + 1, page_next);
            page_next = page_then;
        }
    } else if (warp >= 16) {
        // ---- MMA issuer ----
        give_regs<kRegsMma>();
        if (warp == 16) {
            constexpr uint32_t idesc_s = idesc_f16_f32(128, C::kKeys);
            constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // B is N-major
            auto mma_s = [&](int t, int j) {
                const uint32_t qa = smem_u32(smem + C::kQ + t * C::kTile), ka = smem_u32(smem + C::kK + (j & 1) * C::kTile);
    #pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * C::kHalf + (k & 3) * 32;
                    mma_f16(tmem + t * 128, sw128_kmajor_desc(qa + off), sw128_kmajor_desc(ka + off), idesc_s, k > 0);
                }
            };
            auto mma_pv = [&](int t, int j) {
                const uint32_t va = smem_u32(smem + C::kV + (j & 1) * C::kTile);
    #pragma unroll
                for (int k = 0; k < C::kKeys / 16; ++k)
                    mma_f16_ts(tmem + 256 + t * D, tmem + t * 128 + k * 8, sw128_nmajor_desc(va + k * 2048, C::kHalf), idesc_pv,
                               j > 0 || k > 0);
            };
            auto wait = [&](uint64_t *bar, int phase, int code) {
                return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1, a.err, code));
            };
            bool ok = ntiles > 0 && wait(q_full, 0, TERR_Q) && wait(&k_full[0], 0, TERR_K);
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    for (int t = 0; t < nq; ++t) {
                        mma_s(t, 0);
                        mma_commit(&s_full[t]);
                    }
                    mma_commit(&pair_free[0]);
                }
                __syncwarp();
            }
            for (int j = 0; j < ntiles && ok; ++j) {
                const bool more = j + 1 < ntiles;
                ok = (!more || wait(&k_full[(j + 1) & 1], (j + 1) >> 1, TERR_K)) && wait(&v_full[j & 1], j >> 1, TERR_V);
                for (int t = 0; t < nq && ok; ++t) {
                    ok = wait(&p_full[t], j, TERR_P);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_pv(t, j);
                        if (more) mma_s(t, j + 1);
                        mma_commit(&s_full[t]);
                    }
                    __syncwarp();
                }
                if (ok && more && elect_one()) mma_commit(&pair_free[(j + 1) & 1]);
                __syncwarp();
            }
        }
    } else {
        // ---- softmax: thread = row ----
        take_regs<kRegsSoftmax>();
        const int t = warp >> 2;
        const int64_t r = row0 + threadIdx.x;  // t * 128 + row of the tile
        const bool live = r < R;
        if (t < nq) {
            const int i = static_cast<int>(r / G);
            const int64_t head = kv * static_cast<int64_t>(G) + r % G;
            const int last = live ? kv_last(a, q, i) : -1, first = live ? kv_first(a, last) : 0;
            float row_c = 1.f;
            {  // the row as f16; bf16 rows are brought to [1, 2) by a power of two
                const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.qs.token + head * a.qs.head;
                const uint16_t *src = static_cast<const uint16_t *>(a.q) + at;
                uint8_t *dst = smem + C::kQ + t * C::kTile + (threadIdx.x & 127) * 128;
                auto group8 = [&](int c, float (&x)[8]) {
                    if (!live) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = 0.f;
                    } else if (a.q_bf16) {
                        if (a.qs.aligned16) load8<true>(reinterpret_cast<const __nv_bfloat16 *>(src) + c * 8, x);
                        else load8<false>(reinterpret_cast<const __nv_bfloat16 *>(src) + c * 8, x);
                    } else {
                        if (a.qs.aligned16) load8<true>(reinterpret_cast<const __half *>(src) + c * 8, x);
                        else load8<false>(reinterpret_cast<const __half *>(src) + c * 8, x);
                    }
                };
                float down = 1.f;
                if (a.q_bf16) {
                    float top = 0.f;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        float x[8];
                        group8(c, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[e]));
                    }
                    const int e = min((__float_as_int(top) >> 23) & 0xff, 253);
                    down = e ? __int_as_float((254 - e) << 23) : 1.f;
                    row_c = e ? __int_as_float(e << 23) : 1.f;
                }
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    float x[8];
                    group8(c, x);
                    __half2 h[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(x[2 * e] * down, x[2 * e + 1] * down);
                    *reinterpret_cast<uint4 *>(dst + (c >> 3) * C::kHalf + ((c & 7) ^ (threadIdx.x & 7)) * 16) =
                        *reinterpret_cast<const uint4 *>(h);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const uint32_t base = (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t s_col = tmem + base + t * 128, o_col = tmem + base + 256 + t * D;
            float m = -INFINITY, l = 0.f;
            // tokens that some row of this warp does not see
            const int64_t w_lo = row0 + (threadIdx.x & ~31), w_hi = min(w_lo + 31, R - 1);
            const int all_end = w_lo < R ? kv_last(a, q, static_cast<int>(w_lo / G)) : 0x7fffffff;
            const int all_begin = w_lo < R ? kv_first(a, kv_last(a, q, static_cast<int>(w_hi / G))) : 0;
            bool ok = true;
            for (int j = 0; j < ntiles; ++j) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], j & 1, a.err, TERR_S) &&
                                                 mbar_wait(&sc_full[j % C::kScaleSlots], (j / C::kScaleSlots) & 1, a.err, TERR_K));
                if (!ok) break;
                tc_fence_after();
                const Scales *sc = reinterpret_cast<const Scales *>(smem + C::kScales) + (j % C::kScaleSlots) * 8;
                const int tok = k_begin + j * C::kKeys;
                if (tok + C::kKeys - 1 > all_end || tok < all_begin) {
                    // hidden scores become -inf in place; the row sees columns lo .. hi
                    const int hi = last - tok, lo = first - tok;
#pragma unroll 1
                    for (int c = 0; c < C::kKeys; c += 32) {
                        uint32_t x[32];
                        tmem_ld_32x32b_x32(s_col + c, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (c + e > hi || c + e < lo) x[e] = 0xff800000u;
                        tmem_st_32x32b_x32(s_col + c, x);
                    }
                    tmem_wait_st();
                }
                // P for the maximum known so far; where a row passes it by more than kLazy (always in its first
                // tile, rarely later) the maximum is raised and P formed again
                uint32_t pk[C::kKeys / 2];
                float sum = 0.f;
                for (int pass = 0;; ++pass) {
                    const float less = m == -INFINITY ? 0.f : m - kPUp;
                    float top = -INFINITY;
                    sum = 0.f;
                    uint32_t x[2][16];
                    tmem_ld_32x32b_x16(s_col, x[0]);
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        wait_ld16(x[g & 1]);
                        if (g < 7) tmem_ld_32x32b_x16(s_col + 16 * (g + 1), x[(g + 1) & 1]);
                        const Scales v = sc[g];
                        // a factor of 0 (keys or scale 0) would make NaN of -inf; a tiny one leaves 0 of the others
                        const float k = fmaxf(v.k * row_c, 1e-37f), b = v.lv - less;
                        float s0 = 0.f, s1 = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float y0 = b, y1 = b;
                            ffma2(y0, y1, __uint_as_float(x[g & 1][e]), __uint_as_float(x[g & 1][e + 1]), k, k);
                            top = fmaxf(top, fmaxf(y0, y1));
                            y0 = ex2_approx(y0);
                            y1 = ex2_approx(y1);
                            fadd2(s0, s1, s0, s1, y0, y1);
                            const __half2 h = __floats2half2_rn(y0, y1);
                            pk[8 * g + e / 2] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        sum = fmaf(s0 + s1, v.inv_v, sum);
                    }
                    if (pass == 1 || !__any_sync(0xffffffffu, top > (m == -INFINITY ? -INFINITY : kPUp + kLazy))) break;
                    const float to = fmaxf(m, top + less), alpha = m == to ? 1.f : ex2_approx(m - to);
                    m = to;
                    l *= alpha;
                    if (j == 0) continue;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {  // S_t(j) being there, P_t(j - 1) V_(j - 1) is in O_t
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_col + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st_32x32b_x32(o_col + c, o);
                    }
                }
                l += sum;
#pragma unroll
                for (int c = 0; c < C::kKeys / 2; c += 16) {
                    uint32_t part[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[e] = pk[c + e];
                    tmem_st_32x32b_x16(s_col + c, part);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (ok && ntiles > 0) ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], ntiles & 1, a.err, TERR_S));
            if (ok) {
                tc_fence_after();
                const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees no key yields zeros
                const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.ys.token + head * a.ys.head;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    if (ntiles > 0) {
                        tmem_ld_32x32b_x32(o_col + c, o);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = ntiles > 0 ? __uint_as_float(o[e + k]) * inv : 0.f;
                        if (live) kv_store8(a, at + c + e, v);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 16) tmem_dealloc(tmem, 512);
}

template <int D>
cudaError_t launch_tc(const KvAttnArgs &a, int64_t units, cudaStream_t st) {
    using C = Tc<D>;
    cudaError_t e = cudaFuncSetAttribute(kv_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes f;  // the register shares draw on what the block starts with
    e = cudaFuncGetAttributes(&f, kv_attn_tc_kernel<D>);
    if (e != cudaSuccess) return e;
    if (f.numRegs < kRegsStart) return cudaErrorInvalidConfiguration;
    kv_attn_tc_kernel<D><<<static_cast<unsigned>(units * a.c.heads), C::kThreads, C::kSmem, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv_attn_tc(const KvAttnArgs &a, cudaStream_t st) {
    const int64_t units = ((static_cast<int64_t>(a.b.n_rows) * a.group) >> 8) + a.b.n_seqs;
    if (units * a.c.heads > 0x7fffffff) return cudaErrorInvalidValue;
    return a.c.D == 64 ? launch_tc<64>(a, units, st) : launch_tc<128>(a, units, st);
}

}  // namespace b200
