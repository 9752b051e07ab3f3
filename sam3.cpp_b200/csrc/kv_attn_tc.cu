// kv_attn_tc.cu -- attention over the paged caches of 8 and 4 bits for many
// query rows a kv head (prompts, parts of prompts, cross attention), on the
// 5th-generation tensor cores.
//
// A block owns 256 query rows of one kv head (the group's query heads times
// tokens) as two tiles of 128 and streams the keys in tiles of 128 tokens.
//   warps 0-7:  softmax, one thread a row; warps 0-3 tile 0, 4-7 tile 1;
//   warps 8-11: read the codes (16 bytes a lane straight from the pages, the
//               next tile's in registers meanwhile) and write them as f16,
//               exactly, into 128-byte-swizzled shared memory, and each 16
//               tokens' scales beside them;
//   warps 12, 13: issue the MMAs of tile 0 and 1 (14, 15 only give their
//               registers away; one warp for both was the bottleneck), in
//               steps of 64 tokens: S_t(i) = Q_t K_i^T into one of two
//               buffers, and once softmax t has written its weights over
//               S_t(i), O_t += P_t(i) V_i and S_t(i + 2).  A softmax warp thus
//               finds its next scores ready; the products of one step run
//               under the softmax of the next, and the tiles under each other.
// Keys and values have one layout, [token][64 dimensions] rows of 128 bytes:
// keys are the K-major B operand of the first product, values the N-major B
// operand of the second, so neither is transposed.
// The running maximum is of t = s ks scale log2(e) + log2(vs) (see
// kv_attn.cu), so the scales of 16 tokens enter as one multiply-add in front
// of the exponential.  O stays in tensor memory; it is rescaled only where a
// row's maximum rose by more than kLazy.
// The 4-bit cache's scales, one for 32 dimensions of a token, are multiplied
// in while its codes are widened: of 16 tokens the power of two of the largest
// scale takes the place of the page's scale, and what is left of each, in
// [0, 2), times a code is exact in f16 (8 + 3 bits) down to 2^-10 of it.  Its
// nibbles come out in pairs (0, 4), (1, 5), (2, 6), (3, 7) of 8 dimensions:
// keys and values stay in that order, the queries are staged in it, and the
// results are put back where they are read from tensor memory.
// Tensor memory (512 columns): S_t(i), and P_t(i) over it, at 128 t + 64 (i % 2);
// O_t at 256 + D t.
//
// Bounds, for 128 keys of a block: the products take 2048 cycles at D = 128
// (half at 64), the exponentials 2048 on the special-function unit, 1536 with
// a quarter of them on the FMA pipe.  Measured 2.2 us (about 4100 cycles) at
// D = 128, 1130 TFLOP/s, and 2.0 us at 64, 620 TFLOP/s: the two softmax warps
// of a sub-partition run in step and leave it idle half of their waits.  A
// block's start and end cost about 9 us more (at D = 128 in bf16 6 to 7 to its
// first scores, which wait for the query rows; in f16 at 64 under 5, of which 3
// are the first keys; 3 from the last).  A whole
// prompt of 4096 tokens, 32 heads on 8 of 128: 181 us, 759 TFLOP/s; 5184 rows
// over 10368 tokens, 16 heads of 64: 443 us.  Not kept: two threads a row (212
// us for the prompt then at 193), one lane polling for a warp (277), the
// results by whole rows through shared memory (185 to 188: the loop's
// registers).
// Over the 4-bit cache the same prompt takes 165 to 167 us (832 to 824 TFLOP/s), since half
// the bytes come in and a page has no scale of its own to wait for, the 5184 rows
// 448, and 4 parts of prompts of 400 to 800 tokens behind 2500 to 6700 (32 heads
// on 4 of 128) 290 to 309, in place of 305.
#include <algorithm>
#include <type_traits>

#include "kv_attn.cuh"
#include "kv4_codes.cuh"
#include "ptx.cuh"

namespace b200 {
namespace {

enum { TERR_Q = 1 << 8, TERR_K = 1 << 9, TERR_V = 1 << 10, TERR_FREE = 1 << 11, TERR_S = 1 << 12, TERR_P = 1 << 13 };
static_assert(((TERR_Q | TERR_K | TERR_V | TERR_FREE | TERR_S | TERR_P) & kErrData) == 0, "bits of waits");

// Registers a thread after the split: a block starts with 128 for each of its
// four warpgroups, and the shares may not add up to more.  Those that give
// may not end above the start, nor the one that takes below it: an illegal
// instruction.
constexpr int kRegsStart = 128, kRegsSoftmax = 176, kRegsCodes = 104, kRegsMma = 56;
static_assert(2 * kRegsSoftmax + kRegsCodes + kRegsMma <= 4 * kRegsStart, "register shares");
static_assert(kRegsSoftmax >= kRegsStart && kRegsCodes <= kRegsStart && kRegsMma <= kRegsStart, "register shares' directions");
// (ptxas spills 4 bytes of the D = 128 kernel's 128 registers and 8 of the other's; the shares were measured with that.)
static_assert(kRegsSoftmax % 8 == 0 && kRegsCodes % 8 == 0 && kRegsMma % 8 == 0, "register shares are in eights");

// Of 8 pairs of weights, those whose exponential runs on the FMA pipe (us, prompt and images: 0 pairs 191 and 465, 2
// 185 and 444, 3 186 and 451).
constexpr int kPolyPairs = 2;

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
    static constexpr int kThreads = 16 * 32;
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

// 16 codes of one token as 16 f16: two 16-byte chunks at at and at ^ 16.
__device__ __forceinline__ void put_codes(uint8_t *tile, uint32_t at, const uint4 &x) {
    const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
    *reinterpret_cast<uint4 *>(tile + at) =
        make_uint4(f16_codes(w[0], 0x4140), f16_codes(w[0], 0x4342), f16_codes(w[1], 0x4140), f16_codes(w[1], 0x4342));
    *reinterpret_cast<uint4 *>(tile + (at ^ 16)) =
        make_uint4(f16_codes(w[2], 0x4140), f16_codes(w[2], 0x4342), f16_codes(w[3], 0x4140), f16_codes(w[3], 0x4342));
}

__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int *err, int code) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

// B operand descriptor, N-major, 128-byte swizzle: rows of one k and 64 n;
// 8 k at the stride offset (1024), the next 64 n at the leading offset.
__device__ __forceinline__ uint64_t sw128_nmajor_desc(uint32_t smem_addr, uint32_t next_n) {
    return (sw128_kmajor_desc(smem_addr) & ~(static_cast<uint64_t>(0x3FFF) << 16)) |
           (static_cast<uint64_t>(next_n >> 4) << 16);
}

// Registers that a tcgen05.ld wrote pass through here behind the wait, so that no use of them moves in front of it.
__device__ __forceinline__ void pass32(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// d = a b + c for two numbers at once.
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}

// The largest of three numbers, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^y of two numbers on the FMA pipe, for y <= 127: the magic sum splits y into an integer n and f in [-1/2, 1/2], a
// cubic with nearly the least largest relative error there (7.8e-5; 7.5e-5 by Remez exchange) gives 2^f, n goes to the
// exponent.  At the least y that is let through, -127 + 14 / 2^17, the cubic is 1 (its constant was moved by 2e-6 for
// that), so that n takes all of its bits: the weight of a masked score is 0 exactly, and the weights of a row that sees
// no key add up to 0.  NaN is not kept.
constexpr float kPolyLeast = -127.f + 14.f / 131072.f;
__device__ __forceinline__ void exp2_poly(float &y0, float &y1) {
    y0 = fmaxf(y0, kPolyLeast), y1 = fmaxf(y1, kPolyLeast);
    float n0, n1, f0, f1;
    fadd2(n0, n1, y0, y1, 12582912.f, 12582912.f);
    fadd2(f0, f1, n0, n1, -12582912.f, -12582912.f);
    fadd2(f0, f1, y0, y1, -f0, -f1);
    float a0, a1, b0 = 0.69326097f, b1 = 0.69326097f, c0 = 0.999926f, c1 = 0.999926f;
    fma2(a0, a1, f0, f1, 0.05517167f, 0.24261113f);
    ffma2(b0, b1, a0, a1, f0, f1);
    ffma2(c0, c1, b0, b1, f0, f1);
    y0 = __int_as_float((__float_as_int(n0) << 23) + __float_as_int(c0));
    y1 = __int_as_float((__float_as_int(n1) << 23) + __float_as_int(c1));
}

// 8 elements in the order (0, 4, 1, 5, 2, 6, 3, 7).
__device__ __forceinline__ uint4 paired(const uint4 &x) {
    return make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
}

// The softmax constants of 16 tokens: ks scale log2(e), log2(vs), 1 / vs.
struct Scales {
    float k, lv, inv_v, pad;
};

template <int D, typename Args>
__global__ void __launch_bounds__(Tc<D>::kThreads, 1) kv_attn_tc_kernel(const __grid_constant__ Args a) {
    using C = Tc<D>;
    constexpr bool kFour = std::is_same<Args, Kv4AttnArgs>::value;
    extern __shared__ uint8_t smem_raw[];
    wait_for_stream();
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *q_full = reinterpret_cast<uint64_t *>(smem + C::kBars);
    uint64_t *k_full = q_full + 1;       // [2] keys of tile j in slot j % 2
    uint64_t *v_full = k_full + 2;       // [2]
    uint64_t *k_free = v_full + 2;       // [2] tile j is read by all its MMAs
    uint64_t *v_free = k_free + 2;       // [2]
    uint64_t *s_full = v_free + 2;       // [tile][i % 2] S_t(i) is in tensor memory, and so is O_t with P_t(i - 2) V
    uint64_t *p_full = s_full + 4;       // [tile][i % 2] P_t(i) is there (and O_t rescaled)
    // Scales of key tile j, in slot j % 4: written again for tile j + 4, which waits for P_t(2 j + 3), so a slow
    // softmax warp never sees its phase pass by (the keys run ahead of it: it must not wait on k_full).
    uint64_t *sc_full = p_full + 4;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sc_full + C::kScaleSlots);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % a.splits, kv = blockIdx.x / a.splits % a.c.heads, G = a.group;
    const unsigned unit = (gridDim.x - 1 - blockIdx.x) / a.splits / a.c.heads;  // late rows, with the most keys, come first
    if (blockIdx.x == 0) kv_check(a.b, a.c.page_log2, false, a.err);
    int64_t local;
    KvSeq q;
    if (!kv_find(a.b, unit, G, 8, 1, a.c.page_log2, q, local)) return;
    const int s = q.s;
    const int R = q.n * G;  // the host keeps n_rows * G below 2^31
    if (local * C::kRows >= R) return;
    const int row0 = static_cast<int>(local) * C::kRows, i_lo = row0 / G, i_hi = (min(row0 + C::kRows, R) - 1) / G;
    // the rows' keys, and this block's part of them
    const int all_keys_end = kv_last(a, q, i_hi) + 1, all_keys_begin = kv_first(a, kv_last(a, q, i_lo)) & ~15;
    const int range = max(all_keys_end - all_keys_begin, 0);
    const int part = max(range < a.short_range ? a.chunk_short : a.chunk, ((range + a.splits - 1) / a.splits + 127) & ~127);
    const int n_split = max((range + part - 1) / part, 1);
    if (split >= n_split) return;
    const int k_begin = all_keys_begin + split * part, k_end = min(k_begin + part, all_keys_end);
    const int ntiles = k_end > k_begin ? (k_end - k_begin + C::kKeys - 1) / C::kKeys : 0;  // of 128 tokens, as they are staged
    const int nsteps = k_end > k_begin ? (k_end - k_begin + 63) / 64 : 0;                  // of 64 tokens, as they are used
    const int nq = R - row0 > 128 ? 2 : 1;
    const int64_t group = static_cast<int64_t>(unit) * a.c.heads + kv;
    auto part_of = [&](int k) { return a.part + (group * a.splits + k) * (C::kRows * (D + 2)); };

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4 * nq);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&v_full[i], 4);
            mbar_init(&k_free[i], nq);
            mbar_init(&v_free[i], nq);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < C::kScaleSlots; ++i) mbar_init(&sc_full[i], 4);
        fence_mbar_init();
    }
    __syncthreads();
    constexpr uint32_t tmem = 0;  // all columns are this block's, so they start at 0

    if (warp >= 8 && warp < 12) {
        // ---- codes -> f16 ----
        give_regs<kRegsCodes>();
        // warp w widens tokens 32 w ... 32 w + 31 of each tile: two runs of 16, each in one page
        const int w = warp - 8;
        struct Pages {
            int p[2];  // -1 behind the end
        };
        // Table entries are looked up a tile before they are looked at, so that no load is waited for here.
        auto lookup = [&](int j) {
            Pages r;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int tok = k_begin + j * C::kKeys + w * 32 + g * 16;
                r.p[g] = 0;
                if (j < ntiles && tok < k_end) r.p[g] = a.b.table[s * a.b.table_width + (tok >> a.c.page_log2)];
            }
            return r;
        };
        auto checked = [&](int j, Pages r) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (j >= ntiles || k_begin + j * C::kKeys + w * 32 + g * 16 >= k_end) {
                    r.p[g] = -1;
                } else if (r.p[g] < 0 || r.p[g] >= a.c.n_pages) {
                    atomicOr(a.err, kErrKvPage);
                    r.p[g] = 0;
                }
            }
            return r;
        };
        auto publish = [&](uint64_t *bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        if constexpr (kFour) {
            constexpr int kGroups = D / 32, kTokens = 32 / kGroups, kPer = 32 / kTokens;  // tokens a step, steps a tile
            // A lane takes one group of a token a step: 16 bytes of codes, contiguous over the warp, and 64 bytes of f16.
            const int grp = lane % kGroups, token0 = lane / kGroups, half = grp >> 1;
            // Chunk c of token t's row goes to c ^ (t & 7); lanes of the upper half store chunks 2, 3, 0, 1, so that the 8
            // lanes that store together have different banks.
            const uint32_t at0 = half * C::kHalf + (w * 32 + token0) * 128;
            const int first_any = kv_first(a, kv_last(a, q, i_lo));  // tokens in front of it need not hold numbers
            uint4 kx[kPer], vx[kPer];
            uint16_t kd[kPer], vd[kPer];  // scales
            auto fetch = [&](int which, int j, const Pages &pg, uint4 (&x)[kPer], uint16_t (&d)[kPer]) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int tok = k_begin + j * C::kKeys + w * 32 + g * 16 + token0;
                    const int64_t at = ((static_cast<int64_t>(max(pg.p[g], 0)) * a.c.heads + kv) << a.c.page_log2) + (tok & ((1 << a.c.page_log2) - 1));
#pragma unroll
                    for (int i = 0; i < kPer / 2; ++i) {
                        const int k = g * (kPer / 2) + i, t = tok + i * kTokens;
                        x[k] = make_uint4(0u, 0u, 0u, 0u);
                        d[k] = 0;
                        if (pg.p[g] < 0 || t >= k_end || t < first_any) continue;
                        x[k] = *reinterpret_cast<const uint4 *>(a.c.codes[which] + (at + i * kTokens) * (D / 2) + grp * 16);
                        d[k] = reinterpret_cast<const uint16_t *>(a.c.scale[which])[(at + i * kTokens) * kGroups + grp];
                    }
                }
            };
            // biased exponents of the largest scales of the two runs, in the halves of a word
            auto exponents = [&](const uint16_t (&d)[kPer]) {
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < kPer; ++k) top = __vmaxu2(top, static_cast<uint32_t>(d[k] & 0x7fff) << (k < kPer / 2 ? 0 : 16));
#pragma unroll
                for (int o = 16; o; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
                return (top >> 7) & 0x00ff00ffu;
            };
            auto put = [&](uint8_t *tile, const uint4 (&x)[kPer], const uint16_t (&d)[kPer], uint32_t e) {
#pragma unroll
                for (int k = 0; k < kPer; ++k) {
                    const int er = min(static_cast<int>(k < kPer / 2 ? e & 0xffffu : e >> 16), 253);
                    const float less = er ? __int_as_float((254 - er) << 23) : 0.f;
                    const __half2 by = __float2half2_rn(__uint_as_float(static_cast<uint32_t>(d[k]) << 16) * less);
                    const uint32_t words[4] = {half ? x[k].z : x[k].x, half ? x[k].w : x[k].y, half ? x[k].x : x[k].z, half ? x[k].y : x[k].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t p[4];
                        codes4(words[i], p);
                        __half2 v[4];
#pragma unroll
                        for (int n = 0; n < 4; ++n) v[n] = __hmul2(*reinterpret_cast<const __half2 *>(&p[n]), by);
                        const int chunk = (grp & 1) * 4 + (i ^ (2 * half));
                        *reinterpret_cast<uint4 *>(tile + at0 + k * kTokens * 128 + ((chunk ^ (token0 & 7)) * 16)) = *reinterpret_cast<const uint4 *>(v);
                    }
                }
            };
            auto put_scales = [&](int j, uint32_t ke, uint32_t ve) {
                if (lane >= 2) return;
                const int k = min(static_cast<int>(lane ? ke >> 16 : ke & 0xffffu), 253), v = min(static_cast<int>(lane ? ve >> 16 : ve & 0xffffu), 253);
                Scales z{__int_as_float(k << 23) * a.scale_log2, v ? static_cast<float>(v - 127) : kZeroScaleLog2, 0.f, 0.f};
                z.inv_v = ex2_approx(-z.lv);
                reinterpret_cast<Scales *>(smem + C::kScales)[(j % C::kScaleSlots) * 8 + w * 2 + lane] = z;
            };
            // Codes and scales are loaded a tile ahead, table entries two.
            Pages pg_next = checked(0, lookup(0)), raw = lookup(1);
            fetch(0, 0, pg_next, kx, kd);
            fetch(1, 0, pg_next, vx, vd);
            for (int j = 0; j < ntiles; ++j) {
                pg_next = checked(j + 1, raw);
                raw = lookup(j + 2);
                const uint32_t ke = exponents(kd), ve = exponents(vd);
                if (j >= 2 && !warp_wait(&k_free[j & 1], ((j >> 1) - 1) & 1, a.err, TERR_FREE)) break;
                put(smem + C::kK + (j & 1) * C::kTile, kx, kd, ke);
                put_scales(j, ke, ve);
                publish(&k_full[j & 1]);
                if (lane == 0) mbar_arrive(&sc_full[j % C::kScaleSlots]);
                fetch(0, j + 1, pg_next, kx, kd);
                if (j >= 2 && !warp_wait(&v_free[j & 1], ((j >> 1) - 1) & 1, a.err, TERR_FREE)) break;
                put(smem + C::kV + (j & 1) * C::kTile, vx, vd, ve);
                publish(&v_full[j & 1]);
                fetch(1, j + 1, pg_next, vx, vd);
            }
        } else {
            constexpr int kChunks = D / 16, kPer = C::kKeys * kChunks / 128;  // 16-code chunks a token, a thread
            constexpr int kTokens = 32 / kChunks;                             // tokens a step
            // Lane bits: 0-1 the chunk within 64 dimensions, 2 the token's lowest bit, 3 (D = 128) the half, the rest
            // more of the token.  8 lanes that store together are then 2 neighbouring tokens of one half, whose swizzled
            // chunks have different banks; a token's 128 bytes are still read by lanes of one load.
            const int half = D == 128 ? (lane >> 3) & 1 : 0;
            const int token0 = ((lane >> 2) & 1) + (D == 128 ? (lane >> 4) * 2 : (lane >> 3) * 2);  // of the step's kTokens
            const int chunk = half * 4 + (lane & 3);
            // where this lane's first chunk goes: token t's row, chunk c of it at c ^ (t & 7)
            const uint32_t at0 = half * C::kHalf + (w * 32 + token0) * 128 + ((2 * (lane & 3)) ^ (token0 & 7)) * 16;
            const int64_t own = static_cast<int64_t>(token0) * D + chunk * 16;
            uint4 kx[kPer], vx[kPer];
            float ks = 0.f, vs = 0.f;  // lanes 0, 1: the scales of the two runs
            auto fetch = [&](int which, int j, const Pages &pg, uint4 (&x)[kPer]) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int in_page = (k_begin + j * C::kKeys + w * 32 + g * 16) & ((1 << a.c.page_log2) - 1);
                    const int8_t *from = a.c.codes[which] + kv_slab(a.c, max(pg.p[g], 0), kv) + static_cast<int64_t>(in_page) * D + own;
#pragma unroll
                    for (int i = 0; i < kPer / 2; ++i) {
                        uint4 &v = x[g * (kPer / 2) + i];
                        v = make_uint4(0u, 0u, 0u, 0u);
                        if (pg.p[g] >= 0) v = *reinterpret_cast<const uint4 *>(from + i * kTokens * D);
                    }
                }
            };
            auto fetch_scales = [&](const Pages &pg) {
                if (lane >= 2) return;
                const int page = lane ? pg.p[1] : pg.p[0];
                const int64_t h = static_cast<int64_t>(max(page, 0)) * a.c.heads + kv;
                ks = page < 0 ? 0.f : a.c.scale[0][h];
                vs = page < 0 ? 0.f : a.c.scale[1][h];
            };
            auto put = [&](uint8_t *tile, const uint4 (&x)[kPer]) {
#pragma unroll
                for (int i = 0; i < kPer; ++i)  // a step of 4 tokens (D = 128) flips bit 2 of t & 7
                    put_codes(tile, (kTokens == 4 && (i & 1) ? at0 ^ 64 : at0) + i * kTokens * 128, x[i]);
            };
            auto put_scales = [&](int j) {
                if (lane >= 2) return;
                Scales v{ks * a.scale_log2, vs > 0.f ? __log2f(vs) : kZeroScaleLog2, 0.f, 0.f};
                v.inv_v = ex2_approx(-v.lv);
                reinterpret_cast<Scales *>(smem + C::kScales)[(j % C::kScaleSlots) * 8 + w * 2 + lane] = v;
            };
            // Codes and scales are loaded a tile ahead, table entries two.
            Pages pg_next = checked(0, lookup(0)), raw = lookup(1);
            fetch(0, 0, pg_next, kx);
            fetch_scales(pg_next);
            fetch(1, 0, pg_next, vx);
            for (int j = 0; j < ntiles; ++j) {
                pg_next = checked(j + 1, raw);
                raw = lookup(j + 2);
                if (j >= 2 && !warp_wait(&k_free[j & 1], ((j >> 1) - 1) & 1, a.err, TERR_FREE)) break;
                put(smem + C::kK + (j & 1) * C::kTile, kx);
                put_scales(j);
                publish(&k_full[j & 1]);
                if (lane == 0) mbar_arrive(&sc_full[j % C::kScaleSlots]);
                fetch(0, j + 1, pg_next, kx);
                fetch_scales(pg_next);
                if (j >= 2 && !warp_wait(&v_free[j & 1], ((j >> 1) - 1) & 1, a.err, TERR_FREE)) break;
                put(smem + C::kV + (j & 1) * C::kTile, vx);
                publish(&v_full[j & 1]);
                fetch(1, j + 1, pg_next, vx);
            }
        }
    } else if (warp >= 12) {
        // ---- MMA issuer ----
        give_regs<kRegsMma>();
        if (warp == 12) {  // while keys and queries are on their way
            tmem_alloc(tmem_slot, 512);
            tmem_relinquish();
        }
        asm volatile("bar.sync 2, 128;" ::: "memory");
        tc_fence_after();
        if (warp - 12 < nq) {
            const int t = warp - 12;
            constexpr uint32_t idesc_s = idesc_f16_f32(128, 64);
            constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // B is N-major
            // Descriptors advance by constants (addresses in 16 bytes), so that an MMA costs its issuer little.
            const uint64_t q_desc = sw128_kmajor_desc(smem_u32(smem + C::kQ)), k_desc = sw128_kmajor_desc(smem_u32(smem + C::kK)),
                           v_desc = sw128_nmajor_desc(smem_u32(smem + C::kV), C::kHalf);
            auto mma_s = [&](int i) {
                const uint64_t qd = q_desc + t * (C::kTile >> 4), kd = k_desc + ((i >> 1) & 1) * (C::kTile >> 4) + (i & 1) * (64 * 128 >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = ((k >> 2) * C::kHalf + (k & 3) * 32) >> 4;
                    mma_f16(tmem + t * 128 + (i & 1) * 64, qd + off, kd + off, idesc_s, k > 0);
                }
            };
            auto mma_pv = [&](int i) {
                const uint64_t vd = v_desc + ((i >> 1) & 1) * (C::kTile >> 4) + (i & 1) * (64 * 128 >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_f16_ts(tmem + 256 + t * D, tmem + t * 128 + (i & 1) * 64 + k * 8, vd + (k * 2048 >> 4), idesc_pv, i > 0 || k > 0);
            };
            auto wait = [&](uint64_t *bar, int phase, int code) {
                return warp_wait(bar, phase & 1, a.err, code);
            };
            bool ok = nsteps > 0 && wait(q_full, 0, TERR_Q) && wait(&k_full[0], 0, TERR_K);
            if (ok) {
                tc_fence_after();
                if (elect_one()) {
                    for (int i = 0; i < 2 && i < nsteps; ++i) {
                        mma_s(i);
                        mma_commit(&s_full[2 * t + i]);
                    }
                    mma_commit(&k_free[0]);
                }
                __syncwarp();
            }
            // Step i: O += P(i) V, then S(i + 2) over P(i); S(i + 1) is being worked on meanwhile.
            for (int i = 0; i < nsteps && ok; ++i) {
                const bool more = i + 2 < nsteps, even = (i & 1) == 0;
                ok = (!even || wait(&v_full[(i >> 1) & 1], i >> 2, TERR_V)) &&
                     (!even || !more || wait(&k_full[((i + 2) >> 1) & 1], (i + 2) >> 2, TERR_K)) &&
                     wait(&p_full[2 * t + (i & 1)], i >> 1, TERR_P);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    mma_pv(i);
                    if (more) mma_s(i + 2);
                    mma_commit(&s_full[2 * t + (i & 1)]);
                    if (!even) {  // this tile has read values i / 2 and keys i / 2 + 1
                        mma_commit(&v_free[(i >> 1) & 1]);
                        mma_commit(&k_free[((i + 2) >> 1) & 1]);
                    }
                }
                __syncwarp();
            }
        }
    } else {
        // ---- softmax: thread = row ----
        take_regs<kRegsSoftmax>();
        const int t = warp >> 2;
        const int r = row0 + static_cast<int>(threadIdx.x);  // t * 128 + row of the tile
        const bool live = r < R;
        if (t < nq) {
            const int i = r / G;
            const int64_t head = kv * static_cast<int64_t>(G) + r % G;
            const int last = live ? kv_last(a, q, i) : -1, first = live ? kv_first(a, last) : 0;
            float row_c = 1.f;
            {  // the warp's 32 rows as f16; bf16 rows are brought to [1, 2) by a power of two, undone by row_c
                constexpr int kLanes = D / 8, kRowsStep = 32 / kLanes, kBatch = 8;  // lanes a row, rows a step, steps a batch (4: 0.8 % slower on a whole prompt, 16: 0.5 %)
                const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.qs.token + head * a.qs.head;
                const int part = lane % kLanes;
                for (int step0 = 0; step0 < 32 / kRowsStep; step0 += kBatch) {
                    uint4 raw[kBatch];
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        const int row = (step0 + k) * kRowsStep + lane / kLanes;
                        const int64_t from = __shfl_sync(0xffffffffu, at, row) + part * 8;
                        const bool there = __shfl_sync(0xffffffffu, live, row);
                        const uint16_t *src = static_cast<const uint16_t *>(a.q) + from;
                        raw[k] = make_uint4(0u, 0u, 0u, 0u);
                        if (there && a.qs.aligned16) {
                            raw[k] = *reinterpret_cast<const uint4 *>(src);
                        } else if (there) {
                            uint16_t *e = reinterpret_cast<uint16_t *>(&raw[k]);
#pragma unroll
                            for (int n = 0; n < 8; ++n) e[n] = src[n];
                        }
                    }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (a.q_bf16) {
                            const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
                            float x[8];
#pragma unroll
                            for (int n = 0; n < 4; ++n) x[2 * n] = __uint_as_float(u[n] << 16), x[2 * n + 1] = __uint_as_float(u[n] & 0xffff0000u);
                            // largest of the 8 by their bits; where all lanes' are in [2^-4, 2^15] f16 holds the rows as they are,
                            // to half its smallest step, 2^-25, that is 2^-21 of a row's largest element
                            uint32_t most = __vmaxu2(__vmaxu2(u[0] & 0x7fff7fffu, u[1] & 0x7fff7fffu), __vmaxu2(u[2] & 0x7fff7fffu, u[3] & 0x7fff7fffu));
                            most = max(most & 0xffffu, most >> 16);
                            if (!__all_sync(0xffffffffu, most >= 0x3d80u && most <= 0x4700u)) {
#pragma unroll
                                for (int o = kLanes / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                                const int e = min(static_cast<int>(most >> 7), 253);
                                const float down = e ? __int_as_float((254 - e) << 23) : 1.f;
                                const float up = __shfl_sync(0xffffffffu, e ? __int_as_float(e << 23) : 1.f, lane % kRowsStep * kLanes);
                                if (lane / kRowsStep == step0 + k) row_c = up;
#pragma unroll
                                for (int n = 0; n < 8; ++n) x[n] *= down;
                            }
                            __half2 h[4];
#pragma unroll
                            for (int n = 0; n < 4; ++n) h[n] = __floats2half2_rn(x[2 * n], x[2 * n + 1]);
                            raw[k] = *reinterpret_cast<const uint4 *>(h);
                        }
                        if constexpr (kFour) raw[k] = paired(raw[k]);
                        const int row = (warp & 3) * 32 + (step0 + k) * kRowsStep + lane / kLanes;
                        *reinterpret_cast<uint4 *>(smem + C::kQ + t * C::kTile + (part >> 3) * C::kHalf + row * 128 +
                                                   ((part & 7) ^ (row & 7)) * 16) = raw[k];
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const uint32_t base = (static_cast<uint32_t>((warp & 3) * 32) << 16);
            const uint32_t s_col = tmem + base + t * 128, o_col = tmem + base + 256 + t * D;
            float m = -INFINITY, l = 0.f;
            // tokens that some row of this warp does not see
            const int w_lo = row0 + static_cast<int>(threadIdx.x & ~31u), w_hi = min(w_lo + 31, R - 1);
            const int all_end = w_lo < R ? kv_last(a, q, w_lo / G) : 0x7fffffff;
            const int all_begin = w_lo < R ? kv_first(a, kv_last(a, q, w_hi / G)) : 0;
            bool ok = true;
            for (int i = 0; i < nsteps; ++i) {
                const int j = i >> 1, buf = i & 1;
                const uint32_t s_at = s_col + buf * 64;
                ok = warp_wait(&s_full[2 * t + buf], j & 1, a.err, TERR_S) &&
                     (buf != 0 || warp_wait(&sc_full[j % C::kScaleSlots], (j / C::kScaleSlots) & 1, a.err, TERR_K));
                if (!ok) break;
                tc_fence_after();
                uint32_t x[2][32];
                tmem_ld_32x32b_x32(s_at, x[0]);
                tmem_ld_32x32b_x32(s_at + 32, x[1]);
                // a factor of 0 (keys or scale 0) would make NaN of -inf; a tiny one leaves 0 of the other scores
                float fk[4], lv[4], inv_v[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const Scales v = reinterpret_cast<const Scales *>(smem + C::kScales)[(j % C::kScaleSlots) * 8 + buf * 4 + g];
                    fk[g] = fmaxf(v.k * row_c, 1e-37f), lv[g] = v.lv, inv_v[g] = v.inv_v;
                }
                tmem_wait_ld();
                pass32(x[0]);
                pass32(x[1]);
                const int tok = k_begin + i * 64;
                if (tok + 63 > all_end || tok < all_begin) {  // the row sees columns lo .. hi
                    const int hi = last - tok, lo = first - tok;
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (e > hi || e < lo) x[e >> 5][e & 31] = 0xff800000u;
                }
                float top = -INFINITY;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const uint32_t *y = &x[g >> 1][16 * (g & 1)];
                    float mx = __uint_as_float(y[0]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2) mx = max3_nan(mx, __uint_as_float(y[e]), __uint_as_float(y[e + 1]));
                    top = max3_nan(top, fmaf(mx, fk[g], lv[g]), fmaf(__uint_as_float(y[15]), fk[g], lv[g]));
                }
                float alpha = 1.f;
                if (!(top <= m + kLazy)) {  // a score that is NaN or +inf makes l NaN, and the row
                    alpha = ex2_approx(m - top) + (top - top);
                    m = top;
                    l *= alpha;
                }
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    // P_t(i - 1) V is in O_t when the step after this one has its scores
                    ok = warp_wait(&s_full[2 * t + (buf ^ 1)], ((i + 1) >> 1) & 1, a.err, TERR_S);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_col + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st_32x32b_x16(o_col + c, o);
                    }
                }
                const float less = m == -INFINITY ? 0.f : m - kPUp;
                // in sweeps over 8 pairs, so that many exponentials are on their way at once
                float bb[4], sum[4][2];
#pragma unroll
                for (int g = 0; g < 4; ++g) bb[g] = lv[g] - less, sum[g][0] = sum[g][1] = 0.f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e0 = 0; e0 < 16; e0 += 8) {
                        float y[2][8];
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
#pragma unroll
                            for (int g = 0; g < 2; ++g)
                                fma2(y[g][e], y[g][e + 1], __uint_as_float(x[c][16 * g + e0 + e]),
                                     __uint_as_float(x[c][16 * g + e0 + e + 1]), fk[2 * c + g], bb[2 * c + g]);
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                if ((e0 + e) / 2 >= 8 - kPolyPairs) {
                                    exp2_poly(y[g][e], y[g][e + 1]);
                                } else {
                                    y[g][e] = ex2_approx(y[g][e]);
                                    y[g][e + 1] = ex2_approx(y[g][e + 1]);
                                }
                            }
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
#pragma unroll
                            for (int g = 0; g < 2; ++g) {
                                fadd2(sum[2 * c + g][0], sum[2 * c + g][1], sum[2 * c + g][0], sum[2 * c + g][1], y[g][e], y[g][e + 1]);
                                const __half2 h = __floats2half2_rn(y[g][e], y[g][e + 1]);
                                pk[8 * g + (e0 + e) / 2] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                    }
                    tmem_st_32x32b_x16(s_at + 16 * c, pk);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) l = fmaf(sum[g][0] + sum[g][1], inv_v[g], l);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * t + buf]);
            }
            // the last step's O
            if (ok && nsteps > 0) ok = warp_wait(&s_full[2 * t + ((nsteps + 1) & 1)], ((nsteps + 1) >> 1) & 1, a.err, TERR_S);
            if (ok) {
                tc_fence_after();
                const float inv = n_split > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;  // a row that sees no key yields zeros
                const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.ys.token + head * a.ys.head;
                float *to = part_of(split) + (threadIdx.x & 255);  // [dimension][row]: a warp's rows lie together
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    uint32_t o[32];
                    if (nsteps > 0) {
                        tmem_ld_32x32b_x32(o_col + c, o);
                        tmem_wait_ld();
                        pass32(o);
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            v[kFour ? (k >> 1) + (k & 1) * 4 : k] = nsteps > 0 ? __uint_as_float(o[e + k]) * inv : 0.f;
                        if (n_split > 1) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) to[(c + e + k) * C::kRows] = v[k];
                        } else if (live) {
                            kv_store8(a, at + c + e, v);
                        }
                    }
                }
                if (n_split > 1) to[D * C::kRows] = m, to[(D + 1) * C::kRows] = l;
            }
            if (n_split > 1) {
                // The last of the row tile's blocks joins the parts, in their order.  (Here and not behind the roles:
                // the other warps have given their registers away.)
                auto sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(nq * 128) : "memory"); };
                sync();
                if (threadIdx.x == 0) {
                    __threadfence();
                    *tmem_slot = atomicInc(a.done + group, n_split - 1) == static_cast<unsigned>(n_split - 1);
                    __threadfence();
                }
                sync();
                if (*tmem_slot && live) {
                    const int tid = threadIdx.x;
                    float M = -INFINITY, L = 0.f;
                    for (int k = 0; k < n_split; ++k) M = fmaxf(M, __ldcg(part_of(k) + D * C::kRows + tid));
                    for (int k = 0; k < n_split; ++k) {
                        const float mk = __ldcg(part_of(k) + D * C::kRows + tid);
                        L = fmaf(__ldcg(part_of(k) + (D + 1) * C::kRows + tid), mk == M ? 1.f : ex2_approx(mk - M), L);
                    }
                    const float inv = L == 0.f ? 0.f : 1.f / L;
                    const int64_t at = (q.r0 + static_cast<int64_t>(i)) * a.ys.token + head * a.ys.head;
                    for (int d = 0; d < D; d += 32) {
                        float v[4][8];
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e >> 3][e & 7] = 0.f;
#pragma unroll 2
                        for (int k = 0; k < n_split; ++k) {
                            const float *from = part_of(k) + tid;
                            const float mk = __ldcg(from + D * C::kRows), f = (mk == M ? 1.f : ex2_approx(mk - M)) * inv;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                v[e >> 3][e & 7] = fmaf(__ldcg(from + (d + e) * C::kRows), f, v[e >> 3][e & 7]);
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) kv_store8(a, at + d + 8 * e, v[e]);
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int D, typename Args>
cudaError_t launch_tc(const Args &a, cudaStream_t st) {
    using C = Tc<D>;
    void (*const kernel)(Args) = kv_attn_tc_kernel<D, Args>;
    const unsigned bit = 1u << ((std::is_same<Args, Kv4AttnArgs>::value ? kReadyTc4 : kReadyTc) + (D == 64));
    if (!(*a.ready & bit)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        cudaFuncAttributes f;  // the register shares draw on what the block starts with
        e = cudaFuncGetAttributes(&f, kernel);
        if (e != cudaSuccess) return e;
        if (f.numRegs < kRegsStart) return cudaErrorInvalidConfiguration;
        *a.ready |= bit;
    }
    const int64_t units = ((static_cast<int64_t>(a.b.n_rows) * a.group) >> 8) + a.b.n_seqs;
    return launch_after(kernel, dim3(static_cast<unsigned>(units * a.c.heads * a.splits)), C::kThreads, C::kSmem, st, a);
}

template <typename Args>
cudaError_t run(Args &a, int num_sms, cudaStream_t st) {
    const int64_t units = ((static_cast<int64_t>(a.b.n_rows) * a.group) >> 8) + a.b.n_seqs, groups = units * a.c.heads;
    // Parts of the key range: the number that gives the shortest schedule of one block an SM, counted in tiles of 128
    // tokens (about 2 us), a block's start and end as 4 of them and the join of parts as 3.
    const int64_t span = a.window ? std::min(a.b.max_len, static_cast<int64_t>(a.window) + a.b.max_rows + 16) : a.b.max_len;
    const int64_t tiles = std::max((span + 127) / 128, static_cast<int64_t>(1));
    const int64_t most = std::min(kPartFloats / (256 * (a.c.D + 2)) / std::max(groups, static_cast<int64_t>(1)), static_cast<int64_t>(32));
    int64_t splits = 1, least = 0x7fffffffffffffff;
    for (int64_t n = 1; n <= std::max(most, static_cast<int64_t>(1)) && (n == 1 || 2 * n <= tiles); ++n) {
        const int64_t cost = (groups * n + num_sms - 1) / num_sms * ((tiles + n - 1) / n + (n > 1 ? 7 : 4));
        if (cost < least) least = cost, splits = n;
    }
    if (groups * splits > 0x7fffffff) return cudaErrorInvalidValue;
    a.splits = static_cast<int>(splits);
    a.chunk = static_cast<int>((tiles + splits - 1) / splits * 128);
    // with few row tiles a sequence far shorter than max_len is cut finer, into all parts
    a.chunk_short = 2 * groups < num_sms ? std::min(a.chunk, 256) : a.chunk;
    a.short_range = static_cast<int>(span / 2);
    return a.c.D == 64 ? launch_tc<64>(a, st) : launch_tc<128>(a, st);
}

}  // namespace

cudaError_t kv_attn_tc(KvAttnArgs a, int num_sms, cudaStream_t st) { return run(a, num_sms, st); }
cudaError_t kv_attn_tc(Kv4AttnArgs a, int num_sms, cudaStream_t st) { return run(a, num_sms, st); }

}  // namespace b200
