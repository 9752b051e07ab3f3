// kv_attn_tc.cu -- attention over the paged 8-bit cache for many query rows a
// kv head (prompts, parts of prompts, cross attention), on the
// 5th-generation tensor cores.
//
// A block owns 256 query rows of one kv head (the group's query heads times
// tokens) as two tiles of 128 and streams the keys in tiles of 128 tokens.
//   warps 0-7:  softmax, one thread a row; warps 0-3 tile 0, 4-7 tile 1;
//   warps 8-11: read the codes (16 bytes a lane straight from the pages, the
//               next tile's in registers meanwhile) and write them as f16,
//               exactly, into 128-byte-swizzled shared memory, and each 16
//               tokens' scales beside them;
//   warp 12:    issues the MMAs (13-15 only give their registers away): S_t(j) = Q_t K_j^T, and once softmax t has
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

// Registers a thread after the split: a block starts with 128 for each of its
// four warpgroups, and the shares may not add up to more.
constexpr int kRegsStart = 128, kRegsSoftmax = 176, kRegsCodes = 104, kRegsMma = 56;
static_assert(2 * kRegsSoftmax + kRegsCodes + kRegsMma <= 4 * kRegsStart, "register shares");

constexpr int kPolyPairs = 2;  // of 8 pairs of weights, those whose exponential runs on the FMA pipe

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

// 2^y of two numbers on the FMA pipe, for y <= 127: the magic sum splits y into an integer n and f in [-1/2, 1/2], a
// cubic with the least largest relative error there (7.5e-5, found by Remez exchange) gives 2^f, n goes to the exponent.
// Below -126: 2^-126.
__device__ __forceinline__ void exp2_poly(float &y0, float &y1) {
    y0 = fmaxf(y0, -126.f), y1 = fmaxf(y1, -126.f);
    float n0, n1, f0, f1;
    fadd2(n0, n1, y0, y1, 12582912.f, 12582912.f);
    fadd2(f0, f1, n0, n1, -12582912.f, -12582912.f);
    fadd2(f0, f1, y0, y1, -f0, -f1);
    float a0, a1, b0 = 0.69326097f, b1 = 0.69326097f, c0 = 0.99992806f, c1 = 0.99992806f;
    fma2(a0, a1, f0, f1, 0.05517167f, 0.24261113f);
    ffma2(b0, b1, a0, a1, f0, f1);
    ffma2(c0, c1, b0, b1, f0, f1);
    y0 = __int_as_float((__float_as_int(n0) << 23) + __float_as_int(c0));
    y1 = __int_as_float((__float_as_int(n1) << 23) + __float_as_int(c1));
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
    uint64_t *p_full = s_full + 2;       // [2 tiles] phase j: O_t is rescaled and P_t(j) is there
    // Scales of tile j, in slot j % 4: written again at tile j + 4, which waits for P_t(j + 1), so a slow softmax
    // warp never sees its phase pass by (keys may run two tiles ahead of it: it must not wait on k_full).
    uint64_t *sc_full = p_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sc_full + C::kScaleSlots);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kv = blockIdx.x % a.c.heads, G = a.group;
    if (blockIdx.x == 0) kv_check(a.b, a.c.page_log2, false, a.err);
    int64_t local;
    KvSeq q;  // late rows, with the most keys, come first
    if (!kv_find(a.b, (gridDim.x - 1 - blockIdx.x) / a.c.heads, G, 8, 1, a.c.page_log2, q, local)) return;
    const int s = q.s;
    const int R = q.n * G;  // the host keeps n_rows * G below 2^31
    if (local * C::kRows >= R) return;
    const int row0 = static_cast<int>(local) * C::kRows, i_lo = row0 / G, i_hi = (min(row0 + C::kRows, R) - 1) / G;
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
        for (int i = 0; i < C::kScaleSlots; ++i) mbar_init(&sc_full[i], 4);
        fence_mbar_init();
    }
    if (warp == 12) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;  // all columns are this block's, so they start at 0

    if (warp >= 8 && warp < 12) {
        // ---- codes -> f16 ----
        give_regs<kRegsCodes>();
        // warp w widens tokens 32 w ... 32 w + 31 of each tile: two runs of 16, each in one page
        const int w = warp - 8;
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
                if (j < ntiles && tok < k_end) r.p[g] = __ldg(a.b.table + s * a.b.table_width + (tok >> a.c.page_log2));
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
        auto fetch = [&](int which, int j, const Pages &pg, uint4 (&x)[kPer]) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int in_page = (k_begin + j * C::kKeys + w * 32 + g * 16) & ((1 << a.c.page_log2) - 1);
                const int8_t *from = a.c.codes[which] + kv_slab(a.c, max(pg.p[g], 0), kv) + static_cast<int64_t>(in_page) * D + own;
#pragma unroll
                for (int i = 0; i < kPer / 2; ++i) {
                    uint4 &v = x[g * (kPer / 2) + i];
                    v = make_uint4(0u, 0u, 0u, 0u);
                    if (pg.p[g] >= 0) v = __ldg(reinterpret_cast<const uint4 *>(from + i * kTokens * D));
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
        auto publish = [&](uint64_t *bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // Pair p of the pipeline is keys p and values p - 1; keys j + 1 and values j reuse the slots of pair j - 1.
        // Codes and scales are loaded a tile ahead.
        Pages pg = checked(0, lookup(0)), pg_next = checked(1, lookup(1)), raw = lookup(2);
        fetch(0, 0, pg, kx);
        fetch_scales(pg);
        fetch(1, 0, pg, vx);
        if (ntiles > 0) {
            put(smem + C::kK, kx);
            put_scales(0);
            publish(&k_full[0]);
            if (lane == 0) mbar_arrive(&sc_full[0]);
            fetch(0, 1, pg_next, kx);
            fetch_scales(pg_next);
        }
        for (int j = 0; j < ntiles; ++j) {
            const Pages pg_then = checked(j + 2, raw);
            raw = lookup(j + 3);
            if (j >= 1 && !warp_wait(&pair_free[(j - 1) & 1], ((j - 1) >> 1) & 1, a.err, TERR_FREE))
                break;
            put(smem + C::kV + (j & 1) * C::kTile, vx);
            publish(&v_full[j & 1]);
            fetch(1, j + 1, pg_next, vx);
            if (j + 1 < ntiles) {
                put(smem + C::kK + ((j + 1) & 1) * C::kTile, kx);
                put_scales(j + 1);
                publish(&k_full[(j + 1) & 1]);
                if (lane == 0) mbar_arrive(&sc_full[(j + 1) % C::kScaleSlots]);
                fetch(0, j + 2, pg_then, kx);
                fetch_scales(pg_then);
            }
            pg_next = pg_then;
        }
    } else if (warp >= 12) {
        // ---- MMA issuer ----
        give_regs<kRegsMma>();
        if (warp == 12) {
            constexpr uint32_t idesc_s = idesc_f16_f32(128, C::kKeys);
            constexpr uint32_t idesc_pv = idesc_f16_f32(128, D) | (1u << 16);  // B is N-major
            // Descriptors advance by constants (addresses in 16 bytes), so that an MMA costs its issuer little.
            const uint64_t q_desc = sw128_kmajor_desc(smem_u32(smem + C::kQ)), k_desc = sw128_kmajor_desc(smem_u32(smem + C::kK)),
                           v_desc = sw128_nmajor_desc(smem_u32(smem + C::kV), C::kHalf);
            auto mma_s = [&](int t, int j) {
                const uint64_t qd = q_desc + t * (C::kTile >> 4), kd = k_desc + (j & 1) * (C::kTile >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = ((k >> 2) * C::kHalf + (k & 3) * 32) >> 4;
                    mma_f16(tmem + t * 128, qd + off, kd + off, idesc_s, k > 0);
                }
            };
            auto mma_pv = [&](int t, int j) {
                const uint64_t vd = v_desc + (j & 1) * (C::kTile >> 4);
#pragma unroll
                for (int k = 0; k < C::kKeys / 16; ++k)
                    mma_f16_ts(tmem + 256 + t * D, tmem + t * 128 + k * 8, vd + (k * 2048 >> 4), idesc_pv, j > 0 || k > 0);
            };
            auto wait = [&](uint64_t *bar, int phase, int code) {
                return warp_wait(bar, phase & 1, a.err, code);
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
                ok = wait(&v_full[j & 1], j >> 1, TERR_V);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (t >= nq || !ok) break;
                    ok = (!more || t > 0 || wait(&k_full[(j + 1) & 1], (j + 1) >> 1, TERR_K)) && wait(&p_full[t], j, TERR_P);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_pv(t, j);
                        if (more) mma_s(t, j + 1);
                        mma_commit(&s_full[t]);
                        if (more && t == nq - 1) mma_commit(&pair_free[(j + 1) & 1]);
                    }
                    __syncwarp();
                }
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
                constexpr int kLanes = D / 8, kRowsStep = 32 / kLanes, kBatch = 4;  // lanes a row, rows a step, steps a batch
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
                            float x[8], top = 0.f;
                            const uint32_t u[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
                            for (int n = 0; n < 4; ++n) {
                                x[2 * n] = __uint_as_float(u[n] << 16);
                                x[2 * n + 1] = __uint_as_float(u[n] & 0xffff0000u);
                                top = fmaxf(top, fmaxf(fabsf(x[2 * n]), fabsf(x[2 * n + 1])));
                            }
#pragma unroll
                            for (int o = kLanes / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            const int e = min((__float_as_int(top) >> 23) & 0xff, 253);
                            const float down = e ? __int_as_float((254 - e) << 23) : 1.f;
                            const float up = __shfl_sync(0xffffffffu, e ? __int_as_float(e << 23) : 1.f, lane % kRowsStep * kLanes);
                            if (lane / kRowsStep == step0 + k) row_c = up;
                            __half2 h[4];
#pragma unroll
                            for (int n = 0; n < 4; ++n) h[n] = __floats2half2_rn(x[2 * n] * down, x[2 * n + 1] * down);
                            raw[k] = *reinterpret_cast<const uint4 *>(h);
                        }
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
            for (int j = 0; j < ntiles; ++j) {
                ok = warp_wait(&s_full[t], j & 1, a.err, TERR_S) &&
                     warp_wait(&sc_full[j % C::kScaleSlots], (j / C::kScaleSlots) & 1, a.err, TERR_K);
                if (!ok) break;
                tc_fence_after();
                // a factor of 0 (keys or scale 0) would make NaN of -inf; a tiny one leaves 0 of the other scores
                float fk[8], lv[8], inv_v[8];
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const Scales v = reinterpret_cast<const Scales *>(smem + C::kScales)[(j % C::kScaleSlots) * 8 + g];
                    fk[g] = fmaxf(v.k * row_c, 1e-37f), lv[g] = v.lv, inv_v[g] = v.inv_v;
                }
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
                // columns 64 ... 127, then 0 ... 63, which stay in registers: P goes over columns that were read last
                float top = -INFINITY;
                uint32_t x[2][32];
#pragma unroll
                for (int half = 1; half >= 0; --half) {
                    tmem_ld_32x32b_x32(s_col + 64 * half, x[0]);
                    tmem_ld_32x32b_x32(s_col + 64 * half + 32, x[1]);
                    tmem_wait_ld();
                    pass32(x[0]);
                    pass32(x[1]);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const uint32_t *y = &x[g >> 1][16 * (g & 1)];
                        float mx = __uint_as_float(y[0]);
#pragma unroll
                        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, __uint_as_float(y[e]));
                        top = fmaxf(top, fmaf(mx, fk[4 * half + g], lv[4 * half + g]));
                    }
                }
                float alpha = 1.f;
                if (top > m + kLazy) {
                    alpha = ex2_approx(m - top);
                    m = top;
                    l *= alpha;
                }
                if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {  // S_t(j) being there, P_t(j - 1) V_(j - 1) is in O_t
                        uint32_t o[16];
                        tmem_ld_32x32b_x16(o_col + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st_32x32b_x16(o_col + c, o);
                    }
                }
                const float less = m == -INFINITY ? 0.f : m - kPUp;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    // in three sweeps, so that 32 exponentials are on their way at once
                    float y[32];
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        fma2(y[e], y[e + 1], __uint_as_float(x[c & 1][e]), __uint_as_float(x[c & 1][e + 1]), fk[2 * c + e / 16],
                             lv[2 * c + e / 16] - less);
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        if (e / 2 % 8 >= 8 - kPolyPairs) {
                            exp2_poly(y[e], y[e + 1]);
                        } else {
                            y[e] = ex2_approx(y[e]);
                            y[e + 1] = ex2_approx(y[e + 1]);
                        }
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        float s0 = 0.f, s1 = 0.f;
#pragma unroll
                        for (int e = 16 * g; e < 16 * g + 16; e += 2) {
                            fadd2(s0, s1, s0, s1, y[e], y[e + 1]);
                            const __half2 h = __floats2half2_rn(y[e], y[e + 1]);
                            pk[e / 2] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                        l = fmaf(s0 + s1, inv_v[2 * c + g], l);
                    }
                    tmem_st_32x32b_x16(s_col + 16 * c, pk);
                    if (c > 0 && c < 3) {
                        tmem_wait_ld();
                        pass32(x[(c + 1) & 1]);
                    }
                    if (c < 2) tmem_ld_32x32b_x32(s_col + 64 + 32 * c, x[c]);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t]);
            }
            if (ok && ntiles > 0) ok = warp_wait(&s_full[t], ntiles & 1, a.err, TERR_S);
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
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int D>
cudaError_t launch_tc(const KvAttnArgs &a, int64_t units, cudaStream_t st) {
    using C = Tc<D>;
    if (!(*a.ready & (1u << (16 + (D == 64))))) {
        cudaError_t e = cudaFuncSetAttribute(kv_attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
        if (e != cudaSuccess) return e;
        cudaFuncAttributes f;  // the register shares draw on what the block starts with
        e = cudaFuncGetAttributes(&f, kv_attn_tc_kernel<D>);
        if (e != cudaSuccess) return e;
        if (f.numRegs < kRegsStart) return cudaErrorInvalidConfiguration;
        *a.ready |= 1u << (16 + (D == 64));
    }
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
