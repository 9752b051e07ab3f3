// kv4_cache.cu -- writing rows of keys and values into the paged 4-bit cache
// and reading them back.
//
// 32 consecutive dimensions of one token's head share a scale d:
//   top = the finite element of largest magnitude (the positive one of two)
//   d = bf16(top / -8), its magnitude at most (2 - 2^-7) 2^124,  code = min(round(x / d), 7) + 8,  value = d (code - 8)
// The quotient is exact, ties go to even, so codes depend on nothing but the
// group's 32 numbers.  d has 8 significant bits and code - 8 at most 3 (or is
// -8), so every value has 11 bits: f16 holds it exactly.
//
// A block takes up to 16 rows of a sequence for some of its slabs (a slab: one
// head's keys, or its values), 8 values a thread and step, four threads a
// group, the tokens of a slab side by side so that their codes leave as one
// run; where the rows lie in the cache is looked up once for all slabs.  2 (f16)
// bytes in and 0.56 out per value, and the other way round on
// reading; neither the memory (a third of the copy's rate) nor the issue slots (62 %)
// are full: 983 and 1200 blocks of the ragged prompts below, at 4 and 5 an SM, are 1.66 and 1.62
// waves, the last one two thirds full.  Fewer instructions shortened it most, so both work on packed 16-bit
// numbers where the type has them:
// - the largest magnitude and its sign by the bits (as whole numbers, the largest
//   magnitude m is a maximum without sign, and the positive one exists if the
//   maximum with sign is m too);
// - of a 16-bit x the quotient x / d (d has 8 significant bits) is n + 1/2 exactly
//   or at least 2^-12 away from it, so rounding x * (1 / d), which is off by less
//   than 2^-19, to multiples of 2^-14 first decides every border exactly (f32: the
//   residual is looked at, see round_quotients);
// - code times d in the row's own type is the value rounded once.
// Measured: ragged prompts of 15643 tokens in all, 8 heads of 128 in f16,
// written and the 19116 then cached read back, 47.6 to 48 us (floor 27.9; f32 rows 82, floor 49.7); one token each of 80 sequences and
// its page back 9.8 us, the host's two calls.  With f32 arithmetic and a look up
// of each slab's pages the prompts took 89 us.
#include <algorithm>
#include <type_traits>

#include "kv4_codes.cuh"
#include "kv_cache.cuh"

namespace b200 {
namespace {

constexpr float kMostScale = 0x1.fep+124f;  // (2 - 2^-7) 2^124, the largest whose 8-fold is finite
constexpr int kThreads = 256, kRowsLog2 = 4, kRows = 1 << kRowsLog2;

template <typename Ptr>
struct RowsArgs {
    Kv4View c;
    KvRows b;
    Ptr x[2];  // rows of keys and values
    RowTensor xs[2];
    int slabs, rows_log2;  // of a block; rows that its items are laid out for
    int *err;
};

// Where a thread's work lies: 8 dimensions of one row, of every so many slabs.
template <typename T, typename Ptr>
struct Place {
    Ptr *row[2];             // its elements of head 0's keys and values
    int64_t at;              // its token in the cache, counted in tokens of slab 0; -1: a bad page
    int chunk;               // its dimensions 8 chunk ...
    int slab, step, end;     // slabs
    bool live;               // it has a row
};

// False if the block has nothing to do; every thread of the block calls this.
template <int D, typename T, typename Args, typename Ptr>
__device__ __forceinline__ bool find_place(const Args &a, Place<T, Ptr> &w) {
    constexpr int kChunkLog2 = D == 64 ? 3 : 4;
    __shared__ int64_t s_at[kRows];
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, true, a.err);
    int64_t local;
    KvSeq q;
    if (!kv_find(a.b, blockIdx.x, 1, kRowsLog2, 1, a.c.page_log2, q, local)) return false;
    if ((local << kRowsLog2) >= q.n || q.len < q.n) return false;
    const int first = static_cast<int>(local) << kRowsLog2, rows = min(q.n - first, kRows);
    if (threadIdx.x < rows) {
        const int pos = q.len - q.n + first + threadIdx.x;
        const int page = kv_page(a.c, a.b, q.s, pos >> a.c.page_log2, a.err);
        s_at[threadIdx.x] = page < 0 ? -1 : ((static_cast<int64_t>(page) * a.c.heads) << a.c.page_log2) + (pos & ((1 << a.c.page_log2) - 1));
    }
    __syncthreads();
    // items of a slab: chunk fastest, then row (of 1 << rows_log2); a block's threads are some slabs' items
    const int i = (threadIdx.x >> kChunkLog2) & ((1 << a.rows_log2) - 1);
    w.chunk = threadIdx.x & ((1 << kChunkLog2) - 1);
    w.live = i < rows;
    w.at = w.live ? s_at[i] : -1;
    w.slab = blockIdx.y * a.slabs + (threadIdx.x >> (kChunkLog2 + a.rows_log2));
    w.step = kThreads >> (kChunkLog2 + a.rows_log2);
    w.end = min(static_cast<int>(blockIdx.y + 1) * a.slabs, 2 * a.c.heads);
#pragma unroll
    for (int k = 0; k < 2; ++k)
        w.row[k] = static_cast<Ptr *>(a.x[k]) + (q.r0 + static_cast<int64_t>(w.live ? first + i : 0)) * a.xs[k].token + w.chunk * 8;
    return true;
}

// The lanes of this one's group, which go through the slabs together (a warp's other groups may have one slab less).
__device__ __forceinline__ unsigned four_lanes() { return 0xfu << (threadIdx.x & 28); }

// The largest magnitude of a group of 32 (8 in each of four neighbouring lanes) as the bits of its type, its sign, and
// whether all are finite; the bits of 16-bit types are compared two at a time.
struct Top {
    float value;  // the element of largest magnitude, the positive one of two
    bool finite;
};
__device__ __forceinline__ Top top_of(const Raw8<float> &r) {
    float high = 0.f, low = 0.f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool f = fabsf(r.v[j]) <= kF32Max;
        finite = finite && f;
        high = fmaxf(high, f ? r.v[j] : 0.f), low = fminf(low, f ? r.v[j] : 0.f);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        high = fmaxf(high, __shfl_xor_sync(four_lanes(), high, o));
        low = fminf(low, __shfl_xor_sync(four_lanes(), low, o));
    }
    return Top{high >= -low ? high : low, finite};
}
template <typename T>
__device__ __forceinline__ Top top_of(const Raw8<T> &r) {
    constexpr uint32_t k = 0x7fff7fffu, bias = 0x80008000u;
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint4 w = *reinterpret_cast<const uint4 *>(&r);
    auto halves = [](uint32_t x) { return max(x & 0xffffu, x >> 16); };
    // magnitudes, and numbers with their sign as whole numbers above 0
    uint32_t m = halves(__vmaxu2(__vmaxu2(w.x & k, w.y & k), __vmaxu2(w.z & k, w.w & k)));
    uint32_t s = halves(__vmaxu2(__vmaxu2(w.x ^ bias, w.y ^ bias), __vmaxu2(w.z ^ bias, w.w ^ bias)));
    const bool finite = m < kInf;
    if (!finite) {
        m = 0, s = 0x8000u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t x = reinterpret_cast<const uint16_t *>(&r)[j];
            if ((x & 0x7fffu) < kInf) m = max(m, x & 0x7fffu), s = max(s, x ^ 0x8000u);
        }
    }
    uint32_t both = m << 16 | s;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) both = __vmaxu2(both, __shfl_xor_sync(four_lanes(), both, o));
    m = both >> 16, s = both & 0xffffu;
    const uint16_t bits = static_cast<uint16_t>(m | ((s ^ 0x8000u) == m ? 0u : 0x8000u));
    return Top{to_f32(*reinterpret_cast<const T *>(&bits)), finite};
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T, bool VEC, int D>
__global__ void __launch_bounds__(kThreads) kv4_write_kernel(const __grid_constant__ RowsArgs<const void *> a) {
    wait_for_stream();
    Place<T, const T> w;
    if (!find_place<D>(a, w)) return;
    uint32_t *const codes[2] = {reinterpret_cast<uint32_t *>(a.c.codes[0]) + w.at * (D / 8) + w.chunk,
                                reinterpret_cast<uint32_t *>(a.c.codes[1]) + w.at * (D / 8) + w.chunk};
    __nv_bfloat16 *const scales[2] = {a.c.scale[0] + w.at * (D / 32) + w.chunk / 4, a.c.scale[1] + w.at * (D / 32) + w.chunk / 4};
    constexpr int kFlight = sizeof(T) == 2 ? 4 : 2;  // slabs whose rows a thread has on their way
    Raw8<T> ahead[kFlight];
    for (; w.slab < w.end; w.slab += kFlight * w.step) {  // a group's four threads are neighbours and go together
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int slab = w.slab + k * w.step;
            const bool which = slab >= a.c.heads;
            if (slab < w.end)
                ahead[k] = raw8<VEC>((which ? w.row[1] : w.row[0]) + (which ? slab - a.c.heads : slab) * (which ? a.xs[1].head : a.xs[0].head));
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int slab = w.slab + k * w.step;
            if (slab >= w.end) break;
            const bool which = slab >= a.c.heads;
            const int head = which ? slab - a.c.heads : slab;
            const Raw8<T> raw = ahead[k];
            const Top top = top_of(raw);
            const float eighth = fabsf(top.value) < kKvSmallest ? 0.f : -0.125f * top.value;
            const __nv_bfloat16 held = __float2bfloat16_rn(fminf(fmaxf(eighth, -kMostScale), kMostScale));
            const float d = to_f32(held), s = fabsf(d);
            if (w.at < 0) continue;
            uint32_t packed = 0x88888888u;
            if (s > 0.f) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = to_f32(raw.v[j]);
                if (!top.finite) {
                    const float end = 8.f * s;
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = v[j] == v[j] ? fminf(fmaxf(v[j], -end), end) : 0.f;
                }
                const float inv = rcp_approx(d);
                uint32_t c[8];  // low 16 bits: code + 8, 0 to 16
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)  // 768 + quotient in steps of 2^-14, then 12582920 + quotient in steps of 1
                        c[j] = __float_as_uint(__fadd_rn(__fmaf_rn(v[j], inv, 768.f), 12582920.f - 768.f));
                } else {
                    int n[8];
                    if (d < 0.f) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = -v[j];
                    }
                    round_quotients(v, s, fabsf(inv), n);
#pragma unroll
                    for (int j = 0; j < 8; ++j) c[j] = static_cast<uint32_t>(n[j] + 8);
                }
                uint32_t two[4];  // codes j and j + 4
#pragma unroll
                for (int j = 0; j < 4; ++j) two[j] = __vminu2(__byte_perm(c[j], c[j + 4], 0x5410), 0x000f000fu);
                packed = (two[0] + two[1] * 16u) + (two[2] + two[3] * 16u) * 256u;
            }
            const uint32_t to = static_cast<uint32_t>(head) << a.c.page_log2;  // tokens
            (which ? codes[1] : codes[0])[to * (D / 8)] = packed;
            if ((w.chunk & 3) == 0) (which ? scales[1] : scales[0])[to * (D / 32)] = held;
        }
    }
}

// 8 codes times d as numbers of type T.
__device__ __forceinline__ void widen8(uint32_t w, __nv_bfloat16 held, Raw8<float> &r) {
    const float d = to_f32(held);
#pragma unroll
    for (int j = 0; j < 8; ++j)  // 0x4b00000u is 2^23 + u
        r.v[j] = __fmul_rn(__fsub_rn(__uint_as_float(and_or(w >> (4 * j), 15u, 0x4b000000u)), 8388616.f), d);
}
template <typename T2>
__device__ __forceinline__ uint4 in_order(const T2 (&p)[4]) {  // pairs (j, j + 4) to 8 in a row
    const uint32_t *u = reinterpret_cast<const uint32_t *>(p);
    return make_uint4(__byte_perm(u[0], u[1], 0x5410), __byte_perm(u[2], u[3], 0x5410), __byte_perm(u[0], u[1], 0x7632), __byte_perm(u[2], u[3], 0x7632));
}
__device__ __forceinline__ void widen8(uint32_t w, __nv_bfloat16 held, Raw8<__nv_bfloat16> &r) {
    const __nv_bfloat162 less = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308)), d = __halves2bfloat162(held, held);
    __nv_bfloat162 p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // 0x430u is 128 + u
        const uint32_t x = and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);
        p[j] = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&x), less), d);
    }
    *reinterpret_cast<uint4 *>(&r) = in_order(p);
}
__device__ __forceinline__ void widen8(uint32_t w, __nv_bfloat16 held, Raw8<__half> &r) {
    const float d = to_f32(held);
    if (fabsf(d) >= 6.103515625e-5f && fabsf(d) <= 8160.f) {  // a normal f16 number, and so are all codes times it
        const __half2 by = __float2half2_rn(d);
        uint32_t c[4];
        codes4(w, c);
        __half2 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __hmul2(*reinterpret_cast<const __half2 *>(&c[j]), by);
        *reinterpret_cast<uint4 *>(&r) = in_order(p);
        return;
    }
    Raw8<float> f;
    widen8(w, held, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = __float2half_rn(f.v[j]);
}

template <typename T, bool VEC, int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const __grid_constant__ RowsArgs<void *> a) {
    wait_for_stream();
    Place<T, T> w;
    if (!find_place<D>(a, w) || !w.live) return;
    const int64_t at = max(w.at, static_cast<int64_t>(0));
    const uint32_t *const codes[2] = {reinterpret_cast<const uint32_t *>(a.c.codes[0]) + at * (D / 8) + w.chunk,
                                      reinterpret_cast<const uint32_t *>(a.c.codes[1]) + at * (D / 8) + w.chunk};
    const __nv_bfloat16 *const scales[2] = {a.c.scale[0] + at * (D / 32) + w.chunk / 4, a.c.scale[1] + at * (D / 32) + w.chunk / 4};
    constexpr int kFlight = 4;  // slabs whose codes a thread has on their way
    for (; w.slab < w.end; w.slab += kFlight * w.step) {
        uint32_t packed[kFlight];
        __nv_bfloat16 held[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int slab = w.slab + k * w.step;
            const bool which = slab >= a.c.heads;
            const uint32_t from = static_cast<uint32_t>(which ? slab - a.c.heads : slab) << a.c.page_log2;  // tokens
            packed[k] = 0x88888888u, held[k] = __ushort_as_bfloat16(0);  // a bad page reads as zeros
            if (slab < w.end && w.at >= 0) packed[k] = (which ? codes[1] : codes[0])[from * (D / 8)], held[k] = (which ? scales[1] : scales[0])[from * (D / 32)];
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
            const int slab = w.slab + k * w.step;
            if (slab >= w.end) break;
            const bool which = slab >= a.c.heads;
            const int head = which ? slab - a.c.heads : slab;
            Raw8<T> r;
            widen8(packed[k], held[k], r);
            T *y = (which ? w.row[1] : w.row[0]) + head * (which ? a.xs[1].head : a.xs[0].head);
            if constexpr (VEC) {
#pragma unroll
                for (int e = 0; e < static_cast<int>(sizeof(T) / 2); ++e) reinterpret_cast<uint4 *>(y)[e] = reinterpret_cast<const uint4 *>(&r)[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = r.v[e];
            }
        }
    }
}

// Checks and the launch, which the two directions share.
template <typename Ptr>
int run(const char *op, sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch, int type, Ptr k,
        const int64_t *k_nb, Ptr v, const int64_t *v_nb, bool written, void (*const (&kernels)[3][2][2])(RowsArgs<Ptr>)) {
    auto *be = reinterpret_cast<Backend *>(h);
    RowsArgs<Ptr> a;
    if (!kv_views(op, cache, batch, a.c, a.b)) return SAM3B200_STATUS_FAILED;
    const int bytes = type_bytes(type);
    if (!k || !v || !bytes || reinterpret_cast<uintptr_t>(k) % bytes || reinterpret_cast<uintptr_t>(v) % bytes) {
        if (!k || !v) set_error("%s: null argument", op);
        else set_error("%s: unsupported type %d (F32=0, F16=1, BF16=30) or unaligned rows", op, type);
        return SAM3B200_STATUS_FAILED;
    }
    a.x[0] = k, a.x[1] = v;
    a.xs[0] = row_tensor(k, type, k_nb, a.c.heads, a.c.D);
    a.xs[1] = row_tensor(v, type, v_nb, a.c.heads, a.c.D);
    if (!rows_ok(op, "k", a.xs[0], a.b.n_rows, a.c.heads, a.c.D, written) || !rows_ok(op, "v", a.xs[1], a.b.n_rows, a.c.heads, a.c.D, written))
        return SAM3B200_STATUS_FAILED;
    if (!be) {
        set_error("%s: null backend", op);
        return SAM3B200_STATUS_FAILED;
    }
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return SAM3B200_STATUS_SUCCESS;
    a.err = be->err;
    DeviceScope dev(be->device);
    a.rows_log2 = 0;
    while (1 << a.rows_log2 < std::min(a.b.max_rows, kRows)) ++a.rows_log2;
    const int per_slab = a.c.D / 8 << a.rows_log2;
    // slabs of a thread (us, ragged prompts written and read back: 4 slabs 54.7, 8 48.9, 16 47.6), fewer where the rows alone
    // do not give every SM its blocks
    const int units = (a.b.n_rows >> kRowsLog2) + a.b.n_seqs, steps = units >= 4 * be->num_sms ? 16 : 4;
    a.slabs = std::min(std::max(steps * kThreads / per_slab, 1), 2 * a.c.heads);
    const dim3 grid(units, (2 * a.c.heads + a.slabs - 1) / a.slabs);
    const int t = type == SAM3B200_TYPE_F32 ? 0 : type == SAM3B200_TYPE_F16 ? 1 : 2;
    const cudaError_t e = launch_after(kernels[t][a.xs[0].aligned16 && a.xs[1].aligned16][a.c.D == 128], grid, kThreads, 0, be->stream, a);
    be->count();
    return cuda_ok(e, op) ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int sam3b200_kv4_write(sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch,
                                  int type, const void *k, const int64_t *k_nb, const void *v, const int64_t *v_nb) {
    return run<const void *>("kv4_write", h, cache, batch, type, k, k_nb, v, v_nb, false,
                             {{{kv4_write_kernel<float, false, 64>, kv4_write_kernel<float, false, 128>}, {kv4_write_kernel<float, true, 64>, kv4_write_kernel<float, true, 128>}},
                              {{kv4_write_kernel<__half, false, 64>, kv4_write_kernel<__half, false, 128>}, {kv4_write_kernel<__half, true, 64>, kv4_write_kernel<__half, true, 128>}},
                              {{kv4_write_kernel<__nv_bfloat16, false, 64>, kv4_write_kernel<__nv_bfloat16, false, 128>}, {kv4_write_kernel<__nv_bfloat16, true, 64>, kv4_write_kernel<__nv_bfloat16, true, 128>}}});
}

extern "C" int sam3b200_kv4_read(sam3b200_backend *h, const sam3b200_kv4_cache *cache, const sam3b200_kv_batch *batch,
                                 int type, void *k, const int64_t *k_nb, void *v, const int64_t *v_nb) {
    return run<void *>("kv4_read", h, cache, batch, type, k, k_nb, v, v_nb, true,
                       {{{kv4_read_kernel<float, false, 64>, kv4_read_kernel<float, false, 128>}, {kv4_read_kernel<float, true, 64>, kv4_read_kernel<float, true, 128>}},
                        {{kv4_read_kernel<__half, false, 64>, kv4_read_kernel<__half, false, 128>}, {kv4_read_kernel<__half, true, 64>, kv4_read_kernel<__half, true, 128>}},
                        {{kv4_read_kernel<__nv_bfloat16, false, 64>, kv4_read_kernel<__nv_bfloat16, false, 128>}, {kv4_read_kernel<__nv_bfloat16, true, 64>, kv4_read_kernel<__nv_bfloat16, true, 128>}}});
}
