// kv_cache.cu -- writing rows of keys and values into the paged 8-bit cache
// and reading them back.
//
// A page holds the codes of 16 to 128 consecutive tokens of one sequence for
// each kv head, with one f32 scale s per (page, head): value = code s.
// Writing rows into a page takes
//   s = max(s_old, fl32(amax c))         c = fl32(1 / 127), amax over the finite new values,
//                                        s_old = 0 where the page held no token
//   code = round(x / s)                  of the exact quotient, ties to even
// and rounds the page's older codes again, round(code s_old / s), if s grew.
// Both roundings are decided exactly, so the codes do not depend on how the
// rows of a prompt are cut into calls' blocks or on the order of anything.
//
// A block owns one page of a sequence for several of its slabs (a slab: one
// head's keys, or its values), so that finding the page is paid once; W of
// its 8 warps share a slab.  The new rows of a slab are read once into
// registers, their largest magnitude is reduced over the W warps, and the
// codes are written from the registers; W follows from the rows that a call
// can put into one page, 1 for steps of single tokens.  Bound by memory: 2
// (f16) bytes in and 1 out per value, and the other way round on reading.
//
// Measured: ragged prompts of 5 sequences, pages of 16, 8 heads of 128 in f16,
// written and read back in 44 us, 4.3 TB/s (kernels 26 and 23 us: issue 61 and
// 47 %, about 20 and 12 instructions a value; a block's start, 2 us of
// dependent loads, is the rest).  64 sequences of one token each, written and
// their last pages read back: 9.7 us, on the device as on the host (two
// launches).
#include <algorithm>

#include "kv_cache.cuh"

namespace b200 {
namespace {

constexpr float kF32Max = 3.402823466e38f;

// round(x / s), ties to even, for finite |x| <= 127.5 s, s a normal f32, as
// the low bytes of c.  The magic sum rounds x * inv (inv ~ 1 / s) to an
// integer q that is at most one off; r = x - q s is exact wherever |r| is near
// s / 2 (x and q s are multiples of the smaller of their units, and r needs no
// more bits than s), so comparing it with s / 2 tells on which side of the
// border x lies.  The largest |r| of 8 values decides whether any is looked
// at again.
__device__ __forceinline__ void round_quotients(const float (&x)[8], float s, float inv, int (&c)[8]) {
    float far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float m = __fmaf_rn(x[j], inv, 12582912.f);
        c[j] = __float_as_int(m);
        far = fmaxf(far, fabsf(__fmaf_rn(-__fsub_rn(m, 12582912.f), s, x[j])));
    }
    const float h = 0.5f * s;
    if (far < h) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float r = __fmaf_rn(-__fsub_rn(__int_as_float(c[j]), 12582912.f), s, x[j]);
        if (fabsf(r) > h || (fabsf(r) == h && (c[j] & 1))) c[j] += r > 0.f ? 1 : -1;
    }
}

// The low bytes of four numbers.
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

constexpr int kWarps = 8, kThreads = kWarps * 32;

struct WriteArgs {
    KvView c;
    KvRows b;
    const void *x[2];
    RowTensor xs[2];
    int *err;
};

// 8 values as they come.
template <typename T>
struct alignas(16) Raw8 {
    T v[8];
};

template <bool VEC, typename T>
__device__ __forceinline__ Raw8<T> raw8(const T *p) {
    Raw8<T> r;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
            reinterpret_cast<uint4 *>(&r)[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = p[i];
    }
    return r;
}

// Largest magnitude of 8 values by the bits, as those of an f32: infinities and NaN are above all numbers and show.
__device__ __forceinline__ uint32_t top_bits(const Raw8<float> &r) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(fabsf(r.v[j])));
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw8<T> &r) {  // 16-bit types, two at a time
    const uint4 w = *reinterpret_cast<const uint4 *>(&r);
    constexpr uint32_t k = 0x7fff7fffu;
    uint32_t m = __vmaxu2(__vmaxu2(w.x & k, w.y & k), __vmaxu2(w.z & k, w.w & k));
    m = max(m & 0xffffu, m >> 16);
    const uint16_t h = static_cast<uint16_t>(m);
    return __float_as_uint(to_f32(*reinterpret_cast<const T *>(&h)));
}

// Grid (units of one page, groups of kWarps / W slabs); slab = head + heads * (0 keys, 1 values).
// PER: groups of 8 values that a thread holds.
template <typename T, bool VEC, int W, int PER = 4>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ WriteArgs a) {
    __shared__ float wmax[kWarps];
    wait_for_stream();
    const int D = a.c.D, d_log2 = D == 64 ? 6 : 7;
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, true, a.err);
    int64_t local;
    KvSeq q;
    if (!kv_find(a.b, blockIdx.x, 1, a.c.page_log2, 2, a.c.page_log2, q, local)) return;
    const int begin = q.len - q.n;  // first new position
    if (q.n == 0 || begin < 0) return;
    const int64_t i = (begin >> a.c.page_log2) + local;
    const int64_t p0 = i << a.c.page_log2;
    if (p0 >= q.len) return;
    const int page = kv_page(a.c, a.b, q.s, i, a.err);
    if (page < 0) return;
    const int lo = static_cast<int>(max(begin - p0, static_cast<int64_t>(0)));  // first new token of the page
    const int hi = static_cast<int>(min(q.len - p0, static_cast<int64_t>(1) << a.c.page_log2));
    const int warp = threadIdx.x >> 5, slab = blockIdx.y * (kWarps / W) + warp / W;
    const bool there = slab < 2 * a.c.heads;
    const int w = slab >= a.c.heads, head = there ? slab - w * a.c.heads : 0;
    int8_t *codes = a.c.codes[w] + kv_slab(a.c, page, head);
    float *scale = a.c.scale[w] + static_cast<int64_t>(page) * a.c.heads + head;
    const T *x = static_cast<const T *>(a.x[w]) + head * a.xs[w].head + (q.r0 + p0 - begin) * a.xs[w].token;

    const int first = lo * D, end = there ? hi * D : 0, thread = (warp % W) * 32 + (threadIdx.x & 31);
    Raw8<T> raw[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int e = first + (k * W * 32 + thread) * 8;
        if (e < end) raw[k] = raw8<VEC>(x + (e >> d_log2) * a.xs[w].token + (e & (D - 1)));
    }
    const float held = there && lo > 0 ? *scale : 0.f;
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (first + (k * W * 32 + thread) * 8 < end) bits = max(bits, top_bits(raw[k]));
    const bool finite = bits < 0x7f800000u;
    float amax = finite ? __uint_as_float(bits) : 0.f;
    if (!finite) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (first + (k * W * 32 + thread) * 8 >= end) continue;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float m = fabsf(to_f32(raw[k].v[j]));
                amax = fmaxf(amax, m <= kF32Max ? m : 0.f);
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (W > 1) {
        if ((threadIdx.x & 31) == 0) wmax[warp] = amax;
        __syncthreads();  // also: every thread of the slab has read the old scale
#pragma unroll
        for (int j = 0; j < W; ++j) amax = fmaxf(amax, wmax[warp / W * W + j]);
    } else {
        __syncwarp();
    }
    const float to = fmaxf(held, amax < kKvSmallest ? 0.f : __fmul_rn(amax, 1.f / 127.f));
    const float inv = to > 0.f ? __frcp_rn(to) : 0.f;
    if (finite) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int e = first + (k * W * 32 + thread) * 8;
            if (e >= end) continue;
            float v[8];
            int c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(raw[k].v[j]), c[j] = 0;
            if (to > 0.f) round_quotients(v, to, inv, c);
            *reinterpret_cast<uint2 *>(codes + e) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
        }
    } else {  // NaN is stored as 0, infinities as the ends
        const float top = fminf(__fmul_rn(127.f, to), kF32Max);
#pragma unroll 1
        for (int e = first + thread * 8; e < end; e += W * 32 * 8) {
            const Raw8<T> r = raw8<VEC>(x + (e >> d_log2) * a.xs[w].token + (e & (D - 1)));
            float v[8];
            int c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = to_f32(r.v[j]);
                v[j] = v[j] == v[j] ? fminf(fmaxf(v[j], -top), top) : 0.f;
                c[j] = 0;
            }
            if (to > 0.f) round_quotients(v, to, inv, c);
            *reinterpret_cast<uint2 *>(codes + e) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
        }
    }
    if (there && thread == 0) *scale = to;
    if (to == held) return;
    for (int e = thread * 8; e < (there ? first : 0); e += W * 32 * 8) {  // older tokens, under the grown scale
        const uint2 old = *reinterpret_cast<const uint2 *>(codes + e);
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // code * held is exact in 64 bits, and no quotient rounds onto a tie
            const int8_t o = static_cast<int8_t>((j < 4 ? old.x : old.y) >> (8 * (j & 3)));
            c[j] = __double2int_rn(static_cast<double>(o) * held / to);
        }
        *reinterpret_cast<uint2 *>(codes + e) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
    }
}

struct ReadArgs {
    KvView c;
    KvRows b;
    void *y[2];
    RowTensor ys[2];
    int slabs;  // of a block
    int *err;
};

// Grid (units of one page, groups of a.slabs slabs); 16 codes a thread and step.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a) {
    wait_for_stream();
    const int D = a.c.D;
    if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0) kv_check(a.b, a.c.page_log2, true, a.err);
    int64_t local;
    KvSeq q;
    if (!kv_find(a.b, blockIdx.x, 1, a.c.page_log2, 2, a.c.page_log2, q, local)) return;
    const int begin = q.len - q.n;
    if (q.n == 0 || begin < 0) return;
    const int64_t i = (begin >> a.c.page_log2) + local;
    const int64_t p0 = i << a.c.page_log2;
    if (p0 >= q.len) return;
    const int page = kv_page(a.c, a.b, q.s, i, a.err);  // bad: zeros
    const int lo = static_cast<int>(max(begin - p0, static_cast<int64_t>(0)));
    const int hi = static_cast<int>(min(q.len - p0, static_cast<int64_t>(1) << a.c.page_log2));
    const int64_t row0 = q.r0 + p0 - begin;
    // 16-byte chunks of a slab, counted over the whole page so that shifts take a number apart
    const int chunk_log2 = D == 64 ? 2 : 3, each_log2 = a.c.page_log2 + chunk_log2;
    const int slab0 = blockIdx.y * a.slabs, slabs = min(a.slabs, 2 * a.c.heads - slab0);
    for (int id = threadIdx.x; id < slabs << each_log2; id += kThreads) {
        const int slab = slab0 + (id >> each_log2), t = (id >> chunk_log2) & ((1 << a.c.page_log2) - 1), d = (id & ((1 << chunk_log2) - 1)) * 16;
        if (t < lo || t >= hi) continue;
        const int w = slab >= a.c.heads, head = slab - w * a.c.heads;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        float scale = 0.f;
        if (page >= 0) {
            raw = *reinterpret_cast<const uint4 *>(a.c.codes[w] + kv_slab(a.c, page, head) + t * D + d);
            scale = a.c.scale[w][static_cast<int64_t>(page) * a.c.heads + head];
        }
        T *y = static_cast<T *>(a.y[w]) + head * a.ys[w].head + (row0 + t) * a.ys[w].token + d;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t u[2] = {(h ? raw.z : raw.x) ^ 0x80808080u, (h ? raw.w : raw.y) ^ 0x80808080u};
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // 2^23 + 128 + code by its bits
                const float m = __uint_as_float(__byte_perm(u[j >> 2], 0x4b000000u, 0x7550 | (j & 3)));
                v[j] = __fmul_rn(__fsub_rn(m, 8388736.f), scale);
            }
            store8<VEC>(y + 8 * h, v);
        }
    }
}

template <typename T, bool VEC>
cudaError_t launch_write(const WriteArgs &a, cudaStream_t st) {
    // values that a call can put into one slab of a page, 1024 a warp
    const int most = std::min(1 << a.c.page_log2, a.b.max_rows) * a.c.D;
    const int units = (a.b.n_rows >> a.c.page_log2) + 2 * a.b.n_seqs;
    auto grid = [&](int w) { return dim3(units, (2 * a.c.heads + kWarps / w - 1) / (kWarps / w)); };
    auto go = [&](auto *kernel, int w) { return launch_after(kernel, grid(w), kThreads, 0, st, a); };
    if (most <= 1024) return go(kv_write_kernel<T, VEC, 1>, 1);
    if (most <= 2048) return go(kv_write_kernel<T, VEC, 2>, 2);
    if (most <= 4096) return go(kv_write_kernel<T, VEC, 4>, 4);
    if (most <= 8192) return go(kv_write_kernel<T, VEC, 8>, 8);
    return go(kv_write_kernel<T, VEC, 8, 8>, 8);
}

}  // namespace

bool rows_ok(const char *op, const char *what, const RowTensor &t, int64_t rows, int64_t heads, int64_t D, bool written) {
    const int64_t most = int64_t(1) << 40;
    bool ok = t.token >= 0 && t.head >= 0 && t.token < most && t.head < most;
    if (ok && written)  // no element twice: one of the two strides steps over all that the other reaches
        ok = (t.token >= (heads - 1) * t.head + D || rows == 1) && (t.head >= D || heads == 1);
    if (ok || rows <= 0) return true;
    if (written && t.token >= D && t.head >= (rows - 1) * t.token + D) return true;
    set_error("%s: bad strides of %s: token %lld, head %lld elements", op, what, (long long)t.token, (long long)t.head);
    return false;
}

bool kv_views(const char *op, const sam3b200_kv_cache *c, const sam3b200_kv_batch *b, KvView &cv, KvRows &bv) {
    if (!c || !b || !c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale || !b->table || !b->row_start || !b->kv_len) {
        set_error("%s: null argument", op);
        return false;
    }
    if (c->n_pages < 1 || c->n_kv_heads < 1 || c->n_kv_heads > 32767 ||
        (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) ||
        (c->head_dim != 64 && c->head_dim != 128)) {
        set_error("%s: unsupported cache: %d pages of %d tokens, %d kv heads of %d (pages of 16, 32, 64 or 128 tokens, "
                  "at most 32767 heads, head dims 64 and 128)",
                  op, c->n_pages, c->page_tokens, c->n_kv_heads, c->head_dim);
        return false;
    }
    for (const void *p : {static_cast<const void *>(c->k_codes), static_cast<const void *>(c->v_codes)})
        if (reinterpret_cast<uintptr_t>(p) % 16) {
            set_error("%s: cache codes must be 16-byte aligned", op);
            return false;
        }
    for (const void *p : {static_cast<const void *>(c->k_scale), static_cast<const void *>(c->v_scale),
                          static_cast<const void *>(b->table), static_cast<const void *>(b->row_start),
                          static_cast<const void *>(b->kv_len)})
        if (reinterpret_cast<uintptr_t>(p) % 4) {
            set_error("%s: scales, table, row_start and kv_len must be 4-byte aligned", op);
            return false;
        }
    if (b->n_seqs < 0 || b->n_rows < 0 || b->max_rows < 0 || b->table_width < 1 || b->max_len < 0 ||
        b->n_seqs > (1 << 20) || b->n_rows > (1 << 27) || b->max_len > (1 << 30) || b->table_width > (1 << 30)) {
        set_error("%s: bad batch: %d sequences, %d rows (at most %d a sequence), table width %lld, max_len %lld", op,
                  b->n_seqs, b->n_rows, b->max_rows, (long long)b->table_width, (long long)b->max_len);
        return false;
    }
    int lg = 4;
    while ((1 << lg) < c->page_tokens) ++lg;
    cv = KvView{{static_cast<int8_t *>(c->k_codes), static_cast<int8_t *>(c->v_codes)},
                {c->k_scale, c->v_scale}, c->n_pages, c->n_kv_heads, lg, c->head_dim};
    bv = KvRows{b->table, b->row_start, b->kv_len, b->table_width, b->n_seqs, b->n_rows, b->max_rows, b->max_len};
    return true;
}

}  // namespace b200

using namespace b200;

extern "C" int sam3b200_kv_write(sam3b200_backend *h, const sam3b200_kv_cache *cache, const sam3b200_kv_batch *batch,
                                 int type, const void *k, const int64_t *k_nb, const void *v, const int64_t *v_nb) {
    auto *be = reinterpret_cast<Backend *>(h);
    WriteArgs a;
    if (!kv_views("kv_write", cache, batch, a.c, a.b)) return SAM3B200_STATUS_FAILED;
    const int bytes = type_bytes(type);
    if (!k || !v || !bytes || reinterpret_cast<uintptr_t>(k) % bytes || reinterpret_cast<uintptr_t>(v) % bytes) {
        if (!k || !v) set_error("kv_write: null argument");
        else set_error("kv_write: unsupported type %d (F32=0, F16=1, BF16=30) or unaligned rows", type);
        return SAM3B200_STATUS_FAILED;
    }
    a.x[0] = k, a.x[1] = v;
    a.xs[0] = row_tensor(k, type, k_nb, a.c.heads, a.c.D);
    a.xs[1] = row_tensor(v, type, v_nb, a.c.heads, a.c.D);
    if (!rows_ok("kv_write", "k", a.xs[0], a.b.n_rows, a.c.heads, a.c.D, false) ||
        !rows_ok("kv_write", "v", a.xs[1], a.b.n_rows, a.c.heads, a.c.D, false))
        return SAM3B200_STATUS_FAILED;
    if (!be) {
        set_error("kv_write: null backend");
        return SAM3B200_STATUS_FAILED;
    }
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return SAM3B200_STATUS_SUCCESS;
    a.err = be->err;
    DeviceScope dev(be->device);
    const bool vec = a.xs[0].aligned16 && a.xs[1].aligned16;
    auto go = [&](auto t) {
        using T = decltype(t);
        return vec ? launch_write<T, true>(a, be->stream) : launch_write<T, false>(a, be->stream);
    };
    const cudaError_t e = type == SAM3B200_TYPE_F32 ? go(float()) : type == SAM3B200_TYPE_F16 ? go(__half()) : go(__nv_bfloat16());
    be->count();
    return cuda_ok(e, "kv_write launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}

extern "C" int sam3b200_kv_read(sam3b200_backend *h, const sam3b200_kv_cache *cache, const sam3b200_kv_batch *batch,
                                int type, void *k, const int64_t *k_nb, void *v, const int64_t *v_nb) {
    auto *be = reinterpret_cast<Backend *>(h);
    ReadArgs a;
    if (!kv_views("kv_read", cache, batch, a.c, a.b)) return SAM3B200_STATUS_FAILED;
    const int bytes = type_bytes(type);
    if (!k || !v || !bytes || reinterpret_cast<uintptr_t>(k) % bytes || reinterpret_cast<uintptr_t>(v) % bytes) {
        if (!k || !v) set_error("kv_read: null argument");
        else set_error("kv_read: unsupported type %d (F32=0, F16=1, BF16=30) or unaligned rows", type);
        return SAM3B200_STATUS_FAILED;
    }
    a.y[0] = k, a.y[1] = v;
    a.ys[0] = row_tensor(k, type, k_nb, a.c.heads, a.c.D);
    a.ys[1] = row_tensor(v, type, v_nb, a.c.heads, a.c.D);
    if (!rows_ok("kv_read", "k", a.ys[0], a.b.n_rows, a.c.heads, a.c.D, true) ||
        !rows_ok("kv_read", "v", a.ys[1], a.b.n_rows, a.c.heads, a.c.D, true))
        return SAM3B200_STATUS_FAILED;
    if (!be) {
        set_error("kv_read: null backend");
        return SAM3B200_STATUS_FAILED;
    }
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return SAM3B200_STATUS_SUCCESS;
    a.err = be->err;
    DeviceScope dev(be->device);
    // about 16 K codes a block
    a.slabs = std::min(std::max(16384 / (a.c.D << a.c.page_log2), 1), 2 * a.c.heads);
    const dim3 grid((a.b.n_rows >> a.c.page_log2) + 2 * a.b.n_seqs, (2 * a.c.heads + a.slabs - 1) / a.slabs);
    const bool vec = a.ys[0].aligned16 && a.ys[1].aligned16;
    auto go = [&](auto t) {
        using T = decltype(t);
        return vec ? launch_after(kv_read_kernel<T, true>, grid, kThreads, 0, be->stream, a)
                   : launch_after(kv_read_kernel<T, false>, grid, kThreads, 0, be->stream, a);
    };
    const cudaError_t e = type == SAM3B200_TYPE_F32 ? go(float()) : type == SAM3B200_TYPE_F16 ? go(__half()) : go(__nv_bfloat16());
    be->count();
    return cuda_ok(e, "kv_read launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
