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
// f16 (2^-11 of it).  With t = score scale log2(e), 2^e the power of two above
// the largest |dv| of a block of tokens, and m the running maximum of t + e, the
// weights p = 2^(t + e - m) and the scales dv / 2^e stay within [-1, 1] for f16
// whatever the scales are, and only tokens that count for nothing leave them;
// the sum of the weights l takes p / 2^e, so it has the reference of O, and y = O / l.
//
// The kernel is kv_attn.cu's otherwise: one block of 4 warps per (8 or 16
// query rows of a kv head, part of the key range), blocks of 32 tokens (heads of 64: 64; in
// sixteens, each in one page) through a warp's own ring of shared memory, codes as the 16-row operand.  A lane's
// codes come by ldmatrix: plain for keys, word c of each group of token g (8
// dimensions), and transposed for values, 4 dimensions of tokens 2c and 2c + 1
// side by side, so a nibble and the one 16 bits above it are the pair that the
// instruction wants, in either product, and widening is a mask and a
// subtraction for a pair.  Each warp first widens its block's scales, a lane a
// token, and leaves them in shared memory as pairs of equal f32 numbers: every
// lane then has those of its tokens by one 16-byte load for two groups, ready
// for arithmetic on pairs, in place of two conversions a token and group.
//
// What bounds it: a warp's chain for each block of tokens (copies, scales, scores,
// maximum, exponentials, second product; some 680 instructions for 32 tokens of heads of 128, 4.6
// KB) with four warps a scheduler.  The issue slots are taken in two cycles of
// three (heads of 64: 58 %), no pipe is full (ALU 52 %, LSU 27 %, FMA and tensor
// cores 24 %), memory runs at 60 % of the copy.
// Measured: 64 sequences of 1000 ... 16100 tokens, 8 kv heads of 128, 4 query
// heads each, 157 to 173 us (666 MB, 4.2 to 3.9 TB/s; the 8-bit cache takes 216);
// a window of 1000 over them 38 (floor 11); one sequence
// of 900 7.9 us; 3 ... 5 tokens of each of 4 sequences of 30000 ... 70000, 8
// heads of 64, 37 us.  Scales taken from the stage by each lane: 169 for 161 of
// the first.  Copies by the bulk engine in place of 16-byte ones: 177, since the
// waits take more instructions than the copies; 5 blocks an SM: 195, for lack of
// registers; two stages, since 4 blocks with the widened scales have room for no
// more.
// The parts are cut on the device, from all lengths (few_part): cut by the host
// from the largest length, the last took 45 us, 24 sequences of 3000 ... 30000
// 131 in place of 109, the first 161; the look at all lengths costs one sequence
// of 900 0.7 us, and 64 of one length 157 in place of 149.  Every block reads all
// lengths, 128 sequences in one pass: 64, 128, 256, 512 and 1024 sequences of 500 ...
// 1500 tokens, 8 kv heads of 128, take 35, 53, 85, 165 and 335 us (floors 11, 22, 47, 92, 183).  A
// max_len 300 times the lengths: the first of these 38, 256 of them 87, the 4
// sequences with heads of 64 49 in place of 37, since most blocks then find nothing.  One wave of blocks
// with equal stretches of all the work, a block taking the end of one part and
// the start of the next: 182 us, and 115 in place of 82 for 200 sequences of 100
// ... 2500, whose starts and joins then follow one another.
#include <algorithm>
#include <cmath>

#include "kv4_codes.cuh"
#include "kv_attn_few.cuh"

namespace b200 {
namespace {

__device__ __forceinline__ float low_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The largest of three numbers (NaN is none).
__device__ __forceinline__ float max3(float x, float y, float z) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
    return d;
}
constexpr float kZeroScale = 8.271806125530277e-25f;  // 2^-80: what tokens of zeros count as (2^kZeroScaleLog2)
static_assert(kZeroScaleLog2 == -80.f, "its logarithm");

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

// The words that a lane's rows of four matrices give it, for 16 tokens: w[r][k] of group k and tokens 8 r ... .
template <int D, bool TRANS>
__device__ __forceinline__ void load_half(uint32_t (&w)[2][D / 32], uint32_t from) {
    uint32_t r[4];
    ldmatrix4<TRANS>(r, from);
    if constexpr (D == 128) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[0][k] = r[k];
        ldmatrix4<TRANS>(r, from + 8 * 64);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[1][k] = r[k];
    } else {
        w[0][0] = r[0], w[0][1] = r[1], w[1][0] = r[2], w[1][1] = r[3];
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
    static constexpr int kStages = 2, kBlocks = NT == 1 ? 4 : 2;  // stages of a warp, blocks an SM
    static constexpr int kTurn = 128;                              // least tokens of a part (one token over 900: 64 tokens 8.4 us, 128 7.6, with parts cut by the host)
    static constexpr int kCodeBytes = 16 * D / 2;                  // of 16 tokens
    static constexpr int kScaleBytes = 16 * kGroups * 2;
    // a stage: for each 16 tokens their keys' and values' codes, then for each 16 their scales
    static constexpr int kSixteens = 256 / D, kTokens = 16 * kSixteens;
    static constexpr int kHalfBytes = 2 * kCodeBytes, kScaleAt = kSixteens * kHalfBytes, kStageBytes = kScaleAt + 2 * kSixteens * kScaleBytes;
    // the block's scales as f32, each twice, a pair of groups in 16 bytes: [keys, values][kGroups / 2][kTokens]
    static constexpr int kWideAt = kWarps * kStages * kStageBytes, kWideBytes = kGroups * kTokens * 16;
    static constexpr int kRing = kWideAt + kWarps * kWideBytes;
    static constexpr int kRowFloats = D + 4;                       // a joined row, padded against bank conflicts
    static constexpr int kJoin = kWarps * kRows * kRowFloats * 4;
    static constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
    static_assert(kSmem >= kWarps * kRows * (D + 2) * 4, "shares of the parts");
    static constexpr int kEach = D * kRows / 128 > 8 ? D * kRows / 128 : 8;  // dimensions of a thread that joins
    // Byte of group c of token t within 16 staged tokens, turned so that 8 consecutive tokens' 16 bytes have
    // different banks.  Token t + 8 lies 8 tokens further.
    static __device__ __forceinline__ uint32_t at(int t, int c) {
        if (D == 128) return t * 64 + (c ^ ((t >> 1) & 3)) * 16;
        return t * 32 + (c ^ ((t >> 2) & 1)) * 16;
    }
    static __device__ __forceinline__ int column(int d) { return d; }
};

// A sequence's numbers, cut to the sizes, its tiles (of every kv head), and the keys of each in steps of 64.
template <typename F>
__device__ __forceinline__ void few_seq(const Kv4AttnArgs &a, int s, KvSeq &q, int &tiles, int &steps) {
    const int r0 = a.b.row_start[s], r1 = a.b.row_start[s + 1], len = a.b.kv_len[s];
    const int64_t cap = min(a.b.table_width << a.c.page_log2, a.b.max_len);
    q.s = s;
    q.r0 = min(max(r0, 0), a.b.n_rows);
    q.n = min(min(max(r1, q.r0), a.b.n_rows) - q.r0, a.b.max_rows);
    q.len = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), cap));
    tiles = (q.n * a.group + F::kRows - 1) / F::kRows * a.c.heads;
    steps = max((q.len - (kv_first(a, kv_last(a, q, 0)) & ~15) + 63) / 64, 1);
}

// This block's tile and part, from all sequences' lengths.  With T tiles of W steps in all, parts of W / (S - T) steps
// are at most S in all; S is a.splits, some waves of blocks.  Blocks 0, 1, ... take the parts in the order of the sequences,
// their tiles and kv heads.  Sums are cut where only arrays that contradict the sizes take them.  Runs of rows that follow one
// another make no more tiles than the host counted, so that the parts are at most the blocks; where row_start falls they
// can be more, and then no block does anything, since a tile of which only some parts ran would leave its counter above 0 for
// the calls to come.  The
// part found is one for the block, not one for each warp, so that its numbers are held once a warp (39 us in place of 36 for
// 3 to 5 tokens with heads of 64 otherwise).  Every thread of the block calls this; false if there is nothing to do.
template <typename F>
__device__ __forceinline__ bool few_part(const Kv4AttnArgs &a, FewTile &t) {
    constexpr unsigned kCut = 1u << 24;  // 128 threads' sums stay in 32 bits
    __shared__ unsigned s_tiles[kWarps], s_parts[kWarps];
    __shared__ uint64_t s_steps[kWarps];
    __shared__ KvSeq s_q;
    __shared__ unsigned s_local;  // the part's number within the sequence
    __shared__ int s_split;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int each = (a.b.n_seqs - 1) / (kWarps * 32) + 1;  // consecutive sequences of a thread
    const int s0 = min(static_cast<int>(threadIdx.x) * each, a.b.n_seqs), s1 = s0 + min(each, a.b.n_seqs - s0);
    if (blockIdx.x == gridDim.x - 1) kv_check(a.b, a.c.page_log2, false, a.err);
    KvSeq q;
    int tiles = 0, steps = 1;
    uint64_t T = 0, W = 0;
    for (int s = s0; s < s1; ++s) {
        few_seq<F>(a, s, q, tiles, steps);
        T += tiles, W += static_cast<uint64_t>(tiles) * steps;
    }
    const unsigned tw = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(min(T, static_cast<uint64_t>(kCut))));
    const unsigned low = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(W & 0xffffu));
    const unsigned high = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(min(W >> 16, static_cast<uint64_t>(kCut))));
    if (lane == 0) s_tiles[warp] = tw, s_steps[warp] = (static_cast<uint64_t>(high) << 16) + low;
    __syncthreads();
    T = W = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) T += s_tiles[w], W += s_steps[w];
    const unsigned S = a.splits, room = max(T < S ? S - static_cast<unsigned>(T) : 0u, S / 4);
    W += room - 1;
    const unsigned most = W >> 32 ? static_cast<unsigned>(W / room) : static_cast<unsigned>(W) / room;
    const int chunk = a.chunk ? a.chunk : static_cast<int>(max(min(most, 1u << 25), F::kTurn / 64u));
    uint64_t count = 0;
    if (each == 1) count = static_cast<uint64_t>(tiles) * ((steps + chunk - 1) / chunk);
    else
        for (int s = s0; s < s1; ++s) {
            few_seq<F>(a, s, q, tiles, steps);
            count += static_cast<uint64_t>(tiles) * ((steps + chunk - 1) / chunk);
        }
    const unsigned own = static_cast<unsigned>(min(count, static_cast<uint64_t>(kCut)));
    unsigned front = own;
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, front, i);
        if (lane >= i) front += x;
    }
    if (lane == 31) s_parts[warp] = front;
    __syncthreads();
    front -= own;
    unsigned parts = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) front += s_parts[w];
        parts += s_parts[w];
    }
    const unsigned block = blockIdx.x;
    if (block >= parts || parts > gridDim.x) return false;  // (kv_check names the starts that fall)
    if (front <= block && block < front + own) {
        for (int s = s0; each > 1 && s < s1; ++s) {
            few_seq<F>(a, s, q, tiles, steps);
            const uint64_t n = static_cast<uint64_t>(tiles) * ((steps + chunk - 1) / chunk);
            if (block < front + n) break;
            front += static_cast<unsigned>(n);
        }
        s_q = q, s_local = block - front, s_split = (steps + chunk - 1) / chunk;
    }
    __syncthreads();
    t.q = s_q, t.n_split = s_split;
    const int tile = static_cast<int>(s_local / static_cast<unsigned>(t.n_split));
    t.split = static_cast<int>(s_local) - tile * t.n_split;
    t.slot = static_cast<int64_t>(block) - t.split;
    t.kv = tile % a.c.heads;
    t.R = t.q.n * a.group;
    t.row0 = tile / a.c.heads * F::kRows, t.i_lo = t.row0 / a.group, t.i_hi = (min(t.row0 + F::kRows, t.R) - 1) / a.group;
    const int k_end = kv_last(a, t.q, t.i_hi) + 1, k_begin = kv_first(a, kv_last(a, t.q, t.i_lo)) & ~15;
    t.t_begin = static_cast<int>(min(k_begin + static_cast<int64_t>(t.split) * chunk * 64, static_cast<int64_t>(max(k_end, 0))));
    t.t_end = static_cast<int>(min(t.t_begin + static_cast<int64_t>(chunk) * 64, static_cast<int64_t>(k_end)));
    return true;
}

template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32, (Few4<D, NT>::kBlocks)) kv4_attn_few_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using F = Few4<D, NT>;
    constexpr int kGroups = F::kGroups;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float s_m[kWarps][F::kRows], s_l[kWarps][F::kRows];
    wait_for_stream();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int G = a.group;
    FewTile tile;
    if (!few_part<F>(a, tile)) return;
    const int kv = tile.kv;
    const KvSeq &q = tile.q;
    const int row0 = tile.row0, i_lo = tile.i_lo, i_hi = tile.i_hi, R = tile.R, t_begin = tile.t_begin, t_end = tile.t_end;
    const int n_blocks = t_end > t_begin ? (t_end - t_begin + F::kTokens - 1) / F::kTokens : 0;
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
    // this lane's bytes within a half of a stage: the copy of chunk lane (of 32 a step), and its row of the matrices that it loads
    const uint32_t put0 = F::at(lane / kGroups, lane % kGroups);
    const uint32_t get0 = D == 128 ? F::at(lane & 7, lane >> 3) : F::at((lane & 7) + (lane >> 4) * 8, (lane >> 3) & 1);
    // what this lane copies, for token 0 of the cache's slabs: tokens are counted over all of them, in 32 bits (see kv_views)
    const uint8_t *own_k = a.c.codes[0] + lane * 16, *own_v = a.c.codes[1] + lane * 16;
    constexpr int kScaleChunks = F::kScaleBytes / 16;
    const uint8_t *own_scale = reinterpret_cast<const uint8_t *>(a.c.scale[lane >= kScaleChunks]) + lane % kScaleChunks * 16;
    float4 *wide = reinterpret_cast<float4 *>(smem + F::kWideAt + warp * F::kWideBytes);
    const uint32_t ring_at = smem_u32(ring), put_at = ring_at + put0, put_scale_at = ring_at + F::kScaleAt + lane * 16;
    // lane kSixteens j + h: where the h-th 16 tokens of block kBatch b + j of this warp lie, for batches b and b + 1
    constexpr int kBatch = 32 / F::kSixteens;
    uint32_t at_now = 0, at_next = 0;
    auto look_up = [&](int j) -> uint32_t {
        const int tok = t_begin + (j / F::kSixteens * kWarps + warp) * F::kTokens + j % F::kSixteens * 16;
        if (j / F::kSixteens >= mine || tok >= t_end) return 0;  // (copied all the same, and seen by no row)
        const int page = max(kv_page(a.c, a.b, q.s, tok >> a.c.page_log2, a.err), 0);
        return ((static_cast<uint32_t>(page) * a.c.heads + kv) << a.c.page_log2) + (tok & ((1 << a.c.page_log2) - 1));
    };
    at_next = look_up(lane);
    auto issue = [&](int j, int slot) {  // block j of this warp into a slot
        if (j < mine) {
            if (j % kBatch == 0) {
                at_now = at_next;
                at_next = look_up(F::kSixteens * (j + kBatch) + lane);
            }
#pragma unroll
            for (int h = 0; h < F::kSixteens; ++h) {
                const uint64_t at = __shfl_sync(0xffffffffu, at_now, F::kSixteens * (j % kBatch) + h);
                const uint32_t to = slot * F::kStageBytes;
#pragma unroll
                for (int w = 0; w < 2; ++w)
#pragma unroll
                    for (int k = 0; k < F::kCodeBytes / 512; ++k)  // a step of 8 (D = 128) or 16 tokens
                        cp16(put_at + to + h * F::kHalfBytes + w * F::kCodeBytes + k * 512, (w ? own_v : own_k) + at * (D / 2) + k * 512);
                if (lane < 2 * kScaleChunks) cp16(put_scale_at + to + 2 * h * F::kScaleBytes, own_scale + at * (D / 16));
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
        for (int j = 0; j < 2; ++j)  // a factor of 0 would make NaN of -inf; a tiny one leaves 0 of the scores
            row_c[n][j] = fmaxf(__shfl_sync(0xffffffffu, up, (2 * c + j) * 4), 1e-37f);
    }
    // tokens that some row of the tile does not see, and those that none sees (they need not hold numbers)
    const int seen_by_all = kv_last(a, q, i_lo), window_end = kv_first(a, kv_last(a, q, i_hi)), first_any = kv_first(a, seen_by_all);

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2], high[NT][2], less[NT][2];  // high, less: what follows from m for the next scores
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = high[n][0] = high[n][1] = -INFINITY, l[n][0] = l[n][1] = less[n][0] = less[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    int slot = 0, slot_in = F::kStages - 1;
    for (int j = 0; j < mine; ++j) {
        cp_wait<F::kStages - 2>();
        __syncwarp();  // block j is there for all lanes, and block j - 1 is read by all
        issue(j + F::kStages - 1, slot_in);
        const uint8_t *st = ring + slot * F::kStageBytes;
        const uint32_t st_at = ring_at + slot * F::kStageBytes;
        slot_in = slot;
        slot = slot + 1 == F::kStages ? 0 : slot + 1;
        const int tok = t_begin + (j * kWarps + warp) * F::kTokens;

        // the scales: a lane a token (heads of 64: two); those of values that no row sees are 0
        unsigned top_bits = __float_as_uint(kZeroScale);
        float dv[F::kTokens / 32][kGroups];
#pragma unroll
        for (int u = 0; u < F::kTokens / 32; ++u) {
            const int k = lane + 32 * u;
            const uint8_t *from = st + F::kScaleAt + k / 16 * (2 * F::kScaleBytes) + k % 16 * (2 * kGroups);
            float dk[kGroups];
            scales_of<kGroups>(from, dk);
            scales_of<kGroups>(from + F::kScaleBytes, dv[u]);
            const bool out = tok + k >= t_end || tok + k < first_any;
#pragma unroll
            for (int i = 0; i < kGroups; i += 2) {
                if (out) dv[u][i] = dv[u][i + 1] = 0.f;
                top_bits = max(top_bits, max(__float_as_uint(fabsf(dv[u][i])), __float_as_uint(fabsf(dv[u][i + 1]))));
                wide[i / 2 * F::kTokens + k] = make_float4(dk[i], dk[i], dk[i + 1], dk[i + 1]);
            }
        }
        // 2^e above all of them, and 2^-e
        const int top_e = min(static_cast<int>(__reduce_max_sync(0xffffffffu, top_bits) >> 23), 252);
        const float lv = static_cast<float>(top_e - 126), down = __int_as_float((253 - top_e) << 23);
#pragma unroll
        for (int u = 0; u < F::kTokens / 32; ++u)
#pragma unroll
            for (int i = 0; i < kGroups; i += 2) {
                const float x = dv[u][i] * down, y = dv[u][i + 1] * down;
                wide[(kGroups + i) / 2 * F::kTokens + lane + 32 * u] = make_float4(x, x, y, y);
            }
        __syncwarp();

        // scores of tokens 16 h + g (t[h][n][0], [1]) and 16 h + g + 8 ([2], [3]) for rows 8 n + 2 c, + 1
        float t[F::kSixteens][NT][4];
#pragma unroll
        for (int h = 0; h < F::kSixteens; ++h) {
            uint32_t w[2][kGroups];  // word c of each group of tokens g and g + 8
            load_half<D, false>(w, st_at + h * F::kHalfBytes + get0);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const float4 d0 = wide[k / 2 * F::kTokens + 16 * h + g], d1 = wide[k / 2 * F::kTokens + 16 * h + 8 + g];
                uint32_t u[4], v[4];
                codes4(w[0][k], u);
                codes4(w[1][k], v);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float s[4];
                    mma16816_first(s, u[0], v[0], u[1], v[1], qf[n][k][0], qf[n][k][1]);
                    mma16816(s, u[2], v[2], u[3], v[3], qf[n][k][2], qf[n][k][3]);
                    float *x = t[h][n];
                    if (k == 0) {
                        fmul2(x[0], x[1], s[0], s[1], d0.x, d0.y);
                        fmul2(x[2], x[3], s[2], s[3], d1.x, d1.y);
                    } else {
                        ffma2(x[0], x[1], s[0], s[1], k & 1 ? d0.z : d0.x, k & 1 ? d0.w : d0.y);
                        ffma2(x[2], x[3], s[2], s[3], k & 1 ? d1.z : d1.x, k & 1 ? d1.w : d1.y);
                    }
                }
            }
        }
        if (tok + F::kTokens - 1 > seen_by_all || tok < window_end) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int last = kv_last(a, q, i_lo + (rest0 + 8 * n + 2 * c + k) / G), first = kv_first(a, last);
#pragma unroll
                    for (int h = 0; h < F::kSixteens; ++h)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int at = tok + 16 * h + 8 * r + g;
                            if (at > last || at < first) t[h][n][2 * r + k] = -INFINITY;
                        }
                }
        }
        auto most = [&](int n, int k) {
            float x = fmaxf(t[0][n][k], t[0][n][k + 2]);
#pragma unroll
            for (int h = 1; h < F::kSixteens; ++h) x = max3(x, t[h][n][k], t[h][n][k + 2]);
            return fmaf(x, row_c[n][k], lv);
        };
        bool rise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) rise |= most(n, k) > high[n][k];
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float top = most(n, k);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    const float to = fmaxf(m[n][k], top);
                    const float alpha = m[n][k] == to ? 1.f : ex2_approx(m[n][k] - to);
                    m[n][k] = to;
                    high[n][k] = to + kLazy;
                    less[n][k] = to == -INFINITY ? 0.f : to - kPUp;
                    l[n][k] *= alpha;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) o[n][i][k] *= alpha, o[n][i][k + 2] *= alpha;
                }
        }
        float sum[NT][2], add[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) sum[n][k] = 0.f, add[n][k] = lv - less[n][k];
#pragma unroll
        for (int h = 0; h < F::kSixteens; ++h) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    t[h][n][k] = ex2_approx(fmaf(t[h][n][k], row_c[n][k], add[n][k]));
                    t[h][n][k + 2] = ex2_approx(fmaf(t[h][n][k + 2], row_c[n][k], add[n][k]));
                    sum[n][k] += t[h][n][k] + t[h][n][k + 2];
                    if (h == F::kSixteens - 1) l[n][k] = fmaf(sum[n][k], down, l[n][k]);
                }
            // values: of each group 4 dimensions (4 g ...) of tokens 2c, 2c + 1 and of 8 + 2c, 9 + 2c
            uint32_t w[2][kGroups];
            load_half<D, true>(w, st_at + h * F::kHalfBytes + F::kCodeBytes + get0);
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const float4 d0 = wide[(kGroups + k) / 2 * F::kTokens + 16 * h + g], d1 = wide[(kGroups + k) / 2 * F::kTokens + 16 * h + 8 + g];
                uint32_t u[4], v[4];
                codes4(w[0][k], u);
                codes4(w[1][k], v);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float *y = t[h][n];
                    float x[4];
                    fmul2(x[0], x[1], y[0], y[1], k & 1 ? d0.z : d0.x, k & 1 ? d0.w : d0.y);
                    fmul2(x[2], x[3], y[2], y[3], k & 1 ? d1.z : d1.x, k & 1 ? d1.w : d1.y);
                    const uint32_t p0 = transposed(pack_f16(x[0], x[1])), p1 = transposed(pack_f16(x[2], x[3]));
                    // dimensions 4 g, + 1 of the group are rows g, g + 8 of one product, + 2, + 3 of the next
                    mma16816(o[n][2 * k], u[0], u[1], v[0], v[1], p0, p1);
                    mma16816(o[n][2 * k + 1], u[2], u[3], v[2], v[3], p0, p1);
                }
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
    using F = Few4<D, NT>;
    constexpr unsigned kBit = 1u << (kReadyFew4 + 2 * (NT - 1) + (D == 64));
    // (a batch without rows has one too: its arrays are checked)
    const int64_t most = (static_cast<int64_t>(a.b.max_rows) * a.group + F::kRows - 1) / F::kRows * a.b.n_seqs;
    const int64_t tiles = a.c.heads * std::max(std::min(static_cast<int64_t>(a.b.n_rows) * a.group / F::kRows + a.b.n_seqs, most), int64_t(1));
    const int64_t wave = F::kBlocks * static_cast<int64_t>(num_sms);
    const int64_t span = std::max(a.window ? std::min(a.b.max_len, static_cast<int64_t>(a.window) + a.b.max_rows + 16) : a.b.max_len, int64_t(1));
    // Waves of blocks: more even out lengths (see few_part: the parts of w waves have W / (w wave - T) steps), each costs about
    // 10 steps of 64 tokens.  W from half of the longest, the lengths being on the device.  Measured, heads of 128, 1 and 2
    // waves: 24 sequences of 3000 ... 30000 by 8 heads 133 and 109 us; heads of 64, 16 of 900 ... 6000 16.7 and 25.7.
    const double work = static_cast<double>(tiles) * static_cast<double>(span) / 128;
    int64_t waves = 1;
    double least = 0;
    for (int64_t w = 1; w <= 4; ++w) {
        const double cost = static_cast<double>(w) * (work / static_cast<double>(std::max(w * wave - tiles, w * wave / 4)) + 10);
        if (w == 1 || cost < least) least = cost, waves = w;
    }
    int64_t grid = std::max(waves * wave, waves * wave / 4 + tiles);
    a.splits = static_cast<int>(waves * wave), a.chunk = 0;
    if (grid > kMaxParts) grid = tiles, a.chunk = 1 << 25;  // no parts
    grid = std::min(grid, tiles * ((span + F::kTurn - 1) / F::kTurn));
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    if (!(*a.ready & kBit)) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_attn_few_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem);
        if (e != cudaSuccess) return e;
        *a.ready |= kBit;
    }
    return launch_after(kv4_attn_few_kernel<D, NT>, dim3(static_cast<unsigned>(grid)), kWarps * 32, F::kSmem, st, a);
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
    // us in a graph, 8 kv heads, few rows and tc, for one sequence of 8000 tokens, one of 100000, 16 of 4000.  Heads of 128:
    // 16 rows a kv head 25 and 34, 59 and 116, 50 and 62; 32 rows 31 and 34, 116 and 114, 77 and 62.  Heads of 64: 32 rows 21
    // and 24, 72 and 91, 52 and 58; 48 rows 23 and 24, 89 and 91, 69 and 71; 64 rows 23 and 24, 106 and 91, 82 and 72
    const bool few = static_cast<int64_t>(a.b.max_rows) * a.group <= (a.c.D == 128 ? 16 : 48);
    const cudaError_t e = few ? kv_attn_few(a, k->be->num_sms, k->be->stream) : kv_attn_tc(a, k->be->num_sms, k->be->stream);
    k->be->count();
    return cuda_ok(e, "kv4_attention launch") ? SAM3B200_STATUS_SUCCESS : SAM3B200_STATUS_FAILED;
}
