// paged_attention: causal attention of ragged rows over the paged int8 cache.
//
// Two kernels.  Prompts' codes become 16-bit floats for tcgen05 (below, with what
// that costs in accuracy).  For few rows both products run on integer tensor-core
// instructions over the cache's codes as they lie, so that no code is converted.
// The other operand is written in fixed point, as int8 digits:
//
//   q . K:  a row of q is qs * (65536 d1 + 256 d2 + d3), qs = max|q| / (127 *
//           65536), the digits signed bytes.  The digits' dots with the codes are
//           exact; the score is (65536 D1 + 256 D2 + D3) * qs * scale * s_K[page].
//           (Two digits would do for outputs of 16 bits, but not for lse.)
//   p . V:  p * s_V[page], relative to the largest of it among 32 tokens, is in
//           [0, 1] and becomes 32 bits, whose bytes are unsigned digits; the
//           largest joins the product's factor.
//
// A term of q . K so is off by 2^-24 of the row's largest |q|, a weight by 2^-33 of
// the largest p * s_V of its own 32 tokens and not of the row's: a key that takes
// nearly all of the sum (an attention sink, whose V may be near zero) leaves the
// thousands around it their bits.  (16 bits relative to the row's running maximum
// lost 5% to 27% of such an output.)  Softmax statistics and the output's
// accumulator are fp32.
#include <cmath>

#include "lq_ctx.h"
#include "lq_paged.cuh"
#include "lq_paged_host.h"
#include "lq_tc.cuh"
#include "lq_types.cuh"

namespace lq {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Adding an integer below 2^22 to these bits gives the float 1.5 * 2^23 plus it:
// accumulators that start here are read as floats without a conversion.
constexpr int kBiasBits = 0x4B400000;
constexpr float kBias = 12582912.0f;

struct AttArgs {
    PagedKV c;
    KVBatch b;
    const void* q;
    void* out;
    float* lse;
    int64_t ld_q, ld_out;
    int n_heads, group, type;
    int q_vec;        // rows of q are 16-byte aligned
    int few_rows;     // (token, head) rows of a sequence and kv head that the first kernel takes
    float scale;      // log2(e) times the caller's
    int row_tiles;    // tiles of 8 (token, head) rows of a sequence and kv head
    int plan;         // contexts are split (0: a CTA takes a whole one)
    float* part;      // [split of a sequence][kv head, row tile][its rows][head_size + 8]: out, max, sum
    int* cnt;         // [sequence][kv head, row tile] arrivals
    int* err;
};

// four neighbouring elements of q as they lie: fp32 (PARTS 2) or 16-bit
template <int PARTS>
struct RawQ {
    uint32_t w[2 * PARTS];
    __device__ __forceinline__ void load(const AttArgs& a, int64_t i) {
        if constexpr (PARTS == 2) {
            const float* p = static_cast<const float*>(a.q) + i;
            if (a.q_vec) {
                const uint4 v = ld_after(reinterpret_cast<const uint4*>(p));
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(ld_after(p + e));
            }
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(a.q) + i;
            if (a.q_vec) {
                const uint2 v = ld_after(reinterpret_cast<const uint2*>(p));
                w[0] = v.x, w[1] = v.y;
            } else {
                w[0] = ld_after(p) | (uint32_t)ld_after(p + 1) << 16;
                w[1] = ld_after(p + 2) | (uint32_t)ld_after(p + 3) << 16;
            }
        }
    }
    __device__ __forceinline__ void get(const AttArgs& a, float (&v)[4]) const {
        if constexpr (PARTS == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
        } else if (a.type == LQ_F16) {
            unpack_word<__half>(w[0], v);
            unpack_word<__half>(w[1], v + 2);
        } else {
            unpack_word<__nv_bfloat16>(w[0], v);
            unpack_word<__nv_bfloat16>(w[1], v + 2);
        }
    }
};

__device__ __forceinline__ void store_out(const AttArgs& a, int64_t i, float v) {
    if (a.type == LQ_F32)
        static_cast<float*>(a.out)[i] = v;
    else if (a.type == LQ_F16)
        static_cast<__half*>(a.out)[i] = from_f32<__half>(v);
    else
        static_cast<__nv_bfloat16*>(a.out)[i] = from_f32<__nv_bfloat16>(v);
}

// 4 neighbouring outputs
__device__ __forceinline__ void store_out4(const AttArgs& a, int64_t i, const float (&v)[4]) {
    auto put = [&](auto* p) {
        using T = std::remove_reference_t<decltype(*p)>;
        if (reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0) {
            store_n<4, true>(p, v);
        } else {
            for (int k = 0; k < 4; ++k) p[k] = from_f32<T>(v[k]);
        }
    };
    if (a.type == LQ_F32)
        put(static_cast<float*>(a.out) + i);
    else if (a.type == LQ_F16)
        put(static_cast<__half*>(a.out) + i);
    else
        put(static_cast<__nv_bfloat16*>(a.out) + i);
}

// 16 neighbouring outputs x * f + bad
__device__ __forceinline__ void store_row16(const AttArgs& a, int64_t i, const int (&x)[16], float f, float bad) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = fmaf(__int_as_float(x[k]), f, bad);
    auto put = [&](auto* p) {
        using T = std::remove_reference_t<decltype(*p)>;
        if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
            constexpr int W = 4 / sizeof(T);
            uint32_t w[16 / W];
#pragma unroll
            for (int k = 0; k < 16 / W; ++k) w[k] = pack_word<T>(v + k * W);
#pragma unroll
            for (int k = 0; k < 4 / W; ++k)
                reinterpret_cast<uint4*>(p)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) p[k] = from_f32<T>(v[k]);
        }
    };
    if (a.type == LQ_F32)
        put(static_cast<float*>(a.out) + i);
    else if (a.type == LQ_F16)
        put(static_cast<__half*>(a.out) + i);
    else
        put(static_cast<__nv_bfloat16*>(a.out) + i);
}

// the outputs of a sequence's rows that attend to nothing, for one kv head
__device__ __forceinline__ void zero_rows(const AttArgs& a, const SeqRows& q, int h) {
    const int w = a.group * a.c.head_size;
#pragma unroll 1
    for (int row = q.first; row < q.r0; ++row) {
        for (int d = threadIdx.x; d < w; d += blockDim.x) store_out(a, (int64_t)row * a.ld_out + (int64_t)h * w + d, 0.0f);
        for (int e = threadIdx.x; a.lse && e < a.group; e += blockDim.x)
            a.lse[(int64_t)row * a.n_heads + h * a.group + e] = -INFINITY;
    }
}

template <int N>
__device__ __forceinline__ void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// 2^k for -126 <= k <= 127
__device__ __forceinline__ float lq_exp2i(int k) { return __int_as_float((k + 127) << 23); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

// d += a (16 x 32 signed bytes) * b (32 x 8 signed bytes)
__device__ __forceinline__ void mma_s8(int (&d)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// d += a (16 x 32 unsigned bytes) * b (32 x 8 signed bytes)
__device__ __forceinline__ void mma_u8(int (&d)[4], uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// d += a (16 x 32 signed bytes) * b (32 x 8 unsigned bytes)
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the largest of a warp's values; a NaN among others is passed over
__device__ __forceinline__ float max_redux(float v) {
    float m;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

__device__ __forceinline__ float unbias(int d) { return __int_as_float(d) - kBias; }

// ---------------------------------------------------------------------------
// Few rows per kv head (decode): bound by the cache's bytes from HBM.
//
// One CTA per (sequence, kv head, tile of rows, split of the context); its
// four warps take 32 tokens each in turn, each through a ring of its own of
// bulk copies, and are joined at the end; the splits of a row are joined by
// the last CTA to arrive, in split order.
//
// Tiles of 8 rows (several query heads to a kv head, or several tokens): an
// MMA's 16 rows are the 8 (token, head) rows twice: rows 0-7 hold their first
// digit, rows 8-15 the second, so a thread finds both digits' dots of its row
// in its own registers.  The third and the weights' fourth take a second MMA.
//
// One row (a token, and a query head to each kv head): the codes are the MMA's
// 16 rows, 16 tokens of K or 16 dims of V, and the digits its columns, so that
// one MMA takes all digits and a lane one token's softmax.  64 sequences of the
// case below take 77 us so, 102 us as a tile of 8 rows with seven empty.
//
// How long a split is follows from the contexts, which only the device knows
// (a captured call's max_context is that of its longest replay): the least
// multiple of 128 tokens with which all splits find a CTA slot at once.
//
// Tokens and MMA columns of tiles of 8 rows: the two 8-column tiles over 16 tokens are dealt so
// that a thread's four scores are four neighbouring tokens (the A operand of
// p . V) and that the eight rows an ldmatrix reads lie in different banks:
// column 2j + e of the even tile is token 4j + 2x + e with x = j / 2, of the odd
// tile with x = 1 - j / 2.
//
// Measured, 128 dims: 64 sequences of up to 1100 tokens, 40 heads, fp32 77 us (458
// MB, 5.9 TB/s); 16 of up to 4000, 8 kv heads of 8 query heads each, 26 us (86 MB,
// 3.3 TB/s: DRAM 32% busy, issue slots 36%); 16 of 8192 each 57 us (4.7 TB/s); one
// of 2048, 32 heads, fp32 10.6 us.  What holds the short ones is the chain lengths,
// pages, codes, and the two joins: 5 us with one split to a sequence, 8 us with more.

constexpr int kFewWarps = 4;
constexpr int kFewThreads = 32 * kFewWarps;
constexpr int kItem = 32;   // tokens of one step of a warp
constexpr int kSlots = 2;   // its ring
constexpr float kLeast = 7.9e-31f;  // 2^-100: below it, a weight (of at most 1) counts as zero
constexpr int kFewRows = 32;  // (token, head) rows of a sequence up to which it is taken

// CTAs on an SM: what registers and the rings allow
constexpr int few_ctas(int hs, int rows) { return hs > 128 ? 1 : hs <= 64 && rows == 1 ? 5 : 3; }

template <int HS>
constexpr int few_smem() {
    return kFewWarps * kSlots * kItem * HS * 2;
}

struct Split {
    int s, split, chunk;  // sequence (-1: none), its split, tokens of a split
};

// The unit-th of at most `units` splits of the batch's sequences, each of which
// has one at least.  By one warp; a sequence a lane.
__device__ __forceinline__ Split find_split(const KVBatch& b, int unit, int units, int lane) {
    auto blocks = [&](int i) {  // of 128 tokens
        return i < b.n_seqs ? (min(max(ld_after(b.context + i), 0), b.max_context) + 127) / 128 : 0;
    };
    asm volatile("prefetch.global.L1 [%0];" ::"l"(b.row_start + min(lane, b.n_seqs)));
    if (b.n_seqs == 1) return {0, unit, max(2, (blocks(0) + units - 1) / units) * 128};
    int total = 0;
    for (int i = lane; i < b.n_seqs; i += 32) total += blocks(i);
    total = __reduce_add_sync(0xffffffffu, total);
    int chunk = max(2, (total + units - 1) / units);
    auto parts = [&](int i) { return i < b.n_seqs ? max(1, (blocks(i) + chunk - 1) / chunk) : 0; };
    for (;; chunk += max(1, chunk / 8)) {  // ends: a long chunk leaves one split each, fewer than units
        int n = 0;
        for (int i = lane; i < b.n_seqs; i += 32) n += parts(i);
        if (__reduce_add_sync(0xffffffffu, n) <= units) break;
    }
    int before = 0;
    for (int i0 = 0; i0 < b.n_seqs; i0 += 32) {
        int sum = parts(i0 + lane);
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const int k = __popc(__ballot_sync(0xffffffffu, before + sum <= unit));  // sequences that end before it
        if (k < 32) {
            const int past = __shfl_sync(0xffffffffu, sum, max(k - 1, 0));
            return i0 + k < b.n_seqs ? Split{i0 + k, unit - before - (k > 0 ? past : 0), chunk * 128} : Split{-1, 0, 0};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {-1, 0, 0};
}

// PARTS: 2 for fp32, 1 for the 16-bit types.  ROWS: rows of a tile, 8 or 1
template <int PARTS, int HS, bool EXACT, int ROWS>
__global__ void __launch_bounds__(kFewThreads, few_ctas(HS, ROWS)) attend_few_kernel(const __grid_constant__ AttArgs a) {
    constexpr int KS = HS / 32;       // k steps of q . K
    constexpr int NP = 2;             // MMAs of a tile of q . K: two digits, the third
    constexpr int NT = HS / 8;        // column tiles of p . V
    extern __shared__ __align__(128) unsigned char ring_all[];
    __shared__ uint4 qfrag[ROWS == 8 ? KS * NP * 32 : HS / 4];  // one row: [digit, 4 with zeros][HS / 4] words
    __shared__ uint4 weights[ROWS == 8 ? 1 : kFewWarps * kItem / 4];
    __shared__ float qscale[8];
    __shared__ uint64_t bars[kFewWarps * kSlots];
    __shared__ int last_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hs = EXACT ? HS : a.c.head_size;
    const int P = a.c.page_size, H = a.c.n_kv_heads, g = a.group;
    const int rt = blockIdx.x % a.row_tiles, h = blockIdx.x / a.row_tiles;

    if (tid < kFewWarps * kSlots) mbar_init(&bars[tid], 1);
    fence_mbar_init();
    pdl_trigger();
    pdl_wait();
    int s = blockIdx.y, split = 0, chunk = INT32_MAX;
    if (a.plan) {
        const Split x = find_split(a.b, blockIdx.y, gridDim.y, lane);
        if (x.s < 0) return;
        s = x.s, split = x.split, chunk = x.chunk;
    }
    const SeqRows q = seq_rows(a.b, s, split == 0 && rt == 0 && h == 0 && tid == 0 ? a.err : nullptr);
    if (split == 0 && rt == 0) zero_rows(a, q, h);
    const int rows = q.n * g;
    if (rows > a.few_rows || rt * ROWS >= rows) return;
    const int top = min(rows, rt * ROWS + ROWS) - 1;            // the tile's last row
    const int seen = q.begin + top / g + 1;               // tokens that it sees
    const int splits = a.plan ? (seen + chunk - 1) / chunk : 1;
    if (split >= splits) return;
    const int ta = a.plan ? split * chunk : 0, tb = a.plan ? min(ta + chunk, seen) : seen;
    int* const err = lane == 0 ? a.err : nullptr;

    // the warp's items are kItem tokens at ta + (warp + kFewWarps * j) * kItem; lane L
    // keeps the pages of item j0 + L
    const int items = max(0, ((tb - ta + kItem - 1) / kItem - warp + kFewWarps - 1) / kFewWarps);
    unsigned char* ring = ring_all + warp * kSlots * kItem * HS * 2;
    int held = -1;  // the block of 32 items whose pages are held
    int64_t pg0 = -1, pg1 = -1;
    float2 sc_slot[kSlots];
    const uint64_t policy = l2_evict_first_policy();
    auto issue = [&](int j) {
        if ((j >> 5) != held) {
            held = j >> 5;
            const int t = ta + (warp + kFewWarps * (held * 32 + lane)) * kItem;
            pg0 = t < tb ? page_of(a.c, a.b, s, t / P, a.err) : -1;
            pg1 = P < kItem && t + 16 < tb ? page_of(a.c, a.b, s, t / P + 1, a.err) : -1;
        }
        const int64_t p0 = __shfl_sync(0xffffffffu, pg0, j & 31), p1 = __shfl_sync(0xffffffffu, pg1, j & 31);
        const int slot = j % kSlots;
        uint64_t* bar = &bars[warp * kSlots + slot];
        unsigned char* dst = ring + slot * kItem * HS * 2;
        const int64_t cell = (int64_t)hs * P * 2;
        const int8_t* codes = static_cast<const int8_t*>(a.c.codes);
        const int8_t *c0 = codes + (p0 * H + h) * cell, *c1 = codes + (p1 * H + h) * cell;
        const int bytes = P < kItem ? ((p0 >= 0) + (p1 >= 0)) * (int)cell : p0 >= 0 ? kItem * hs * 2 : 0;
        __syncwarp();  // every lane has read the slot's last item
        if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
        __syncwarp();
        if (P <= kItem) {
            // whole pages, K and V together
            if (lane == 0 && p0 >= 0) bulk_g2s(dst, c0, (uint32_t)cell, bar, policy);
            if (lane == 1 && p1 >= 0) bulk_g2s(dst + cell, c1, (uint32_t)cell, bar, policy);
        } else if (p0 >= 0) {
            const int off = (ta + (warp + kFewWarps * j) * kItem) % P;
            if (lane < hs / 16)  // 16 dims of the item's tokens
                bulk_g2s(dst + lane * kItem * 16, c0 + ((int64_t)lane * P + off) * 16, kItem * 16, bar, policy);
            else if (lane == hs / 16)
                bulk_g2s(dst + kItem * hs, c0 + (int64_t)hs * (P + off), kItem * hs, bar, policy);
        }
        // the scales of the item's pages, by lane 0 (and 1): used one step later
        const int64_t pl = lane == 1 ? p1 : p0;
        float2 sc = make_float2(NAN, NAN);
        if (lane < 2 && pl >= 0) sc = ld_after(reinterpret_cast<const float2*>(a.c.scales) + pl * H + h);
        return sc;
    };
    __syncthreads();  // barriers are ready
#pragma unroll
    for (int j = 0; j < kSlots; ++j)
        if (j < items) sc_slot[j] = issue(j);

    // the digits of the tile's rows, in the order of the MMA's operand: two rows
    // per warp, or one by the first warp
#pragma unroll
    for (int i = 0; i < (ROWS == 8 ? 2 : 1); ++i) {
        if (ROWS == 1 && warp > 0) break;
        const int r8 = 2 * warp + i, r = rt * ROWS + r8;
        const bool have = r < rows;
        const int64_t base = have ? (int64_t)(q.r0 + r / g) * a.ld_q + (int64_t)(h * g + r % g) * hs : 0;
        float x[(HS + 127) / 128][4];
        uint32_t m = 0;
#pragma unroll
        for (int b = 0; b < (HS + 127) / 128; ++b) {
            const int d = b * 128 + lane * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][e] = 0.0f;
            if (have && d < hs) {
                RawQ<PARTS> raw;
                raw.load(a, base + d);
                raw.get(a, x[b]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max(m, abs_bits(x[b][e]));
        }
        m = __reduce_max_sync(0xffffffffu, m);
        constexpr float kTop = 8323072.0f;  // 127 * 256^2
        const float peak = __uint_as_float(m);
        const bool fine = m < kInfBits && peak > 1e-30f;
        const float inv = fine ? kTop / peak : 0.0f;
        if (lane == 0) qscale[r8] = m >= kInfBits ? NAN : fine ? peak / kTop * a.scale : 0.0f;
#pragma unroll
        for (int b = 0; b < (HS + 127) / 128; ++b) {
            const int d = b * 128 + lane * 4;
            if (d >= HS) continue;
            uint32_t w[3] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                int n = m >= kInfBits ? 0 : __float2int_rn(x[b][e] * inv);
                const int d3 = (int)(int8_t)n;
                n = (n - d3) >> 8;
                w[2] |= (uint32_t)(d3 & 255) << (8 * e);
                const int d2 = (int)(int8_t)n;
                w[1] |= (uint32_t)(d2 & 255) << (8 * e);
                w[0] |= (uint32_t)(((n - d2) >> 8) & 255) << (8 * e);
            }
            if constexpr (ROWS == 8) {
                const int ks = d / 32, half = d % 32 / 16, L = r8 * 4 + d % 16 / 4;
                uint32_t* f = reinterpret_cast<uint32_t*>(&qfrag[ks * NP * 32 + L]);
                f[half * 2] = w[0];
                f[half * 2 + 1] = w[1];
                f[32 * 4 + half * 2] = w[2];
                f[32 * 4 + half * 2 + 1] = 0;
            } else {
                uint32_t* f = reinterpret_cast<uint32_t*>(qfrag) + d / 4;
                f[0] = w[0];
                f[HS / 4] = w[1];
                f[HS / 2] = w[2];
                f[HS / 4 * 3] = 0;
            }
        }
    }
    __syncthreads();

    const int r8 = ROWS == 8 ? lane >> 2 : 0, jj = lane & 3;
    const int r = rt * ROWS + r8;
    const int pos = r < rows ? q.begin + r / g : -1;  // the row's last token
    const float fs = qscale[r8];
    float m = -INFINITY, l = 0.0f, poison = 0.0f;
    // rows of 8: [column tile][2]; one row: [tile of 16 dims][2][2]
    float o[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = 0.0f;
    uint32_t qd[ROWS == 8 ? 1 : KS][2];  // one row: digit (lane / 4) % 4 of q, the B operand
    if constexpr (ROWS == 1) {
        const uint32_t* f = reinterpret_cast<const uint32_t*>(qfrag) + (lane >> 2 & 3) * (HS / 4) + jj;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qd[ks][0] = f[ks * 8];
            qd[ks][1] = f[ks * 8 + 4];
        }
    }

    // strides of an item in shared memory: 16 tokens on, 16 dims on (K), V's start
    const int cell = hs * P * 2;
    const int k16 = P < kItem ? cell : 256, kc = P < kItem ? 256 : kItem * 16;
    const int v0 = P < kItem ? cell / 2 : kItem * hs, v16 = P < kItem ? cell : hs * 16;
    // ldmatrix rows of this lane: matrix mi = lane / 8, row lane % 8
    const int mi = lane >> 3, mr = lane & 7, mj = mr >> 1;
    const int ktok = 4 * mj + 2 * ((mi >> 1) ? 1 - (mj >> 1) : mj >> 1) + (mr & 1);
    const int last_chunk = hs / 16 - 1;

    for (int j = 0; j < items; ++j) {
        const int slot = j % kSlots;
        const float2 sc_lane = slot == 0 ? sc_slot[0] : sc_slot[1];
        const uint32_t base = smem_addr(ring + slot * kItem * HS * 2);
        const bool ok = mbar_wait(&bars[warp * kSlots + slot], (uint32_t)((j / kSlots) & 1), err, DEV_TIMEOUT_FULL);
        if (!__all_sync(0xffffffffu, ok)) {
            // confirm the copies still in flight before anything else is written there
            for (int k = j; k < min(j + kSlots, items); ++k)
                mbar_wait(&bars[warp * kSlots + k % kSlots], (uint32_t)((k / kSlots) & 1), err, DEV_TIMEOUT_DRAIN);
            __syncwarp();
            break;
        }
        const int t0 = ta + (warp + kFewWarps * j) * kItem;
        float sk[2], sv[2];
        sk[0] = __shfl_sync(0xffffffffu, sc_lane.x, 0);
        sv[0] = __shfl_sync(0xffffffffu, sc_lane.y, 0);
        sk[1] = sk[0];
        sv[1] = sv[0];
        if (P < kItem) {
            sk[1] = __shfl_sync(0xffffffffu, sc_lane.x, 1);
            sv[1] = __shfl_sync(0xffffffffu, sc_lane.y, 1);
        }
        const bool two = t0 + 16 < tb;
        // a scale that is not finite takes the rows that see its page with it
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (!(sv[c] < INFINITY)) {
                if (t0 + 16 * c <= pos && (c == 0 || two)) poison = NAN;
                sv[c] = 0.0f;
            }
        // a page that the row does not see has no say in what its weights are relative to
        if (P < kItem) {
            if (t0 > pos) sv[0] = 0.0f;
            if (t0 + 16 > pos) sv[1] = 0.0f;
        }
        const float svm = fmaxf(sv[0], sv[1]);
        // the largest weight, 2^32 less an ulp; its first digit is a unit of the products
        constexpr float kOne = 4294967040.0f, kUnitOf = 16777216.0f / kOne;
        if constexpr (ROWS == 1) {
            // scores: the codes of 16 tokens are the A operand, q's digits the
            // columns 0-2 and, again, 4-6.  A lane so finds one digit pair or third
            // digit of four tokens, and trades with its neighbour for one token whole.
            int d[2][4];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) d[c][e] = kBiasBits;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (!EXACT && ks * 32 >= hs) break;
                const int chunk = EXACT ? 2 * ks + (mi >> 1) : min(2 * ks + (mi >> 1), last_chunk);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t k[4];
                    ldsm4(base + c * k16 + chunk * kc + ((mi & 1) * 8 + mr) * 16, k);
                    mma_s8(d[c], make_uint4(k[0], k[1], k[2], k[3]), qd[ks][0], qd[ks][1]);
                }
            }
            const bool odd = jj & 1, late = jj >> 1;  // the lane's token: 16 late + 8 odd + lane / 4
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = unbias(late ? d[1][e] : d[0][e]);
            const float y0 = odd ? y[0] : fmaf(y[0], 256.0f, y[1]), y1 = odd ? y[2] : fmaf(y[2], 256.0f, y[3]);
            const float mine = odd ? y1 : y0, other = __shfl_xor_sync(0xffffffffu, odd ? y0 : y1, 1);
            float x = (odd ? fmaf(other, 256.0f, mine) : fmaf(mine, 256.0f, other)) * (fs * (late ? sk[1] : sk[0]));
            const int at = 16 * late + 8 * odd + (lane >> 2);
            if (t0 + at > pos) x = -INFINITY;
            const float top = max_redux(x), top_new = fmaxf(m, top);
            const float mref = top_new == -INFINITY ? 0.0f : top_new;
            const float corr = exp2_fast(m - mref);  // 0 for the first tokens
            const float rise = exp2_fast(top - mref);
            m = top_new;
            const float p = exp2_fast(x - (top == -INFINITY ? 0.0f : top));
            l = fmaf(l, corr, p * rise);
            // the weight in fixed point; its bytes are the B operand's columns
            float w = p, of = svm * rise * kUnitOf;
            if (P < kItem) {  // two pages
                w = svm > 0.0f ? p * ((late ? sv[1] : sv[0]) / svm) : 0.0f;
                const float most = max_redux(w);
                w = most > kLeast ? w / most : 0.0f;
                of *= most;
            }
            uint32_t* wt = reinterpret_cast<uint32_t*>(weights) + warp * kItem;
            wt[at] = __float2uint_rn(w * kOne);
            __syncwarp();
            uint32_t b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 u = weights[warp * (kItem / 4) + 4 * i + jj];
                const int byte = 3 - min(lane >> 2, 3);
                const uint32_t sel = ((4u + byte) << 4) | byte;
                b[i] = __byte_perm(__byte_perm(u.x, u.y, sel), __byte_perm(u.z, u.w, sel), 0x5410u);
                if (lane >> 2 >= 4) b[i] = 0;
            }
            const bool turn = corr != 1.0f;  // alike in all lanes
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                if (!EXACT && t * 8 >= hs) break;
                uint32_t v[4];
                int e4[4] = {kBiasBits, kBiasBits, kBiasBits, kBiasBits};
                ldsm4(base + v0 + (mi >> 1) * v16 + (t * 8 + (mi & 1) * 8 + mr) * 16, v);
                mma_s8u8(e4, v, b[0], b[1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float& f = o[t + (e >> 1)][e & 1];
                    if (turn) f *= corr;
                    f = fmaf(unbias(e4[e]), of, f);
                }
            }
            __syncwarp();  // the weights are read
        } else {
            float top = -INFINITY;
            float x[4][2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // 16 tokens: tiles 2c and 2c + 1
                int d[2][NP][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[i][p][e] = kBiasBits;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (!EXACT && ks * 32 >= hs) break;
                    uint32_t b[4];
                    const int chunk = EXACT ? 2 * ks + (mi & 1) : min(2 * ks + (mi & 1), last_chunk);
                    ldsm4(base + c * k16 + chunk * kc + ktok * 16, b);
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        const uint4 f = qfrag[(ks * NP + p) * 32 + lane];
                        mma_s8(d[0][p], f, b[0], b[1]);
                        mma_s8(d[1][p], f, b[2], b[3]);
                    }
                }
                const float f = fs * sk[c];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int t = t0 + 16 * c + 4 * jj + 2 * (i ? 1 - (jj >> 1) : jj >> 1);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = fmaf(unbias(d[i][0][e]), 256.0f, unbias(d[i][0][2 + e]));
                        v = fmaf(v, 256.0f, unbias(d[i][1][e]));
                        v *= f;
                        if (t + e > pos) v = -INFINITY;
                        x[2 * c + i][e] = v;
                        top = fmaxf(top, v);
                    }
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float top_new = fmaxf(m, top), top_ref = top == -INFINITY ? 0.0f : top;
            const float mref = top_new == -INFINITY ? 0.0f : top_new;
            const float corr = exp2_fast(m - mref);  // 0 for the first tokens
            const float rise = exp2_fast(top - mref);
            m = top_new;
            float sum = 0.0f, of = svm * rise * kUnitOf;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    x[t][e] = exp2_fast(x[t][e] - top_ref);
                    sum += x[t][e];
                }
            l = fmaf(l, corr, sum * rise);
            if (P < kItem) {  // two pages
                float most = 0.0f;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const float w = svm > 0.0f ? sv[t / 2] / svm : 0.0f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[t][e] *= w;
                        most = fmaxf(most, x[t][e]);
                    }
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) x[t][e] = most > kLeast ? x[t][e] / most : 0.0f;
                of *= most;
            }
            // weights in fixed point; their bytes are the A operand
            uint4 pa, pb;
            uint32_t* pw[2] = {reinterpret_cast<uint32_t*>(&pa), reinterpret_cast<uint32_t*>(&pb)};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t u[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) u[i][e] = __float2uint_rn(x[2 * c + i][e] * kOne);
                const uint32_t order = jj < 2 ? 0x5410u : 0x1054u;
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // byte 3 - k of the four weights
                    const uint32_t sel = ((7u - k) << 4) | (3u - k);
                    const uint32_t word =
                        __byte_perm(__byte_perm(u[0][0], u[0][1], sel), __byte_perm(u[1][0], u[1][1], sel), order);
                    pw[k / 2][c * 2 + k % 2] = word;
                }
            }
            const bool turn = __any_sync(0xffffffffu, corr != 1.0f);
#pragma unroll
            for (int t = 0; t < NT; t += 2) {
                if (!EXACT && t * 8 >= hs) break;
                uint32_t b[4];
                ldsm4(base + v0 + (mi & 1) * v16 + ((t + (mi >> 1)) * 8 + mr) * 16, b);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    int d[4] = {kBiasBits, kBiasBits, kBiasBits, kBiasBits};
                    int d3[4] = {kBiasBits, kBiasBits, kBiasBits, kBiasBits};
                    mma_u8(d, pa, b[2 * i], b[2 * i + 1]);
                    mma_u8(d3, pb, b[2 * i], b[2 * i + 1]);
                    if (turn) {
                        o[t + i][0] *= corr;
                        o[t + i][1] *= corr;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = fmaf(unbias(d3[2 + e]), 0.00390625f, unbias(d3[e]));
                        v = fmaf(v, 0.00390625f, unbias(d[2 + e]));
                        v = fmaf(v, 0.00390625f, unbias(d[e]));
                        o[t + i][e] = fmaf(v, of, o[t + i][e]);
                    }
                }
            }
        }
        if (j + kSlots < items) {
            const float2 sc = issue(j + kSlots);
            if (slot == 0)
                sc_slot[0] = sc;
            else
                sc_slot[1] = sc;
        }
    }
    if constexpr (ROWS == 8) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
    } else {
        l = warp_sum(l);
    }

    // join the warps: [warp][ROWS][hs + 8] over the rings (8 more: a row's stores
    // then fall into other banks than its neighbours')
    __syncthreads();
    float* join = reinterpret_cast<float*>(ring_all);
    const int w1 = hs + 8;
    {
        float* mine = join + (warp * ROWS + r8) * w1;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!EXACT && t * 8 >= hs) break;
            if constexpr (ROWS == 8) {
                *reinterpret_cast<float2*>(mine + t * 8 + 2 * jj) = make_float2(o[t][0] + poison, o[t][1] + poison);
            } else {  // dim 8 t + lane / 4: two digits here, the others by the next lane
                float v = fmaf(o[t][1], 0.00390625f, o[t][0]);
                v = fmaf(__shfl_down_sync(0xffffffffu, v, 1), 1.52587890625e-5f, v);
                if (jj == 0) mine[t * 8 + (lane >> 2)] = v + poison;
            }
        }
        if (ROWS == 8 ? jj == 0 : lane == 0) {
            mine[hs] = m;
            mine[hs + 1] = l;
        }
    }
    __syncthreads();
    // the split's part, and how far it is to the next one's
    const int64_t hop = (int64_t)gridDim.x * ROWS * w1;
    float* part = a.part + blockIdx.y * hop + blockIdx.x * ROWS * w1;
    // W neighbouring dims of a row to a thread: one row has a thread for each dim
    constexpr int W = ROWS == 8 ? 4 : 1;
    auto finish = [&](int rr, int d, const float (&v)[W], float mm, float ll) {
        const int row = q.r0 + rr / g, head = h * g + rr % g;
        const int64_t at = (int64_t)row * a.ld_out + (int64_t)head * hs + d;
        if constexpr (W == 4)
            store_out4(a, at, {v[0] / ll, v[1] / ll, v[2] / ll, v[3] / ll});
        else
            store_out(a, at, v[0] / ll);
        if (a.lse && d == 0) a.lse[(int64_t)row * a.n_heads + head] = (mm + log2f(ll)) * kLn2;
    };
    const int shares = (top + 1 - rt * ROWS) * (hs / W);
    for (int i = tid; i < shares; i += kFewThreads) {
        const int row8 = i / (hs / W), d = i % (hs / W) * W;
        float mm = -INFINITY, ll = 0.0f, v[W] = {};
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) mm = fmaxf(mm, join[(w * ROWS + row8) * w1 + hs]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float* src = join + (w * ROWS + row8) * w1;
            const float c = exp2_fast(src[hs] - ref);
            ll = fmaf(src[hs + 1], c, ll);
            float x[W];
            if constexpr (W == 4)
                load_n<4, true>(src + d, x);
            else
                x[0] = src[d];
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] = fmaf(x[e], c, v[e]);
        }
        if (splits == 1) {
            finish(rt * ROWS + row8, d, v, mm, ll);
        } else {
            float* to = part + row8 * w1;
            if constexpr (W == 4)
                __stcg(reinterpret_cast<float4*>(to + d), make_float4(v[0], v[1], v[2], v[3]));
            else
                __stcg(to + d, v[0]);
            if (d == 0) __stcg(reinterpret_cast<float2*>(to + hs), make_float2(mm, ll));
        }
    }
    if (splits == 1) return;
    __syncthreads();
    if (tid == 0) {
        __threadfence();  // for the whole CTA: its stores were before the barrier
        int* cnt = a.cnt + s * (int)gridDim.x + blockIdx.x;
        const int n = atomicAdd(cnt, 1);
        last_flag = n == splits - 1;
        if (last_flag) *cnt = 0;  // as the next launch expects it
        __threadfence();
    }
    __syncthreads();
    if (!last_flag) return;
    // eight splits at a time, all their loads before the first use (one at a time
    // the join of three splits of 8 rows took 15 us)
    const float* all = part - split * hop;
    for (int i = tid; i < shares; i += kFewThreads) {
        const int row8 = i / (hs / W), d = i % (hs / W) * W;
        const float* src = all + row8 * w1;
        float mm = -INFINITY, ll = 0.0f, v[W] = {};
#pragma unroll 1
        for (int k = 0; k < splits; k += 8) {
            float x[8][W];
            float2 ml[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ml[e] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int c = 0; c < W; ++c) x[e][c] = 0.0f;
                if (k + e < splits) {
                    const float* from = src + (k + e) * hop;
                    if constexpr (W == 4) {
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(from + d));
                        x[e][0] = y.x, x[e][1] = y.y, x[e][2] = y.z, x[e][3] = y.w;
                    } else {
                        x[e][0] = __ldcg(from + d);
                    }
                    ml[e] = __ldcg(reinterpret_cast<const float2*>(from + hs));
                }
            }
            const float was = mm;
#pragma unroll
            for (int e = 0; e < 8; ++e) mm = fmaxf(mm, ml[e].x);
            const float ref = mm == -INFINITY ? 0.0f : mm, c = exp2_fast(was - ref);
            ll *= c;
#pragma unroll
            for (int z = 0; z < W; ++z) v[z] *= c;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = exp2_fast(ml[e].x - ref);
                ll = fmaf(ml[e].y, f, ll);
#pragma unroll
                for (int z = 0; z < W; ++z) v[z] = fmaf(x[e][z], f, v[z]);
            }
        }
        finish(rt * ROWS + row8, d, v, mm, ll);
    }
}

template <int PARTS, int HS, bool EXACT, int ROWS>
cudaError_t few_launch(const AttArgs& a, dim3 grid, cudaStream_t st) {
    auto kern = attend_few_kernel<PARTS, HS, EXACT, ROWS>;
    constexpr int join = kFewWarps * ROWS * (HS + 8) * 4;
    constexpr int smem = few_smem<HS>() > join ? few_smem<HS>() : join;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int PARTS, int ROWS>
cudaError_t few_launch(const AttArgs& a, dim3 grid, cudaStream_t st) {
    const int hs = a.c.head_size;
    if (hs == 64) return few_launch<PARTS, 64, true, ROWS>(a, grid, st);
    if (hs == 128) return few_launch<PARTS, 128, true, ROWS>(a, grid, st);
    if (hs == 256) return few_launch<PARTS, 256, true, ROWS>(a, grid, st);
    if (hs < 64) return few_launch<PARTS, 64, false, ROWS>(a, grid, st);
    if (hs < 128) return few_launch<PARTS, 128, false, ROWS>(a, grid, st);
    return few_launch<PARTS, 256, false, ROWS>(a, grid, st);
}

// ---------------------------------------------------------------------------
// Many rows per kv head (prompts): bound by arithmetic, on tcgen05.
//
// One CTA per NQ tiles of 128 (token, head) rows of a sequence and kv head,
// which walk the context together in tiles of TK tokens.  Codes become f16 or
// bf16 exactly.  q of the 16-bit types is taken as it is (K in q's type); an fp32
// row is scaled by a power of two to fill f16's range and is two f16 (22
// bits); the weights are one or two f16 (V in f16).  Products accumulate in
// fp32 in tensor memory.
//
//   warps 0-3, 4-7   softmax of one row tile each: a thread per row reads its
//                    scores from tensor memory, writes its weights over them
//                    as the A operand of the second product, 2 x (32 columns
//                    of scores -> 16 of f16 pairs, the second ones for fp32)
//   4 or 8 warps     convert codes: global -> registers (a tile ahead) -> f16 in
//                    shared memory (128-byte swizzle)
//   then 4 warps     the first (and the third) issue the MMAs, the second looks
//                    up pages and scales, up to four tiles ahead
//
// The 16-bit types keep two buffers of scores per row tile, of 64 tokens each:
// the next scores are computed while softmax is at these, and each row tile
// has an issuing warp of its own.  fp32's two parts do not leave the tensor
// pipe the time for such short tiles (an MMA of 64 columns takes as long as one
// of 128): one buffer of 128 tokens, a row tile's products run while the other
// is in softmax.
//
// s_K multiplies scores by 16-token granules (one FMA with the exponent's
// shift); s_V enters as its logarithm: a weight's exponent gets log2(s_V / the
// first s_V of the sequence), so O needs no second scaling, and the sum divides it
// out again per granule.  The maximum that a row follows is that of score plus
// logarithm, over what the row sees: the weights that count are the ones with bits,
// however far apart the pages' scales lie, and pages that a row does not see or
// hardly attends to take none.  O is rescaled only when that maximum has grown by
// more than 2^kGrow since its last one: weights are 2^kUnit at that maximum, 2^14 at
// most, and have 11 bits, down to 2^-31 of the largest (fp32: 22, down to 2^-36).
//
// Measured, 1024 rows at the end of 4096 tokens, 32 heads of 128: bf16 119 us
// (60 GFLOP, 505 TFLOP/s), fp32 162 us.  What bounds it is the conversion (93 us
// without it), then a row tile's chain from scores through softmax to the next
// product, which two row tiles on an SM hide only in part (tensor pipe and issue
// slots are both under half busy).  Tiles of 128 tokens with one buffer of scores
// were level in bf16, and slower in f16 with 8 heads to a kv head and pages of 16
// (176 us against 164) and at head size 64 (103 us against 98).

// Converting warps: codes to 16 bits are two or three instructions each, and with
// four warps they held up the 16-bit types (132 us in the case above, 85 us without
// any conversion).
constexpr int many_converters(int ns) { return ns == 2 ? 8 : 4; }
constexpr int many_threads(int ns) { return 32 * (8 + many_converters(ns) + 4); }
// A row's maximum may grow by 2^kGrow before O is rescaled.  Their sum is 14, of f16's
// 16 bits upwards (a score of some 10^7 rounds by a bit); what kGrow leaves to kUnit is
// what small weights keep.  fp32 with 11 + 3 160 us, 6 + 8 159 us, 4 + 10 154 us in the case
// above; f16 with 8 heads to a kv head 177, 161 and 159 us.
constexpr float grow_bits(int parts) { return parts == 2 ? 3.0f : 8.0f; }
// s_V relative to the sequence's first: beyond 2^kFar either way it counts as that,
// and as no less than 2^-kBelow of the largest so far, so that a weight's share of the sum
// (its product with `inv`) stays a normal number
constexpr float kFar = 100.0f, kBelow = 80.0f;

struct Granule {  // 16 tokens
    float sk, shift, inv, bad;  // s_K, log2(s_V / first), 2^-shift, NaN where s_V is not finite
};

struct ManyBars {
    uint64_t qfull[2], kfull[4], kempty[4], vfull[4], vempty[4], sfull[2][2], pfull[2][2], pvdone[2], last[2], done[2];
    uint64_t tabfull[4], tabempty[4];
    uint32_t tmem_base;
    int abort_flag;
    float first;         // the s_V that the others are relative to
    Granule gran[4][8];  // by tile, four deep
    int64_t cell[4][8];  // the granules' pages: byte offset of the head's codes, or -1
    float fs[256];       // rows' factors of the scores
};

// NQ row tiles, TK tokens a tile, NS score buffers per row tile, NB buffers of K and of V
template <int HS, int TYPE, int NQ, int TK, int NS, int NB>
struct ManyLayout {
    static constexpr int kParts = TYPE == LQ_F32 ? 2 : 1;
    static constexpr int kQ = 128 * HS * 2 * kParts;       // one row tile: [part][64 dims][128][128 bytes]
    static constexpr int kK = TK * HS * 2, kV = TK * HS * 2;
    static constexpr int kSmem = 1024 + NQ * kQ + NB * (kK + kV) + (int)sizeof(ManyBars);
    static_assert(kSmem <= 227 * 1024 && HS % 64 == 0, "shared memory");
    static_assert(NQ * (NS * TK + HS) <= 512, "tensor memory");
};

// 4 codes to 2 x 2 f16: bytes + 128 as the low mantissa of 1024, minus 1152
__device__ __forceinline__ uint2 codes_f16(uint32_t w) {
    w ^= 0x80808080u;
    const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off);
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// 4 codes to 2 x 2 bf16, times 2^-16 (kBf16Codes undoes it): the low 7 bits as the
// mantissa of 128, minus 128 (a code of 0 to 127) or 256 (a negative one), which its
// sign bit makes of 128.  Any finite q of bf16 then has dots within fp32's range.
constexpr float kBf16Codes = 65536.0f;
__device__ __forceinline__ uint2 codes_bf16(uint32_t w) {
    auto two = [](uint32_t x) {
        const uint32_t m = (x & 0x007F007Fu) | 0x3B003B00u, off = (x & 0x00800080u) | 0x3B003B00u;
        const __nv_bfloat162 r =
            __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&m), *reinterpret_cast<const __nv_bfloat162*>(&off));
        return *reinterpret_cast<const uint32_t*>(&r);
    };
    return make_uint2(two(__byte_perm(w, 0, 0x4140)), two(__byte_perm(w, 0, 0x4342)));
}

// 16 codes to two 16-byte chunks (2 * pair, 2 * pair + 1) of row `row` of 128-byte swizzled rows
template <bool BF16>
__device__ __forceinline__ void put_codes(unsigned char* block, int row, int pair, uint4 w) {
    const uint2 x = BF16 ? codes_bf16(w.x) : codes_f16(w.x), y = BF16 ? codes_bf16(w.y) : codes_f16(w.y);
    const uint2 z = BF16 ? codes_bf16(w.z) : codes_f16(w.z), u = BF16 ? codes_bf16(w.w) : codes_f16(w.w);
    const uint32_t at = row * 128 + ((row & 7) << 4);
    *reinterpret_cast<uint4*>(block + (at ^ (pair << 5))) = make_uint4(x.x, x.y, y.x, y.y);
    *reinterpret_cast<uint4*>(block + (at ^ (pair << 5) ^ 16)) = make_uint4(z.x, z.y, u.x, u.y);
}

template <int HS, int TYPE, int NQ, int TK, int NS, int NB, bool EXACT>
__global__ void __launch_bounds__(many_threads(NS), 1) attend_many_kernel(const __grid_constant__ AttArgs a) {
    using Lay = ManyLayout<HS, TYPE, NQ, TK, NS, NB>;
    constexpr int kIssuers = NS == 2 ? NQ : 1;  // warps that issue MMAs: one per row tile, or one for all
    constexpr int PARTS = Lay::kParts;
    constexpr bool kBf16 = TYPE == LQ_BF16;
    constexpr float kGrow = grow_bits(PARTS), kUnit = 14.0f - kGrow;
    constexpr int kConv = many_converters(NS), kIssue = 8 + kConv;  // converting warps; the first issuing warp
    constexpr int kLoads = HS / 16 * TK / (32 * kConv);  // 16-byte pieces of K (and of V) per converting thread
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    unsigned char *sq = sm, *sk = sq + NQ * Lay::kQ, *sv = sk + NB * Lay::kK;
    ManyBars* bars = reinterpret_cast<ManyBars*>(sv + NB * Lay::kV);
    volatile int* abort_flag = &bars->abort_flag;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hs = EXACT ? HS : a.c.head_size;
    const int P = a.c.page_size, H = a.c.n_kv_heads, g = a.group;
    const int tile = gridDim.x - 1 - blockIdx.x;  // long ones first
    const int h = blockIdx.y, s = blockIdx.z;

    pdl_wait();
    const SeqRows q = seq_rows(a.b, s, a.few_rows == 0 && tile == 0 && h == 0 && tid == 0 ? a.err : nullptr);
    const int rows = q.n * g, base_row = tile * NQ * 128;
    if (a.few_rows == 0 && tile == 0) zero_rows(a, q, h);
    if (rows <= a.few_rows || base_row >= rows) return;
    int n[NQ];  // token tiles that each row tile sees
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int lo = base_row + i * 128, hi = min(rows, lo + 128) - 1;
        n[i] = lo < rows ? (q.begin + hi / g) / TK + 1 : 0;
    }
    int tiles = n[0];
    if (NQ == 2 && n[NQ - 1] > tiles) tiles = n[NQ - 1];
    const int seen = q.begin + (min(rows, base_row + NQ * 128) - 1) / g + 1;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->qfull[i], 4);
            for (int b = 0; b < 2; ++b) {
                mbar_init(&bars->sfull[i][b], 1);
                mbar_init(&bars->pfull[i][b], 4);
            }
            mbar_init(&bars->pvdone[i], 1);
            mbar_init(&bars->last[i], 1);
            mbar_init(&bars->done[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bars->tabfull[i], 1);
            mbar_init(&bars->tabempty[i], kIssuers);
            mbar_init(&bars->kfull[i], kConv);
            mbar_init(&bars->vfull[i], kConv);
            mbar_init(&bars->kempty[i], kIssuers);
            mbar_init(&bars->vempty[i], kIssuers);
        }
        bars->abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kIssue) tmem_alloc<1, 512>(&bars->tmem_base);
    const int lp2 = __ffs(P) - 1;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    // not before: a later kernel that takes tensor memory while it waits for this one
    // (matmul_rows) would keep it from CTAs of this one that have none yet
    pdl_trigger();
    const int8_t* codes = static_cast<const int8_t*>(a.c.codes);

    // 512 threads have 128 registers each; 128 scores a thread take a larger share,
    // dealt to warpgroups within that sum
    constexpr bool kDeal = NS == 1;
    constexpr int kSoftRegs = 168, kConvRegs = 104, kIssueRegs = 72;
    static_assert(!kDeal || 8 * kSoftRegs + kConv * kConvRegs + 4 * kIssueRegs <= (12 + kConv) * 128, "registers");
    if (warp >= 8 && warp < kIssue) {
        // ---------------- conversion ----------------
        if constexpr (kDeal) regs_down<kConvRegs>();
        const int t = tid - 256;
        uint4 kr[kLoads], vr[kLoads];
        // K: token t % TK, every kcs-th piece of its dims
        constexpr int kcs = 32 * kConv / TK;
        const int kt = t % TK, kc0 = t / TK;
        // V: every 32 * kConv-th piece of the tile: piece tc * hs + d is 16 tokens of dim d
        int pd[kLoads], ptc[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            ptc[i] = (t + 32 * kConv * i) / hs;
            pd[i] = (t + 32 * kConv * i) - ptc[i] * hs;
        }
        bool ok = true;
        auto load_k = [&](int j) {
            ok = ok && __all_sync(0xffffffffu, qwait(&bars->tabfull[j & 3], (uint32_t)((j >> 2) & 1), a.err,
                                                     DEV_TIMEOUT_FULL, abort_flag));
            const int64_t at = ok ? bars->cell[j & 3][kt >> 4] : -1;
            const uint4* src = reinterpret_cast<const uint4*>(codes + at) + ((j * TK + kt) & (P - 1));
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int c = kc0 + i * kcs;
                kr[i] = at >= 0 && c * 16 < hs ? ld_after(src + c * P) : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_v = [&](int j) {  // after load_k(j)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int64_t at = ok && ptc[i] < TK / 16 ? bars->cell[j & 3][ptc[i]] : -1;
                const uint4* src = reinterpret_cast<const uint4*>(codes + at) + (hs >> 4) * P +
                                   (((j * TK + ptc[i] * 16) & (P - 1)) >> 4) * hs + pd[i];
                vr[i] = at >= 0 ? ld_after(src) : make_uint4(0, 0, 0, 0);
            }
        };
        load_k(0);
        load_v(0);
        for (int j = 0; j < tiles; ++j) {
            const int buf = j % NB;
            const uint32_t par = (uint32_t)((j / NB) & 1);
            ok = ok && __all_sync(0xffffffffu, qwait(&bars->kempty[buf], par ^ 1u, a.err, DEV_TIMEOUT_EMPTY, abort_flag));
            if (!ok) break;
            unsigned char* kb = sk + buf * Lay::kK;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int c = kc0 + i * kcs;
                if (c * 16 < hs) put_codes<kBf16>(kb + (c >> 2) * (TK * 128), kt, c & 3, kr[i]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->kfull[buf]);
            if (j + 1 < tiles) load_k(j + 1);
            ok = ok && __all_sync(0xffffffffu, qwait(&bars->vempty[buf], par ^ 1u, a.err, DEV_TIMEOUT_EMPTY, abort_flag));
            if (!ok) break;
            unsigned char* vb = sv + buf * Lay::kV;
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (ptc[i] < TK / 16) put_codes<false>(vb + (ptc[i] >> 2) * (hs * 128), pd[i], ptc[i] & 3, vr[i]);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->vfull[buf]);
            if (j + 1 < tiles) load_v(j + 1);
        }
    } else if (warp >= kIssue) {
        if constexpr (kDeal) regs_down<kIssueRegs>();
        if ((warp - kIssue) / 2 < kIssuers && warp % 2 == 0) {
            // ---------------- MMA issue ----------------
            // f32 += f16 x f16 (or bf16 x bf16), M 128
            const uint32_t id_s =
                (1u << 4) | (kBf16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)(TK >> 3) << 17) | (8u << 24);
            const uint32_t id_o = (1u << 4) | ((uint32_t)(hs >> 3) << 17) | (8u << 24);
            const uint64_t dq = smem_desc_sw128(smem_addr(sq)), dk = smem_desc_sw128(smem_addr(sk)),
                           dv = smem_desc_sw128(smem_addr(sv));
            const int steps = hs / 16, me = (warp - kIssue) / 2;
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                ok = ok && __all_sync(0xffffffffu, qwait(bar, parity, a.err, code, abort_flag));
            };
            // whether this warp's last use of token tile j is row tile i's
            auto last_use = [&](int i, int j) { return NS == 2 || i == NQ - 1 || j >= n[NQ - 1]; };
            auto scores = [&](int i, int j) {  // row tile i, token tile j
                if (NS == 1 && j >= n[i]) return;
                wait(&bars->kfull[j % NB], (uint32_t)((j / NB) & 1), DEV_TIMEOUT_FULL);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    if (j < n[i]) {
                        const uint32_t dst = tmem + (i * NS + j % NS) * TK;
                        const uint64_t kd = dk + (uint32_t)((j % NB) * Lay::kK >> 4);
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) {
                            const uint64_t qd = dq + (uint32_t)((i * Lay::kQ + p * (Lay::kQ / PARTS)) >> 4);
                            for (int k = 0; k < steps; ++k)  // 64 dims a block of 128-byte rows, 32 bytes a step
                                mma_f16(dst, qd + (uint32_t)((k >> 2) * (128 * 128) >> 4) + 2 * (k & 3),
                                        kd + (uint32_t)((k >> 2) * (TK * 128) >> 4) + 2 * (k & 3), id_s, k > 0 || p > 0);
                        }
                        mma_commit(&bars->sfull[i][j % NS]);
                        if (last_use(i, j)) mma_commit(&bars->kempty[j % NB]);
                    } else {  // not a tile of this row tile's
                        mbar_arrive(&bars->kempty[j % NB]);
                    }
                }
                __syncwarp();
            };
            auto values = [&](int i, int j) {
                if (NS == 1 && j >= n[i]) return;
                if (j < n[i]) wait(&bars->pfull[i][j % NS], (uint32_t)((j / NS) & 1), DEV_TIMEOUT_FULL);
                wait(&bars->vfull[j % NB], (uint32_t)((j / NB) & 1), DEV_TIMEOUT_FULL);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
                    if (j < n[i]) {
                        const uint32_t dst = tmem + NQ * NS * TK + i * HS, src = tmem + (i * NS + j % NS) * TK;
                        const uint64_t vd = dv + (uint32_t)((j % NB) * Lay::kV >> 4);
#pragma unroll
                        for (int k = 0; k < TK / 16; ++k)
#pragma unroll
                            for (int p = 0; p < PARTS; ++p)
                                mma_f16_ts(dst, src + (k >> 1) * 32 + p * 16 + (k & 1) * 8,
                                           vd + (uint32_t)((k >> 2) * (hs * 128) >> 4) + 2 * (k & 3), id_o,
                                           j > 0 || k > 0 || p > 0);
                        // the last tile's on a barrier of its own: softmax may come to it
                        // before the tile before it is done, whose phase has the other parity
                        mma_commit(j == n[i] - 1 ? &bars->last[i] : &bars->pvdone[i]);
                        if (last_use(i, j)) {
                            mma_commit(&bars->vempty[j % NB]);
                            mma_commit(&bars->tabempty[j & 3]);
                        }
                    } else {
                        mbar_arrive(&bars->vempty[j % NB]);
                        mbar_arrive(&bars->tabempty[j & 3]);
                    }
                }
                __syncwarp();
            };
            if constexpr (NS == 2) {
                if (n[me] > 0) wait(&bars->qfull[me], 0, DEV_TIMEOUT_FULL);
                if (ok) scores(me, 0);
                for (int j = 0; ok && j < tiles; ++j) {
                    if (j + 1 < tiles) scores(me, j + 1);
                    if (ok) values(me, j);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NQ; ++i)
                    if (ok && n[i] > 0) {
                        wait(&bars->qfull[i], 0, DEV_TIMEOUT_FULL);
                        if (ok) scores(i, 0);
                    }
                for (int j = 0; ok && j < tiles; ++j) {
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        if (ok) values(i, j);
                        if (ok) scores(i, j + 1);
                    }
                }
            }
            if (elect_one()) mma_commit(&bars->done[me]);
            __syncwarp();
            mbar_wait(&bars->done[me], 0, a.err, DEV_TIMEOUT_MMA);  // every MMA is done before the memory is freed
        } else if (warp == kIssue + 1) {
            // ---------------- pages and scales ----------------
            // a granule a lane, the next 32 looked up while these are handed out: two
            // dependent loads from memory for each tile took longer than its products
            constexpr int kGran = TK / 16, kRound = 32 / kGran;  // granules of a tile, tiles of a round
            int64_t p = -1, p_next = -1;
            float2 sc = make_float2(NAN, NAN), sc_next = sc;
            auto look_up = [&](int j) {  // tiles j .. j + kRound - 1
                const int tok = (j * kGran + lane) * 16;
                p_next = -1;
                sc_next = make_float2(NAN, NAN);
                if (tok < seen) {
                    p_next = page_of(a.c, a.b, s, tok >> lp2, a.err);
                    if (p_next >= 0) sc_next = ld_after(reinterpret_cast<const float2*>(a.c.scales) + p_next * H + h);
                }
            };
            Granule gr = {};
            float first = 1.0f, most = -kFar;
            look_up(0);
            for (int j = 0; j < tiles; ++j) {
                if (j % kRound == 0) {
                    p = p_next;
                    sc = sc_next;
                    look_up(j + kRound);
                    const bool fine = sc.y < INFINITY;
                    if (j == 0) {
                        const uint32_t some = __ballot_sync(0xffffffffu, fine && sc.y > 0.0f);
                        if (some) first = __shfl_sync(0xffffffffu, sc.y, __ffs(some) - 1);
                        if (lane == 0) bars->first = first;
                    }
                    float shift = fine ? fminf(fmaxf(log2f(sc.y / first), -kFar), kFar) : -kFar, up = shift;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {  // the largest up to this granule
                        const float x = __shfl_up_sync(0xffffffffu, up, o);
                        if (lane >= o) up = fmaxf(up, x);
                    }
                    up = fmaxf(up, most);
                    most = __shfl_sync(0xffffffffu, up, 31);
                    shift = fmaxf(shift, up - kBelow);
                    gr = {sc.x, shift, exp2f(-shift), fine ? 0.0f : NAN};
                }
                if (!__all_sync(0xffffffffu, qwait(&bars->tabempty[j & 3], (uint32_t)(((j >> 2) & 1) ^ 1), a.err,
                                                   DEV_TIMEOUT_EMPTY, abort_flag)))
                    break;
                const int i = lane - j % kRound * kGran;
                if (i >= 0 && i < kGran) {
                    bars->gran[j & 3][i] = gr;
                    bars->cell[j & 3][i] = p >= 0 ? (p * H + h) * (int64_t)(hs * P * 2) : -1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->tabfull[j & 3]);
            }
        }
    } else {
        // ---------------- softmax ----------------
        if constexpr (kDeal) regs_up<kSoftRegs>();
        if (warp < 4 * NQ && (warp < 4 ? n[0] : n[NQ - 1]) > 0) {
            const int i = warp >> 2, w4 = warp & 3;
            const int n_i = i == 0 ? n[0] : n[NQ - 1];
            // q of this warp's 32 rows
            const int first = base_row + i * 128 + w4 * 32;
            if constexpr (PARTS == 1) {
                // as it is, in 16-byte pieces: a short loop of asynchronous copies (its
                // unrolled form was bound by fetching instructions that run once)
                const int per = hs / 8;  // pieces of a row
#pragma unroll 1
                for (int pc = lane; pc < 32 * per; pc += 32) {
                    const int rr = pc / per, ck = pc - rr * per, row = w4 * 32 + rr, r = min(first + rr, rows - 1);
                    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (int64_t)(q.r0 + r / g) * a.ld_q +
                                          (int64_t)(h * g + r % g) * hs + ck * 8;
                    unsigned char* dst =
                        sq + i * Lay::kQ + (ck >> 3) * (128 * 128) + row * 128 + (((ck & 7) ^ (row & 7)) << 4);
                    if (a.q_vec) {
                        cp_async16(dst, src);
                    } else {
                        for (int k = 0; k < 8; ++k) reinterpret_cast<uint16_t*>(dst)[k] = ld_after(src + k);
                    }
                }
                cp_async_wait();
                bars->fs[i * 128 + w4 * 32 + lane] = fabsf(a.scale) * (kBf16 ? kBf16Codes : 1.0f);
            } else {
                // scaled and split, a few rows at a time (all their loads before the
                // first use), 4 dims a lane
                constexpr int kB = (HS + 127) / 128, kBatch = 8 / kB;
                int tok = min(first, rows - 1) / g, head = min(first, rows - 1) - tok * g;
                for (int r0 = 0; r0 < 32; r0 += kBatch) {
                    RawQ<2> raw[kBatch][kB];
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const int64_t at = (int64_t)(q.r0 + tok) * a.ld_q + (int64_t)(h * g + head) * hs;
#pragma unroll
                        for (int b = 0; b < kB; ++b) raw[u][b].load(a, at + min(b * 128 + lane * 4, hs - 4));
                        if (first + r0 + u + 1 < rows && ++head == g) {
                            head = 0;
                            ++tok;
                        }
                    }
                    float x[kBatch][kB][4];
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const bool have = first + r0 + u < rows;
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            raw[u][b].get(a, x[u][b]);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (!have || b * 128 + lane * 4 >= hs) x[u][b][e] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        const int row = w4 * 32 + r0 + u;
                        uint32_t m = 0;
#pragma unroll
                        for (int b = 0; b < kB; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) m = max(m, abs_bits(x[u][b][e]));
                        m = __reduce_max_sync(0xffffffffu, m);
                        // a power of two that takes the largest into [2^13, 2^14)
                        int ex = (int)(m >> 23) - 127;
                        ex = max(-114, min(100, 13 - ex));
                        const float up = m >= kInfBits ? 0.0f : a.scale < 0.0f ? -lq_exp2i(ex) : lq_exp2i(ex);
                        if (lane == 0) bars->fs[i * 128 + row] = m >= kInfBits ? NAN : fabsf(a.scale) * lq_exp2i(-ex);
#pragma unroll
                        for (int b = 0; b < kB; ++b) {
                            const int d = b * 128 + lane * 4;
                            if (d >= hs) continue;
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[u][b][e] = up == 0.0f ? 0.0f : x[u][b][e] * up;
#pragma unroll
                            for (int p = 0; p < PARTS; ++p) {
                                const uint32_t w0 = pack_word<__half>(x[u][b]), w1 = pack_word<__half>(x[u][b] + 2);
                                unsigned char* dst = sq + i * Lay::kQ + p * (Lay::kQ / PARTS) + (d >> 6) * (128 * 128) +
                                                     row * 128 + ((((d & 63) >> 3) ^ (row & 7)) << 4) + (d & 4) * 2;
                                *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
                                if (p + 1 < PARTS) {  // what the first part leaves
                                    float y[4];
                                    unpack_word<__half>(w0, y);
                                    unpack_word<__half>(w1, y + 2);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) x[u][b][e] -= y[e];
                                }
                            }
                        }
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->qfull[i]);

            const int row = w4 * 32 + lane, r = base_row + i * 128 + row;
            const int pos = r < rows ? q.begin + r / g : -1;
            const float fs = bars->fs[i * 128 + row];
            const uint32_t to = tmem + ((uint32_t)(w4 * 32) << 16) + NQ * NS * TK + i * HS;
            float mref = 0.0f, l = 0.0f, poison = 0.0f;
            bool ok = true;
            for (int j = 0; j < n_i; ++j) {
                ok = __all_sync(0xffffffffu, qwait(&bars->sfull[i][j % NS], (uint32_t)((j / NS) & 1), a.err,
                                                    DEV_TIMEOUT_TFULL, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint32_t ts = tmem + ((uint32_t)(w4 * 32) << 16) + (i * NS + j % NS) * TK;
                const Granule* gr = bars->gran[j & 3];
                const int left = pos - j * TK;  // the tile's last token that this row sees
                float x[TK / 32][32];
#pragma unroll
                for (int c = 0; c < TK / 32; ++c) tmem_ld<32>(ts + c * 32, reinterpret_cast<int(&)[32]>(x[c]));
                tmem_ld_wait();
                if (PARTS == 1 && a.scale < 0.0f) {  // the factors are positive
#pragma unroll
                    for (int c = 0; c < TK / 32; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[c][k] = -x[c][k];
                }
                if (__any_sync(0xffffffffu, left < TK - 1)) {
#pragma unroll
                    for (int c = 0; c < TK / 32; ++c)
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (c * 32 + k > left) x[c][k] = -INFINITY;
                }
                float m = -INFINITY;
#pragma unroll
                for (int e = 0; e < TK / 16; ++e) {
                    const float* y = &x[e / 2][(e & 1) * 16];
                    float t[5];
#pragma unroll
                    for (int k = 0; k < 5; ++k) t[k] = max3(y[3 * k], y[3 * k + 1], y[3 * k + 2]);
                    m = fmaxf(m, fmaf(fmaxf(max3(t[0], t[1], t[2]), max3(t[3], t[4], y[15])), fs * gr[e].sk, gr[e].shift));
                }
                const bool grown = j == 0 ? m > -INFINITY : m > mref + (kUnit + kGrow);
                if (__any_sync(0xffffffffu, grown)) {
                    const float next = grown ? m - kUnit : mref;
                    const float f = exp2_fast(mref - next);
                    mref = next;
                    if (j > 0) {
                        l *= f;
                        if constexpr (NS == 2) {  // else the scores were issued after the product before them
                            ok = __all_sync(0xffffffffu, qwait(&bars->pvdone[i], (uint32_t)((j - 1) & 1), a.err,
                                                               DEV_TIMEOUT_TFULL, abort_flag));
                            if (!ok) break;
                        }
                        tc_fence_after();
                        // a short loop: it runs rarely, and fetching its instructions took
                        // longer than they do (fp32 170 us unrolled, 162 us)
#pragma unroll 1
                        for (int c = 0; c < hs; c += 16) {
                            int y[16];
                            tmem_ld<16>(to + c, y);
                            tmem_ld_wait();
                            uint32_t z[16];
#pragma unroll
                            for (int k = 0; k < 16; ++k) z[k] = __float_as_uint(__int_as_float(y[k]) * f);
                            tmem_st16(to + c, z);
                        }
                    }
                }
                uint64_t total[2] = {};
#pragma unroll
                for (int c = 0; c < TK / 32; ++c) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const Granule gg = gr[2 * c + e];
                        // a masked -infinity has to stay one: no factor of zero, and
                        // no NaN from a granule that the row does not see
                        const bool sees = c * 32 + e * 16 <= left;
                        float f = sees ? fs * gg.sk : 1.4e-45f;
                        if (f == 0.0f) f = 1.4e-45f;
                        if (sees) poison += gg.bad;
                        const uint64_t f2 = f2_pack(f, f), b2 = f2_pack(gg.shift - mref, gg.shift - mref);
                        uint64_t sum[2];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint64_t z = f2_fma(f2_pack(x[c][e * 16 + 2 * k], x[c][e * 16 + 2 * k + 1]), f2, b2);
                            const float y[2] = {exp2_fast(f2_lo(z)), exp2_fast(f2_hi(z))};
                            const uint64_t w = f2_pack(y[0], y[1]);
                            sum[k & 1] = k < 2 ? w : f2_add(sum[k & 1], w);
                            hi[e * 8 + k] = pack_word<__half>(y);
                            if (PARTS == 2) {
                                float u[2];
                                unpack_word<__half>(hi[e * 8 + k], u);
                                u[0] = y[0] - u[0];
                                u[1] = y[1] - u[1];
                                lo[e * 8 + k] = pack_word<__half>(u);
                            }
                        }
                        total[e] = f2_fma(f2_add(sum[0], sum[1]), f2_pack(gg.inv, gg.inv), total[e]);
                    }
                    tmem_st16(ts + c * 32, hi);
                    if (PARTS == 2) tmem_st16(ts + c * 32 + 16, lo);
                }
                l += (f2_lo(total[0]) + f2_hi(total[0])) + (f2_lo(total[1]) + f2_hi(total[1]));
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->pfull[i][j % NS]);
            }
            if (ok)
                ok = __all_sync(0xffffffffu, qwait(&bars->last[i], 0, a.err, DEV_TIMEOUT_TFULL, abort_flag));
            tc_fence_after();
            if (ok) {
                const float f = bars->first / l;
                const int64_t at = (int64_t)(q.r0 + r / g) * a.ld_out + (int64_t)(h * g + r % g) * hs;
                for (int c = 0; c < hs; c += 16) {
                    int y[16];
                    tmem_ld<16>(to + c, y);
                    tmem_ld_wait();
                    if (r < rows) store_row16(a, at + c, y, f, poison);
                }
                if (a.lse && r < rows)
                    a.lse[(int64_t)(q.r0 + r / g) * a.n_heads + h * g + r % g] = (mref + log2f(l)) * kLn2;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssue) {
        tc_fence_after();
        tmem_free<1, 512>(tmem);
    }
}

template <int HS, int TYPE, int NQ, int TK, int NS, int NB, bool EXACT>
cudaError_t many_launch_t(const AttArgs& a, cudaStream_t st) {
    using Lay = ManyLayout<HS, TYPE, NQ, TK, NS, NB>;
    auto kern = attend_many_kernel<HS, TYPE, NQ, TK, NS, NB, EXACT>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Lay::kSmem);
    if (e != cudaSuccess) return e;
    const int64_t x = ((int64_t)a.b.max_rows * a.group + NQ * 128 - 1) / (NQ * 128);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)x, (unsigned)a.c.n_kv_heads, (unsigned)a.b.n_seqs);
    cfg.blockDim = dim3(many_threads(NS));
    cfg.dynamicSmemBytes = Lay::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

// Two row tiles of 128 up to 128 dims, one beyond (their accumulators and
// operands would not fit twice); 64 and 128 dims with their addresses at compile
// time.
template <int TYPE>
cudaError_t many_launch(const AttArgs& a, cudaStream_t st) {
    constexpr bool f32 = TYPE == LQ_F32;
    constexpr int TK = f32 ? 128 : 64, NS = f32 ? 1 : 2;
    const int hs = a.c.head_size;
    if (hs == 64) return many_launch_t<64, TYPE, 2, TK, NS, f32 ? 2 : 4, true>(a, st);
    if (hs == 128) return many_launch_t<128, TYPE, 2, TK, NS, f32 ? 1 : 3, true>(a, st);
    if (hs < 64) return many_launch_t<64, TYPE, 2, TK, NS, f32 ? 2 : 4, false>(a, st);
    if (hs < 128) return many_launch_t<128, TYPE, 2, TK, NS, f32 ? 1 : 3, false>(a, st);
    return many_launch_t<256, TYPE, 1, f32 ? 64 : 128, 1, 1, false>(a, st);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" int paged_attention(void* out, int64_t ld_out, const void* q, int64_t ld_q, int type, int n_heads,
                               const PagedKV* cache, const KVBatch* batch, float scale, float* lse) {
    int rc = check_paged(cache, batch, n_heads, type, "paged_attention");
    if (rc) return rc;
    if (n_heads <= 0) return lq_fail(LQ_EINVAL, "paged_attention: %d query heads", n_heads);
    if (!(scale == scale) || std::isinf(scale)) return lq_fail(LQ_EINVAL, "paged_attention: scale is not finite");
    if (batch->n_seqs == 0 || batch->n_rows == 0) return LQ_OK;
    const int64_t row = (int64_t)n_heads * cache->head_size;
    if (!out || !q || ld_out < row || ld_q < row)
        return lq_fail(LQ_EINVAL, "paged_attention: out or q not set, or rows closer than %lld elements", (long long)row);
    const uintptr_t size = type == LQ_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % size || reinterpret_cast<uintptr_t>(q) % size ||
        (reinterpret_cast<uintptr_t>(lse) & 3u))
        return lq_fail(LQ_EINVAL, "paged_attention: a tensor is not aligned to its elements");
    DevCtx* c = ctx();
    if (!c) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
    AttArgs a = {};
    a.c = *cache;
    a.b = *batch;
    if (a.b.max_rows > a.b.n_rows) a.b.max_rows = a.b.n_rows;  // a bound, however far above: grids follow it
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.ld_q = ld_q;
    a.ld_out = ld_out;
    a.n_heads = n_heads;
    a.group = n_heads / cache->n_kv_heads;
    a.type = type;
    a.q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld_q * size % 16 == 0;
    a.scale = scale * kLog2e;
    a.err = c->err;
    // few rows: every (sequence, kv head, row tile) is cut into splits of the context
    const int64_t most_rows = (int64_t)a.b.max_rows * a.group;
    const int tile_rows = most_rows <= 1 ? 1 : 8;
    a.row_tiles = (int)(((most_rows < kFewRows ? most_rows : kFewRows) + tile_rows - 1) / tile_rows);
    if (a.row_tiles < 1) a.row_tiles = 1;
    // Splits of contexts, as many as find a CTA slot each (few_ctas of them to an
    // SM): a second round costs more than uneven contexts (16 sequences of the 70B
    // shape 26 us in one, 32 us in two).
    const int64_t x = (int64_t)cache->n_kv_heads * a.row_tiles;
    const int64_t slots = few_ctas(cache->head_size, tile_rows) * c->num_sms;
    const int64_t most_splits = (int64_t)batch->n_seqs * ((batch->max_context + 255) / 256);
    int64_t units = slots / x < most_splits ? slots / x : most_splits;
    a.plan = units > batch->n_seqs;
    if (!a.plan) units = batch->n_seqs;
    void* part = nullptr;
    if (a.plan) {
        rc = stream_workspace(c, (size_t)(units * x * tile_rows * (cache->head_size + 8)) * sizeof(float), &a.cnt, &part);
        if (rc) return rc;
    }
    a.part = static_cast<float*>(part);
    // one sequence with many rows leaves nothing to the first kernel
    a.few_rows = batch->n_seqs == 1 && most_rows > kFewRows && (int64_t)batch->n_rows * a.group > kFewRows ? 0 : kFewRows;
    const dim3 grid((unsigned)x, (unsigned)units);
    cudaError_t e = cudaSuccess;
    if (a.few_rows && tile_rows == 1)
        e = type == LQ_F32 ? few_launch<2, 1>(a, grid, stream()) : few_launch<1, 1>(a, grid, stream());
    else if (a.few_rows)
        e = type == LQ_F32 ? few_launch<2, 8>(a, grid, stream()) : few_launch<1, 8>(a, grid, stream());
    if (e != cudaSuccess) return cuda_fail(e, "paged_attention launch");
    if (most_rows > kFewRows) {
        e = type == LQ_F32   ? many_launch<LQ_F32>(a, stream())
            : type == LQ_F16 ? many_launch<LQ_F16>(a, stream())
                             : many_launch<LQ_BF16>(a, stream());
        if (e != cudaSuccess) return cuda_fail(e, "paged_attention launch");
    }
    return LQ_OK;
}
