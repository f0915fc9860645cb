// kv_append: rotation by position, int8 quantization into the paged cache, and
// the host checks that the paged-cache entry points share.
#include <cmath>

#include "lq_ctx.h"
#include "lq_paged.cuh"
#include "lq_paged_host.h"
#include "lq_types.cuh"

namespace lq {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;

struct AppendArgs {
    PagedKV c;
    KVBatch b;
    KVRows r;
    int* err;
    int kv_blocks;  // blocks for keys and values; the others rotate queries
    int q_parts;    // warps that share a row of queries
};

// dims d .. d + 3 of a row, rotated as its position asks.  d is a multiple of
// 4.  The products and sums are separate fp32 operations (no fused multiply-add).
template <typename T, bool VEC>
__device__ __forceinline__ void rotated4(const T* x, const float* tab, int hs, int mode, int d, float (&v)[4]) {
    load_n<4, VEC>(x + d, v);
    if (!tab) return;
    if (mode == LQ_ROPE_PAIRS) {
        const float2 t0 = reinterpret_cast<const float2*>(tab)[d / 2], t1 = reinterpret_cast<const float2*>(tab)[d / 2 + 1];
        const float a0 = v[0], b0 = v[1], a1 = v[2], b1 = v[3];
        v[0] = a0 * t0.x - b0 * t0.y;
        v[1] = a0 * t0.y + b0 * t0.x;
        v[2] = a1 * t1.x - b1 * t1.y;
        v[3] = a1 * t1.y + b1 * t1.x;
    } else {
        const int half = hs / 2;  // a multiple of 8: the four dims lie in one half
        const bool up = d >= half;
        float o[4];
        load_n<4, VEC>(x + (up ? d - half : d + half), o);
        const float2* t = reinterpret_cast<const float2*>(tab) + (up ? d - half : d);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = up ? o[e] * t[e].y + v[e] * t[e].x : v[e] * t[e].x - o[e] * t[e].y;
    }
}

__device__ __forceinline__ float append_scale(uint32_t amax_bits, float old) {
    const float s = __uint_as_float(amax_bits) / 127.0f;
    float m = s > old ? s : old;
    if (m == 0.0f) m = 1e-8f;
    if (amax_bits >= kInfBits || !(old < __uint_as_float(kInfBits))) m = __uint_as_float(0x7FC00000u);
    return m;
}

// the last sequence whose key (by its index) is at most `at`, keys ascending; -1: none
template <typename F>
__device__ __forceinline__ int find_seq(int n, int at, int lane, F key) {
    int s = -1;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int c = __popc(__ballot_sync(0xffffffffu, i0 + lane < n && key(i0 + lane) <= at));
        s += c;
        if (c < 32) break;
    }
    return s;
}

// 8 dims by their four pairs' (cos, sin): u and v are the pairs' first and second
// dims (halves), or 4 dims each
__device__ __forceinline__ void turn8(bool halves, const float4& t0, const float4& t1, float (&u)[4], float (&v)[4]) {
    const float c[4] = {t0.x, t0.z, t1.x, t1.z}, n[4] = {t0.y, t0.w, t1.y, t1.w};
    if (halves) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float p = u[k], r = v[k];
            u[k] = p * c[k] - r * n[k];
            v[k] = p * n[k] + r * c[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float p = u[2 * k], r = u[2 * k + 1], p2 = v[2 * k], r2 = v[2 * k + 1];
            u[2 * k] = p * c[k] - r * n[k];
            u[2 * k + 1] = p * n[k] + r * c[k];
            v[2 * k] = p2 * c[k + 2] - r2 * n[k + 2];
            v[2 * k + 1] = p2 * n[k + 2] + r2 * c[k + 2];
        }
    }
}

constexpr int kNoRope = 2;  // MODE: LQ_ROPE_*, or this, or -1 for whichever at run time

// A warp's share of a row of queries: 8 dims a lane, 256 neighbouring ones at a
// time.  The four pairs of 8 dims at d are the table's d / 2 .. d / 2 + 3 for
// either mode: dims d .. d + 7, or d / 2 .. d / 2 + 3 of both halves.
template <typename T, bool VEC, int MODE>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, int unit, int lane) {
    const int hs = a.c.head_size, row = unit / a.q_parts, part = unit - row * a.q_parts;
    if (row >= a.b.n_rows) return;
    const int s = find_seq(a.b.n_seqs, row, lane, [&](int i) { return ld_after(a.b.row_start + i); });
    if (s < 0) return;
    const SeqRows q = seq_rows(a.b, s, lane == 0 ? a.err : nullptr);
    if (row < q.r0 || row >= q.r0 + q.n) return;
    const int pos = q.begin + (row - q.r0);
    if (a.r.rope && pos >= a.r.rope_rows) {
        if (lane == 0) set_err(a.err, DEV_BAD_POS);
        return;
    }
    const float4* tab = reinterpret_cast<const float4*>(a.r.rope + (int64_t)pos * hs);
    const T* x = static_cast<const T*>(a.r.q) + (int64_t)row * a.r.ld_q;
    T* y = static_cast<T*>(a.r.q_out) + (int64_t)row * a.r.ld_q_out;
    const int width = a.r.n_heads * hs, step = 256 * a.q_parts;
    const bool turn = MODE < 0 ? a.r.rope != nullptr : MODE != kNoRope;
    const bool halves = MODE < 0 ? turn && a.r.rope_mode == LQ_ROPE_HALVES : MODE == LQ_ROPE_HALVES;
    const bool fixed = step % hs == 0;  // a lane's dims are the same in every head: one look at the table
    float4 t0 = make_float4(1.0f, 0.0f, 1.0f, 0.0f), t1 = t0;
    int i = part * 256 + lane * 8, d = i % hs;
    if (turn && fixed && i < width) {
        t0 = tab[d / 4];
        t1 = tab[d / 4 + 1];
    }
    auto turned = [&](float (&u)[4], float (&v)[4]) {
        if (turn) turn8(halves, t0, t1, u, v);
    };
    if (fixed) {
        const int o0 = halves ? d / 2 - d : 0, o1 = halves ? o0 + hs / 2 : 4;
        for (; i + 3 * step < width; i += 4 * step) {  // four steps' loads together
            float u[4][4], v[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                load_n<4, VEC>(x + i + k * step + o0, u[k]);
                load_n<4, VEC>(x + i + k * step + o1, v[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                turned(u[k], v[k]);
                store_n<4, VEC>(y + i + k * step + o0, u[k]);
                store_n<4, VEC>(y + i + k * step + o1, v[k]);
            }
        }
    }
    for (; i < width; i += step) {
        if (!fixed) {
            d = i % hs;
            if (turn) {
                t0 = tab[d / 4];
                t1 = tab[d / 4 + 1];
            }
        }
        const int e0 = halves ? i - d + d / 2 : i, e1 = halves ? e0 + hs / 2 : i + 4;
        float u[4], v[4];
        load_n<4, VEC>(x + e0, u);
        load_n<4, VEC>(x + e1, v);
        turned(u, v);
        store_n<4, VEC>(y + e0, u);
        store_n<4, VEC>(y + e1, v);
    }
}

// codes of a word at a grown scale
__device__ __forceinline__ uint32_t again(uint32_t word, float ratio) {
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (uint32_t)__float2int_rn((float)code_of(word >> (8 * e)) * ratio);
    return pack8(o[0], o[1], o[2], o[3]);
}

// the first `keep` bytes of a word (4 and more: all) at a grown scale
__device__ __forceinline__ uint32_t again(uint32_t word, float ratio, int keep) {
    const uint32_t mask = keep >= 4 ? 0xFFFFFFFFu : (1u << (8 * keep)) - 1u;
    return (again(word, ratio) & mask) | (word & ~mask);
}

// One new token per sequence: a warp per (sequence, kv head), 4 dims a lane.
// Bound by the chain of dependent loads (lengths, page, scales).  Measured, fp32
// with 128 dims: one sequence of 32 heads 3.7 us, 64 of 40 heads 6.5 us (12.6 us
// by the kernel for any rows, with a block per sequence and head).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) append_one_kernel(const __grid_constant__ AppendArgs a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= a.kv_blocks) {
        rotate_queries<T, VEC, -1>(a, (blockIdx.x - a.kv_blocks) * kAppendWarps + warp, lane);
        return;
    }
    const int hs = a.c.head_size, P = a.c.page_size, H = a.c.n_kv_heads;
    const int per = (H + kAppendWarps - 1) / kAppendWarps;
    const int s = blockIdx.x / per, h = blockIdx.x % per * kAppendWarps + warp;
    if (h >= H) return;
    int* const err = lane == 0 ? a.err : nullptr;
    const SeqRows q = seq_rows(a.b, s, err);
    if (q.n != 1) return;
    const int pos = q.begin, lp = pos / P, off = pos - lp * P;
    if (a.r.rope && pos >= a.r.rope_rows) {
        set_err(err, DEV_BAD_POS);
        return;
    }
    const int64_t page = page_of(a.c, a.b, s, lp, err);
    const T* kr = static_cast<const T*>(a.r.k) + (int64_t)q.r0 * a.r.ld_k + (int64_t)h * hs;
    const T* vr = static_cast<const T*>(a.r.v) + (int64_t)q.r0 * a.r.ld_v + (int64_t)h * hs;
    const float* tab = a.r.rope ? a.r.rope + (int64_t)pos * hs : nullptr;
    float k[2][4] = {}, v[2][4] = {};
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = i * 128 + lane * 4;
        if (d < hs) {
            rotated4<T, VEC>(kr, tab, hs, a.r.rope_mode, d, k[i]);
            load_n<4, VEC>(vr + d, v[i]);
        }
    }
    if (page < 0) return;
    const int64_t cell = page * H + h;
    float2* const sc = reinterpret_cast<float2*>(a.c.scales) + cell;
    const float2 old = off > 0 ? *sc : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mk = max(mk, abs_bits(k[i][e]));
            mv = max(mv, abs_bits(v[i][e]));
        }
    const float sk = append_scale(__reduce_max_sync(0xffffffffu, mk), old.x);
    const float sv = append_scale(__reduce_max_sync(0xffffffffu, mv), old.y);
    const Quant8 qk(sk), qv(sv);
    __syncwarp();  // every lane has read the old scales
    if (lane == 0) *sc = make_float2(sk, sv);
    int8_t* kc = static_cast<int8_t*>(a.c.codes) + cell * 2 * hs * P;
    int8_t* vc = kc + (int64_t)hs * P;
    if (off > 0 && sk != old.x) {
        const float ratio = qk.bad ? 0.0f : old.x / sk;
        for (int i = lane; i < off * (hs / 4); i += 32) {
            const int t = i % off, w = i / off;
            uint32_t* p = reinterpret_cast<uint32_t*>(kc + ((int64_t)(w / 4) * P + t) * 16) + (w & 3);
            *p = again(*p, ratio);
        }
    }
    if (off > 0 && sv != old.y) {
        const float ratio = qv.bad ? 0.0f : old.y / sv;
        for (int i = lane; i < (off + 3) / 4 * hs; i += 32) {
            const int w = i / hs, d = i - w * hs;
            uint32_t* p = reinterpret_cast<uint32_t*>(vc + ((int64_t)(w / 4) * hs + d) * 16) + (w & 3);
            *p = again(*p, ratio, off - 4 * w);
        }
        __syncwarp();  // the new token's bytes may lie in these words
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = i * 128 + lane * 4;
        if (d >= hs) continue;
        const uint32_t ck = qk(k[i][0], k[i][1], k[i][2], k[i][3]), cv = qv(v[i][0], v[i][1], v[i][2], v[i][3]);
        *reinterpret_cast<uint32_t*>(kc + ((int64_t)(d / 16) * P + off) * 16 + d % 16) = ck;
        int8_t* vp = vc + ((int64_t)(off / 16) * hs + d) * 16 + off % 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) vp[16 * e] = (int8_t)(cv >> (8 * e));
        const int64_t at = (int64_t)q.r0 * a.r.ld_kv_out + (int64_t)h * hs + d;
        float o[4];
        if (a.r.k_out) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (float)code_of(ck >> (8 * e)) * sk;
            store_n<4, VEC>(static_cast<T*>(a.r.k_out) + at, o);
        }
        if (a.r.v_out) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (float)code_of(cv >> (8 * e)) * sv;
            store_n<4, VEC>(static_cast<T*>(a.r.v_out) + at, o);
        }
    }
}

// i = q * n + r, advanced by a fixed step without dividing again
struct Walk {
    int q, r, dq, dr, n;
    __device__ Walk(int i, int step, int n_) : q(i / n_), r(i - i / n_ * n_), dq(step / n_), dr(step - step / n_ * n_), n(n_) {}
    __device__ __forceinline__ void next() {
        q += dq;
        r += dr;
        if (r >= n) {
            r -= n;
            ++q;
        }
    }
};

// Any rows: a block per (page, kv head) that receives tokens.  Sequence s owns
// the jobs from row_start[s] / page + 2 s on, which are at least as many as the
// pages that its rows touch.  The rows are read twice, for the maxima and (from
// L1 or L2) for the codes, in short loops by many threads: keeping the values in
// registers between the two unrolled the code, whose instructions run once per
// block, and was slower (69 us against 45 for 2048 fp32 tokens of 32 heads,
// without queries).  Prompts of 64 + 2 x 8 heads, 220 MB of bf16 rows and codes in
// pages of 16, take 47 us (4.7 TB/s): neither DRAM (46%) nor the issue slots (54%)
// are full, a block's chain of loads from its page's look-up to its codes is what a
// small page costs.

template <typename T, bool VEC, int MODE>
__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const __grid_constant__ AppendArgs a) {
    pdl_trigger();
    pdl_wait();
    const int threads = blockDim.x;
    const int tid = threadIdx.x, lane = tid & 31;
    if (blockIdx.x >= a.kv_blocks) {
        rotate_queries<T, VEC, MODE>(a, (blockIdx.x - a.kv_blocks) * (threads / 32) + (tid >> 5), lane);
        return;
    }
    const int hs = a.c.head_size, P = a.c.page_size, H = a.c.n_kv_heads;
    const int job = blockIdx.x / H, h = blockIdx.x % H;
    const int s = find_seq(a.b.n_seqs, job, lane, [&](int i) { return ld_after(a.b.row_start + i) / P + 2 * i; });
    if (s < 0) return;
    const SeqRows q = seq_rows(a.b, s, tid == 0 ? a.err : nullptr);
    if (q.n <= 0) return;
    const int lp = q.begin / P + (job - (ld_after(a.b.row_start + s) / P + 2 * s));
    const int t0 = max(q.begin, lp * P), t1 = min(q.ctx, lp * P + P);  // the page's new tokens
    if (t0 >= t1) return;
    if (a.r.rope && t1 > a.r.rope_rows) {
        if (tid == 0) set_err(a.err, DEV_BAD_POS);
        return;
    }
    const int64_t page = page_of(a.c, a.b, s, lp, tid == 0 ? a.err : nullptr);
    if (page < 0) return;
    const int64_t cell = page * H + h;
    int8_t* kc = static_cast<int8_t*>(a.c.codes) + cell * 2 * hs * P;
    int8_t* vc = kc + (int64_t)hs * P;
    const int row0 = q.r0 + (t0 - q.begin), nt = t1 - t0, off = t0 - lp * P;
    const T* kr = static_cast<const T*>(a.r.k) + (int64_t)row0 * a.r.ld_k + (int64_t)h * hs;
    const T* vr = static_cast<const T*>(a.r.v) + (int64_t)row0 * a.r.ld_v + (int64_t)h * hs;
    const float* tab0 = a.r.rope ? a.r.rope + (int64_t)t0 * hs : nullptr;

    // K: 8 dims of a token at a time, as in rotate_queries.  V: 4 tokens of 4 dims,
    // a word of codes for each dim; words wf .. w1 - 1 hold new tokens, and four
    // neighbouring threads take the words of 16 tokens.
    const int hw = hs / 8, nk = nt * hw, wf = off / 4, w1 = (off + nt + 3) / 4, g0 = wf / 4, nv = ((w1 + 3) / 4 - g0) * hs;
    const Walk k0(tid, threads, hw), v0(tid / 4, threads / 4, hs / 4);
    const bool turn = MODE < 0 ? tab0 != nullptr : MODE != kNoRope;
    const bool halves = MODE < 0 ? turn && a.r.rope_mode == LQ_ROPE_HALVES : MODE == LQ_ROPE_HALVES;
    auto dims = [&](const Walk& i, int& e0, int& e1) {
        e0 = halves ? 4 * i.r : 8 * i.r;
        e1 = halves ? e0 + hs / 2 : e0 + 4;
    };
    auto load_k = [&](const Walk& i, float (&u)[4], float (&v)[4]) {
        int e0, e1;
        dims(i, e0, e1);
        const T* row = kr + i.q * a.r.ld_k;
        load_n<4, VEC>(row + e0, u);
        load_n<4, VEC>(row + e1, v);
        if (turn) {
            const float4* t = reinterpret_cast<const float4*>(tab0 + i.q * hs) + 2 * i.r;
            turn8(halves, t[0], t[1], u, v);
        }
    };
    uint32_t mk = 0, mv = 0;
    Walk ki = k0, vi = v0;
#pragma unroll 2
    for (int i = tid; i < nk; i += threads, ki.next()) {
        float u[4], v[4], x[4], y[4];
        load_k(ki, u, v);
        const T* row = vr + ki.q * a.r.ld_v + 8 * ki.r;
        load_n<4, VEC>(row, x);
        load_n<4, VEC>(row + 4, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mk = max(mk, max(abs_bits(u[e]), abs_bits(v[e])));
            mv = max(mv, max(abs_bits(x[e]), abs_bits(y[e])));
        }
    }
    float old_k = 0.0f, old_v = 0.0f;  // a page whose first token arrives now starts afresh
    if (off > 0) {
        old_k = a.c.scales[cell * 2];
        old_v = a.c.scales[cell * 2 + 1];
    }
    __shared__ uint32_t wk[kAppendWarps], wv[kAppendWarps];
    mk = __reduce_max_sync(0xffffffffu, mk);
    mv = __reduce_max_sync(0xffffffffu, mv);
    if (lane == 0) {
        wk[tid >> 5] = mk;
        wv[tid >> 5] = mv;
    }
    __syncthreads();
    for (int w = 0; w < threads / 32; ++w) {
        mk = max(mk, wk[w]);
        mv = max(mv, wv[w]);
    }
    const float sk = append_scale(mk, old_k), sv = append_scale(mv, old_v);
    const Quant8 qk(sk), qv(sv);
    if (tid == 0) {
        a.c.scales[cell * 2] = sk;
        a.c.scales[cell * 2 + 1] = sv;
    }
    // earlier tokens at the grown scale (a NaN scale leaves nothing to keep)
    const bool grow_k = off > 0 && sk != old_k, grow_v = off > 0 && sv != old_v;
    if (grow_k) {
        const float ratio = qk.bad ? 0.0f : old_k / sk;
        for (int i = tid; i < off * (hs / 4); i += threads) {
            const int t = i % off, w = i / off;  // word w (4 dims) of token t
            uint32_t* p = reinterpret_cast<uint32_t*>(kc + ((int64_t)(w / 4) * P + t) * 16) + (w & 3);
            *p = again(*p, ratio);
        }
    }
    const float ratio_v = qv.bad ? 0.0f : old_v / sv;
    if (grow_v) {  // whole words of earlier tokens
        for (int i = tid; i < wf * hs; i += threads) {
            const int w = i / hs, d = i - w * hs;
            uint32_t* p = reinterpret_cast<uint32_t*>(vc + ((int64_t)(w / 4) * hs + d) * 16) + (w & 3);
            *p = again(*p, ratio_v);
        }
    }
    auto store_k = [&](int t, int d, float (&k)[4]) {
        const uint32_t c = qk(k[0], k[1], k[2], k[3]);
        *reinterpret_cast<uint32_t*>(kc + ((d >> 4) * P + off + t) * 16 + (d & 15)) = c;
        if (a.r.k_out) {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = (float)code_of(c >> (8 * e)) * sk;
            store_n<4, VEC>(static_cast<T*>(a.r.k_out) + (int64_t)(row0 + t) * a.r.ld_kv_out + (int64_t)h * hs + d, k);
        }
    };
    ki = k0;
#pragma unroll 2
    for (int i = tid; i < nk; i += threads, ki.next()) {
        float u[4], v[4];
        load_k(ki, u, v);
        int e0, e1;
        dims(ki, e0, e1);
        store_k(ki.q, e0, u);
        store_k(ki.q, e1, v);
    }
#pragma unroll 1
    for (int i = tid; i < nv; i += threads, vi.next()) {
        const int w = 4 * (g0 + vi.q) + (tid & 3), d = 4 * vi.r, t = 4 * w - off;
        if (w < wf || w >= w1) continue;
        const T* x = vr + t * a.r.ld_v + d;
        float v[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[e][k] = 0.0f;
            if (t + e >= 0 && t + e < nt) load_n<4, VEC>(x + e * a.r.ld_v, v[e]);
        }
        uint32_t c[4];  // by token
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = qv(v[e][0], v[e][1], v[e][2], v[e][3]);
        const uint32_t a0 = __byte_perm(c[0], c[1], 0x5140), a1 = __byte_perm(c[2], c[3], 0x5140);
        const uint32_t b0 = __byte_perm(c[0], c[1], 0x7362), b1 = __byte_perm(c[2], c[3], 0x7362);
        uint32_t word[4] = {__byte_perm(a0, a1, 0x5410), __byte_perm(a0, a1, 0x7632), __byte_perm(b0, b1, 0x5410),
                            __byte_perm(b0, b1, 0x7632)};  // by dim
        // a word at either end: earlier tokens kept or rescaled, later bytes kept
        const int lo = max(-t, 0), hi = min(nt - t, 4);  // its new bytes
        uint32_t* p = reinterpret_cast<uint32_t*>(vc + ((w >> 2) * hs + d) * 16) + (w & 3);
        if (lo > 0 || hi < 4) {
            const uint32_t mask = (hi >= 4 ? 0xFFFFFFFFu : (1u << (8 * hi)) - 1u) & ~((1u << (8 * lo)) - 1u);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t was = p[4 * k];
                if (grow_v && lo > 0) was = again(was, ratio_v, lo);
                word[k] = (word[k] & mask) | (was & ~mask);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) p[4 * k] = word[k];
        if (a.r.v_out) {
            T* out = static_cast<T*>(a.r.v_out) + (row0 + t) * a.r.ld_kv_out + (int64_t)h * hs + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (e < lo || e >= hi) continue;
                float o[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) o[k] = (float)code_of(c[e] >> (8 * k)) * sv;
                store_n<4, VEC>(out + e * a.r.ld_kv_out, o);
            }
        }
    }
}

template <typename T>
cudaError_t append_t(AppendArgs& a, int sms, cudaStream_t st) {
    const KVRows& r = a.r;
    const uintptr_t bytes = 4 * sizeof(T);
    auto fits = [&](const void* p, int64_t ld) { return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld % 4 == 0); };
    const bool vec = fits(r.q, r.ld_q) && fits(r.k, r.ld_k) && fits(r.v, r.ld_v) && fits(r.q_out, r.ld_q_out) &&
                     fits(r.k_out, r.ld_kv_out) && fits(r.v_out, r.ld_kv_out);
    const bool one = a.b.max_rows <= 1;
    int64_t kv = one ? (int64_t)a.b.n_seqs * ((a.c.n_kv_heads + kAppendWarps - 1) / kAppendWarps)
                     : ((int64_t)a.b.n_rows / a.c.page_size + 2 * a.b.n_seqs) * a.c.n_kv_heads;
    // Threads for a page: no more than fill the GPU (768 an SM, of the 1024 that
    // registers allow), since a block's start costs every warp as much as some
    // hundred elements.  2424 pages of 16 tokens: 64 threads 47 us, 256 58 us;
    // 576 pages of 32 tokens: 25 us and 17 us.
    int threads = kAppendThreads;
    while (!one && threads > 32 && kv * (threads / 2) >= (int64_t)sms * 768) threads /= 2;
    // a row of queries is cut into 256-dim parts until there are 8 warps per SM
    int64_t q_blocks = 0;
    a.q_parts = 1;
    if (r.q) {
        const int most = (r.n_heads * a.c.head_size + 255) / 256, want = 8 * sms / a.b.n_rows;
        a.q_parts = want < 1 ? 1 : want < most ? want : most;
        q_blocks = ((int64_t)a.b.n_rows * a.q_parts + threads / 32 - 1) / (threads / 32);
    }
    if (kv + q_blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    a.kv_blocks = (int)kv;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(kv + q_blocks));
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto kern = one ? (vec ? append_one_kernel<T, true> : append_one_kernel<T, false>)
                : !vec    ? append_kernel<T, false, -1>
                : !r.rope ? append_kernel<T, true, kNoRope>
                : r.rope_mode == LQ_ROPE_HALVES ? append_kernel<T, true, LQ_ROPE_HALVES>
                                                : append_kernel<T, true, LQ_ROPE_PAIRS>;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace

int check_paged(const PagedKV* c, const KVBatch* b, int n_heads, int type, const char* fn) {
    if (!c || !b) return lq_fail(LQ_EINVAL, "%s: null argument", fn);
    if (type != LQ_F32 && type != LQ_F16 && type != LQ_BF16) return lq_fail(LQ_EINVAL, "%s: type %d", fn, type);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return lq_fail(LQ_EINVAL, "%s: page size %d (16, 32, 64 or 128)", fn, c->page_size);
    if (c->head_size < 16 || c->head_size > 256 || c->head_size % 16)
        return lq_fail(LQ_EINVAL, "%s: head size %d (a multiple of 16, 16 to 256)", fn, c->head_size);
    if (c->n_kv_heads <= 0 || c->n_kv_heads > 65535 || n_heads < 0 || n_heads % c->n_kv_heads)
        return lq_fail(LQ_EINVAL, "%s: %d query heads over %d kv heads", fn, n_heads, c->n_kv_heads);
    if (c->n_pages < 0 || c->n_pages > INT32_MAX || b->n_seqs < 0 || b->n_rows < 0 || b->max_pages < 0 ||
        b->max_rows < 0 || b->max_context < 0)
        return lq_fail(LQ_EINVAL, "%s: a count is negative or too large", fn);
    if (b->n_seqs > 65535 || b->n_rows > (1 << 24) || b->max_context > (1 << 28))
        return lq_fail(LQ_EUNSUPPORTED, "%s: at most 65535 sequences, 2^24 rows and contexts of 2^28", fn);
    if (b->n_seqs == 0 || b->n_rows == 0) return LQ_OK;
    if (!c->codes || !c->scales || !b->row_start || !b->context || (b->max_pages > 0 && !b->pages))
        return lq_fail(LQ_EINVAL, "%s: the cache's or the batch's memory is not set", fn);
    if ((reinterpret_cast<uintptr_t>(c->codes) & 15u) || (reinterpret_cast<uintptr_t>(c->scales) & 7u) ||
        ((reinterpret_cast<uintptr_t>(b->row_start) | reinterpret_cast<uintptr_t>(b->context) |
          reinterpret_cast<uintptr_t>(b->pages)) & 3u))
        return lq_fail(LQ_EINVAL, "%s: codes must be 16-byte, scales 8-byte and the batch's arrays 4-byte aligned", fn);
    return LQ_OK;
}

}  // namespace lq

using namespace lq;

extern "C" {

int lq_rope_table(float* table, int positions, int head_size, float base) {
    if (!table || positions < 0 || head_size <= 0 || head_size % 2 || !(base > 0.0f))
        return lq_fail(LQ_EINVAL, "lq_rope_table: null table, odd head size or base <= 0");
    for (int pos = 0; pos < positions; ++pos)
        for (int i = 0; i < head_size / 2; ++i) {
            const float freq = 1.0f / powf(base, (2 * i) / (float)head_size);
            const float val = pos * freq;
            float* t = table + ((size_t)pos * (head_size / 2) + i) * 2;
            t[0] = cosf(val);
            t[1] = sinf(val);
        }
    return LQ_OK;
}

int kv_append(const PagedKV* cache, const KVBatch* batch, const KVRows* rows) {
    if (!rows) return lq_fail(LQ_EINVAL, "kv_append: null argument");
    int rc = check_paged(cache, batch, rows->q ? rows->n_heads : 0, rows->type, "kv_append");
    if (rc) return rc;
    if (rows->rope && (rows->rope_rows < 0 || (rows->rope_mode != LQ_ROPE_PAIRS && rows->rope_mode != LQ_ROPE_HALVES) ||
                       (reinterpret_cast<uintptr_t>(rows->rope) & 15u)))
        return lq_fail(LQ_EINVAL, "kv_append: rope mode %d, or a table that is not 16-byte aligned", rows->rope_mode);
    if (batch->n_seqs == 0 || batch->n_rows == 0) return LQ_OK;
    const int64_t kv = (int64_t)cache->n_kv_heads * cache->head_size;
    if (!rows->k || !rows->v || rows->ld_k < kv || rows->ld_v < kv)
        return lq_fail(LQ_EINVAL, "kv_append: k or v not set, or rows closer than %lld elements", (long long)kv);
    if ((rows->k_out || rows->v_out) && rows->ld_kv_out < kv)
        return lq_fail(LQ_EINVAL, "kv_append: ld_kv_out=%lld is less than %lld", (long long)rows->ld_kv_out, (long long)kv);
    const int64_t qd = (int64_t)rows->n_heads * cache->head_size;
    if (rows->q && (!rows->q_out || rows->ld_q < qd || rows->ld_q_out < qd))
        return lq_fail(LQ_EINVAL, "kv_append: q_out not set, or rows closer than %lld elements", (long long)qd);
    const uintptr_t size = rows->type == LQ_F32 ? 4 : 2;
    const void* all[] = {rows->q, rows->k, rows->v, rows->q ? rows->q_out : nullptr, rows->k_out, rows->v_out};
    for (const void* p : all)
        if (reinterpret_cast<uintptr_t>(p) % size)
            return lq_fail(LQ_EINVAL, "kv_append: a tensor is not aligned to its elements");
    DevCtx* c = ctx();
    if (!c) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
    AppendArgs a;
    a.c = *cache;
    a.b = *batch;
    if (a.b.max_rows > a.b.n_rows) a.b.max_rows = a.b.n_rows;
    a.r = *rows;
    a.err = c->err;
    if (rows->q && rows->n_heads == 0) a.r.q = nullptr;
    cudaError_t e = rows->type == LQ_F32   ? append_t<float>(a, c->num_sms, stream())
                    : rows->type == LQ_F16 ? append_t<__half>(a, c->num_sms, stream())
                                           : append_t<__nv_bfloat16>(a, c->num_sms, stream());
    return e == cudaSuccess ? LQ_OK : cuda_fail(e, "kv_append launch");
}

}  // extern "C"
