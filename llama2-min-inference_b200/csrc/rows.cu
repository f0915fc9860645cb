// Token-scaled int8 products: quantize_rows (one scale per row) and
// matmul_rows (int8 x int8 with a scale per token and per output channel).
#include "lq_ctx.h"
#include "lq_device.cuh"
#include "lq_ops.h"
#include "lq_tc.cuh"
#include "lq_types.cuh"

namespace lq {
namespace {

// ---------------------------------------------------------------------------
// quantize_rows: s = max|x| / 127 (0 -> 1e-8), q = rint(x / s), one CTA per row.
// The row is read once: each thread keeps up to kKeep quads of it between the
// maximum and the rounding; longer rows are read again (from L2).

constexpr int kQuantThreads = 256;
constexpr int kKeep = 16;  // quads per thread: rows of up to 16384 stay in registers

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const T* __restrict__ x, int64_t ld, int n,
                                                                      int8_t* __restrict__ q, int pitch,
                                                                      float* __restrict__ s) {
    pdl_trigger();
    pdl_wait();
    const T* xr = x + (int64_t)blockIdx.x * ld;
    const int quads = pitch / 4;
    float keep[kKeep][4];
    uint32_t m = 0;
    auto load = [&](int i, float (&v)[4]) {
        if (4 * i + 4 <= n) {
            load_n<4, VEC>(xr + 4 * i, v);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = 4 * i + e < n ? to_f32(xr[4 * i + e]) : 0.0f;
        }
    };
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
        const int i = threadIdx.x + j * kQuantThreads;
        if (i < quads) load(i, keep[j]);
    }
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
        if (threadIdx.x + j * kQuantThreads < quads) {
#pragma unroll
            for (int e = 0; e < 4; ++e) m = max(m, abs_bits(keep[j][e]));
        }
    }
    for (int i = threadIdx.x + kKeep * kQuantThreads; i < quads; i += kQuantThreads) {
        float v[4];
        load(i, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, abs_bits(v[e]));
    }
    __shared__ uint32_t wm[kQuantThreads / 32];
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) wm[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantThreads / 32; ++w) m = max(m, wm[w]);
    const bool bad = m >= kInfBits;  // a NaN or an infinity: scale NaN, codes 0
    float sc = __uint_as_float(m) / 127.0f;
    if (sc == 0.0f) sc = 1e-8f;
    uint32_t* qr = reinterpret_cast<uint32_t*>(q + (int64_t)blockIdx.x * pitch);
    auto store = [&](int i, const float (&v)[4]) {
        qr[i] = bad ? 0u : pack8(quant8(v[0], sc), quant8(v[1], sc), quant8(v[2], sc), quant8(v[3], sc));
    };
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
        const int i = threadIdx.x + j * kQuantThreads;
        if (i < quads) store(i, keep[j]);
    }
    for (int i = threadIdx.x + kKeep * kQuantThreads; i < quads; i += kQuantThreads) {
        float v[4];
        load(i, v);
        store(i, v);
    }
    if (threadIdx.x == 0) s[blockIdx.x] = bad ? __uint_as_float(0x7FC00000u) : sc;
}

template <typename T>
cudaError_t quantize_rows_t(const void* x, int64_t ld, int64_t rows, int n, int8_t* q, float* s, cudaStream_t st) {
    const T* xt = static_cast<const T*>(x);
    const int pitch = LQ_ROW8_PITCH(n);
    const bool vec = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 && ld % 4 == 0;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows);
    cfg.blockDim = dim3(kQuantThreads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return vec ? cudaLaunchKernelEx(&cfg, quantize_rows_kernel<T, true>, xt, ld, n, q, pitch, s)
               : cudaLaunchKernelEx(&cfg, quantize_rows_kernel<T, false>, xt, ld, n, q, pitch, s);
}

// ---------------------------------------------------------------------------
// matmul_rows on the tensor cores: tcgen05.mma kind::i8, int32 accumulators in
// tensor memory.  The channels are the MMA's M (128, or 256 by a pair of CTAs)
// and the tokens its N, for every token count: one token is N = 16 with zeros,
// the weights then stream at memory speed, and a thread of the epilogue holds
// one channel of all tokens, so that a warp's store is 32 neighbouring channels.
//
// One CTA per SM: warp 0 issues the TMA copies (128-byte K stages, 128-byte
// swizzle; bytes past the row or the tensor read as zeros), warp 1 the MMAs,
// warps 2-5 turn a finished accumulator into outputs while the MMAs fill the
// other.  Tiles that fill whole rounds of the grid are done by one CTA each;
// the stages of the remaining ones are cut into equal runs over all CTAs
// (stream-K).  A tile cut so leaves int32 partials, which the last of its CTAs
// to arrive adds: integer sums, the same whatever the order.

constexpr int kRowsThreads = 192;
constexpr int kStageBytes = 128;  // K bytes per stage
constexpr int kMaxStages = 12;

struct RowsArgs {
    CUtensorMap wmap, xmap;
    const float *xs, *ws;
    void* y;
    int64_t ld;
    int rows, d, type;
    int kst;                // K stages
    int ttiles;             // tiles along the tokens
    int whole, shared;      // tiles done by one CTA group each; tiles cut by stages
    int sk_grid;            // CTA groups that share them
    int stages;
    int early;              // the weights may be read before the previous kernel ends
    int *part, *cnt, *err;
};

struct RowsBars {
    uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2], done;
    uint32_t tmem_base;
    int abort_flag, last_flag;
};

// the (tile, K range) pieces of one CTA group: first its run of shared stages, then whole tiles
struct Pieces {
    int64_t s, s1;
    int t, whole, groups, kst;
    __device__ Pieces(const RowsArgs& a, int group, int groups_) {
        const int64_t w = (int64_t)a.shared * a.kst;
        s = group < a.sk_grid ? sk_start(group, w, a.sk_grid) : 0;
        s1 = group < a.sk_grid ? sk_start(group + 1, w, a.sk_grid) : 0;
        t = group;
        whole = a.whole;
        groups = groups_;
        kst = a.kst;
    }
    __device__ bool next(int& tile, int& k0, int& k1) {
        if (s < s1) {
            const int q = (int)(s / kst);
            tile = whole + q;
            k0 = (int)(s - (int64_t)q * kst);
            k1 = (int)min((int64_t)kst, k0 + (s1 - s));
            s += k1 - k0;
            return true;
        }
        if (t < whole) {
            tile = t;
            k0 = 0;
            k1 = kst;
            t += groups;
            return true;
        }
        return false;
    }
};

template <int N, int CTAS>
constexpr int rows_stage_bytes() {
    return 128 * kStageBytes + N / CTAS * kStageBytes;
}

template <int CH, typename T>
__device__ __forceinline__ void store_columns(T* y, int64_t ld, const int (&acc)[CH], float xsv, float wsv, int n,
                                              bool ok) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const float f = (float)acc[j] * (__shfl_sync(0xffffffffu, xsv, j) * wsv);
        if (j < n && ok) y[j * ld] = from_f32<T>(f);
    }
}

template <int N, int CTAS>
__global__ void __launch_bounds__(kRowsThreads, 1) matmul_rows_kernel(const __grid_constant__ RowsArgs a) {
    constexpr int kA = 128 * kStageBytes, kB = N / CTAS * kStageBytes, kStage = kA + kB;
    constexpr int kCols = 2 * N < 32 ? 32 : 2 * N;
    constexpr int CH = N < 32 ? N : 32;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    RowsBars* bars = reinterpret_cast<RowsBars*>(sm + (size_t)a.stages * kStage);
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = blockIdx.x / CTAS, groups = gridDim.x / CTAS, rank = CTAS == 2 ? blockIdx.x & 1 : 0;
    const int S = a.stages;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&bars->full[i], 1);
            mbar_init(&bars->empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bars->tfull[i], 1);
            mbar_init(&bars->tempty[i], 4 * CTAS);
        }
        mbar_init(&bars->done, 1);
        bars->abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc<CTAS>(&bars->tmem_base, kCols);
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    pdl_trigger();
    if (!(warp == 0 && a.early)) pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pw = l2_evict_first_policy(), px = l2_evict_last_policy();
            const uint64_t pol_w = a.ttiles > 1 ? px : pw;  // weights that several token tiles read stay in L2
            Pieces p(a, group, groups);
            int tile, k0, k1, slot = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            uint64_t* full0 = bars->full;
            const uint32_t lead = CTAS == 2 ? cluster_addr(full0, 0) : smem_addr(full0);
            if (CTAS == 1 && a.early) {
                // the ring's first weight tiles, then the previous kernel's end, then the activations
                Pieces e(a, group, groups);
                int n = 0;
                while (n < S && e.next(tile, k0, k1))
                    for (int k = k0; k < k1 && n < S; ++k, ++n) {
                        mbar_arrive_expect_tx(&bars->full[n], kStage);
                        tma_load_2d(sm + n * kStage, &a.wmap, k * kStageBytes, tile / a.ttiles * 128, &bars->full[n], pol_w);
                    }
                pdl_wait();
            }
            while (ok && p.next(tile, k0, k1)) {
                const int ch = tile / a.ttiles * (128 * CTAS) + rank * 128, tok = tile % a.ttiles * N + rank * (N / CTAS);
                for (int k = k0; k < k1; ++k) {
                    if (!qwait(&bars->empty[slot], ph ^ 1u, a.err, DEV_TIMEOUT_EMPTY, abort_flag)) {
                        ok = false;
                        break;
                    }
                    unsigned char* at = sm + slot * kStage;
                    if (CTAS == 1) {
                        if (!(a.early && issued < S)) {
                            mbar_arrive_expect_tx(&bars->full[slot], kStage);
                            tma_load_2d(at, &a.wmap, k * kStageBytes, ch, &bars->full[slot], pol_w);
                        }
                        tma_load_2d(at + kA, &a.xmap, k * kStageBytes, tok, &bars->full[slot], px);
                    } else {
                        if (rank == 0) mbar_arrive_expect_tx(&bars->full[slot], 2 * kStage);
                        tma_load_2d_pair(at, &a.wmap, k * kStageBytes, ch, lead + slot * 8, pol_w);
                        tma_load_2d_pair(at + kA, &a.xmap, k * kStageBytes, tok, lead + slot * 8, px);
                    }
                    ++issued;
                    if (++slot == S) {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (*abort_flag && rank == 0) {  // confirm the copies still in flight
                for (int j = max(0, issued - S); j < issued; ++j)
                    if (!mbar_wait(&bars->full[j % S], (uint32_t)((j / S) & 1), a.err, DEV_TIMEOUT_DRAIN)) break;
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // s32 += s8 x s8, both K-major
            const uint32_t idesc =
                (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(8 * CTAS) << 24);
            Pieces p(a, group, groups);
            int tile, k0, k1, slot = 0, buf = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true, issued = false;
            while (ok && p.next(tile, k0, k1)) {
                if (!qwait(&bars->tempty[buf], bph ^ 1u, a.err, DEV_TIMEOUT_TEMPTY, abort_flag)) break;
                tc_fence_after();
                const uint32_t dst = tmem + (uint32_t)(buf * N);
                for (int k = k0; k < k1; ++k) {
                    if (!qwait(&bars->full[slot], ph, a.err, DEV_TIMEOUT_FULL, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t ad = smem_desc_sw128(smem_addr(sm + slot * kStage));
                    const uint64_t bd = smem_desc_sw128(smem_addr(sm + slot * kStage + kA));
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // 32 bytes of K each: 2 descriptor units
                        mma_i8_n<CTAS>(dst, ad + 2 * j, bd + 2 * j, idesc, k > k0 || j > 0);
                    issued = true;
                    mma_commit_n<CTAS>(&bars->empty[slot]);
                    if (++slot == S) {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
                if (ok) mma_commit_n<CTAS>(&bars->tfull[buf]);
                buf ^= 1;
                if (buf == 0) bph ^= 1u;
            }
            if (issued) {  // every MMA has completed before the tensor memory is freed
                mma_commit_n<CTAS>(&bars->done);
                mbar_wait(&bars->done, 0, a.err, DEV_TIMEOUT_MMA);
            }
        }
    } else {
        const int q = warp & 3, rr = 32 * q + lane;  // channel within the CTA's 128 = TMEM lane
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const int64_t w = (int64_t)a.shared * a.kst;
        const int64_t my0 = group < a.sk_grid ? sk_start(group, w, a.sk_grid) : 0;
        Pieces p(a, group, groups);
        int tile, k0, k1, buf = 0;
        uint32_t bph = 0;
        while (p.next(tile, k0, k1)) {
            if (!__all_sync(0xffffffffu, qwait(&bars->tfull[buf], bph, a.err, DEV_TIMEOUT_TFULL, abort_flag))) break;
            tc_fence_after();
            const uint32_t src = tl + (uint32_t)(buf * N);
            const int ch = tile / a.ttiles * (128 * CTAS) + rank * 128 + rr, tok0 = tile % a.ttiles * N;
            int first = 0, pieces = 1;
            const int64_t tk0 = (int64_t)(tile - a.whole) * a.kst;
            if (k1 - k0 < a.kst) {
                first = sk_owner(tk0, w, a.sk_grid);
                pieces = sk_owner(tk0 + a.kst - 1, w, a.sk_grid) - first + 1;
            }
            bool finish = true;
            if (pieces > 1) {
                int* pb = a.part + ((size_t)blockIdx.x * 2 + (my0 >= tk0 ? 0 : 1)) * (N * 128) + rr;
                for (int c = 0; c < N && tok0 + c < a.rows; c += CH) {
                    int v[CH];
                    tmem_ld<CH>(src + c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < CH; ++j) __stcg(pb + (c + j) * 128, v[j]);
                }
                __threadfence();
                named_bar_sync(1, 128);
                if (threadIdx.x == 64) {
                    int* cnt = a.cnt + (tile - a.whole) * CTAS + rank;
                    const int last = atomicAdd(cnt, 1) == pieces - 1;
                    if (last) *cnt = 0;  // as the next launch expects it
                    bars->last_flag = last;
                }
                named_bar_sync(1, 128);
                finish = bars->last_flag != 0;
                named_bar_sync(1, 128);  // the next piece writes last_flag again
                if (finish) __threadfence();
            }
            if (finish) {
                const float wsv = ch < a.d ? __ldg(a.ws + ch) : 0.0f;
                for (int c = 0; c < N && tok0 + c < a.rows; c += CH) {
                    int v[CH];
                    tmem_ld<CH>(src + c, v);
                    tmem_ld_wait();
                    for (int o = 0; o < pieces; ++o) {
                        if (first + o == group || pieces == 1) continue;
                        const int64_t o0 = sk_start(first + o, w, a.sk_grid);
                        const int* pb = a.part + ((size_t)((first + o) * CTAS + rank) * 2 + (o0 >= tk0 ? 0 : 1)) * (N * 128) + rr;
#pragma unroll
                        for (int j = 0; j < CH; ++j) v[j] += __ldcg(pb + (c + j) * 128);
                    }
                    const int n = min(CH, a.rows - tok0 - c);
                    const float xsv = lane < n ? __ldg(a.xs + tok0 + c + lane) : 0.0f;
                    const int64_t at = (int64_t)(tok0 + c) * a.ld + ch;
                    if (a.type == LQ_F32)
                        store_columns<CH>(static_cast<float*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
                    else if (a.type == LQ_F16)
                        store_columns<CH>(static_cast<__half*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
                    else
                        store_columns<CH>(static_cast<__nv_bfloat16*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CTAS == 2)
                    mbar_arrive_cluster(cluster_addr(&bars->tempty[buf], 0));
                else
                    mbar_arrive(&bars->tempty[buf]);
            }
            buf ^= 1;
            if (buf == 0) bph ^= 1u;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<CTAS>(tmem, kCols);
    }
}

template <int N, int CTAS>
cudaError_t rows_launch(RowsArgs a, int grid, cudaStream_t st) {
    constexpr int kStage = rows_stage_bytes<N, CTAS>();
    const int most = (227 * 1024 - 1024 - (int)sizeof(RowsBars)) / kStage;
    a.stages = most < kMaxStages ? most : kMaxStages;
    const int smem = a.stages * kStage + 1024 + (int)sizeof(RowsBars);
    auto kern = matmul_rows_kernel<N, CTAS>;
    static bool set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) set[dev] = true;
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CTAS;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = CTAS == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" {

int quantize_rows(QuantizedTensor* out, const void* x, int type, int64_t ld, int n) {
    if (!out || n <= 0 || n > 131072 || out->rows < 0 || out->rows > INT32_MAX)
        return lq_fail(LQ_EINVAL, "quantize_rows: null argument, n outside 1..131072 or bad row count");
    if (type != LQ_F32 && type != LQ_F16 && type != LQ_BF16) return lq_fail(LQ_EINVAL, "quantize_rows: type %d", type);
    if (ld < n) return lq_fail(LQ_EINVAL, "quantize_rows: ld=%lld is less than n=%d", (long long)ld, n);
    if (out->rows > 0) {
        if (!x || !out->q || !out->s) return lq_fail(LQ_EINVAL, "quantize_rows: x, out->q or out->s not set");
        const int size = type == LQ_F32 ? 4 : 2;
        if ((reinterpret_cast<uintptr_t>(out->q) & 15u) || (reinterpret_cast<uintptr_t>(out->s) & 3u) ||
            reinterpret_cast<uintptr_t>(x) % size)
            return lq_fail(LQ_EINVAL, "quantize_rows: out->q must be 16-byte aligned, x and out->s to their elements");
        if (!ctx()) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
        int8_t* q = static_cast<int8_t*>(out->q);
        cudaError_t e = type == LQ_F32   ? quantize_rows_t<float>(x, ld, out->rows, n, q, out->s, stream())
                        : type == LQ_F16 ? quantize_rows_t<__half>(x, ld, out->rows, n, q, out->s, stream())
                                         : quantize_rows_t<__nv_bfloat16>(x, ld, out->rows, n, q, out->s, stream());
        if (e != cudaSuccess) return cuda_fail(e, "quantize_rows launch");
    }
    out->cols = out->group_size = n;
    out->kind = LQ_KIND_ROW8;
    return LQ_OK;
}

int matmul_rows(void* xout, int type, int64_t ld, const QuantizedTensor* x, const QuantizedTensor* w, int n, int d) {
    if (!x || !w) return lq_fail(LQ_EINVAL, "matmul_rows: null argument");
    if (type != LQ_F32 && type != LQ_F16 && type != LQ_BF16) return lq_fail(LQ_EINVAL, "matmul_rows: type %d", type);
    if (n <= 0 || n > 131072 || d <= 0) return lq_fail(LQ_EINVAL, "matmul_rows: n=%d (1..131072), d=%d", n, d);
    if (x->kind != LQ_KIND_ROW8 || w->kind != LQ_KIND_ROW8)
        return lq_fail(LQ_EINVAL, "matmul_rows: x and w must be LQ_KIND_ROW8");
    if (x->cols != n || w->cols != n || x->group_size != n || w->group_size != n || w->rows != d || x->rows < 0 ||
        x->rows > INT32_MAX - 256)
        return lq_fail(LQ_EINVAL, "matmul_rows: shape mismatch (x is %lld x %lld, w is %lld x %lld, n=%d d=%d)",
                       (long long)x->rows, (long long)x->cols, (long long)w->rows, (long long)w->cols, n, d);
    if (ld < d) return lq_fail(LQ_EINVAL, "matmul_rows: ld=%lld is less than d=%d", (long long)ld, d);
    if (x->rows == 0) return LQ_OK;
    if (!xout || !x->q || !x->s || !w->q || !w->s) return lq_fail(LQ_EINVAL, "matmul_rows: null tensor");
    const int size = type == LQ_F32 ? 4 : 2;
    if (((reinterpret_cast<uintptr_t>(x->q) | reinterpret_cast<uintptr_t>(w->q)) & 15u) ||
        ((reinterpret_cast<uintptr_t>(x->s) | reinterpret_cast<uintptr_t>(w->s)) & 3u) ||
        reinterpret_cast<uintptr_t>(xout) % size)
        return lq_fail(LQ_EINVAL, "matmul_rows: x->q and w->q must be 16-byte aligned, the rest to their elements");
    DevCtx* c = ctx();
    if (!c) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
    const int rows = (int)x->rows, pitch = LQ_ROW8_PITCH(n);
    RowsArgs a;
    a.xs = x->s;
    a.ws = w->s;
    a.y = xout;
    a.ld = ld;
    a.rows = rows;
    a.d = d;
    a.type = type;
    a.kst = (pitch + kStageBytes - 1) / kStageBytes;
    a.early = (launch_flags() & LQ_LAUNCH_PDL) != 0;
    a.err = c->err;
    // Tokens per tile: the fewest that hold them all up to 128; beyond, 256
    // wherever that leaves a tile per SM, else 128.  (Pairs of CTAs: below.)
    const int64_t ct = (d + 127) / 128;
    int N = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    if (N == 256 && ct * ((rows + 255) / 256) < c->num_sms) N = 128;
    const int ctas = 1;
    const int64_t ctiles = (d + 128 * ctas - 1) / (128 * ctas);
    a.ttiles = (rows + N - 1) / N;
    const int64_t tiles = ctiles * a.ttiles;
    if (tiles > INT32_MAX) return lq_fail(LQ_EUNSUPPORTED, "matmul_rows: %lld tiles", (long long)tiles);
    const int groups = c->num_sms / ctas;
    // whole rounds of tiles, the rest cut by stages so that every CTA gets an
    // equal run of at least kMinRun (a cut costs a partial tile's round trip)
    constexpr int kMinRun = 4;
    int64_t shared = tiles % groups;
    int64_t sk = shared * a.kst / kMinRun;
    if (sk > groups) sk = groups;
    if (sk <= shared) shared = sk = 0;  // nothing gained
    a.shared = (int)shared;
    a.whole = (int)(tiles - shared);
    a.sk_grid = (int)sk;
    const int64_t most = tiles - shared > sk ? tiles - shared : sk;
    const int grid = (int)(most < groups ? most : groups) * ctas;
    void* part = nullptr;
    a.cnt = nullptr;
    if (a.shared) {
        int rc = stream_workspace(c, (size_t)grid * 2 * N * 128 * sizeof(int), &a.cnt, &part);
        if (rc) return rc;
    }
    a.part = static_cast<int*>(part);
    if (!byte_map_2d(&a.wmap, w->q, pitch, d, pitch, kStageBytes, 128, true) ||
        !byte_map_2d(&a.xmap, x->q, pitch, rows, pitch, kStageBytes, N / ctas, true))
        return lq_fail(LQ_ECUDA, "matmul_rows: tensor map of %d x %d or %d x %d", d, pitch, rows, pitch);
    cudaError_t e = N == 16   ? rows_launch<16, 1>(a, grid, stream())
                    : N == 32 ? rows_launch<32, 1>(a, grid, stream())
                    : N == 64 ? rows_launch<64, 1>(a, grid, stream())
                    : N == 128 ? rows_launch<128, 1>(a, grid, stream())
                               : rows_launch<256, 1>(a, grid, stream());
    if (e != cudaSuccess) return cuda_fail(e, "matmul_rows launch");
    return LQ_OK;
}

}  // extern "C"
