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
// Each element is read once and one byte written.  A thread keeps
// up to KEEP 16-byte pieces of the row, as they lie in memory, in registers
// between the maximum and the rounding, all loaded at once; rows longer than
// that are read again.  Measured: 2048 rows of 4096 bf16 9 us (2.8 TB/s; DRAM is
// 18% busy, issue slots 56%).  What bounds it is a row's chain of load, maximum,
// barrier, divide and store, and the instructions of the rounding beside it.  40
// registers a thread keep three CTAs of 512 threads on an SM.

template <typename T, bool VEC, int KEEP>
__global__ void __maxnreg__(40)
    quantize_rows_kernel(const T* x, int64_t ld, int n, int8_t* __restrict__ q, int pitch, float* __restrict__ s) {
    constexpr int E = 16 / sizeof(T);  // elements of a piece; their codes are E bytes
    constexpr int W = E / 4;           // elements of a word
    pdl_trigger();
    pdl_wait();
    const T* xr = x + (int64_t)blockIdx.x * ld;
    const int pieces = pitch / E, step = blockDim.x;
    uint4 keep[KEEP];
    uint32_t m = 0;
    auto load = [&](int i) {
        if (VEC && E * i + E <= n) return *reinterpret_cast<const uint4*>(xr + E * i);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[W];
#pragma unroll
            for (int e = 0; e < W; ++e) v[e] = E * i + W * k + e < n ? to_f32(xr[E * i + W * k + e]) : 0.0f;
            w[k] = pack_word<T>(v);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto peak = [&](uint4 p) {
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[W];
            unpack_word<T>(w[k], v);
#pragma unroll
            for (int e = 0; e < W; ++e) m = max(m, abs_bits(v[e]));
        }
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int i = threadIdx.x + j * step;
        if (i < pieces) keep[j] = load(i);
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j)
        if (threadIdx.x + j * step < pieces) peak(keep[j]);
    for (int i = threadIdx.x + KEEP * step; i < pieces; i += step) peak(load(i));
    __shared__ uint32_t wm[32];
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) wm[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, (threadIdx.x & 31) < (step >> 5) ? wm[threadIdx.x & 31] : 0u);
    float sc = __uint_as_float(m) / 127.0f;
    if (sc == 0.0f) sc = 1e-8f;
    if (m >= kInfBits) sc = __uint_as_float(0x7FC00000u);  // a NaN or an infinity: scale NaN, codes 0
    const Quant8 code(sc);
    int8_t* qr = q + (int64_t)blockIdx.x * pitch;
    auto store = [&](int i, uint4 p) {
        float v[E];
        unpack_word<T>(p.x, v);
        unpack_word<T>(p.y, v + W);
        unpack_word<T>(p.z, v + 2 * W);
        unpack_word<T>(p.w, v + 3 * W);
        if constexpr (E == 4)
            reinterpret_cast<uint32_t*>(qr)[i] = code(v[0], v[1], v[2], v[3]);
        else
            reinterpret_cast<uint2*>(qr)[i] = make_uint2(code(v[0], v[1], v[2], v[3]), code(v[4], v[5], v[6], v[7]));
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int i = threadIdx.x + j * step;
        if (i < pieces) store(i, keep[j]);
    }
    for (int i = threadIdx.x + KEEP * step; i < pieces; i += step) store(i, load(i));
    if (threadIdx.x == 0) s[blockIdx.x] = sc;
}

template <typename T>
cudaError_t quantize_rows_t(const void* x, int64_t ld, int64_t rows, int n, int8_t* q, float* s, int sms,
                            cudaStream_t st) {
    constexpr int E = 16 / sizeof(T);
    const T* xt = static_cast<const T*>(x);
    const int pitch = LQ_ROW8_PITCH(n), pieces = pitch / E;
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld % E == 0;
    // Few rows: the time of one, so two pieces a thread.  Many: four, so that
    // more rows are in flight on an SM.
    const int want = rows <= 4 * sms ? 2 : 4;
    int threads = 64;
    while (threads < 1024 && threads * want < pieces) threads *= 2;
    const int keep = (pieces + threads - 1) / threads;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto kern = !vec      ? quantize_rows_kernel<T, false, 4>
                : keep <= 1 ? quantize_rows_kernel<T, true, 1>
                : keep <= 2 ? quantize_rows_kernel<T, true, 2>
                            : quantize_rows_kernel<T, true, 4>;
    return cudaLaunchKernelEx(&cfg, kern, xt, ld, n, q, pitch, s);
}

// ---------------------------------------------------------------------------
// matmul_rows on the tensor cores: tcgen05.mma kind::i8, int32 accumulators in
// tensor memory.  The channels are the MMA's M (128, or 256 by a pair of CTAs)
// and the tokens its N, for every token count: one token is N = 16 with zeros,
// the weights then stream at memory speed, and a thread of the epilogue holds
// one channel of all tokens, so that a warp's store is 32 neighbouring channels.
//
// One persistent CTA (or half a pair) per SM: warps 0 and 6 issue the TMA
// copies (128-byte swizzle; bytes past the row or the tensor read as zeros),
// warp 1 the MMAs, warps 2-5 turn a finished accumulator into outputs while the
// MMAs fill the other.  A tile may hold fewer than 128
// channels, so that the tiles fill whole rounds of the grid: the copies, which
// bound every size here (HBM for few tokens, L2 to SM for many), then are only
// those of its channels, and the MMA's other rows, which compute with whatever
// follows in shared memory, are not read out.
//
// Measured, with quantize_rows before it: 1 x 4096 x 11008 13.5 us (45 MB, 3.3
// TB/s: two launches and one ring of copies to fill and drain are half of it),
// 32 x 5120 x 13824 18.9 us (3.9 TB/s), 2048 x 4096 x 11008 104 us, 87 us of
// them this kernel's (2.1 PTOP/s: the pairs' copies from L2, and the power limit).

constexpr int kRowsThreads = 224;
constexpr int kMaxStages = 12;

// K bytes per stage, in 128-byte halves (the swizzle's width): two halves for
// up to 64 tokens, whose MMAs are short (64 cycles each, 128 x N x 32 for any
// N up to 128), so that waiting and committing once per stage (about 250
// cycles of the issuing thread) is spread over eight of them; one beyond, for
// a deeper ring.
template <int N>
constexpr int rows_halves() {
    return N <= 64 ? 2 : 1;
}

struct RowsArgs {
    CUtensorMap wmap, xmap;
    const float *xs, *ws;
    void* y;
    int64_t ld;
    int rows, d, type;
    int pitch, kst;  // bytes of a row, K stages
    int ttiles;  // tiles along the tokens
    int tiles;
    int m;       // channels per tile and CTA: a multiple of 8, at most 128
    int xbox;    // tokens of an activation copy: no more than there are (an MMA
                 // column past them holds anything and is not read out)
    int stages, rot;
    int* err;
};

struct RowsBars {
    uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2], done;
    uint32_t tmem_base;
    int abort_flag;
};

// one channel of CH tokens: fl(fl(sum) * fl(sx * sw)), rounded to the type
template <int CH, typename T>
__device__ __forceinline__ void store_columns(T* y, int64_t ld, const int (&acc)[CH], float xsv, float wsv, int n,
                                              bool ok) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
        const float f = (float)acc[j] * (__shfl_sync(0xffffffffu, xsv, j) * wsv);
        if (j < n && ok) y[j * ld] = from_f32<T>(f);
    }
}

template <int CH>
__device__ __forceinline__ void store_columns(const RowsArgs& a, int tok, int ch, const int (&v)[CH], int lane) {
    const int n = min(CH, a.rows - tok);
    const float xsv = lane < n ? ld_after(a.xs + tok + lane) : 0.0f;
    const float wsv = ch < a.d ? ld_after(a.ws + ch) : 0.0f;
    const int64_t at = (int64_t)tok * a.ld + ch;
    if (a.type == LQ_F32)
        store_columns<CH>(static_cast<float*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
    else if (a.type == LQ_F16)
        store_columns<CH>(static_cast<__half*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
    else
        store_columns<CH>(static_cast<__nv_bfloat16*>(a.y) + at, a.ld, v, xsv, wsv, n, ch < a.d);
}

// s32 += s8 x s8, both K-major
template <int N, int CTAS>
constexpr uint32_t rows_idesc() {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(8 * CTAS) << 24);
}

template <int N, int CTAS>
__global__ void __launch_bounds__(kRowsThreads, 1) matmul_rows_kernel(const __grid_constant__ RowsArgs a) {
    constexpr int kCols = 2 * N;
    constexpr int CH = N < 32 ? N : 32;
    constexpr int kHalves = rows_halves<N>(), kB = N / CTAS * 128;
    const int kA = a.m * 128, kHalf = kA + kB, kStage = kHalves * kHalf;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    RowsBars* bars = reinterpret_cast<RowsBars*>(sm);
    sm += 1024;
    volatile int* abort_flag = &bars->abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = blockIdx.x / CTAS, groups = gridDim.x / CTAS, rank = CTAS == 2 ? blockIdx.x & 1 : 0;
    const int S = a.stages;
    // Where the weights of a CTA are its own, the CTAs begin at different K
    // stages (an integer sum has no order): together they would all ask L2
    // for the same few lines of the activations.
    const int k0 = a.rot ? (int)((int64_t)group * a.kst / groups) : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&bars->full[i], 2);  // both producers
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
    if (warp == 1) tmem_alloc<CTAS, kCols>(&bars->tmem_base);
    tc_fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    pdl_trigger();
    if (threadIdx.x == 0) {
        prefetch_map(&a.wmap);
        prefetch_map(&a.xmap);
        if (group < a.tiles)  // no read: what the previous kernel still writes is seen by the copies below
            for (int i = 0; i < S * kHalves && 128 * i < a.pitch; ++i)
                tma_prefetch_2d(&a.wmap, (k0 * kHalves + i) * 128 % (a.kst * kHalves * 128),
                                (group / a.ttiles * CTAS + rank) * a.m);
    }
    pdl_wait();

    if (warp == 0 || warp == 6) {
        // warp 0 copies weights, warp 6 activations
        const CUtensorMap* map = warp == 0 ? &a.wmap : &a.xmap;
        const int bytes = warp == 0 ? kA : a.xbox * 128, off = warp == 0 ? 0 : kA;
        const uint64_t pol = l2_normal_policy();
        const uint32_t lead = CTAS == 2 ? cluster_addr(bars->full, 0) : 0;
        int slot = 0, issued = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int tile = group; ok && tile < a.tiles; tile += groups) {
            const int y = warp == 0 ? (tile / a.ttiles * CTAS + rank) * a.m : tile % a.ttiles * N + rank * (N / CTAS);
            for (int i = 0; i < a.kst; ++i) {
                const int k = i + k0 < a.kst ? i + k0 : i + k0 - a.kst;
                ok = __all_sync(0xffffffffu, qwait(&bars->empty[slot], ph ^ 1u, a.err, DEV_TIMEOUT_EMPTY, abort_flag));
                if (!ok) break;
                if (elect_one()) {
                    const int halves = kHalves == 2 && k * 256 + 128 < a.pitch ? 2 : 1;
                    // a pair's copies are all counted on CTA 0's barrier
                    if (rank == 0) mbar_arrive_expect_tx(&bars->full[slot], CTAS * halves * bytes);
#pragma unroll
                    for (int j = 0; j < kHalves; ++j) {
                        unsigned char* at = sm + slot * kStage + j * kHalf + off;
                        const int x = (k * kHalves + j) * 128;
                        if (j < halves) {
                            if (CTAS == 1)
                                tma_load_2d(at, map, x, y, &bars->full[slot], pol);
                            else
                                tma_load_2d_pair(at, map, x, y, lead + slot * 8, pol);
                        }
                    }
                }
                __syncwarp();
                ++issued;
                if (++slot == S) {
                    slot = 0;
                    ph ^= 1u;
                }
            }
        }
        if (*abort_flag && rank == 0 && warp == 0)  // confirm the copies still in flight
            for (int j = max(0, issued - S); j < issued; ++j)
                if (!__all_sync(0xffffffffu, mbar_wait(&bars->full[j % S], (uint32_t)((j / S) & 1), a.err, DEV_TIMEOUT_DRAIN)))
                    break;
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint64_t desc0 = smem_desc_sw128(smem_addr(sm));
            constexpr uint32_t idesc = rows_idesc<N, CTAS>();
            int slot = 0, buf = 0;
            uint32_t ph = 0, bph = 0;
            bool ok = true;
            for (int tile = group; ok && tile < a.tiles; tile += groups) {
                ok = __all_sync(0xffffffffu, qwait(&bars->tempty[buf], bph ^ 1u, a.err, DEV_TIMEOUT_TEMPTY, abort_flag));
                if (!ok) break;
                tc_fence_after();
                const uint32_t dst = tmem + (uint32_t)(buf * N);
                for (int i = 0; i < a.kst; ++i) {
                    const int k = i + k0 < a.kst ? i + k0 : i + k0 - a.kst;
                    ok = __all_sync(0xffffffffu, qwait(&bars->full[slot], ph, a.err, DEV_TIMEOUT_FULL, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t ad = desc0 + (uint32_t)(slot * kStage >> 4), bd = ad + (uint32_t)(kA >> 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j)  // 32 bytes of K each: 2 descriptor units
                            mma_i8_n<CTAS>(dst, ad + 2 * j, bd + 2 * j, idesc, i > 0 || j > 0);
                        if (kHalves == 2 && k * 256 + 128 < a.pitch) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma_i8_n<CTAS>(dst, ad + (uint32_t)(kHalf >> 4) + 2 * j, bd + (uint32_t)(kHalf >> 4) + 2 * j,
                                               idesc, 1);
                        }
                        mma_commit_n<CTAS>(&bars->empty[slot]);
                        if (i == a.kst - 1) mma_commit_n<CTAS>(&bars->tfull[buf]);
                    }
                    __syncwarp();
                    if (++slot == S) {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
                buf ^= 1;
                if (buf == 0) bph ^= 1u;
            }
            if (elect_one()) mma_commit_n<CTAS>(&bars->done);
            __syncwarp();
            mbar_wait(&bars->done, 0, a.err, DEV_TIMEOUT_MMA);  // every MMA is done before the memory is freed
        }
        __syncwarp();
    } else {
        const int q = warp & 3, rr = 32 * q + lane;  // channel within the CTA's 128 = TMEM lane
        int buf = 0;
        uint32_t bph = 0;
        for (int tile = group; tile < a.tiles; tile += groups) {
            if (!__all_sync(0xffffffffu, qwait(&bars->tfull[buf], bph, a.err, DEV_TIMEOUT_TFULL, abort_flag))) break;
            tc_fence_after();
            const uint32_t src = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(buf * N);
            const int tok0 = tile % a.ttiles * N;
            const int ch = rr < a.m ? (tile / a.ttiles * CTAS + rank) * a.m + rr : a.d;
            for (int c = 0; 32 * q < a.m && c < N && tok0 + c < a.rows; c += CH) {
                int v[CH];
                tmem_ld<CH>(src + c, v);
                tmem_ld_wait();
                store_columns<CH>(a, tok0 + c, ch, v, lane);
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
        tmem_free<CTAS, kCols>(tmem);
    }
}

constexpr int kRowsSmem = 227 * 1024;

template <int N, int CTAS>
cudaError_t rows_launch(RowsArgs& a, int sms, cudaStream_t st) {
    // barriers (1 KB), the ring, and what an MMA reads past the last stage's channels
    const int stage = rows_halves<N>() * (a.m + N / CTAS) * 128, slack = (128 - a.m) * 128;
    a.kst = (a.pitch + rows_halves<N>() * 128 - 1) / (rows_halves<N>() * 128);
    const int most = (kRowsSmem - 2048 - slack) / stage;
    a.stages = most < kMaxStages ? most : kMaxStages;
    const int smem = 2048 + a.stages * stage + slack;
    auto kern = matmul_rows_kernel<N, CTAS>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CTAS;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    const int groups = sms / CTAS;
    cfg.gridDim = dim3((a.tiles < groups ? a.tiles : groups) * CTAS);
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = CTAS == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

struct RowsPlan {
    int n, ctas, m;  // tokens per tile, CTAs per tile, channels per CTA
    int64_t rounds;
};

// The narrowest channels per tile with which all tiles of n tokens fit the
// fewest rounds that 128 channels need.
RowsPlan rows_plan(int n, int ctas, int rows, int d, int sms) {
    const int64_t groups = sms / ctas, tt = (rows + n - 1) / n, ct = (d + 128 * ctas - 1) / (128 * ctas);
    const int64_t rounds = (tt * ct + groups - 1) / groups;
    int64_t most = rounds * groups / tt;  // channel tiles that fit
    if (most < ct) most = ct;
    const int64_t m = ((d + most - 1) / most + ctas - 1) / ctas;
    return {n, ctas, (int)((m + 7) / 8 * 8), rounds};
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
        DevCtx* c = ctx();
        if (!c) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
        int8_t* q = static_cast<int8_t*>(out->q);
        cudaError_t e = type == LQ_F32   ? quantize_rows_t<float>(x, ld, out->rows, n, q, out->s, c->num_sms, stream())
                        : type == LQ_F16 ? quantize_rows_t<__half>(x, ld, out->rows, n, q, out->s, c->num_sms, stream())
                                         : quantize_rows_t<__nv_bfloat16>(x, ld, out->rows, n, q, out->s, c->num_sms, stream());
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
    a.pitch = pitch;
    a.rot = 0;
    a.err = c->err;
    // The plan with the least time by rounds * K * time per K + start.
    // Measured, per 128 bytes of K: the copies, about 90 bytes per ns and SM
    // (128 channels x 128 tokens: 0.34 us, x 256: 0.48 us; a pair's 256 x 256:
    // 0.50 us), and at least the MMAs with their waits, 0.17 us (0.19 us
    // beyond 64 tokens); starting and ending take about 6 us, the last tile's
    // outputs 1 us per 64 tokens.
    RowsPlan best = {};
    double least = 0;
    for (int i = 0; i < 6; ++i) {
        const int n = i < 5 ? 16 << i : 256, ctas = i < 5 ? 1 : 2;
        if (n > 16 && n / 2 >= rows) break;  // half of it would do
        const RowsPlan p = rows_plan(n, ctas, rows, d, c->num_sms);
        double stage = ctas == 2 ? 0.50 * (p.m + 128) / 256 : (p.m + n) * 128 / 90e3;
        const double mma = n <= 64 ? 0.17 : 0.19;
        if (stage < mma) stage = mma;
        const double us = 6 + n / 64.0 + p.rounds * (pitch / 128.0) * stage;
        if (!best.n || us < least) {
            best = p;
            least = us;
        }
    }
    const int N = best.n;
    a.m = best.m;
    a.ttiles = (rows + N - 1) / N;
    const int64_t tiles = (int64_t)((d + a.m * best.ctas - 1) / (a.m * best.ctas)) * a.ttiles;
    if (tiles > INT32_MAX / 2) return lq_fail(LQ_EUNSUPPORTED, "matmul_rows: %d x %d outputs", rows, d);
    a.tiles = (int)tiles;
    a.rot = a.ttiles == 1;
    a.xbox = N / best.ctas < rows ? N / best.ctas : rows;
    if (!byte_map_2d(&a.wmap, w->q, pitch, d, pitch, 128, a.m, true) ||
        !byte_map_2d(&a.xmap, x->q, pitch, rows, pitch, 128, a.xbox, true))
        return lq_fail(LQ_ECUDA, "matmul_rows: tensor map of %d x %d or %d x %d", d, pitch, rows, pitch);
    cudaStream_t st = stream();
    const int sms = c->num_sms;
    cudaError_t e = best.ctas == 2 ? rows_launch<256, 2>(a, sms, st)
                    : N == 16      ? rows_launch<16, 1>(a, sms, st)
                    : N == 32      ? rows_launch<32, 1>(a, sms, st)
                    : N == 64      ? rows_launch<64, 1>(a, sms, st)
                    : N == 128     ? rows_launch<128, 1>(a, sms, st)
                                   : rows_launch<256, 1>(a, sms, st);
    if (e != cudaSuccess) return cuda_fail(e, "matmul_rows launch");
    return LQ_OK;
}

}  // extern "C"
