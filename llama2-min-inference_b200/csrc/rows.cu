// Token-scaled int8 products: quantize_rows (one scale per row) and
// matmul_rows (int8 x int8 with a scale per token and per output channel).
#include "lq_ctx.h"
#include "lq_device.cuh"
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
// matmul_rows: a warp per (8 tokens, channel), dp4a over the row.

template <typename T>
__global__ void __launch_bounds__(256) matmul_rows_kernel(const int8_t* __restrict__ x, const float* __restrict__ xs,
                                                          int rows, const int8_t* __restrict__ w,
                                                          const float* __restrict__ ws, int d, int pitch,
                                                          T* __restrict__ y, int64_t ld) {
    const int lane = threadIdx.x & 31;
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int b0 = blockIdx.y * 8;
    if (i >= d) return;
    const int nb = min(8, rows - b0);
    int acc[8] = {};
    const uint4* wr = reinterpret_cast<const uint4*>(w + (int64_t)i * pitch);
    for (int k = lane; k < pitch / 16; k += 32) {
        const uint4 a = wr[k];
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            if (b < nb) {
                const uint4 v = reinterpret_cast<const uint4*>(x + (int64_t)(b0 + b) * pitch)[k];
                acc[b] = __dp4a((int)a.x, (int)v.x, acc[b]);
                acc[b] = __dp4a((int)a.y, (int)v.y, acc[b]);
                acc[b] = __dp4a((int)a.z, (int)v.z, acc[b]);
                acc[b] = __dp4a((int)a.w, (int)v.w, acc[b]);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const int t = __reduce_add_sync(0xffffffffu, acc[b]);
        if (lane == 0 && b < nb) y[(int64_t)(b0 + b) * ld + i] = from_f32<T>((float)t * (xs[b0 + b] * ws[i]));
    }
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
    const int rows = (int)x->rows;
    const int pitch = LQ_ROW8_PITCH(n);
    const int8_t *xq = static_cast<const int8_t*>(x->q), *wq = static_cast<const int8_t*>(w->q);
    for (int r0 = 0; r0 < rows; r0 += 65535 * 8) {
        const int rn = rows - r0 < 65535 * 8 ? rows - r0 : 65535 * 8;
        const dim3 grid((d + 7) / 8, (rn + 7) / 8);
        const int8_t* xp = xq + (int64_t)r0 * pitch;
        if (type == LQ_F32)
            matmul_rows_kernel<float><<<grid, 256, 0, stream()>>>(xp, x->s + r0, rn, wq, w->s, d, pitch,
                                                                  static_cast<float*>(xout) + r0 * ld, ld);
        else if (type == LQ_F16)
            matmul_rows_kernel<__half><<<grid, 256, 0, stream()>>>(xp, x->s + r0, rn, wq, w->s, d, pitch,
                                                                   static_cast<__half*>(xout) + r0 * ld, ld);
        else
            matmul_rows_kernel<__nv_bfloat16><<<grid, 256, 0, stream()>>>(
                xp, x->s + r0, rn, wq, w->s, d, pitch, static_cast<__nv_bfloat16*>(xout) + r0 * ld, ld);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "matmul_rows launch");
    }
    return LQ_OK;
}

}  // extern "C"
