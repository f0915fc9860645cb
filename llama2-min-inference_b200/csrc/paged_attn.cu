// paged_attention: causal attention of ragged rows over the paged int8 cache.
#include <cfloat>
#include <cmath>

#include "lq_ctx.h"
#include "lq_paged.cuh"
#include "lq_paged_host.h"
#include "lq_types.cuh"

namespace lq {
namespace {

struct AttArgs {
    PagedKV c;
    KVBatch b;
    const void* q;
    void* out;
    float* lse;
    int64_t ld_q, ld_out;
    int n_heads;
    float scale;
    int* err;
};

// one warp per (row, head); the cache is walked token by token
template <typename T>
__global__ void __launch_bounds__(128) attend_kernel(const __grid_constant__ AttArgs a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int row = (int)(w / a.n_heads), head = (int)(w % a.n_heads);
    if (row >= a.b.n_rows) return;
    int s = -1;
    for (int i = 0; i < a.b.n_seqs && a.b.row_start[i] <= row; ++i) s = i;
    const int hs = a.c.head_size, P = a.c.page_size, H = a.c.n_kv_heads;
    const int kvh = head / (a.n_heads / H);
    int last = -1;
    if (s >= 0) {
        const SeqRows q = seq_rows(a.b, s, a.err);
        if (row >= q.r0 && row < q.r0 + q.n) last = q.begin + row - q.r0;
    }
    float qv[8], o[8] = {};
    const T* qp = static_cast<const T*>(a.q) + row * a.ld_q + (int64_t)head * hs;
    for (int j = 0; j < 8; ++j) qv[j] = lane + 32 * j < hs ? to_f32(qp[lane + 32 * j]) : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int t = 0; t <= last; ++t) {
        const int64_t page = page_of(a.c, a.b, s, t / P, a.err);
        if (page < 0) continue;
        const int64_t cell = page * H + kvh;
        const int8_t* kc = static_cast<const int8_t*>(a.c.codes) + cell * 2 * hs * P;
        const int8_t* vc = kc + (int64_t)hs * P;
        const float sk = a.c.scales[cell * 2], sv = a.c.scales[cell * 2 + 1];
        const int u = t % P;
        float d = 0.0f;
        for (int j = 0; j < 8; ++j) {
            const int e = lane + 32 * j;
            if (e < hs) d += qv[j] * (float)kc[((int64_t)(e / 16) * P + u) * 16 + e % 16];
        }
        d = warp_sum(d) * (sk * a.scale);
        const float mn = fmaxf(m, d);
        const float c = m == -INFINITY ? 0.0f : expf(m - mn), p = d != d ? d : expf(d - mn);
        l = l * c + p;
        for (int j = 0; j < 8; ++j) {
            const int e = lane + 32 * j;
            if (e < hs) o[j] = o[j] * c + p * sv * (float)vc[((int64_t)(u / 16) * hs + e) * 16 + u % 16];
        }
        m = mn;
    }
    T* op = static_cast<T*>(a.out) + row * a.ld_out + (int64_t)head * hs;
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < hs) op[lane + 32 * j] = from_f32<T>(last < 0 ? 0.0f : o[j] / l);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.n_heads + head] = last < 0 ? -INFINITY : m + logf(l);
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
    if (batch->n_rows == 0) return LQ_OK;
    const int64_t row = (int64_t)n_heads * cache->head_size;
    if (!out || !q || ld_out < row || ld_q < row)
        return lq_fail(LQ_EINVAL, "paged_attention: out or q not set, or rows closer than %lld elements", (long long)row);
    const uintptr_t size = type == LQ_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % size || reinterpret_cast<uintptr_t>(q) % size ||
        (reinterpret_cast<uintptr_t>(lse) & 3u))
        return lq_fail(LQ_EINVAL, "paged_attention: a tensor is not aligned to its elements");
    DevCtx* c = ctx();
    if (!c) return lq_fail(LQ_ECUDA, "no CUDA device context (no device, or first use inside a graph capture)");
    AttArgs a = {*cache, *batch, q, out, lse, ld_q, ld_out, n_heads, scale, c->err};
    const int64_t blocks = ((int64_t)batch->n_rows * n_heads + 3) / 4;
    if (blocks > INT32_MAX) return lq_fail(LQ_EUNSUPPORTED, "paged_attention: too many rows and heads");
    if (type == LQ_F32)
        attend_kernel<float><<<(unsigned)blocks, 128, 0, stream()>>>(a);
    else if (type == LQ_F16)
        attend_kernel<__half><<<(unsigned)blocks, 128, 0, stream()>>>(a);
    else
        attend_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, stream()>>>(a);
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? LQ_OK : cuda_fail(e, "paged_attention launch");
}
