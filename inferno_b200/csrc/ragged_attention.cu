// Causal attention of a ragged batch over paged K/V: every sequence brings its own number of new tokens (a prompt chunk,
// a few drafts, one decode token, or none), their keys and values already in the pages.
//
// Row t of sequence b stands at p = past_b + t and sees the keys [max(0, p + 1 - window), p]:
//     o = softplus(gate) * sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q . k_j,  m = max_j s_j
// in one pass over the keys with a running maximum and sum.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "ptx.cuh"

using namespace inf;

namespace {

constexpr int D = 128;
constexpr float M_INIT = -1.0e30f;

struct RaggedParams {
    const __half* q;
    const __half *k, *v;
    const int *pages, *lens, *starts;
    int batch, max_pages, tokens, q_heads, kv_heads, group, page_size, num_pages, window;
    float scale_log2;
    const float* gate;
    void* out;
    int out_f16;
    int* status;
};

// log(1 + e^v): log1p, because 1 + e^v keeps nothing but 2^-24 of e^v, which is 1e-3 of it at v = -10.
__device__ __forceinline__ float softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// A sequence's rows and cached keys; false (and the status word) where they do not fit what the launch was given.
__device__ __forceinline__ bool sequence_of(const RaggedParams& p, int b, int& start, int& n, int& past) {
    start = p.starts[b];
    n = p.starts[b + 1] - start;
    past = p.lens[b];
    if (n == 0) return false;
    if (start < 0 || n < 0 || (long long)start + n > p.tokens || past < 0 || (long long)past + n > (long long)p.max_pages * p.page_size) {
        atomicOr(p.status, INF_STATUS_BAD_LEN);
        return false;
    }
    return true;
}

// One warp per (token, query head): lane holds four of the 128 dims, keys one after the other.
__global__ void __launch_bounds__(256)
ragged_attention_kernel(RaggedParams p) {
    inf_pdl_wait();
    inf_pdl_release();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int t = (int)(row / p.q_heads), h = (int)(row % p.q_heads);
    if (t >= p.tokens) return;
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.starts[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    int start, n, past;
    if (!sequence_of(p, lo, start, n, past) || t < start || t >= start + n) return;
    const int pos = past + t - start;
    const int first = p.window > 0 ? max(0, pos + 1 - p.window) : 0;
    const uint2 qraw = reinterpret_cast<const uint2*>(p.q + row * D)[lane];
    const float2 q0 = __half22float2(*reinterpret_cast<const __half2*>(&qraw.x)), q1 = __half22float2(*reinterpret_cast<const __half2*>(&qraw.y));
    float m = M_INIT, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int key = first; key <= pos; ++key) {
        const int page = p.pages[(long long)lo * p.max_pages + key / p.page_size];
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) atomicOr(p.status, INF_STATUS_BAD_PAGE);
            continue;
        }
        const long long at = (((long long)page * p.kv_heads + h / p.group) * p.page_size + key % p.page_size) * D;
        const uint2 kr = reinterpret_cast<const uint2*>(p.k + at)[lane], vr = reinterpret_cast<const uint2*>(p.v + at)[lane];
        const float2 k0 = __half22float2(*reinterpret_cast<const __half2*>(&kr.x)), k1 = __half22float2(*reinterpret_cast<const __half2*>(&kr.y));
        float s = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= p.scale_log2;
        const float m_new = fmaxf(m, s), alpha = ex2_approx(m - m_new), w = ex2_approx(s - m_new);
        const float2 v0 = __half22float2(*reinterpret_cast<const __half2*>(&vr.x)), v1 = __half22float2(*reinterpret_cast<const __half2*>(&vr.y));
        m = m_new;
        l = l * alpha + w;
        o[0] = o[0] * alpha + w * v0.x, o[1] = o[1] * alpha + w * v0.y;
        o[2] = o[2] * alpha + w * v1.x, o[3] = o[3] * alpha + w * v1.y;
    }
    float gain = l > 0.f ? 1.0f / l : 0.f;
    if (p.gate) gain *= softplus(p.gate[row]);
    if (p.out_f16)
        reinterpret_cast<uint2*>((__half*)p.out + row * D)[lane] = make_uint2(pack_half2(o[0] * gain, o[1] * gain), pack_half2(o[2] * gain, o[3] * gain));
    else
        reinterpret_cast<float4*>((float*)p.out + row * D)[lane] = make_float4(o[0] * gain, o[1] * gain, o[2] * gain, o[3] * gain);
}

}  // namespace

extern "C" int32_t inf_gqa_attention_ragged(inf_ctx* ctx, const void* q_f16, const inf_kv_pool* pool,
                                            const inf_page_table* table, const int32_t* q_starts, int32_t tokens,
                                            int32_t q_heads, int32_t sliding_window, const float* gate, float scale,
                                            void* out, int32_t out_dtype) {
    INF_CHECK_CTX(ctx);
    return inf_entry(ctx, [&]() -> int {
        const char* what = "gqa_attention_ragged";
        if (!pool || !table) return inf_fail(ctx, INF_E_ARG, "%s: null pool or page table", what);
        if (!pool->k || !pool->v) return inf_fail(ctx, INF_E_ARG, "%s: pool has no storage", what);
        if (pool->head_dim != D) return inf_fail(ctx, INF_E_SHAPE, "%s: head_dim must be 128, got %d", what, pool->head_dim);
        if (pool->num_pages <= 0 || pool->kv_heads <= 0 || pool->page_size <= 0 || pool->page_size % 16 != 0)
            return inf_fail(ctx, INF_E_CACHE, "%s: page_size must be a positive multiple of 16, got %d", what, pool->page_size);
        if ((long long)pool->num_pages * pool->kv_heads * pool->page_size >= 0x7fffffffLL)
            return inf_fail(ctx, INF_E_CACHE, "%s: the pool's rows must be countable in 31 bits", what);
        if (tokens < 0) return inf_fail(ctx, INF_E_SHAPE, "%s: tokens must not be negative", what);
        if (q_heads <= 0 || q_heads % pool->kv_heads != 0)
            return inf_fail(ctx, INF_E_SHAPE, "%s: q_heads %d must be a positive multiple of kv_heads %d", what, q_heads, pool->kv_heads);
        if (q_heads / pool->kv_heads > 128) return INF_UNSUPPORTED;
        if (sliding_window < 0) return inf_fail(ctx, INF_E_CONFIG, "%s: sliding_window must be >= 0", what);
        if (!isfinite(scale)) return inf_fail(ctx, INF_E_CONFIG, "%s: scale must be finite", what);
        if (out_dtype != INF_DTYPE_F32 && out_dtype != INF_DTYPE_F16)
            return inf_fail(ctx, INF_E_DTYPE, "%s: output dtype must be f32 or f16", what);
        int rc = inf_validate_table(ctx, table, pool->num_pages, pool->page_size, 0, what, sliding_window, 1);
        if (rc != INF_OK) return rc;
        if (tokens == 0) return INF_OK;
        if (!q_f16 || !q_starts || !out) return inf_fail(ctx, INF_E_ARG, "%s: null pointer", what);
        if (((uintptr_t)q_f16 | (uintptr_t)out | (uintptr_t)pool->k | (uintptr_t)pool->v) & 15u)
            return inf_fail(ctx, INF_E_ARG, "%s: tensors must be 16-byte aligned", what);
        RaggedParams p{};
        p.q = (const __half*)q_f16;
        p.k = (const __half*)pool->k;
        p.v = (const __half*)pool->v;
        p.pages = table->pages;
        p.lens = table->lens;
        p.starts = q_starts;
        p.batch = table->batch;
        p.max_pages = table->max_pages;
        p.tokens = tokens;
        p.q_heads = q_heads;
        p.kv_heads = pool->kv_heads;
        p.group = q_heads / pool->kv_heads;
        p.page_size = pool->page_size;
        p.num_pages = pool->num_pages;
        p.window = sliding_window;
        p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf((float)D)) * 1.4426950408889634f;
        p.gate = gate;
        p.out = out;
        p.out_f16 = out_dtype == INF_DTYPE_F16;
        p.status = ctx->status;
        const long long rows = (long long)tokens * q_heads;
        if ((rows + 7) / 8 > 0x7fffffffLL) return inf_fail(ctx, INF_E_SHAPE, "%s: tokens x heads exceeds the launch grid", what);
        INF_CUDA(ctx, inf_launch_pdl(ragged_attention_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, ctx->stream, p));
        return INF_OK;
    });
}
