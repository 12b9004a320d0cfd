// Per-head RMSNorm + half-split RoPE + paged append for a ragged batch: every token comes with its own position and its
// own slot of the pools (inf_device_index_append makes both), so one launch serves chunks, drafts and decodes together.
//
//     x' = x w / sqrt(mean x^2 + eps);  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs (d, d + rotary / 2)
//
// HBM-bound: a token's q, k and v rows are read once and written once as fp16.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "rows.cuh"

namespace {

constexpr int D = 128;
constexpr int THREADS = 256;

struct AppendArgs {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;  // elements between tokens
    const float *qw, *kw, *inv_freq;
    int rotary_dim;
    float factor, eps;
    __half *k_pool, *v_pool, *q_out;
    const int *positions, *slots;
    int tokens, q_heads, kv_heads, page_size, num_pages;
    int* status;
};

// cos and sin of position * inv_freq.  The product has up to 55 significant bits and only its remainder by a turn
// matters: in 32 bits the angle of position 30 000 is off by 1e-3, so the product and its remainder are taken in 64 and
// cos / sin of an angle of at most half a turn in 32.
__device__ __forceinline__ float2 turn_of(int position, float inv_freq, float factor) {
    constexpr double TURN = 6.283185307179586476925;
    const double angle = (double)position * (double)inv_freq;
    const float r = (float)fma(-rint(angle * (1.0 / TURN)), TURN, angle);
    float s, c;
    sincosf(r, &s, &c);
    return make_float2(c * factor, s * factor);
}

// One CTA per token; 16 threads hold a row of 128 values, eight consecutive ones each, and the rotation partner sits
// rotary / 16 lanes away.
template <typename T>
__global__ void __launch_bounds__(THREADS)
rope_append_ragged_kernel(AppendArgs p) {
    __shared__ float2 s_cs[64];
    inf_pdl_wait();
    inf_pdl_release();
    const int t = blockIdx.x, tid = threadIdx.x, sub = tid & 15, d0 = sub * 8;
    const int position = p.positions[t], slot = p.slots[t];
    if (position < 0) return;  // a padding row
    const int half = p.rotary_dim >> 1;
    if (p.inv_freq && tid < half) s_cs[tid] = turn_of(position, p.inv_freq[tid], p.factor);
    const bool stored = slot >= 0 && slot < (long long)p.num_pages * p.page_size;
    if (!stored && tid == 0) atomicOr(p.status, INF_STATUS_BAD_PAGE);
    __syncthreads();
    const int rows = p.q_heads + 2 * p.kv_heads, partner = half >> 3;
    for (int base = 0; base < rows; base += THREADS / 16) {  // the same trips for every thread
        const int rr = base + (tid >> 4);
        const int kind = rr < p.q_heads ? 0 : (rr < p.q_heads + p.kv_heads ? 1 : 2);
        const int head = kind == 0 ? rr : (kind == 1 ? rr - p.q_heads : rr - p.q_heads - p.kv_heads);
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (rr < rows) {
            const T* src = (const T*)(kind == 0 ? p.q : (kind == 1 ? p.k : p.v)) +
                           (long long)t * (kind == 0 ? p.q_stride : (kind == 1 ? p.k_stride : p.v_stride)) + (long long)head * D + d0;
            Raw8<T> raw;
            raw.load(src);
            raw.to_f32(x);
        }
        if (p.inv_freq) {  // whole warps take part in the shuffles; rows that are not turned drop the result
            const float* w = kind == 0 ? p.qw : p.kw;
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (kind != 2 && w) {
                const float inv_rms = rsqrtf(ss / (float)D + p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = x[j] * w[d0 + j] * inv_rms;
            }
            const bool first = d0 < half, second = !first && d0 < p.rotary_dim;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float other = __shfl_xor_sync(0xffffffffu, x[j], partner);
                if (kind != 2 && (first || second)) {
                    const float2 cs = s_cs[first ? d0 + j : d0 + j - half];
                    x[j] = first ? x[j] * cs.x - other * cs.y : x[j] * cs.x + other * cs.y;
                }
            }
        }
        if (rr >= rows) continue;
        if (kind == 0) {
            st8_as_f16(p.q_out + ((long long)t * p.q_heads + head) * D + d0, x);
        } else if (stored) {
            const int page = slot / p.page_size;
            const long long row = ((long long)page * p.kv_heads + head) * p.page_size + (slot - page * p.page_size);
            st8_as_f16((kind == 1 ? p.k_pool : p.v_pool) + row * D + d0, x);
        }
    }
}

}  // namespace

extern "C" int32_t inf_rope_append_gqa_ragged(inf_ctx* ctx, const void* q, const void* k, const void* v, int64_t q_stride,
                                              int64_t k_stride, int64_t v_stride, int32_t in_dtype,
                                              const float* q_norm_weight, const float* k_norm_weight, float eps,
                                              const inf_rope_table* rope, const inf_kv_pool* pool,
                                              const int32_t* positions, const int32_t* slots, int32_t tokens,
                                              int32_t q_heads, void* q_out_f16) {
    INF_CHECK_CTX(ctx);
    return inf_entry(ctx, [&]() -> int {
        const char* what = "rope_append_gqa_ragged";
        if (!pool) return inf_fail(ctx, INF_E_ARG, "%s: null pool", what);
        if (!pool->k || !pool->v) return inf_fail(ctx, INF_E_ARG, "%s: pool has no storage", what);
        if (pool->head_dim != D) return inf_fail(ctx, INF_E_SHAPE, "%s: head_dim must be 128, got %d", what, pool->head_dim);
        if (pool->num_pages <= 0 || pool->page_size <= 0 || pool->kv_heads <= 0)
            return inf_fail(ctx, INF_E_CACHE, "%s: pool sizes must be positive", what);
        if ((long long)pool->num_pages * pool->page_size > 0x7fffffffLL)
            return inf_fail(ctx, INF_E_CACHE, "%s: token slots must be countable in 31 bits", what);
        if (tokens < 0) return inf_fail(ctx, INF_E_SHAPE, "%s: tokens must not be negative", what);
        if (q_heads <= 0 || q_heads % pool->kv_heads != 0)
            return inf_fail(ctx, INF_E_SHAPE, "%s: q_heads %d must be a positive multiple of kv_heads %d", what, q_heads, pool->kv_heads);
        if (in_dtype != INF_DTYPE_F32 && in_dtype != INF_DTYPE_F16)
            return inf_fail(ctx, INF_E_DTYPE, "%s: input dtype must be f32 or f16", what);
        if (!isfinite(eps) || eps < 0.f) return inf_fail(ctx, INF_E_CONFIG, "%s: eps must be finite and not negative", what);
        if (rope) {
            if (!rope->inv_freq) return inf_fail(ctx, INF_E_ARG, "%s: rope table has no device frequencies", what);
            if (rope->rotary_dim != 64 && rope->rotary_dim != 128)
                return inf_fail(ctx, INF_E_BACKEND, "%s: rotary dimension must be 64 or 128, got %d", what, rope->rotary_dim);
        } else if (q_norm_weight || k_norm_weight) {
            return inf_fail(ctx, INF_E_CONFIG, "%s: a norm without a rope table is not offered", what);
        }
        if (tokens == 0) return INF_OK;
        if (!q || !k || !v || !positions || !slots || !q_out_f16) return inf_fail(ctx, INF_E_ARG, "%s: null pointer", what);
        const long long esz = in_dtype == INF_DTYPE_F16 ? 2 : 4;
        if (q_stride < (long long)q_heads * D || k_stride < (long long)pool->kv_heads * D || v_stride < (long long)pool->kv_heads * D)
            return inf_fail(ctx, INF_E_SHAPE, "%s: token strides %lld, %lld, %lld are shorter than a token's heads", what,
                            (long long)q_stride, (long long)k_stride, (long long)v_stride);
        if ((q_stride * esz) % 16 || (k_stride * esz) % 16 || (v_stride * esz) % 16 ||
            (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out_f16 | (uintptr_t)pool->k | (uintptr_t)pool->v) & 15u))
            return inf_fail(ctx, INF_E_ARG, "%s: tensors and token strides must be 16-byte aligned", what);
        AppendArgs p{q, k, v, q_stride, k_stride, v_stride, q_norm_weight, k_norm_weight, rope ? rope->inv_freq : nullptr,
                     rope ? rope->rotary_dim : 64, rope ? rope->attention_factor : 1.0f, eps, (__half*)pool->k, (__half*)pool->v,
                     (__half*)q_out_f16, positions, slots, tokens, q_heads, pool->kv_heads, pool->page_size, pool->num_pages, ctx->status};
        auto kernel = in_dtype == INF_DTYPE_F16 ? rope_append_ragged_kernel<__half> : rope_append_ragged_kernel<float>;
        INF_CUDA(ctx, inf_launch_pdl(kernel, dim3((unsigned)tokens), dim3(THREADS), 0, ctx->stream, p));
        return INF_OK;
    });
}
