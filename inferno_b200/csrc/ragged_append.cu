// Per-head RMSNorm + half-split RoPE + paged append for a ragged batch: every token comes with its own position and its
// own slot of the pools (inf_device_index_append makes both), so one launch serves chunks, drafts and decodes together.
//
//     x' = x w / sqrt(mean x^2 + eps);  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs (d, d + rotary / 2)
//
// HBM-bound: a token's q, k and v rows are read once and written once as fp16.  8192 tokens of 48 + 2 x 8 fp16 heads move
// 268 MB in 49.8 us, 0.82 of the measured copy bandwidth; a single token takes 4.1 us of a graph.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "ptx.cuh"

using namespace inf;

namespace {

constexpr int D = 128;
constexpr int THREADS = 128;

struct AppendArgs {
    const void *q, *k, *v;
    long long q_stride, k_stride, v_stride;  // elements between tokens
    const float *qw, *kw, *inv_freq;
    float factor, eps;
    __half *k_pool, *v_pool, *q_out;
    const int *positions, *slots;
    int tokens, parts;  // warps of a token
    int q_heads, kv_heads, page_size, slots_total;
    int* status;
};

// cos and sin of position * inv_freq.  The product has up to 55 significant bits and only its remainder by a turn
// matters: in 32 bits the angle of position 30 000 is off by 1e-3, so it is counted in half turns and reduced to at most
// one of them in 64 bits, and cos / sin are taken of the remainder in 32.
__device__ __forceinline__ float2 turn_of(int position, float inv_freq, float factor) {
    const double turns = (double)position * (double)inv_freq * 0.15915494309189533577;
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    return make_float2(c * factor, s * factor);
}

// Two pieces of four consecutive values of a row, as they lie in memory.
template <typename T>
struct Pieces;
template <>
struct Pieces<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* at, int apart) {
        a = *reinterpret_cast<const float4*>(at);
        b = *reinterpret_cast<const float4*>(at + apart);
    }
    __device__ __forceinline__ void to_f32(uint64_t (&x)[2], uint64_t (&y)[2]) const {
        x[0] = pack_f32x2(a.x, a.y), x[1] = pack_f32x2(a.z, a.w), y[0] = pack_f32x2(b.x, b.y), y[1] = pack_f32x2(b.z, b.w);
    }
};
template <>
struct Pieces<__half> {
    uint2 a, b;
    __device__ __forceinline__ void load(const __half* at, int apart) {
        a = *reinterpret_cast<const uint2*>(at);
        b = *reinterpret_cast<const uint2*>(at + apart);
    }
    static __device__ __forceinline__ uint64_t pair(uint32_t h) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        return pack_f32x2(f.x, f.y);
    }
    __device__ __forceinline__ void to_f32(uint64_t (&x)[2], uint64_t (&y)[2]) const {
        x[0] = pair(a.x), x[1] = pair(a.y), y[0] = pair(b.x), y[1] = pair(b.y);
    }
};
__device__ __forceinline__ void st4_as_f16(__half* p, const uint64_t (&x)[2]) {
    float f[4];
    unpack_f32x2(x[0], f[0], f[1]);
    unpack_f32x2(x[1], f[2], f[3]);
    __half2 h[2] = {__floats2half2_rn(f[0], f[1]), __floats2half2_rn(f[2], f[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
}
__device__ __forceinline__ uint64_t shfl_xor2(uint64_t v, int o) {
    float a, b;
    unpack_f32x2(v, a, b);
    return pack_f32x2(__shfl_xor_sync(0xffffffffu, a, o), __shfl_xor_sync(0xffffffffu, b, o));
}

// A warp works on one token, or with `parts` > 1 on every parts-th pair of its rows.  16 lanes hold a row, each four
// values and their four rotation partners, so a rotation needs no other lane, its four cosines and sines stay in
// registers for all rows, and a warp's 8-byte accesses still fill whole sectors.  Eight neighbouring values a lane need
// eight shuffles a step for the partners and twice the cosines: 69 us instead of 49.8 for those 8192 tokens.  Rows are
// requested AHEAD steps before they are worked on, the first ones before the position is known.  No barriers.
template <typename T, int HALF>  // HALF: half the rotary dimension, what lies between partners
__global__ void __launch_bounds__(THREADS, 8)
rope_append_ragged_kernel(AppendArgs p) {
    constexpr int AHEAD = sizeof(T) == 2 ? 4 : 2;  // what 64 registers hold
    inf_pdl_wait();
    inf_pdl_release();
    const int lane = threadIdx.x & 31, sub = lane & 15, upper = lane >> 4;
    const long long unit = (long long)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const int t = (int)(unit / p.parts), part = (int)(unit - (long long)t * p.parts);
    if (t >= p.tokens) return;
    // a row's rotated part is HALF / 4 lanes wide, what is left of it the others'
    const bool turned = 4 * sub < HALF && p.inv_freq;
    const int column = 4 * sub < HALF ? 4 * sub : HALF + 4 * sub;
    const int rows = p.q_heads + 2 * p.kv_heads, keys_from = p.q_heads, values_from = p.q_heads + p.kv_heads;
    // rows are counted through queries, keys and values: each base stands where row 0 would
    const T* q = (const T*)p.q + t * p.q_stride + column;
    const T* k = (const T*)p.k + t * p.k_stride + column - (long long)keys_from * D;
    const T* v = (const T*)p.v + t * p.v_stride + column - (long long)values_from * D;
    const int first = 2 * part + upper, stride = 2 * p.parts;  // this half-warp's rows
    auto request = [&](Pieces<T>& raw, int rr) {
        rr = min(rr, rows - 1);
        raw.load((rr < keys_from ? q : (rr < values_from ? k : v)) + (long long)rr * D, HALF);
    };
    Pieces<T> raw[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) request(raw[u], first + u * stride);
    const int position = p.positions[t], slot = p.slots[t];
    if (position < 0) return;  // a padding row
    const bool stored = slot >= 0 && slot < p.slots_total;
    if (!stored && part == 0 && lane == 0) atomicOr(p.status, INF_STATUS_BAD_PAGE);
    const int page = stored ? slot / p.page_size : 0;
    const long long pool_step = (long long)p.page_size * D;  // from a head to the next one of a page
    const long long pool_row = ((long long)page * p.kv_heads * p.page_size + (slot - page * p.page_size)) * D + column;
    __half* const q_to = p.q_out + (long long)t * p.q_heads * D + column;
    __half* const k_to = p.k_pool + pool_row - keys_from * pool_step;
    __half* const v_to = p.v_pool + pool_row - values_from * pool_step;
    uint64_t c[2] = {0, 0}, s[2] = {0, 0};
    if (p.inv_freq) {
        // the half-warps make two of the four each
        const int f = turned ? 4 * sub + 2 * upper : 0;
        const float2 e0 = turn_of(position, p.inv_freq[f], p.factor), e1 = turn_of(position, p.inv_freq[f + 1], p.factor);
        const uint64_t my_c = pack_f32x2(e0.x, e1.x), my_s = pack_f32x2(e0.y, e1.y);
        const uint64_t its_c = shfl_xor2(my_c, 16), its_s = shfl_xor2(my_s, 16);
        c[0] = upper ? its_c : my_c, c[1] = upper ? my_c : its_c;
        s[0] = upper ? its_s : my_s, s[1] = upper ? my_s : its_s;
    }
#pragma unroll 1
    for (int base = first; base - upper < rows; base += AHEAD * stride) {  // the same trips for the whole warp
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int rr = base + u * stride;
            uint64_t x[2], y[2];
            raw[u].to_f32(x, y);
            request(raw[u], rr + AHEAD * stride);
            if (p.inv_freq && rr - upper < values_from) {  // a query or a key among the warp's two rows
                const float* w = rr < keys_from ? p.qw : p.kw;
                if (p.qw || p.kw) {
                    const uint64_t sq = fma_f32x2(y[1], y[1], fma_f32x2(y[0], y[0], fma_f32x2(x[1], x[1], mul_f32x2(x[0], x[0]))));
                    float sum, odd;
                    unpack_f32x2(sq, sum, odd);
                    sum += odd;
#pragma unroll
                    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (w && rr < values_from) {
                        const float scale = rsqrtf(sum * (1.0f / D) + p.eps);
                        const uint64_t scale2 = pack_f32x2(scale, scale);
                        const float4 wa = *reinterpret_cast<const float4*>(w + column), wb = *reinterpret_cast<const float4*>(w + column + HALF);
                        x[0] = mul_f32x2(mul_f32x2(x[0], pack_f32x2(wa.x, wa.y)), scale2);
                        x[1] = mul_f32x2(mul_f32x2(x[1], pack_f32x2(wa.z, wa.w)), scale2);
                        y[0] = mul_f32x2(mul_f32x2(y[0], pack_f32x2(wb.x, wb.y)), scale2);
                        y[1] = mul_f32x2(mul_f32x2(y[1], pack_f32x2(wb.z, wb.w)), scale2);
                    }
                }
                if (turned && rr < values_from) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint64_t a = x[j], b = y[j];
                        x[j] = fma_f32x2(b ^ 0x8000000080000000ull, s[j], mul_f32x2(a, c[j]));
                        y[j] = fma_f32x2(a, s[j], mul_f32x2(b, c[j]));
                    }
                }
            }
            if (rr < rows && (rr < keys_from || stored)) {
                __half* to = (rr < keys_from ? q_to : (rr < values_from ? k_to : v_to)) + rr * (rr < keys_from ? (long long)D : pool_step);
                st4_as_f16(to, x);
                st4_as_f16(to + HALF, y);
            }
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
            (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out_f16 | (uintptr_t)pool->k | (uintptr_t)pool->v |
              (uintptr_t)q_norm_weight | (uintptr_t)k_norm_weight) & 15u))
            return inf_fail(ctx, INF_E_ARG, "%s: tensors and token strides must be 16-byte aligned", what);
        // A token's rows in one warp, unless that leaves SMs without work: then up to eight warps share them.
        int parts = 1;
        while (parts < 8 && (long long)tokens * parts < 8LL * ctx->sm_count) parts *= 2;
        AppendArgs p{q, k, v, q_stride, k_stride, v_stride, q_norm_weight, k_norm_weight, rope ? rope->inv_freq : nullptr,
                     rope ? rope->attention_factor : 1.0f, eps, (__half*)pool->k, (__half*)pool->v,
                     (__half*)q_out_f16, positions, slots, tokens, parts, q_heads, pool->kv_heads, pool->page_size, pool->num_pages * pool->page_size, ctx->status};
        const bool wide = rope && rope->rotary_dim == 128, f16 = in_dtype == INF_DTYPE_F16;
        auto kernel = f16 ? (wide ? rope_append_ragged_kernel<__half, 64> : rope_append_ragged_kernel<__half, 32>)
                          : (wide ? rope_append_ragged_kernel<float, 64> : rope_append_ragged_kernel<float, 32>);
        const long long blocks = ((long long)tokens * parts + THREADS / 32 - 1) / (THREADS / 32);
        INF_CUDA(ctx, inf_launch_pdl(kernel, dim3((unsigned)blocks), dim3(THREADS), 0, ctx->stream, p));
        return INF_OK;
    });
}
