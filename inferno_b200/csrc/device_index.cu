// Page bookkeeping on the GPU: the device twin of paged_index.cu, for batches whose request lengths live on the GPU.
//
// With past_b tokens cached and n_b new ones, P tokens per page, sequence b needs
//     need_b = ceil((past_b + n_b) / P) - ceil(past_b / P)
// pages; the free list is a stack, and page j of sequence b's is the (sum_{b' < b} need_b' + j)-th from its top, which
// is the page inf_paged_index_append called for one sequence after the other would hand out.  Dropping tokens pushes
// pages in the reverse order (the last sequence's last page first), so an append followed by a truncate to the old
// lengths restores the free list exactly.  Both are prefix sums over the batch; a few KB move, so what counts is the
// length of the chain of dependent loads.
#include "common.cuh"

namespace {

constexpr int THREADS = 1024;
constexpr int WARPS = THREADS / 32;

struct IndexArgs {
    int* pages;
    int* lens;
    int* free_pages;
    int* free_count;
    int num_pages, page_size, seqs, max_pages;
    int* status;
};

// Sum over the block of one value per thread and, per thread, the sum over the threads before it.
__device__ __forceinline__ long long block_scan(long long v, long long& before, long long* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    __syncthreads();  // the warp sums of the call before this one have been read
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    long long base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const long long x = s_warp[w];
        if (w < warp) base += x;
        total += x;
    }
    before = base + inc - v;
    return total;
}

__device__ __forceinline__ int pages_of(long long tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }

__global__ void __launch_bounds__(THREADS)
device_index_append_kernel(IndexArgs a, const int* __restrict__ new_tokens, int max_tokens, int* __restrict__ past_lens,
                           int* __restrict__ q_starts, int* __restrict__ positions, int* __restrict__ slots) {
    __shared__ long long s_warp[WARPS];
    inf_pdl_wait();
    inf_pdl_release();
    const int tid = threadIdx.x;
    const long long capacity = (long long)a.max_pages * a.page_size;
    const int free_count = *a.free_count;
    // ---- a step that does not fit is refused as a whole, before anything of the index changes
    int bad = free_count < 0 || free_count > a.num_pages ? INF_STATUS_NO_PAGES : 0;
    long long tokens = 0, need = 0;
    for (int b = tid; b < a.seqs; b += THREADS) {
        const int past = a.lens[b], n = new_tokens[b];
        if (past < 0 || n < 0 || (long long)past + n > capacity) {
            bad |= INF_STATUS_BAD_LEN;
        } else {
            tokens += n;
            need += pages_of((long long)past + n, a.page_size) - pages_of(past, a.page_size);
        }
    }
    long long unused;
    const long long total = block_scan(tokens, unused, s_warp);
    const long long fresh_total = block_scan(need, unused, s_warp);
    if (total > max_tokens) bad |= INF_STATUS_BAD_LEN;
    if (fresh_total > free_count) bad |= INF_STATUS_NO_PAGES;
    if (__syncthreads_or(bad)) {
        if (bad) atomicOr(a.status, bad);
        for (int b = tid; b < a.seqs; b += THREADS) past_lens[b] = a.lens[b];
        for (int b = tid; b <= a.seqs; b += THREADS) q_starts[b] = 0;
        for (int t = tid; t < max_tokens; t += THREADS) positions[t] = slots[t] = -1;
        return;
    }
    // ---- pages and starts, a block of sequences at a time
    long long token0 = 0, page0 = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += THREADS) {
        const int b = b0 + tid;
        const int past = b < a.seqs ? a.lens[b] : 0, n = b < a.seqs ? new_tokens[b] : 0;
        const int mapped = pages_of(past, a.page_size), fresh = pages_of((long long)past + n, a.page_size) - mapped;
        long long tokens_before, pages_before;
        const long long tokens_here = block_scan(n, tokens_before, s_warp);
        const long long pages_here = block_scan(fresh, pages_before, s_warp);
        if (b < a.seqs) {
            past_lens[b] = past;
            q_starts[b] = (int)(token0 + tokens_before);
            for (int j = 0; j < fresh; ++j)
                a.pages[(long long)b * a.max_pages + mapped + j] = a.free_pages[free_count - 1 - (int)(page0 + pages_before) - j];
            a.lens[b] = past + n;
        }
        token0 += tokens_here;
        page0 += pages_here;
    }
    if (tid == 0) {
        q_starts[a.seqs] = (int)total;
        *a.free_count = free_count - (int)fresh_total;
    }
    __syncthreads();
    // ---- every token's position and slot; rows behind the last token hold -1
    for (int t = tid; t < max_tokens; t += THREADS) {
        int position = -1, slot = -1;
        if (t < total) {
            int lo = 0, hi = a.seqs;  // the sequence whose [start, next start) holds t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (q_starts[mid] <= t)
                    lo = mid;
                else
                    hi = mid;
            }
            position = past_lens[lo] + t - q_starts[lo];
            const int page = a.pages[(long long)lo * a.max_pages + position / a.page_size];
            if (page >= 0 && page < a.num_pages)
                slot = page * a.page_size + position % a.page_size;
            else
                atomicOr(a.status, INF_STATUS_BAD_PAGE);
        }
        positions[t] = position;
        slots[t] = slot;
    }
}

__global__ void __launch_bounds__(THREADS)
device_index_truncate_kernel(IndexArgs a, const int* __restrict__ keep) {
    __shared__ long long s_warp[WARPS];
    inf_pdl_wait();
    inf_pdl_release();
    const int tid = threadIdx.x;
    const int free_count = *a.free_count;
    int bad = free_count < 0 ? INF_STATUS_NO_PAGES : 0;
    long long gone = 0, unused;
    for (int b = tid; b < a.seqs; b += THREADS) {
        const int len = a.lens[b], k = keep[b];
        if (k >= 0) {
            if (k > len || len > (long long)a.max_pages * a.page_size)
                bad |= INF_STATUS_BAD_LEN;
            else
                gone += pages_of(len, a.page_size) - pages_of(k, a.page_size);
        }
    }
    const long long gone_total = block_scan(gone, unused, s_warp);
    if (gone_total + free_count > a.num_pages) bad |= INF_STATUS_NO_PAGES;
    if (__syncthreads_or(bad)) {
        if (bad) atomicOr(a.status, bad);
        return;
    }
    // from the last sequence to the first, each from its last page down
    long long pushed0 = 0;
    for (int r0 = 0; r0 < a.seqs; r0 += THREADS) {
        const int b = a.seqs - 1 - (r0 + tid);
        const int len = b >= 0 ? a.lens[b] : 0, k = b >= 0 ? keep[b] : -1;
        const int have = pages_of(len, a.page_size), hold = k >= 0 ? pages_of(k, a.page_size) : have;
        long long before;
        const long long here = block_scan(have - hold, before, s_warp);
        if (b >= 0 && k >= 0) {
            for (int j = 0; j < have - hold; ++j) {
                int* slot = a.pages + (long long)b * a.max_pages + have - 1 - j;
                a.free_pages[free_count + (int)(pushed0 + before) + j] = *slot;
                *slot = -1;
            }
            a.lens[b] = k;
        }
        pushed0 += here;
    }
    if (tid == 0) *a.free_count = free_count + (int)gone_total;
}

__global__ void device_index_reset_kernel(IndexArgs a) {
    inf_pdl_wait();
    inf_pdl_release();
    const long long stride = (long long)gridDim.x * blockDim.x, i0 = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    for (long long i = i0; i < (long long)a.seqs * a.max_pages; i += stride) a.pages[i] = -1;
    for (long long i = i0; i < a.seqs; i += stride) a.lens[i] = 0;
    for (long long i = i0; i < a.num_pages; i += stride) a.free_pages[i] = a.num_pages - 1 - (int)i;
    if (i0 == 0) *a.free_count = a.num_pages;
}

int index_args(inf_ctx* ctx, const inf_device_index* x, const char* what, IndexArgs* out) {
    if (!x || !x->pages || !x->lens || !x->free_pages || !x->free_count) return inf_fail(ctx, INF_E_ARG, "%s: null pointer", what);
    if (x->num_pages <= 0 || x->page_size <= 0 || x->max_seqs <= 0 || x->max_pages <= 0)
        return inf_fail(ctx, INF_E_CACHE, "%s: num_pages %d, page_size %d, max_seqs %d and max_pages %d must be positive", what,
                        x->num_pages, x->page_size, x->max_seqs, x->max_pages);
    if ((long long)x->num_pages * x->page_size > 0x7fffffffLL || (long long)x->max_pages * x->page_size > 0x7fffffffLL)
        return inf_fail(ctx, INF_E_CACHE, "%s: token slots must be countable in 31 bits", what);
    *out = IndexArgs{x->pages, x->lens, x->free_pages, x->free_count, x->num_pages, x->page_size, x->max_seqs, x->max_pages, ctx->status};
    return INF_OK;
}

}  // namespace

extern "C" int32_t inf_device_index_reset(inf_ctx* ctx, const inf_device_index* index) {
    INF_CHECK_CTX(ctx);
    return inf_entry(ctx, [&]() -> int {
        IndexArgs a;
        const int rc = index_args(ctx, index, "device_index_reset", &a);
        if (rc != INF_OK) return rc;
        const long long most = (long long)a.seqs * a.max_pages > a.num_pages ? (long long)a.seqs * a.max_pages : a.num_pages;
        const long long blocks = (most + 255) / 256;
        INF_CUDA(ctx, inf_launch_pdl(device_index_reset_kernel, dim3((unsigned)(blocks < 4LL * ctx->sm_count ? blocks : 4LL * ctx->sm_count)),
                                     dim3(256), 0, ctx->stream, a));
        return INF_OK;
    });
}

extern "C" int32_t inf_device_index_append(inf_ctx* ctx, const inf_device_index* index, const int32_t* new_tokens,
                                           int32_t max_tokens, int32_t* past_lens, int32_t* q_starts, int32_t* positions,
                                           int32_t* slots) {
    INF_CHECK_CTX(ctx);
    return inf_entry(ctx, [&]() -> int {
        IndexArgs a;
        const int rc = index_args(ctx, index, "device_index_append", &a);
        if (rc != INF_OK) return rc;
        if (!new_tokens || !past_lens || !q_starts || !positions || !slots)
            return inf_fail(ctx, INF_E_ARG, "device_index_append: null pointer");
        if (max_tokens <= 0) return inf_fail(ctx, INF_E_SHAPE, "device_index_append: max_tokens must be positive, got %d", max_tokens);
        INF_CUDA(ctx, inf_launch_pdl(device_index_append_kernel, dim3(1), dim3(THREADS), 0, ctx->stream, a, new_tokens, max_tokens,
                                     past_lens, q_starts, positions, slots));
        return INF_OK;
    });
}

extern "C" int32_t inf_device_index_truncate(inf_ctx* ctx, const inf_device_index* index, const int32_t* keep_lens) {
    INF_CHECK_CTX(ctx);
    return inf_entry(ctx, [&]() -> int {
        IndexArgs a;
        const int rc = index_args(ctx, index, "device_index_truncate", &a);
        if (rc != INF_OK) return rc;
        if (!keep_lens) return inf_fail(ctx, INF_E_ARG, "device_index_truncate: null pointer");
        INF_CUDA(ctx, inf_launch_pdl(device_index_truncate_kernel, dim3(1), dim3(THREADS), 0, ctx->stream, a, keep_lens));
        return INF_OK;
    });
}
