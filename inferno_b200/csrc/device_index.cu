// Page bookkeeping on the GPU: the device twin of paged_index.cu, for batches whose request lengths live on the GPU.
//
// With past_b tokens cached and n_b new ones, P tokens per page, sequence b needs
//     need_b = ceil((past_b + n_b) / P) - ceil(past_b / P)
// pages; the free list is a stack, and page j of sequence b's is the (sum_{b' < b} need_b' + j)-th from its top, which
// is the page inf_paged_index_append called for one sequence after the other would hand out.  Dropping tokens pushes
// pages in the reverse order (the last sequence's last page first), so an append followed by a truncate to the old
// lengths restores the free list exactly.  Both are prefix sums over the batch; a few KB move, so what counts is the
// length of the chain of dependent loads.
//
// A cluster of up to sixteen CTAs shares a call.  Each takes the prefix sums over the whole batch into its own shared
// memory, which is cheaper than waiting for another's, and then its share of the tokens and of the pages:
// a search of the prefix sums gives the sequence, and a fresh page is read from the free list itself.  Whether a page id is
// none of the pool's is known behind those reads, to the CTA that met it; the CTAs tell each other, and the cluster's barrier
// stands between the last read and the first write of the index, so that a refused call leaves all of it as it was.
// An append and a truncate in a graph take 9.1 us for 32 decodes, 11.0 for 300 sequences of up to 9 new tokens, and 18.2
// for 1000 of up to 127 (65 000 rows), of which the two launches are about 5.  Without the check of the page ids, whose
// barrier and second search stand in the chain, it was 8.2, 9.4 and 15.9 (with eight CTAs 19.1 for the last, with one 94).
#include "common.cuh"

namespace {

constexpr int THREADS = 1024;
constexpr int WARPS = THREADS / 32;
constexpr int MOST_CTAS = 16;  // of a cluster; more than eight are not possible on every GPU
constexpr int MOST_SEQS = 16384;  // three words of shared memory each

struct IndexArgs {
    int* pages;
    int* lens;
    int* free_pages;
    int* free_count;
    int num_pages, page_size, seqs, max_pages;
    int* status;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int cluster_rank() {
    int r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Whether `mine` holds for a thread of any of the cluster's CTAs (one cluster is the grid).  All threads call it, after a
// cluster_arrive() of their own; everything they read before it has been read when it returns.
__device__ __forceinline__ bool any_of_cluster(bool mine, int* s_flags) {
    const bool here = __syncthreads_or(mine);
    cluster_wait();  // the others run: their shared memory may be written
    const int ctas = (int)gridDim.x;
    if ((int)threadIdx.x < ctas) {
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                     : "=r"(there)
                     : "r"((uint32_t)__cvta_generic_to_shared(s_flags + cluster_rank())), "r"((int)threadIdx.x));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(here ? 1 : 0) : "memory");
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    bool any = false;
    for (int c = 0; c < ctas; ++c) any |= s_flags[c] != 0;
    return any;
}

// Replaces x[0 .. n) by the sums of the values before them and writes the whole sum to x[n]; y likewise if given.  The
// sums themselves (returned) are taken in 64 bits.  A thread takes ceil(n / THREADS) neighbours.
struct Sums {
    long long x, y;
};
__device__ __forceinline__ Sums prefix_sums(int* x, int* y, int n, Sums* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int each = (n + THREADS - 1) / THREADS, from = min((int)threadIdx.x * each, n), to = min(from + each, n);
    Sums mine{0, 0};
    for (int i = from; i < to; ++i) {
        mine.x += x[i];
        if (y) mine.y += y[i];
    }
    Sums inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ux = __shfl_up_sync(0xffffffffu, inc.x, o);
        if (lane >= o) inc.x += ux;
        if (y) {
            const long long uy = __shfl_up_sync(0xffffffffu, inc.y, o);
            if (lane >= o) inc.y += uy;
        }
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    Sums base{0, 0}, total{0, 0};
    const int used = (n + 32 * each - 1) / (32 * each);  // warps that hold values
    for (int w = 0; w < used; ++w) {
        const Sums v = s_warp[w];
        if (w < warp) base.x += v.x, base.y += v.y;
        total.x += v.x, total.y += v.y;
    }
    Sums run{base.x + inc.x - mine.x, base.y + inc.y - mine.y};
    for (int i = from; i < to; ++i) {
        const int vx = x[i];
        x[i] = (int)run.x;
        run.x += vx;
        if (y) {
            const int vy = y[i];
            y[i] = (int)run.y;
            run.y += vy;
        }
    }
    if (threadIdx.x == 0) {
        x[n] = (int)total.x;
        if (y) y[n] = (int)total.y;
    }
    __syncthreads();
    return total;
}

// The last i of [0, n) with sums[i] <= v, for sums[0] <= v < sums[n]: its own value is not zero.
__device__ __forceinline__ int holder_of(const int* sums, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= v)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(long long tokens, int page_size) { return (int)((tokens + page_size - 1) / page_size); }

// A thread takes EACH neighbouring tokens at a time: one while the cluster has a thread for every token, four (one search,
// 16-byte stores) when it has not.
template <int EACH>
__global__ void __launch_bounds__(THREADS)
device_index_append_kernel(IndexArgs a, const int* __restrict__ new_tokens, int max_tokens, int* __restrict__ past_lens,
                           int* __restrict__ q_starts, int* __restrict__ positions, int* __restrict__ slots) {
    __shared__ Sums s_warp[WARPS];
    __shared__ int s_flags[MOST_CTAS];
    extern __shared__ int s_seqs[];
    int *s_past = s_seqs, *s_start = s_past + a.seqs, *s_fresh = s_start + a.seqs + 1;
    cluster_arrive();
    inf_pdl_wait();
    inf_pdl_release();
    const int tid = threadIdx.x, rank = cluster_rank(), i0 = rank * THREADS + tid, stride = (int)gridDim.x * THREADS;
    const long long capacity = (long long)a.max_pages * a.page_size;
    const int free_count = *a.free_count;
    // ---- a step that does not fit is refused as a whole, before anything of the index changes
    int bad = free_count < 0 || free_count > a.num_pages ? INF_STATUS_NO_PAGES : 0;
    for (int b = tid; b < a.seqs; b += THREADS) {
        const int past = a.lens[b], n = new_tokens[b];
        const bool fits = past >= 0 && n >= 0 && (long long)past + n <= capacity;
        if (!fits) bad |= INF_STATUS_BAD_LEN;
        s_past[b] = past;
        s_start[b] = fits ? n : 0;
        s_fresh[b] = fits ? pages_of((long long)past + n, a.page_size) - pages_of(past, a.page_size) : 0;
    }
    const bool any_bad = __syncthreads_or(bad);
    const Sums total = prefix_sums(s_start, s_fresh, a.seqs, s_warp);
    if (total.x > max_tokens) bad |= INF_STATUS_BAD_LEN;
    if (total.y > free_count) bad |= INF_STATUS_NO_PAGES;
    auto describe_no_tokens = [&] {
        for (int b = i0; b < a.seqs; b += stride) past_lens[b] = s_past[b];
        for (int b = i0; b <= a.seqs; b += stride) q_starts[b] = 0;
        for (long long t = i0; t < max_tokens; t += stride) positions[t] = slots[t] = -1;
    };
    if (any_bad || total.x > max_tokens || total.y > free_count) {
        if (bad && rank == 0) atomicOr(a.status, bad);
        describe_no_tokens();
        cluster_wait();
        return;
    }
    // ---- every token's position and slot; rows behind the last token hold -1.  Every page that the step fills or takes has
    // a token, so this meets all of their ids.
    bool lost = false;
    const bool aligned = EACH == 4 && (((uintptr_t)positions | (uintptr_t)slots) & 15u) == 0;
    for (long long t0 = (long long)EACH * i0; t0 < max_tokens; t0 += (long long)EACH * stride) {
        int position[EACH], slot[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) position[j] = slot[j] = -1;
        if (t0 < total.x) {
            int b = holder_of(s_start, a.seqs, (int)t0), seen = -1, page = 0;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                if (t0 + j >= total.x) break;
                if (EACH > 1)
                    while (t0 + j >= s_start[b + 1]) ++b, seen = -1;
                const int past = s_past[b], at_token = past + (int)(t0 + j) - s_start[b], at = at_token / a.page_size;
                if (at != seen) {
                    const int fresh = at - pages_of(past, a.page_size);
                    page = fresh >= 0 ? a.free_pages[free_count - 1 - s_fresh[b] - fresh] : a.pages[(long long)b * a.max_pages + at];
                    seen = at;
                }
                const bool there = page >= 0 && page < a.num_pages;
                lost |= !there;
                position[j] = at_token;
                slot[j] = there ? page * a.page_size + at_token - at * a.page_size : -1;
            }
        }
        if (aligned && t0 + EACH <= max_tokens) {
            *reinterpret_cast<int4*>(positions + t0) = make_int4(position[0], position[1 % EACH], position[2 % EACH], position[3 % EACH]);
            *reinterpret_cast<int4*>(slots + t0) = make_int4(slot[0], slot[1 % EACH], slot[2 % EACH], slot[3 % EACH]);
        } else {
#pragma unroll
            for (int j = 0; j < EACH; ++j)
                if (t0 + j < max_tokens) positions[t0 + j] = position[j], slots[t0 + j] = slot[j];
        }
    }
    if (any_of_cluster(lost, s_flags)) {  // (the barrier inside also orders the two stores to a row of the outputs)
        if (i0 == 0) atomicOr(a.status, INF_STATUS_BAD_PAGE);
        describe_no_tokens();
        return;
    }
    // ---- the fresh pages, and the batch's lengths and starts
    for (int f = i0; f < (int)total.y; f += stride) {
        const int b = holder_of(s_fresh, a.seqs, f);
        a.pages[(long long)b * a.max_pages + pages_of(s_past[b], a.page_size) + f - s_fresh[b]] = a.free_pages[free_count - 1 - f];
    }
    for (int b = i0; b <= a.seqs; b += stride) {
        q_starts[b] = s_start[b];
        if (b < a.seqs) {
            past_lens[b] = s_past[b];
            a.lens[b] = s_past[b] + s_start[b + 1] - s_start[b];
        }
    }
    if (i0 == 0) *a.free_count = free_count - (int)total.y;
}

__global__ void __launch_bounds__(THREADS)
device_index_truncate_kernel(IndexArgs a, const int* __restrict__ keep) {
    __shared__ Sums s_warp[WARPS];
    __shared__ int s_flags[MOST_CTAS];
    extern __shared__ int s_seqs[];
    int *s_have = s_seqs, *s_hold = s_have + a.seqs, *s_gone = s_hold + a.seqs;  // from the last sequence to the first
    cluster_arrive();
    inf_pdl_wait();
    inf_pdl_release();
    const int tid = threadIdx.x, rank = cluster_rank(), i0 = rank * THREADS + tid, stride = (int)gridDim.x * THREADS;
    const int free_count = *a.free_count;
    int bad = free_count < 0 ? INF_STATUS_NO_PAGES : 0;
    for (int r = tid; r < a.seqs; r += THREADS) {
        const int b = a.seqs - 1 - r, len = a.lens[b], k = keep[b];
        const bool fits = k <= len && len <= (long long)a.max_pages * a.page_size;
        if (k >= 0 && !fits) bad |= INF_STATUS_BAD_LEN;
        s_hold[r] = k;
        s_have[r] = pages_of(len, a.page_size);
        s_gone[r] = k >= 0 && fits ? s_have[r] - pages_of(k, a.page_size) : 0;
    }
    const bool any_bad = __syncthreads_or(bad);
    const Sums gone = prefix_sums(s_gone, nullptr, a.seqs, s_warp);
    const bool overfull = gone.x + free_count > a.num_pages;
    if (any_bad || overfull) {
        bad |= overfull ? INF_STATUS_NO_PAGES : 0;
        if (bad && rank == 0) atomicOr(a.status, bad);
        cluster_wait();
        return;
    }
    auto slot_of = [&](int g) {  // where the g-th page to be pushed stands
        const int r = holder_of(s_gone, a.seqs, g);
        return a.pages + (long long)(a.seqs - 1 - r) * a.max_pages + s_have[r] - 1 - (g - s_gone[r]);
    };
    bool lost = false;
    for (int g = i0; g < (int)gone.x; g += stride) {
        const int page = *slot_of(g);
        lost |= page < 0 || page >= a.num_pages;
    }
    if (any_of_cluster(lost, s_flags)) {
        if (i0 == 0) atomicOr(a.status, INF_STATUS_BAD_PAGE);
        return;
    }
    for (int g = i0; g < (int)gone.x; g += stride) {
        int* slot = slot_of(g);
        a.free_pages[free_count + g] = *slot;
        *slot = -1;
    }
    for (int r = i0; r < a.seqs; r += stride)
        if (s_hold[r] >= 0) a.lens[a.seqs - 1 - r] = s_hold[r];
    if (i0 == 0) *a.free_count = free_count + (int)gone.x;
}

// The CTAs that a cluster of these kernels may have on the context's GPU: sixteen where they fit, else the portable eight.
int most_ctas(inf_ctx* ctx) {
    if (ctx->index_ctas) return ctx->index_ctas;
    const void* kernels[] = {(const void*)device_index_append_kernel<1>, (const void*)device_index_append_kernel<4>,
                             (const void*)device_index_truncate_kernel};
    int fits = MOST_CTAS;
    for (const void* kernel : kernels) {
        const int smem = (3 * MOST_SEQS + 2) * (int)sizeof(int);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(MOST_CTAS);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {MOST_CTAS, 1, 1};
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1)
            fits = 8;
    }
    cudaGetLastError();  // what did not fit is no error
    return ctx->index_ctas = fits;
}

// One cluster for `work` threads' work.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(inf_ctx* ctx, void (*kernel)(KArgs...), long long work, int seqs, Args... args) {
    const int most = most_ctas(ctx);
    int ctas = 1;
    while (ctas < most && (long long)ctas * THREADS < work) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (3 * (size_t)seqs + 2) * sizeof(int);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)ctas, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
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
    if (x->max_seqs > MOST_SEQS) return inf_fail(ctx, INF_E_CACHE, "%s: at most %d sequences, got %d", what, MOST_SEQS, x->max_seqs);
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
        const bool few = max_tokens <= most_ctas(ctx) * THREADS;
        INF_CUDA(ctx, launch_cluster(ctx, few ? device_index_append_kernel<1> : device_index_append_kernel<4>, max_tokens, a.seqs, a, new_tokens, max_tokens,
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
        // how many pages go is known on the GPU alone: four a sequence are expected
        INF_CUDA(ctx, launch_cluster(ctx, device_index_truncate_kernel, 4LL * a.seqs, a.seqs, a, keep_lens));
        return INF_OK;
    });
}
