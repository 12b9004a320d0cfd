// Causal attention of a ragged batch over paged K/V: every sequence brings its own number of new tokens (a prompt chunk,
// a few drafts, one decode token, or none), their keys and values already in the pages.
//
// Row t of sequence b stands at p = past_b + t and sees the keys [max(0, p + 1 - window), p]:
//     o = softplus(gate) * sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = scale q . k_j,  m = max_j s_j
// in one pass over the keys with a running maximum and sum.
//
// Work.  The G query heads of a KV head share its keys, so the rows of a KV head are packed: row = token * G + head, a
// STREAM is up to 128 rows (Ts = 128 / G tokens), and an ITEM is (sequence, KV head, up to 2 Ts tokens): two streams that
// read every 128-key tile together.  An item of one stream's tokens (decodes, drafts) has both streams on the same rows,
// tile by tile in turn, and merges them at the end.
//
// One persistent CTA per SM.  The lengths are on the GPU, so the CTAs divide the work themselves: an item costs its keys
// plus a fixed amount, the costs of all items stand in one line (sequence, KV head, tile of tokens), and CTA c takes the
// c-th of equal parts of it.  Sums over a sequence's items have a closed form, so a scan over the batch and a binary
// search find both ends.  A part's ends fall inside items, at tiles of keys; such an item's pieces leave (max, sum, row)
// in scratch, and the CTA that finishes its last piece joins them in the order of the keys: nothing depends on timing.
//
// Twelve warps:
//   warps 0-3, 4-7   softmax and epilogue of stream 0 / 1
//   warp 8           walks the CTA's items, describes each in shared memory for the others, loads the K ring (TMA)
//   warp 9           issues every MMA, in the order  S(0) S(1) | PV(0) S(2) | PV(1) S(3) | ...  over the streams' tiles in turn
//   warp 10          loads the V ring (TMA)
//   warp 11          loads Q
// S = Q K^T is an SS MMA (M128 N128 K16), O += P V a TS MMA: P, packed fp16, lies over its own S in TMEM, 64 keys of it over
// the columns 0-31 and 64 over 64-95, V is read MN-major straight from its [key][dim] tile.  One thread's MMAs run in order,
// so S of a stream's next tile, issued behind PV, may overwrite that P, and its barrier also says that PV has retired: a
// softmax warp waits for one barrier per tile, and while it works on one stream the tensor cores have PV and S of the other.
// TMEM: S 128 columns and O 128 columns per stream.  Shared memory: Q 2 x 32 KB, K 3 x 32 KB, V 2 x 32 KB.
//
// Rows of few items fill few of the 128 lanes, and a warp's exponentials go through one of the four special-function
// units.  Up to 32 rows (decodes, short drafts) are therefore dealt out to the four lane quarters, and each is held by four
// threads (16x256 TMEM shape): 32 exponentials a thread and tile instead of 128 on one warp.  Their MMAs are of M64, whose
// rows are lanes 0-15 of each quarter: a batch of decodes holds the GPU at its power limit, and half the multiplications
// leave the clock 8 % higher (139 -> 133 us).
//
// What bounds it, and what it takes on a B200 (a floor is the keys' bytes at the measured copy bandwidth or the products at the
// measured cuBLAS rate; the first figure from a cool GPU, the second held at its power limit):
//   32 decodes of 1 024-16 384 keys, 48 / 8 heads   125, 131 us   floor 114: memory
//   24 sequences of 6 drafts, 64 / 8 heads           79, 83        60: memory, then the CTAs' start (5 us), unequal SMs, the join
//   46 decodes and two chunks of 1 024, 48 / 8      151, 173       84: the chunks' tiles (softmax and MMAs in turn), joins
//   40 decodes and a chunk of 777, window 512        51, 51        10: five tiles an item, so its start and end; the largest part is
//                                                                  worth 1.5 times the mean
//   a chunk of 4 096 on 8 192 keys, 48 / 8          945, 1 040    626: a stream's tile takes softmax 2 100 + MMAs 1 300 cycles,
//                                                                  and the other stream covers half of that
//   one decode of 100 keys                             9 in a graph: launch, cold code, a chain of five waits
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "ptx.cuh"
#include "ragged_parts.h"

using namespace inf;

namespace {

constexpr int D = 128;
constexpr int BM = 128, BN = RAGGED_TILE;
constexpr int THREADS = 384;
constexpr int KS = 3, VS = 2;          // tiles in the K and V rings
constexpr int SR = 4;                  // rotation of the barriers that free their slots: one is looked at up to three tiles late
constexpr int TILE_BYTES = BN * D * 2;  // also the bytes of a stream's Q
constexpr int BLK_BYTES = BN * 128;    // [128 rows][64 columns] with the 128-byte swizzle
constexpr int RING = 4;                // item descriptions in flight
constexpr int FEW_ROWS = 32;           // rows that are dealt out to the lane quarters, eight each
constexpr int LIGHT_ROWS = 64;         // rows up to which an item's time is that of its keys' way from memory
constexpr float M_INIT = -1.0e30f;
constexpr float RESCALE_THRESHOLD = 8.0f;
constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_O = 256;  // 128 columns per stream each

struct Item {
    int b, kvh, tok0, ntok;        // tokens [tok0, tok0 + ntok) of the step
    int qpos0, kv_total, lowest;   // position of the first token, keys of the sequence, lowest key any row sees
    int kt0, kt1;                  // key tiles of this piece; kt0 == kt1 ends the CTA's work
    int pieces, ordinal, group;    // of an item cut over several CTAs: how many, which one, the CTA of the first
};

struct Found {
    long long at;  // where the sequence begins in the line
    int b, n, past;
};

struct Shared {
    uint64_t q_full[2], q_free[2], k_full[KS], v_full[VS];
    uint64_t s_full[2][SR];   // S of a stream's tile is in TMEM, PV of its tile before has retired
    uint64_t p_full[2][2];    // keys 64-127 / 0-63 of a stream's P are in TMEM
    uint64_t o_ready[2][SR];  // PV of a stream's tile has retired
    uint64_t item_full[RING], item_free[RING];
    uint64_t v_patched[VS];   // dead slots of the V tile in this ring slot have been cleared
    uint64_t join[2];         // shared rows: stream 1's maxima and sums are in ml / its O has been read
    uint64_t drained;         // every MMA has retired
    uint64_t part_bar, flag_bar;  // the CTA's pieces are in scratch / whether they were their items' last
    uint32_t tmem;
    int last_piece[2];
    Item piece[2];                 // the CTA's pieces of cut items
    Item items[RING];
    long long scan[THREADS / 32];
    Found found[2];                // the sequences that hold the part's ends
    int end[4], begin[4];          // (sequence, KV head, tile of tokens, key tile)
    int cut[2][3];                 // pieces, ordinal, group of the first and of the last item
    float ml[BM][2];
};

constexpr int OFF_K = 2 * TILE_BYTES, OFF_V = OFF_K + KS * TILE_BYTES, OFF_SHARED = OFF_V + VS * TILE_BYTES;
constexpr int SMEM_BYTES = OFF_SHARED + (int)sizeof(Shared);
static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");

struct RaggedParams {
    const __half* q;
    const int *pages, *lens, *starts;
    int batch, max_pages, tokens, q_heads, kv_heads, group, page_size, num_pages, window;
    int stream_tokens;              // Ts
    int few_tokens, light_tokens;   // of an item of FEW_ROWS / LIGHT_ROWS rows at most
    int box_rows;       // keys of one TMA box
    float scale_log2;
    const float* gate;
    void* out;
    int out_f16, out_sectors;  // fp16 rows; rows begin at whole 32-byte sectors
    float *part_acc, *part_ml;  // [2 grid][256] rows
    int* counters;              // [grid], zero between launches
    int* status;
};

// log(1 + e^v): log1p, because 1 + e^v keeps nothing but 2^-24 of e^v, which is 1e-3 of it at v = -10.
__device__ __forceinline__ float softplus(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// ---------------------------------------------------------------------------------------------- the line of work
struct Seq {
    int start, n, past;
};

// A sequence's rows and cached keys; n = 0 (and a status bit) where they do not fit what the launch was given.
__device__ __forceinline__ Seq sequence_of(const RaggedParams& p, int b, int& bad) {
    Seq s;
    s.start = p.starts[b];
    s.n = p.starts[b + 1];
    s.past = p.lens[b];
    const long long n = (long long)s.n - s.start;
    s.n = (int)n;
    if (n < 0 || (n > 0 && (s.start < 0 || s.start + n > p.tokens || s.past < 0 || s.past + n > (long long)p.max_pages * p.page_size))) {
        bad = INF_STATUS_BAD_LEN;
        s.n = 0;
    }
    return s;
}

template <typename T>
__device__ __forceinline__ T block_sum_before(T v, T& before, T* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    T base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += s_warp[w];
        total += s_warp[w];
    }
    before = base + inc - v;
    return total;
}

__device__ __forceinline__ RaggedHead head_of(const RaggedParams& p, int n, int past) {
    return RaggedHead(n, past, 2 * p.stream_tokens, p.light_tokens, p.window);
}

// Where CTA c's part of the line begins and ends.  Returns false where it has none.  The threads sum the sequences' costs and
// find the two sequences, then one warp each finds the place inside (read after the caller's barrier): its lanes take the
// cuts that fall into the item, 32 at a time.
__device__ __forceinline__ bool find_part(const RaggedParams& p, Shared& sh) {
    const int tid = threadIdx.x, c = blockIdx.x;
    const int per = (p.batch + THREADS - 1) / THREADS, b0 = min(tid * per, p.batch), b1 = min(b0 + per, p.batch);
    int bad = 0;
    long long mine = 0, before;
    Seq s{0, 0, 0};
#pragma unroll 1
    for (int b = b0; b < b1; ++b) {
        s = sequence_of(p, b, bad);
        mine += p.kv_heads * head_of(p, s.n, s.past).total();
    }
    if (bad && c == 0) atomicOr(p.status, bad);
    if (tid == 0) sh.found[1].b = p.batch;
    const RaggedLine line(block_sum_before(mine, before, sh.scan), (int)gridDim.x);
    if (c >= line.parts) return false;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
        const long long x = line.cut(c + e);
        if (x >= before && x < before + mine) {
            long long at = before;
            int b = b0;
            for (; per > 1; ++b) {
                s = sequence_of(p, b, bad);
                const long long cost = p.kv_heads * head_of(p, s.n, s.past).total();
                if (x < at + cost) break;
                at += cost;
            }
            sh.found[e] = Found{at, b, s.n, s.past};
        }
    }
    __syncthreads();
    if (tid < 64) {
        const int e = tid >> 5, lane = tid & 31;
        const Found f = sh.found[e];
        int* out = e == 0 ? sh.begin : sh.end;
        int inside = 0, first = 0, tile = 0, kvh = 0, item = 0;
        if (f.b < p.batch) {
            const RaggedHead h = head_of(p, f.n, f.past);
            const RaggedPlace place(h, f.at, line.cut(c + e));
            kvh = place.kvh;
            item = place.i;
            const int first_tile = h.first_tile(item), end_tile = h.end_tile(item);
            tile = place.tile_of(h, line, c + e);
            for (int k0 = place.first_cut(line);; k0 += 32) {
                const int t = place.tile_of(h, line, k0 + lane);
                const uint32_t in = __ballot_sync(0xffffffffu, t > first_tile && t < end_tile);
                if (in && inside == 0) first = k0 + __ffs(in) - 1;
                inside += __popc(in);
                if (__any_sync(0xffffffffu, t == end_tile)) break;  // these cuts reach the item's end
            }
        }
        if (lane == 0) {
            out[0] = f.b;
            out[1] = kvh;
            out[2] = item;
            out[3] = tile;
            sh.cut[e][0] = inside + 1;
            sh.cut[e][1] = c - (first - 1);
            sh.cut[e][2] = first - 1;
        }
    }
    return true;
}

// ---------------------------------------------------------------------------------------------- the kernel
// A bounded wait in few instructions, because the code of the twelve warps has to fit the instruction caches: up to 2^21
// tries of at most a microsecond each.
__device__ __forceinline__ bool lone_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 tries;\n\t"
        "mov.u32 tries, 0;\n"
        "again:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "add.u32 tries, tries, 1;\n\t"
        "setp.lt.u32 q, tries, 0x200000;\n\t"
        "@p bra done;\n\t"
        "@q bra again;\n"
        "done:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// of a whole warp, with one answer for all its lanes
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, lone_wait(bar, parity)); }

// of a whole warp without a vote, so that its branches stay uniform: a wait that gave up leaves the ones after it no tries
__device__ __forceinline__ void uniform_wait(uint64_t* bar, uint32_t parity, uint32_t& tries) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 tried;\n\t"
        "mov.u32 tried, 0;\n"
        "again:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "add.u32 tried, tried, 1;\n\t"
        "setp.lt.u32 q, tried, %3;\n\t"
        "@p bra done;\n\t"
        "@q bra again;\n"
        "done:\n\t"
        "selp.u32 %0, %3, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(tries)
        : "memory");
    tries = ok;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t leader;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(leader));
    return leader != 0;
}

// A role's view of the items: the next one's description, copied to registers.
struct ItemReader {
    int count = 0;
    __device__ __forceinline__ bool next(Shared& sh, Item& it) {
        const int slot = count % RING;
        if (!warp_wait(&sh.item_full[slot], (uint32_t)(count / RING) & 1u)) return false;
        it = sh.items[slot];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.item_free[slot]);
        ++count;
        return true;
    }
};

// Both streams on the same rows, tiles in turn.
__device__ __forceinline__ bool shares_rows(const RaggedParams& p, const Item& it) { return it.ntok <= p.stream_tokens; }

// Slots of key tile t behind the sequence's last key that a box brings all the same.
__device__ __forceinline__ int dead_slots(const RaggedParams& p, const Item& it, int t) {
    const int live = it.kv_total - t * BN;
    return live < BN ? (live + p.box_rows - 1) / p.box_rows * p.box_rows - live : 0;
}

// Slots of key tile t below the lowest key any row sees, in the box that brings that key.
__device__ __forceinline__ int dead_below(const RaggedParams& p, const Item& it, int t) {
    const int under = it.lowest - t * BN;
    return under > 0 && under < BN ? under % p.box_rows : 0;
}

// Who reads a tile last: (stream, that stream's count of tiles) of the last three tiles, so that a producer knows which
// barrier says that a ring slot is free.  MMAs of one thread retire in order, so the last reader speaks for both.
struct TileLog {
    int cnt0 = 0, cnt1 = 0, back0 = 0, back1 = 0, back2 = 0;
    __device__ __forceinline__ int back(int tiles) const { return tiles == 2 ? back1 : back2; }
    __device__ __forceinline__ void add(bool shared_rows, int turn) {
        back2 = back1;
        back1 = back0;
        if (shared_rows && turn == 0) {
            back0 = cnt0++ << 1;
        } else {
            back0 = cnt1++ << 1 | 1;
            if (!shared_rows) ++cnt0;
        }
    }
};
static_assert(KS >= 2 && KS <= 3 && VS >= 2 && VS <= 3, "the last three tiles are remembered");

template <int N>
struct RingPlace {
    uint32_t slot = 0, parity = 0;
    __device__ __forceinline__ void step() {
        if (++slot == N) {
            slot = 0;
            parity ^= 1u;
        }
    }
};

// Row coordinates of the TMA boxes of 128 / box_rows tiles at a time, one box per lane, the next group looked up ahead.
struct PageWalk {
    int per_tile, tiles;  // boxes per tile, tiles per group of 32 boxes
    int group = -1, y = 0, ahead = 0;
    __device__ __forceinline__ explicit PageWalk(const RaggedParams& p) : per_tile(BN / p.box_rows), tiles(32 / (BN / p.box_rows)) {}
    __device__ __forceinline__ int lookup(const RaggedParams& p, const Item& it, int g) const {
        const int token = (g * tiles * BN) + (int)(threadIdx.x & 31) * p.box_rows;
        int row = p.num_pages * p.kv_heads * p.page_size;  // outside the tensor: zeros
        // boxes wholly below the lowest visible key may lie in pages that were given back
        if (token < it.kv_total && token / BN < it.kt1 && token + p.box_rows > it.lowest) {
            const int page = p.pages[(long long)it.b * p.max_pages + token / p.page_size];
            if (page >= 0 && page < p.num_pages)
                row = (page * p.kv_heads + it.kvh) * p.page_size + token % p.page_size;
            else
                atomicOr(p.status, INF_STATUS_BAD_PAGE);
        }
        return row;
    }
    __device__ __forceinline__ void begin(const RaggedParams& p, const Item& it) {
        group = it.kt0 / tiles;
        y = lookup(p, it, group);
        ahead = lookup(p, it, group + 1);
    }
    __device__ __forceinline__ void step_to(const RaggedParams& p, const Item& it, int kt) {
        if (kt / tiles == group) return;
        group = kt / tiles;
        y = ahead;
        ahead = lookup(p, it, group + 1);
    }
    // one [128 keys][128 dims] tile as two blocks of 64 columns; every lane issues its boxes
    __device__ __forceinline__ void load(const CUtensorMap* tm, const RaggedParams& p, int kt, uint8_t* dst, uint64_t* bar) const {
        const int lane = threadIdx.x & 31, box = lane >> 1, blk = lane & 1;
        const int row = __shfl_sync(0xffffffffu, y, (kt % tiles) * per_tile + (box < per_tile ? box : 0));
        if (lane == 0) mbar_arrive_expect_tx(bar, TILE_BYTES);
        __syncwarp();
        if (box < per_tile) tma_load_2d(dst + blk * BLK_BYTES + box * p.box_rows * 128, tm, blk * 64, row, bar);
    }
};

__device__ __forceinline__ bool few_rows(const RaggedParams& p, const Item& it) { return it.ntok <= p.few_tokens; }

// ---- one tile of a stream: S in TMEM -> P over it, and the row's running maximum and sum.  The maximum is kept as it comes out
// of S and subtracted before the scale: rounded after the scale it is off by as much as half a step of itself, which the
// exponents of large scores (2^28 and more) do not survive, and the row's top key must get a weight of 1 (one instruction more
// for two keys: the chunk of 4 096 took 912 us before).  A row of O is scaled only when its maximum grew by more than 2^8 in
// weight: until then the weights stay below 2^8.  Each row decides for itself, so that its bits do
// not depend on what else is in the warp.  The weights enter PV as fp16, half a step of 2^-11 each; their sum stays in 32 bits.

// weights of 64 keys of a row, packed, and their sum
__device__ __forceinline__ void exponentials(const uint32_t* x, float scale_log2, float m, uint32_t* packed, uint64_t* sums) {
    const uint64_t scale2 = pack_f32x2(scale_log2, scale_log2), neg_m2 = pack_f32x2(-m, -m);  // one rounding each, relative
#pragma unroll
    for (int i = 0; i < 64; i += 2) {
        float a, b;
        unpack_f32x2(mul_f32x2(add_f32x2(pack_f32x2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), neg_m2), scale2), a, b);
        a = ex2_approx(a);
        b = ex2_approx(b);
        sums[(i >> 1) & 1] = add_f32x2(sums[(i >> 1) & 1], pack_f32x2(a, b));
        packed[i / 2] = pack_half2(a, b);
    }
}
// hides keys of a tile from a row: S is masked where it lies, so that the code below serves every tile
__device__ __forceinline__ void mask_scores(uint32_t col_s, int k0, int qpos, int first_key) {
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
        uint32_t x[32];
        tmem_ld32(col_s + c, x);
        tc_wait_ld32(x);
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (k0 + c + i > qpos || k0 + c + i < first_key) x[i] = 0xff800000u;  // -inf
        tmem_st32(col_s + c, x);
    }
    tc_wait_st();
}
__device__ __forceinline__ float max_of(const uint32_t* x) {
    float mx[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]), __uint_as_float(x[3])};
#pragma unroll
    for (int i = 4; i < 60; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(x[i + e]), __uint_as_float(x[i + 4 + e]));
    return max3(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), fmaxf(__uint_as_float(x[60]), __uint_as_float(x[61])),
                fmaxf(__uint_as_float(x[62]), __uint_as_float(x[63])));
}

// thread = row.  Loops over the halves of the row keep the code short: three warps with different code share a scheduler's
// instruction cache, and the warp that issues the MMAs must not wait for its instructions.  The maximum leaves keys 64-127 in
// registers; their weights come first, and the scores of keys 0-63 are read again behind them.
__device__ __forceinline__ void softmax_tile(Shared& sh, const RaggedParams& p, uint32_t col_s, uint32_t col_o, int st, int k0,
                                             int qpos, int first_key, bool masked, bool valid, bool first, float& m_used, float& l) {
    const int lane = threadIdx.x & 31;
    if (masked) mask_scores(col_s, k0, qpos, first_key);
    float top = -INFINITY;
    uint32_t x[64];
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        tmem_ld32(col_s + h * 64, x);
        tmem_ld32(col_s + h * 64 + 32, x + 32);
        tc_wait_ld64(x);
        top = fmaxf(top, max_of(x));
    }
    const float m_new = fmaxf(m_used, top), growth = (m_new - m_used) * p.scale_log2;  // the scale is positive
    const bool grew = valid && growth > RESCALE_THRESHOLD;
    if (first) {
        m_used = m_new;
    } else if (__any_sync(0xffffffffu, grew)) {
        const float alpha = grew ? ex2_approx(-growth) : 1.0f;
        m_used = grew ? m_new : m_used;
        l *= alpha;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(col_o + c * 32, o);
            tc_wait_ld32(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(col_o + c * 32, o);
        }
        tc_wait_st();
    }
    uint64_t sums[2] = {0, 0};
#pragma unroll 1
    for (int h = 0;; ++h) {  // keys 64-127, which are there, then keys 0-63
        uint32_t packed[32];
        exponentials(x, p.scale_log2, m_used, packed, sums);
        tmem_st32(col_s + (h == 0 ? 64 : 0), packed);  // over columns of S that have been read
        if (h == 0) {
            tmem_ld32(col_s, x);
            tmem_ld32(col_s + 32, x + 32);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[st][h]);  // 64 keys of P are there: their PV may start
        if (h == 1) break;
        tc_wait_ld64(x);
    }
    float a, b;
    unpack_f32x2(add_f32x2(sums[0], sums[1]), a, b);
    l += a + b;
}

// a quad of threads = row: thread q of it has columns 8 k + 2 q + {0, 1}; key0 is the first of them
__device__ __forceinline__ void softmax_tile_few(Shared& sh, const RaggedParams& p, uint32_t col_s, uint32_t col_o, int st, int key0,
                                                 int qpos, int first_key, bool masked, bool valid, bool first, float& m_used, float& l) {
    const int lane = threadIdx.x & 31;
    uint32_t x[64];
    tmem_ld_16x256(col_s, x);
    tc_wait_ld64(x);
    if (masked) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (key0 + 8 * k + e > qpos || key0 + 8 * k + e < first_key) x[4 * k + e] = 0xff800000u;
    }
    float mx[4] = {__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[4]), __uint_as_float(x[5])};
#pragma unroll
    for (int k = 2; k < 16; k += 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(x[4 * (k + (e >> 1)) + (e & 1)]));
    float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m_new = fmaxf(m_used, top), growth = (m_new - m_used) * p.scale_log2;
    if (first) {
        m_used = m_new;
    } else {
        const bool grew = valid && growth > RESCALE_THRESHOLD;
        if (__any_sync(0xffffffffu, grew)) {
            const float alpha = grew ? ex2_approx(-growth) : 1.0f;
            m_used = grew ? m_new : m_used;
            l *= alpha;
            uint32_t o[64];
            tmem_ld_16x256(col_o, o);
            tc_wait_ld64(o);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                o[4 * k] = __float_as_uint(__uint_as_float(o[4 * k]) * alpha);
                o[4 * k + 1] = __float_as_uint(__uint_as_float(o[4 * k + 1]) * alpha);
            }
            tmem_st_16x256(col_o, o);
            tc_wait_st();
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {  // keys 64-127 first
        uint32_t y[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float a = ex2_approx((__uint_as_float(x[4 * (8 - half * 8 + k)]) - m_used) * p.scale_log2);
            const float b = ex2_approx((__uint_as_float(x[4 * (8 - half * 8 + k) + 1]) - m_used) * p.scale_log2);
            sum += a + b;
            y[2 * k] = pack_half2(a, b);
            y[2 * k + 1] = 0u;  // lanes 8-15 hold no row
        }
        tmem_st_16x128_x8(col_s + 64 - half * 64, y);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[st][half]);
    }
    l += sum;
}

// 32 bytes of a thread's own row: one whole sector where the address allows it
__device__ __forceinline__ void store_sector(void* at, const uint32_t* r, bool aligned) {
    if (aligned) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                     "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(at)[0] = make_uint4(r[0], r[1], r[2], r[3]);
        reinterpret_cast<uint4*>(at)[1] = make_uint4(r[4], r[5], r[6], r[7]);
    }
}

// ---- pieces of a cut item: row r of a stream of piece q in the scratch rows
__device__ __forceinline__ long long piece_row(const Item& it, int q, int st, int r) {
    return ((long long)(q > 0 ? 2 * (it.group + q) : 2 * it.group + 1) * 2 + st) * BM + r;
}

// Joins the pieces in the order of the keys; `warps` warps take the rows in turn, eight of them with four pieces each at a
// time: the time is latency, so what counts is how many loads are under way.
__device__ __forceinline__ void join_pieces(const RaggedParams& p, const Item& it, int warp, int warps, int lane) {
    constexpr int ROWS = 8, PIECES = 4;
    const int per = p.stream_tokens * p.group, all = it.ntok * p.group;  // rows of a full stream, of the item
    auto row_in_piece = [&](int rr) { return rr < per ? rr : BM + rr - per; };
#pragma unroll 1
    for (int r0 = warp; r0 < all; r0 += ROWS * warps) {
        // lane = (row, one of four pieces); rows behind the last are read as the last and not stored
        const int mine = min(r0 + lane / PIECES * warps, all - 1);
        const long long out_mine = (long long)(it.tok0 + mine / p.group) * p.q_heads + it.kvh * p.group + mine % p.group;
        auto max_and_sum = [&](int q) {  // of one of this lane's pieces
            return q < it.pieces ? __ldcg(reinterpret_cast<const float2*>(p.part_ml) + piece_row(it, q, 0, 0) + row_in_piece(mine))
                                 : make_float2(M_INIT, 0.f);
        };
        auto merge = [&](float& m, float& sum, float m2, float sum2) {
            const float top = fmaxf(m, m2);
            sum = sum * ex2_approx((m - top) * p.scale_log2) + sum2 * ex2_approx((m2 - top) * p.scale_log2);
            m = top;
        };
        const float gate = p.gate ? p.gate[out_mine] : 0.f;
        float m = M_INIT, gain = 0.f;
        float4 acc[ROWS];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int q = 0; q < it.pieces; q += PIECES) {
            const float2 ml = max_and_sum(q + lane % PIECES);
            float4 v[PIECES][ROWS];
#pragma unroll
            for (int e = 0; e < PIECES; ++e) {
                if (q + e < it.pieces) {
                    const float4* base = reinterpret_cast<const float4*>(p.part_acc + piece_row(it, q + e, 0, 0) * D) + lane;
#pragma unroll
                    for (int u = 0; u < ROWS; ++u) v[e][u] = __ldcg(base + row_in_piece(min(r0 + u * warps, all - 1)) * (D / 4));
                }
            }
            if (q == 0) {  // while the rows of the first pieces are on their way
                m = ml.x;
                float sum = ml.y;
#pragma unroll 1
                for (int r = PIECES + lane % PIECES; r < it.pieces; r += PIECES) {
                    const float2 more = max_and_sum(r);
                    merge(m, sum, more.x, more.y);
                }
#pragma unroll
                for (int o = 1; o < PIECES; o <<= 1) {
                    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), sum2 = __shfl_xor_sync(0xffffffffu, sum, o);
                    merge(m, sum, m2, sum2);
                }
                gain = (p.gate ? softplus(gate) : 1.0f) / sum;
            }
            const float w = ex2_approx((ml.x - m) * p.scale_log2) * gain;  // 0 behind the last piece
#pragma unroll
            for (int e = 0; e < PIECES; ++e) {
                if (q + e < it.pieces) {
#pragma unroll
                    for (int u = 0; u < ROWS; ++u) {
                        const float wu = __shfl_sync(0xffffffffu, w, u * PIECES + e);
                        acc[u].x = fmaf(wu, v[e][u].x, acc[u].x);
                        acc[u].y = fmaf(wu, v[e][u].y, acc[u].y);
                        acc[u].z = fmaf(wu, v[e][u].z, acc[u].z);
                        acc[u].w = fmaf(wu, v[e][u].w, acc[u].w);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const long long row = __shfl_sync(0xffffffffu, out_mine, u * PIECES);
            if (r0 + u * warps >= all) break;
            if (p.out_f16)
                reinterpret_cast<uint2*>((__half*)p.out + row * D)[lane] = make_uint2(pack_half2(acc[u].x, acc[u].y), pack_half2(acc[u].z, acc[u].w));
            else
                reinterpret_cast<float4*>((float*)p.out + row * D)[lane] = acc[u];
        }
    }
}

__global__ void __launch_bounds__(THREADS, 1)
ragged_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_q_light,
                        const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, RaggedParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *sQ = smem, *sK = smem + OFF_K, *sV = smem + OFF_V;
    Shared& sh = *reinterpret_cast<Shared*>(smem + OFF_SHARED);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool smem_ok = (smem_u32(smem) & 1023u) == 0;  // the swizzled tiles need a 1024-byte aligned base
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.q_full[i], 1);
            mbar_init(&sh.q_free[i], 1);
            for (int j = 0; j < SR; ++j) {
                mbar_init(&sh.s_full[i][j], 1);
                mbar_init(&sh.o_ready[i][j], 1);
            }
            for (int j = 0; j < 2; ++j) mbar_init(&sh.p_full[i][j], 4);  // one arrival per warp: tcgen05.wait is warp-wide
            mbar_init(&sh.join[i], 4);
        }
        for (int i = 0; i < KS; ++i) mbar_init(&sh.k_full[i], 1);
        for (int i = 0; i < VS; ++i) {
            mbar_init(&sh.v_full[i], 1);
            mbar_init(&sh.v_patched[i], 1);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(&sh.item_full[i], 1);
            mbar_init(&sh.item_free[i], 11);  // every warp but the one that writes
        }
        mbar_init(&sh.drained, 1);
        mbar_init(&sh.part_bar, 8);
        mbar_init(&sh.flag_bar, 1);
        sh.last_piece[0] = sh.last_piece[1] = 0;
        mbar_fence_init();
    }
    if (warp == 9) {
        tmem_alloc(&sh.tmem, TMEM_COLS);
        tmem_relinquish();
    }
    if (warp == 8 && lane == 0) {
        tma_prefetch_desc(&tm_q);
        tma_prefetch_desc(&tm_q_light);
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
    }
    for (int i = tid; i < TILE_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    inf_pdl_wait();  // queries, appended rows, lengths and page table come from work earlier in the stream
    inf_pdl_release();
    const bool has_work = find_part(p, sh) && smem_ok;
    if (!smem_ok && tid == 0) atomicOr(p.status, INF_STATUS_BAD_SMEM);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = sh.tmem;

    if (!has_work) {
        // nothing to do for this CTA
    } else if (warp >= 8) {
        setmaxnreg_dec<72>();
        ItemReader reader;
        Item it;
        bool alive = true;
        if (warp == 8) {
            // ------------------------------------------------ items and the K ring
            int b = sh.begin[0], kvh = sh.begin[1], i = sh.begin[2], kt = sh.begin[3], bad = 0;
            const int eb = sh.end[0], ekvh = sh.end[1], ei = sh.end[2], ekt = sh.end[3];
            bool first = true;  // still in the item the part begins in
            int items = 0, tiles = 0, base = -32;
            Seq s{0, 0, 0};
            TileLog log;
            PageWalk walk(p);
            while (b < p.batch && b <= eb) {
                // ---- the sequence: metadata of 32 at a time, one per lane
                if (b >= base + 32) {
                    base = b;
                    if (base + lane < p.batch)
                        s = sequence_of(p, base + lane, bad);
                    else
                        s.n = 0;
                }
                const int n = __shfl_sync(0xffffffffu, s.n, b - base), past = __shfl_sync(0xffffffffu, s.past, b - base),
                          start = __shfl_sync(0xffffffffu, s.start, b - base);
                const RaggedHead h = head_of(p, n, past);
                if (i >= h.items) {
                    i = 0;
                    if (n == 0 || ++kvh >= p.kv_heads) {
                        kvh = 0;
                        ++b;
                    }
                    continue;
                }
                // ---- the item, and how much of it is this CTA's
                if (b == eb && (kvh > ekvh || (kvh == ekvh && i > ei))) break;
                const bool last = b == eb && kvh == ekvh && i == ei;
                const int* cut = first ? sh.cut[0] : sh.cut[1];
                it.pieces = first || last ? cut[0] : 1;
                it.ordinal = first || last ? cut[1] : 0;
                it.group = first || last ? cut[2] : 0;
                it.kt0 = first ? kt : h.first_tile(i);
                it.kt1 = last ? ekt : h.end_tile(i);
                it.b = b;
                it.kvh = kvh;
                it.tok0 = start + i * h.T;
                it.ntok = min(h.T, n - i * h.T);
                it.qpos0 = past + i * h.T;
                it.kv_total = past + n;
                it.lowest = h.lo(i);
                first = false;
                ++i;
                if (it.kt0 < it.kt1) {
                    // ---- tell the others
                    const int slot = items % RING;
                    if (items >= RING) alive = warp_wait(&sh.item_free[slot], (uint32_t)(items / RING - 1) & 1u);
                    if (!alive) break;
                    if (lane == 0) sh.items[slot] = it;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.item_full[slot]);
                    ++items;
                    const bool shared_rows = shares_rows(p, it);
                    walk.begin(p, it);
                    for (int t = it.kt0; t < it.kt1; ++t, ++tiles) {
                        walk.step_to(p, it, t);
                        if (tiles >= KS) {
                            const int who = log.back(KS), c = who >> 1;
                            alive = warp_wait(&sh.s_full[who & 1][c % SR], (uint32_t)(c / SR) & 1u);
                            if (!alive) break;
                        }
                        walk.load(&tm_k, p, t, sK + (tiles % KS) * TILE_BYTES, &sh.k_full[tiles % KS]);
                        log.add(shared_rows, (t - it.kt0) & 1);
                    }
                    if (!alive) break;
                }
                if (last) break;
            }
            if (alive) {
                const int slot = items % RING;
                if (items >= RING) alive = warp_wait(&sh.item_free[slot], (uint32_t)(items / RING - 1) & 1u);
                if (alive && lane == 0) {
                    sh.items[slot].kt0 = sh.items[slot].kt1 = 0;
                    mbar_arrive(&sh.item_full[slot]);
                }
            }
            if (!alive)  // copies in flight land before the block ends
                for (int t = max(0, tiles - KS); t < tiles; ++t) warp_wait(&sh.k_full[t % KS], (uint32_t)(t / KS) & 1u);
        } else if (warp == 10) {
            // ------------------------------------------------ the V ring
            int tiles = 0;
            TileLog log;
            PageWalk walk(p);
            while ((alive = reader.next(sh, it)) && it.kt0 < it.kt1) {
                const bool shared_rows = shares_rows(p, it);
                walk.begin(p, it);
                for (int t = it.kt0; t < it.kt1; ++t, ++tiles) {
                    walk.step_to(p, it, t);
                    if (tiles >= VS) {
                        const int who = log.back(VS), c = who >> 1;
                        alive = warp_wait(&sh.o_ready[who & 1][c % SR], (uint32_t)(c / SR) & 1u);
                        if (!alive) break;
                    }
                    walk.load(&tm_v, p, t, sV + (tiles % VS) * TILE_BYTES, &sh.v_full[tiles % VS]);
                    log.add(shared_rows, (t - it.kt0) & 1);
                    // slots that no row sees may hold anything, and 0 * NaN is NaN
                    const int behind = dead_slots(p, it, t), below = dead_below(p, it, t);
                    if (behind | below) {
                        alive = warp_wait(&sh.v_full[tiles % VS], (uint32_t)(tiles / VS) & 1u);
                        auto clear = [&](int row, int rows) {
                            uint8_t* at = sV + (tiles % VS) * TILE_BYTES + row * 128;
                            for (int c = lane; c < rows * 16; c += 32)
                                *reinterpret_cast<uint4*>(at + ((c >> 3) & 1) * BLK_BYTES + (c >> 4) * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                        };
                        clear(it.kv_total - t * BN, behind);
                        clear(it.lowest - t * BN - below, below);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.v_patched[tiles % VS]);
                        if (!alive) break;
                    }
                }
                if (!alive) break;
            }
            if (!alive)
                for (int t = max(0, tiles - VS); t < tiles; ++t) warp_wait(&sh.v_full[t % VS], (uint32_t)(t / VS) & 1u);
        } else if (warp == 11) {
            // ------------------------------------------------ Q: a stream's tile is free when its last S has retired.  An item of
            // few rows finds zeros in the tile's other rows, a light one in the upper 64 (below them its box may bring the next
            // tokens' rows and leave older ones, which nothing reads the products of): the tensor cores work on all 128, and what
            // they draw for multiplying by zero leaves the clock higher when the GPU is at its power limit.
            int uses0 = 0, uses1 = 0;
            int held = 0;  // rows of stream 0's tile that are not zero: of an item of few rows, or -1: light, -2: any
            auto few_row = [](int r) { return (r & 3) * 16 + (r >> 2); };  // row r of few lies there
            auto zero_chunk = [&](int row, int chunk) {
                *reinterpret_cast<uint4*>(sQ + (chunk >> 3) * BLK_BYTES + row * 128 + ((chunk & 7) << 4)) = make_uint4(0, 0, 0, 0);
            };
            while ((alive = reader.next(sh, it)) && it.kt0 < it.kt1) {
                if (uses0 > 0) alive = warp_wait(&sh.q_free[0], (uint32_t)(uses0 - 1) & 1u);
                if (!alive) break;
                ++uses0;
                const int rows = it.ntok * p.group;
                if (few_rows(p, it)) {
                    // as a TMA load with the swizzle would have written them
                    if (held < 0) {
                        for (int c = lane; c < BM * 16; c += 32) zero_chunk(c >> 4, c & 15);
                        __syncwarp();
                    } else {
                        for (int c = rows * 16 + lane; c < held * 16; c += 32) zero_chunk(few_row(c >> 4), c & 15);
                    }
                    held = rows;
                    for (int c0 = 0; c0 < rows * 16; c0 += 4 * 32) {
                        uint4 v[4];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int c = c0 + u * 32 + lane, r = c >> 4;
                            if (r < rows)
                                v[u] = *reinterpret_cast<const uint4*>(
                                    p.q + ((long long)(it.tok0 + r / p.group) * p.q_heads + it.kvh * p.group + r % p.group) * D + (c & 15) * 8);
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int c = c0 + u * 32 + lane, r = c >> 4, row = few_row(r);
                            if (r < rows)
                                *reinterpret_cast<uint4*>(sQ + ((c >> 3) & 1) * BLK_BYTES + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[u];
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.q_full[0]);
                    continue;
                }
                const bool light = it.ntok <= p.light_tokens;
                if (light && held != -1) {
                    for (int c = LIGHT_ROWS * 16 + lane; c < BM * 16; c += 32) zero_chunk(c >> 4, c & 15);
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                held = light ? -1 : -2;
                const uint32_t bytes = (uint32_t)(p.stream_tokens * p.group) * 256u;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.q_full[0], light ? (uint32_t)(p.light_tokens * p.group) * 256u : bytes);
                    for (int blk = 0; blk < 2; ++blk)
                        tma_load_3d(sQ + blk * BLK_BYTES, light ? &tm_q_light : &tm_q, blk * 64, it.kvh * p.group, it.tok0, &sh.q_full[0]);
                }
                if (shares_rows(p, it)) continue;
                if (uses1 > 0) alive = warp_wait(&sh.q_free[1], (uint32_t)(uses1 - 1) & 1u);
                if (!alive) break;
                ++uses1;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.q_full[1], bytes);
                    for (int blk = 0; blk < 2; ++blk)
                        tma_load_3d(sQ + TILE_BYTES + blk * BLK_BYTES, &tm_q, blk * 64, it.kvh * p.group, it.tok0 + p.stream_tokens,
                                    &sh.q_full[1]);
                }
            }
            if (!alive) {  // copies in flight land before the block ends
                if (uses0 > 0) warp_wait(&sh.q_full[0], (uint32_t)(uses0 - 1) & 1u);
                if (uses1 > 0) warp_wait(&sh.q_full[1], (uint32_t)(uses1 - 1) & 1u);
            }
        } else {
            // ------------------------------------------------ every MMA.  The warp runs about four MMAs (256 cycles) ahead of the
            // tensor cores; what it does between two groups must not take longer.  So its branches depend on values that are the
            // same in all lanes, which keeps descriptors and addresses in uniform registers (as a lone thread's, moved there for
            // each MMA, the chunk of 4096 took 5 % longer), and ring positions and parities are stepped, not computed.
            constexpr uint32_t idesc_s128 = umma_idesc_f16(BM, BN, 0, 0), idesc_o128 = umma_idesc_f16(BM, D, 0, 1),
                               idesc_s64 = umma_idesc_f16(BM / 2, BN, 0, 0), idesc_o64 = umma_idesc_f16(BM / 2, D, 0, 1);
            constexpr uint32_t hi = umma_desc_hi(1024, UMMA_SW128);
            const uint32_t q_lo0 = umma_desc_lo(smem_u32(sQ), 16), k_lo0 = umma_desc_lo(smem_u32(sK), 16),
                           v_lo0 = umma_desc_lo(smem_u32(sV), BLK_BYTES);
            RingPlace<KS> k_at;
            RingPlace<VS> v_at;
            RingPlace<SR> s_at[2], o_at[2];  // which barriers the next S and PV of a stream report to
            uint32_t patched = 0, p_parity = 0, q_parity = 0;  // a bit for each V slot, stream, stream
            const uint32_t tb = __shfl_sync(0xffffffffu, tbase, 0);
            uint32_t tries = 0x200000u;  // none once a wait gave up
            while ((alive = reader.next(sh, it)) && it.kt0 < it.kt1) {
                const bool shared_rows = __shfl_sync(0xffffffffu, shares_rows(p, it) ? 1 : 0, 0) != 0;
                const uint32_t few = __shfl_sync(0xffffffffu, few_rows(p, it) ? 1u : 0u, 0);
                const uint32_t idesc_s = few ? idesc_s64 : idesc_s128, idesc_o = few ? idesc_o64 : idesc_o128;
                const int steps = __shfl_sync(0xffffffffu, (it.kt1 - it.kt0) * (shared_rows ? 1 : 2), 0);  // one tile of one stream each, the streams in turn
                // steps whose V tile is cleared first: the one of the item's last key, the one of its lowest
                const int dead_step = __shfl_sync(0xffffffffu, dead_slots(p, it, it.kt1 - 1) ? (shared_rows ? steps - 1 : steps - 2) : -1, 0);
                const int low_step = __shfl_sync(0xffffffffu, dead_below(p, it, it.kt0) ? 0 : -1, 0);
                uint32_t k_lo = 0, v_lo = 0;
                uniform_wait(&sh.q_full[0], q_parity & 1u, tries);
                q_parity ^= 1u;
                if (!shared_rows) {
                    uniform_wait(&sh.q_full[1], q_parity >> 1, tries);
                    q_parity ^= 2u;
                }
                // step w: PV of tile w - 2 of the steps, then S of tile w
                auto scores = [&](int st, uint32_t col_s, bool last) {
                    const uint32_t q_lo = q_lo0 + (shared_rows ? 0u : (uint32_t)st * (TILE_BYTES >> 4));
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) {
                        const uint32_t off = (uint32_t)((kk >> 2) * BLK_BYTES + (kk & 3) * 32) >> 4;
                        umma_ss(col_s, umma_desc_pack(q_lo + off, hi), umma_desc_pack(k_lo + off, hi), idesc_s, kk > 0);
                    }
                    tc_commit(&sh.s_full[st][st ? s_at[1].slot : s_at[0].slot]);
                    if (last) tc_commit(&sh.q_free[shared_rows ? 0 : st]);  // the last S that reads this Q
                };
#pragma unroll 1
                for (int w = 0; w < steps + 2; ++w) {
                    const int st = w & 1;
                    const uint32_t col_s = tb + COL_S + st * BN, col_o = tb + COL_O + st * D;
                    const bool new_tile = shared_rows || st == 0, more = w < steps;
                    const bool last = w + 1 == steps || (!shared_rows && w + 2 == steps);
                    if (w >= 2) {
                        if (new_tile) {
                            uniform_wait(&sh.v_full[v_at.slot], v_at.parity, tries);
                            if (w - 2 == dead_step || w - 2 == low_step) {
                                uniform_wait(&sh.v_patched[v_at.slot], (patched >> v_at.slot) & 1u, tries);
                                patched ^= 1u << v_at.slot;
                            }
                            v_lo = v_lo0 + v_at.slot * (TILE_BYTES >> 4);
                            v_at.step();
                        }
                        // the halves of P arrive separately
                        uniform_wait(&sh.p_full[st][0], (p_parity >> st) & 1u, tries);
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                umma_ts(col_o, col_s + 64 + kk * 8, umma_desc_pack(v_lo + (4 + kk) * (2048 >> 4), hi), idesc_o, kk > 0 || w >= 4);
                        }
                        __syncwarp();
                    }
                    if (more && new_tile) {
                        uniform_wait(&sh.k_full[k_at.slot], k_at.parity, tries);
                        k_lo = k_lo0 + k_at.slot * (TILE_BYTES >> 4);
                        k_at.step();
                    }
                    if (w >= 2) {
                        uniform_wait(&sh.p_full[st][1], (p_parity >> st) & 1u, tries);
                        tc_fence_after();
                        p_parity ^= 1u << st;
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk)
                                umma_ts(col_o, col_s + kk * 8, umma_desc_pack(v_lo + kk * (2048 >> 4), hi), idesc_o, 1u);
                            tc_commit(&sh.o_ready[st][st ? o_at[1].slot : o_at[0].slot]);
                            if (more) scores(st, col_s, last);
                        }
                        __syncwarp();
                        if (st)
                            o_at[1].step();
                        else
                            o_at[0].step();
                    } else if (more) {
                        if (elect_one()) scores(st, col_s, last);
                        __syncwarp();
                    }
                    if (more) {
                        if (st)
                            s_at[1].step();
                        else
                            s_at[0].step();
                    }
                }
                alive = __all_sync(0xffffffffu, tries != 0);
                if (!alive) break;
            }
            if (elect_one()) tc_commit(&sh.drained);  // also after a wait that gave up: TMEM is freed behind the last MMA
            __syncwarp();
            alive = warp_wait(&sh.drained, 0) && alive;
        }
        if (!alive && lane == 0) atomicOr(p.status, INF_STATUS_WAIT_TIMEOUT);
    } else {
        setmaxnreg_inc<216>();
        // ------------------------------------------------ softmax and epilogue
        const int st = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t col_s = tbase + lanes + COL_S + st * BN, col_o = tbase + lanes + COL_O + st * D;
        ItemReader reader;
        Item it;
        int cnt = 0, joins = 0, pieces = 0;  // tiles, items that both streams' rows were joined in, pieces of cut items
        bool ok = true;  // a wait that gave up: the rest runs through without waiting, so that nobody waits for this warp
        while (reader.next(sh, it) ? it.kt0 < it.kt1 : (ok = false)) {
            const bool shared_rows = shares_rows(p, it), few = few_rows(p, it);
            const int n_all = it.kt1 - it.kt0;
            const int first_tile = shared_rows ? it.kt0 + st : it.kt0, step = shared_rows ? 2 : 1;
            const int n = shared_rows ? (n_all + 1 - st) >> 1 : n_all;
            const int tok_in = shared_rows ? 0 : st * p.stream_tokens;          // first token of the stream in the item
            const int rows = min(p.stream_tokens, it.ntok - tok_in) * p.group;  // of the stream
            // this thread's row: its lane's, or with few rows the one it shares with the three other threads of its quad
            const int r = few ? (lane >> 2) * 4 + quarter : quarter * 32 + lane;
            const bool valid = r < rows, busy = few ? quarter < rows : quarter * 32 < rows;
            const int row_tok = r / p.group;
            const int qpos_lo = it.qpos0 + tok_in, qpos_hi = qpos_lo + (rows - 1) / p.group;  // of the stream's rows
            const int qpos = qpos_lo + row_tok, first_key = p.window > 0 ? qpos + 1 - p.window : 0;
            float m_used = valid ? M_INIT : -M_INIT, l = 0.f;  // no row there: its weights are zeros
            for (int j = 0; j < n; ++j, ++cnt) {
                const int k0 = (first_tile + j * step) * BN;
                if (ok) ok = warp_wait(&sh.s_full[st][cnt % SR], (uint32_t)(cnt / SR) & 1u);
                tc_fence_after();
                const bool masked = k0 + BN - 1 > qpos_lo || (p.window > 0 && k0 < qpos_hi + 1 - p.window);
                if (!busy) {  // no row of this warp is used: keep step with the others
                    if (lane < 2) mbar_arrive(&sh.p_full[st][lane]);
                } else if (few) {
                    softmax_tile_few(sh, p, col_s, col_o, st, k0 + 2 * (lane & 3), qpos, first_key, masked, valid, j == 0, m_used, l);
                } else {
                    softmax_tile(sh, p, col_s, col_o, st, k0, qpos, first_key, masked, valid, j == 0, m_used, l);
                }
            }
            if (n > 0) {
                if (ok) ok = warp_wait(&sh.o_ready[st][(cnt - 1) % SR], (uint32_t)((cnt - 1) / SR) & 1u);
                tc_fence_after();
            }
            if (few) {  // each thread of the quad has summed its own columns
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
            }
            // ---- shared rows: stream 0 joins the two; the same lanes hold the same rows, so it reads stream 1's O in place
            const bool two = shared_rows && n_all > 1;
            const bool cut = it.pieces > 1;
            if (two && st == 1) {
                sh.ml[quarter * 32 + lane][0] = m_used;
                sh.ml[quarter * 32 + lane][1] = l;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.join[0]);
                if (ok) ok = warp_wait(&sh.join[1], (uint32_t)joins & 1u);  // before this stream's next PV
            }
            if (st == 0 || !shared_rows) {
                float w0 = 1.f, w1 = 0.f;
                if (two) {
                    if (ok) ok = warp_wait(&sh.join[0], (uint32_t)joins & 1u);
                    tc_fence_after();
                    const float m1 = sh.ml[quarter * 32 + lane][0], m_all = fmaxf(m_used, m1);
                    w0 = ex2_approx((m_used - m_all) * p.scale_log2);
                    w1 = ex2_approx((m1 - m_all) * p.scale_log2);
                    l = l * w0 + sh.ml[quarter * 32 + lane][1] * w1;
                    m_used = m_all;
                }
                if (busy) {
                    const long long out_row =
                        valid ? (long long)(it.tok0 + tok_in + row_tok) * p.q_heads + it.kvh * p.group + (r - row_tok * p.group) : 0;
                    const long long part_row = piece_row(it, it.ordinal, st, r);
                    if (!cut) {
                        float gain = 1.0f / l;
                        if (p.gate && valid) gain *= softplus(p.gate[out_row]);
                        w0 *= gain;
                        w1 *= gain;
                    } else if (valid && (!few || (lane & 3) == 0)) {
                        p.part_ml[part_row * 2] = m_used;
                        p.part_ml[part_row * 2 + 1] = l;
                    }
                    float* out32 = cut ? p.part_acc + part_row * D : (float*)p.out + out_row * D;  // f32 rows
                    __half* out16 = cut || !p.out_f16 ? nullptr : (__half*)p.out + out_row * D;
                    if (few) {
                        uint32_t o[64];
                        float y[32];
                        tmem_ld_16x256(col_o, o);
                        tc_wait_ld64(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            y[2 * k] = __uint_as_float(o[4 * k]) * w0;
                            y[2 * k + 1] = __uint_as_float(o[4 * k + 1]) * w0;
                        }
                        if (two) {
                            tmem_ld_16x256(col_o + D, o);
                            tc_wait_ld64(o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                y[2 * k] = fmaf(__uint_as_float(o[4 * k]), w1, y[2 * k]);
                                y[2 * k + 1] = fmaf(__uint_as_float(o[4 * k + 1]), w1, y[2 * k + 1]);
                            }
                        }
                        if (valid) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const int d = 8 * k + 2 * (lane & 3);
                                if (out16)
                                    *reinterpret_cast<uint32_t*>(out16 + d) = pack_half2(y[2 * k], y[2 * k + 1]);
                                else
                                    *reinterpret_cast<float2*>(out32 + d) = make_float2(y[2 * k], y[2 * k + 1]);
                            }
                        }
                    } else {
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            float y[32];
                            tmem_ld32(col_o + c * 32, o);
                            tc_wait_ld32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) y[i] = __uint_as_float(o[i]) * w0;
                            if (two) {
                                tmem_ld32(col_o + D + c * 32, o);
                                tc_wait_ld32(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) y[i] = fmaf(__uint_as_float(o[i]), w1, y[i]);
                            }
                            if (valid && out16) {
#pragma unroll
                                for (int i = 0; i < 32; i += 16) {
#pragma unroll
                                    for (int e = 0; e < 8; ++e) o[e] = pack_half2(y[i + 2 * e], y[i + 2 * e + 1]);
                                    store_sector(out16 + c * 32 + i, o, p.out_sectors);
                                }
                            } else if (valid) {
#pragma unroll
                                for (int i = 0; i < 32; i += 8) {
#pragma unroll
                                    for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(y[i + e]);
                                    store_sector(out32 + c * 32 + i, o, p.out_sectors || cut);
                                }
                            }
                            __syncwarp();
                        }
                    }
                }
                tc_fence_before();  // the next item's first PV overwrites O
                __syncwarp();
                if (two && lane == 0) mbar_arrive(&sh.join[1]);
            }
            if (two) ++joins;
            if (cut) {
                if (tid == 0) sh.piece[pieces] = it;
                ++pieces;
            }
        }
        // ---- cut items (the part's first and last at most): whoever finishes the last piece joins them in the order of the keys
        if (pieces > 0) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.part_bar);
            if (ok) ok = warp_wait(&sh.part_bar, 0);
            if (tid < pieces) {
                const Item& mine = sh.piece[tid];
                // One thread counts for its CTA: the pieces that a barrier has shown to it before the count, and the others' pieces
                // behind it, which a barrier shows to the warps that join.
                __threadfence();
                const int before = atomicAdd(&p.counters[mine.group], 1);
                __threadfence();
                sh.last_piece[tid] = before + 1 == mine.pieces;
                if (before + 1 == mine.pieces) p.counters[mine.group] = 0;  // for the next launch
            }
            __syncwarp();
            if (tid == 0) mbar_arrive(&sh.flag_bar);
            if (ok) ok = warp_wait(&sh.flag_bar, 0);
            const bool one = sh.last_piece[0], other = pieces == 2 && sh.last_piece[1], both = one && other;
            // half of the warps each where there are two; none behind a wait that gave up, whose items may never have been written
            if (ok && (one || other))
                join_pieces(p, sh.piece[both ? warp >> 2 : (one ? 0 : 1)], both ? warp & 3 : warp, both ? 4 : 8, lane);
        }
        if (!ok && lane == 0) atomicOr(p.status, INF_STATUS_WAIT_TIMEOUT);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tbase, TMEM_COLS);
}

// Scratch for the pieces of cut items (a CTA has at most two) and their counters, made by the context's first call.
int ragged_scratch(inf_ctx* ctx, int grid, float** acc, float** ml, int** counters) {
    const size_t rows = (size_t)grid * 2 * 2 * BM, bytes = rows * (D + 2) * sizeof(float) + (size_t)grid * sizeof(int);
    if (!ctx->ragged_scratch) {
        void* fresh = nullptr;
        INF_CUDA(ctx, cudaMalloc(&fresh, bytes));
        cudaError_t e = cudaMemsetAsync(fresh, 0, bytes, ctx->stream);
        if (e == cudaSuccess) e = cudaStreamSynchronize(ctx->stream);  // the next call may be on another stream
        if (e != cudaSuccess) {
            cudaFree(fresh);
            return inf_fail(ctx, INF_E_BACKEND, "gqa_attention_ragged: clearing the scratch failed: %s", cudaGetErrorString(e));
        }
        ctx->ragged_scratch = fresh;
        ctx->ragged_counters = (int*)((float*)fresh + rows * (D + 2));
    }
    *acc = (float*)ctx->ragged_scratch;
    *ml = *acc + rows * D;
    *counters = ctx->ragged_counters;
    return INF_OK;
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
        if ((long long)table->max_pages * pool->page_size > (1LL << 29))
            return inf_fail(ctx, INF_E_CACHE, "%s: a page-table row must not hold more than 2^29 tokens", what);
        if (tokens < 0) return inf_fail(ctx, INF_E_SHAPE, "%s: tokens must not be negative", what);
        if (q_heads <= 0 || q_heads % pool->kv_heads != 0)
            return inf_fail(ctx, INF_E_SHAPE, "%s: q_heads %d must be a positive multiple of kv_heads %d", what, q_heads, pool->kv_heads);
        if (q_heads / pool->kv_heads > 128) return INF_UNSUPPORTED;
        if (sliding_window < 0) return inf_fail(ctx, INF_E_CONFIG, "%s: sliding_window must be >= 0", what);
        if (!(scale <= 1e15f)) return inf_fail(ctx, INF_E_CONFIG, "%s: scale must be finite and at most 1e15", what);
        if (out_dtype != INF_DTYPE_F32 && out_dtype != INF_DTYPE_F16)
            return inf_fail(ctx, INF_E_DTYPE, "%s: output dtype must be f32 or f16", what);
        int rc = inf_validate_table(ctx, table, pool->num_pages, pool->page_size, 0, what, sliding_window, 0);
        if (rc != INF_OK) return rc;
        RaggedParams p{};
        const int grid = ctx->sm_count;
        rc = ragged_scratch(ctx, grid, &p.part_acc, &p.part_ml, &p.counters);  // also of a call without tokens, which may be the first
        if (rc != INF_OK) return rc;
        if (tokens == 0) return INF_OK;
        if (!q_f16 || !q_starts || !out) return inf_fail(ctx, INF_E_ARG, "%s: null pointer", what);
        if (((uintptr_t)q_f16 | (uintptr_t)out | (uintptr_t)pool->k | (uintptr_t)pool->v) & 15u)
            return inf_fail(ctx, INF_E_ARG, "%s: tensors must be 16-byte aligned", what);
        const int group = q_heads / pool->kv_heads;
        p.q = (const __half*)q_f16;
        p.pages = table->pages;
        p.lens = table->lens;
        p.starts = q_starts;
        p.batch = table->batch;
        p.max_pages = table->max_pages;
        p.tokens = tokens;
        p.q_heads = q_heads;
        p.kv_heads = pool->kv_heads;
        p.group = group;
        p.page_size = pool->page_size;
        p.num_pages = pool->num_pages;
        p.window = sliding_window < table->max_pages * pool->page_size ? sliding_window : 0;  // a window no sequence can fill
        p.stream_tokens = BM / group;
        p.few_tokens = FEW_ROWS / group;
        p.light_tokens = LIGHT_ROWS / group;
        p.box_rows = 16;  // the widest box of whole pages' rows: a page holds a multiple of 16
        while (p.box_rows < BN && pool->page_size % (2 * p.box_rows) == 0) p.box_rows *= 2;
        p.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf((float)D)) * 1.4426950408889634f;
        p.gate = gate;
        p.out = out;
        p.out_f16 = out_dtype == INF_DTYPE_F16;
        p.out_sectors = ((uintptr_t)out & 31u) == 0;
        p.status = ctx->status;
        CUtensorMap tq, tq_light, tk, tv;
        {
            const uint64_t dims[3] = {D, (uint64_t)q_heads, (uint64_t)tokens}, strides[2] = {D * 2, (uint64_t)q_heads * D * 2};
            const uint32_t box[3] = {64, (uint32_t)group, (uint32_t)p.stream_tokens};
            rc = inf_make_tmap(ctx, q_f16, 3, dims, strides, box, &tq);
            if (rc != INF_OK) return rc;
            const uint32_t light_box[3] = {64, (uint32_t)group, (uint32_t)(p.light_tokens > 0 ? p.light_tokens : 1)};
            rc = inf_make_tmap(ctx, q_f16, 3, dims, strides, light_box, &tq_light);
            if (rc != INF_OK) return rc;
        }
        {
            const uint64_t dims[2] = {D, (uint64_t)pool->num_pages * pool->kv_heads * pool->page_size}, strides[1] = {D * 2};
            const uint32_t box[2] = {64, (uint32_t)p.box_rows};
            rc = inf_make_tmap(ctx, pool->k, 2, dims, strides, box, &tk);
            if (rc == INF_OK) rc = inf_make_tmap(ctx, pool->v, 2, dims, strides, box, &tv);
            if (rc != INF_OK) return rc;
        }
        constexpr uint32_t attr_bit = 1u << 30;
        if (!(ctx->func_attr_done & attr_bit)) {
            INF_CUDA(ctx, cudaFuncSetAttribute(ragged_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
            ctx->func_attr_done |= attr_bit;
        }
        {
            inf_prof_scope prof(ctx, "ragged_attention_kernel");
            INF_CUDA(ctx, inf_launch_pdl(ragged_attention_kernel, dim3((unsigned)grid), dim3(THREADS), (size_t)SMEM_BYTES, ctx->stream, tq, tq_light, tk, tv, p));
        }
        return INF_OK;
    });
}
