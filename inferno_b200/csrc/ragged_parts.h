// How the CTAs of the ragged attention divide its work: the arithmetic of the line of items (see ragged_attention.cu),
// free of CUDA so that a host program can check every part of it.
#pragma once

#ifdef __CUDACC__
#define RAGGED_FN __host__ __device__ __forceinline__
#else
#define RAGGED_FN inline
#endif

constexpr int RAGGED_TILE = 128;  // keys of a tile
// Costs, in halves of a key of a light item.  A key of an item of two streams costs two and a half times as much (with twice:
// two chunks of 1 024 among 46 decodes 158 us instead of 151, a window of 512 50 instead of 51.5), of one stream of many rows one
// and a half times (items of 33 to 64 rows count as light: 24 sequences' drafts 95 us as heavy ones, 82 as light); an item
// costs some keys besides (256 light ones; with 192 or 384 the window takes 54 us).  A CTA's part is worth a tile of two
// streams at least, which keeps two cuts of one item from falling on the same tile, and no more, so that short decodes are
// parts of their own (with three light tiles a decode of 100 keys and 8 heads was seven parts: 11.6 us instead of 9.3).  Cuts
// near an end of an item of two streams move to it (RAGGED_SNAP; with one tile instead of two the window's items of five
// tiles fall apart: 68 us).
constexpr int RAGGED_ITEM_COST = 512;
constexpr int RAGGED_MIN_PART = 5 * (RAGGED_TILE + 1);  // one key more: cuts are rounded
constexpr int RAGGED_SNAP = 2;

// The items of T tokens of one KV head of a sequence: n new tokens behind `past` cached ones, past + n at most 2^29.  An item
// of more than T / 2 tokens has two streams, one of up to `light` tokens is light.
struct RaggedHead {
    enum { PAIR = 5 };
    int n, past, T, light, window, items;
    RAGGED_FN RaggedHead(int n_, int past_, int T_, int light_, int window_)
        : n(n_), past(past_), T(T_), light(light_), window(window_), items((int)((unsigned)(n_ + T_ - 1) / (unsigned)T_)) {}
    RAGGED_FN static int least(int a, int b) { return a < b ? a : b; }
    RAGGED_FN static int most(int a, int b) { return a > b ? a : b; }
    // keys [lo, hi) that some row of item i sees
    RAGGED_FN int lo(int i) const { return window > 0 ? most(0, past + i * T + 1 - window) : 0; }
    RAGGED_FN int hi(int i) const { return past + least((i + 1) * T, n); }
    RAGGED_FN int first_tile(int i) const { return lo(i) / RAGGED_TILE; }
    RAGGED_FN int end_tile(int i) const { return (hi(i) + RAGGED_TILE - 1) / RAGGED_TILE; }
    RAGGED_FN int weight(int i) const {
        const int tokens = n - i * T;
        return tokens > T / 2 ? PAIR : (tokens > light ? 3 : 2);
    }
    RAGGED_FN long long cost(int i) const { return RAGGED_ITEM_COST + (long long)weight(i) * (hi(i) - lo(i)); }
    // cost of the items before item i (all of T tokens): past + (i + 1) T keys each, or T + window - 1 where the window bites
    RAGGED_FN long long before(int i) const {
        int m = i;  // items that the window does not reach
        if (window > 0) m = least(m, (int)((unsigned)most(0, T + window - 1 - past) / (unsigned)T));
        const long long keys = (long long)m * past + (long long)T * (((long long)m * (m + 1)) >> 1) + (long long)(i - m) * (T + window - 1);
        return (long long)i * RAGGED_ITEM_COST + PAIR * keys;
    }
    RAGGED_FN long long total() const { return items > 0 ? before(items - 1) + cost(items - 1) : 0; }
    RAGGED_FN int item_at(long long y) const {  // largest i with before(i) <= y
        int a = 0, z = items;
        while (z - a > 1) {
            const int mid = (a + z) >> 1;
            if (before(mid) <= y)
                a = mid;
            else
                z = mid;
        }
        return a;
    }
    // The key tile at which a cut z into the cost of item i falls.  A cut within RAGGED_SNAP tiles of an end of an item of two
    // streams goes there: the pieces of up to 256 rows cost more than so many tiles.
    RAGGED_FN int tile_at(int i, long long z) const {
        const int first = first_tile(i), end = end_tile(i), w = weight(i), snap = w == PAIR ? RAGGED_SNAP : 0;
        if (z <= RAGGED_ITEM_COST) return first;
        const unsigned past_fixed = (unsigned)(z - RAGGED_ITEM_COST);  // below 5 * 2^29
        const int tile = (int)(((unsigned)lo(i) + past_fixed / (unsigned)w + RAGGED_TILE / 2) / RAGGED_TILE);
        if (tile <= first + snap) return first;
        return tile >= end - snap ? end : tile;
    }
};

// The line of all items and its equal parts.  A cut is one 64-bit product: every CTA finds the same ones.
struct RaggedLine {
    long long total;
    int parts;
    double step;
    RAGGED_FN RaggedLine(long long total_, int grid) : total(total_) {
        const double most = (double)total_ * (1.0 / RAGGED_MIN_PART);
        parts = total_ == 0 ? 0 : (most < 1.0 ? 1 : (most < grid ? (int)most : grid));
        step = parts == 0 ? 1.0 : (double)total_ / parts;
    }
    RAGGED_FN long long cut(int c) const { return c >= parts ? total : (long long)(c * step); }
};

// Position x of the line, in a sequence that begins at `at`: which of its KV heads, which item, where that item stands.
struct RaggedPlace {
    int kvh, i;
    long long start, end;
    RAGGED_FN RaggedPlace(const RaggedHead& h, long long at, long long x) {
        const long long head_cost = h.total();
        kvh = (int)((double)(x - at) / (double)head_cost);  // at most one off
        long long in_head = x - at - kvh * head_cost;
        if (in_head < 0) {
            --kvh;
            in_head += head_cost;
        } else if (in_head >= head_cost) {
            ++kvh;
            in_head -= head_cost;
        }
        i = h.item_at(in_head);
        start = x - in_head + h.before(i);
        end = start + h.cost(i);
    }
    // the first cut at or behind the item's start
    RAGGED_FN int first_cut(const RaggedLine& line) const {
        int c = (int)((double)start / line.step);
        if (c > 0 && line.cut(c - 1) >= start) --c;
        while (line.cut(c) < start) ++c;
        return c;
    }
    // the key tile of cut c; cuts behind the item's end give its last
    RAGGED_FN int tile_of(const RaggedHead& h, const RaggedLine& line, int c) const {
        const long long x = line.cut(c);
        return x < end ? h.tile_at(i, x - start) : h.end_tile(i);
    }
};
