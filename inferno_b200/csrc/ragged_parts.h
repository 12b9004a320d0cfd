// How the CTAs of the ragged attention divide its work: the arithmetic of the line of items (see ragged_attention.cu),
// free of CUDA so that a host program can check every part of it.
#pragma once

#ifdef __CUDACC__
#define RAGGED_FN __host__ __device__ __forceinline__
#else
#define RAGGED_FN inline
#endif

constexpr int RAGGED_TILE = 128;  // keys of a tile
// Costs in keys: what an item costs besides its keys, and the least part of the work that a CTA is given.  Parts of three
// tiles or more also keep two cuts of one item from falling on the same tile.
constexpr int RAGGED_ITEM_COST = 128;
constexpr int RAGGED_MIN_PART = 3 * RAGGED_TILE;
constexpr int RAGGED_SNAP = 2;

// The items of T tokens of one KV head of a sequence: n new tokens behind `past` cached ones.
struct RaggedHead {
    int n, past, T, window, items;
    RAGGED_FN RaggedHead(int n_, int past_, int T_, int window_) : n(n_), past(past_), T(T_), window(window_), items((n_ + T_ - 1) / T_) {}
    RAGGED_FN static long long least(long long a, long long b) { return a < b ? a : b; }
    RAGGED_FN static long long most(long long a, long long b) { return a > b ? a : b; }
    // keys [lo, hi) that some row of item i sees
    RAGGED_FN int lo(int i) const { return window > 0 ? (int)most(0, past + i * T + 1 - window) : 0; }
    RAGGED_FN int hi(int i) const { return past + (int)least((i + 1) * T, n); }
    RAGGED_FN int first_tile(int i) const { return lo(i) / RAGGED_TILE; }
    RAGGED_FN int end_tile(int i) const { return (hi(i) + RAGGED_TILE - 1) / RAGGED_TILE; }
    RAGGED_FN long long cost(int i) const { return RAGGED_ITEM_COST + hi(i) - lo(i); }
    // cost of the items before item i (all of T tokens): past + (i + 1) T keys each, or T + window - 1 where the window bites
    RAGGED_FN long long before(int i) const {
        long long m = i;  // items that the window does not reach
        if (window > 0) m = least(m, most(0, T + window - 1 - past) / T);
        return (long long)i * RAGGED_ITEM_COST + m * past + T * (m * (m + 1) / 2) + (i - m) * (T + window - 1);
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
        const int snap = n - i * T > T / 2 ? RAGGED_SNAP : 0;
        if (z <= RAGGED_ITEM_COST) return first_tile(i);
        const int tile = (lo(i) + (int)(z - RAGGED_ITEM_COST) + RAGGED_TILE / 2) / RAGGED_TILE;
        if (tile <= first_tile(i) + snap) return first_tile(i);
        return tile >= end_tile(i) - snap ? end_tile(i) : tile;
    }
};

// Parts of a line of `total` keys for `grid` CTAs, and where cut c between them falls.
RAGGED_FN int ragged_parts(long long total, int grid) {
    return total == 0 ? 0 : (int)RaggedHead::most(1, RaggedHead::least(grid, total / RAGGED_MIN_PART));
}
RAGGED_FN long long ragged_cut(long long total, int parts, int c) { return total * c / parts; }

// Where position x of the line falls in a sequence that begins at `at`: (KV head, item, key tile).  cut: into how many
// pieces the line's cuts divide that item, which one of them CTA c has, and the CTA of the first.
RAGGED_FN void ragged_locate(const RaggedHead& h, long long at, long long x, long long total, int parts, int c, int* where, int* cut) {
    const long long head_cost = h.total();
    const int kvh = (int)((x - at) / head_cost);
    const int i = h.item_at(x - at - kvh * head_cost);
    const long long xs = at + kvh * head_cost + h.before(i), xe = xs + h.cost(i);
    where[0] = kvh;
    where[1] = i;
    where[2] = h.tile_at(i, x - xs);
    int f = (int)(xs * parts / total), l = (int)RaggedHead::least(parts, xe * parts / total + 1);
    while (f > 0 && ragged_cut(total, parts, f - 1) >= xs) --f;
    while (f <= l && (ragged_cut(total, parts, f) < xs || h.tile_at(i, ragged_cut(total, parts, f) - xs) <= h.first_tile(i))) ++f;
    while (l >= f && (ragged_cut(total, parts, l) >= xe || h.tile_at(i, ragged_cut(total, parts, l) - xs) >= h.end_tile(i))) --l;
    cut[0] = l >= f ? l - f + 2 : 1;  // cuts f .. l fall inside
    cut[1] = c - (f - 1);
    cut[2] = f - 1;
}
