// Paged key-value cache: places of rows in the pages and the keys that a query
// row sees, shared by the kernels (rope.hip, paged_decode.hip,
// paged_prefill.hpp), their launchers and a host-side check.
#pragma once

#include <stdint.h>

namespace uocr_hip {

#ifdef __HIP__
#define UOCR_HD __host__ __device__
#else
#define UOCR_HD
#endif

constexpr int kPagedShareRows = 1024;   // sequences of a decode call that is cut into shares
constexpr int kPagedShareGroups = 256;  // workgroups that it aims at: one per CU
constexpr int kPagedCounters = 16384;   // (sequence, KV head, 16 query heads) of such a call
constexpr int kPagedMagic = 0x70616765; // first word of a workspace that was set up
constexpr int kPagedHead = 64 + kPagedCounters * 4;  // bytes before a workspace's partial results
constexpr int kPagedUnitTiles = 8;     // tiles of keys that one workgroup takes alone
constexpr int kPagedPrefillTarget = 1024;  // workgroups of 128 pairs of a split prefill call at most
constexpr int kPagedMaxSplits = 128;

// n / d for 0 <= n < 2^31 by a multiplication: with s = ceil(log2 d) and
// mul = floor(2^(31+s) / d) + 1, the excess mul * d - 2^(31+s) is at most d <= 2^s,
// so n * mul / 2^(31+s) is n / d plus less than 1 / d.
struct FastDiv {
    uint32_t d, mul, shift;
    UOCR_HD uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> shift); }
};
inline FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return FastDiv{d, (uint32_t)((1ull << (31 + s)) / d + 1), 31 + s};
}

// The cache as the kernels see it; strides in bytes.
struct PagedCache {
    char* k;
    char* v;
    const int* table;  // [n_seqs][max_pages], rows table_stride apart
    long long page_bytes, row_bytes, head_bytes, table_stride;
    int n_pages, n_seqs, max_pages;
    FastDiv ps;  // page size

    // rows that the table has room for
    UOCR_HD long long capacity() const { return (long long)max_pages * ps.d; }
    // Byte offset of row `pos` of sequence `seq` (both in range: pos < capacity);
    // -1 where the table names no page of the cache.
    UOCR_HD long long offset(int seq, int pos) const {
        const uint32_t t = ps.div((uint32_t)pos);
        const int page = table[seq * table_stride + t];
        if ((uint32_t)page >= (uint32_t)n_pages) return -1;
        return page * page_bytes + (long long)((uint32_t)pos - t * ps.d) * row_bytes;
    }
};

// What a query row sees: keys [b0, e0) and [b1, e1), e0 <= b1, either may be empty.
struct Span {
    int b0, e0, b1, e1;
    UOCR_HD bool has(int j) const { return (j >= b0 && j < e0) || (j >= b1 && j < e1); }
    UOCR_HD int count() const { return (e0 - b0) + (e1 - b1); }
};

struct MaskArgs {
    int causal, window, both_ways;  // window 0: none
    const int* prefix_len;          // [n_seqs] or null
    const int* key_begin;           // [rows] or null
    const int* key_end;             // [rows] or null
};

UOCR_HD inline int imin(int a, int b) { return a < b ? a : b; }
UOCR_HD inline int imax(int a, int b) { return a > b ? a : b; }

// Row at position `pos` of a sequence of `len` keys, `prefix` of them its prefix, that sees
// keys [begin, end) at most: key j with j <= pos and j > pos - window (one token has
// causal set too), or j < prefix (and j <= pos unless the prefix is seen both ways).
UOCR_HD inline Span row_span(int causal, int window, int both_ways, int pos, int len, int prefix, int begin, int end) {
    const int hi = causal ? imin(len, pos + 1) : len;          // pos < len <= 2^31 - 1
    const int lo = window && pos >= window ? pos - window + 1 : 0;
    const int first = imin(both_ways ? len : hi, prefix);      // the prefix's keys are [0, first)
    begin = imax(begin, 0);
    end = imin(end, len);
    Span s;
    s.b0 = begin;
    s.e0 = imax(begin, imin(first, end));
    s.b1 = imax(imax(lo, s.e0), begin);
    s.e1 = imax(s.b1, imin(hi, end));
    // one interval where they touch
    if (s.b1 == s.e0) {
        s.e0 = s.e1;
        s.b1 = s.e1;
    } else if (s.e0 == s.b0) {
        s.b0 = s.e0 = s.b1;
    }
    return s;
}

// The keys that rows at positions first .. last see together (no limits of their own), as two
// ranges that may overlap; hi 0 or lo >= hi: empty.
UOCR_HD inline void tile_range(int causal, int window, int both_ways, int first, int last, int len, int prefix, int& lo0,
                               int& hi0, int& lo1, int& hi1) {
    const int hi = causal ? imin(len, last + 1) : len;
    lo0 = 0;
    hi0 = imax(imin(both_ways ? len : hi, prefix), 0);
    lo1 = window && first >= window ? first - window + 1 : 0;
    hi1 = imax(hi, 0);
    if (lo1 >= hi1) hi1 = 0;
}

// A row's span as tiles of W keys on W-aligned positions: the first tile that
// holds a key of each interval, and how many there are. Neighbouring intervals may share a
// tile; it is walked once for each, with that interval's keys.
struct TileWalk {
    int t0, n0, t1, n1;
    UOCR_HD int count() const { return n0 + n1; }
};
template <int W>
UOCR_HD inline TileWalk tile_walk(const Span& s) {
    TileWalk w;
    w.t0 = s.b0 / W;
    w.n0 = s.e0 > s.b0 ? (s.e0 - 1) / W - w.t0 + 1 : 0;
    w.t1 = s.b1 / W;
    w.n1 = s.e1 > s.b1 ? (s.e1 - 1) / W - w.t1 + 1 : 0;
    return w;
}

// How a decode call is shared out: one workgroup per (sequence, KV head, 16 query heads) where
// `max_keys` is short or the rows (or the `room` for their keys) too many for the shares' table, else (shares > 0) equal
// shares of all rows' tiles, one workgroup per share and KV head, and a join.
// A workgroup of 8 waves takes 8 tiles at a time, one of one wave leaves room for seven
// others: us of 8 / 1 waves: 1128 units of one key 19.3 / 6.1, 640 of up to
// 120 keys 14.5 / 11.8, 320 of up to 200 12.6 / 16.5.
struct DecodePlan {
    int blocks;   // of 16 query heads per KV head
    int unit_waves;
    int shares;   // 0: one workgroup per unit
    unsigned long long records;  // partial results of one (workgroup, first or last sequence, query head) each
};
inline DecodePlan paged_decode_plan(long long batch, int heads, int kv_heads, int tile_keys, long long max_keys, long long room) {
    DecodePlan p{(heads / kv_heads + 15) / 16, 8, 0, 0};
    // rounds on the chip (256 workgroups of 8 waves, 2048 of one) times the tiles one after the other, 2 tiles'
    // time for the beginning and the end
    const long long units = batch * kv_heads * p.blocks, longest = (max_keys + tile_keys - 1) / tile_keys;
    if ((units + 2047) / 2048 * (2 + longest) < (units + 255) / 256 * (2 + (longest + 7) / 8)) p.unit_waves = 1;
    if (batch > kPagedShareRows || max_keys <= kPagedUnitTiles * tile_keys) return p;
    const long long kvb = (long long)kv_heads * p.blocks;
    // (a row has two more tiles than its keys fill at most, and the line's length is an int)
    if (batch * kvb > kPagedCounters || batch * (room / tile_keys + 3) > 0x7fffffff) return p;
    const long long tiles = batch * ((max_keys + tile_keys - 1) / tile_keys);
    long long n = kPagedShareGroups / kvb;  // (no more than the chip holds at once)
    if (n < 1) n = 1;
    if (n > tiles) n = tiles;
    p.shares = (int)n;
    p.records = (unsigned long long)n * kvb * 2 * (heads / kv_heads < 16 ? heads / kv_heads : 16);
    return p;
}

// How a prefill call is shared out: workgroups of 4 waves (16-bit heads above 128: 8), `row_waves` of them along the
// (row, head) pairs of a KV head (32 each), the others on other tiles of keys; `tiles` of pairs per KV head at
// most (each entry rounds up by less than one), each of which sees min_keys to max_keys keys; the keys split over
// `splits` workgroups, 256 keys in each at least. Taken is what costs the least by this model, in quarters of the
// time that a tile of keys (64; f32: 32) takes a workgroup of 128 pairs on a full chip:
//   * a tile of keys, and a workgroup's beginning and end, by shape, below;
//   * rounds of `slots` workgroups; where they fill the chip the longest go first, and what the last round
//     leaves idle is as long as the shortest;
//   * splits: their sums' way through memory, a join with its launch.
// 128 pairs per workgroup share K and V best, 64 or 32 leave fewer rounds one after the other and more
// workgroups. us with 4 / 2 / 1 row waves, head_dim 128 (workgroups of 128 pairs):
//   bf16  10 heads, 64 rows (10) 7.5 / 9.0, 256 (30) 13.2 / 11.6, 1024 (90) 35 / 30, 4096 (330) 126 / 97;
//         32 heads over 8, 1024 rows (264) 51 / 30, 4096 (1032) 188 / 227, 1100 on 16000 keys (280) 456 / 711
//   f32   10 heads, 64 rows 16.4 / 13.9 / 15.5, 256 46 / 30 / 23, 1024 91 / 65 / 64, 4096 481 / 470 / 565;
//         32 heads over 8, 1024 rows 169 / 121 / 147, 4096 1230 / 1201 / 1720
// Heads above 128 keep 4 where they fill the chip (64 pairs: one wave per SIMD, bf16 376 us instead of 216 for 4096
// rows of 16 heads of 256 over 4); smaller calls of those heads: 64 rows bf16 16.9 / 13.2, f32 32 / 31, 256 rows 24 / 21
// and 91 / 77, heads of 192 in f32 26 / 22 and 70 / 47 (in 16 bits 64 pairs gain nothing there: 11.3 / 11.9).
// Splits, bf16: 64 rows of 32 heads on 16000 keys 1 split 351 us, 3 129, 12 61; 2100 rows of 16 heads of 256 (264
// workgroups) on 20000 keys 1 1785, 2 1345, 3 1211.
struct PrefillPlan {
    int row_waves, splits;
    long long tiles;
};
inline PrefillPlan paged_prefill_plan(long long rows, long long batch, int heads, int kv_heads, int head_dim, bool f32,
                                      long long max_keys, long long min_keys = 0) {
    struct Shape {
        int row_waves, slots;
        double tile, ends, way;
    };
    constexpr Shape kShapes[] = {{4, 512, 4.0, 16.0, 12.0}, {2, 512, 2.4, 18.0, 6.0},   // 16 bits, heads up to 128
                                 {4, 256, 4.0, 16.0, 12.0}, {2, 256, 4.2, 12.0, 6.0},   // above
                                 {2, 256, 2.0, 7.0, 3.5},   {1, 256, 1.2, 11.0, 1.7},   // f32
                                 {4, 256, 4.0, 6.0, 7.0},   {2, 256, 3.0, 5.0, 3.5}};
    const int first = (f32 ? 4 : 0) + (head_dim > 128 ? 2 : 0);
    const int last = !f32 && head_dim > 128 && head_dim <= 192 ? first : first + 1;
    const long long pairs = rows * (heads / kv_heads);
    const double longest = (double)max_keys / (f32 ? 32 : 64), shortest = (double)min_keys / (f32 ? 32 : 64);
    PrefillPlan p{4, 1, 0};
    double best = 1e300;
    for (int k = first; k <= last; ++k) {
        const Shape& s = kShapes[k];
        const long long across = 32 * s.row_waves;
        // the workgroups that there are likely to be
        long long units = batch == 1 ? (pairs + across - 1) / across : pairs / across + (batch + 1) / 2;
        units = (units < batch ? batch : units) * kv_heads;
        const bool full = units >= s.slots;
        if (full && k > first && head_dim > 128) continue;
        const double mean = full ? (longest + shortest) / 2 : longest, least = full ? shortest : longest;
        for (long long n = 1; n <= kPagedMaxSplits; ++n) {
            if (n > 1 && (n > max_keys / 256 || units * n * s.row_waves > 4 * kPagedPrefillTarget)) break;
            const double turns = (double)(units * n) / s.slots;
            const long long whole = (units * n + s.slots - 1) / s.slots;
            double cost = turns * (s.tile * mean / n + s.ends) + (whole - turns) * (s.tile * least / n + s.ends);
            if (n > 1) cost += (f32 ? 6.0 + 0.3 * n : 16.0 + 0.5 * n) + whole * s.way * (full ? 2 : 1);
            if (cost < best) {
                best = cost;
                p.row_waves = s.row_waves;
                p.splits = (int)n;
            }
        }
    }
    p.tiles = pairs / (32 * p.row_waves) + batch;
    return p;
}

// Partial results that calls of up to `rows` rows may hold. Decode: 2 per workgroup and query head;
// prefill: a unit is 32 (row, head) pairs of a KV head per row wave at most, and units * splits * row waves
// stays within 4 kPagedPrefillTarget.
inline unsigned long long paged_workspace_records(long long rows, int heads, int kv_heads) {
    const long long group = heads / kv_heads, kvb = kv_heads * ((group + 15) / 16), cols = group < 16 ? group : 16;
    const long long decode = (kPagedShareGroups + kvb) * 2 * cols;
    const long long all = rows * heads * kPagedMaxSplits, most = 128ll * kPagedPrefillTarget, prefill = all < most ? all : most;
    return (unsigned long long)(decode > prefill ? decode : prefill);
}

}  // namespace uocr_hip
