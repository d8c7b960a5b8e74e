"""CPU check of paged.hpp: what a query row sees, the tiles that walk it, where rows lie in the
pages (bad entries included), division by the page size, and the split's workspace."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unlimited-ocr.cpp_amd", "csrc")
MAIN = r"""
#include "paged.hpp"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace uocr_hip;
#define CHECK(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)

static int spans() {
    const int M = 2147483647;
    for (int causal = 0; causal < 2; ++causal)
    for (int both = 0; both < 2; ++both)
    for (int window : {0, 1, 2, 5, 9, M}) {
        if (window && !causal) continue;
        for (int len = 0; len < 12; ++len)
        for (int pos = -2; pos < len; ++pos)
        for (int prefix : {-1, 0, 1, 3, 7, 11, 20, M})
        for (int begin : {-M - 1, -1, 0, 2, 6, 20, M})
        for (int end : {-M - 1, 0, 1, 4, 9, 12, M}) {
            const Span s = row_span(causal, window, both, pos, len, prefix, begin, end);
            int n = 0;
            for (int j = 0; j < len; ++j) {
                bool seen = !causal || j <= pos;
                if (window) seen = seen && (long long)j > (long long)pos - window;
                seen = seen || (j < prefix && (both || !causal || j <= pos));
                seen = seen && j >= begin && j < end;
                n += seen;
                CHECK(s.has(j) == seen);
            }
            CHECK(s.count() == n && s.b0 <= s.e0 && s.e0 <= s.b1 && s.b1 <= s.e1);
            if (n) CHECK((s.b0 == s.e0 || (s.b0 >= 0 && s.e0 <= len)) && (s.b1 == s.e1 || (s.b1 >= 0 && s.e1 <= len)));
            // every seen key in exactly one tile of its interval, no tile without one
            const TileWalk w = tile_walk<4>(s);
            int found = 0;
            for (int t = 0; t < w.count(); ++t) {
                const bool first = t < w.n0;
                const int base = (first ? w.t0 + t : w.t1 + t - w.n0) * 4, b = first ? s.b0 : s.b1, e = first ? s.e0 : s.e1;
                int here = 0;
                for (int j = base; j < base + 4; ++j) here += j >= b && j < e;
                CHECK(here > 0);
                found += here;
            }
            CHECK(found == n);
        }
    }
    // rows first .. last together: every key that one of them sees is in a range, and none beyond the sequence
    for (int causal = 0; causal < 2; ++causal)
    for (int both = 0; both < 2; ++both)
    for (int window : {0, 1, 2, 5, 9, M}) {
        if (window && !causal) continue;
        for (int len = 0; len < 12; ++len)
        for (int first = -3; first < len; ++first)
        for (int last = first; last < len; ++last)
        for (int prefix : {-1, 0, 1, 3, 7, 20, M}) {
            int l0, h0, l1, h1;
            tile_range(causal, window, both, first, last, len, prefix, l0, h0, l1, h1);
            CHECK(l0 >= 0 && l1 >= 0 && h0 <= len && h1 <= len && h0 >= 0 && h1 >= 0);
            for (int j = 0; j < len; ++j) {
                bool seen = false;
                for (int p = first; p <= last; ++p) seen = seen || row_span(causal, window, both, p, len, prefix, 0, M).has(j);
                const bool in = (j >= l0 && j < h0) || (j >= l1 && j < h1);
                CHECK(!seen || in);
                // and no key that none sees, but where prefix rows before the first position stand for the last's
                CHECK(!in || seen || first < 0);
            }
        }
    }
    // the far end of int
    const Span s = row_span(1, 100, 0, M - 1, M, 50, 0, M);
    CHECK(s.b0 == 0 && s.e0 == 50 && s.b1 == M - 100 && s.e1 == M);
    CHECK(tile_walk<32>(s).count() == 2 + (M - 1) / 32 - (M - 100) / 32 + 1);
    return 0;
}

static int places() {
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 16u, 24u, 48u, 100u, 255u, 256u, 1000003u, 1u << 30}) {
        const FastDiv f = fast_div(d);
        for (uint64_t n = 0; n < 3000; ++n) CHECK(f.div((uint32_t)n) == n / d);
        for (uint64_t k = 1; k * d < (1ull << 31); k += 1 + k / 3)
            for (long long n = (long long)(k * d) - 2; n < (long long)(k * d) + 2; ++n)
                if (n >= 0 && n < (1ll << 31)) CHECK(f.div((uint32_t)n) == n / d);
        for (long long n = (1ll << 31) - 3; n < (1ll << 31); ++n) CHECK(f.div((uint32_t)n) == n / d);
    }
    const int table[8] = {3, 0, -1, 5, 2, 4, 2147483647, 1};
    PagedCache c{};
    c.table = table;
    c.page_bytes = 3ll << 32;
    c.row_bytes = 1000;
    c.table_stride = 4;
    c.n_pages = 5;
    c.n_seqs = 2;
    c.max_pages = 4;
    c.ps = fast_div(6);
    CHECK(c.capacity() == 24);
    for (int s = 0; s < 2; ++s)
        for (int j = 0; j < 24; ++j) {
            const int page = table[s * 4 + j / 6];
            const long long want = page >= 0 && page < 5 ? page * (3ll << 32) + j % 6 * 1000 : -1;
            CHECK(c.offset(s, j) == want);
        }
    c.max_pages = 2147483647;
    CHECK(c.capacity() == 6ll * 2147483647);
    return 0;
}

static int splits() {
    for (int kv : {1, 2, 8, 10, 40})
        for (int g : {1, 4, 7, 16, 17, 33})
            for (long long rows : {1, 2, 3, 9, 33, 100, 257, 1000, 1024, 1025, 100000})
                for (long long r = 1; r <= rows; r += 1 + r / 5)
                    for (long long keys : {1ll, 17ll, 512ll, 1024ll, 1025ll, 5000ll, 2147483647ll}) {
                        const unsigned long long most = paged_workspace_records(rows, kv * g, kv);
                        for (int kt : {16, 32}) for (long long room : {keys, 2147483647ll}) {
                            const DecodePlan p = paged_decode_plan(r, kv * g, kv, kt, keys, room);
                            if (p.shares) CHECK(r * (room / kt + 3) <= 2147483647ll);
                            CHECK(p.blocks == (g + 15) / 16 && p.shares >= 0 && p.records <= most);
                            // a record for every wave, of its first and its last sequence, and query head
                            if (p.shares) CHECK(p.records == 2ull * p.shares * kv * p.blocks * (g < 16 ? g : 16) && r <= kPagedShareRows && r * kv * p.blocks <= kPagedCounters);
                        }
                        // prefill: r rows of one entry
                        for (int d : {8, 128, 256}) for (int f32 : {0, 1}) {
                            const PrefillPlan p = paged_prefill_plan(r, 1, kv * g, kv, d, f32, keys);
                            CHECK(p.row_waves == 4 || p.row_waves == 2 || p.row_waves == 1);
                            CHECK(p.tiles * p.row_waves * 32 >= r * g && p.splits >= 1 && p.splits <= kPagedMaxSplits);
                            if (p.splits > 1) CHECK((unsigned long long)r * kv * g * p.splits <= most);
                            // several entries, whose rows all see some of the keys
                            for (long long batch : {2ll, 7ll, r}) for (long long least : {0ll, keys / 2, keys}) {
                                const PrefillPlan b = paged_prefill_plan(r, batch, kv * g, kv, d, f32, keys, least);
                                CHECK(b.row_waves == 4 || b.row_waves == 2 || b.row_waves == 1);
                                CHECK(b.tiles >= r * g / (b.row_waves * 32) + batch && b.splits >= 1 && b.splits <= kPagedMaxSplits);
                                if (b.splits > 1) CHECK((unsigned long long)r * kv * g * b.splits <= most);
                            }
                        }
                    }
    return 0;
}

int main(int, char** v) { return v[1][0] == 's' ? spans() : v[1][0] == 'p' ? places() : splits(); }
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "m.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC,
                    str(d / "m.cpp"), "-o", str(d / "m")], check=True)
    return lambda what: subprocess.run([d / "m", what], capture_output=True, text=True)


@pytest.mark.parametrize("what", ["spans", "places", "workspace"])
def test_arithmetic(run, what):
    r = run(what)
    assert r.returncode == 0, r.stdout + r.stderr
