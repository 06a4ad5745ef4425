// paged_split.hpp -- how the attention over the multi-sequence cache is split: tiles of
// how many rows, kv ranges cut into how many parts (paged_attn.hip).  Plain host
// arithmetic on a call's sizes, without HIP, so that it can be looked at by itself.  The
// lengths are on the device, so every range is taken to be as long as max_len says,
// and which parts an entry has is settled there; the result is the same but for
// its rounding whatever is chosen here.
#pragma once

#include <algorithm>

#include "../../include/hymt_hip.h"

namespace hymt {

constexpr int kCus = 256;
constexpr int kMaxParts = 64;  // parts of a split range

struct PagedSplit {
    int tiles;           // of one kv head, at most
    int parts, span;     // a kv range (shared: the prefix) is cut into parts of about `span` pages, `parts` at most
    int own, own_span;   // shared: the same of an entry's own range
    int blocks16;        // of 16 q heads in a group
    int groups;          // of waves in a tile workgroup
    int rows;            // of a tile
};

inline long ceil_div(long a, long b) { return (a + b - 1) / b; }

// Cut ranges of up to `longest` pages, `average` on average, of `wgs` workgroups so
// that every one of `slots` gets its share, `least` pages at least, unless that saves
// less than `worth` pages' time on the longest.
inline void cut(long wgs, int longest, long average, int slots, int least, int worth, int &parts, int &span) {
    // a share of all workgroups' pages may pass 2^31; what is kept is `longest` at most
    const long share = std::max({(long)least, ceil_div(wgs * average, slots), ceil_div(longest, kMaxParts), 1L});
    span = longest <= share + worth ? std::max(longest, 1) : (int)share;
    parts = (int)std::max(1L, ceil_div(longest, span));
}

inline PagedSplit paged_split(const hymt_paged &p, const hymt_batch &b, int heads, int prefix, bool shared) {
    const int group = heads / p.kv_heads;
    const long room = (long)p.blocks * HYMT_PAGE_TOKENS, longest = b.max_len > 0 ? std::min<long>(b.max_len, room) : room;
    const int pages = (int)ceil_div(longest, HYMT_PAGE_TOKENS);
    PagedSplit s{0, 1, 1, 1, 1, (group + 15) / 16, 1, 128};
    if (shared) {
        const int common = (int)std::min<long>(prefix, longest) / HYMT_PAGE_TOKENS;
        // tiles of 64 rows until a CU has more than 8 pages of them (128 rows and 64: 8
        // rows behind 512 positions 9.4 and 8.6 us, 64 behind 4096 20.3 and 18.3, 128 22.1 and
        // 21.3; 256 behind 16384 73 and 88)
        if (ceil_div((long)b.n * group, 64) * p.kv_heads * common <= 8 * kCus) s.rows = 64;
        s.tiles = prefix ? (int)ceil_div((long)b.n * group, s.rows) : 0;
        const long rows = (long)b.n * p.kv_heads * s.blocks16;
        // Short sequences, and not too many rows: each row by itself through the prefix too, in one
        // launch without a join.  With tiles and without, us: 8 rows behind 512 positions and 64
        // of their own 8.7 and 6.8, 64 rows 12.8 and 8.1, 256 rows 21.2 and 19.0; behind 1024 8
        // rows 10.6 and 9.2, 128 18.0 and 15.9, 256 21.6 and 27.3; behind 1536 8 rows 10.3 and 11.4.
        if (s.tiles && pages <= 20 && rows * pages <= 40 * kCus) {
            s.tiles = 0;
            s.own_span = pages;
            return s;
        }
        // One tile a CU, beside it the rows: at 256 rows behind 16384 positions 75 us
        // (tiles in both places first, rows after them, 94).  Short parts, as
        // the join is launched anyway, yet not one page each of a longer prefix,
        // which moves more partials than it saves (64 rows behind 1024: one page 15.6 us,
        // three 13.9; 16 behind 8192: two 16.8, three 15.5; 8 behind 512: one 9.4, two 10.1).
        if (s.tiles) cut((long)s.tiles * p.kv_heads, common, common, kCus, common <= 8 ? 1 : 3, 0, s.parts, s.span);
        cut(rows, pages - common, pages - common, kCus, 4, 0, s.own, s.own_span);
        // Without tiles whole ranges need no join: cut in two or three they gain less (cut and whole,
        // us: 8 rows of 4 kv heads over 576 positions 9.3 and 7.9, over 2048 13.1 and 15.5; 32 over
        // 832 16.0 and 12.6, over 2048 30.3 and 28.8; 48 over 8192 146 and 134, over 32768 549 and
        // 518; 60 over 32768 663 and 657), except that a workgroup for every other CU is too
        // few for long ranges (32 rows over 4096 52.3 and 51.8, over 8192 97.7 and 98.2, over
        // 32768 360 and 375).
        const bool few = rows <= kCus / 2 && pages > 128;
        if (!s.tiles && !few && pages <= 2 * s.own_span + 4) {
            s.own = 1;
            s.own_span = std::max(pages, 1);
        }
    } else {
        auto tiles = [&](int rows) {
            return (int)(b.cu ? (long)b.rows * group / rows + b.n : (long)b.n * ceil_div(group, rows));
        };
        s.tiles = tiles(s.rows);
        // the rows are an entry's last ones: the first of them attend to less
        const int average = pages - (int)(std::min<long>(b.rows, longest) / HYMT_PAGE_TOKENS / 2);
        const long wgs = (long)s.tiles * p.kv_heads;
        // Two groups of waves, which halve a tile's own time, where the longest
        // tile takes about as long as the chip needs for all: one prompt of 2048
        // 48 -> 38 us, of 4096 93 -> 80; three of 2048 would go from 73 to 84, one of
        // 8192 from 262 to 277.
        if (pages >= 8 && 5L * pages * kCus >= 4 * wgs * average) s.groups = 2;
        // Few tiles of long ranges are cut besides (two chunks of 256 over 8192: 68
        // us with two parts, 50 with four).  Shorter ranges or more tiles are not: one
        // prompt of 1000 cut in four 34 us, whole 17; of 2048 47 and 38.
        if (wgs <= kCus / 2) cut(wgs, pages, average, 2 * kCus / s.groups, 4, 24, s.parts, s.span);
        else s.span = pages;
        // Tiles of half the rows, as a tile's time is mostly its own chain of reads
        // and products, as long as they do not queue for the CUs (128 rows and 64: one
        // sentence 8.6 and 6.6 us, 32 of them 11.0 and 10.0, one prompt of 700 18.8 and
        // 13.5, of 2048 37.6 and 34.2; but 12 of 200 16.0 and 17.1, 64 of 61 16.1 and 18.2).
        if (s.parts == 1 && 8 * wgs <= 9 * kCus) {
            s.rows = 64;
            s.tiles = tiles(s.rows);
        }
    }
    return s;
}

}  // namespace hymt
