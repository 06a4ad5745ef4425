// How the attention over the multi-sequence cache is split (paged_split.hpp), at every
// size that its entry points accept: ranges stay inside what they are cut from, and
// what fills the chip as it is is not cut.
#include <cstdio>

#include "../../hymt2sharp_amd/csrc/paged_split.hpp"

using namespace hymt;

static int failures = 0;
static const char *where;
static long at[6];
#define CHECK(x)                                                                                                     \
    do {                                                                                                             \
        if (!(x)) {                                                                                                  \
            std::printf("%s: %s: n %ld kv_heads %ld group %ld blocks %ld max_len %ld prefix/rows %ld\n", where, #x,  \
                        at[0], at[1], at[2], at[3], at[4], at[5]);                                                   \
            failures++;                                                                                              \
        }                                                                                                            \
    } while (0)

static PagedSplit split(int n, int kv_heads, int group, int blocks, int max_len, int prefix, bool shared, int rows) {
    hymt_paged p{};
    p.kv_heads = kv_heads;
    p.blocks = blocks;
    hymt_batch b{};
    static const int32_t offsets = 0;
    b.cu = shared ? nullptr : &offsets;
    b.n = n;
    b.rows = rows;
    b.max_len = max_len;
    at[0] = n, at[1] = kv_heads, at[2] = group, at[3] = blocks, at[4] = max_len, at[5] = shared ? prefix : rows;
    return paged_split(p, b, group * kv_heads, prefix, shared);
}

static const int kEntries[] = {1, 2, 31, 32, 33, 64, 256, 511, 1024};
static const int kHeads[] = {1, 3, 4, 8, 32, 256};
static const int kGroups[] = {1, 4, 17, 64};
static const int kBlocks[] = {1, 9, 512, 1 << 14, 1 << 24};
static const int kLens[] = {0, 1, 64, 65, 8192, 1 << 20, 0x7FFFFFFF};

// A range of up to `pages` pages in `parts` parts of about `span`.
static void ranges(int parts, int span, long pages) {
    CHECK(parts >= 1 && parts <= kMaxParts);
    CHECK(span >= 1 && span <= (pages > 1 ? pages : 1));
    CHECK((long)parts * span >= pages);       // the longest range has its parts
    CHECK((long)(parts - 1) * span < pages || parts == 1);
}

static void every_size() {
    for (int n : kEntries)
        for (int h : kHeads)
            for (int g : kGroups)
                for (int blocks : kBlocks)
                    for (int len : kLens) {
                        const long longest = len ? std::min<long>(len, blocks * 64L) : blocks * 64L, pages = (longest + 63) / 64;
                        where = "shared";
                        for (int prefix : {0, 64, 4096, 1 << 20}) {
                            const PagedSplit s = split(n, h, g, blocks, len, prefix, true, n);
                            const long common = std::min<long>(prefix, longest) / 64, rows = (long)n * h * s.blocks16;
                            CHECK(s.blocks16 == (g + 15) / 16 && (s.rows == 64 || s.rows == 128));
                            CHECK(s.tiles == 0 || (prefix > 0 && s.tiles == ((long)n * g + s.rows - 1) / s.rows));
                            ranges(s.own, s.own_span, s.tiles ? pages - common : pages);
                            if (s.tiles) ranges(s.parts, s.span, common);
                            CHECK(rows < 256 || s.own == 1);                         // a workgroup a CU already
                            CHECK((long)s.tiles * h < 256 || s.parts == 1);
                            CHECK(rows * s.own <= std::max(rows, 2 * 256L));         // and not many more than that
                            CHECK((long)s.tiles * h * s.parts <= std::max((long)s.tiles * h, 2 * 256L));
                        }
                        where = "packed";
                        for (long rows : {1L, (long)n, 700L, 8192L, std::min(1L << 22, (1L << 28) / (h * g))}) {
                            const PagedSplit s = split(n, h, g, blocks, len, 0, false, (int)rows);
                            CHECK(s.rows == 64 || s.rows == 128);
                            CHECK(s.tiles == rows * g / s.rows + n);
                            CHECK(s.groups == 1 || s.groups == 2);
                            ranges(s.parts, s.span, pages);
                            const long wgs = (rows * g / 128 + n) * h;
                            CHECK(wgs <= 128 || s.parts == 1);
                            CHECK(wgs * s.parts <= std::max(wgs, 4 * 256L));
                        }
                    }
}

int main() {
    every_size();
    // one page too many for 31 bits: 2^15 rows' share of 2^24 pages each
    where = "the largest";
    const PagedSplit s = split(1024, 32, 1, 1 << 24, 0, 0, true, 1024);
    CHECK(s.own == 1 && s.own_span == 1 << 24);
    // long ranges of half as many rows as CUs are cut in two, short ones and those of more
    // rows stay whole
    where = "single rows";
    CHECK(split(32, 4, 4, 1 << 14, 32768, 0, true, 32).own == 2);
    CHECK(split(16, 8, 4, 1 << 14, 8256, 0, true, 16).own == 2);
    CHECK(split(32, 4, 4, 1 << 14, 8192, 0, true, 32).own == 1);
    CHECK(split(33, 4, 4, 1 << 14, 32768, 0, true, 33).own == 1);
    CHECK(split(48, 4, 4, 1 << 14, 32768, 0, true, 48).own == 1);
    if (failures) std::printf("%d failures\n", failures);
    return failures != 0;
}
