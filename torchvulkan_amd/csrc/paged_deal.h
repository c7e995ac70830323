// How paged attention deals a call's tiles to its workgroups: the arithmetic
// between the lengths' totals and a workgroup's pieces. Plain constexpr functions
// without a wave in them, so that the kernel (paged_attention_mfma.h) and a model
// of whole launches on the host (tests/paged_deal_model.cpp) run the same ones.
// Sums of tiles and units stay below 2^31 (paged_attn_mfma); products of a
// workgroup's number and a stretch's length do only where the workgroup has one.
#pragma once

#include <cstdint>

namespace tvk {

#define TVK_DEAL [[gnu::always_inline]] constexpr

// n / d for a quotient below 2^22, rd being 1 / d: a float estimate that is at most one off.
TVK_DEAL uint32_t small_div(uint32_t n, uint32_t d, float rd) {
    uint32_t q = (uint32_t)((float)n * rd);
    const int r = (int)(n - q * d);
    if (r < 0) --q;
    else if (r >= (int)d) ++q;
    return q;
}

// What a launch is dealt with.
struct PagedPlan {
    int wgs;        // workgroups of the launch
    int resident;   // workgroups that run together
    int many;       // segments enough to fill the chip: chunks only
    int shared;     // rows of neighbouring heads share 128-byte lines
};

// Keys of a segment, in tiles of 32, up to which it takes one wave and one workgroup. A wave spares the merge of four
// (float16 98 x 64/8 heads x 16 keys of 128: 6.0 us, 10.9 with four) and takes the tiles one after another. More segments
// than run together wait less for shorter workgroups; segments that fill a third of the chip have no use for being cut
// (bfloat16 52 x 64/16 heads x 743 keys of 64: 20.9 us whole, 24.3 in pieces), few long ones do (float32 6 x 32/8 heads x
// 640 keys of 256: 16 us in pieces, 35 whole).
constexpr int PM_WAVE = 2, PM_WAVE_MANY = 4, PM_WHOLE = 17, PM_WHOLE_MANY = 49;
constexpr double PM_MANY = 0.35;

TVK_DEAL bool paged_many(int64_t segments, int64_t resident) { return (double)segments > (double)resident * PM_MANY; }
// Whether segments of up to `keys` keys are cut at all.
TVK_DEAL bool paged_is_dealt(bool many, int64_t keys) { return keys > 32 * (many ? PM_WHOLE_MANY : PM_WHOLE); }

// Workgroups a launch of `segments` segments of at most `tiles` tiles is given: one for every 4 tiles the sequences may
// have, as many as are resident together, or what the chunks of many segments may come to.
TVK_DEAL int64_t paged_wgs(bool many, int64_t segments, int64_t tiles, int64_t resident) {
    const int64_t some = segments * (tiles / 4);
    return many ? segments + 2 * resident : some < resident ? some : resident;
}

// Workgroups whose pieces have a place in the scratch: those that share a segment with others. Many segments are cut into
// at most 2 * resident chunks beside the whole ones, or into a stretch for each resident workgroup.
TVK_DEAL int64_t paged_places(bool many, int64_t wgs, int64_t resident) { return many ? 2 * resident : wgs; }

struct PagedDeal {
    int shift;        // segments are cut into chunks of at least 2^shift tiles; -1: stretches
    uint32_t per;     // tiles a workgroup's stretch has
    uint32_t snap;    // an end of a stretch this near to a segment's moves there: a short piece costs more than its tiles
    uint32_t total;   // tiles of the call
    uint32_t used;    // workgroups that get any (chunks: if heads share lines)
    TVK_DEAL uint32_t units(uint32_t tiles) const { return shift < 0 ? tiles : tiles >> shift > 1 ? tiles >> shift : 1; }
};

// count(d): the units of the whole call as d cuts it. rcp(x): 1 / x to a float's last places.
template <int BN, class Count, class Rcp>
TVK_DEAL PagedDeal paged_deal(const PagedPlan& p, uint32_t total, Count count, Rcp rcp) {
    PagedDeal d{2, 0, 0, total, 0};
    // at least a resident workgroup's share: the float product is off by less than one in 2^22
    d.per = (uint32_t)((float)total * rcp((float)(p.wgs < p.resident ? p.wgs : p.resident)) * 1.000001f) + 1;
    d.snap = 128u / BN < d.per / 4 ? 128u / BN : d.per / 4;
    // Many segments and short stretches: a piece's start and end would cost more than its tiles (float32 20 x 16/16 heads x
    // 1442 keys of 64: 44 us in chunks, 56 in stretches). At most a chunk a segment and two for each of the resident
    // workgroups: they fit the launch.
    const bool chunks = p.many && d.per < 1536 / BN;
    if (chunks) {
        d.shift = BN == 32 ? 3 : 4;
        while (((uint64_t)p.resident << (d.shift + 1)) < total) ++d.shift;
        if (!p.shared) return d;
    }
    if (chunks || !p.many) {
        for (;; ++d.shift) {
            d.used = count(d);
            if (chunks || d.used <= (uint32_t)p.wgs) return d;
            if (d.shift == 4) break;
        }
    }
    d.shift = -1;
    d.used = small_div(total + d.per - 1, d.per, rcp((float)d.per));
    return d;
}

// Workgroup wg's first unit x, and the tile its stretch ends at; false where no stretch is left for it. A launch of many
// segments has more workgroups than there are stretches, and wg * per of those would pass 2^32.
TVK_DEAL bool paged_start(const PagedDeal& d, uint32_t wg, uint32_t& x, uint32_t& stop) {
    x = wg;
    if (d.shift >= 0) return true;
    if (wg >= d.used) return false;
    x = wg * d.per;
    stop = d.total - x < d.per ? d.total : x + d.per;
    return true;
}

// Piece i of a segment: a stretch of its tiles, [c0, c1); how many there are, and the place of the first.
struct PagedPiece {
    int item, hk;
    uint32_t c0, c1;
    uint32_t first, pieces, i;
};

// Where the end of a stretch at tile x of a segment's tiles lies.
TVK_DEAL uint32_t paged_cut(const PagedDeal& d, uint32_t x, uint32_t tiles) {
    return x <= d.snap ? 0 : tiles - x <= d.snap ? tiles : x;
}

// The chunk `at` of a segment that is cut into `units`; it is workgroup x's. `begin`: the segment's first tile of the call,
// which says where its pieces are kept where many segments are whole: k chunks have 2^shift * k tiles and more, and floor(a)
// + floor(b) <= floor(a + b).
TVK_DEAL void paged_chunk(const PagedPlan& p, const PagedDeal& d, uint32_t x, uint32_t begin, uint32_t at, uint32_t tiles,
                          uint32_t units, float r_units, PagedPiece& pc) {
    const uint32_t q = small_div(tiles, units, r_units), r = tiles - q * units;
    pc.c0 = at * q + (at < r ? at : r);
    pc.c1 = pc.c0 + q + (at < r);
    pc.first = p.many ? begin >> d.shift : x - at;
    pc.pieces = units;
    pc.i = at;
}

// The piece of a segment from its tile `at`, tile x of the call, on, of workgroup wg's stretch that ends at `stop`. Ends of
// stretches inside a segment that do not move to its ends cut it.
TVK_DEAL void paged_stretch(const PagedDeal& d, uint32_t wg, uint32_t x, uint32_t at, uint32_t tiles, uint32_t stop, float r_per, PagedPiece& pc) {
    const uint32_t begin = x - at;
    pc.first = small_div(begin + d.snap, d.per, r_per);
    const uint32_t last = tiles > 2 * d.snap ? small_div(begin + tiles - d.snap - 1, d.per, r_per) : 0;
    pc.pieces = last > pc.first ? last - pc.first + 1 : 1;
    pc.i = wg - pc.first;
    pc.c0 = paged_cut(d, at, tiles);
    pc.c1 = stop - x < tiles - at ? paged_cut(d, at + (stop - x), tiles) : tiles;
}

// Where a segment's piece i is kept: a workgroup has at most one piece that does not begin its segment and one that does
// and does not end it.
TVK_DEAL uint32_t paged_slot(uint32_t first, uint32_t i) { return 2 * (first + i) + (i == 0); }

#undef TVK_DEAL

}  // namespace tvk
