// Model of a whole paged-attention launch on the host: every workgroup runs the
// arithmetic of torchvulkan_amd/csrc/paged_deal.h as the kernel does, with the
// sums over items that a wave takes there taken here. Checks that
//   1. every tile of every segment belongs to one piece;
//   2. a segment's pieces agree on their number and on the first, and come once;
//   3. a segment in one piece is whole;
//   4. pieces that are kept for a join lie in places of their own, inside the buffer.
// Arguments: BN CT resident kvh group new window shared batch longest shortest power: lengths rise to the longest as the power of a
// line.
// Prints "ok", the launch's workgroups (0: segments of so few keys are not cut) and the kept pieces' places; a violation
// ends it with a message.
#include "paged_deal.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <vector>

using namespace tvk;

namespace {

[[noreturn]] void die(const char* what, long long a, long long b) {
    std::fprintf(stderr, "paged deal model: %s (%lld, %lld)\n", what, a, b);
    std::exit(1);
}

struct Kept {
    uint32_t c0, c1, first, pieces, i;
    bool operator<(const Kept& o) const { return c0 < o.c0; }
};

// A reciprocal a step above or below the nearest float, as a hardware one may be.
int g_off = 0;
float rcp(float x) {
    const float r = 1.0f / x;
    return g_off ? std::nextafterf(r, g_off > 0 ? 2.0f * r : 0.0f) : r;
}

struct Call {
    int bn, ct, resident, kvh, group;
    int64_t fresh, window;
    int shared;
    std::vector<int64_t> lens;
};

template <int BN>
void run(const Call& c, int64_t& launch, uint32_t& places) {
    const int64_t rows = c.fresh * c.group, block = 16 * c.ct, nrb = (rows + block - 1) / block;
    const int64_t items = (int64_t)c.lens.size() * nrb, segments = items * c.kvh;
    std::vector<uint32_t> tiles((size_t)items);
    for (int64_t e = 0; e < items; ++e) {
        const int64_t len = c.lens[(size_t)(e / nrb)], r0 = e % nrb * block, r1 = std::min(rows, r0 + block) - 1;
        const int64_t t0 = r0 / c.group, t1 = r1 / c.group;
        const int64_t hi = std::max<int64_t>(0, len - c.fresh + t1 + 1), top = len - c.fresh + t0 + 1;
        const int64_t lo = std::min(hi, c.window && top > c.window ? top - c.window : 0);
        tiles[(size_t)e] = hi > lo ? (uint32_t)((hi + BN - 1) / BN - lo / BN) : 1;
    }
    const int64_t longest = *std::max_element(c.lens.begin(), c.lens.end());
    const int64_t keys = c.window ? std::min(longest, c.window + c.fresh + BN) : longest;
    PagedPlan p{};
    p.resident = c.resident;
    p.many = paged_many(segments, c.resident);
    p.shared = c.shared;
    if (!paged_is_dealt(p.many, (keys + BN - 1) / BN * BN)) return;
    p.wgs = (int)(launch = paged_wgs(p.many, segments, (keys + BN - 1) / BN, c.resident));
    uint64_t total = 0;
    for (const uint32_t t : tiles) total += (uint64_t)t * c.kvh;
    if (total >= 1u << 31) die("more tiles than the kernel takes", (long long)total, 0);
    const auto count = [&](const PagedDeal& d) {
        uint64_t n = 0;
        for (const uint32_t t : tiles) n += (uint64_t)d.units(t) * c.kvh;
        return (uint32_t)n;
    };
    const PagedDeal d = paged_deal<BN>(p, (uint32_t)total, count, rcp);
    std::vector<uint64_t> unit0((size_t)items + 1, 0);   // units before an item
    for (int64_t e = 0; e < items; ++e) unit0[(size_t)e + 1] = unit0[(size_t)e] + (uint64_t)d.units(tiles[(size_t)e]) * c.kvh;

    std::vector<std::vector<Kept>> of((size_t)segments);
    places = 0;
    std::vector<char> taken((size_t)2 * paged_places(p.many, p.wgs, p.resident), 0);
    std::vector<uint64_t> tile0((size_t)items + 1, 0);   // tiles before an item
    for (int64_t e = 0; e < items; ++e) tile0[(size_t)e + 1] = tile0[(size_t)e] + (uint64_t)tiles[(size_t)e] * c.kvh;
    for (uint32_t launched = 0; launched < (uint32_t)p.wgs; ++launched) {
        uint32_t wg = launched, x, stop = 0;
        if (p.shared && wg < d.used / 8 * 8) wg = wg % 8 * (d.used / 8) + wg / 8;
        if (!paged_start(d, wg, x, stop) || x >= unit0.back()) continue;
        PagedPiece pc{};
        pc.item = (int)(std::upper_bound(unit0.begin(), unit0.end(), (uint64_t)x) - unit0.begin()) - 1;
        uint32_t at = x - (uint32_t)unit0[(size_t)pc.item];
        for (bool more = true; more;) {
            const uint32_t n = tiles[(size_t)pc.item], units = d.units(n);
            more = false;
            pc.hk = (int)small_div(at, units, rcp((float)units));
            at -= (uint32_t)pc.hk * units;
            const int64_t segment = (int64_t)pc.item * c.kvh + pc.hk;
            if (pc.hk >= c.kvh) die("a head past the last", pc.item, pc.hk);
            if (d.shift >= 0) {
                paged_chunk(p, d, x, (uint32_t)tile0[(size_t)pc.item] + (uint32_t)pc.hk * n, at, n, units, rcp((float)units), pc);
            } else {
                paged_stretch(d, wg, x, at, n, stop, rcp((float)d.per), pc);
                x += n - at;
                more = x < stop;
                at = (uint32_t)(pc.hk + 1) * n;
            }
            if (more && pc.hk + 1 == c.kvh) {
                ++pc.item;
                at = 0;
            }
            if (pc.c0 >= pc.c1) continue;
            if (pc.c1 > n) die("tiles past a segment's last", (long long)segment, pc.c1);
            of[(size_t)segment].push_back(Kept{pc.c0, pc.c1, pc.first, pc.pieces, pc.i});
            if (pc.pieces == 1) continue;
            if (pc.i >= pc.pieces || (pc.i == 0) != (pc.c0 == 0)) die("a piece that is not one of its segment's", (long long)segment, pc.i);
            const uint32_t slot = paged_slot(pc.first, pc.i);
            if (slot >= taken.size()) die("a place past the buffer", (long long)segment, slot);
            if (taken[slot]++) die("a place that is kept twice", (long long)segment, slot);
            places = std::max(places, slot + 1);
        }
    }
    for (int64_t s = 0; s < segments; ++s) {
        auto& v = of[(size_t)s];
        std::sort(v.begin(), v.end());
        uint32_t at = 0;
        for (const Kept& k : v) {
            if (k.c0 != at) die("a tile that none or two pieces have", (long long)s, k.c0);
            if (k.first != v[0].first || k.pieces != v.size()) die("pieces that disagree", (long long)s, k.pieces);
            if (v.size() > 1 && k.i != (uint32_t)(&k - v.data())) die("pieces out of order", (long long)s, k.i);
            at = k.c1;
        }
        if (at != tiles[(size_t)(s / c.kvh)]) die("tiles that no piece has", (long long)s, at);
    }
}

}  // namespace

int main(int argc, char** argv) {
    if (argc != 13) return 2;
    long long a[12];
    for (int i = 0; i < 12; ++i) a[i] = std::atoll(argv[i + 1]);
    Call c{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4], a[5], a[6], (int)a[7], {}};
    for (long long i = 0; i < a[8]; ++i) c.lens.push_back(a[10] + (int64_t)((double)(a[9] - a[10]) * std::pow((double)(i + 1) / (double)a[8], (double)a[11])));
    int64_t launch = 0;
    uint32_t places = 0;
    for (g_off = -1; g_off <= 1; ++g_off) {
        uint32_t n = 0;
        c.bn == 32 ? run<32>(c, launch, n) : run<16>(c, launch, n);
        places = std::max(places, n);
    }
    std::printf("ok %lld %u\n", (long long)launch, places);
    return 0;
}
