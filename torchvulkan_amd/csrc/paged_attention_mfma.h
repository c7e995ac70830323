// MFMA kernel of tvk_paged_attention.
//
// The new_tokens * group query rows that share a key/value head are the
// columns of the products, 16 or 32 (CT) of them a row block. Keys go by tiles
// of 32, a wave a tile: S^T = K Q^T, an online softmax per column in log2
// units, O^T += V^T P^T. The call reads each key and value once and is bound
// by that stream, so nothing stands between a wave and its loads: no LDS and no
// barrier in the loop, both tiles of the next step in flight while one is
// computed.
//   K: lane (g, c) = (lane / 16, lane % 16) holds row c of each 16-key half, 16
//      bytes of every 64: the A operand of S^T as it lies in memory. The order
//      of a row's values in the products is that of these chunks, for K and Q
//      alike.
//   V: lane (g, c) holds EV neighbouring values, from EV * c, of the rows
//      4g .. 4g + 3 of each half. Those eight rows are the keys whose
//      probabilities the lane holds after S^T, so A operands of V^T are pairs of
//      16-bit values picked out of the lane's own registers (v_perm); row m of
//      the product for value e is column EV * m + e of the output. float32
//      values and probabilities are operands of the 16x16x4 product as they are.
//
// Work is dealt by every workgroup itself (paged_deal.h), from the lengths on the device: a
// batch's lengths are not on the host, and a launch sized by the longest would
// leave the others' workgroups idle. A segment is a row block of a sequence and a
// key/value head. Short ones take a wave or a workgroup each, as max_len tells the
// host. Else segments are cut into chunks of at least 4 (8, 16) tiles where those
// do not exceed the workgroups that run together; where they do, all tiles of the
// call, in segment order, are cut into equal stretches, and a workgroup's stretch
// may end one segment and begin others. Its 4 waves take a stretch's tiles in turn
// and are merged through LDS in wave order. A segment that lies in one workgroup is
// written out; the pieces of another go to scratch as float32 (max, sum, O), written
// through to memory as the skinny GEMM's split_fixup does. They are joined in runs,
// and the runs' results in order, by the last workgroup to finish; where that is
// more than one workgroup reads in a few microseconds, by the last of each run and
// then the last of all, or by a second launch, which a stream without counters takes
// too. All give the same bits every run. Segments count 128 bytes apart: those that
// count on one line wait for each other, 13 ns each (6 x 15334 keys of one head of 32,
// 120 pieces each: 16.7 us on one line, 12.5 apart).
//
// Slots with rows of less than whole 128-byte lines share lines between heads, and an
// XCD that reads one head fetches its neighbours' values too. Workgroups go to the XCDs
// in turn, so the heads of a sequence are numbered to meet on one (bfloat16 73 x 64/16
// heads x 1149 keys of 32: 42 us, 61 in the order of the heads; 128-byte rows keep
// that order, which spreads long sequences better: 65 us, 69 for 110 x 1149 keys of 128).
//
// Measured: one sequence of 100001 keys (32/8 heads of 128, bfloat16) 82 us, 5.0
// TB/s; 32 of up to 8000 keys 110 us, 4.9 TB/s; 24 of up to 6001 in 8 bits with 4
// tokens each 53-57 us, 3.4-3.1 TB/s: 592 chunks of 32 to 58 tiles, 37 on average, and
// the call ends with the longest; 16 with windows of 1000 keys, 12 heads of 80 in
// float16 16.5 us, 3.1 TB/s. Prompts are far from the products' rate: a tile feeds 32
// rows only (bfloat16 32/8 heads of 128, one prompt of 8192 tokens 3.9 ms, 140 TFLOP/s).
#pragma once

#include "attention_kernels.h"
#include "paged.h"
#include "paged_deal.h"

namespace tvk {

struct PagedMfmaArgs {
    PagedAttnArgs a;
    uint32_t kp, ks, vp, vs;   // page and slot strides of keys and values, in 16 bytes
    int rows;              // new_tokens * group
    int items;             // batch * row blocks of a key/value head
    PagedPlan plan;        // wgs 0: a workgroup a segment
    Div32 nrb, kvh, group;
    int places;            // workgroups whose pieces are kept
    float* part_o;         // [2 * places][16 * CT][hd]
    float* part_ml;        // [2][2 * places][16 * CT][2]: max, sum; again where a run's result is kept
    unsigned part_bytes;   // of both
    // finished pieces (or runs) of every segment, then finished pieces of the run that begins in every slot; zero before
    // and after the launch. NULL: a second launch joins, one of `slices` workgroups some of a segment's rows, and
    // `seg` [items * kvh][2] tells it a segment's first workgroup and its pieces
    unsigned* count;
    int spread;            // log2 of the words from a segment's counter to the next
    uint32_t* seg;
    int slices;
};

namespace {

constexpr int PM_WAVES = 4;   // paged_wgs: a tile for each

template <int DT, bool F8, int D>
struct PagedTile {
    static constexpr int NB = DT == TVK_F32 ? 1 : 2;            // blocks of 16 keys in a tile
    static constexpr int BN = 16 * NB;
    static constexpr int ES = F8 ? 1 : DT == TVK_F32 ? 4 : 2;   // bytes of a cached value
    static constexpr int KL = (D * ES + 63) / 64;               // 16-byte K chunks a lane holds of a row
    static constexpr int QS = F8 ? 2 * KL : KL;                 // Q fragments of 16 bytes
    static constexpr int EV = D == 96 ? 8 : D / 16;             // V values a lane holds of a row
    static constexpr int DV = 16 * EV;
    static constexpr int VW = EV * ES / 4;                      // the same in 32-bit words
    // Workgroups a CU that calls are dealt for: an estimate by the registers, K and V tiles, Q, O and S, and 90 beside them.
    // It is what the kernels for pages of any size get; those for whole pages of 8 bits up to 128 columns and one row block,
    // of 64 and two, of 256 and one, and of bfloat16 with 128 and two take fewer, and one workgroup more fits.
    // Three of bfloat16 and 128 columns would fit their loop, but 12 waves with a tile each on its way read slower than 8
    // (32 x 8000 keys: 124 us, 112).
    static constexpr int regs(int ct) { return 4 * NB * (KL + VW) + ct * (4 * QS + 4 * EV + 4 * NB) + 90; }
    static constexpr int occ(int ct) { return regs(ct) <= 128 ? 4 : regs(ct) <= 168 ? 3 : regs(ct) <= 256 ? 2 : 1; }
};

// ---------------------------------------------------------------------------
// dealing
// ---------------------------------------------------------------------------

struct PagedSpan {
    int b, len;
    int t0, t1;   // the row block's first and last token
    int pad;      // tokens in front that are padding
    int lo, hi;   // keys that some row of the block sees
    int tiles;    // at least one: a segment without keys writes its zeros
};

// Keys below it are seen by token t of a sequence; of those, the ones from window_lo on.
__device__ __forceinline__ int window_lo(int hi, uint32_t window) { return window && hi > (int)window ? hi - (int)window : 0; }

template <int BN, int CT>
__device__ __forceinline__ PagedSpan paged_span(const PagedMfmaArgs& p, int e) {
    PagedSpan s;
    s.b = (int)div32((uint32_t)e, p.nrb);
    const int r0 = (e - s.b * (int)p.nrb.d) * 16 * CT, r1 = min(p.rows, r0 + 16 * CT) - 1;
    s.len = (int)min((uint32_t)paged_len(p.a.c, s.b), p.a.max_len);
    s.t0 = (int)div32((uint32_t)r0, p.group);
    s.t1 = (int)div32((uint32_t)r1, p.group);
    s.pad = paged_padding(p.a.c, s.b, p.a.new_tokens);
    s.hi = s.t1 < s.pad ? 0 : max(0, s.len - p.a.new_tokens + s.t1 + 1);
    s.lo = min(s.hi, window_lo(s.len - p.a.new_tokens + max(s.t0, s.pad) + 1, p.a.window));
    s.tiles = s.hi > s.lo ? (s.hi + BN - 1) / BN - s.lo / BN : 1;
    return s;
}

__device__ __forceinline__ float wave_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ uint32_t wave_div(uint32_t n, uint32_t d) { return small_div(n, d, wave_rcp((float)d)); }

// v + the lane's value from lanes below it by a DPP move (0 where there is none), in the rows of 16 lanes that MASK names.
template <int CTRL, int MASK>
__device__ __forceinline__ uint32_t plus_moved(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, MASK, 0xf, false);
}
// Inclusive sums over a wave's lanes.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v = plus_moved<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8
    v = plus_moved<0x112, 0xf>(v);
    v = plus_moved<0x114, 0xf>(v);
    v = plus_moved<0x118, 0xf>(v);
    v = plus_moved<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3
    return plus_moved<0x143, 0xc>(v);   // row_bcast 31 into rows 2 and 3
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63); }

// mine: the tiles of item `lane`.
template <int BN, int CT>
__device__ __forceinline__ PagedDeal paged_deal_of(const PagedMfmaArgs& p, int lane, uint32_t mine) {
    uint32_t n = mine;
    for (int e = lane + 64; e < p.items; e += 64) n += (uint32_t)paged_span<BN, CT>(p, e).tiles;
    auto count = [&](const PagedDeal& d) {
        uint32_t u = mine ? d.units(mine) : 0;
        for (int e = lane + 64; e < p.items; e += 64) u += d.units((uint32_t)paged_span<BN, CT>(p, e).tiles);
        return wave_sum(u) * p.kvh.d;
    };
    return paged_deal<BN>(p.plan, wave_sum(n) * p.kvh.d, count, [](float x) { return wave_rcp(x); });
}

// The item that holds unit x of the call, the unit's place among the item's, and, where many segments are cut into chunks,
// the item's first tile of the call; false past the last.
template <int BN, int CT>
__device__ __forceinline__ bool paged_locate(const PagedMfmaArgs& p, const PagedDeal& d, uint32_t x, int lane, uint32_t mine, int& item,
                                             uint32_t& at, uint32_t& begin) {
    uint32_t base = 0, tiles = 0;
    const bool begins = p.plan.many && d.shift >= 0;
    for (int e0 = 0;;) {
        const uint32_t n = mine ? d.units(mine) * p.kvh.d : 0;
        const uint32_t s = base + wave_scan(n);
        const uint32_t ts = begins ? tiles + wave_scan(mine * p.kvh.d) : 0;
        const uint64_t past = __ballot(s > x);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            item = e0 + l;
            at = x - (uint32_t)__builtin_amdgcn_readlane((int)(s - n), l);
            begin = (uint32_t)__builtin_amdgcn_readlane((int)(ts - mine * p.kvh.d), l);
            return true;
        }
        e0 += 64;
        if (e0 >= p.items) return false;
        base = (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
        tiles = (uint32_t)__builtin_amdgcn_readlane((int)ts, 63);
        mine = e0 + lane < p.items ? (uint32_t)paged_span<BN, CT>(p, e0 + lane).tiles : 0;
    }
}

// ---------------------------------------------------------------------------
// partials and outputs
// ---------------------------------------------------------------------------

// Query row r of (b, hk), its softmax's max and sum known: where it goes, and the factor of its products.
struct PagedRow {
    int64_t o, lse;
    float f, l;
    __device__ __forceinline__ PagedRow(const PagedMfmaArgs& p, int b, int hk, int r, float m, float sum) {
        const int t = (int)div32((uint32_t)r, p.group), h = hk * (int)p.group.d + (r - t * (int)p.group.d);
        o = (int64_t)b * p.a.so[0] + (int64_t)t * p.a.so[1] + (int64_t)h * p.a.so[2];
        lse = (int64_t)b * p.a.sl[0] + (int64_t)t * p.a.sl[1] + (int64_t)h * p.a.sl[2];
        // a NaN sum is a NaN row; only a row without keys is zeros, as its products are
        const bool none = sum == 0.0f;
        f = none ? 0.0f : (p.a.c.v_scale ? p.a.c.v_scale[hk] : 1.0f) * __builtin_amdgcn_rcpf(sum);   // sum >= 1, or no number
        l = none ? INFINITY : (m + __builtin_amdgcn_logf(sum)) * AT_LN2;
    }
    // columns dv .. dv + 3
    template <int DT>
    __device__ __forceinline__ void store(const PagedMfmaArgs& p, int dv, f32x4 v) const {
        if (dv == 0 && p.a.lse) p.a.lse[lse] = l;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= f;
        if constexpr (DT == TVK_F32) {
            typedef float V __attribute__((ext_vector_type(4), aligned(4)));
            *reinterpret_cast<V*>(static_cast<float*>(p.a.out) + o + dv) = v;
        } else {
            *reinterpret_cast<u32x2u*>(static_cast<uint16_t*>(p.a.out) + o + dv) =
                u32x2u{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
        }
    }
};

// A running (max, sum, O) takes in another.
struct PagedSum {
    float m = -INFINITY, l = 0.0f;
    f32x4 o = f32x4{0, 0, 0, 0};
    __device__ __forceinline__ void raise(float mn) {
        const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= f;
        m = mn;
    }
    __device__ __forceinline__ void add(float ms, float ls, f32x4 os) {   // ms <= m
        const float f = ms == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ms - m);
        l += ls * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += os[i] * f;
    }
};

// The runs that a segment's pieces are joined in: run r is the pieces [at(r), at(r + 1)).
struct PagedRuns {
    uint32_t pieces, n;
    bool apart;   // by several workgroups
    __device__ __forceinline__ uint32_t at(uint32_t r) const { return pieces * r / n; }
    __device__ __forceinline__ uint32_t of(uint32_t i) const { return ((i + 1) * n - 1) / pieces; }
};

__device__ __forceinline__ PagedRuns paged_runs(uint32_t pieces, uint32_t quads) {   // quads of columns in all of the rows
    PagedRuns r{pieces, 1, pieces * quads > 8192};   // 128 KB
    if (r.apart) r.n = min(32u, (pieces + 7) / 8);
    else if (quads <= 128 && pieces >= 8)
        r.n = min(min(32u, 256u / quads), pieces / 4);   // threads that would be idle take one each
    return r;
}

// Partials in memory. SHARED: other workgroups of the launch write and read them, through the L2 (an XCD's lines may be
// older than another's stores); else an earlier launch wrote them.
template <int CT, bool SHARED>
struct PagedParts {
    const PagedMfmaArgs& p;
    __amdgpu_buffer_rsrc_t rs;
    __device__ __forceinline__ PagedParts(const PagedMfmaArgs& a)
        : p(a), rs(__builtin_amdgcn_make_buffer_rsrc((void*)a.part_o, 0, (int)a.part_bytes, 0x00020000)) {}
    // byte offsets: below 2 GiB; of a run's result in the place of its first piece, whose max and sum others still read
    __device__ __forceinline__ int run_ml_at(uint32_t slot, int lr) const { return ml_at(slot + 2 * p.places, lr); }
    __device__ __forceinline__ int o_at(uint32_t slot, int lr, int dv) const {
        return (int)(((slot * 16 * CT + lr) * (uint32_t)p.a.c.hd + dv) * 4);
    }
    __device__ __forceinline__ int ml_at(uint32_t slot, int lr) const {
        return (int)((const char*)p.part_ml - (const char*)p.part_o) + (int)(slot * 16 * CT + lr) * 8;
    }
    __device__ __forceinline__ f32x2v ml(int at) const {
        return __builtin_bit_cast(f32x2v, __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, SHARED ? kCoherent : 0));
    }
    __device__ __forceinline__ f32x4 o(uint32_t slot, int lr, int dv) const {
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o_at(slot, lr, dv), 0, SHARED ? kCoherent : 0));
    }
    __device__ __forceinline__ void store(uint32_t slot, int lr, int dv, const PagedSum& s, bool piece) const {
        const u32x2 w = __builtin_bit_cast(u32x2, f32x2v{s.m, s.l});
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s.o), rs, o_at(slot, lr, dv), 0, kCoherent);
        if (dv == 0) __builtin_amdgcn_raw_buffer_store_b64(w, rs, run_ml_at(slot, lr), 0, kCoherent);   // a run of one piece
        if (dv == 0 && piece) __builtin_amdgcn_raw_buffer_store_b64(w, rs, ml_at(slot, lr), 0, kCoherent);
    }
    // Joins pieces i0 .. i1 - 1 in order, eight on their way together. Past the last piece it is read again, and masked: a
    // weight of 0 would make NaN of an infinite sum, and a branch lets the loads sink to their uses.
    __device__ __forceinline__ PagedSum run(uint32_t first, uint32_t i0, uint32_t i1, int lr, int dv) const {
        PagedSum s;
        constexpr uint32_t U = 8;
        for (uint32_t i = i0; i < i1; i += U) {
            f32x2v w[U];
            f32x4 os[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) w[u] = ml(ml_at(paged_slot(first, min(i + u, i1 - 1)), lr));
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) os[u] = o(paged_slot(first, min(i + u, i1 - 1)), lr, dv);
            __builtin_amdgcn_sched_barrier(0);
            float mn = s.m;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                if (i + u >= i1) w[u][0] = -INFINITY;
                mn = fmaxf(mn, w[u][0]);
            }
            s.raise(mn);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const u32x4 kept = __builtin_bit_cast(u32x4, os[u]) & (i + u < i1 ? ~0u : 0u);
                s.add(w[u][0], w[u][1], __builtin_bit_cast(f32x4, kept));
            }
        }
        return s;
    }
    // Joins the results of runs, kept where each run's first piece was.
    __device__ __forceinline__ PagedSum runs(uint32_t first, const PagedRuns& r, int lr, int dv) const {
        PagedSum s;
        constexpr uint32_t U = 8;
        for (uint32_t i = 0; i < r.n; i += U) {
            f32x2v w[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) w[u] = ml(run_ml_at(paged_slot(first, r.at(min(i + u, r.n - 1))), lr));
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) s.m = fmaxf(s.m, w[u][0]);
        }
        for (uint32_t i = 0; i < r.n; i += U) {
            f32x2v w[U];
            f32x4 os[U];
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                const uint32_t slot = paged_slot(first, r.at(min(i + u, r.n - 1)));
                w[u] = ml(run_ml_at(slot, lr));
                os[u] = o(slot, lr, dv);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                if (i + u < r.n) s.add(w[u][0], w[u][1], os[u]);
        }
        return s;
    }
};

// Joins `n` runs whose results lie in LDS, `step` apart.
__device__ __forceinline__ PagedSum paged_runs_lds(const f32x4* o, const f32x2v* ml, uint32_t n, uint32_t step) {
    PagedSum s;
    constexpr uint32_t U = 8;   // read together
    for (uint32_t i = 0; i < n; i += U) {
        f32x2v w[U];
        f32x4 os[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t k = min(i + u, n - 1) * step;
            w[u] = ml[k];
            os[u] = o[k];
        }
        float mn = s.m;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) mn = fmaxf(mn, w[u][0]);
        s.raise(mn);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
            if (i + u < n) s.add(w[u][0], w[u][1], os[u]);
    }
    return s;
}

// This workgroup has stored a piece: whether it is the last of the `n` that count on cnt, which is then zero again.
__device__ __forceinline__ bool paged_last(unsigned* cnt, uint32_t n, int* flag) {
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's partials are in memory
    __syncthreads();
    if (threadIdx.x == 0) {
        *flag = atomicAdd_system(cnt, 1u) + 1 == n;
        if (*flag) atomicExch_system(cnt, 0u);
    }
    __syncthreads();
    return *flag;
}

constexpr int PM_JOIN_BYTES = 256 * 24;   // of LDS that paged_join uses

// After a workgroup of 256 threads has stored its piece i of a segment: the last one joins.
template <int DT, int CT>
__device__ __forceinline__ void paged_join(const PagedMfmaArgs& p, int item, int hk, uint32_t first, uint32_t pieces, uint32_t i,
                                           char* lds, int* flag) {
    const PagedParts<CT, true> parts(p);
    const int tid = threadIdx.x, b = (int)div32((uint32_t)item, p.nrb), r0 = (item - b * (int)p.nrb.d) * 16 * CT;
    const int quads = p.a.c.hd / 4, all = min(16 * CT, p.rows - r0) * quads;
    const PagedRuns r = paged_runs(pieces, all);
    unsigned* cnt = p.count + (((int64_t)item * p.a.c.kvh + hk) << p.spread);
    if (r.apart) {
        const uint32_t run = r.of(i), i0 = r.at(run), i1 = r.at(run + 1), slot = paged_slot(first, i0);
        if (i1 - i0 > 1) {
            if (!paged_last(p.count + ((int64_t)p.items * p.a.c.kvh << p.spread) + slot, i1 - i0, flag)) return;
            for (int c = tid; c < all; c += 256) {
                const int lr = c / quads, dv = (c - lr * quads) * 4;
                parts.store(slot, lr, dv, parts.run(first, i0, i1, lr, dv), false);
            }
        }
        if (!paged_last(cnt, r.n, flag)) return;
        for (int c = tid; c < all; c += 256) {
            const int lr = c / quads, dv = (c - lr * quads) * 4;
            const PagedSum s = parts.runs(first, r, lr, dv);
            PagedRow(p, b, hk, r0 + lr, s.m, s.l).template store<DT>(p, dv, s.o);
        }
        return;
    }
    if (!paged_last(cnt, pieces, flag)) return;
    if (r.n == 1) {
        for (int c = tid; c < all; c += 256) {
            const int lr = c / quads, dv = (c - lr * quads) * 4;
            const PagedSum s = parts.run(first, 0, pieces, lr, dv);
            PagedRow(p, b, hk, r0 + lr, s.m, s.l).template store<DT>(p, dv, s.o);
        }
        return;
    }
    f32x4* o = reinterpret_cast<f32x4*>(lds);
    f32x2v* ml = reinterpret_cast<f32x2v*>(lds + 256 * 16);
    const uint32_t run = tid / all, c = tid - run * all;
    const int lr = c / quads, dv = (c - lr * quads) * 4;
    if (run < r.n) {
        const PagedSum s = parts.run(first, r.at(run), r.at(run + 1), lr, dv);
        o[tid] = s.o;
        ml[tid] = f32x2v{s.m, s.l};
    }
    __syncthreads();
    if (run) return;
    const PagedSum s = paged_runs_lds(o + c, ml + c, r.n, all);
    PagedRow(p, b, hk, r0 + lr, s.m, s.l).template store<DT>(p, dv, s.o);
}

// ---------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------

// The kernel's one argument, read again from where it was passed: values that only a piece's start or end needs would
// otherwise be held in scalar registers across the loop over keys, which they overflow.
__device__ __forceinline__ const PagedMfmaArgs& paged_args() {
    auto* k = (const __attribute__((address_space(4))) PagedMfmaArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    return *(const PagedMfmaArgs*)k;
}

template <int W>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[W]) {
    if constexpr (W == 1) w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (W == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        w[0] = x[0];
        w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = x[j];
        }
    }
}

// Two of a word's four e4m3 values as a packed pair of DT: exact, e4m3 has 3 bits after the leading one and exponents
// from 2^-9.
template <int DT>
__device__ __forceinline__ uint32_t widen8(uint32_t w, bool hi) {
    if constexpr (DT == TVK_F16)
        return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    else
        return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}

// Bits of the keys k0 .. k0 + 31 that lie in [lo, hi).
__device__ __forceinline__ uint32_t key_bits(int k0, int lo, int hi) {
    const int n = min(max(hi - k0, 0), 32), f = min(max(lo - k0, 0), 32);
    return (n == 32 ? ~0u : (1u << n) - 1) & (f == 32 ? 0u : ~0u << f);
}

// FAST: the page size is a multiple of 16, so that a half tile lies in one page and its address is the wave's, not a
// lane's, and rows fill their KL chunks of 64 bytes. WAVES 1: a wave a segment, for short sequences.
template <int DT, bool F8, int D, int CT, bool FAST, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (PagedTile<DT, F8, D>::occ(CT))) void paged_attn_mfma_kernel(PagedMfmaArgs) {
    typedef PagedTile<DT, F8, D> G;
    constexpr bool F32 = DT == TVK_F32;
    constexpr int NB = G::NB, BN = G::BN, KL = G::KL, QS = G::QS, EV = G::EV, DV = G::DV, VW = G::VW, ES = G::ES;
    constexpr int COLS = 16 * CT, LDO = DV + 4;
    constexpr int RED = WAVES == 1 ? 16 * DV : WAVES * COLS * LDO;
    __shared__ __attribute__((aligned(16))) float red[RED];
    __shared__ float ml[2][WAVES][COLS];
    __shared__ int flag;
    static_assert(WAVES == 1 || (sizeof(red) >= PM_JOIN_BYTES && WAVES == 4), "the join of pieces reuses the waves'");
    __shared__ int has_marks;
    __shared__ uint32_t marks[CT * DV];   // two bits for each row and column: the infinities (1, 2) it takes in, both for NaN
    const int tid = threadIdx.x, lane = tid % 64, wave = WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid / 64);
    const int g = lane / 16, c16 = lane % 16;
    uint32_t wg = blockIdx.x;
    PagedDeal deal{31, 0, 0, 0, 0};
    PagedPiece pc, part[2];   // part: pieces of segments that others share, the one that begins its segment second
    int parts = 0;
    uint32_t at = 0, x = wg, stop = 0, begin = 0;
    const bool dealt = WAVES > 1 && paged_args().plan.wgs;
    if (!dealt) {
        const PagedMfmaArgs& p = paged_args();
        // the heads of an item on one XCD, as long as there are items for all of them
        const uint32_t grouped = p.plan.shared ? (uint32_t)p.items / 8 * 8 * p.kvh.d : 0;
        const uint32_t of = wg < grouped ? wg / 8 : wg, n = div32(of, p.kvh);
        pc.item = (int)(wg < grouped ? 8 * n + wg % 8 : n);
        pc.hk = (int)(of - n * p.kvh.d);
    } else {
        const PagedMfmaArgs& p = paged_args();
        const uint32_t mine = lane < p.items ? (uint32_t)paged_span<BN, CT>(p, lane).tiles : 0;
        deal = paged_deal_of<BN, CT>(p, lane, mine);
        // a stretch of neighbours' work for each XCD
        if (p.plan.shared && wg < deal.used / 8 * 8) wg = wg % 8 * (deal.used / 8) + wg / 8;
        if (!paged_start(deal, wg, x, stop) || !paged_locate<BN, CT>(p, deal, x, lane, mine, pc.item, at, begin)) return;
    }

    for (bool more_pieces = true; more_pieces;) {
        if (WAVES > 1) __syncthreads();   // the piece before has been merged
        const PagedMfmaArgs& p = paged_args();
        const PagedAttnArgs& a = p.a;
        const bool several = a.new_tokens > 1;
        if (several) {
            for (int i = tid; i < CT * DV; i += 64 * WAVES) marks[i] = 0;
            if (tid == 0) has_marks = 0;
            if (WAVES > 1) __syncthreads();
        }
        const PagedSpan sp = paged_span<BN, CT>(p, pc.item);
        const uint32_t tiles = (uint32_t)sp.tiles;
        more_pieces = false;
        pc.c0 = 0;
        pc.c1 = tiles;
        pc.pieces = 1;
        if (dealt) {
            const uint32_t units = deal.units(tiles);
            pc.hk = (int)wave_div(at, units);
            at -= (uint32_t)pc.hk * units;   // of the segment
            if (deal.shift >= 0) {
                paged_chunk(p.plan, deal, x, begin + (uint32_t)pc.hk * tiles, at, tiles, units, wave_rcp((float)units), pc);
            } else {
                paged_stretch(deal, wg, x, at, tiles, stop, wave_rcp((float)deal.per), pc);
                // the next segment: the item's next head, or the next item's first
                x += tiles - at;
                more_pieces = x < stop;
                at = (uint32_t)(pc.hk + 1) * tiles;
            }
        }
        const int item = pc.item;
        if (more_pieces && pc.hk + 1 == (int)p.kvh.d) {
            ++pc.item;
            at = 0;
        }
        if (pc.c0 >= pc.c1) continue;
        const int b = sp.b, hk = pc.hk, r0 = (item - b * (int)p.nrb.d) * COLS;

        // ---- queries: scores in log2 units are c2 * q.k, with q's signs turned where c2 would be negative
        const float cs = a.scale * (F8 && a.c.k_scale ? a.c.k_scale[hk] : 1.0f) * AT_LOG2E;
        const float c2 = cs < 0.0f ? -cs : cs;
        u32x4 qf[CT][QS];
        int last_c[CT];   // keys below it are seen by the column's row
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int r = min(r0 + 16 * ct + c16, p.rows - 1);   // columns past the rows repeat the last one, unused
            const int t = (int)div32((uint32_t)r, p.group), h = hk * (int)p.group.d + (r - t * (int)p.group.d);
            last_c[ct] = t < sp.pad ? 0 : sp.len - a.new_tokens + t + 1;
            constexpr int QES = F32 ? 4 : 2;
            const char* Q = static_cast<const char*>(a.q) +
                            ((int64_t)b * a.sq[0] + (int64_t)t * a.sq[1] + (int64_t)h * a.sq[2]) * QES;
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                // the first value of the fragment that K's chunk s (8-bit: half a chunk) meets
                const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : (64 * s + 16 * g) / ES;
                qf[ct][s] = FAST || d < a.c.hd ? *reinterpret_cast<const u32x4*>(Q + d * QES) : u32x4{0, 0, 0, 0};
            }
        }
        if (__builtin_expect(cs < 0.0f, 0)) {
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                for (int s = 0; s < QS; ++s) qf[ct][s] ^= F32 ? 0x80000000u : 0x80008000u;
        }

        f32x4 oacc[EV][CT];
        float m_run[CT], l_run[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
            for (int i = 0; i < EV; ++i) oacc[i][ct] = f32x4{0, 0, 0, 0};
            m_run[ct] = -INFINITY;
            l_run[ct] = 0.0f;
        }

        // ---- where a tile's keys are
        // lane offsets, in bytes, of a row's chunks and values
        const uint32_t krow = p.ks * 16, vrow = p.vs * 16;
        const uint32_t kbytes = (uint32_t)a.c.hd * ES;
        uint32_t kcol[FAST ? 1 : KL];   // chunks past the row are its last one, and zeros when it comes to the product
        if constexpr (FAST) kcol[0] = c16 * krow + 16 * g;
        else
#pragma unroll
            for (int s = 0; s < KL; ++s) kcol[s] = min(16u * g + 64 * s, kbytes - 16);
        // columns past the head dim are not stored
        const uint32_t vcol = EV * c16 < a.c.hd ? EV * ES * c16 : 0;
        uint32_t vfast[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) vfast[r] = (4 * g + r) * vrow + vcol;

        typedef const __attribute__((address_space(4))) int32_t* table_ptr;   // scalar loads: no store of a kernel goes there
        const int32_t* trow = a.c.table + (int64_t)b * a.c.table_stride;
        const char* Kh = static_cast<const char*>(a.c.k) + (int64_t)hk * a.c.sk[2] * ES;
        const char* Vh = static_cast<const char*>(a.c.v) + (int64_t)hk * a.c.sv[2] * ES;
        constexpr uint32_t ALL = BN == 32 ? ~0u : (1u << BN) - 1;
        constexpr int NE = FAST ? NB : 1;
        uint32_t entry[NE], slot[NE];      // of the tile after next: table entries on their way
        const char* kbase[NB];             // FAST: a block's first row
        const char* vbase[NB];
        uint32_t koff = 0, voff = 0;       // else: lane j's for key j % BN, in 16 bytes
        uint32_t ok = 0;                   // keys that have a page
        const uint32_t kp = p.kp, ks = p.ks, vp = p.vp, vs = p.vs;
        const int reach = (int)a.c.reach - 1;
        auto fetch = [&](int t) {          // past the table its last entry is read again
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const uint32_t pos = FAST ? min(t * BN + 16 * i, reach & ~15) : min(t * BN + lane % BN, reach);
                const uint32_t n = div32(pos, a.c.page);
                slot[i] = pos - n * a.c.page.d;
                if constexpr (FAST) entry[i] = (uint32_t)((table_ptr)(uintptr_t)trow)[n];
                else entry[i] = (uint32_t)trow[n];
            }
        };
        auto resolve = [&]() {   // keys without a page read page 0 and are masked
            uint32_t page[NE];
#pragma unroll
            for (int i = 0; i < NE; ++i) page[i] = entry[i] < a.c.pages ? entry[i] : 0;
            if constexpr (FAST) {
                ok = 0;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    ok |= entry[i] < a.c.pages ? 0xffffu << (16 * i) : 0u;
                    kbase[i] = Kh + (uint64_t)(page[i] * kp + slot[i] * ks) * 16;
                    vbase[i] = Vh + (uint64_t)(page[i] * vp + slot[i] * vs) * 16;
                }
            } else {
                ok = (uint32_t)__ballot(entry[0] < a.c.pages) & ALL;
                koff = page[0] * kp + slot[0] * ks;
                voff = page[0] * vp + slot[0] * vs;
            }
        };
        u32x4 kr[NB][KL];
        uint32_t vr[4 * NB][VW];
        auto load_k = [&]() {
#pragma unroll
            for (int kb = 0; kb < NB; ++kb) {
                const char* row = Kh;
                if constexpr (!FAST) row += (uint64_t)__shfl(koff, 16 * kb + c16) * 16;
#pragma unroll
                for (int s = 0; s < KL; ++s)
                    kr[kb][s] = *reinterpret_cast<const u32x4*>(FAST ? kbase[kb] + kcol[0] + 64 * s : row + kcol[FAST ? 0 : s]);
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < 4 * NB; ++j) {
                if constexpr (FAST) load_words<VW>(vbase[j / 4] + vfast[j % 4], vr[j]);
                else load_words<VW>(Vh + (uint64_t)__shfl(voff, 16 * (j / 4) + 4 * g + j % 4) * 16 + vcol, vr[j]);
            }
        };

        int t = 0;
        auto next_k = [&]() {
            resolve();
            fetch(t + 2 * WAVES);
            load_k();
        };

        const int tile0 = sp.lo / BN;
        const int end = sp.hi > sp.lo ? tile0 + (int)pc.c1 : 0;
        // keys that every row of the block sees
        const int all_lo = window_lo(sp.hi, a.window);
        const int all_hi = sp.t0 < sp.pad ? 0 : sp.len - a.new_tokens + sp.t0 + 1;
        t = tile0 + (int)pc.c0 + wave;
        if (t < end) {
            fetch(t);
            resolve();
            load_k();
            load_v();
            fetch(t + WAVES);
        }
        for (; t < end; t += WAVES) {
            const int k0 = t * BN;
            const uint32_t keys = ok & key_bits(k0, sp.lo, sp.hi);
            const bool plain = keys == ALL && k0 >= all_lo && k0 + BN <= all_hi;
            const bool more = t + WAVES < end;
            // ---- S^T = K Q^T
            if constexpr (!FAST) {
#pragma unroll
                for (int s = 0; s < KL; ++s)
#pragma unroll
                    for (int kb = 0; kb < NB; ++kb)
                        if (16 * g + 64 * s >= (int)kbytes) kr[kb][s] = u32x4{0, 0, 0, 0};
            }
            f32x4 sacc[NB][CT];
#pragma unroll
            for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) sacc[kb][ct] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KL; ++s)
#pragma unroll
                for (int kb = 0; kb < NB; ++kb) {
                    const u32x4 kv = kr[kb][s];
                    if constexpr (F32) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int ct = 0; ct < CT; ++ct)
                                sacc[kb][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __builtin_bit_cast(float, (uint32_t)kv[i]), __builtin_bit_cast(float, (uint32_t)qf[ct][s][i]),
                                    sacc[kb][ct], 0, 0, 0);
                    } else if constexpr (F8) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const u32x4 w = u32x4{widen8<DT>(kv[2 * i], false), widen8<DT>(kv[2 * i], true),
                                                  widen8<DT>(kv[2 * i + 1], false), widen8<DT>(kv[2 * i + 1], true)};
#pragma unroll
                            for (int ct = 0; ct < CT; ++ct) sacc[kb][ct] = mfma16<DT>(w, qf[ct][2 * s + i], sacc[kb][ct]);
                        }
                    } else {
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) sacc[kb][ct] = mfma16<DT>(kv, qf[ct][s], sacc[kb][ct]);
                    }
                }
            // on a masked tile the next keys wait: the registers of both do not fit
            if (more && plain) next_k();
            // ---- online softmax per column
            float alpha[CT];
            bool rescale = false;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                float tmax = -INFINITY;
                if (!plain) {
                    const uint32_t mine = (keys & key_bits(k0, window_lo(last_c[ct], a.window), last_c[ct])) >> (4 * g);
#pragma unroll
                    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sacc[kb][ct][r] = (mine >> (16 * kb + r)) & 1 ? sacc[kb][ct][r] * c2 : -INFINITY;
                }
#pragma unroll
                for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) tmax = fmaxf(tmax, sacc[kb][ct][r]);
                tmax = lanes4_max(tmax);
                if (plain) tmax *= c2;
                const float m_old = m_run[ct], m_new = fmaxf(m_old, tmax);
                const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                alpha[ct] = (m_old == m_new || m_old == -INFINITY) ? 1.0f : __builtin_amdgcn_exp2f(m_old - m_use);
                rescale = rescale || alpha[ct] != 1.0f;
                float rsum = 0.0f;
#pragma unroll
                for (int kb = 0; kb < NB; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = __builtin_amdgcn_exp2f(plain ? __builtin_fmaf(sacc[kb][ct][r], c2, -m_use) : sacc[kb][ct][r] - m_use);
                        sacc[kb][ct][r] = e;
                        rsum += e;
                    }
                l_run[ct] = l_run[ct] * alpha[ct] + rsum;
                m_run[ct] = m_new;
            }
            if (__any(rescale)) {
#pragma unroll
                for (int i = 0; i < EV; ++i)
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
                        for (int r = 0; r < 4; ++r) oacc[i][ct][r] *= alpha[ct];
            }
            // ---- O^T += V^T P^T
            // values of keys that no row sees may be anything: zeros
            if (!plain) {
#pragma unroll
                for (int j = 0; j < 4 * NB; ++j)
#pragma unroll
                    for (int w = 0; w < VW; ++w) vr[j][w] = (keys >> (4 * g + 16 * (j / 4) + j % 4)) & 1 ? vr[j][w] : 0u;
            }
            // Keys that some rows see and others do not, with values that are not finite: a probability of zero must not
            // meet them. They are marked for the rows that see them, and zeros in the product.
            if (__builtin_expect(!plain && several, 0)) {
                typedef typename std::conditional<F8, uint8_t, typename std::conditional<F32, uint32_t, uint16_t>::type>::type U;
                // a value's bits that are all set in infinities and NaN (8 bits: in NaN alone)
                constexpr uint32_t top = F8 ? 0x7fu : F32 ? 0x7f800000u : DT == TVK_F16 ? 0x7c00u : 0x7f80u;
                constexpr uint32_t sign = F8 ? 0x80u : F32 ? 0x80000000u : 0x8000u;
                constexpr int PER = 4 / ES;   // values in a word
                // any value's such bits all set, a word's values together
                bool odd;
                if constexpr (F8) {
                    uint32_t any = 0;
#pragma unroll
                    for (int j = 0; j < 4 * NB; ++j)
#pragma unroll
                        for (int w = 0; w < VW; ++w) any |= (vr[j][w] & 0x7f7f7f7fu) + 0x01010101u;
                    odd = any & 0x80808080u;
                } else {
                    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
                    u16x2 most = {0, 0};
                    uint32_t most32 = 0;
#pragma unroll
                    for (int j = 0; j < 4 * NB; ++j)
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            if constexpr (F32) most32 = max(most32, vr[j][w] & top);
                            else most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, vr[j][w] & (top | top << 16)));
                        }
                    odd = F32 ? most32 == top : most[0] == top || most[1] == top;
                }
                if (__any(odd)) {
                    if (lane == 0) has_marks = 1;
                    U* tile = reinterpret_cast<U*>(red + wave * (WAVES == 1 ? 0 : COLS * LDO));   // the wave's own: a block's values
#pragma unroll
                    for (int kb = 0; kb < NB; ++kb) {
                        __builtin_amdgcn_wave_barrier();
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int w = 0; w < VW; ++w) {
                                uint32_t& v = vr[4 * kb + j][w];
                                reinterpret_cast<uint32_t*>(tile)[((4 * g + j) * 16 + c16) * VW + w] = v;
#pragma unroll
                                for (int i = 0; i < PER; ++i)
                                    if ((v >> (8 * ES * i) & top) == top) v &= ~((top | sign) << (8 * ES * i));
                            }
                        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                        for (int i = lane; i < 16 * DV; i += 64) {
                            const int key = 16 * kb + i / DV, dv = i % DV;
                            const uint32_t v = tile[i];
                            if ((v & top) != top) continue;
                            const uint32_t mark = F8 || (v & ~sign) != top ? 3u : v & sign ? 2u : 1u;
#pragma unroll 1
                            for (int col = 0; col < COLS; ++col) {
                                const int tok = (int)div32((uint32_t)min(r0 + col, p.rows - 1), p.group);
                                const int hi = tok < sp.pad ? 0 : sp.len - a.new_tokens + tok + 1;
                                if ((keys & key_bits(k0, window_lo(hi, a.window), hi)) >> key & 1) atomicOr(&marks[(col * DV + dv) / 16], mark << 2 * (dv % 16));
                            }
                        }
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 4 * NB; ++j)
#pragma unroll
                    for (int i = 0; i < EV; ++i)
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct)
                            oacc[i][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[j][i]),
                                                                               sacc[j / 4][ct][j % 4], oacc[i][ct], 0, 0, 0);
            } else {
                u32x4 pf[CT];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const f32x4 y = sacc[0][ct], z = sacc[NB - 1][ct];
                    pf[ct] = u32x4{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]), pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3])};
                }
#pragma unroll
                for (int w = 0; w < EV / 2; ++w) {
                    uint32_t two[8];   // values 2w, 2w + 1 of the lane's eight keys
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if constexpr (F8) two[j] = widen8<DT>(vr[j % (4 * NB)][w / 2], w % 2);
                        else two[j] = vr[j % (4 * NB)][w % VW];
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t sel = i ? 0x07060302u : 0x05040100u;
                        const u32x4 vf = u32x4{__builtin_amdgcn_perm(two[1], two[0], sel), __builtin_amdgcn_perm(two[3], two[2], sel),
                                               __builtin_amdgcn_perm(two[5], two[4], sel), __builtin_amdgcn_perm(two[7], two[6], sel)};
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) oacc[2 * w + i][ct] = mfma16<DT>(vf, pf[ct], oacc[2 * w + i][ct]);
                    }
                }
            }
            if (more) {
                if (!plain) next_k();
                load_v();
            }
        }

        const PagedMfmaArgs& pe = paged_args();
        auto marked = [&](int lr, int dv, f32x4 o) {   // with the infinities and NaN that were kept out of the products
            const uint32_t mark = marks[(lr * DV + dv) / 16] >> 2 * (dv % 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t two = mark >> 2 * i & 3;
                if (two) o[i] += two == 1 ? INFINITY : two == 2 ? -INFINITY : NAN;
            }
            return o;
        };
        // a lane's values are the 4 EV columns of its row from EV * 4g on
        auto quad = [&](int ct, int j) {
            f32x4 o;
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = oacc[(4 * j + u) % EV][ct][(4 * j + u) / EV];
            return o;
        };
        if constexpr (WAVES == 1) {
            const bool mark = several && has_marks;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float l = lanes4_sum(l_run[ct]);
                const int lr = 16 * ct + c16;
                if (r0 + lr >= pe.rows) continue;
                const PagedRow row(pe, b, hk, r0 + lr, m_run[ct], l);
#pragma unroll
                for (int j = 0; j < EV; ++j) {
                    const int dv = 4 * (EV * g + j);
                    f32x4 o = quad(ct, j);
                    if ((!FAST || DV != D) && dv >= pe.a.c.hd) continue;
                    if (__builtin_expect(mark, 0)) o = marked(lr, dv, o);
                    row.template store<DT>(pe, dv, o);
                }
            }
        } else {
            // ---- merge the waves
            const bool whole = pc.pieces == 1;
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
                const float l_tot = lanes4_sum(l_run[ct]);
                if (g == 0) {
                    ml[0][wave][16 * ct + c16] = m_run[ct];
                    ml[1][wave][16 * ct + c16] = l_tot;
                }
#pragma unroll
                for (int j = 0; j < EV; ++j)
                    *reinterpret_cast<f32x4*>(&red[(wave * COLS + 16 * ct + c16) * LDO + 4 * (EV * g + j)]) = quad(ct, j);
            }
            __syncthreads();
            for (int c = tid; c < min(COLS, pe.rows - r0) * (DV / 4); c += 64 * WAVES) {
                const int lr = c / (DV / 4), dv = (c % (DV / 4)) * 4;
                if ((!FAST || DV != D) && dv >= pe.a.c.hd) continue;
                PagedSum s;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) s.m = fmaxf(s.m, ml[0][w][lr]);
#pragma unroll
                for (int w = 0; w < WAVES; ++w)
                    s.add(ml[0][w][lr], ml[1][w][lr], *reinterpret_cast<const f32x4*>(&red[(w * COLS + lr) * LDO + dv]));
                if (__builtin_expect(several && has_marks, 0)) s.o = marked(lr, dv, s.o);
                if (whole) PagedRow(pe, b, hk, r0 + lr, s.m, s.l).template store<DT>(pe, dv, s.o);
                else PagedParts<CT, true>(pe).store(paged_slot(pc.first, pc.i), lr, dv, s, true);
            }
            if (!whole && pe.count) {
                const int second = pc.c0 == 0;
                part[second] = pc;
                part[second].item = item;
                parts |= 1 << second;
            } else if (dealt && !pe.count && pc.c0 == 0 && tid == 0) {
                *reinterpret_cast<u32x2*>(pe.seg + 2 * ((int64_t)item * pe.kvh.d + hk)) = u32x2{pc.first, pc.pieces};
            }
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
            if (!(parts >> i & 1)) continue;
            const PagedPiece& q = part[0];
            const int item = i ? part[1].item : q.item, hk = i ? part[1].hk : q.hk;
            const uint32_t first = i ? part[1].first : q.first, pieces = i ? part[1].pieces : q.pieces;
            paged_join<DT, CT>(paged_args(), item, hk, first, pieces, i ? part[1].i : q.i, reinterpret_cast<char*>(red), &flag);
        }
    }
}

// The join as a launch of its own: a workgroup a segment, or one of `slices` that take its rows in turn. A row's quads of
// columns are shared by as many threads as there are, every so-manieth run to each.
constexpr int PM_JOIN_THREADS = 512;
template <int DT, int CT>
__global__ __launch_bounds__(PM_JOIN_THREADS) void paged_attn_join_kernel(PagedMfmaArgs p) {
    constexpr int RUNS = 32;   // paged_runs
    __shared__ f32x4 o[RUNS * 64];
    __shared__ f32x2v ml[RUNS * 64];
    const uint32_t slice = blockIdx.x % (uint32_t)p.slices, id = blockIdx.x / (uint32_t)p.slices;
    const uint32_t first = p.seg[2 * (int64_t)id], pieces = p.seg[2 * (int64_t)id + 1];
    if (pieces == 1) return;
    const PagedParts<CT, false> parts(p);
    const int item = (int)div32(id, p.kvh), hk = (int)(id - item * p.kvh.d);
    const int b = (int)div32((uint32_t)item, p.nrb), r0 = (item - b * (int)p.nrb.d) * 16 * CT;
    const int nr = min(16 * CT, p.rows - r0), quads = p.a.c.hd / 4, share = PM_JOIN_THREADS / quads;
    const int part = threadIdx.x / quads, c = threadIdx.x - part * quads;
    const PagedRuns r = paged_runs(pieces, nr * quads);
    for (int lr = slice; lr < nr; lr += p.slices) {
        __syncthreads();   // the row before has been read
        PagedSum s;
        for (uint32_t run = part; part < share && run < r.n; run += share) {
            s = parts.run(first, r.at(run), r.at(run + 1), lr, 4 * c);
            o[run * quads + c] = s.o;
            ml[run * quads + c] = f32x2v{s.m, s.l};
        }
        __syncthreads();
        if (part) continue;
        if (r.n > 1) s = paged_runs_lds(o + c, ml + c, r.n, quads);
        PagedRow(p, b, hk, r0 + lr, s.m, s.l).template store<DT>(p, 4 * c, s.o);
    }
}

constexpr int PM_CUS = 256;
// Quads of columns and pieces of an average segment up to which its last workgroup joins it: beyond, the second launch's
// many workgroups are faster (float16 1 x 16/4 heads, 4 tokens, 32576 keys of 128: 22 us, 28 joined by the last ones).
constexpr double PM_JOIN_ALONE = 4096;
// Values of the row blocks from which segments are whole whatever their keys (bfloat16 32/8 heads of 128, 512 new tokens of
// 4000 for 128 sequences: 9.3 ms whole, 18.4 in stretches).
constexpr double PM_WHOLE_VALUES = 0x1p28;
constexpr int PM_SPREAD = 5, PM_COUNTERS = 16384;

// False, and nothing queued, where the launch would have too many threads.
template <int DT, bool F8, int D, int CT>
bool paged_launch(PagedMfmaArgs& p, int64_t batch, hipStream_t s) {
    typedef PagedTile<DT, F8, D> G;
    const int nrb = (p.rows + 16 * CT - 1) / (16 * CT);
    p.nrb = make_div((uint32_t)nrb);
    p.kp = (uint32_t)(p.a.c.sk[0] * G::ES / 16);
    p.ks = (uint32_t)(p.a.c.sk[1] * G::ES / 16);
    p.vp = (uint32_t)(p.a.c.sv[0] * G::ES / 16);
    p.vs = (uint32_t)(p.a.c.sv[1] * G::ES / 16);
    p.kvh = make_div((uint32_t)p.a.c.kvh);
    p.group = make_div((uint32_t)p.a.group);
    p.items = (int)(batch * nrb);
    const int64_t segments = (int64_t)p.items * p.a.c.kvh;
    // Workgroups go to the XCDs in turn, and each XCD reads for itself a line that its heads share with another's.
    const auto partial = [&](const int64_t* stride) { return stride[2] * G::ES % 128 != 0; };
    p.plan.shared = p.a.c.kvh > 1 && (partial(p.a.c.sk) || partial(p.a.c.sv));
    const bool fast = p.a.c.page.d % 16 == 0 && p.a.c.hd * G::ES == G::KL * 64;
    const int64_t keys = p.a.window ? std::min<int64_t>(p.a.max_len, (int64_t)p.a.window + p.a.new_tokens + G::BN) : p.a.max_len;
    const int64_t tiles = (keys + G::BN - 1) / G::BN;   // at most, of a segment
    p.plan.resident = PM_CUS * G::occ(CT);
    if (tiles * G::BN <= 32 * (segments > p.plan.resident ? PM_WAVE_MANY : PM_WAVE)) {
        if (segments * 64 > kGridThreads) return false;
        const dim3 grid((unsigned)segments), block(64);
        if (fast) hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, true, 1>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, false, 1>), grid, block, 0, s, p);
        return true;
    }
    if (segments * 64 * PM_WAVES > kGridThreads) return false;
    Scratch scratch;
    p.plan.many = paged_many(segments, p.plan.resident);
    const int64_t wgs = paged_wgs(p.plan.many, segments, tiles, p.plan.resident);
    const bool most = (double)wgs * 16 * CT * (p.a.c.hd + 4) >= PM_WHOLE_VALUES;
    if (paged_is_dealt(p.plan.many, tiles * G::BN) && !most && segments * PM_JOIN_THREADS <= kGridThreads) {
        const int64_t places = paged_places(p.plan.many, wgs, p.plan.resident);
        const size_t rows = (size_t)2 * places * 16 * CT, bytes = rows * (p.a.c.hd + 4) * 4;
        float* part = static_cast<float*>(scratch.get(bytes + (size_t)segments * 8, s));   // (at most 2^28 bytes of partials)
        if (part) {
            p.plan.wgs = (int)wgs;
            p.places = (int)places;
            p.part_o = part;
            p.part_ml = part + rows * p.a.c.hd;
            p.part_bytes = (unsigned)bytes;
            p.seg = reinterpret_cast<uint32_t*>(p.part_ml + rows * 4);
            const double pieces = std::min((double)p.plan.resident / segments, (double)tiles / PM_WAVES);
            const double wide = std::max(1.0, pieces) * std::min(p.rows, 16 * CT) * p.a.c.hd / 4;
            p.spread = PM_SPREAD;
            while (p.spread > 0 && (segments << p.spread) + 2 * places > PM_COUNTERS) --p.spread;
            p.count = wide > PM_JOIN_ALONE ? nullptr : split_counters(s, (segments << p.spread) + 2 * places);
        } else {
            clear_error();
        }
    }
    const dim3 grid((unsigned)(p.plan.wgs ? p.plan.wgs : segments)), block(64 * PM_WAVES);
    if (fast) hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, true, PM_WAVES>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, false, PM_WAVES>), grid, block, 0, s, p);
    if (p.plan.wgs && !p.count) {
        p.slices = (int)std::min<int64_t>(std::min(p.rows, 16 * CT), std::max<int64_t>(1, 2048 / segments));
        hipLaunchKernelGGL((paged_attn_join_kernel<DT, CT>), dim3((unsigned)(segments * p.slices)), dim3(PM_JOIN_THREADS), 0, s, p);
    }
    return true;
}

template <int DT, bool F8>
bool paged_dispatch(PagedMfmaArgs& p, int64_t batch, hipStream_t s) {
    const bool two = p.rows > 16;
    const int hd = p.a.c.hd;
#define TVK_PAGED(D) (two ? paged_launch<DT, F8, D, 2>(p, batch, s) : paged_launch<DT, F8, D, 1>(p, batch, s))
    if constexpr (!F8) {   // 8-bit rows of 32 bytes would be values of half a word a lane
        if (hd <= 32) return TVK_PAGED(32);
    }
    if (hd <= 64) return TVK_PAGED(64);
    if (hd <= 96) return TVK_PAGED(96);
    if (hd <= 128) return TVK_PAGED(128);
    if constexpr (DT == TVK_F32) return paged_launch<DT, F8, 256, 1>(p, batch, s);   // two row blocks' registers would spill
    else return TVK_PAGED(256);
#undef TVK_PAGED
}

}  // namespace

// One translation unit each (paged_attention_f16.hip and its neighbours).
bool paged_attn_f16(PagedMfmaArgs& p, bool f8, int64_t batch, hipStream_t s);
bool paged_attn_bf16(PagedMfmaArgs& p, bool f8, int64_t batch, hipStream_t s);
bool paged_attn_f32(PagedMfmaArgs& p, int64_t batch, hipStream_t s);

}  // namespace tvk
