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
// Work is dealt to a fixed number of workgroups by every workgroup itself, from
// the lengths on the device: a batch's lengths are not on the host, and a launch
// sized by the longest would leave the others' workgroups idle. A segment is a
// row block of a sequence and a key/value head. Where every segment can be cut
// into chunks of at least 4 (8, 16) tiles without exceeding the workgroups, each
// takes one chunk; else all tiles of the call, in segment order, are cut into
// equal stretches, and a workgroup's stretch may end one segment and begin
// others. Its 4 waves take a stretch's tiles in turn and are merged through LDS
// in wave order. A segment that lies in one workgroup is written out; the pieces
// of another go to scratch as float32 (max, sum, O), written through to memory
// as the skinny GEMM's split_fixup does, and the last workgroup to finish merges
// them in order; without counters for the stream a second launch does. Both
// give the same bits every run.
#pragma once

#include "attention_kernels.h"
#include "paged.h"

namespace tvk {

struct PagedMfmaArgs {
    PagedAttnArgs a;
    int rows;              // new_tokens * group
    int nrb;               // row blocks of a key/value head
    int items;             // batch * nrb
    int wgs;               // workgroups the tiles are dealt to; 0: one a segment
    int out_vec;           // output rows take vector stores
    float* part_o;         // [2 * wgs][16 * CT][hd]
    float* part_ml;        // [2 * wgs][16 * CT][2]: max, sum
    unsigned part_bytes;   // of both
    unsigned* count;       // a segment's finished pieces, zero before and after the launch; NULL: a second launch merges
};

namespace {

constexpr int PM_WAVES = 4;
constexpr int PM_BN = 32;   // keys per tile

template <int DT, bool F8, int D>
struct PagedTile {
    static constexpr int ES = F8 ? 1 : DT == TVK_F32 ? 4 : 2;   // bytes of a cached value
    static constexpr int KL = (D * ES + 63) / 64;               // 16-byte K chunks a lane holds of a row
    static constexpr int QS = F8 ? 2 * KL : KL;                 // Q fragments of 16 bytes
    static constexpr int EV = D == 96 ? 8 : D / 16;             // V values a lane holds of a row
    static constexpr int DV = 16 * EV;
    static constexpr int VW = EV * ES / 4;                      // the same in 32-bit words
    // workgroups a CU by the registers: K and V tiles, Q and O, and some 100 more
    static constexpr int regs(int ct) { return 8 * KL + 8 * VW + ct * (4 * QS + 4 * EV + 8) + 100; }
    static constexpr int occ(int ct) { return regs(ct) <= 128 ? 4 : regs(ct) <= 168 ? 3 : regs(ct) <= 256 ? 2 : 1; }
};

// ---------------------------------------------------------------------------
// dealing
// ---------------------------------------------------------------------------

struct PagedSpan {
    int b, len;
    int t0, t1;   // the row block's first and last token
    int lo, hi;   // keys that some row of the block sees
    int tiles;    // at least one: a segment without keys writes its zeros
};

template <int CT>
__device__ __forceinline__ PagedSpan paged_span(const PagedMfmaArgs& p, int e) {
    PagedSpan s;
    s.b = e / p.nrb;
    const int r0 = (e - s.b * p.nrb) * 16 * CT, r1 = min(p.rows, r0 + 16 * CT) - 1;
    s.len = (int)min((uint32_t)paged_len(p.a.c, s.b), p.a.max_len);
    s.t0 = r0 / p.a.group;
    s.t1 = r1 / p.a.group;
    s.hi = max(0, s.len - p.a.new_tokens + s.t1 + 1);
    const int64_t first = (int64_t)s.len - p.a.new_tokens + s.t0 + 1 - (int64_t)p.a.window;
    s.lo = p.a.window ? (int)min((int64_t)s.hi, max((int64_t)0, first)) : 0;
    s.tiles = s.hi > s.lo ? (s.hi + PM_BN - 1) / PM_BN - s.lo / PM_BN : 1;
    return s;
}

struct PagedDeal {
    uint32_t chunk;   // tiles a segment's chunks have at least; 0: stretches
    uint32_t per;     // tiles a workgroup's stretch has
    uint32_t total;   // tiles of the call
    __device__ uint32_t units(uint32_t tiles) const { return chunk ? max(1u, tiles / chunk) : tiles; }
};

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return __builtin_amdgcn_readfirstlane(v);
}

// Sums stay below 2^31 (paged_attn_mfma).
template <int CT>
__device__ __forceinline__ PagedDeal paged_deal(const PagedMfmaArgs& p, int lane) {
    PagedDeal d{0x7fffffff, 0, 0};
    if (!p.wgs) return d;
    uint32_t n = 0, n4 = 0, n8 = 0, n16 = 0;
    for (int e = lane; e < p.items; e += 64) {
        const uint32_t t = (uint32_t)paged_span<CT>(p, e).tiles;
        n += t;
        n4 += max(1u, t / 4);
        n8 += max(1u, t / 8);
        n16 += max(1u, t / 16);
    }
    const uint32_t most = (uint32_t)p.wgs / (uint32_t)p.a.c.kvh;
    n4 = wave_sum(n4);
    n8 = wave_sum(n8);
    n16 = wave_sum(n16);
    d.total = wave_sum(n) * (uint32_t)p.a.c.kvh;
    d.chunk = n4 <= most ? 4 : n8 <= most ? 8 : n16 <= most ? 16 : 0;
    d.per = (d.total + (uint32_t)p.wgs - 1) / (uint32_t)p.wgs;
    return d;
}

// Units of the items before `stop` (all of a wave's lanes take part).
template <int CT>
__device__ __forceinline__ uint32_t paged_before(const PagedMfmaArgs& p, const PagedDeal& d, int stop, int lane) {
    uint32_t n = 0;
    for (int e = lane; e < stop; e += 64) n += d.units((uint32_t)paged_span<CT>(p, e).tiles);
    return wave_sum(n);
}

// The item that holds unit x of the call, and the unit's place among the item's; false past the last.
template <int CT>
__device__ __forceinline__ bool paged_locate(const PagedMfmaArgs& p, const PagedDeal& d, uint32_t x, int lane, int& item, uint32_t& at) {
    uint32_t base = 0;
    for (int e0 = 0; e0 < p.items; e0 += 64) {
        const int e = e0 + lane;
        const uint32_t n = e < p.items ? d.units((uint32_t)paged_span<CT>(p, e).tiles) * (uint32_t)p.a.c.kvh : 0;
        uint32_t s = n;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint32_t o = __shfl_up(s, m);
            s += lane >= m ? o : 0;
        }
        s += base;
        const uint64_t past = __ballot(s > x);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            item = e0 + l;
            at = x - (uint32_t)__builtin_amdgcn_readlane((int)(s - n), l);
            return true;
        }
        base = (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
    }
    return false;
}

// A stretch of a segment's tiles, [c0, c1), and the workgroups whose pieces make up the segment.
struct PagedPiece {
    int item, hk;
    uint32_t c0, c1;
    uint32_t first, pieces;
};

__device__ __forceinline__ void paged_pieces(const PagedDeal& d, uint32_t begin, uint32_t tiles, PagedPiece& pc) {
    pc.first = begin / d.per;
    pc.pieces = (begin + tiles - 1) / d.per - pc.first + 1;
}

// Where a segment's piece i is kept: a workgroup has at most one piece that does not begin its segment and one that does
// and does not end it.
__device__ __forceinline__ uint32_t paged_slot(uint32_t first, uint32_t i) { return 2 * (first + i) + (i == 0); }

// ---------------------------------------------------------------------------
// partials and outputs
// ---------------------------------------------------------------------------

template <int DT>
__device__ __forceinline__ void paged_store(const PagedMfmaArgs& p, int64_t off, f32x4 o) {
    if constexpr (DT == TVK_F32) {
        float* op = static_cast<float*>(p.a.out) + off;
        if (p.out_vec) *reinterpret_cast<f32x4*>(op) = o;
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) op[i] = o[i];
    } else {
        uint16_t* op = static_cast<uint16_t*>(p.a.out) + off;
        if (p.out_vec) *reinterpret_cast<u32x2*>(op) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) op[i] = __builtin_bit_cast(uint16_t, elem<DT>::from_f32(o[i]));
    }
}

// Columns dv .. dv + 3 of query row r of (b, hk), from its softmax's max, sum and products.
template <int DT>
__device__ __forceinline__ void paged_finish(const PagedMfmaArgs& p, int b, int hk, int r, int dv, float m, float l, f32x4 o) {
    const int t = r / p.a.group, h = hk * p.a.group + (r - t * p.a.group);
    // a NaN sum is a NaN row; only a row without keys is zeros
    const bool none = l == 0.0f;
    const float f = p.a.c.v_scale ? p.a.c.v_scale[hk] / l : 1.0f / l;
    paged_store<DT>(p, (int64_t)b * p.a.so[0] + (int64_t)t * p.a.so[1] + (int64_t)h * p.a.so[2] + dv,
                    none ? f32x4{0, 0, 0, 0} : f32x4{o[0] * f, o[1] * f, o[2] * f, o[3] * f});
    if (dv == 0 && p.a.lse)
        p.a.lse[(int64_t)b * p.a.sl[0] + (int64_t)t * p.a.sl[1] + (int64_t)h * p.a.sl[2]] =
            none ? INFINITY : m * AT_LN2 + logf(l);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t paged_rsrc(const PagedMfmaArgs& p) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p.part_o, 0, (int)p.part_bytes, 0x00020000);
}
// Byte offsets of the partials: below 2 GiB (paged_attn_mfma).
__device__ __forceinline__ int paged_o_at(const PagedMfmaArgs& p, uint32_t row, int dv) { return (int)((row * (uint32_t)p.a.c.hd + dv) * 4); }
__device__ __forceinline__ int paged_ml_at(const PagedMfmaArgs& p, uint32_t row) {
    return (int)((const char*)(p.part_ml + (int64_t)row * 2) - (const char*)p.part_o);
}

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

constexpr int PM_MERGE_BYTES = 64 * PM_WAVES * 24;   // of LDS that paged_merge uses

// Merges a segment's pieces in order and writes its rows. Where the rows' quads of columns are few, each is shared by
// several threads, a run of pieces to each, whose sums are then joined through LDS in order.
template <int DT, int CT>
__device__ __forceinline__ void paged_merge(const PagedMfmaArgs& p, int item, int hk, uint32_t first, uint32_t pieces, char* lds) {
    const __amdgpu_buffer_rsrc_t rs = paged_rsrc(p);
    const int tid = threadIdx.x, b = item / p.nrb, r0 = (item - b * p.nrb) * 16 * CT;
    const int nr = min(16 * CT, p.rows - r0), quads = p.a.c.hd / 4, all = nr * quads;
    const int share = all <= 128 && pieces >= 8 ? (int)min(64u * PM_WAVES / (uint32_t)all, pieces / 4) : 1;
    auto sum = [&](int row, int dv, uint32_t i0, uint32_t i1) __attribute__((always_inline)) {
        PagedSum s;
        constexpr uint32_t U = 8;
        for (uint32_t i = i0; i < i1; i += U) {
            u32x2 w[U];
            u32x4 os[U];
            // past the last piece it is read again, and its max and sums masked: a weight of 0 would make NaN of an
            // infinite sum, and a branch lets the loads sink to their uses
            auto at = [&](uint32_t u) { return paged_slot(first, min(i + u, i1 - 1)) * 16 * CT + row; };
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                w[u] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, paged_ml_at(p, at(u)), 0, kCoherent));
#pragma unroll
            for (uint32_t u = 0; u < U; ++u)
                os[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, paged_o_at(p, at(u), dv), 0, kCoherent));
            __builtin_amdgcn_sched_barrier(0);
            float mn = s.m;
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                if (i + u >= i1) w[u][0] = 0xff800000u;
                mn = fmaxf(mn, __builtin_bit_cast(float, (uint32_t)w[u][0]));
            }
            s.raise(mn);
#pragma unroll
            for (uint32_t u = 0; u < U; ++u) {
                os[u] = os[u] & (i + u < i1 ? ~0u : 0u);
                s.add(__builtin_bit_cast(float, (uint32_t)w[u][0]), __builtin_bit_cast(float, (uint32_t)w[u][1]),
                      __builtin_bit_cast(f32x4, os[u]));
            }
        }
        return s;
    };
    if (share == 1) {
        for (int c = tid; c < all; c += 64 * PM_WAVES) {
            const int row = c / quads, dv = (c - row * quads) * 4;
            const PagedSum s = sum(row, dv, 0, pieces);
            paged_finish<DT>(p, b, hk, r0 + row, dv, s.m, s.l, s.o);
        }
        return;
    }
    f32x4* po = reinterpret_cast<f32x4*>(lds);
    float* pm = reinterpret_cast<float*>(lds + 64 * PM_WAVES * 16);
    float* pl = pm + 64 * PM_WAVES;
    const int part = tid / all, c = tid - part * all, row = c / quads, dv = (c - row * quads) * 4;
    if (part < share) {
        const PagedSum s = sum(row, dv, pieces * part / share, pieces * (part + 1) / share);
        po[tid] = s.o;
        pm[tid] = s.m;
        pl[tid] = s.l;
    }
    __syncthreads();
    if (part) return;
    PagedSum s;
    for (int i = 0; i < share; ++i) s.m = fmaxf(s.m, pm[i * all + c]);
    for (int i = 0; i < share; ++i) s.add(pm[i * all + c], pl[i * all + c], po[i * all + c]);
    paged_finish<DT>(p, b, hk, r0 + row, dv, s.m, s.l, s.o);
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

// Bits i of a mask spread over the halves of a word.
__device__ __forceinline__ uint32_t half_bits(uint32_t m, int lo, int hi) {
    return ((m >> lo) & 1 ? 0xffffu : 0u) | ((m >> hi) & 1 ? 0xffff0000u : 0u);
}

// Bits of the keys k0 .. k0 + 31 that lie in [lo, hi).
__device__ __forceinline__ uint32_t key_bits(int k0, int lo, int hi) {
    const int n = min(max(hi - k0, 0), 32), f = min(max(lo - k0, 0), 32);
    return (n == 32 ? ~0u : (1u << n) - 1) & (f == 32 ? 0u : ~0u << f);
}

// FAST: the page size is a multiple of 16, so that a half tile lies in one page and its address is the wave's, not a
// lane's, and rows fill their KL chunks of 64 bytes.
template <int DT, bool F8, int D, int CT, bool FAST>
__global__ __launch_bounds__(64 * PM_WAVES, (PagedTile<DT, F8, D>::occ(CT))) void paged_attn_mfma_kernel(PagedMfmaArgs) {
    typedef PagedTile<DT, F8, D> G;
    constexpr bool F32 = DT == TVK_F32;
    constexpr int KL = G::KL, QS = G::QS, EV = G::EV, DV = G::DV, VW = G::VW, ES = G::ES;
    constexpr int LDO = DV + 4;
    __shared__ __attribute__((aligned(16))) float red[PM_WAVES * 16 * LDO];
    __shared__ float ml[2][PM_WAVES][16 * CT];
    __shared__ int last;
    static_assert(sizeof(red) >= PM_MERGE_BYTES, "the merge of pieces reuses the waves'");

    __shared__ uint32_t marks[CT * DV];   // two bits for each row and column: the infinities (1, 2) it takes in, both for NaN
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int g = lane / 16, c16 = lane % 16;
    const uint32_t wg = blockIdx.x;
    const PagedDeal deal = paged_deal<CT>(paged_args(), lane);
    PagedPiece pc;
    uint32_t at;
    uint32_t x = deal.chunk ? wg : wg * deal.per;
    if (!paged_locate<CT>(paged_args(), deal, x, lane, pc.item, at)) return;
    const uint32_t stop = deal.chunk ? x + 1 : min(deal.total, x + deal.per);

    for (bool more_pieces = true; more_pieces;) {
        __syncthreads();   // the piece before has been merged
        const PagedMfmaArgs& p = paged_args();
        const PagedAttnArgs& a = p.a;
        const bool several = a.new_tokens > 1;
        if (several) {
            for (int i = tid; i < CT * DV; i += 64 * PM_WAVES) marks[i] = 0;
            __syncthreads();
        }
        const PagedSpan sp = paged_span<CT>(p, pc.item);
        const uint32_t units = deal.units((uint32_t)sp.tiles);
        pc.hk = (int)(at / units);
        at -= (uint32_t)pc.hk * units;
        if (deal.chunk) {
            pc.c0 = (uint32_t)((uint64_t)at * (uint32_t)sp.tiles / units);
            pc.c1 = (uint32_t)((uint64_t)(at + 1) * (uint32_t)sp.tiles / units);
            pc.first = x - at;
            pc.pieces = units;
            more_pieces = false;
        } else {
            pc.c0 = at;
            pc.c1 = min((uint32_t)sp.tiles, at + (stop - x));
            paged_pieces(deal, x - at, (uint32_t)sp.tiles, pc);
        }
        const int b = sp.b, hk = pc.hk, r0 = (pc.item - b * p.nrb) * 16 * CT;

        // ---- queries: scores in log2 units are c2 * q.k, with q's signs turned where c2 would be negative
        const float cs = a.scale * (F8 && a.c.k_scale ? a.c.k_scale[hk] : 1.0f) * AT_LOG2E;
        const float c2 = cs < 0.0f ? -cs : cs;
        const uint32_t flip = cs < 0.0f ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
        u32x4 qf[CT][QS];
        int first_c[CT], last_c[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int r = min(r0 + 16 * ct + c16, p.rows - 1);   // columns past the rows repeat the last one, unused
            const int t = r / a.group, h = hk * a.group + (r - t * a.group);
            
            last_c[ct] = sp.len - a.new_tokens + t + 1;
            first_c[ct] = a.window ? (int)max((int64_t)0, (int64_t)last_c[ct] - (int64_t)a.window) : 0;
            constexpr int QES = F32 ? 4 : 2;
            const char* Q = static_cast<const char*>(a.q) +
                            ((int64_t)b * a.sq[0] + (int64_t)t * a.sq[1] + (int64_t)h * a.sq[2]) * QES;
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                // the first value of the fragment that K's chunk s (8-bit: half a chunk) meets
                const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : (64 * s + 16 * g) / ES;
                u32x4 v = d < a.c.hd ? *reinterpret_cast<const u32x4*>(Q + d * QES) : u32x4{0, 0, 0, 0};
                v ^= flip;
                qf[ct][s] = v;
            }
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
        const uint32_t krow = (uint32_t)a.c.sk[1] * ES, vrow = (uint32_t)a.c.sv[1] * ES;
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
        constexpr int NE = FAST ? 2 : 1;
        uint32_t entry[NE], slot[NE];      // of the tile after next: table entries on their way
        const char* kbase[2];              // FAST: a half's first row
        const char* vbase[2];
        uint32_t koff = 0, voff = 0;       // else: lane j's for key j % 32, in 16 bytes
        uint32_t ok = 0;                   // keys that have a page
        auto fetch = [&](int t) {          // hi > 0; past the last key its own entry is read again
#pragma unroll
            for (int i = 0; i < NE; ++i) {
                const uint32_t pos = FAST ? min(t * PM_BN + 16 * i, (sp.hi - 1) & ~15) : min(t * PM_BN + lane % 32, sp.hi - 1);
                const uint32_t n = div32(pos, a.c.page);
                slot[i] = pos - n * a.c.page.d;
                if constexpr (FAST) entry[i] = (uint32_t)((table_ptr)(uintptr_t)trow)[n];
                else entry[i] = (uint32_t)trow[n];
            }
        };
        auto resolve = [&]() {   // keys without a page read page 0 and are masked
            if constexpr (FAST) {
                ok = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bool in = entry[i] < a.c.pages;
                    const int64_t page = in ? entry[i] : 0;
                    ok |= in ? 0xffffu << (16 * i) : 0u;
                    kbase[i] = Kh + (page * a.c.sk[0] + (int64_t)slot[i] * a.c.sk[1]) * ES;
                    vbase[i] = Vh + (page * a.c.sv[0] + (int64_t)slot[i] * a.c.sv[1]) * ES;
                }
            } else {
                const bool in = entry[0] < a.c.pages;
                const int64_t page = in ? entry[0] : 0;
                ok = (uint32_t)__ballot(in);
                koff = (uint32_t)((uint64_t)((page * a.c.sk[0] + (int64_t)slot[0] * a.c.sk[1]) * ES) / 16);
                voff = (uint32_t)((uint64_t)((page * a.c.sv[0] + (int64_t)slot[0] * a.c.sv[1]) * ES) / 16);
            }
        };
        u32x4 kr[2][KL];
        uint32_t vr[8][VW];
        auto load_k = [&]() {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const char* row = Kh;
                if constexpr (!FAST) row += (uint64_t)__shfl(koff, 16 * kb + c16) * 16;
#pragma unroll
                for (int s = 0; s < KL; ++s)
                    kr[kb][s] = *reinterpret_cast<const u32x4*>(FAST ? kbase[kb] + kcol[0] + 64 * s : row + kcol[FAST ? 0 : s]);
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (FAST) load_words<VW>(vbase[j / 4] + vfast[j % 4], vr[j]);
                else load_words<VW>(Vh + (uint64_t)__shfl(voff, 16 * (j / 4) + 4 * g + j % 4) * 16 + vcol, vr[j]);
            }
        };

        int t = 0;
        auto next_k = [&]() {
            resolve();
            fetch(t + 2 * PM_WAVES);
            load_k();
        };

        const int tile0 = sp.lo / PM_BN;
        const int end = sp.hi > sp.lo ? tile0 + (int)pc.c1 : 0;
        // keys that every row of the block sees
        const int all_lo = a.window ? (int)max((int64_t)0, (int64_t)sp.hi - (int64_t)a.window) : 0;
        const int all_hi = sp.len - a.new_tokens + sp.t0 + 1;
        t = tile0 + (int)pc.c0 + wave;
        if (t < end) {
            fetch(t);
            resolve();
            load_k();
            load_v();
            fetch(t + PM_WAVES);
        }
        for (; t < end; t += PM_WAVES) {
            const int k0 = t * PM_BN;
            const uint32_t keys = ok & key_bits(k0, sp.lo, sp.hi);
            const bool plain = keys == ~0u && k0 >= all_lo && k0 + PM_BN <= all_hi;
            const bool more = t + PM_WAVES < end;
            // ---- S^T = K Q^T
            if constexpr (!FAST) {
#pragma unroll
                for (int s = 0; s < KL; ++s)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        if (16 * g + 64 * s >= (int)kbytes) kr[kb][s] = u32x4{0, 0, 0, 0};
            }
            f32x4 sacc[2][CT];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) sacc[kb][ct] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KL; ++s)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
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
                    const uint32_t mine = (keys & key_bits(k0, first_c[ct], last_c[ct])) >> (4 * g);
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sacc[kb][ct][r] = (mine >> (16 * kb + r)) & 1 ? sacc[kb][ct][r] * c2 : -INFINITY;
                }
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
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
                for (int kb = 0; kb < 2; ++kb)
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
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < VW; ++w) vr[j][w] = (keys >> (4 * g + 16 * (j / 4) + j % 4)) & 1 ? vr[j][w] : 0u;
            }
            constexpr int RW = EV * (F32 ? 4 : 2) / 4;
            uint32_t vw[8][RW];   // 8-bit values widened
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int w = 0; w < RW; ++w) {
                    if constexpr (F8) vw[j][w] = widen8<DT>(vr[j][w / 2], w % 2);
                    else vw[j][w] = vr[j][w];
                }
            // Keys that some rows see and others do not, with values that are not finite: a probability of zero must not
            // meet them. They are marked for the rows that see them, and zeros in the product.
            if (__builtin_expect(!plain && several, 0)) {
                constexpr uint32_t top = F32 ? 0x7f800000u : DT == TVK_F16 ? 0x7c00u : 0x7f80u;
                int odd = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < RW; ++w)
                        odd |= (int)((vw[j][w] & top) == top) | (F32 ? 0 : (int)((vw[j][w] >> 16 & top) == top));
                if (__any(odd)) {
                    uint32_t* tile = reinterpret_cast<uint32_t*>(red + wave * 16 * LDO);   // the wave's own: a half's values
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        __builtin_amdgcn_wave_barrier();
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int w = 0; w < RW; ++w) {
                                uint32_t& v = vw[4 * kb + j][w];
                                tile[((4 * g + j) * 16 + c16) * RW + w] = v;
                                if constexpr (F32) v = (v & top) == top ? 0u : v;
                                else v &= ((v & top) == top ? 0u : 0xffffu) | ((v >> 16 & top) == top ? 0u : 0xffff0000u);
                            }
                        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
                        for (int i = lane; i < 16 * DV; i += 64) {
                            const int key = 16 * kb + i / DV, dv = i % DV;
                            const uint32_t v = F32 ? tile[i] : reinterpret_cast<const uint16_t*>(tile)[i];
                            if ((v & top) != top) continue;
                            const uint32_t sign = F32 ? 0x80000000u : 0x8000u;
                            const uint32_t mark = (v & ~sign) != top ? 3u : v & sign ? 2u : 1u;
#pragma unroll 1
                            for (int col = 0; col < 16 * CT; ++col) {
                                const int hi = sp.len - a.new_tokens + min(r0 + col, p.rows - 1) / a.group + 1;
                                const int lo = a.window ? (int)max((int64_t)0, (int64_t)hi - (int64_t)a.window) : 0;
                                if ((keys & key_bits(k0, lo, hi)) >> key & 1) atomicOr(&marks[(col * DV + dv) / 16], mark << 2 * (dv % 16));
                            }
                        }
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < EV; ++i)
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct)
                            oacc[i][ct] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vw[j][i]),
                                                                               sacc[j / 4][ct][j % 4], oacc[i][ct], 0, 0, 0);
            } else {
                u32x4 pf[CT];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    const f32x4 y = sacc[0][ct], z = sacc[1][ct];
                    pf[ct] = u32x4{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3]), pack2<DT>(z[0], z[1]), pack2<DT>(z[2], z[3])};
                }
#pragma unroll
                for (int i = 0; i < EV; ++i) {   // value i of the lane's eight keys
                    const uint32_t sel = i % 2 ? 0x07060302u : 0x05040100u;
                    const u32x4 vf = u32x4{__builtin_amdgcn_perm(vw[1][i / 2], vw[0][i / 2], sel),
                                           __builtin_amdgcn_perm(vw[3][i / 2], vw[2][i / 2], sel),
                                           __builtin_amdgcn_perm(vw[5][i / 2], vw[4][i / 2], sel),
                                           __builtin_amdgcn_perm(vw[7][i / 2], vw[6][i / 2], sel)};
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) oacc[i][ct] = mfma16<DT>(vf, pf[ct], oacc[i][ct]);
                }
            }
            if (more) {
                if (!plain) next_k();
                load_v();
            }
        }

        // ---- merge the waves, one 16-column block at a time
        const PagedMfmaArgs& pe = paged_args();
        const bool whole = pc.pieces == 1;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const float l_tot = lanes4_sum(l_run[ct]);
            __syncthreads();   // the block (piece) before has been read
            if (g == 0) {
                ml[0][wave][16 * ct + c16] = m_run[ct];
                ml[1][wave][16 * ct + c16] = l_tot;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < EV; i += 4)
                    *reinterpret_cast<f32x4*>(&red[(wave * 16 + c16) * LDO + EV * (4 * g + r) + i]) =
                        f32x4{oacc[i][ct][r], oacc[i + 1][ct][r], oacc[i + 2][ct][r], oacc[i + 3][ct][r]};
            __syncthreads();
            for (int c = tid; c < 16 * (DV / 4); c += 64 * PM_WAVES) {
                const int col = c / (DV / 4), dv = (c % (DV / 4)) * 4;
                const int lr = 16 * ct + col, r = r0 + lr;
                if (r >= pe.rows || dv >= pe.a.c.hd) continue;
                PagedSum s;
#pragma unroll
                for (int w = 0; w < PM_WAVES; ++w) s.m = fmaxf(s.m, ml[0][w][lr]);
#pragma unroll
                for (int w = 0; w < PM_WAVES; ++w)
                    s.add(ml[0][w][lr], ml[1][w][lr], *reinterpret_cast<const f32x4*>(&red[(w * 16 + col) * LDO + dv]));
                if (several) {
                    const uint32_t mark = marks[(lr * DV + dv) / 16] >> 2 * (dv % 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t two = mark >> 2 * i & 3;
                        if (two) s.o[i] += two == 1 ? INFINITY : two == 2 ? -INFINITY : NAN;
                    }
                }
                if (whole) {
                    paged_finish<DT>(pe, b, hk, r, dv, s.m, s.l, s.o);
                } else {
                    const __amdgpu_buffer_rsrc_t rs = paged_rsrc(pe);
                    const uint32_t row = (2 * wg + (pc.c0 == 0)) * 16 * CT + lr;
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, s.o), rs, paged_o_at(pe, row, dv), 0, kCoherent);
                    if (dv == 0)
                        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2v{s.m, s.l}), rs, paged_ml_at(pe, row), 0, kCoherent);
                }
            }
        }
        if (!whole && pe.count) {
            // ---- the last workgroup of the segment merges its pieces; none waits for another
            __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's partials are in memory
            __syncthreads();
            if (tid == 0) {
                unsigned* cnt = pe.count + (pc.item * pe.a.c.kvh + hk);
                last = atomicAdd_system(cnt, 1u) + 1 == pc.pieces;
                if (last) atomicExch_system(cnt, 0u);
            }
            __syncthreads();
            if (last) paged_merge<DT, CT>(pe, pc.item, hk, pc.first, pc.pieces, reinterpret_cast<char*>(red));
        }
        if (more_pieces) {
            x += pc.c1 - pc.c0;
            more_pieces = x < stop;
            // the next segment: the item's next head, or the next item's first
            at = (uint32_t)(hk + 1) * (uint32_t)sp.tiles;
            if (hk + 1 == pe.a.c.kvh) {
                ++pc.item;
                at = 0;
            }
        }
    }
}

// The merge as a launch of its own: a workgroup a segment.
template <int DT, int CT>
__global__ __launch_bounds__(64 * PM_WAVES) void paged_attn_merge_kernel(PagedMfmaArgs p) {
    __shared__ __attribute__((aligned(16))) char lds[PM_MERGE_BYTES];
    const int item = blockIdx.x / p.a.c.kvh, hk = blockIdx.x % p.a.c.kvh, lane = threadIdx.x % 64;
    const PagedDeal deal = paged_deal<CT>(p, lane);
    const uint32_t tiles = (uint32_t)paged_span<CT>(p, item).tiles, units = deal.units(tiles);
    PagedPiece pc;
    const uint32_t begin = paged_before<CT>(p, deal, item, lane) * (uint32_t)p.a.c.kvh + (uint32_t)hk * units;
    if (deal.chunk) {
        pc.first = begin;
        pc.pieces = units;
    } else {
        paged_pieces(deal, begin, tiles, pc);
    }
    if (pc.pieces > 1) paged_merge<DT, CT>(p, item, hk, pc.first, pc.pieces, lds);
}

constexpr int PM_CUS = 256;

template <int DT, bool F8, int D, int CT>
void paged_launch(PagedMfmaArgs& p, int64_t batch, hipStream_t s) {
    typedef PagedTile<DT, F8, D> G;
    p.nrb = (p.rows + 16 * CT - 1) / (16 * CT);
    p.items = (int)(batch * p.nrb);
    const int64_t segments = (int64_t)p.items * p.a.c.kvh;
    // a workgroup for every 4 tiles the sequences may have, as many as are resident together
    const int64_t tiles = ((int64_t)p.a.max_len + PM_BN - 1) / PM_BN + 1;
    const int64_t most = (int64_t)PM_CUS * G::occ(CT);
    int64_t wgs = tiles / PM_WAVES > most ? most : std::min<int64_t>(most, segments * (tiles / PM_WAVES));
    Scratch scratch;
    if (wgs > 0 && (tiles / PM_WAVES > 1)) {
        const size_t rows = (size_t)2 * wgs * 16 * CT, bytes = rows * (p.a.c.hd + 2) * 4;
        float* part = s == hipStreamPerThread ? nullptr : static_cast<float*>(scratch.get(bytes, s));
        if (part) {
            p.wgs = (int)wgs;
            p.part_o = part;
            p.part_ml = part + rows * p.a.c.hd;
            p.part_bytes = (unsigned)bytes;
            p.count = split_counters(s, segments);
        } else {
            clear_error();
        }
    }
    const dim3 grid((unsigned)(p.wgs ? p.wgs : segments)), block(64 * PM_WAVES);
    if (p.a.c.page.d % 16 == 0 && p.a.c.hd * G::ES == G::KL * 64) hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, true>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((paged_attn_mfma_kernel<DT, F8, D, CT, false>), grid, block, 0, s, p);
    if (p.wgs && !p.count)
        hipLaunchKernelGGL((paged_attn_merge_kernel<DT, CT>), dim3((unsigned)segments), block, 0, s, p);
}

template <int DT, bool F8>
void paged_dispatch(PagedMfmaArgs& p, int64_t batch, hipStream_t s) {
    const bool two = p.rows > 16;
    const int hd = p.a.c.hd;
#define TVK_PAGED(D) (two ? paged_launch<DT, F8, D, 2>(p, batch, s) : paged_launch<DT, F8, D, 1>(p, batch, s))
    if (hd <= 64) TVK_PAGED(64);
    else if (hd <= 96) TVK_PAGED(96);
    else if (hd <= 128) TVK_PAGED(128);
    else if constexpr (DT == TVK_F32) paged_launch<DT, F8, 256, 1>(p, batch, s);   // two row blocks' registers would spill
    else TVK_PAGED(256);
#undef TVK_PAGED
}

}  // namespace

// One translation unit each (paged_attention_f16.hip and its neighbours).
void paged_attn_f16(PagedMfmaArgs& p, bool f8, int64_t batch, hipStream_t s);
void paged_attn_bf16(PagedMfmaArgs& p, bool f8, int64_t batch, hipStream_t s);
void paged_attn_f32(PagedMfmaArgs& p, int64_t batch, hipStream_t s);

}  // namespace tvk
