// Products of 8-bit floats in blocks of 128 for more than 64 rows (tvk_gemm_f8):
// workgroup tiles of BM rows of A by BN rows of W, one block of 128 values of k a
// step, its operands and scales fetched from memory straight into LDS by buffer
// loads while the matrix unit works on the step before.
//
// A wave's tile is FN x FM blocks of 16 x 16. Its matrix instructions go row of
// blocks by row of blocks: those of row i into fresh registers, while row i - 1's
// sums are added to the running ones times their scales, and row i + 1's fragment is
// read. Before the last row of a step everything of the step has been read: there
// the one barrier of a step stands, behind which the next step's operands, which
// have landed, are read in place of those that the last row has used, and the step
// after that is fetched over the one that ends.
//
// LDS layout: 128 bytes a row and step, eight chunks of 16 bytes, chunk c of row r
// at slot c ^ ((r / 2) % 8). A fragment read takes 16 rows; its lanes l / 16 = g
// read chunk g + 4 j in read j (any order of k does, the same for both operands),
// and a read is served in groups of 16 lanes: {0-3, 12-15, 20-27}, {16-19, 28-31,
// 4-11} and the same two shifted by 32. Each group's rows of one parity are then
// (for c and c + 1) at the eight slots c ^ {0, 1, 6, 7}, c + 1 ^ {2, 3, 4, 5}: no
// two units on one bank.
//
// Measured: 8192 x 14336 x 4096 475 to 492 us, 8192^3 486 us (1.95 to 2.0 and 2.3 PFLOP/s; a library's bfloat16 product of 8192^3 958 us). The
// matrix unit is busy for half of the cycles there: a step's fragments and what is put into LDS take it three
// quarters of the time that the products take, and a wave's next step starts behind a barrier.
#include "gemm_dma.h"
#include "gemm_f8.h"

using namespace tvk;

namespace {

// Buffer resource over [p, p + bytes): loads past the end return zeros. The same for all lanes of a wave.
__device__ __forceinline__ i32x4 f8_rsrc(const void* p, int64_t bytes) {
    const uint64_t a = (uint64_t)p;
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)),
                 __builtin_amdgcn_readfirstlane((int)min(bytes, (int64_t)0x7fffffff)), 0x00020000};
}

// As dma16, 4 bytes per lane, to lds_addr + 4 * lane. (From inline assembly: a compiler-visible load into LDS would make every
// later LDS read wait for it.)
__device__ __forceinline__ void f8_dma4(i32x4 r, uint32_t lds_addr, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :: "s"(lds_addr), "v"(voff), "s"(r) : "memory");
}

// BM x BN tiles, WM x WN waves, NS steps in LDS.
template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_;
    static constexpr int NW = WM * WN, THREADS = 64 * NW;
    static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;   // fragments of a wave
    static constexpr int OPERANDS = (BM + BN) * F8_BLOCK;        // bytes of LDS a step
    static constexpr int STAGE = OPERANDS + 2048;                // with A's scales and 64 places for W's
    static constexpr int LOADS = OPERANDS / 1024 / NW;           // of a wave, each 8 rows; and one of scales
    static constexpr int A_LOADS = BM / 8;                       // of all
    static_assert(LOADS * 1024 * NW == OPERANDS, "whole loads a wave");
    static_assert(BN / WN <= F8_BLOCK && F8_BLOCK % (BN / WN) == 0, "one scale of W a wave and step");
    static_assert(NW > BM / 64 && BM * 4 + 256 <= 2048, "waves and places for both kinds of scales");
    static_assert(NS * STAGE <= 160 * 1024, "LDS");
};

template <class T, bool WIDE>
__global__ __launch_bounds__(T::THREADS) void gemm_f8_ring_kernel(GemmF8Args p) {
    constexpr int FM = T::FM, FN = T::FN, NS = T::NS;
    __shared__ __attribute__((aligned(1024))) char lds_raw[NS * T::STAGE];
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(TVK_LDS char*)lds_raw);
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wm = wave / T::WN, wn = wave % T::WN;
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m * p.tiles_n, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = tm * T::BM, n0 = tn * T::BN;
    const int first = blockIdx.y * p.split_blocks, steps = min(p.split_blocks, p.blocks - first);
    // the tile's rows from its first on: offsets within 32 bits whatever the matrix holds
    const int rows_a = min(T::BM, p.M - m0), rows_b = min(T::BN, p.N - n0);
    const i32x4 ra = f8_rsrc(static_cast<const uint8_t*>(p.a) + m0 * p.lda, (rows_a - 1) * p.lda + p.K);
    const i32x4 rb = f8_rsrc(p.b + n0 * p.ldb, (rows_b - 1) * p.ldb + p.K);
    const int k_left = p.K % F8_BLOCK;   // bytes of a last block that is not whole
    uint32_t off[T::LOADS], tail[2];     // (the chunks of a wave's loads depend on their parity alone)
#pragma unroll
    for (int q = 0; q < T::LOADS; ++q) {
        const int blk = wave * T::LOADS + q;
        const bool is_a = blk < T::A_LOADS;
        const int row = (is_a ? blk : blk - T::A_LOADS) * 8 + lane / 8;
        const int c = (lane % 8) ^ ((row / 2) % 8);
        off[q] = row < (is_a ? rows_a : rows_b) ? (uint32_t)(row * (is_a ? p.lda : p.ldb)) + 16 * c : kOOB;
        if (q < 2) tail[q] = k_left && 16 * c >= k_left ? kOOB : 0;
    }
    static_assert(T::LOADS % 2 == 0 && T::A_LOADS % 2 == 0, "parity");
    // one load of scales a wave: 64 of A's, or W's
    const bool scales_a = wave < T::BM / 64;
    const float* const sbase = scales_a ? p.sa + (m0 + wave * 64) * p.sa_m : p.sb + (int64_t)(n0 / F8_BLOCK) * p.sb_n;
    const int64_t sstep = scales_a ? p.sa_b : p.sb_b;
    const int sstride = (int)(scales_a ? p.sa_m : p.sb_n);
    const int srows = scales_a ? rows_a - wave * 64 : (rows_b + F8_BLOCK - 1) / F8_BLOCK;
    const uint32_t soff = lane < srows ? (uint32_t)(lane * sstride) * 4 : kOOB;
    const uint32_t sat = T::OPERANDS + (scales_a ? wave * 256 : T::BM * 4);
    // The waits count on as many loads for every step, so those past the last go through resources without records: they
    // put zeros into LDS and read no memory.
    auto fetch_one = [&](int step, int q) {
        const uint32_t slot = lds0 + (uint32_t)(step % NS * T::STAGE);
        const int b = first + step;
        const int live = step < steps;
        if (q < T::LOADS) {
            const int blk = wave * T::LOADS + q;
            const uint32_t end = b == p.blocks - 1 ? ~0u : 0u;
            i32x4 r = blk < T::A_LOADS ? ra : rb;
            r[2] = live ? r[2] : 0;
            dma16(r, slot + (uint32_t)(blk * 1024), (off[q] + (uint32_t)(b * F8_BLOCK)) | (tail[q % 2] & end));
        } else {
            f8_dma4(f8_rsrc(sbase + b * sstep, live ? 0x7fffffff : 0), slot + sat, soff);
        }
    };
    auto fetch = [&](int step) {
#pragma unroll
        for (int q = 0; q <= T::LOADS; ++q) fetch_one(step, q);
    };
    const int r = lane % 16, g = lane / 16;
    const uint32_t frag[2] = {(uint32_t)(r * F8_BLOCK + ((g ^ (r / 2)) * 16)), (uint32_t)(r * F8_BLOCK + (((g + 4) ^ (r / 2)) * 16))};
    auto read = [&](uint32_t base) {
        union { u32x4 h[2]; i32x8 v; } u;
        u.h[0] = *(const TVK_LDS u32x4*)(uintptr_t)(base + frag[0]);
        u.h[1] = *(const TVK_LDS u32x4*)(uintptr_t)(base + frag[1]);
        return u.v;
    };
    auto scale_at = [&](uint32_t at) { return *(const TVK_LDS float*)(uintptr_t)at; };
    const uint32_t at_x = lds0 + (uint32_t)(wm * FM * 16 * F8_BLOCK), at_w = lds0 + (uint32_t)((T::BM + wn * FN * 16) * F8_BLOCK);
    const uint32_t at_sx = lds0 + T::OPERANDS + (uint32_t)(wm * FM * 16 + r) * 4, at_sw = lds0 + T::OPERANDS + T::BM * 4 + wn * FN * 16 / F8_BLOCK * 4;
    f32x4 acc[FN][FM], d[2][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < FM; ++j) d[(FN - 1) % 2][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    i32x8 fx[FM], fw[2];
    float s[FM], s_before[FM], sx[FM], sw = 0.0f;
#pragma unroll
    for (int j = 0; j < FM; ++j) s[j] = 0.0f;
    if (steps > 0) {
#pragma unroll
        for (int k = 0; k < NS - 1; ++k) fetch(k);
        wait_vmcnt<(NS - 2) * (T::LOADS + 1)>();
        __syncthreads();
        fetch(NS - 1);
#pragma unroll
        for (int j = 0; j < FM; ++j) fx[j] = read(at_x + j * 16 * F8_BLOCK);
        fw[0] = read(at_w);
#pragma unroll
        for (int j = 0; j < FM; ++j) sx[j] = scale_at(at_sx + j * 64);
        sw = scale_at(at_sw);
    }
    for (int step = 0; step < steps; ++step) {
        const uint32_t here = (uint32_t)(step % NS * T::STAGE), next = (uint32_t)((step + 1) % NS * T::STAGE);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            s_before[j] = s[j];
            s[j] = sx[j] * sw;
        }
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const bool last = i == FN - 1;
            if (last) {
                // everything of this step is read and everything of the next has landed, for all waves
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                wait_vmcnt<(NS - 2) * (T::LOADS + 1)>();
                __syncthreads();
            }
            fw[(i + 1) % 2] = read(last ? at_w + next : at_w + here + (i + 1) * 16 * F8_BLOCK);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                d[i % 2][j] = f8_mfma<WIDE>(fw[i % 2], fx[j]);
                if (last) {
                    fx[j] = read(at_x + next + j * 16 * F8_BLOCK);
                    sx[j] = scale_at(at_sx + next + j * 64);
                    if (j == 0) sw = scale_at(at_sw + next);
                }
                // row i - 1, of the step before for i == 0
                const int before = (i + FN - 1) % FN;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[before][j][e] = fmaf(d[(i + 1) % 2][j][e], i ? s[j] : s_before[j], acc[before][j][e]);
                asm volatile("" : "+v"(acc[before][j]));   // here, and not when the sum is wanted
                __builtin_amdgcn_sched_barrier(0);
            }
            if (last) fetch(step + NS);
        }
    }
    wait_vmcnt<0>();
    static_assert(FN % 2 == 0, "rows of blocks in turn");
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[FN - 1][j][e] = fmaf(d[1][j][e], s[j], acc[FN - 1][j][e]);
    if (p.part) {   // a lane has four neighbouring sums of row m
        float* part = p.part + (int64_t)blockIdx.y * p.M * p.part_n;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = m0 + (wm * FM + j) * 16 + r;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int n = n0 + (wn * FN + i) * 16 + 4 * g;
                if (m < p.M && n < p.part_n) *reinterpret_cast<f32x4*>(part + (int64_t)m * p.part_n + n) = acc[i][j];
            }
        }
        return;
    }
    // Through LDS, so that stores are whole lines: row m's chunk c of 16 bytes at slot c ^ m, within the row.
    __syncthreads();   // every wave has left the ring (what it read past its last step is not used)
    auto finish = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        typedef typename elem<DT>::T O;
        constexpr int PER = 16 / (int)sizeof(O), PITCH = T::BN * (int)sizeof(O), CHUNKS = T::BN / PER;
        static_assert(T::BM * PITCH <= NS * T::STAGE || sizeof(O) == 4, "the tile fits the ring");
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = (wm * FM + j) * 16 + r;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int n = (wn * FN + i) * 16 + 4 * g;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = acc[i][j][e];
                    if (p.bias) v[e] += f8_bias<DT>(p, min(n0 + n + e, p.N - 1));
                }
                char* to = lds_raw + m * PITCH + ((n / PER) ^ (m % CHUNKS)) * 16 + n % PER * (int)sizeof(O);
                store_words<4 * sizeof(O), 4 * sizeof(O)>(to, pack<DT, 4>(v));
            }
        }
        __syncthreads();
        for (int q = threadIdx.x; q < T::BM * CHUNKS; q += T::THREADS) {
            const int m = q / CHUNKS, c = q % CHUNKS, n = n0 + c * PER;
            if (m0 + m >= p.M || n >= p.N) continue;
            const Words<16> w = load_words<16, 16>(lds_raw + m * PITCH + (c ^ (m % CHUNKS)) * 16);
            O* o = static_cast<O*>(p.out) + (m0 + m) * p.ldo + n;
            if (n + PER <= p.N) store_words<16, sizeof(O)>(o, w);
            else
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (n + e < p.N) {
                        if constexpr (sizeof(O) == 4) o[e] = __builtin_bit_cast(O, w.w[e]);
                        else o[e] = __builtin_bit_cast(O, (uint16_t)(w.w[e / 2] >> e % 2 * 16));
                    }
        }
    };
    if constexpr (WIDE) finish(std::integral_constant<int, TVK_F32>{});
    else if (p.out_dtype == TVK_F16) finish(std::integral_constant<int, TVK_F16>{});
    else finish(std::integral_constant<int, TVK_BF16>{});
}

// Sums the partials of a split K in their order: four neighbouring outputs a thread.
__global__ __launch_bounds__(256) void gemm_f8_join_kernel(GemmF8Args p, int splits) {
    const int64_t all = (int64_t)p.M * (p.part_n / 4);
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
        const int m = (int)(q / (p.part_n / 4)), n = (int)(q % (p.part_n / 4)) * 4;
        f32x4 v = *reinterpret_cast<const f32x4*>(p.part + q * 4);
#pragma unroll 4
        for (int k = 1; k < splits; ++k) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(p.part + (k * all + q) * 4);
            v = f32x4{v[0] + o[0], v[1] + o[1], v[2] + o[2], v[3] + o[3]};
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N) f8_put(p, m, n + e, v[e]);
    }
}

template <class T, bool WIDE>
void launch(GemmF8Args p, int splits, hipStream_t s) {
    p.tiles_m = (p.M + T::BM - 1) / T::BM;
    p.tiles_n = (p.N + T::BN - 1) / T::BN;
    p.split_blocks = (p.blocks + splits - 1) / splits;
    hipLaunchKernelGGL((gemm_f8_ring_kernel<T, WIDE>), dim3((unsigned)(p.tiles_m * p.tiles_n), (unsigned)splits), dim3(T::THREADS), 0, s, p);
    if (p.part) {
        const int64_t groups = ((int64_t)p.M * (p.part_n / 4) + 255) / 256;
        hipLaunchKernelGGL(gemm_f8_join_kernel, dim3((unsigned)std::min<int64_t>(groups, 1 << 20)), dim3(256), 0, s, p, splits);
    }
}

}  // namespace

namespace tvk {

// K is split where there are 128 x 128 tiles for half the CUs or fewer, into stretches of 4 blocks or more: 128 x 4096 x 4096 in
// 1, 2, 4 and 8 parts 27.4, 21.2, 18.5 and 19.8 us, 1024 x 1024 x 14336 in 1, 2 and 4 85.5, 50.9 and 36.5; 512 x 4096 x 4096 in
// 1, 2 (a workgroup a CU) and 4 27.9, 25.5 and 36.3.
int f8_ring_splits(const GemmF8Args& p) {
    const int64_t tiles = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    return (int)std::max<int64_t>(1, std::min<int64_t>(256 / tiles, p.blocks / 4));
}

void f8_ring(const GemmF8Args& p, int splits, hipStream_t s) {
    // float32 results need a wave's registers for wider operands
    if (p.out_dtype == TVK_F32) return launch<Tile<128, 128, 2, 2, 2>, true>(p, splits, s);
    // A round of a tile on every CU takes about 30, 42 and 60 us of 4096 values of k for tiles of 128 x 128, 128 x 256 and
    // 256 x 256 (that is 1.15, 1.6 and 2 PFLOP/s, the smaller ones waiting for LDS): the size whose rounds take least.
    // 2048 x 4096 x 4096 59.8, 49.7 and 64.8 us; 1024 x 4096 x 4096 29.9, 40.4 and 57.5; 3000 x 4096 x 4096 83.7, 85.5 and 68.0.
    auto rounds = [&](int64_t bm, int64_t bn) { return ((p.M + bm - 1) / bm * ((p.N + bn - 1) / bn) + 255) / 256; };
    const int64_t small = 5 * rounds(128, 128), middle = 7 * rounds(128, 256), large = 10 * rounds(256, 256);
    if (splits > 1 || small <= std::min(middle, large)) launch<Tile<128, 128, 2, 2, 4>, false>(p, splits, s);
    else if (middle < large) launch<Tile<128, 256, 2, 4, 3>, false>(p, splits, s);
    else launch<Tile<256, 256, 4, 2, 2>, false>(p, splits, s);
}

}  // namespace tvk
