// Append to a paged key/value cache (tvk_paged_append): rotation of the new
// tokens' queries and keys, and their keys and values into their slots.
//
// The call moves each value once and is bound by that. The queries', keys' and
// values' heads of a token follow each other. A thread takes two chunks of VEC
// values of a head, 16 bytes each: the two that are rotated into each other, or
// neighbours; rotated values are read and written by one thread, so q_out may be
// q. A token's chunks are taken by as many waves as it needs for the call to fill
// the chip, and where a lane meets the same place of every head, it keeps its
// angles. Rotations that do not split into chunks run one pair a thread.
//
// Measured: 8192 tokens of 32 queries, 8 keys and 8 values of 128 in bfloat16 44 us,
// 4.6 TB/s (a 2 GiB copy moves 4.9); 240 such tokens to 8 bits 4.5 us, one token 3.7 us,
// the launch.
#include "paged.h"
#include "words.h"

#include <algorithm>

using namespace tvk;

namespace tvk {

tvk_status check_paged_cache(const char* who, const tvk_paged_cache& c, int32_t dtype, int64_t batch) {
    auto bad = [&](tvk_status st, const char* m) { return fail(st, std::string(who) + ": " + m); };
    if (dtype != TVK_F32 && dtype != TVK_F16 && dtype != TVK_BF16)
        return bad(TVK_ERR_UNSUPPORTED, "dtype must be float32, float16 or bfloat16");
    if (c.dtype != dtype && c.dtype != TVK_F8E4M3FN)
        return bad(TVK_ERR_UNSUPPORTED, "the cache's dtype must be the tokens' or float8_e4m3fn");
    if (c.dtype != TVK_F8E4M3FN && (c.k_scale || c.v_scale))
        return bad(TVK_ERR_INVALID, "scales belong to a float8_e4m3fn cache");
    if (batch < 0 || c.pages < 0 || c.page_size <= 0 || c.heads_kv <= 0 || c.head_dim <= 0 || c.table_width < 0)
        return bad(TVK_ERR_INVALID, "a negative size, or a cache without slots or heads");
    if (c.pages > 0x7fffffff || c.page_size > 0x7fffffff || c.heads_kv > 65535 || batch > 0x7fffffff)
        return bad(TVK_ERR_UNSUPPORTED, "pages, page size and batch up to 2^31 - 1, key/value heads up to 65535 only");
    if (c.table_width > 0x7fffffff)
        return bad(TVK_ERR_UNSUPPORTED, "table rows up to 2^31 - 1 entries only");
    for (int i = 0; i < 3; ++i)
        if (c.k_stride[i] < 0 || c.v_stride[i] < 0) return bad(TVK_ERR_INVALID, "negative cache stride");
    if (batch > 0 && (!c.seq_lens || (c.table_width > 0 && !c.table))) return bad(TVK_ERR_INVALID, "NULL table or lengths");
    if (batch > 0 && c.pages > 0 && (!c.k || !c.v)) return bad(TVK_ERR_INVALID, "NULL cache");
    if (batch > 1 && c.table_stride < 0) return bad(TVK_ERR_INVALID, "negative table stride");
    return TVK_OK;
}

PagedCache paged_cache(const tvk_paged_cache& c) {
    PagedCache p{};
    p.k = c.k;
    p.v = c.v;
    for (int i = 0; i < 3; ++i) {
        p.sk[i] = c.k_stride[i];
        p.sv[i] = c.v_stride[i];
    }
    p.k_scale = c.k_scale;
    p.v_scale = c.v_scale;
    p.table = c.table;
    p.lens = c.seq_lens;
    p.news = c.new_lens;
    p.table_stride = c.table_stride;
    p.pages = (uint32_t)c.pages;
    p.reach = (uint32_t)(c.table_width > kMaxReach / c.page_size ? kMaxReach : c.table_width * c.page_size);
    p.page = make_div((uint32_t)c.page_size);
    p.kvh = (int)c.heads_kv;
    p.hd = (int)c.head_dim;
    return p;
}

}  // namespace tvk

namespace {

constexpr int AP_THREADS = 256;

struct AppendArgs {
    PagedCache c;
    const void* q;
    const void* k;
    const void* v;
    void* qo;
    int64_t sq[3], sk[3], sv[3], so[3];   // batch, token, head strides
    const float* rotary;
    int64_t srot;
    uint32_t rot_len;
    int half;               // rotated pairs of a head
    int interleaved;
    int heads_q;
    int64_t tokens;         // batch * new tokens
    Div32 split;            // waves a token
    uint32_t width;         // workgroups in the grid's first dimension, which does not hold those of 2^26 tokens
    int same_place;         // a lane's chunks lie in the same place of every head it meets
    Div32 per_head, per_token, new_tokens;
};

// A product and a sum, each rounded: (a cos - b sin, b cos + a sin) is the same from any kernel.
__device__ inline void rotate(float& a, float& b, float cs, float sn) {
#pragma clang fp contract(off)
    const float x = a * cs - b * sn;
    b = b * cs + a * sn;
    a = x;
}

__device__ inline float saturated(float f, float s) {
    f /= s;
    return f != f ? f : fminf(fmaxf(f, -448.0f), 448.0f);
}

// A token's place; false for padding, a position past the angles and a page that is none.
__device__ inline bool place(const AppendArgs& p, int64_t token, uint32_t& b, uint32_t& t, int& pos, uint32_t& page, uint32_t& slot) {
    b = div32((uint32_t)token, p.new_tokens);
    t = (uint32_t)token - b * p.new_tokens.d;
    pos = paged_len(p.c, b) - (int)p.new_tokens.d + (int)t;
    page = slot = 0;
    return (int)t >= paged_padding(p.c, b, (int)p.new_tokens.d) && pos >= 0 && (!p.rotary || (uint32_t)pos < p.rot_len) && paged_find(p.c, b, (uint32_t)pos, page, slot);
}

template <int DT, bool F8>
__global__ __launch_bounds__(AP_THREADS) void paged_append_any_kernel(AppendArgs p) {
    typedef typename elem<DT>::T T;
    const uint32_t items = p.per_token.d;
    for (int64_t token = blockIdx.x; token < p.tokens; token += gridDim.x) {
        uint32_t b, t, page, slot;
        int pos;
        const bool placed = place(p, token, b, t, pos, page, slot);
        const float* rot = p.rotary + (placed ? pos * p.srot : 0);
        for (uint32_t i = threadIdx.x; i < items; i += AP_THREADS) {
            const int head = (int)div32(i, p.per_head), j = (int)(i - head * p.per_head.d);
            const bool is_q = head < p.heads_q, is_k = !is_q && head < p.heads_q + p.c.kvh;
            const int h = is_q ? head : is_k ? head - p.heads_q : head - p.heads_q - p.c.kvh;
            if (!placed && !is_q) continue;
            const T* src = is_q ? static_cast<const T*>(p.q) + b * p.sq[0] + t * p.sq[1] + h * p.sq[2]
                         : is_k ? static_cast<const T*>(p.k) + b * p.sk[0] + t * p.sk[1] + h * p.sk[2]
                                : static_cast<const T*>(p.v) + b * p.sv[0] + t * p.sv[1] + h * p.sv[2];
            const bool turn = (is_q || is_k) && j < p.half;
            // the item's two values: a rotated pair, or two neighbours (the last one alone)
            const int d0 = turn && !p.interleaved ? j : 2 * j, d1 = turn && !p.interleaved ? j + p.half : 2 * j + 1;
            const bool two = d1 < p.c.hd;
            const T x0 = src[d0], y0 = two ? src[d1] : T(0);
            float x = elem<DT>::to_f32(x0), y = elem<DT>::to_f32(y0);
            if (turn && placed) rotate(x, y, rot[j], rot[p.half + j]);
            if (is_q) {
                T* o = static_cast<T*>(p.qo) + b * p.so[0] + t * p.so[1] + h * p.so[2];
                // values that are not rotated keep their bits
                o[d0] = !placed ? T(0) : turn ? elem<DT>::from_f32(x) : x0;
                if (two) o[d1] = !placed ? T(0) : turn ? elem<DT>::from_f32(y) : y0;
                continue;
            }
            const int64_t* st = is_k ? p.c.sk : p.c.sv;
            const int64_t off = (int64_t)page * st[0] + (int64_t)slot * st[1] + (int64_t)h * st[2];
            if (F8) {
                uint8_t* o = static_cast<uint8_t*>(is_k ? p.c.k : p.c.v) + off;
                const float* sc = is_k ? p.c.k_scale : p.c.v_scale;
                const float s = sc ? sc[h] : 1.0f;
                o[d0] = f32_to_f8(saturated(x, s), TVK_F8E4M3FN);
                if (two) o[d1] = f32_to_f8(saturated(y, s), TVK_F8E4M3FN);
            } else {
                T* o = static_cast<T*>(is_k ? p.c.k : p.c.v) + off;
                o[d0] = turn ? elem<DT>::from_f32(x) : x0;
                if (two) o[d1] = turn ? elem<DT>::from_f32(y) : y0;
            }
        }
    }
}

template <int DT, bool F8, int VEC>
__global__ __launch_bounds__(AP_THREADS) void paged_append_kernel(AppendArgs p) {
    typedef typename elem<DT>::T T;
    constexpr int B = VEC * (int)sizeof(T), A = (int)sizeof(T);
    const uint32_t wave = __builtin_amdgcn_readfirstlane((blockIdx.y * p.width + blockIdx.x) * (AP_THREADS / 64) + threadIdx.x / 64);
    const uint32_t token = div32(wave, p.split), part = wave - token * p.split.d;
    if (token >= p.tokens) return;
    uint32_t b, t, page, slot;
    int pos;
    const bool placed = place(p, token, b, t, pos, page, slot);
    const float* rot = p.rotary + (placed ? pos * p.srot : 0);
    const uint32_t items = placed ? p.per_token.d : (uint32_t)p.heads_q * p.per_head.d;   // without a place: zeros in q_out
    const int turned = p.half / VEC;   // chunk pairs that are rotated into each other
    float cs[VEC], sn[VEC];
    bool angles = false;
    for (uint32_t i = part * 64 + threadIdx.x % 64; i < items; i += 64 * p.split.d) {
        const int head = (int)div32(i, p.per_head), j = (int)(i - head * p.per_head.d);
        const bool is_q = head < p.heads_q, is_k = !is_q && head < p.heads_q + p.c.kvh;
        const int h = is_q ? head : is_k ? head - p.heads_q : head - p.heads_q - p.c.kvh;
        const T* src = is_q ? static_cast<const T*>(p.q) + b * p.sq[0] + t * p.sq[1] + h * p.sq[2]
                     : is_k ? static_cast<const T*>(p.k) + b * p.sk[0] + t * p.sk[1] + h * p.sk[2]
                            : static_cast<const T*>(p.v) + b * p.sv[0] + t * p.sv[1] + h * p.sv[2];
        // chunks of pairs (i, i + half) first; interleaved pairs lie inside a chunk
        const bool across = !p.interleaved && j < turned;
        const int d0 = across ? VEC * j : 2 * VEC * j, d1 = across ? d0 + p.half : d0 + VEC;
        const bool two = d1 < p.c.hd;
        const bool turn0 = !is_q && !is_k ? false : p.interleaved ? d0 < 2 * p.half : across;
        const bool turn1 = turn0 && (!p.interleaved || d1 < 2 * p.half);
        Words<B> w0 = load_words<B, A>(src + d0), w1 = two ? load_words<B, A>(src + d1) : Words<B>{};
        if (placed && turn0 && (!angles || !p.same_place)) {
            // across: VEC angles, from d0; interleaved: VEC / 2 for each of the two chunks, from d0 / 2
            const int from = across ? d0 : d0 / 2, n = p.half - from;
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
                const bool in = k < n;
                const Words<8> c2 = load_words<8, 4>(rot + from + (in ? k : 0)), s2 = load_words<8, 4>(rot + p.half + from + (in ? k : 0));
                cs[k] = __builtin_bit_cast(float, c2.w[0]);
                cs[k + 1] = __builtin_bit_cast(float, c2.w[1]);
                sn[k] = __builtin_bit_cast(float, s2.w[0]);
                sn[k + 1] = __builtin_bit_cast(float, s2.w[1]);
            }
            angles = true;
        }
        float x[VEC], y[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            x[k] = word_at<DT>(w0, k);
            y[k] = word_at<DT>(w1, k);
        }
        if (placed && turn0) {
            if (across) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) rotate(x[k], y[k], cs[k], sn[k]);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; k += 2) rotate(x[k], x[k + 1], cs[k / 2], sn[k / 2]);
                if (turn1)
#pragma unroll
                    for (int k = 0; k < VEC; k += 2) rotate(y[k], y[k + 1], cs[(VEC + k) / 2], sn[(VEC + k) / 2]);
            }
        }
        // values that are not rotated keep their bits
        const Words<B> o0 = !placed ? Words<B>{} : turn0 ? pack<DT, VEC>(x) : w0;
        const Words<B> o1 = !placed ? Words<B>{} : turn1 ? pack<DT, VEC>(y) : w1;
        if (is_q) {
            T* o = static_cast<T*>(p.qo) + b * p.so[0] + t * p.so[1] + h * p.so[2];
            store_words<B, A>(o + d0, o0);
            if (two) store_words<B, A>(o + d1, o1);
            continue;
        }
        const int64_t* st = is_k ? p.c.sk : p.c.sv;
        const int64_t off = (int64_t)page * st[0] + (int64_t)slot * st[1] + (int64_t)h * st[2];
        if constexpr (F8) {
            uint8_t* o = static_cast<uint8_t*>(is_k ? p.c.k : p.c.v) + off;
            const float* sc = is_k ? p.c.k_scale : p.c.v_scale;
            const float s = sc ? sc[h] : 1.0f;
            Words<VEC> e0, e1;
#pragma unroll
            for (int k = 0; k < VEC; k += 4) {
                e0.w[k / 4] = pack4_f8(saturated(x[k], s), saturated(x[k + 1], s), saturated(x[k + 2], s), saturated(x[k + 3], s));
                e1.w[k / 4] = pack4_f8(saturated(y[k], s), saturated(y[k + 1], s), saturated(y[k + 2], s), saturated(y[k + 3], s));
            }
            store_words<VEC, 1>(o + d0, e0);
            if (two) store_words<VEC, 1>(o + d1, e1);
        } else {
            T* o = static_cast<T*>(is_k ? p.c.k : p.c.v) + off;
            store_words<B, A>(o + d0, o0);
            if (two) store_words<B, A>(o + d1, o1);
        }
    }
}

template <int DT, bool F8>
void append(AppendArgs& p, hipStream_t s) {
    const uint32_t heads = (uint32_t)(p.heads_q + 2 * p.c.kvh);
    auto fits = [&](int vec) { return p.c.hd % vec == 0 && (p.interleaved ? 2 * p.half : p.half) % vec == 0; };
    const int vec = DT != TVK_F32 && fits(8) ? 8 : fits(4) ? 4 : 0;
    if (!vec) {
        const uint32_t per_head = (uint32_t)((p.c.hd + 1) / 2);
        p.per_head = make_div(per_head);
        p.per_token = make_div(heads * per_head);
        const dim3 grid((unsigned)std::min<int64_t>(p.tokens, 1 << 20)), block(AP_THREADS);
        hipLaunchKernelGGL((paged_append_any_kernel<DT, F8>), grid, block, 0, s, p);
        return;
    }
    const uint32_t per_head = (uint32_t)((p.c.hd / vec + 1) / 2), items = heads * per_head;
    p.per_head = make_div(per_head);
    p.per_token = make_div(items);
    // waves a token: all it has work for while the chip is not full (32 waves a CU)
    const int64_t all = (items + 63) / 64, room = std::max<int64_t>(1, 8192 / p.tokens);
    const int64_t split = std::min(all, room);
    p.split = make_div((uint32_t)split);
    p.same_place = 64 * split % per_head == 0;
    const int64_t wgs = (p.tokens * split + 3) / 4;   // below 2^30: more than 8192 tokens take a wave each
    p.width = (uint32_t)std::min<int64_t>(wgs, 1 << 23);
    const dim3 grid(p.width, (unsigned)((wgs + p.width - 1) / p.width)), block(AP_THREADS);
    if constexpr (DT != TVK_F32) {
        if (vec == 8) {
            hipLaunchKernelGGL((paged_append_kernel<DT, F8, 8>), grid, block, 0, s, p);
            return;
        }
    }
    hipLaunchKernelGGL((paged_append_kernel<DT, F8, 4>), grid, block, 0, s, p);
}

}  // namespace

extern "C" tvk_status tvk_paged_append(const tvk_paged_append_desc* d) {
    const char* who = "tvk_paged_append";
    auto bad = [&](tvk_status st, const char* m) { return fail(st, std::string(who) + ": " + m); };
    if (!d) return bad(TVK_ERR_INVALID, "desc is NULL");
    const tvk_paged_cache& c = d->cache;
    tvk_status st = check_paged_cache(who, c, d->dtype, d->batch);
    if (st != TVK_OK) return st;
    if (d->new_tokens < 0 || d->heads_q < 0) return bad(TVK_ERR_INVALID, "negative size");
    if (c.head_dim > 1024 || d->heads_q > 65535) return bad(TVK_ERR_UNSUPPORTED, "head dims up to 1024, heads up to 65535 only");
    if (d->new_tokens > 0x7fffffff || (d->new_tokens > 0 && d->batch > 0x7fffffff / d->new_tokens))
        return bad(TVK_ERR_UNSUPPORTED, "batch * new_tokens up to 2^31 - 1 only");
    if (d->rotary) {
        if (d->rotary_dim <= 0 || d->rotary_dim % 2 != 0 || d->rotary_dim > c.head_dim)
            return bad(TVK_ERR_INVALID, "rotary_dim must be even, above zero and at most head_dim");
        if (d->rotary_len < 0 || d->rotary_stride < 0) return bad(TVK_ERR_INVALID, "negative rotary size or stride");
    }
    for (const int64_t* s3 : {d->q_stride, d->k_stride, d->v_stride, d->q_out_stride})
        for (int i = 0; i < 3; ++i)
            if (s3[i] < 0) return bad(TVK_ERR_INVALID, "negative stride");
    if (d->batch == 0 || d->new_tokens == 0) return TVK_OK;
    if (!d->k || !d->v || (d->heads_q > 0 && (!d->q || !d->q_out))) return bad(TVK_ERR_INVALID, "NULL tensor");
    AppendArgs p{};
    p.c = paged_cache(c);
    p.q = d->q;
    p.k = d->k;
    p.v = d->v;
    p.qo = d->q_out;
    for (int i = 0; i < 3; ++i) {
        p.sq[i] = d->q_stride[i];
        p.sk[i] = d->k_stride[i];
        p.sv[i] = d->v_stride[i];
        p.so[i] = d->q_out_stride[i];
    }
    p.rotary = d->rotary;
    p.srot = d->rotary_stride;
    p.rot_len = d->rotary ? (uint32_t)std::min<int64_t>(d->rotary_len, 0x7fffffff) : 0;
    p.half = d->rotary ? (int)(d->rotary_dim / 2) : 0;
    p.interleaved = d->interleaved != 0;
    p.heads_q = (int)d->heads_q;
    p.tokens = d->batch * d->new_tokens;
    p.new_tokens = make_div((uint32_t)d->new_tokens);
    const hipStream_t s = resolve_stream(d->stream);
    const bool f8 = c.dtype == TVK_F8E4M3FN;
    if (d->dtype == TVK_F32) f8 ? append<TVK_F32, true>(p, s) : append<TVK_F32, false>(p, s);
    else if (d->dtype == TVK_F16) f8 ? append<TVK_F16, true>(p, s) : append<TVK_F16, false>(p, s);
    else f8 ? append<TVK_BF16, true>(p, s) : append<TVK_BF16, false>(p, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string(who) + ": launch failed: " + hipGetErrorString(e));
    return TVK_OK;
}
