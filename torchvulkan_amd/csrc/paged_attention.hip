// Attention of the newest tokens over a paged key/value cache
// (tvk_paged_attention): checks and the general kernel.
//
// General kernel: a workgroup a query row (batch, token, head). Its 4 waves
// take the keys in turn; a lane holds every 64th value of the head dim, a
// wave's lanes add up a key's dot product, and each wave keeps a running
// maximum, sum and output that are merged at the end in wave order.
#include "paged.h"

#include <algorithm>
#include <cmath>

using namespace tvk;

namespace {

constexpr int PA_WAVES = 4;
constexpr int PA_MAX_DIM = 512;
constexpr int PA_UNROLL = 4;

template <int DT, bool F8>
__device__ inline float cached(const void* p, int64_t i) {
    if (F8) return f8_to_f32(static_cast<const uint8_t*>(p)[i], TVK_F8E4M3FN);
    return elem<DT>::to_f32(static_cast<const typename elem<DT>::T*>(p)[i]);
}

template <int DT, bool F8, int ND>
__global__ __launch_bounds__(64 * PA_WAVES) void paged_attn_any_kernel(PagedAttnArgs p, int64_t rows) {
    typedef typename elem<DT>::T T;
    __shared__ float red[PA_WAVES][64 * ND];
    __shared__ float ml[PA_WAVES][2];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;   // a dimension of the grid does not hold them all
    if (row >= rows) return;
    const int h = (int)(row % p.heads), bt = (int)(row / p.heads);
    const int t = bt % p.new_tokens, b = bt / p.new_tokens, hk = h / p.group;
    const int hd = p.c.hd;
    const int len = (int)min((uint32_t)paged_len(p.c, b), p.max_len);
    const int last = t < paged_padding(p.c, b, p.new_tokens) ? 0 : len - p.new_tokens + t + 1;   // keys below it are seen
    const int first = p.window ? (int)max((int64_t)0, (int64_t)last - (int64_t)p.window) : 0;
    const T* q = static_cast<const T*>(p.q) + b * p.sq[0] + t * p.sq[1] + h * p.sq[2];
    const float ks = F8 && p.c.k_scale ? p.c.k_scale[hk] : 1.0f, vs = F8 && p.c.v_scale ? p.c.v_scale[hk] : 1.0f;
    float qv[ND], o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        qv[i] = lane + 64 * i < hd ? elem<DT>::to_f32(q[lane + 64 * i]) : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j0 = first + wave * PA_UNROLL; j0 < last; j0 += PA_WAVES * PA_UNROLL) {
        float s[PA_UNROLL];
        int64_t vo[PA_UNROLL];
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) {
            uint32_t page = 0, slot = 0;
            const bool in = j0 + u < last && paged_find(p.c, b, (uint32_t)(j0 + u), page, slot);
            const int64_t ko = (int64_t)page * p.c.sk[0] + (int64_t)slot * p.c.sk[1] + (int64_t)hk * p.c.sk[2];
            vo[u] = in ? (int64_t)page * p.c.sv[0] + (int64_t)slot * p.c.sv[1] + (int64_t)hk * p.c.sv[2] : -1;
            float acc = 0.0f;
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (in && lane + 64 * i < hd) acc = fmaf(qv[i], cached<DT, F8>(p.c.k, ko + lane + 64 * i), acc);
#pragma unroll
            for (int x = 32; x > 0; x >>= 1) acc += __shfl_xor(acc, x);
            s[u] = in ? acc * ks * p.scale : -INFINITY;
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) mn = fmaxf(mn, s[u]);
        const float mu = mn == -INFINITY ? 0.0f : mn;
        const float f = m == -INFINITY ? 0.0f : expf(m - mu);
        l *= f;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= f;
        m = mn;
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) {
            if (vo[u] < 0) continue;
            const float e = expf(s[u] - mu);
            l += e;
#pragma unroll
            for (int i = 0; i < ND; ++i)
                if (lane + 64 * i < hd) o[i] = fmaf(e, cached<DT, F8>(p.c.v, vo[u] + lane + 64 * i), o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) red[wave][lane + 64 * i] = o[i];
    if (lane == 0) {
        ml[wave][0] = m;
        ml[wave][1] = l;
    }
    __syncthreads();
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < PA_WAVES; ++w) mt = fmaxf(mt, ml[w][0]);
    float lt = 0.0f, f[PA_WAVES];
#pragma unroll
    for (int w = 0; w < PA_WAVES; ++w) {
        f[w] = ml[w][0] == -INFINITY ? 0.0f : expf(ml[w][0] - mt);
        lt += ml[w][1] * f[w];
    }
    // a NaN sum is a NaN row; only a row without keys is zeros
    const bool none = lt == 0.0f;
    T* out = static_cast<T*>(p.out) + b * p.so[0] + t * p.so[1] + h * p.so[2];
    for (int d = threadIdx.x; d < hd; d += 64 * PA_WAVES) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < PA_WAVES; ++w) x += red[w][d] * f[w];
        out[d] = elem<DT>::from_f32(none ? 0.0f : x / lt * vs);
    }
    if (p.lse && threadIdx.x == 0) p.lse[b * p.sl[0] + t * p.sl[1] + h * p.sl[2]] = none ? INFINITY : mt + logf(lt);
}

template <int DT, bool F8>
void launch_any(const PagedAttnArgs& p, int64_t rows, hipStream_t s) {
    const int64_t x = std::min<int64_t>(rows, 1 << 23);
    const dim3 grid((unsigned)x, (unsigned)((rows + x - 1) / x)), block(64 * PA_WAVES);
    if (p.c.hd <= 64) hipLaunchKernelGGL((paged_attn_any_kernel<DT, F8, 1>), grid, block, 0, s, p, rows);
    else if (p.c.hd <= 128) hipLaunchKernelGGL((paged_attn_any_kernel<DT, F8, 2>), grid, block, 0, s, p, rows);
    else if (p.c.hd <= 256) hipLaunchKernelGGL((paged_attn_any_kernel<DT, F8, 4>), grid, block, 0, s, p, rows);
    else hipLaunchKernelGGL((paged_attn_any_kernel<DT, F8, 8>), grid, block, 0, s, p, rows);
}

}  // namespace

extern "C" tvk_status tvk_paged_attention(const tvk_paged_attention_desc* d) {
    const char* who = "tvk_paged_attention";
    auto bad = [&](tvk_status st, const char* m) { return fail(st, std::string(who) + ": " + m); };
    if (!d) return bad(TVK_ERR_INVALID, "desc is NULL");
    const tvk_paged_cache& c = d->cache;
    tvk_status st = check_paged_cache(who, c, d->dtype, d->batch);
    if (st != TVK_OK) return st;
    if (d->new_tokens < 0 || d->heads_q < 0 || d->max_len < 0 || d->window < 0) return bad(TVK_ERR_INVALID, "negative size");
    if (d->heads_q % c.heads_kv != 0) return bad(TVK_ERR_INVALID, "heads_q is not a multiple of heads_kv");
    if (c.head_dim > PA_MAX_DIM) return bad(TVK_ERR_UNSUPPORTED, "head dims up to 512 only");
    for (const int64_t* s3 : {d->q_stride, d->out_stride, d->lse_stride})
        for (int i = 0; i < 3; ++i)
            if (s3[i] < 0) return bad(TVK_ERR_INVALID, "negative stride");
    if (d->batch == 0 || d->new_tokens == 0 || d->heads_q == 0) return TVK_OK;
    if (d->heads_q > 65535 || d->new_tokens > (int64_t)0x7fffffff / d->heads_q ||
        d->batch > (int64_t)0x7fffffff / (d->heads_q * d->new_tokens))
        return bad(TVK_ERR_UNSUPPORTED, "heads up to 65535, query rows up to 2^31 - 1 only");
    if (!d->q || !d->out) return bad(TVK_ERR_INVALID, "NULL tensor");
    PagedAttnArgs p{};
    p.c = paged_cache(c);
    p.q = d->q;
    p.out = d->out;
    p.lse = d->lse;
    for (int i = 0; i < 3; ++i) {
        p.sq[i] = d->q_stride[i];
        p.so[i] = d->out_stride[i];
        p.sl[i] = d->lse_stride[i];
    }
    p.heads = (int)d->heads_q;
    p.group = (int)(d->heads_q / c.heads_kv);
    p.new_tokens = (int)d->new_tokens;
    p.max_len = (uint32_t)std::min<int64_t>(d->max_len > 0 ? d->max_len : p.c.reach, p.c.reach);
    p.window = (uint32_t)std::min<int64_t>(d->window, 0x7fffffff);
    p.scale = (float)d->scale;
    const hipStream_t s = resolve_stream(d->stream);
    const int64_t rows = d->batch * d->new_tokens * d->heads_q;
    const bool f8 = c.dtype == TVK_F8E4M3FN;
    if (!paged_attn_mfma(p, d->dtype, f8, d->batch, s)) {
        if (d->dtype == TVK_F32) f8 ? launch_any<TVK_F32, true>(p, rows, s) : launch_any<TVK_F32, false>(p, rows, s);
        else if (d->dtype == TVK_F16) f8 ? launch_any<TVK_F16, true>(p, rows, s) : launch_any<TVK_F16, false>(p, rows, s);
        else f8 ? launch_any<TVK_BF16, true>(p, rows, s) : launch_any<TVK_BF16, false>(p, rows, s);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string(who) + ": launch failed: " + hipGetErrorString(e));
    return TVK_OK;
}
