// The paged attention's MFMA kernels for float32 queries and caches, and the rule for all types' calls.
#include "paged_attention_mfma.h"

namespace tvk {

bool paged_attn_f32(PagedMfmaArgs& p, int64_t batch, hipStream_t s) { return paged_dispatch<TVK_F32, false>(p, batch, s); }

// Head dims in 16s up to 256, rows whose 16-byte chunks are aligned, cache offsets that fit 32 bits in units of 16 bytes.
bool paged_attn_mfma(const PagedAttnArgs& a, int dtype, bool f8, int64_t batch, hipStream_t s) {
    const PagedCache& c = a.c;
    const bool f32 = dtype == TVK_F32;
    if (c.hd % 16 != 0 || c.hd > 256 || (f32 && f8) || c.pages == 0 || c.reach == 0) return false;
    const int64_t es = f8 ? 1 : f32 ? 4 : 2, qes = f32 ? 4 : 2;
    // strides of a dimension of one entry do not matter
    auto even = [](const void* p, const int64_t* st, std::initializer_list<int64_t> sizes, int64_t es, int64_t by) {
        if (reinterpret_cast<uintptr_t>(p) % by != 0) return false;
        int i = 0;
        for (const int64_t n : sizes) {
            if (n > 1 && st[i] * es % by != 0) return false;
            ++i;
        }
        return true;
    };
    const std::initializer_list<int64_t> cache = {(int64_t)c.pages, (int64_t)c.page.d, (int64_t)c.kvh};
    const std::initializer_list<int64_t> rows = {batch, (int64_t)a.new_tokens, (int64_t)a.heads};
    if (!even(c.k, c.sk, cache, es, 16) || !even(c.v, c.sv, cache, es, 16) || !even(a.q, a.sq, rows, qes, 16)) return false;
    for (const int64_t* st : {c.sk, c.sv}) {
        if (st[1] * es * 32 >= (int64_t)0x7fffffff || st[0] >= (int64_t)1 << 40 || st[2] >= (int64_t)1 << 40) return false;
        const double reach = ((double)(c.pages - 1) * st[0] + (double)(c.page.d - 1) * st[1]) * es;
        if (reach >= 0x1p36) return false;
    }
    PagedMfmaArgs p{};
    p.a = a;
    const int64_t nr = (int64_t)a.new_tokens * a.group;
    // every sum of tiles, pieces and segments below 2^31
    const double tiles = (a.max_len + 15.0) / 16 + 1.0;
    if (nr > 0x7fffffff || (double)batch * ((nr + 15) / 16) * c.kvh * tiles >= 0x1p31) return false;
    p.rows = (int)nr;
    return f32 ? paged_attn_f32(p, batch, s) : dtype == TVK_F16 ? paged_attn_f16(p, f8, batch, s) : paged_attn_bf16(p, f8, batch, s);
}

}  // namespace tvk
