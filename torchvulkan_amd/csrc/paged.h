// The paged key/value cache of tvk_paged_append and tvk_paged_attention, as
// the kernels see it, and the checks both entry points share.
#pragma once

#include "convert.h"

namespace tvk {

constexpr int64_t kGridThreads = 0xffffffff;     // of a launch in one dimension of its grid
constexpr int64_t kMaxReach = (int64_t)1 << 30;   // positions: index sums stay in 32 bits

struct PagedCache {
    void* k;
    void* v;
    int64_t sk[3], sv[3];   // page, slot, head strides, elements
    const float* k_scale;
    const float* v_scale;
    const int32_t* table;
    const int32_t* lens;
    const int32_t* news;    // or NULL
    int64_t table_stride;
    uint32_t pages;
    uint32_t reach;         // positions a table row spans (at most kMaxReach)
    Div32 page;             // by the page size
    int kvh, hd;
};

struct PagedAttnArgs {
    PagedCache c;
    const void* q;
    void* out;
    float* lse;
    int64_t sq[3], so[3], sl[3];   // batch, token, head strides
    int heads, group, new_tokens;
    uint32_t max_len;
    uint32_t window;               // 0: none
    float scale;
};

// Queues the MFMA kernel (paged_attention_mfma.h) when it takes the call; false when it does not, its launch having too
// many workgroups among the reasons.
bool paged_attn_mfma(const PagedAttnArgs& a, int dtype, bool f8, int64_t batch, hipStream_t s);

// TVK_OK when the cache is one the kernels take and its pointers are there.
tvk_status check_paged_cache(const char* who, const tvk_paged_cache& c, int32_t dtype, int64_t batch);
PagedCache paged_cache(const tvk_paged_cache& c);

// Positions of sequence b: never below zero nor past its table row.
__device__ inline int paged_len(const PagedCache& c, int b) {
    // not written while a kernel reads it: a scalar load where b is a wave's
    const int n = ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)c.lens)[b];
    return n < 0 ? 0 : (uint32_t)n > c.reach ? (int)c.reach : n;
}

// Of a call's `new_tokens` tokens, those in front of sequence b's own.
__device__ inline int paged_padding(const PagedCache& c, int b, int new_tokens) {
    if (!c.news) return 0;
    const int n = ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)c.news)[b];
    return new_tokens - min(max(n, 0), new_tokens);
}

// The page and slot of position p (0 <= p < c.reach) of sequence b; false where its entry is no page.
__device__ inline bool paged_find(const PagedCache& c, int b, uint32_t p, uint32_t& page, uint32_t& slot) {
    const uint32_t i = div32(p, c.page);
    slot = p - i * c.page.d;
    page = (uint32_t)c.table[(int64_t)b * c.table_stride + i];
    return page < c.pages;
}

}  // namespace tvk
