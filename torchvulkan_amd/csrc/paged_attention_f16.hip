// The paged attention's MFMA kernels for float16 queries.
#include "paged_attention_mfma.h"

namespace tvk {

bool paged_attn_f16(PagedMfmaArgs& p, bool f8, int64_t batch, hipStream_t s) {
    return f8 ? paged_dispatch<TVK_F16, true>(p, batch, s) : paged_dispatch<TVK_F16, false>(p, batch, s);
}

}  // namespace tvk
