// k_attn_paged_f16.hip -- attention over a K/V cache in pages: the kernels of f16 caches.
#include "attn_paged.h"

namespace slate_hip {

template <>
void launch_attention_paged_type<_Float16>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    launch_paged_hd<_Float16>(a, pb, s);
}

}  // namespace slate_hip
