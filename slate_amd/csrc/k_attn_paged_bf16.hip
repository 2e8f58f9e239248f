// k_attn_paged_bf16.hip -- attention over a K/V cache in pages: the kernels of bf16 caches.
#include "attn_paged.h"

namespace slate_hip {

template <>
void launch_attention_paged_type<__bf16>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    launch_paged_hd<__bf16>(a, pb, s);
}

}  // namespace slate_hip
