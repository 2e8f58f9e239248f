// k_attn_paged.hip -- attention over a K/V cache in pages: its workspace, the choice
// of the type's kernels, and those of f32 caches.  How they work: attn_paged.h.
#include "attn_paged.h"

namespace slate_hip {

int64_t attention_paged_bytes(int hd) {
    return plan_bytes(paged_wgs(hd), hd <= 128 ? 64 : 32, hd <= 64 ? 64 : hd <= 128 ? 128 : 256);
}

template <>
void launch_attention_paged_type<float>(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    launch_paged_hd<float>(a, pb, s);
}

int launch_attention_paged(const PagedAttn& a, const PagedBatch& pb, hipStream_t s) {
    if (a.kv.dtype == KV_F32)
        launch_attention_paged_type<float>(a, pb, s);
    else if (a.kv.dtype == KV_F16)
        launch_attention_paged_type<_Float16>(a, pb, s);
    else
        launch_attention_paged_type<__bf16>(a, pb, s);
    SH_CHECK_LAUNCH();
    return 0;
}

}  // namespace slate_hip
