// attention_pages_bf16.cu -- the paged attention kernels over a bf16 cache.
#include "paged_classes.cuh"

namespace ftc {

FTC_DEVSTAT_READER(devstat_pages_bf16)

namespace paged {

int launch_bf16(const PagedJob& j, int q_dtype) {
    if (q_dtype == FTC_F32) return launch_hd<float, __nv_bfloat16>(j);
    return launch_hd<__nv_bfloat16, __nv_bfloat16>(j);
}

PagedSet geom_bf16(int64_t hd, int q_dtype, int cls) {
    if (q_dtype == FTC_F32) return geom_hd<float, __nv_bfloat16>(hd, cls);
    return geom_hd<__nv_bfloat16, __nv_bfloat16>(hd, cls);
}

}  // namespace paged
}  // namespace ftc
