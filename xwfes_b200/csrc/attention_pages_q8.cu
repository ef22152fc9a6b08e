// attention_pages_q8.cu -- the paged attention kernels over an 8-bit cache.
#include "paged_classes.cuh"

namespace ftc {

FTC_DEVSTAT_READER(devstat_pages_q8)

namespace paged {

int launch_q8(const PagedJob& j, int q_dtype) {
    if (q_dtype == FTC_F32) return launch_hd<float, int8_t>(j);
    if (q_dtype == FTC_F16) return launch_hd<__half, int8_t>(j);
    return launch_hd<__nv_bfloat16, int8_t>(j);
}

PagedSet geom_q8(int64_t hd, int q_dtype, int cls) {
    if (q_dtype == FTC_F32) return geom_hd<float, int8_t>(hd, cls);
    if (q_dtype == FTC_F16) return geom_hd<__half, int8_t>(hd, cls);
    return geom_hd<__nv_bfloat16, int8_t>(hd, cls);
}

}  // namespace paged
}  // namespace ftc
