// attention_pages_f16.cu -- the paged attention kernels over an f16 cache.
#include "paged_classes.cuh"

namespace ftc {

FTC_DEVSTAT_READER(devstat_pages_f16)

namespace paged {

int launch_f16(const PagedJob& j, int q_dtype) {
    if (q_dtype == FTC_F32) return launch_hd<float, __half>(j);
    return launch_hd<__half, __half>(j);
}

PagedSet geom_f16(int64_t hd, int q_dtype, int cls) {
    if (q_dtype == FTC_F32) return geom_hd<float, __half>(hd, cls);
    return geom_hd<__half, __half>(hd, cls);
}

}  // namespace paged
}  // namespace ftc
