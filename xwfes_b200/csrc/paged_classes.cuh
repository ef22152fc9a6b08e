// paged_classes.cuh -- the kernel of each class of sequences, for every type.
#pragma once

#include "attention_pages_tc.cuh"

namespace ftc {
namespace paged {

// Class 3 runs on tcgen05 with 16-bit queries: fp32 ones need their sums kept
// out of the matrix unit's accumulator, and head_dim 256 its tensor memory.
template <typename X, int HD>
constexpr bool kTc = sizeof(X) == 2 && HD < 256;

// fp32 queries over a bf16 cache of head_dim 64 have no 64-row shape: one of
// this type with several groups of warps (not in the tree) stopped with an
// illegal access that reading did not explain, and a shape that no test had run
// is not the place to look for it.  17 to 64 rows take the 128-row shape.
template <typename X, typename C, int HD>
constexpr bool kNo64 = sizeof(X) == 4 && std::is_same<C, __nv_bfloat16>::value && HD == 64;

// The class's shape elsewhere: 4 warps in turn on 8 rows and on 16, one group
// of 4 warps of 16 rows, and of 8 (head_dim 256: 4 again, nine warps leave a
// thread too few registers).  Below 64 rows the tcgen05 kernel does not pay
// over an 8-bit cache (32 sequences of 900 to 6000, 32 heads on 8 of 128, bf16
// q: 24 rows 303 us there, 202 here; 64 rows 316 and 209).  Over 16 bits it
// would (24 rows 151 and 229, 64 rows 164 and 237; head_dim 64 114 and 124, 119
// and 130); one rule for all caches stands for now.
template <typename X, typename C, int HD, class Fn>
auto with_class(int cls, Fn fn) {
    if (cls == 0) return fn((Cfg<X, C, HD, 1, 1, 4>*)nullptr);
    if (cls == 1) return fn((Cfg<X, C, HD, 2, 1, 4>*)nullptr);
    if constexpr (HD == 256 || kTc<X, HD>) {
        return fn((Cfg<X, C, HD, 2, 4, 4>*)nullptr);
    } else {
        if constexpr (!kNo64<X, C, HD>) {
            if (cls == 2) return fn((Cfg<X, C, HD, 2, 4, 4>*)nullptr);
        }
        return fn((Cfg<X, C, HD, 2, 8, 8>*)nullptr);
    }
}

template <typename X, typename C, int HD>
int launch_class(const PagedJob& j) {
    if constexpr (kTc<X, HD>) {
        if (j.cls == 3) return launch_tc<X, C, HD>(j);
    }
    return with_class<X, C, HD>(j.cls, [&](auto* f) {
        return launch_cfg<typename std::remove_pointer<decltype(f)>::type>(j);
    });
}

template <typename X, typename C, int HD>
PagedSet geom_class(int cls) {
    if constexpr (kTc<X, HD>) {
        if (cls == 3) return {device_sms(), TcCfg<X, C, HD>::TR};
    }
    return with_class<X, C, HD>(cls, [&](auto* f) {
        return geom_cfg<typename std::remove_pointer<decltype(f)>::type>();
    });
}

template <typename X, typename C>
int launch_hd(const PagedJob& j) {
    return j.c->head_dim == 64    ? launch_class<X, C, 64>(j)
           : j.c->head_dim == 128 ? launch_class<X, C, 128>(j)
                                  : launch_class<X, C, 256>(j);
}

template <typename X, typename C>
PagedSet geom_hd(int64_t hd, int cls) {
    return hd == 64 ? geom_class<X, C, 64>(cls)
                    : hd == 128 ? geom_class<X, C, 128>(cls) : geom_class<X, C, 256>(cls);
}

}  // namespace paged
}  // namespace ftc
