// Attention over a paged cache of 8-bit numbers, each block of positions and head with a scale.
#pragma once

#include "paged_sdpa.hpp"

namespace fth {
namespace paged {

struct ScaledArgs : PagedArgs {
    static constexpr bool kScaled = true;
    fth_paged_scales sc;
    const float *k_scales, *v_scales;
    fth::Divisor by_block;
};

template <typename T> int32_t launch_scaled(ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st) {
    a.even = 0;
    FTH_ARG(pl.rows * a.nsplit <= 2147483647LL, "paged_sdpa_scaled: too many rows for one launch");
    paged_sdpa_rows_kernel<T, ScaledArgs><<<dim3((unsigned)(pl.rows * a.nsplit)), dim3(64), 0, st>>>(a);
    FTH_CHECK_LAUNCH("paged_sdpa_scaled");
    return launch_join(a, pl, st);
}

int32_t launch_e4m3(ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st);
int32_t launch_i8(ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st);

}  // namespace paged
}  // namespace fth
