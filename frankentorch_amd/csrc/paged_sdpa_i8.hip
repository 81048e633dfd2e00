// Attention over a paged cache of scaled 8-bit numbers: the kernels for i8.

#include "paged_sdpa_scaled.hpp"

namespace fth {
namespace paged {

int32_t launch_i8(const ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st) { return launch_scaled<fth::i8>(a, pl, tiles, st); }

}  // namespace paged
}  // namespace fth
