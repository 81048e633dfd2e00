// Attention of the last one to eight tokens of every sequence over a paged K/V cache of 8-bit numbers: the entry points.

#include "paged_sdpa_scaled.hpp"

using namespace fth::paged;

extern "C" {

size_t fth_dev_paged_sdpa_scaled_workspace_bytes(const fth_paged_cache *c, const fth_paged_scales *sc, const fth_paged_sdpa_desc *d) {
    return check(c, d, true) == FTH_OK && fth::check_paged_scales(sc, c, "paged_sdpa_scaled") == FTH_OK ? workspace_bytes_of(plan(*c, *d), *c) : 0;
}

int32_t fth_dev_paged_sdpa_scaled_f32(const fth_paged_cache *c, const fth_paged_scales *sc, const fth_paged_sdpa_desc *d, float scale, const float *q, const void *k_cache,
                                      const void *v_cache, const float *k_scales, const float *v_scales, const int32_t *block_table, const int32_t *lens, float *out,
                                      int64_t *bad_index, void *workspace, size_t workspace_bytes, fth_stream s) {
    if (int32_t rc = check(c, d, true)) return rc;
    if (int32_t rc = fth::check_paged_scales(sc, c, "paged_sdpa_scaled")) return rc;
    FTH_ARG(c->num_seqs == 0 || (q && lens && out && (block_table || c->max_pages == 0) && ((k_cache && v_cache && k_scales && v_scales) || c->num_pages == 0)),
            "paged_sdpa_scaled: NULL operand");
    const Plan pl = plan(*c, *d);
    const size_t need = workspace_bytes_of(pl, *c);
    FTH_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15u) == 0), "paged_sdpa_scaled: needs a workspace of %zu bytes, 16-byte aligned", need);
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("paged_sdpa_scaled(bad_index reset)");
    }
    if (c->num_seqs == 0) return FTH_OK;
    ScaledArgs a;
    const bool tiles = fill_args(a, *c, *d, pl, scale, q, k_cache, v_cache, block_table, lens, out, bad_index, workspace);
    a.sc = *sc;
    a.k_scales = k_scales; a.v_scales = v_scales;
    a.by_block = fth::Divisor((uint32_t)sc->block);
    return c->dtype == FTH_DTYPE_I8 ? launch_i8(a, pl, tiles, st) : launch_e4m3(a, pl, tiles, st);
}

}  // extern "C"
