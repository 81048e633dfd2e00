// How a call of the attention over a paged cache is cut into shares, the same for caches of every type, and the kernel that joins them.

#include "paged_sdpa.hpp"

namespace {

using namespace fth::paged;

// ---- shares joined in their order -----------------------------------------------------------------------------------------

// SL lanes of a wavefront walk the shares of four columns of a row side by side (each over every SL-th of them, in order) and are
// added up in a fixed tree; 64 / SL neighbouring groups of columns make the wavefront. SL grows with the shares, so that no lane
// has more than a few loads to wait for.
template <int SL, bool EVEN> __global__ __launch_bounds__(256) void paged_sdpa_join_kernel(const PagedArgs p, int items) {
    constexpr int CL = 64 / SL;
    fetch_arguments<PagedArgs>();
    const int item = (int)((blockIdx.x * 4 + (threadIdx.x >> 6)) * CL + (threadIdx.x & (CL - 1)));
    const int lane_s = (threadIdx.x & 63) / CL;
    const bool there = item < items;
    const int row32 = there ? (int)p.by_group4((uint32_t)item) : 0, c = there ? (item - row32 * (p.pitch / 4)) * 4 : 0;
    const int token = (int)p.by_q_heads((uint32_t)row32), h = row32 - token * (int)p.d.q_heads;
    const int seq32 = (int)p.by_new((uint32_t)token), i = token - seq32 * (int)p.d.new_tokens;
    const int64_t seq = seq32;
    const int len = p.lens[seq], hk = (int)p.by_group((uint32_t)h), in_pair = (h - hk * p.group) * (int)p.d.new_tokens + i;
    // The slots of the row's shares, `apart` from each other; `first`: the first of even shares may stand further on. Rows of one share
    // are written; so are those of an invalid length.
    int shares = 0;
    int64_t slot0, apart, first = 0;
    const int share = EVEN ? p.starts[p.c.num_seqs] : 0;
    if (!EVEN || share == 0) {
        if (there && len > p.share && len <= p.most) shares = (len - 1) / p.share + 1;
        apart = p.rows;
        slot0 = (seq * p.c.kv_heads + hk) * p.nsplit * apart + in_pair;
    } else {
        const int steps = steps_of(p, len);
        const int begin = p.starts[seq] + hk * (steps + 1) + 1, from = begin / share, to = (begin + steps - 1) / share;
        if (there && steps > 0 && to > from) shares = to - from + 1;
        apart = 2 * p.rows;
        slot0 = from * apart + in_pair;
        if (from * share < begin) first = p.rows;
    }
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml);
    auto slot = [&](int s) __attribute__((always_inline)) { return slot0 + s * apart + (EVEN && s == 0 ? first : 0); };
    const float *o = p.part_o + c;
    float m = -__builtin_inff();
    for (int s = lane_s; s < shares; s += SL) m = fmaxf(m, ml[slot(s)].x);
#pragma unroll
    for (int d = CL; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float ref = m == -__builtin_inff() ? 0.f : m;
    F4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 8
    for (int s = lane_s; s < shares; s += SL) {
        const float2 part = ml[slot(s)];
        const F4 v = *reinterpret_cast<const F4 *>(o + slot(s) * p.pitch);
        const float w = __builtin_amdgcn_exp2f(part.x - ref);
        l += part.y * w;
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += v[j] * w;
    }
#pragma unroll
    for (int d = CL; d < 64; d <<= 1) {
        l += __shfl_xor(l, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], d);
    }
    if (shares == 0 || lane_s != 0) return;
    float *dst = out_row(p, seq, i, h) + c;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < p.c.head_dim) dst[j] = acc[j] / l;
}
// ---- host -------------------------------------------------------------------------------------------------------------------

}  // namespace

namespace fth {
namespace paged {

Plan plan(const fth_paged_cache &c, const fth_paged_sdpa_desc &d) {
    Plan p;
    const int64_t size = fth::element_size(c.dtype), ch = 16 / size;
    p.rows = c.num_seqs * d.new_tokens * d.q_heads;
    p.tiles = c.head_dim % ch == 0 && c.row_stride % ch == 0 && c.head_stride % ch == 0 && c.page_stride % ch == 0 &&
              c.row_stride <= ((int64_t)1 << 24) && c.num_pages > 0;
    p.pitch = (int)fth::ceil_div(c.head_dim, 4) * 4;
    const int64_t most = p.most = c.max_pages * c.page_size < d.max_len ? c.max_pages * c.page_size : d.max_len;
    p.row_tiles = fth::ceil_div(d.q_heads / c.kv_heads * d.new_tokens, 16);
    const int64_t pairs = c.num_seqs * c.kv_heads, units = p.tiles ? pairs * p.row_tiles : p.rows;
    const int64_t key_bytes = 2 * c.head_dim * size;
    // Shares of one length: about 256 workgroups, of 256 keys at least. A join costs 4 to 5 us, so nothing is cut that fills the chip whole (32
    // sequences of 1000 keys: 18.6 us in one share, 23.6 in two) or has 512 keys (8 K/V heads of 128: 10.5 / 12.0). 128 keys where 256
    // would not make 128 workgroups (12 heads of 64, 1024 keys: 10.6 / 12.4; 8 of 128, 4096 keys: 13.4 / 14.7). From 129 workgroups on one
    // share each (8 heads of 128, up to 4000 keys, bf16, one / two shares: 24 sequences 57 / 63.5, 31 64 / 69, fp32 24 123 / 136, up to 1000 keys 15.3 / 20;
    // 17 sequences 51.5 / 42.7).
    // In a batch that fills the chip, shares of 512 KB where a sequence has more than 1 MB: the chip does not wait for the longest one
    // (64 of up to 8191 keys, bf16: 244 us in one share each, 224 in shares of 1 MB, 218 of 512 KB, 227 of 256 KB; 64 of up to 4000,
    // fp32: 255, 232, 225, 234; 32 of up to 1000, fp32: 39 in one, 45 in 512 KB). At most 16 of the longest: where max_len is far
    // above the lengths, workgroups without keys take the time (256 sequences of 300 keys, max_len 131072: 248 us in 128 shares, 96).
    const int64_t step = kTile * kWaves, least = units * fth::ceil_div(most, 256) <= 128 ? 128 : 256;
    static_assert(step == 1 << 7, "a step is a tile of every wavefront");
    const bool large = units >= 256 && most * key_bytes > (1 << 20);
    int64_t share = fth::ceil_div(most, units > 0 && units < 256 ? 256 / units : 1);
    if (large) {
        const int64_t part = fth::ceil_div(most, 16), cut = (512 << 10) / key_bytes > part ? (512 << 10) / key_bytes : part;
        share = share < cut ? share : cut;
    }
    share = share < least ? least : share;
    if (p.tiles && most <= 512) share = most;
    p.share = (int)(fth::ceil_div(share > 0 ? share : 1, step) * step);
    p.nsplit = (int)fth::ceil_div(most, p.share);
    if (p.nsplit < 1) p.nsplit = 1;
    // There even shares are better for up to 256 sequences that turn out to have 576 KB each on average, at one workgroup a compute unit
    // (us, shares of 512 KB / even ones: 64 of up to 8191, bf16: 225 / 204; 64 of up to 4000, fp32: 225 / 202; 64 on 12 heads of 64 of
    // up to 5000, bf16: 117 / 103; 128 on heads of 256 of up to 1500, bf16: 198 / 165; 512 of 1000 on one head: 51 / 56, 1024 of 20 keys:
    // 19 / 33, where beginning a pair costs more than waiting for one), two where their tiles would not keep enough bytes on the way (the first
    // of these: 204 / 209, the second 202 / 210, heads of 64, bf16: 108 / 103).
    // Caches of 8 bits by the same bytes (us): even / shares of 512 KB / one each, 64 of up to 8191 120 / 132 / 139, on 12 heads of 64 of up to 12000 129 / 136 /
    // 153, 128 on heads of 256 of up to 3000 180 / 213 / 183; shares from 512 KB on instead, 64 of up to 3000 56 / 60, on 12 heads of 64 of up to 5000 69 / 77, 128 on
    // heads of 256 of up to 1500 104 / 129; two workgroups a compute unit / one, the first two of these 120 / 129 and 129 / 156.
    p.even = p.enough = 0;
    p.step_log2 = 7;
    if (p.tiles && large && c.num_seqs <= 256) {
        p.even = (int)((key_bytes < 512 ? 512 : 256) / p.row_tiles / 8 * 8);
        p.even = p.even < 8 ? 8 : p.even;
        while (pairs * ((most >> p.step_log2) + 2) > (1 << 30)) ++p.step_log2;  // places in the line are 32-bit numbers
        const int64_t enough = pairs * fth::ceil_div((int64_t)(576 << 10) / key_bytes, (int64_t)1 << p.step_log2);
        p.enough = (int)(enough < 2147483647LL ? enough : 2147483647LL);
    }
    // Nontemporal loads for what the 256 MB last-level cache cannot hold until the next call, if sequences are half of max_len on
    // average, and that is read once (us, with / without: one sequence of 131071, bf16 87 / 99, fp32 180 / 196; 64 of up to 8191,
    // bf16 217 / 229 in shares of 512 KB; 16 of up to 3967, four queries, f16, 260 MB 38.5 / 36.3, fp32, 520 MB 79 / 72; by the even
    // shares of today 196 / 220). The host knows the bound alone: where it is far above the lengths, calls that read one cache again and
    // again lose (under 131072: 4 sequences of 3000 keys 47.5 / 34, 16 of 1000 22.4 / 17.2, 64 of 300 or 600 level). Caches of 8 bits, with / without: 64 of up to
    // 8191 120 / 127, on 12 heads of 64 of up to 12000 129 / 137, 128 on heads of 256 of up to 3000 180 / 186; below the bound 64 of up to 4000 level, 24 38.6 / 34.2, one
    // of 131071, 269 MB, 50.6 / 55.5 where two take turns and 49 / 46 where it is read again.
    p.nt = p.row_tiles == 1 && 2.0 * (double)c.num_seqs * (double)most * (double)c.kv_heads * (double)c.head_dim * (double)size > 500.0 * (1 << 20);
    return p;
}

// Partial results: of the shares of every row, or of two pairs a share.
static int64_t slots_of(const Plan &p, const fth_paged_cache &c, bool tiles) {
    const int64_t one = p.nsplit > 1 ? p.rows * p.nsplit : 0, even = tiles && p.even ? 2 * p.even * (p.rows / (c.num_seqs * c.kv_heads)) : 0;
    return even > one ? even : one;
}
size_t workspace_bytes_of(const Plan &p, const fth_paged_cache &c) {
    return (size_t)slots_of(p, c, true) * (p.pitch + 2) * sizeof(float) + (p.even ? (size_t)(c.num_seqs + 1) * sizeof(int32_t) : 0);
}

int32_t check(const fth_paged_cache *c, const fth_paged_sdpa_desc *d, bool scaled) {
    if (int32_t rc = fth::check_paged_cache(c, "paged_sdpa", scaled)) return rc;
    FTH_ARG(d, "paged_sdpa: NULL descriptor");
    if (d->q_heads > (1 << 24)) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "paged_sdpa: more than 2^24 query heads");
    FTH_ARG(d->q_heads >= 1 && d->q_heads % c->kv_heads == 0, "paged_sdpa: %lld query heads on %lld K/V heads", (long long)d->q_heads, (long long)c->kv_heads);
    FTH_ARG(d->new_tokens >= 1 && d->new_tokens <= 8, "paged_sdpa: new_tokens %lld is outside 1..8", (long long)d->new_tokens);
    FTH_ARG(d->max_len >= 0 && d->max_len <= (1 << 30), "paged_sdpa: max_len %lld is outside 0..2^30", (long long)d->max_len);
    for (int64_t x : {d->q_seq_stride, d->q_row_stride, d->q_head_stride, d->o_seq_stride, d->o_row_stride, d->o_head_stride})
        FTH_ARG(fth::stride_in_range(x), "paged_sdpa: a stride is negative or over 2^40");
    int64_t rows = 0;
    if (__builtin_mul_overflow(c->num_seqs * d->new_tokens, d->q_heads, &rows) || rows > (1 << 24))
        return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "paged_sdpa: more than 2^24 query rows");
    return FTH_OK;
}

bool fill_args(PagedArgs &a, const fth_paged_cache &c, const fth_paged_sdpa_desc &d, const Plan &pl, float scale, const float *q, const void *k_cache, const void *v_cache,
               const int32_t *block_table, const int32_t *lens, float *out, int64_t *bad_index, void *workspace) {
    a.c = c;
    a.d = d;
    a.q = q; a.k = k_cache; a.v = v_cache; a.table = block_table; a.lens = lens; a.out = out; a.bad = bad_index;
    a.part_o = static_cast<float *>(workspace);
    const bool tiles = pl.tiles && (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15u) == 0;
    const int64_t slots = slots_of(pl, c, tiles);
    a.part_ml = a.part_o + slots * pl.pitch;
    a.starts = reinterpret_cast<int32_t *>(a.part_ml + 2 * slots);
    a.scale2 = scale * kLog2e;
    a.most = pl.most;
    a.group = (int)(d.q_heads / c.kv_heads);
    a.rows = a.group * (int)d.new_tokens;
    a.row_tiles = (int)pl.row_tiles;
    a.nsplit = pl.nsplit; a.share = pl.share; a.pitch = pl.pitch;
    a.even = tiles ? pl.even : 0; a.enough = pl.enough; a.step_log2 = pl.step_log2;
    a.seqs_a_lane = (int)fth::ceil_div(c.num_seqs, 64);
    a.pairs = (int)(c.num_seqs * c.kv_heads);
    a.by_page = fth::Divisor((uint32_t)c.page_size);
    a.by_tiles = fth::Divisor((uint32_t)a.row_tiles);
    a.by_pairs = fth::Divisor((uint32_t)a.pairs);
    a.by_even = fth::Divisor((uint32_t)(a.even ? a.even : 1));
    a.by_heads = fth::Divisor((uint32_t)c.kv_heads);
    a.by_new = fth::Divisor((uint32_t)d.new_tokens);
    a.by_q_heads = fth::Divisor((uint32_t)d.q_heads);
    a.by_group = fth::Divisor((uint32_t)a.group);
    a.by_group4 = fth::Divisor((uint32_t)(a.pitch / 4));
    return tiles;
}

int64_t tiles_grid(const PagedArgs &a) {
    const int64_t cut = (int64_t)a.pairs * a.nsplit;
    return fth::ceil_div(cut > a.even ? cut : a.even, 8) * 8 * a.row_tiles;
}

int32_t launch_join(const PagedArgs &a, const Plan &pl, hipStream_t st) {
    if (a.even || a.nsplit > 1) {
        const int items = (int)(pl.rows * (a.pitch / 4));  // at most 2^24 rows of 64 groups
        // (us, 1 / 4 / 16 / 64 lanes: 2048 rows of up to 16 shares 5.9 / 5.1 / 11.8 / 41; 32 rows of 256 shares 44 / 15 / 9.6 / 6.3)
        // (in a batch that fills the chip a row has about one share, though the longest have more)
        const int lanes = a.nsplit <= 4 ? 1 : a.nsplit <= 16 || a.even ? 4 : a.nsplit <= 64 ? 16 : 64;
        const dim3 blocks((unsigned)fth::ceil_div((int64_t)items * lanes, 256));
        auto go = [&](auto kernel) { kernel<<<blocks, dim3(256), 0, st>>>(a, items); };
        if (a.even) go(lanes == 1 ? paged_sdpa_join_kernel<1, true> : paged_sdpa_join_kernel<4, true>);
        else if (lanes == 1) go(paged_sdpa_join_kernel<1, false>);
        else if (lanes == 4) go(paged_sdpa_join_kernel<4, false>);
        else if (lanes == 16) go(paged_sdpa_join_kernel<16, false>);
        else go(paged_sdpa_join_kernel<64, false>);
        FTH_CHECK_LAUNCH("paged_sdpa_join");
    }
    return FTH_OK;
}

}  // namespace paged
}  // namespace fth
