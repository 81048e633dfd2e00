// Attention of the last one to eight tokens of every sequence over a paged K/V cache of 8-bit numbers, each block of positions and
// head with a scale.
//
//   out = sum_j w_j s'_j v_j / sum_j w_j,   w_j = exp(x_j - max x),   x_j = scale s_j (q . k_j),   k, v codes, s, s' the scales of the key's blocks
//
// Bound by reading the cache once. Shares, tiles of 32 keys and the way keys and query rows lie in the lanes are those of the kernels
// for 16-bit caches; both products run on the 16-bit matrix units against codes turned into numbers of 16 bits, which hold them exactly:
//   * K as f16, against a query row scaled by a power of two and cut into two parts of f16 (22 bits of an element, or 2^-39 of the row's largest). A
//     score meets the scale of its key's block in fp32 afterwards.
//   * V as bf16, against weights that have met the scale of their key's block in fp32 and are cut into three parts of bf16, whose sum they
//     are. They carry a factor of 2^40, which keeps the third part of every weight an output of fp32 can show above the smallest bf16; where that
//     overflows (scales of V beyond 2^70) the share is walked twice more, for the keys with scales of V below 2^48, and for the others with 2^-24.
// e4m3 becomes either type two at a time by one instruction of gfx950; whole numbers become f16 by the bits of 1024 + 128 + x, bf16 through fp32.
//
// Measured: 64 sequences of 1024 to 8191 keys, 32 query heads on 8 of 128, e4m3, blocks of 16 (614 MB): 111 us, 5.6 TB/s (one wavefront a row 3660;
// a bf16 cache of the same keys, 1.22 GB, 193). One sequence of 131071: 53 us (5.1 TB/s). 16 of up to 3967, four queries, i8: 27.6. Bound by the loads, of which the
// two workgroups of a compute unit keep too few bytes on the way: the loop without its products takes 110 / 49 / 26 us. Of two workgroups with equal
// shares the older one ends at 82 us, the younger at 105; lengthening the shares of the older by 6 to 25 % was level, and so were three workgroups a
// compute unit, tiles of 64 keys, raised wavefront priorities, and twice or four times as many shares (one sequence: 57 / 58 / 60).
// Half tiles looked up 64 at a time took the loop from 460 to 330 instructions a tile (134 -> 111 us).
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

using H2 = _Float16 __attribute__((ext_vector_type(2)));
using H8 = _Float16 __attribute__((ext_vector_type(8)));
using B2 = __bf16 __attribute__((ext_vector_type(2)));
using B8 = __bf16 __attribute__((ext_vector_type(8)));
using ConstF = const float __attribute__((address_space(4))) *;

// Where the scales of 16 keys come from: one number (blocks and pages are multiples of 16: a scalar load); one for each four (blocks are
// multiples of 4, pages of 16); one for each key, four in a 128-bit load (blocks of one, pages of 16); one for each key, whose page every
// lane looks up (any pages and blocks).
enum class ScaleOf { sixteen, four, one, any };

// 8 codes (two words) as f16.
template <typename T> __device__ __forceinline__ H8 to_f16(uint32_t a, uint32_t b) {
    H2 x[4];
    const uint32_t w[2] = {a, b};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (std::is_same<T, fth::e4m3>::value) {
            x[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.f, false);
            x[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w[i], 1.f, true);
        } else {  // 0x6400 + u is the f16 1024 + u; u = 128 + the number
            const uint32_t u = w[i] ^ 0x80808080u;
            const H2 bias = {(_Float16)1152.f, (_Float16)1152.f};
            x[2 * i] = __builtin_bit_cast(H2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
            x[2 * i + 1] = __builtin_bit_cast(H2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
        }
    }
    return H8{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

// Byte b (a constant) of two words as two bf16.
template <typename T> __device__ __forceinline__ uint32_t to_bf16(uint32_t first, uint32_t second, int b) {
    if constexpr (std::is_same<T, fth::e4m3>::value) {
        const uint32_t pairs = __builtin_amdgcn_perm(second, first, b < 2 ? 0x05010400u : 0x07030602u);  // bytes 0 and 1 (2 and 3) of both
        return __builtin_bit_cast(uint32_t, (b & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)pairs, 1.f, true)
                                                    : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)pairs, 1.f, false));
    } else {  // 8 bits: the upper halves of fp32
        const float x = (float)(int8_t)(first >> (8 * b)), y = (float)(int8_t)(second >> (8 * b));
        return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    }
}

// Bit 7 of every byte that is a NaN of e4m3.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// One segment: keys key_lo .. key_hi - 1 of a pair of `len` keys, with row tile rt of its queries. FULL: head_dim == DP; otherwise what lies past
// head_dim counts as zero. NT: K and V leave no trace in the caches.
template <typename T, int DP, bool FULL, bool NT, ScaleOf OF>
__device__ __forceinline__ void scaled_segment(const ScaledArgs &p, float *lds_o, float *lds_ml, int seq32, int hk, int rt, int len, bool bad, int key_lo, int key_hi, bool alone, int64_t slot0) {
    constexpr bool ANY = OF == ScaleOf::any, SIXTEEN = OF == ScaleOf::sixteen, FOUR = OF == ScaleOf::four, kNan = std::is_same<T, fth::e4m3>::value;
    constexpr int NK = DP / 64;   // 128-bit loads of a lane's quarter of a K row
    constexpr int NE = DP / 16;   // output columns of a lane, consecutive ones
    constexpr int NV = NE / 4;    // words of its part of a V row
    constexpr int NS = SIXTEEN || FOUR ? 1 : 4;  // scales of a lane's four keys
    constexpr int NL = ANY ? 1 : NS;             // as they are loaded: ANY has that of this lane's row
    constexpr int H = 2, kKeys = 16 * H;  // 16 keys so many times make a tile of a wavefront
    const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t seq = seq32;
    const int hd = (int)p.c.head_dim, new_tokens = (int)p.d.new_tokens, rows = p.rows;
    const int tiles = (key_hi - key_lo + kKeys - 1) / kKeys, last16 = (key_hi - 1) >> 4;
    const uint8_t *K = static_cast<const uint8_t *>(p.k) + hk * p.c.head_stride, *V = static_cast<const uint8_t *>(p.v) + hk * p.c.head_stride;
    const float *KS = p.k_scales + hk * p.sc.head_stride, *VS = p.v_scales + hk * p.sc.head_stride;
    const Const table = constant(p.table) + seq * p.c.table_stride;
    const int t16_lo = key_lo >> 4;
    const int rs = (int)p.c.row_stride, num_pages = (int)p.c.num_pages;
    if (len == 0) {
        store_empty(p, seq, hk, rt, bad);
        return;
    }

    // this lane's query row (rows past the last repeat it and are never stored) and how many keys it sees
    int rr = rt * 16 + lr;
    rr = rr < rows ? rr : rows - 1;
    const int in_group = (int)p.by_new((uint32_t)rr), qi = rr - in_group * new_tokens, qh = hk * p.group + in_group;
    const int sees = len - new_tokens + 1 + qi;
    const float *qr = p.q + seq * p.d.q_seq_stride + qi * p.d.q_row_stride + qh * p.d.q_head_stride;
    float q[2 * NK][8];
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = (4 * (i / 2) + g) * 16 + 8 * (i % 2) + e;
            q[i][e] = FULL || c < hd ? qr[c] : 0.f;
        }

    // The 16 keys number t16 (of the sequence): the page and the row in it of the first (ANY: of this lane's); half tiles past the
    // end repeat the last one (ANY: keys past the end repeat the last one).
    auto page_of = [&](int t16) __attribute__((always_inline)) {
        int key;
        if constexpr (ANY) {
            key = (t16 << 4) + lr;
            key = key < len ? key : len - 1;
        } else {
            key = (t16 < last16 ? t16 : last16) << 4;
        }
        const int index = (int)p.by_page((uint32_t)key);
        return make_int2(table[index], key - index * (int)p.c.page_size);
    };
    struct Place {
        int64_t row;   // the offset of the row
        int64_t page;  // of the page's scales
        int in_page;   // the row in its page
    };
    auto place_of = [&](int2 page) __attribute__((always_inline)) {
        const bool there = page.x >= 0 && page.x < num_pages;
        bad = bad || !there;
        return Place{(int64_t)(there ? page.x : 0) * p.c.page_stride + (int64_t)page.y * rs, (int64_t)(there ? page.x : 0) * p.sc.page_stride, page.y};
    };
    // Where the next 64 of this wavefront's half tiles are, one a lane (a half tile costs some 60 scalar instructions by itself, as many
    // as half of its products take): half tile j is number t16_lo + H wave + s + H kWaves (j / H), s = j % H.
    Place mine;
    float my_ks = 0.f, my_vs = 0.f;  // SIXTEEN: the scales
    auto page_ahead = [&](int j0) __attribute__((always_inline)) {
        const int j = j0 + lane, t16 = t16_lo + H * wave + j % H + H * kWaves * (j / H), key = (t16 < last16 ? t16 : last16) << 4, index = (int)p.by_page((uint32_t)key);
        return make_int2(p.table[seq * p.c.table_stride + index], key - index * (int)p.c.page_size);
    };
    int2 ahead64;
    // Which keys this walk has, 0: all, 1: those with scales of V below 2^48, 2: the others; their scales (of the others: 0).
    int part = 0;
    bool others = false;
    auto of_part = [&](float s) __attribute__((always_inline)) {
        if (part == 0) return s;
        const bool below = fabsf(s) < 0x1p48f;
        others |= !below;
        return below == (part == 1) ? s : 0.f;
    };
    auto look_ahead = [&](int j0) __attribute__((always_inline)) {
        mine = place_of(ahead64);
        if constexpr (SIXTEEN) {
            const int64_t at = mine.page + p.by_block((uint32_t)mine.in_page);
            my_ks = KS[at];
            my_vs = VS[at];
            my_vs = of_part(my_vs);
        }
        ahead64 = page_ahead(j0 + 64);
    };
    auto one_of = [&](int64_t x, int j) __attribute__((always_inline)) {
        return (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)x, j);
    };
    auto half_tile = [&](int j) __attribute__((always_inline)) {
        Place at = {one_of(mine.row, j & 63), 0, 0};
        if constexpr (!SIXTEEN) {
            at.page = one_of(mine.page, j & 63);
            at.in_page = __builtin_amdgcn_readlane(mine.in_page, j & 63);
        }
        return at;
    };
    // the offset of row `row` of a half tile
    auto row_offset = [&](const Place &at, int row) __attribute__((always_inline)) {
        if constexpr (ANY) return (int64_t)__shfl((int)(at.row >> 32), row) << 32 | (uint32_t)__shfl((int)at.row, row);
        return at.row + row * rs;
    };
    U4 kf[H][NK];
    uint32_t vf[H][4][NV];
    float ks[H][NL], vs[H][NL];  // of 16 keys, of this lane's keys 4 g .. 4 g + 3, or of each of them
    const uint32_t k_lane = (uint32_t)((ANY ? 0 : lr * rs) + g * 16);
    uint32_t v_lane[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v_lane[r] = (uint32_t)((ANY ? 0 : (4 * g + r) * rs) + lr * NE);
    auto load_scales = [&](float (&s)[H][NL], const float *from, const Place (&at)[H]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if constexpr (SIXTEEN) {  // in the lanes, see above
            } else if constexpr (ANY) {
                s[h][0] = from[at[h].page + p.by_block((uint32_t)at[h].in_page)];  // (handed round where it is used: it is on its way until then)
            } else if constexpr (FOUR) {
                s[h][0] = from[at[h].page + p.by_block((uint32_t)(at[h].in_page + 4 * g))];
            } else {
                const F4 x = *reinterpret_cast<const F4 *>(from + at[h].page + at[h].in_page + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[h][r] = x[r];
            }
        }
    };
    auto load_k = [&](const Place (&at)[H]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < H; ++s) {
            const uint8_t *base = K + at[s].row;
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                if (!FULL) kf[s][i] = U4{0u, 0u, 0u, 0u};
                if (FULL || (4 * i + g) * 16 < hd) kf[s][i] = load128<NT>(base + k_lane + 64 * i);
            }
        }
        load_scales(ks, KS, at);
    };
    auto load_v = [&](const Place (&at)[H]) __attribute__((always_inline)) {
        using Row = uint32_t __attribute__((ext_vector_type(NV)));
#pragma unroll
        for (int s = 0; s < H; ++s) {
            const uint8_t *base = V + at[s].row;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (ANY) base = V + row_offset(at[s], 4 * g + r);
                if (!FULL)
#pragma unroll
                    for (int i = 0; i < NV; ++i) vf[s][r][i] = 0u;
                if (FULL || lr * NE < hd) {
                    const Row *src = reinterpret_cast<const Row *>(base + v_lane[r]);
                    const Row w = NT ? __builtin_nontemporal_load(src) : *src;
#pragma unroll
                    for (int i = 0; i < NV; ++i) vf[s][r][i] = w[i];
                }
            }
        }
        load_scales(vs, VS, at);
    };

    int2 ahead[H];  // ANY: of the next tile
    auto begin = [&]() __attribute__((always_inline)) {
        Place at[H];
        if constexpr (ANY) {
            int2 now[H];
#pragma unroll
            for (int s = 0; s < H; ++s) {
                now[s] = page_of(t16_lo + H * wave + s);
                ahead[s] = page_of(t16_lo + H * (wave + kWaves) + s);
            }
#pragma unroll
            for (int s = 0; s < H; ++s) at[s] = place_of(now[s]);
        } else {
            ahead64 = page_ahead(0);
            look_ahead(0);
            __builtin_amdgcn_sched_barrier(0);  // the scales before K and V: who waits for them would wait for V
#pragma unroll
            for (int s = 0; s < H; ++s) at[s] = half_tile(s);
        }
        load_k(at);  // (a wavefront without a tile reads the last one)
        load_v(at);
    };
    begin();
    __builtin_amdgcn_sched_barrier(0);

    // The query row times a power of two that brings its largest element to [2^14, 2^15), in two parts (one that is not finite gives NaN).
    H8 qp[2][2 * NK];
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(q[i][e]));
    big = rows_reduce(big, MaxOp());
    const int up = big > 0.f && big < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(big) : 0;
    // What a score is multiplied by beside its key's scale: 2^-up scale2, of which `rest` has the power of two that would take it out of range (queries near
    // the ends of float32).
    const int over = __builtin_amdgcn_frexp_expf(p.scale2) - up, cut = over > 96 ? over - 96 : over < -96 ? over + 96 : 0;
    const float factor = __builtin_ldexpf(p.scale2, -up - cut), rest = __builtin_ldexpf(1.f, cut);
    const bool far = __any(cut != 0);
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = __builtin_ldexpf(q[i][e], up);
            qp[0][i][e] = (_Float16)x;
            qp[1][i][e] = (_Float16)(x - (float)qp[0][i][e]);
        }

    F4 o[NE], before[NE];          // of the last tiles; of those before them
    float m_run, l_run, l_before;  // likewise the sums of the weights, of this lane's keys only
    const int limit = sees < key_hi ? sees : key_hi;

    // One tile. `more` (a constant): another one of this wavefront follows, whose loads go out on the way (what a query
    // may not see lies in the last two tiles of the sequence, which are the last ones of their wavefronts). `unit`: the factor of the weights.
    auto step = [&](int t, float unit, auto more) __attribute__((always_inline)) {
        const int key0 = key_lo + t * kKeys;
        F4 sc[H], low[H];
#pragma unroll
        for (int s = 0; s < H; ++s) sc[s] = low[s] = F4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i)
#pragma unroll
            for (int s = 0; s < H; ++s) {
                const H8 k8 = to_f16<T>(kf[s][i / 2][2 * (i % 2)], kf[s][i / 2][2 * (i % 2) + 1]);
                low[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qp[1][i], low[s], 0, 0, 0);
                sc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qp[0][i], sc[s], 0, 0, 0);
            }
        float by[H][NS];
        const int j = H * (t - wave) / kWaves;
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
            for (int r = 0; r < NS; ++r) {
                if constexpr (SIXTEEN) {
                    ks[s][r] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_ks), (j + s) & 63));
                    vs[s][r] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_vs), (j + s) & 63));
                }
                const float k_scale = ANY ? __shfl(ks[s][0], 4 * g + r) : ks[s][r % NL];
                by[s][r] = __builtin_fmaf(k_scale, 0.f, k_scale * factor);  // NaN for an infinite one, whatever its scores' sign (V's give NaN by their parts)
            }
        if (far || (!SIXTEEN && part > 0)) {
#pragma unroll
            for (int s = 0; s < H; ++s) {
#pragma unroll
                for (int r = 0; r < NS; ++r) by[s][r] *= rest;
                if constexpr (!SIXTEEN)
#pragma unroll
                    for (int r = 0; r < NL; ++r) vs[s][r] = of_part(vs[s][r]);
            }
        }
        Place next[H];
        if constexpr (more) {
            if constexpr (ANY) {
#pragma unroll
                for (int s = 0; s < H; ++s) {
                    next[s] = place_of(ahead[s]);
                    ahead[s] = page_of(t16_lo + H * (t + 2 * kWaves) + s);
                }
            } else {
                if (((j + H) & 63) == 0) look_ahead(j + H);
#pragma unroll
                for (int s = 0; s < H; ++s) next[s] = half_tile(j + H + s);
            }
            load_k(next);
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = (sc[s][r] + low[s][r]) * by[s][NS == 1 ? 0 : r];
                sc[s][r] = more || key0 + 16 * s + 4 * g + r < limit ? x : -__builtin_inff();
                mx = fmaxf(mx, sc[s][r]);
            }
        mx = rows_reduce(mx, MaxOp());
        if (__any(mx > m_run)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -__builtin_inff() ? 0.f : m_new));
            m_run = m_new;
            l_run *= alpha;
            l_before *= alpha;
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    o[e][r] *= alpha;
                    before[e][r] *= alpha;
                }
        }
        // nothing visible so far: every weight is exp(-inf) = 0; a key that is not seen has weight 0 whatever its scale is
        const float ref = m_run == -__builtin_inff() ? 0.f : m_run;
        float w[H][4], l_tile = 0.f;
#pragma unroll
        for (int s = 0; s < H; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(sc[s][r] - ref);
                l_tile += e;
                const float v_scale = ANY ? __shfl(vs[s][0], 4 * g + r) : vs[s][NS == 1 ? 0 : r % NL];
                w[s][r] = more || key0 + 16 * s + 4 * g + r < limit ? e * (v_scale * unit) : 0.f;
            }
        l_run += l_tile;
        // A NaN code under a weight of 0 would be NaN: what lies past the keys counts as zero, and so does, in keys that only the later of the new
        // tokens see, a NaN, which is added below to the rows that see it.
        const int partly = len - new_tokens + 1;
        bool held = false;
        if constexpr (kNan && !more) {
#pragma unroll
            for (int s = 0; s < H; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = key0 + 16 * s + 4 * g + r;
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const uint32_t nan = key >= partly && key < key_hi ? nan_bytes(vf[s][r][i]) : 0u;
                        held |= nan != 0u;
                        vf[s][r][i] = key >= key_hi ? 0u : vf[s][r][i] & ~((nan >> 7) * 255u);
                    }
                }
        }
        // The weights in three parts of bf16, and the products with the columns of V, 32 keys at a time.
#pragma unroll
        for (int two = 0; two < H; two += 2) {
            B8 wp[3];
#pragma unroll
            for (int j = 0; j < 3; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float &x = w[two + (e >> 2)][e & 3];
                    wp[j][e] = (__bf16)x;
                    x -= (float)wp[j][e];
                }
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                U4 column;
#pragma unroll
                for (int j = 0; j < 4; ++j) column[j] = to_bf16<T>(vf[two + (j >> 1)][2 * (j & 1)][e / 4], vf[two + (j >> 1)][2 * (j & 1) + 1][e / 4], e % 4);
#pragma unroll
                for (int j = 2; j >= 0; --j) o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, column), wp[j], o[e], 0, 0, 0);
            }
        }
        if constexpr (kNan && !more) {
            if (__any(held)) {
                const int from = partly > key0 ? partly : key0, to = key_hi < key0 + kKeys ? key_hi : key0 + kKeys;
                for (int key = from; key < to; ++key) {
                    const Place place = place_of(page_of(key >> 4));
                    const uint8_t *vr = V + row_offset(place, key & 15);
#pragma unroll
                    for (int e = 0; e < NE; ++e)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int c = (4 * g + r) * NE + e;
                            if (key < sees && (FULL || c < hd) && (vr[c] & 127) == 127) o[e][r] = __builtin_nanf("");
                        }
                }
            }
        }
        if constexpr (more) {
            load_v(next);
            // Every eighth tile the sums begin anew: a sum over tens of thousands of keys that a few outweigh drops the others' last bits all to one
            // side (28000 keys in one share: sums of weights were off by up to 200 units of 2^-24), and those of the matrix units err to one side too.
            if ((j & (8 * H - 1)) == 7 * H) {
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    before[e] += o[e];
                    o[e] = F4{0.f, 0.f, 0.f, 0.f};
                }
                l_before += l_run;
                l_run = 0.f;
            }
        }
    };
    // All tiles of this wavefront; whether something in the outputs is not finite.
    auto walk = [&]() __attribute__((always_inline)) {
        const float unit = part < 2 ? 0x1p40f : 0x1p-24f;
        m_run = -__builtin_inff();
        l_run = l_before = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e) o[e] = before[e] = F4{0.f, 0.f, 0.f, 0.f};
        if (wave >= tiles) return false;
        int t = wave;
        for (; t + kWaves < tiles; t += kWaves) step(t, unit, std::true_type());
        step(t, unit, std::false_type());
        l_run += l_before;
        float check = 0.f;
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                o[e][r] += before[e][r];
                check = __builtin_fmaf(o[e][r], 0.f, check);
                o[e][r] *= part < 2 ? 0x1p-40f : 0x1p24f;
            }
        return __any(!(check == 0.f)) != 0;
    };
    if (walk()) {  // with code of its own (as one loop, in which a branch of every tile asks which part it is: heads of 80, i8, 64 sequences of up to 8191 keys 116 -> 122 us)
        for (;;) {
            ++part;
            begin();
            walk();
            if (part == 1 && !__any(others)) break;  // (the same as before: what is not finite comes from elsewhere)
            float *mine = lds_o + (wave * 16 + lr) * (DP + 4);  // this wavefront's place holds the first part for the second
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float &x = mine[(4 * g + r) * NE + e];
                    if (part == 1) x = o[e][r];
                    else o[e][r] += x;
                }
            if (part == 2) break;
        }
    }

    bad = __any(bad);
    join_wavefronts<DP>(p, lds_o, lds_ml, seq, hk, rt, len, bad, alone, slot0, o, m_run, l_run,
                        [&](int e, int r) __attribute__((always_inline)) { return (4 * g + r) * NE + e; });
}

template <typename T, int DP, bool FULL, bool NT, ScaleOf OF, bool EVEN>
__global__ __launch_bounds__(64 * kWaves, DP > 128 ? 1 : 2) void paged_sdpa_scaled_kernel(const ScaledArgs p) {
    __shared__ __attribute__((aligned(16))) float lds_o[kWaves * 16 * (DP + 4)];
    __shared__ float lds_ml[kWaves * 16 * 2];
    fetch_arguments<ScaledArgs>();
    walk_shares<EVEN>(p, [&](int seq, int hk, int rt, int len, bool bad, int key_lo, int key_hi, bool alone, int64_t slot) __attribute__((always_inline)) {
        scaled_segment<T, DP, FULL, NT, OF>(p, lds_o, lds_ml, seq, hk, rt, len, bad, key_lo, key_hi, alone, slot);
    });
}

template <typename T> int32_t launch_scaled(const ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st) {
    if (tiles) {
        const int64_t grid = tiles_grid(a);
        FTH_ARG(grid <= 2147483647LL, "paged_sdpa_scaled: too many workgroups for one launch");
        auto go = [&](auto kernel) { kernel<<<dim3((unsigned)grid), dim3(64 * kWaves), 0, st>>>(a); };
        const bool nt = pl.nt, full = a.c.head_dim == 64 || a.c.head_dim == 128 || a.c.head_dim == 256;
        const bool pages = a.c.page_size % 16 == 0, sixteen = pages && a.sc.block % 16 == 0, four = pages && full && a.sc.block % 4 == 0;
        const bool one = pages && full && a.sc.block == 1 && ((uintptr_t)a.k_scales % 16 | (uintptr_t)a.v_scales % 16 | a.sc.page_stride % 4 | a.sc.head_stride % 4) == 0;
        // (us for 64 sequences of up to 8191 keys, scales by four and by one / looked up by every lane: blocks of 8 133 / 164, of 4 136 / 163, of 1 136 / 166; of 16 128)
        auto pick = [&](auto even) {
            constexpr bool E = decltype(even)::value;
            auto size = [&](auto dp) {
                constexpr int DP = decltype(dp)::value;
                if (sixteen && full) go(nt ? paged_sdpa_scaled_kernel<T, DP, true, true, ScaleOf::sixteen, E> : paged_sdpa_scaled_kernel<T, DP, true, false, ScaleOf::sixteen, E>);
                else if (sixteen) go(paged_sdpa_scaled_kernel<T, DP, false, false, ScaleOf::sixteen, E>);
                else if (one) go(nt ? paged_sdpa_scaled_kernel<T, DP, true, true, ScaleOf::one, E> : paged_sdpa_scaled_kernel<T, DP, true, false, ScaleOf::one, E>);
                else if (four) go(paged_sdpa_scaled_kernel<T, DP, true, false, ScaleOf::four, E>);
                else go(paged_sdpa_scaled_kernel<T, DP, false, false, ScaleOf::any, E>);
            };
            if (a.c.head_dim <= 64) size(std::integral_constant<int, 64>());
            else if (a.c.head_dim <= 128) size(std::integral_constant<int, 128>());
            else size(std::integral_constant<int, 256>());
        };
        if (a.even) pick(std::true_type());
        else pick(std::false_type());
    } else {
        FTH_ARG(pl.rows * a.nsplit <= 2147483647LL, "paged_sdpa_scaled: too many rows for one launch");
        paged_sdpa_rows_kernel<T, ScaledArgs><<<dim3((unsigned)(pl.rows * a.nsplit)), dim3(64), 0, st>>>(a);
    }
    FTH_CHECK_LAUNCH("paged_sdpa_scaled");
    return launch_join(a, pl, st);
}

int32_t launch_e4m3(const ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st);
int32_t launch_i8(const ScaledArgs &a, const Plan &pl, bool tiles, hipStream_t st);

}  // namespace paged
}  // namespace fth
