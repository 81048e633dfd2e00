// Attention of the last one to eight tokens of every sequence over a paged K/V cache.
//
//   out[s, i, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(x_j - max x),   x_j = scale q . k_j,   j < lens[s] - new_tokens + i + 1
//
// Bound by reading the cache once. The keys of a sequence are cut into shares; a workgroup takes one share of one K/V head for up to
// 16 of the query rows that read it (query heads of the group x new tokens), so K and V are read once for all of them. Every 16 rows
// more walk the share again, from the L2 that the first 16 have filled, and pay its products, loads and unpacking again (32 sequences of up to 3967 keys,
// 8 K/V heads of 128, bf16, 304 MB: 8 rows a K/V head 67 us, 16 70, 32 90, 64 144). Shares have one length, or, in large batches of long sequences, are cut from the keys of the whole batch end to end, so that the chip does
// not wait for the longest ones (see steps_of). The four wavefronts of a workgroup walk a share in tiles of 32 keys, each on its own (running
// maximum and sum per row in fp32, no barrier), and are joined through LDS at the end; a second small kernel joins the shares of a
// row in order.
//   * S^T[key, row] = K . Q^T with a key row and a query row per lane (16 x 16 tiles); the lane that gets scores of row lr holds
//     them as it needs them for O^T[d, row] += V^T . P^T, so P never moves; V rows are read whole (16 lanes side by side).
//   * 16-bit caches: both products run on the 16-bit matrix units against the bits as they are stored. The fp32 side is cut into
//     parts of the storage type whose sum it is (struct Parts), so that the result is that of fp32 arithmetic but for queries against f16
//     keys (22 bits of an element, or 2^-39 of the row's largest); what parts cannot do (values that are not finite) is found
//     and computed again, small weights of f16 caches are cut more than once. fp32 caches: fp32 matrix units, 16 times slower a product.
//   * The loads of the next tile's K go out when the scores have consumed this one's, those of V after the outputs have, with
//     nothing conditional in between: the waits are then for K or V alone, never for both.
// Pages: with a page size that is a multiple of 16 each half tile lies in one page, whose number is a scalar load one tile
// ahead; with other sizes every lane looks up a row. Strides, head sizes and alignments that 128-bit loads cannot take go to a
// kernel of one wavefront a row.
//
// Measured: 64 sequences of 1024 to 8191 keys, 32 query heads on 8 K/V heads of 128, bf16 (1.22 GB): 7.6 ms on one wavefront a
// row, 283 us with both products on fp32 units, 235 with the scores on 16-bit ones (MFMA-busy 0.31, wavefronts waiting to
// issue), 212 + 5 with both in shares of 512 KB, 192 + 5 in even ones (6.4 TB/s; a kernel that only reads pages of 4 KB in random
// order reaches 5.9, with nontemporal loads 6.7). One sequence of 131071: 80 + 5 us (6.7 TB/s). Joining the shares in the last workgroup to arrive instead of a
// second launch was slower in every case (release and acquire across the XCDs): 90 -> 109 us.

#include "paged_sdpa.hpp"

namespace {

using namespace fth::paged;

// ---- tiles of 32 keys on the matrix units ---------------------------------------------------------------------------------

// Element e of 16 bytes of storage, as a float.
template <typename T> struct Chunk {  // f16, bf16
    static constexpr int kElems = 8;
    static __device__ __forceinline__ float get(const U4 &v, int e) {
        const uint32_t w = v[e >> 1];
        if constexpr (std::is_same<T, fth::bf16>::value) {
            return __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
        } else {
            return (float)__builtin_bit_cast(fth::f16, (uint16_t)((e & 1) ? w >> 16 : w));
        }
    }
};
template <> struct Chunk<float> {
    static constexpr int kElems = 4;
    static __device__ __forceinline__ float get(const U4 &v, int e) { return __uint_as_float(v[e]); }
};

// (Registers: the fp32 instances for heads of 256 spill 10 to 56 of them, those with even shares the most.)
//
// Scores against 16-bit keys go to the 16-bit matrix units: a query row is scaled by a power of two so that its largest element
// lies in [2^kTop, 2^(kTop + 1)), and cut into parts of the keys' type whose sum it is (bf16: 3 x 8 bits; f16: 2 x 11 bits, off by
// 2^-22 of an element or 2^-39 of the largest). Weights, of which the smallest may be all that V lets through, are cut into as many
// parts as they need (see there).
template <typename T> struct Parts {  // fp32 keys and values: none
    static constexpr int kParts = 0, kArray = 1, kTop = 0;
    static constexpr float kScale = 1.f;  // of the weights that are cut
    using Vec = __attribute__((ext_vector_type(8))) _Float16;
    static __device__ __forceinline__ F4 mfma(const U4 &, const U4 &, F4 c) { return c; }
};
template <> struct Parts<fth::bf16> {
    static constexpr int kParts = 3, kArray = 3, kTop = 0;
    static constexpr float kScale = 0x1p64f;
    using Vec = __attribute__((ext_vector_type(8))) __bf16;
    static __device__ __forceinline__ F4 mfma(const U4 &a, const U4 &b, F4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Vec, a), __builtin_bit_cast(Vec, b), c, 0, 0, 0);
    }
};
template <> struct Parts<fth::f16> {
    static constexpr int kParts = 2, kArray = 2, kTop = 14;
    static constexpr float kScale = 0x1p15f;
    using Vec = __attribute__((ext_vector_type(8))) _Float16;
    static __device__ __forceinline__ F4 mfma(const U4 &a, const U4 &b, F4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Vec, a), __builtin_bit_cast(Vec, b), c, 0, 0, 0);
    }
};

// v[0..7] as kParts vectors of the storage type whose sum they are (up to the last part's rounding).
template <typename T> __device__ __forceinline__ void split_parts(float *v, U4 (&parts)[Parts<T>::kArray]) {
    using V8 = typename Parts<T>::Vec;
#pragma unroll
    for (int j = 0; j < Parts<T>::kParts; ++j) {
        V8 part;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            part[e] = (typename std::remove_reference<decltype(part[0])>::type)v[e];
            v[e] -= (float)part[e];
        }
        parts[j] = __builtin_bit_cast(U4, part);
    }
}

template <typename T, int DP> struct TileShape {
    static constexpr int CH = Chunk<T>::kElems;     // elements of a 128-bit load
    static constexpr int NK = DP / 4 / CH;          // loads of a lane's quarter of a K row
    static constexpr int NE = DP / 16;              // output columns of a lane
    static constexpr int CV = NE < CH ? NE : CH;    // consecutive ones
    static constexpr int NV = NE / CV;              // loads of its part of a V row
};

// FULL: head_dim == DP; otherwise what lies past head_dim counts as zero. NT: K and V leave no trace in the caches. ANY: pages of any
// size: every lane looks its K row up, and V rows are found through the lane that has the same key.
//
// One segment: keys key_lo .. key_hi - 1 of a pair of `len` keys, with row tile rt of its queries. `alone`: these are all of them, and
// the outputs are written; otherwise they go to the slots from `slot` on.
template <typename T, int DP, bool FULL, bool NT, bool ANY>
__device__ __forceinline__ void tiles_segment(const PagedArgs &p, float *lds_o, float *lds_ml, int seq32, int hk, int rt, int len, bool bad, int key_lo, int key_hi, bool alone, int64_t slot0) {
    using S = TileShape<T, DP>;
    constexpr int CH = S::CH, NK = S::NK, NE = S::NE, CV = S::CV, NV = S::NV, kParts = Parts<T>::kParts;
    const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t seq = seq32;
    const int hd = (int)p.c.head_dim, new_tokens = (int)p.d.new_tokens, rows = p.rows;
    const int tiles = (key_hi - key_lo + kTile - 1) / kTile, last16 = (key_hi - 1) >> 4;
    const T *K = static_cast<const T *>(p.k) + hk * p.c.head_stride, *V = static_cast<const T *>(p.v) + hk * p.c.head_stride;
    const Const table = constant(p.table) + seq * p.c.table_stride;
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
    float q[NK][CH];
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int e = 0; e < CH; ++e) {
            const int c = (4 * i + g) * CH + e;
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
    auto offset_of = [&](int2 page) __attribute__((always_inline)) {
        const bool there = page.x >= 0 && page.x < num_pages;
        bad = bad || !there;
        const int64_t at = (int64_t)(there ? page.x : 0) * p.c.page_stride + (int64_t)page.y * rs;
        if constexpr (ANY) return at;
        return (int64_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);  // one for all lanes
    };
    // the offset of row `row` of a half tile, from what offset_of gave
    auto row_offset = [&](int64_t at, int row) __attribute__((always_inline)) {
        if constexpr (ANY) return (int64_t)__shfl((int)(at >> 32), row) << 32 | (uint32_t)__shfl((int)at, row);
        return at + row * rs;
    };
    U4 kf[2][NK], vf[2][4][NV];
    const uint32_t k_lane = (uint32_t)(((ANY ? 0 : lr * rs) + g * CH) * (int)sizeof(T));
    uint32_t v_lane[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v_lane[r] = (uint32_t)(((ANY ? 0 : (4 * g + r) * rs) + lr * CV) * (int)sizeof(T));
    auto load_k = [&](const int64_t (&off)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const char *base = reinterpret_cast<const char *>(K + off[s]);
#pragma unroll
            for (int i = 0; i < NK; ++i) {
                if (!FULL) kf[s][i] = U4{0u, 0u, 0u, 0u};
                if (FULL || (4 * i + g) * CH < hd) kf[s][i] = load128<NT>(base + k_lane + 64 * i);
            }
        }
    };
    auto load_v = [&](const int64_t (&off)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const char *base = reinterpret_cast<const char *>(V + off[s]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (ANY) base = reinterpret_cast<const char *>(V + row_offset(off[s], 4 * g + r));
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const char *src = base + v_lane[r] + 16 * CV * (int)sizeof(T) * i;
                    if (!FULL) vf[s][r][i] = U4{0u, 0u, 0u, 0u};
                    if (FULL || (16 * i + lr) * CV < hd) {
                        if constexpr (CV * sizeof(T) == 16) {
                            vf[s][r][i] = load128<NT>(src);
                        } else {
                            const U2 w = NT ? __builtin_nontemporal_load(reinterpret_cast<const U2 *>(src)) : *reinterpret_cast<const U2 *>(src);
                            vf[s][r][i][0] = w[0];
                            vf[s][r][i][1] = w[1];
                        }
                    }
                }
            }
        }
    };

    const int t16_lo = key_lo >> 4;
    int64_t off[2];
    int2 ahead[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        off[s] = offset_of(page_of(t16_lo + 2 * wave + s));
        ahead[s] = page_of(t16_lo + 2 * (wave + kWaves) + s);
    }
    load_k(off);  // (a wavefront without a tile reads the last one)
    load_v(off);
    __builtin_amdgcn_sched_barrier(0);

    U4 qp[Parts<T>::kArray][NK];
    float scale2 = p.scale2;
    bool finite = true;  // the query row
    if constexpr (kParts != 0) {
        float big = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                big = fmaxf(big, fabsf(q[i][e]));
                sum += q[i][e] * 0.f;
            }
        big = rows_reduce(big, MaxOp());
        finite = rows_reduce(sum, AddOp()) == 0.f;
        const int up = big > 0.f && big < __builtin_inff() ? Parts<T>::kTop + 1 - __builtin_amdgcn_frexp_expf(big) : 0;
        scale2 = __builtin_ldexpf(scale2, -up);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            U4 parts[Parts<T>::kArray];
#pragma unroll
            for (int e = 0; e < CH; ++e) q[i][e] = __builtin_ldexpf(q[i][e], up);
            split_parts<T>(q[i], parts);
#pragma unroll
            for (int j = 0; j < kParts; ++j) qp[j][i] = parts[j];
        }
    }

    F4 o[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = F4{0.f, 0.f, 0.f, 0.f};
    float m_run = -__builtin_inff(), l_run = 0.f;  // the sum: this lane's keys only
    const int limit = sees < key_hi ? sees : key_hi;

    // One tile of 32 keys. Constants: `more`: another one of this wavefront follows, whose loads go out on the way (what a query
    // may not see lies in the last two tiles of the sequence, which are the last ones of their wavefronts); `parts`: weights
    // and V on the 16-bit matrix units.
    auto step = [&](int t, auto more, auto parts) __attribute__((always_inline)) {
        const int key0 = key_lo + t * kTile;
        F4 sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, low[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            if constexpr (kParts == 0) {
#pragma unroll
                for (int e = 0; e < CH; ++e)
#pragma unroll
                    for (int s = 0; s < 2; ++s) sc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(Chunk<T>::get(kf[s][i], e), q[i][e], sc[s], 0, 0, 0);
            } else {
#pragma unroll
                for (int j = kParts - 1; j >= 0; --j)
#pragma unroll
                    for (int s = 0; s < 2; ++s) (j ? low : sc)[s] = Parts<T>::mfma(kf[s][i], qp[j][i], (j ? low : sc)[s]);
            }
        }
        int64_t next[2];
        if constexpr (more) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                next[s] = offset_of(ahead[s]);
                ahead[s] = page_of(t16_lo + 2 * (t + 2 * kWaves) + s);
            }
            load_k(next);
        }
        float check = 0.f;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = (kParts ? sc[s][r] + low[s][r] : sc[s][r]) * scale2;
                const bool seen = more || key0 + 16 * s + 4 * g + r < limit;
                check = __builtin_fmaf(seen ? x : 0.f, 0.f, check);
                sc[s][r] = seen ? x : -__builtin_inff();
            }
        if constexpr (kParts != 0) {
            // An infinity against the parts of a query is no longer what it is against the query, and the scaled query may
            // overflow where it does not: such scores are computed again. (A query row that is not finite gives NaN either way.)
            if (__any(!(check == 0.f) && finite)) {
#pragma unroll 1
                for (int j = 0; j < 8; ++j) {
                    float x = sc[0][0];
#pragma unroll
                    for (int y = 1; y < 8; ++y) x = j == y ? sc[y >> 2][y & 3] : x;
                    const int row = 16 * (j >> 2) + 4 * g + (j & 3);
                    const T *kr = K + row_offset(off[j >> 2], row & 15);
                    if (finite && !(fabsf(x) < __builtin_inff()) && key0 + row < limit) {
                        float dot = 0.f;
                        for (int c = 0; c < hd; ++c) dot = __builtin_fmaf(qr[c], fth::to_f32(kr[c]), dot);
                        x = dot * p.scale2;
                    }
#pragma unroll
                    for (int y = 0; y < 8; ++y) sc[y >> 2][y & 3] = j == y ? x : sc[y >> 2][y & 3];
                }
            }
        }
        float mx = -__builtin_inff();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[s][r]);
        mx = rows_reduce(mx, MaxOp());
        if (__any(mx > m_run)) {
            const float m_new = fmaxf(m_run, mx);
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -__builtin_inff() ? 0.f : m_new));
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][r] *= alpha;
        }
        // nothing visible so far: every weight is exp(-inf) = 0. The power of two that parts are scaled by is a factor, not a part of the
        // exponent, which would be rounded by it (64 more: weights off by 22 units of 2^-24).
        const float ref = m_run == -__builtin_inff() ? 0.f : m_run;
        float w[8];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w[4 * s + r] = __builtin_amdgcn_exp2f(sc[s][r] - ref);
                l_run += w[4 * s + r];
                if constexpr (parts) w[4 * s + r] *= Parts<T>::kScale;
            }
        if constexpr (!more) {  // weight 0 times what an unused row holds would be NaN
            if (key0 + kTile > key_hi) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key0 + 16 * s + 4 * g + r >= key_hi)
#pragma unroll
                            for (int i = 0; i < NV; ++i) vf[s][r][i] = U4{0u, 0u, 0u, 0u};
            }
        }
        if constexpr (parts) {
            U4 wp[Parts<T>::kArray];
            // elements e of the eight V rows, in the order of the weights
            auto column_of = [&](int e, uint32_t even, uint32_t odd) __attribute__((always_inline)) {
                U4 column;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a = vf[j >> 1][2 * (j & 1)][e / CV][e % CV / 2], b = vf[j >> 1][2 * (j & 1) + 1][e / CV][e % CV / 2];
                    column[j] = __builtin_amdgcn_perm(b, a, e & 1 ? odd : even);
                }
                return column;
            };
            // Two parts of f16, which ends at 2^-24, hold 22 bits of a weight from 2^-3 on. Of smaller ones they leave up to 2^-25, and numbers
            // below 2^-14 are added by the matrix units with no more digits than 2^-14 has. So weights below 2^-14, and what the parts of those from
            // there on leave, are cut again times 2^29, until the smallest that is not zero has its 22 bits: V may be zero under all larger ones.
            // (What is left of weights so large that it would not fit is below their 22 bits.) 64 sequences of up to 8191 keys, 16 of up to 3967 with four
            // queries, without / with it: scores of 1.5 around their mean 194 / 194, 40.1 / 40.4 us, of 6 (two turns) 194 / 203, 40.0 / 47.4, of 20 194 / 276, 39.8 / 64.8.
            uint32_t least = ~0u;  // the bits of the smallest weight that is not zero, less one
            if constexpr (kParts == 2) {
#pragma unroll
                for (int j = 0; j < 8; ++j) least = min(least, __float_as_uint(w[j]) - 1u);
            }
            float unit = 1.f;
            auto small = [&]() __attribute__((always_inline)) { return kParts == 2 && __any(least < __float_as_uint(0x1p-3f * unit) - 1u); };
            float in[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) in[j] = w[j];
            if (small()) {
#pragma unroll
                for (int j = 0; j < 8; ++j) in[j] = in[j] < 0x1p-14f ? 0.f : in[j];
            }
            split_parts<T>(in, wp);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const U4 column = column_of(e, 0x05040100u, 0x07060302u);
#pragma unroll
                for (int j = kParts - 1; j >= 0; --j) o[e] = Parts<T>::mfma(column, wp[j], o[e]);
            }
            if constexpr (kParts == 2) {
#pragma unroll 1
                for (int turn = 0; turn < 5 && small(); ++turn) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {  // what the parts so far leave
                        const float left = w[j] - (float)(_Float16)w[j];
                        w[j] = fabsf(w[j]) < 0x1p-14f ? w[j] : left - (float)(_Float16)left;
                        w[j] = fabsf(w[j]) < 0x1p-14f ? w[j] * 0x1p29f : 0.f;
                        in[j] = fabsf(w[j]) < 0x1p-14f ? 0.f : w[j];
                    }
                    unit *= 0x1p-29f;
                    split_parts<T>(in, wp);
                    uint32_t even = 0x05040100u, odd = 0x07060302u;
                    asm volatile("" : "+s"(even), "+s"(odd));  // columns made again each time need no registers across the loop
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        const U4 column = column_of(e, even, odd);
                        F4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = kParts - 1; j >= 0; --j) sum = Parts<T>::mfma(column, wp[j], sum);
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[e][r] = __builtin_fmaf(sum[r], unit, o[e][r]);
                        if (e & 1) __builtin_amdgcn_sched_barrier(0);  // two sums at a time, for their registers' sake
                    }
                }
            }
        } else {
            // A key that only the later of the new tokens see: what is not finite in its V row would be NaN under a weight of 0. It
            // counts as zero here and is added below to the rows that see it.
            const int partly = len - new_tokens + 1;
            bool held = false;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        float v = Chunk<T>::get(vf[s][r][e / CV], e % CV);
                        if constexpr (!more) {
                            const bool hold = key0 + 16 * s + 4 * g + r >= partly && !(fabsf(v) < __builtin_inff());
                            held |= hold;
                            v = hold ? 0.f : v;
                        }
                        o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[4 * s + r], o[e], 0, 0, 0);
                    }
            if constexpr (!more) {
                if (__any(held)) {
                    const int from = partly > key0 ? partly : key0, to = key_hi < key0 + kTile ? key_hi : key0 + kTile;
                    for (int key = from; key < to; ++key) {
                        const int at = key - key0, in_lane = 4 * (at >> 4) + (at & 3);
                        float mine = w[0];
#pragma unroll
                        for (int y = 1; y < 8; ++y) mine = in_lane == y ? w[y] : mine;
                        const float weight = __shfl(mine, (at >> 2 & 3) * 16 + lr);
                        const T *vr = V + row_offset(off[at >> 4], at & 15);
#pragma unroll
                        for (int e = 0; e < NE; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int c = ((e / CV) * 16 + 4 * g + r) * CV + e % CV;
                                const float v = FULL || c < hd ? fth::to_f32(vr[c]) : 0.f;
                                if (key < sees && !(fabsf(v) < __builtin_inff())) o[e][r] += weight * v;
                            }
                    }
                }
            }
        }
        if constexpr (more) {
            load_v(next);
            off[0] = next[0];
            off[1] = next[1];
        }
    };
    using Yes = std::true_type;
    using No = std::false_type;
    auto walk = [&](auto parts) __attribute__((always_inline)) {
        int t = wave;
        for (; t + kWaves < tiles; t += kWaves) step(t, Yes(), parts);
        step(t, No(), parts);
    };
    if (wave < tiles) {
        if constexpr (kParts == 0) {
            walk(No());
        } else {
            walk(Yes());
            float check = 0.f;
#pragma unroll
            for (int e = 0; e < NE; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    check = __builtin_fmaf(o[e][r], 0.f, check);
                    o[e][r] *= 1.f / Parts<T>::kScale;
                }
            // What is not finite in V meets the parts of a weight, not the weight, and large values times the scaled weights
            // may overflow where they do not: once more on fp32 units, unless the query row gives NaN anyway.
            if (__any(!(check == 0.f) && finite)) {
                m_run = -__builtin_inff();
                l_run = 0.f;
#pragma unroll
                for (int e = 0; e < NE; ++e) o[e] = F4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    off[s] = offset_of(page_of(t16_lo + 2 * wave + s));
                    ahead[s] = page_of(t16_lo + 2 * (wave + kWaves) + s);
                }
                load_k(off);
                load_v(off);
                walk(No());
            }
        }
    }

    if constexpr (ANY) bad = __any(bad);
    // MFMA row 4 g + r of column tile e is output column ((e / CV) * 16 + 4 g + r) * CV + e % CV
    join_wavefronts<DP>(p, lds_o, lds_ml, seq, hk, rt, len, bad, alone, slot0, o, m_run, l_run,
                        [&](int e, int r) __attribute__((always_inline)) { return ((e / CV) * 16 + 4 * g + r) * CV + e % CV; });
}

template <typename T, int DP, bool FULL, bool NT, bool ANY, bool EVEN> __global__ __launch_bounds__(64 * kWaves, DP > 128 ? 1 : 2) void paged_sdpa_tiles_kernel(const PagedArgs p) {
    __shared__ __attribute__((aligned(16))) float lds_o[kWaves * 16 * (DP + 4)];
    __shared__ float lds_ml[kWaves * 16 * 2];
    fetch_arguments<PagedArgs>();
    walk_shares<EVEN>(p, [&](int seq, int hk, int rt, int len, bool bad, int key_lo, int key_hi, bool alone, int64_t slot) __attribute__((always_inline)) {
        tiles_segment<T, DP, FULL, NT, ANY>(p, lds_o, lds_ml, seq, hk, rt, len, bad, key_lo, key_hi, alone, slot);
    });
}

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
    // again lose (under 131072: 4 sequences of 3000 keys 47.5 / 34, 16 of 1000 22.4 / 17.2, 64 of 300 or 600 level).
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

namespace {

template <typename T> int32_t launch(const PagedArgs &a, const Plan &pl, bool tiles, hipStream_t st) {
    if (tiles) {
        const int64_t grid = tiles_grid(a);
        FTH_ARG(grid <= 2147483647LL, "paged_sdpa: too many workgroups for one launch");
        const dim3 blocks((unsigned)grid);
        const bool nt = pl.nt;
        auto go = [&](auto kernel) { kernel<<<blocks, dim3(64 * kWaves), 0, st>>>(a); };
        auto pick = [&](auto even) {
            constexpr bool E = decltype(even)::value;
            if (a.c.page_size % 16 != 0) {
                if (a.c.head_dim <= 64) go(paged_sdpa_tiles_kernel<T, 64, false, false, true, E>);
                else if (a.c.head_dim <= 128) go(paged_sdpa_tiles_kernel<T, 128, false, false, true, E>);
                else go(paged_sdpa_tiles_kernel<T, 256, false, false, true, E>);
            } else switch (a.c.head_dim) {
                case 64: go(nt ? paged_sdpa_tiles_kernel<T, 64, true, true, false, E> : paged_sdpa_tiles_kernel<T, 64, true, false, false, E>); break;
                case 128: go(nt ? paged_sdpa_tiles_kernel<T, 128, true, true, false, E> : paged_sdpa_tiles_kernel<T, 128, true, false, false, E>); break;
                case 256: go(nt ? paged_sdpa_tiles_kernel<T, 256, true, true, false, E> : paged_sdpa_tiles_kernel<T, 256, true, false, false, E>); break;
                default:
                    if (a.c.head_dim < 64) go(paged_sdpa_tiles_kernel<T, 64, false, false, false, E>);
                    else if (a.c.head_dim < 128) go(paged_sdpa_tiles_kernel<T, 128, false, false, false, E>);
                    else go(paged_sdpa_tiles_kernel<T, 256, false, false, false, E>);
            }
        };
        if (a.even) pick(std::true_type());
        else pick(std::false_type());
    } else {
        FTH_ARG(pl.rows * a.nsplit <= 2147483647LL, "paged_sdpa: too many rows for one launch");
        paged_sdpa_rows_kernel<T, PagedArgs><<<dim3((unsigned)(pl.rows * a.nsplit)), dim3(64), 0, st>>>(a);
    }
    FTH_CHECK_LAUNCH("paged_sdpa");
    return launch_join(a, pl, st);
}

}  // namespace

extern "C" {

size_t fth_dev_paged_sdpa_workspace_bytes(const fth_paged_cache *c, const fth_paged_sdpa_desc *d) {
    return check(c, d) == FTH_OK ? workspace_bytes_of(plan(*c, *d), *c) : 0;
}

int32_t fth_dev_paged_sdpa_f32(const fth_paged_cache *c, const fth_paged_sdpa_desc *d, float scale, const float *q, const void *k_cache, const void *v_cache,
                               const int32_t *block_table, const int32_t *lens, float *out, int64_t *bad_index, void *workspace, size_t workspace_bytes,
                               fth_stream s) {
    if (int32_t rc = check(c, d)) return rc;
    FTH_ARG(c->num_seqs == 0 || (q && lens && out && (block_table || c->max_pages == 0) && ((k_cache && v_cache) || c->num_pages == 0)), "paged_sdpa: NULL operand");
    const Plan pl = plan(*c, *d);
    const size_t need = workspace_bytes_of(pl, *c);
    FTH_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15u) == 0), "paged_sdpa: needs a workspace of %zu bytes, 16-byte aligned", need);
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("paged_sdpa(bad_index reset)");
    }
    if (c->num_seqs == 0) return FTH_OK;
    PagedArgs a;
    const bool tiles = fill_args(a, *c, *d, pl, scale, q, k_cache, v_cache, block_table, lens, out, bad_index, workspace);
    switch (c->dtype) {
        case FTH_DTYPE_F32: return launch<float>(a, pl, tiles, st);
        case FTH_DTYPE_F16: return launch<fth::f16>(a, pl, tiles, st);
        default: return launch<fth::bf16>(a, pl, tiles, st);
    }
}

}  // extern "C"
