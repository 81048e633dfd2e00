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
