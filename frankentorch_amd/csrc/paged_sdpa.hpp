// What the attention kernels over a paged cache share: the arguments, how a call is cut into shares, the walk over the shares, and the
// kernel of one wavefront a row that takes what 128-bit loads cannot. Caches of fp32 and of 16 bits and caches of 8 bits with
// scales each have their tiles on the matrix units; the shares are joined by one kernel.
#pragma once

#include <type_traits>

#include "paged.hpp"

namespace fth {
namespace paged {

using F4 = float __attribute__((ext_vector_type(4)));
using U4 = uint32_t __attribute__((ext_vector_type(4)));
using U2 = uint32_t __attribute__((ext_vector_type(2)));

// What no kernel here writes: such loads stay scalar ones also behind stores.
using Const = const int32_t __attribute__((address_space(4))) *;
__device__ __forceinline__ Const constant(const int32_t *x) { return (Const)(uintptr_t)x; }

constexpr float kLog2e = 1.44269502162933349609375f;
constexpr int kTile = 32, kWaves = 4;

struct PagedArgs {
    static constexpr bool kScaled = false;
    fth_paged_cache c;
    fth_paged_sdpa_desc d;
    const float *q;
    const void *k, *v;
    const int32_t *table, *lens;
    float *out;
    int64_t *bad;
    float *part_o;    // [slot][pitch] unnormalised outputs of the shares (rows with more than one)
    float *part_ml;   // [slot][2] their maxima (of scores times log2 e) and sums
    int32_t *starts;  // even shares: where each sequence begins in the line of steps; behind the last one the length of a share
    float scale2;     // scale * log2(e)
    int64_t most;     // the longest valid sequence
    int group, rows, row_tiles, pitch;                    // rows: queries that read a K/V head, group * new_tokens
    int pairs;                                            // of a sequence and a K/V head
    int nsplit, share;                                    // shares of `share` keys from the first key of a pair on, nsplit of the longest
    int even, enough, step_log2, seqs_a_lane;             // or this many even shares, if the keys make `enough` steps (0: the former)
    fth::Divisor by_page, by_tiles, by_pairs, by_heads;   // by page_size, row_tiles, pairs, kv_heads
    fth::Divisor by_new, by_q_heads, by_group, by_group4, by_even;  // by new_tokens, q_heads, group, pitch / 4, even
};

// Even shares: all pairs of a sequence and a K/V head stand in one line, each as one step for beginning it and the steps of
// 2^step_log2 keys that it has, and every workgroup takes the same stretch of that line. A stretch has at most two pairs in part, its
// first and its last, so a workgroup has two groups of `rows` slots.
__device__ __forceinline__ int steps_of(const PagedArgs &p, int len) { return len < 0 || len > p.most ? 0 : (int)(((uint32_t)len + (1u << p.step_log2) - 1) >> p.step_log2); }

// All lines of the arguments at once: the compiler reads them as it needs them, in several round trips one after the other (8
// sequences of up to 1024 keys, 12 heads of 64: 10.8 + 3.8 -> 10.3 + 3.1 us).
template <typename A> __device__ __forceinline__ void fetch_arguments() {
    const auto a = (const uint32_t __attribute__((address_space(4))) *)__builtin_amdgcn_kernarg_segment_ptr();
    uint32_t any = 0;
#pragma unroll
    for (unsigned i = 0; i < sizeof(A) / 4; i += 16) any |= a[i];
    asm volatile("" ::"s"(any));
}

struct MaxOp { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct AddOp { __device__ float operator()(float a, float b) const { return a + b; } };
template <typename F> __device__ __forceinline__ float wave_reduce(float x, F op) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    return x;
}
// over the four 16-lane rows of a wavefront, the result in every lane
template <typename F> __device__ __forceinline__ float rows_reduce(float x, F op) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Where a row (sequence, new token, query head) of the output lies.
__device__ __forceinline__ float *out_row(const PagedArgs &p, int64_t seq, int i, int h) {
    return p.out + seq * p.d.o_seq_stride + i * p.d.o_row_stride + h * p.d.o_head_stride;
}

// ---- one wavefront a row and share: any page size, head size, stride and alignment ----------------------------------------

template <typename T, typename Args> __global__ __launch_bounds__(64) void paged_sdpa_rows_kernel(const Args p) {
    __shared__ float qs[256], ps[64];
    __shared__ float vs[64];  // scales of V
    __shared__ int64_t at[64];
    const int lane = threadIdx.x, hd = (int)p.c.head_dim, page_size = (int)p.c.page_size;
    const int split = (int)(blockIdx.x % (unsigned)p.nsplit), row32 = (int)(blockIdx.x / (unsigned)p.nsplit);
    const int token = (int)p.by_q_heads((uint32_t)row32), h = row32 - token * (int)p.d.q_heads;
    const int seq32 = (int)p.by_new((uint32_t)token), i = token - seq32 * (int)p.d.new_tokens;
    const int64_t seq = seq32, hk = p.by_group((uint32_t)h);
    const T *K = static_cast<const T *>(p.k) + hk * p.c.head_stride, *V = static_cast<const T *>(p.v) + hk * p.c.head_stride;
    int len = p.lens[seq];
    bool bad = len < 0 || len > p.most;
    if (bad) len = 0;
    const int key_lo = split * p.share;
    if (split > 0 && key_lo >= len) return;
    const bool alone = len <= p.share;  // no other share of this row
    const int end = len - key_lo < p.share ? len : key_lo + p.share;
    const int sees = len - (int)p.d.new_tokens + i + 1, key_hi = sees < end ? sees : end;  // pages are looked at up to `end`, so that all rows of a sequence find a bad one
    const float *q = p.q + seq * p.d.q_seq_stride + i * p.d.q_row_stride + h * p.d.q_head_stride;
    for (int c = lane; c < hd; c += 64) qs[c] = q[c];
    __syncthreads();
    float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -__builtin_inff(), l = 0.f;
    for (int key0 = key_lo; key0 < end; key0 += 64) {
        const int key = key0 + lane, n = key_hi - key0 < 64 ? key_hi - key0 : 64;
        float x = -__builtin_inff();
        if (key < end) {
            const int index = (int)p.by_page((uint32_t)key);
            int page = p.table[seq * p.c.table_stride + index];
            if (page < 0 || page >= p.c.num_pages) {
                bad = true;
                page = -1;
            }
            const int64_t off = page < 0 ? -1 : (int64_t)page * p.c.page_stride + (int64_t)(key - index * page_size) * p.c.row_stride;
            at[lane] = off;
            float ks = 1.f;
            if constexpr (Args::kScaled) {
                if (page >= 0 && lane < n) {
                    const int64_t i = (int64_t)page * p.sc.page_stride + hk * p.sc.head_stride + (int)p.by_block((uint32_t)(key - index * page_size));
                    ks = p.k_scales[i];
                    const float v = p.v_scales[i];
                    ks = __builtin_fmaf(ks, 0.f, ks);  // infinite: NaN
                    vs[lane] = __builtin_fmaf(v, 0.f, v);
                }
            }
            if (page >= 0 && lane < n) {
                float dot[4] = {0.f, 0.f, 0.f, 0.f};  // short chains of roundings
                for (int c = 0; c < hd; ++c) dot[c & 3] = __builtin_fmaf(qs[c], fth::to_f32(K[off + c]), dot[c & 3]);
                x = (dot[0] + dot[1]) + (dot[2] + dot[3]);
                if constexpr (Args::kScaled) x *= ks;
                x *= p.scale2;
            }
        }
        const float m_new = fmaxf(m, wave_reduce(x, MaxOp()));
        const float ref = m_new == -__builtin_inff() ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - ref), w = lane < n ? __builtin_amdgcn_exp2f(x - ref) : 0.f;
        m = m_new;
        l = l * alpha + wave_reduce(w, AddOp());
        ps[lane] = w;
        __syncthreads();
        for (int j = 0; j < 4; ++j) {
            const int c = lane + 64 * j;
            if (c >= hd) break;
            float acc = 0.f;
            for (int r = 0; r < n; ++r)
                if (at[r] >= 0) {
                    float x = fth::to_f32(V[at[r] + c]);
                    if constexpr (Args::kScaled) x *= vs[r];
                    acc = __builtin_fmaf(ps[r], x, acc);
                }
            o[j] = o[j] * alpha + acc;
        }
        __syncthreads();
    }
    bad = __any(bad);
    if (bad && lane == 0) fth::report_bad_entry(p.bad, seq);
    if (bad) l = __builtin_nanf("");
    float *dst = out_row(p, seq, i, h);
    if (!alone) {
        const int64_t slot = ((seq * p.c.kv_heads + hk) * p.nsplit + split) * p.rows + (h - hk * p.group) * p.d.new_tokens + i;
        dst = p.part_o + slot * p.pitch;
        if (lane == 0) {
            p.part_ml[2 * slot] = m;
            p.part_ml[2 * slot + 1] = l;
        }
    }
    for (int j = 0; j < 4; ++j) {
        const int c = lane + 64 * j;
        if (c < hd) dst[c] = !alone ? o[j] : sees <= 0 && !bad ? 0.f : o[j] / l;
    }
}

// ---- what every kernel of tiles ends with ------------------------------------------------------------------------------------

// A pair without keys: row tile rt of its queries gives zeros, or NaN for a sequence that is invalid.
__device__ __forceinline__ void store_empty(const PagedArgs &p, int64_t seq, int hk, int rt, bool bad) {
    const int hd = (int)p.c.head_dim, new_tokens = (int)p.d.new_tokens, stored = p.rows - rt * 16 < 16 ? p.rows - rt * 16 : 16;
    if (bad && threadIdx.x == 0) fth::report_bad_entry(p.bad, seq);
    for (int x = threadIdx.x; x < stored * hd; x += 64 * kWaves) {
        const int row = rt * 16 + x / hd;
        out_row(p, seq, row % new_tokens, hk * p.group + row / new_tokens)[x % hd] = bad ? __builtin_nanf("") : 0.f;
    }
}

// The wavefronts of a workgroup joined through LDS, and the result written: to the outputs (`alone`) or to the slots from slot0 on. A lane
// holds o[e][r], column(e, r) of query row lane % 16, its maximum, and the sum over its own keys.
template <int DP, int NE, typename F>
__device__ __forceinline__ void join_wavefronts(const PagedArgs &p, float *lds_o, float *lds_ml, int64_t seq, int hk, int rt, int len, bool bad, bool alone, int64_t slot0, const F4 (&o)[NE],
                                                float m_run, float l_run, F column) {
    constexpr int P = DP + 4;
    const int lane = threadIdx.x & 63, lr = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hd = (int)p.c.head_dim, new_tokens = (int)p.d.new_tokens, stored = p.rows - rt * 16 < 16 ? p.rows - rt * 16 : 16;
    const float l_wave = rows_reduce(l_run, AddOp());
    if (g == 0) {
        lds_ml[(wave * 16 + lr) * 2] = m_run;
        lds_ml[(wave * 16 + lr) * 2 + 1] = bad ? __builtin_nanf("") : l_wave;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) lds_o[(wave * 16 + lr) * P + column(e, r)] = o[e][r];
    if (bad && lane == 0) fth::report_bad_entry(p.bad, seq);
    __syncthreads();
    for (int x = threadIdx.x; x < stored * (DP / 4); x += 64 * kWaves) {
        const int row = x / (DP / 4), c = x % (DP / 4) * 4;
        if (c >= hd) continue;
        float m = -__builtin_inff(), l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, lds_ml[(w * 16 + row) * 2]);
        const float ref = m == -__builtin_inff() ? 0.f : m;
        F4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float weight = __builtin_amdgcn_exp2f(lds_ml[(w * 16 + row) * 2] - ref);
            l += lds_ml[(w * 16 + row) * 2 + 1] * weight;
            const F4 part = *reinterpret_cast<const F4 *>(&lds_o[(w * 16 + row) * P + c]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += part[j] * weight;
        }
        const int head = (int)p.by_new((uint32_t)(rt * 16 + row)), ri = rt * 16 + row - head * new_tokens, rh = hk * p.group + head;
        if (alone) {
            float *dst = out_row(p, seq, ri, rh);
            const bool nothing = !(l != l) && len - new_tokens + 1 + ri <= 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[c + j] = nothing ? 0.f : acc[j] / l;
        } else {
            const int64_t slot = slot0 + rt * 16 + row;
            *reinterpret_cast<F4 *>(p.part_o + slot * p.pitch + c) = acc;
            if (c == 0) {
                p.part_ml[2 * slot] = m;
                p.part_ml[2 * slot + 1] = l;
            }
        }
    }
}

// ---- shares -----------------------------------------------------------------------------------------------------------------

// The shares of a workgroup one after the other: segment(seq, hk, rt, len, bad, key_lo, key_hi, alone, slot) attends to keys key_lo .. key_hi - 1
// of a pair of `len` keys with row tile rt of its queries.
template <bool EVEN, typename F> __device__ __forceinline__ void walk_shares(const PagedArgs &p, F segment) {
    // Workgroup ids go round the 8 XCDs: the row tiles of one share of a K/V head come 8 apart, so that they find its K and V in
    // one L2 (16 sequences of up to 3967 keys, 64 query heads on 8 of 128: four queries, bf16 64.6 -> 57.3 us; eight, fp32 202 -> 155).
    const int block8 = (int)(blockIdx.x >> 3), item8 = (int)p.by_tiles((uint32_t)block8), rt = block8 - item8 * p.row_tiles;
    const int item = item8 * 8 + (int)(blockIdx.x & 7), heads = (int)p.c.kv_heads;
    const Const lens = constant(p.lens);
    int seq = 0, hk = 0, raw = 0, split = 0, pos = 0, end = 0, within = 0;
    bool line = false;  // even shares
    if constexpr (EVEN) {
        if (item >= p.even) {  // nothing to do either way? (most workgroups, where max_len is far above the lengths)
            const int at = (int)p.by_pairs((uint32_t)item), len = lens[p.by_heads((uint32_t)(item - at * p.pairs))];
            if (at >= p.nsplit || (at > 0 && (len <= at * p.share || len > p.most))) return;
        }
        const int lane = threadIdx.x & 63, first = lane * p.seqs_a_lane, num_seqs = (int)p.c.num_seqs;
        const int last = num_seqs - first < p.seqs_a_lane ? num_seqs : first + p.seqs_a_lane;
        int mine = 0;
        for (int j = first; j < last; ++j) mine += heads * (steps_of(p, lens[j]) + 1);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(upto, d);
            upto += lane >= d ? x : 0;
        }
        const int total = __builtin_amdgcn_readlane(upto, 63), share = (int)p.by_even((uint32_t)(total + p.even - 1));
        line = total - p.pairs >= p.enough;
        if (blockIdx.x == 0 && threadIdx.x < 64) {
            int at = upto - mine;
            for (int j = first; j < last; ++j) {
                p.starts[j] = at;
                at += heads * (steps_of(p, lens[j]) + 1);
            }
            if (lane == 0) p.starts[num_seqs] = line ? share : 0;
        }
        if (line) {  // this workgroup's place in the line
            pos = item * share;
            if (item >= p.even || pos >= total) return;
            end = total - pos < share ? total : pos + share;
            const int in_lane = __builtin_ctzll(__ballot(upto > pos));
            int at = __builtin_amdgcn_readlane(upto - mine, in_lane);
            seq = in_lane * p.seqs_a_lane;
            for (;;) {
                raw = lens[seq];
                const int behind = at + heads * (steps_of(p, raw) + 1);
                if (pos < behind) break;
                at = behind;
                ++seq;
            }
            hk = (pos - at) / (steps_of(p, raw) + 1);
            within = pos - at - hk * (steps_of(p, raw) + 1);
        }
    }
    if (!line) {
        split = (int)p.by_pairs((uint32_t)item);
        if (split >= p.nsplit) return;
        const int pair = item - split * p.pairs;
        seq = (int)p.by_heads((uint32_t)pair);
        hk = pair - seq * heads;
        raw = lens[seq];
    }
    for (;;) {
        const bool bad = raw < 0 || raw > p.most;
        const int len = bad ? 0 : raw, steps = steps_of(p, raw), stop = steps + 1 - within < end - pos ? steps + 1 : within + end - pos;
        int key_lo, key_hi;
        int64_t slot;
        if (EVEN && line) {
            key_lo = (within > 1 ? within - 1 : 0) << p.step_log2;
            key_hi = stop > steps ? len : (stop - 1) << p.step_log2;
            slot = 2 * item + (within == 0);
        } else {
            key_lo = split * p.share;
            key_hi = len - key_lo < p.share ? len : key_lo + p.share;
            slot = ((int64_t)seq * heads + hk) * p.nsplit + split;
        }
        if (key_lo < key_hi || (len == 0 && key_lo == 0))
            segment(seq, hk, rt, len, bad, key_lo, key_hi, key_lo == 0 && key_hi == len, slot * p.rows);
        if (!EVEN || !line) break;
        pos += stop - within;
        if (pos >= end) break;
        within = 0;
        if (++hk == heads) {
            hk = 0;
            raw = lens[++seq];
        }
        __syncthreads();  // the segment's LDS has been read
    }
}

template <bool NT> __device__ __forceinline__ U4 load128(const void *p) {
    const U4 *v = static_cast<const U4 *>(p);
    return NT ? __builtin_nontemporal_load(v) : *v;
}

// ---- how a call is cut, and the join --------------------------------------------------------------------------------------

// The same for a call's workspace and its launch.
struct Plan {
    bool tiles;  // head size and strides that the 128-bit loads take (the pointers' alignment is looked at later)
    bool nt;     // loads that leave no trace in the caches
    int even, enough, step_log2, nsplit, share, pitch;
    int64_t rows, row_tiles, most;
};
Plan plan(const fth_paged_cache &c, const fth_paged_sdpa_desc &d);
size_t workspace_bytes_of(const Plan &p, const fth_paged_cache &c);
int32_t check(const fth_paged_cache *c, const fth_paged_sdpa_desc *d, bool scaled = false);  // scaled: a cache of 8 bits
// The operands of a call that check() and the workspace's size have passed; returns whether the tiles take them, else it is one wavefront a row.
bool fill_args(PagedArgs &a, const fth_paged_cache &c, const fth_paged_sdpa_desc &d, const Plan &pl, float scale, const float *q, const void *k_cache, const void *v_cache,
               const int32_t *block_table, const int32_t *lens, float *out, int64_t *bad_index, void *workspace);
int64_t tiles_grid(const PagedArgs &a);
int32_t launch_join(const PagedArgs &a, const Plan &pl, hipStream_t st);

}  // namespace paged
}  // namespace fth
