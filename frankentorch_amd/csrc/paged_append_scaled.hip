// Keys and values of new tokens into a paged cache of 8-bit numbers with a scale for each block of positions and head.
//
// A block's scale s is the smallest power of two whose 127 (448) multiples reach the largest element it was given: x / s is exact, so
// that an element is rounded once, and a scale that grows by 2^k takes what the block holds to code / 2^k. A run is the tokens of one block that stand
// one after the other in the call; whoever has its first token does all of it, so that no two workgroups touch one block.

#include <type_traits>

#include "paged.hpp"

namespace {

struct Args {
    fth_paged_cache c;
    fth_paged_append_desc d;
    fth_paged_scales sc;
    const float *q, *k, *v, *cosines, *sines;
    const int32_t *table, *seq_ids, *positions;
    float *q_out;
    void *k_cache, *v_cache;
    float *k_scales, *v_scales;
    int64_t *bad;
    fth::Divisor by_page, by_block;
};

// Where position pos of a sequence is: its page and the row in it; false when there is no such place.
__device__ __forceinline__ bool find_row(const Args &p, int seq, int pos, int *page, int *row) {
    if (pos < 0 || (p.d.rotary_dim > 0 && pos >= p.d.max_pos)) return false;
    if (seq < 0 || seq >= p.c.num_seqs || pos >= p.c.max_pages * p.c.page_size) return false;
    const int index = (int)p.by_page((uint32_t)pos);
    *page = p.table[(int64_t)seq * p.c.table_stride + index];
    *row = pos - index * (int)p.c.page_size;
    return *page >= 0 && *page < p.c.num_pages;
}

struct Run {
    int tokens;     // 0: token t begins none
    int pos, page;
    int row, first; // of its first token: the row in the page; the block's first row
};

// The run that token t begins. All lanes of a wavefront ask for the same one.
__device__ __forceinline__ Run run_at(const Args &p, int64_t t, bool report) {
    Run r = {0, p.positions[t], 0, 0, 0};
    if (r.pos == -1) return r;
    const int lane = threadIdx.x & 63, block = (int)p.sc.block, seq = p.seq_ids[t];
    if (!find_row(p, seq, r.pos, &r.page, &r.row)) {
        if (report && lane == 0) fth::report_bad_entry(p.bad, t);
        return r;
    }
    r.first = (int)p.by_block((uint32_t)r.row) * block;
    const int in_block = r.row - r.first;
    if (t > 0 && p.seq_ids[t - 1] == seq) {
        const int before = p.positions[t - 1], start = r.pos - in_block;
        if (before >= start && before - start < block) {  // of the same block
            if (before != r.pos - 1 && report && lane == 0) fth::report_bad_entry(p.bad, t);
            return r;
        }
    }
    int64_t most = p.d.tokens - t;
    most = block - in_block < most ? block - in_block : most;
    int last = p.d.rotary_dim > 0 ? (int)(p.d.max_pos < 2147483647LL ? p.d.max_pos : 2147483647LL) : 2147483647;
    int n = 1;
    for (;;) {
        const int i = n + lane;
        const bool goes_on = i < most && p.positions[t + i] == r.pos + i && p.seq_ids[t + i] == seq && r.pos + i < last;
        const uint64_t on = __ballot(goes_on);
        if (~on) {
            n += __builtin_ctzll(~on);
            break;
        }
        n += 64;
    }
    r.tokens = n;
    return r;
}

template <typename T> constexpr float kLargest = std::is_same<T, fth::i8>::value ? 127.f : 448.f;

// The scale that elements up to `largest` need (see above): 0 for zeros, NaN for what is not finite.
template <typename T> __device__ __forceinline__ float scale_for(float largest) {
    if (largest == 0.f) return 0.f;
    if (!(largest < __builtin_inff())) return __builtin_nanf("");
    // largest = m 2^e, m in [1/2, 1), against 127 = (127 / 128) 2^7 and 448 = (7 / 8) 2^9
    const float m = __builtin_amdgcn_frexp_mantf(largest);
    const int e = __builtin_amdgcn_frexp_expf(largest) - (std::is_same<T, fth::i8>::value ? 7 : 9) + (m > (std::is_same<T, fth::i8>::value ? 0.9921875f : 0.875f));
    return __builtin_ldexpf(1.f, e < -126 ? -126 : e);
}
// Which of two scales holds: the larger, NaN before all.
__device__ __forceinline__ float larger_scale(float had, float needs) { return had != had || needs != needs ? __builtin_nanf("") : had > needs ? had : needs; }
// What elements are multiplied by: 0 under a scale that is none.
__device__ __forceinline__ float per_scale(float s) { return s > 0.f ? 1.f / s : 0.f; }

// To nearest even; |x| is within the type's range, or x is not finite (0).
__device__ __forceinline__ uint32_t to_code(float x, fth::i8) {
    x = fabsf(x) < __builtin_inff() ? __builtin_rintf(x) : 0.f;
    return (uint32_t)(int)fminf(fmaxf(x, -127.f), 127.f) & 255u;
}
__device__ __forceinline__ uint32_t to_code(float x, fth::e4m3) {
    x = fabsf(x) < __builtin_inff() ? fminf(fmaxf(x, -448.f), 448.f) : 0.f;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 255u;
}

struct Turn {
    const float *c, *s;  // of the position
    int pairs;
    bool inter;
};
__device__ __forceinline__ Turn turn_at(const Args &p, int pos) {
    const int pairs = (int)p.d.rotary_dim / 2;
    return {p.cosines + (int64_t)pos * pairs, p.sines + (int64_t)pos * pairs, pairs, p.d.interleaved != 0};
}
// Element c of a row, rotated.
__device__ __forceinline__ float turned(const float *x, int c, const Turn &t) {
    if (c >= 2 * t.pairs) return x[c];
    const int i = t.inter ? c >> 1 : c < t.pairs ? c : c - t.pairs;
    const float a = x[t.inter ? 2 * i : i], b = x[t.inter ? 2 * i + 1 : i + t.pairs];
    const bool first = t.inter ? !(c & 1) : c < t.pairs;
    return first ? a * t.c[i] - b * t.s[i] : b * t.c[i] + a * t.s[i];
}

// ---- one wavefront a run and head, element by element: any head size, stride and alignment ---------------------------------

template <typename T> __global__ __launch_bounds__(64) void append_scaled_kernel(const Args p, int per_token) {
    const int64_t t = blockIdx.x / (unsigned)per_token;
    const int item = (int)(blockIdx.x % (unsigned)per_token), lane = threadIdx.x, hd = (int)p.c.head_dim, hkv = (int)p.c.kv_heads;
    if (item == 2 * hkv) {  // the queries of a token: pairs, so that they may be rotated in place
        const int pos = p.positions[t];
        int page, row;
        if (pos == -1 || !find_row(p, p.seq_ids[t], pos, &page, &row)) return;
        const Turn turn = turn_at(p, pos);
        const int units = hd - turn.pairs;
        for (int64_t u = lane; u < p.d.q_heads * units; u += 64) {
            const int64_t h = u / units;
            const int i = (int)(u % units), ia = i >= turn.pairs ? i + turn.pairs : turn.inter ? 2 * i : i, ib = turn.inter ? 2 * i + 1 : i + turn.pairs;
            const float *x = p.q + t * p.d.q_row_stride + h * p.d.q_head_stride;
            float *y = p.q_out + t * p.d.out_row_stride + h * p.d.out_head_stride;
            const float a = turned(x, ia, turn), b = i < turn.pairs ? turned(x, ib, turn) : 0.f;
            y[ia] = a;
            if (i < turn.pairs) y[ib] = b;
        }
        return;
    }
    const Run run = run_at(p, t, item == 0);
    if (run.tokens == 0) return;
    const bool keys = item < hkv;
    const int64_t h = keys ? item : item - hkv;
    const float *src = keys ? p.k + t * p.d.k_row_stride + h * p.d.k_head_stride : p.v + t * p.d.v_row_stride + h * p.d.v_head_stride;
    const int64_t pitch = keys ? p.d.k_row_stride : p.d.v_row_stride;
    T *dst = static_cast<T *>(keys ? p.k_cache : p.v_cache) + run.page * p.c.page_stride + h * p.c.head_stride;
    float *scale = (keys ? p.k_scales : p.v_scales) + run.page * p.sc.page_stride + h * p.sc.head_stride + (int)p.by_block((uint32_t)run.first);
    auto element = [&](int i, int c) {
        const float *x = src + i * pitch;
        return keys ? turned(x, c, turn_at(p, run.pos + i)) : x[c];
    };
    uint32_t largest = 0;  // bits of |x|: those of NaN are above infinity's
    for (int64_t x = lane; x < (int64_t)run.tokens * hd; x += 64) {
        const uint32_t bits = __float_as_uint(element((int)(x / hd), (int)(x % hd))) & 0x7fffffffu;
        largest = bits > largest ? bits : largest;
    }
    for (int m = 32; m > 0; m >>= 1) {
        const uint32_t other = __shfl_xor(largest, m);
        largest = other > largest ? other : largest;
    }
    const float had = run.row > run.first ? *scale : 0.f, now = larger_scale(had, scale_for<T>(__uint_as_float(largest))), per = per_scale(now);
    __syncthreads();  // every lane has read the scale
    auto store = [&](int row, int c, float x) { reinterpret_cast<uint8_t *>(dst)[row * p.c.row_stride + c] = (uint8_t)to_code(x, T()); };
    if (run.row == run.first || now != had) {
        const float shrink = had * per;
        for (int64_t x = lane; x < (int64_t)(run.row - run.first) * hd; x += 64) {
            const int row = run.first + (int)(x / hd), c = (int)(x % hd);
            store(row, c, fth::to_f32(dst[row * p.c.row_stride + c]) * shrink);
        }
        if (lane == 0) *scale = now;
    }
    for (int64_t x = lane; x < (int64_t)run.tokens * hd; x += 64) {
        const int i = (int)(x / hd), c = (int)(x % hd);
        store(run.row + i, c, element(i, c) * per);
    }
}

// ---- whole vectors ----------------------------------------------------------------------------------------------------------

using F4 = float __attribute__((ext_vector_type(4)));

template <bool NT> __device__ __forceinline__ F4 load4(const float *p) {
    const F4 *v = reinterpret_cast<const F4 *>(p);
    return NT ? __builtin_nontemporal_load(v) : *v;
}

// Four codes as they are stored. x is within the type's range (its scale sees to that).
template <typename T> __device__ __forceinline__ uint32_t codes4(F4 x) {
    if constexpr (std::is_same<T, fth::e4m3>::value) {
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false), true);
    } else {  // to nearest even by the sum with 1.5 * 2^23, whose last bits are the number
        uint32_t b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(x[e] + 12582912.f);
        const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        return lo | hi;
    }
}
template <typename T> __device__ __forceinline__ F4 values4(uint32_t w) {
    if constexpr (std::is_same<T, fth::e4m3>::value) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return F4{lo[0], lo[1], hi[0], hi[1]};
    } else {
        return F4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
    }
}

// A lane has two chunks of four elements of a row, so that every access of the lanes of a row covers whole lines: of a rotated row the two sides
// of four pairs (i, i + rotary_dim / 2), else, and of adjacent pairs, chunks from the two halves of what they cover.
struct Chunks {
    int a, b;
    bool turn_a, turn_b;
};
template <bool INTER> __device__ __forceinline__ Chunks chunks_of(int i, int hd, int rotary, bool turns) {
    Chunks c = {4 * i, hd / 2 + 4 * i, false, false};
    if (!turns) return c;
    if constexpr (INTER) {
        c.turn_a = c.a < rotary;
        c.turn_b = c.b < rotary;
    } else if (8 * i < rotary) {
        c.b = rotary / 2 + 4 * i;
        c.turn_a = c.turn_b = true;
    } else {
        c.a = rotary + 4 * (i - rotary / 8);
        c.b = c.a + (hd - rotary) / 2;
    }
    return c;
}
struct Angles {
    F4 c, s;  // of four pairs; INTER: of two of chunk a, two of chunk b
};
template <bool INTER> __device__ __forceinline__ Angles angles_at(const Args &p, int pos, int i, const Chunks &at) {
    const int pairs = (int)p.d.rotary_dim / 2;
    const float *c = p.cosines + (int64_t)pos * pairs, *s = p.sines + (int64_t)pos * pairs;
    Angles r = {F4{1.f, 1.f, 1.f, 1.f}, F4{0.f, 0.f, 0.f, 0.f}};
    if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (at.turn_a) r.c[e] = c[at.a / 2 + e], r.s[e] = s[at.a / 2 + e];
            if (at.turn_b) r.c[2 + e] = c[at.b / 2 + e], r.s[2 + e] = s[at.b / 2 + e];
        }
    } else if (at.turn_a) {
        r.c = load4<false>(c + 4 * i);
        r.s = load4<false>(s + 4 * i);
    }
    return r;
}
template <bool INTER> __device__ __forceinline__ void turn(F4 &x, F4 &y, const Angles &g, const Chunks &at) {
    const F4 a = x, b = y;
    if constexpr (INTER) {
        if (at.turn_a) x = F4{a[0] * g.c[0] - a[1] * g.s[0], a[1] * g.c[0] + a[0] * g.s[0], a[2] * g.c[1] - a[3] * g.s[1], a[3] * g.c[1] + a[2] * g.s[1]};
        if (at.turn_b) y = F4{b[0] * g.c[2] - b[1] * g.s[2], b[1] * g.c[2] + b[0] * g.s[2], b[2] * g.c[3] - b[3] * g.s[3], b[3] * g.c[3] + b[2] * g.s[3]};
    } else if (at.turn_a) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = a[e] * g.c[e] - b[e] * g.s[e];
            y[e] = b[e] * g.c[e] + a[e] * g.s[e];
        }
    }
}

// The bits of the largest |x| (those of NaN are above infinity's).
__device__ __forceinline__ uint32_t largest_of(F4 x, F4 y, uint32_t so_far) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t a = __float_as_uint(x[e]) & 0x7fffffffu, b = __float_as_uint(y[e]) & 0x7fffffffu;
        so_far = a > so_far ? a : so_far;
        so_far = b > so_far ? b : so_far;
    }
    return so_far;
}

constexpr int kWaves = 4, kHeld = 4;

// One wavefront a run and head: 64 / (head_dim / 8) rows side by side, kHeld times of them in registers; longer runs are read twice.
template <typename T, bool INTER, bool NT> __device__ __forceinline__ void store_run(const Args &p, const Run &run, int64_t t, int item) {
    const int lane = threadIdx.x & 63, hd = (int)p.c.head_dim, hkv = (int)p.c.kv_heads, per_row = hd / 8, abreast = 64 / per_row;
    const int slot = lane / per_row, i = lane % per_row;
    const bool keys = item < hkv, there = slot < abreast;
    const int64_t h = keys ? item : item - hkv, pitch = keys ? p.d.k_row_stride : p.d.v_row_stride;
    const float *src = keys ? p.k + t * pitch + h * p.d.k_head_stride : p.v + t * pitch + h * p.d.v_head_stride;
    uint8_t *dst = static_cast<uint8_t *>(keys ? p.k_cache : p.v_cache) + run.page * p.c.page_stride + h * p.c.head_stride;
    float *scale = (keys ? p.k_scales : p.v_scales) + run.page * p.sc.page_stride + h * p.sc.head_stride + (int)p.by_block((uint32_t)run.first);
    const bool turns = keys && p.d.rotary_dim > 0;
    const Chunks at = chunks_of<INTER>(i, hd, (int)p.d.rotary_dim, turns);
    const float had = run.row > run.first ? *scale : 0.f;
    F4 x[kHeld], y[kHeld];
    auto fetch = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int row = row0 + j * abreast + slot;
            x[j] = y[j] = F4{0.f, 0.f, 0.f, 0.f};
            if (there && row < run.tokens) {
                x[j] = load4<NT>(src + row * pitch + at.a);
                y[j] = load4<NT>(src + row * pitch + at.b);
            }
        }
        if (turns) {
            Angles g[kHeld];
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int row = row0 + j * abreast + slot;
                if (there && row < run.tokens) g[j] = angles_at<INTER>(p, run.pos + row, i, at);
            }
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                const int row = row0 + j * abreast + slot;
                if (there && row < run.tokens) turn<INTER>(x[j], y[j], g[j], at);
            }
        }
    };
    uint32_t largest = 0;
    const int held = kHeld * abreast;
    for (int row0 = 0; row0 < run.tokens; row0 += held) {
        fetch(row0);
#pragma unroll
        for (int j = 0; j < kHeld; ++j) largest = largest_of(x[j], y[j], largest);
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const uint32_t other = __shfl_xor(largest, m);
        largest = other > largest ? other : largest;
    }
    const float now = larger_scale(had, scale_for<T>(__uint_as_float(largest))), per = per_scale(now);
    if (run.row == run.first || now != had) {
        const float shrink = had * per;
        for (int row = run.first + slot; there && row < run.row; row += abreast) {
            uint32_t *w = reinterpret_cast<uint32_t *>(dst + row * p.c.row_stride + 8 * i);
            const uint32_t u = w[0], v = w[1];
            w[0] = now == now ? codes4<T>(values4<T>(u) * shrink) : 0u;
            w[1] = now == now ? codes4<T>(values4<T>(v) * shrink) : 0u;
        }
        if (lane == 0) *scale = now;
    }
    for (int row0 = 0; row0 < run.tokens; row0 += held) {
        if (run.tokens > held) fetch(row0);
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int row = row0 + j * abreast + slot;
            if (!there || row >= run.tokens) continue;
            uint8_t *to = dst + (run.row + row) * p.c.row_stride;
            *reinterpret_cast<uint32_t *>(to + at.a) = now == now ? codes4<T>(x[j] * per) : 0u;
            *reinterpret_cast<uint32_t *>(to + at.b) = now == now ? codes4<T>(y[j] * per) : 0u;
        }
    }
}

// `chunk` tokens for a wavefront, of which it does the runs that begin there; behind those the queries, 4 kHeld rows of a token for a wavefront.
template <typename T, bool INTER, bool NT> __global__ __launch_bounds__(64 * kWaves) void append_scaled_vec_kernel(const Args p, int chunk, int64_t kv_items, int q_parts) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hkv = (int)p.c.kv_heads;
    const int64_t work = (int64_t)blockIdx.x * kWaves + wave;
    if (work < kv_items) {
        const int item = (int)(work % (2 * hkv));
        const int64_t t0 = work / (2 * hkv) * chunk, end = t0 + chunk < p.d.tokens ? t0 + chunk : p.d.tokens;
        uint64_t begins = 1;
        if (chunk > 1) {  // not those that go on from the token before them
            const int64_t t = t0 + lane;
            bool first = t < end && p.positions[t] != -1;
            if (first && t > 0 && p.seq_ids[t] == p.seq_ids[t - 1] && p.positions[t] == p.positions[t - 1] + 1)
                first = (uint32_t)p.positions[t] == p.by_block((uint32_t)p.positions[t]) * (uint32_t)p.sc.block;  // (pages are whole blocks)
            begins = __ballot(first);
        }
        for (; begins; begins &= begins - 1) {
            const int64_t t = t0 + __builtin_ctzll(begins);
            const Run run = run_at(p, t, item == 0);
            if (run.tokens) store_run<T, INTER, NT>(p, run, t, item);
        }
        return;
    }
    const int64_t rest = work - kv_items, t = rest / q_parts;
    if (t >= p.d.tokens) return;
    const int pos = p.positions[t];
    int page, row;
    if (pos == -1 || !find_row(p, p.seq_ids[t], pos, &page, &row)) return;
    const int hd = (int)p.c.head_dim, per_row = hd / 8, abreast = 64 / per_row, slot = lane / per_row, i = lane % per_row;
    if (slot >= abreast) return;
    const Chunks at = chunks_of<INTER>(i, hd, (int)p.d.rotary_dim, p.d.rotary_dim > 0);
    const int h0 = (int)(rest % q_parts) * kHeld * abreast + slot, hq = (int)p.d.q_heads;
    F4 x[kHeld], y[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int h = h0 + j * abreast;
        if (h >= hq) continue;
        const float *src = p.q + t * p.d.q_row_stride + h * p.d.q_head_stride;
        x[j] = load4<NT>(src + at.a);
        y[j] = load4<NT>(src + at.b);
    }
    const Angles g = angles_at<INTER>(p, pos, i, at);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int h = h0 + j * abreast;
        if (h >= hq) continue;
        if (p.d.rotary_dim > 0) turn<INTER>(x[j], y[j], g, at);
        float *dst = p.q_out + t * p.d.out_row_stride + h * p.d.out_head_stride;
        if constexpr (NT) {
            __builtin_nontemporal_store(x[j], reinterpret_cast<F4 *>(dst + at.a));
            __builtin_nontemporal_store(y[j], reinterpret_cast<F4 *>(dst + at.b));
        } else {
            *reinterpret_cast<F4 *>(dst + at.a) = x[j];
            *reinterpret_cast<F4 *>(dst + at.b) = y[j];
        }
    }
}

bool aligned(const void *p, int64_t row_stride, int64_t head_stride) { return ((uintptr_t)p & 15u) == 0 && row_stride % 4 == 0 && head_stride % 4 == 0; }

// Rows, pairs and strides that 128-bit accesses take (32-bit ones in the caches).
bool takes_vectors(const Args &a) {
    const bool cache = (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache) & 3u) == 0 && a.c.page_stride % 4 == 0 && a.c.head_stride % 4 == 0 && a.c.row_stride % 4 == 0;
    const bool rows = a.c.head_dim % 8 == 0 && a.d.rotary_dim % 8 == 0 && aligned(a.k, a.d.k_row_stride, a.d.k_head_stride) && aligned(a.v, a.d.v_row_stride, a.d.v_head_stride);
    const bool queries = a.d.q_heads == 0 || (aligned(a.q, a.d.q_row_stride, a.d.q_head_stride) && aligned(a.q_out, a.d.out_row_stride, a.d.out_head_stride));
    return cache && rows && queries && (a.d.rotary_dim == 0 || (((uintptr_t)a.cosines | (uintptr_t)a.sines) & 15u) == 0);
}

template <typename T> int32_t launch(const Args &a, hipStream_t st) {
    if (takes_vectors(a)) {
        const int64_t heads = 2 * a.c.kv_heads, abreast = 64 / (a.c.head_dim / 8);
        const int chunk = a.d.tokens * heads <= 8192 ? 1 : (int)(a.sc.block < 64 ? a.sc.block : 64);
        const int64_t kv_items = fth::ceil_div(a.d.tokens, chunk) * heads, q_parts = fth::ceil_div(a.d.q_heads, abreast * kHeld);
        const int64_t blocks = fth::ceil_div(kv_items + a.d.tokens * q_parts, kWaves);
        FTH_ARG(blocks <= 2147483647LL, "paged_append_scaled: too many tokens for one launch");
        const bool nt = (double)a.d.tokens * a.c.head_dim * (8.0 * a.d.q_heads + 10.0 * a.c.kv_heads) > 0x1p28;
        auto go = [&](auto kernel) { kernel<<<dim3((unsigned)blocks), dim3(64 * kWaves), 0, st>>>(a, chunk, kv_items, (int)(q_parts ? q_parts : 1)); };
        if (a.d.interleaved && a.d.rotary_dim > 0) go(nt ? append_scaled_vec_kernel<T, true, true> : append_scaled_vec_kernel<T, true, false>);
        else go(nt ? append_scaled_vec_kernel<T, false, true> : append_scaled_vec_kernel<T, false, false>);
        FTH_CHECK_LAUNCH("paged_append_scaled");
        return FTH_OK;
    }
    const int per_token = (int)(2 * a.c.kv_heads + (a.d.q_heads > 0));
    FTH_ARG(a.d.tokens * per_token <= 2147483647LL, "paged_append_scaled: too many tokens for one launch");
    append_scaled_kernel<T><<<dim3((unsigned)(a.d.tokens * per_token)), dim3(64), 0, st>>>(a, per_token);
    FTH_CHECK_LAUNCH("paged_append_scaled");
    return FTH_OK;
}

}  // namespace

extern "C" {

void fth_dev_paged_scales_contiguous(fth_paged_scales *sc, const fth_paged_cache *c, int64_t block) {
    if (!sc || !c) return;
    sc->block = block;
    sc->head_stride = block > 0 ? c->page_size / block : 0;
    sc->page_stride = (int64_t)((uint64_t)c->kv_heads * (uint64_t)sc->head_stride);
}

int32_t fth_dev_paged_append_scaled_f32(const fth_paged_cache *c, const fth_paged_scales *sc, const fth_paged_append_desc *d, const float *q, const float *k, const float *v,
                                        const float *cosines, const float *sines, const int32_t *block_table, const int32_t *seq_ids, const int32_t *positions, float *q_out,
                                        void *k_cache, void *v_cache, float *k_scales, float *v_scales, int64_t *bad_index, fth_stream s) {
    if (int32_t rc = fth::check_paged_cache(c, "paged_append_scaled", true)) return rc;
    if (int32_t rc = fth::check_paged_scales(sc, c, "paged_append_scaled")) return rc;
    // what the call shares with the one for other caches, checked there; with queries alone that is all of it
    fth_paged_cache plain = *c;
    plain.dtype = FTH_DTYPE_F32;
    if (!k && !v) return fth_dev_paged_append_f32(&plain, d, q, nullptr, nullptr, cosines, sines, block_table, seq_ids, positions, q_out, nullptr, nullptr, bad_index, s);
    if (int32_t rc = fth::check_paged_append(&plain, d, q, k, v, cosines, sines, block_table, seq_ids, positions, q_out, k_cache, v_cache, "paged_append_scaled")) return rc;
    FTH_ARG(d->tokens == 0 || c->num_pages == 0 || (k_scales && v_scales), "paged_append_scaled: NULL scales");
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("paged_append_scaled(bad_index reset)");
    }
    if (d->tokens == 0) return FTH_OK;
    Args a;
    a.c = *c; a.d = *d; a.sc = *sc;
    a.q = q; a.k = k; a.v = v; a.cosines = cosines; a.sines = sines;
    a.table = block_table; a.seq_ids = seq_ids; a.positions = positions;
    a.q_out = q_out; a.k_cache = k_cache; a.v_cache = v_cache; a.k_scales = k_scales; a.v_scales = v_scales; a.bad = bad_index;
    a.by_page = fth::Divisor((uint32_t)c->page_size);
    a.by_block = fth::Divisor((uint32_t)sc->block);
    return c->dtype == FTH_DTYPE_I8 ? launch<fth::i8>(a, st) : launch<fth::e4m3>(a, st);
}

}  // extern "C"
