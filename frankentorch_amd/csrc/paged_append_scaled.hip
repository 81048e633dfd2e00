// Keys and values of new tokens into a paged cache of 8-bit numbers with a scale for each block of positions and head.
//
// A block's scale s is the smallest power of two whose 127 (448) multiples reach the largest element it was given: x / s is exact, so
// that an element is rounded once, and a scale that grows by 2^k takes what the block holds to code / 2^k. A run is the tokens of one block that stand
// one after the other in the call; whoever has its first token does all of it, so that no two workgroups touch one block. A run ends at the first token
// that is not at the next position: that one is reported, and what follows it in the block belongs to no run.
//
// Bound by reading the rows and writing the queries once: 3 prompts of up to 7001 tokens, 32 query heads on 8 of 128, e4m3, blocks of 48: 113 us, 6.0
// TB/s (element by element 473; a wavefront a run that first asks for its place 156). Short calls wait for loads that depend on each
// other, position -> page -> scale: 5.6 us for a step of 64 sequences, where an empty launch takes 5.

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
// Which of two scales holds: the larger (what was there may be negative, where something else has filled the cache), NaN before all.
__device__ __forceinline__ float larger_scale(float had, float needs) { return had != had || needs != needs ? __builtin_nanf("") : fabsf(had) > needs ? had : needs; }
// What elements are multiplied by: 0 under a scale that is none or subnormal (such a one holds for zeros alone).
__device__ __forceinline__ float per_scale(float s) { return fabsf(s) >= 0x1p-126f ? 1.f / s : 0.f; }

// To nearest even; |x| is within the type's range. NaN is for e4m3 alone, which has a code for it.
__device__ __forceinline__ uint32_t to_code(float x, fth::i8) {
    return (uint32_t)(int)fminf(fmaxf(__builtin_rintf(x), -127.f), 127.f) & 255u;
}
__device__ __forceinline__ uint32_t to_code(float x, fth::e4m3) {
    x = x == x ? fminf(fmaxf(x, -448.f), 448.f) : x;
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
            store(row, c, now == now ? fth::to_f32(dst[row * p.c.row_stride + c]) * shrink : 0.f);
        }
        if (lane == 0) *scale = now;
    }
    for (int64_t x = lane; x < (int64_t)run.tokens * hd; x += 64) {
        const int i = (int)(x / hd), c = (int)(x % hd);
        store(run.row + i, c, now == now ? element(i, c) * per : 0.f);
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

constexpr int kWaves = 4;

// `tokens` tokens from t on, all of one block from position `pos` of sequence `seq` on: one wavefront (TEAM: the workgroup) for their rows of one head, 64 /
// (head_dim / 8) of them side by side, HELD times as many in registers; longer runs are read twice. The rows are asked for before it is
// known where they go.
constexpr int kHeld = 4;  // at most
struct Team {
    uint32_t largest[kWaves];
    float had;
};
template <typename T, bool INTER, bool NT, bool TEAM, int HELD> __device__ __forceinline__ void store_run(const Args &p, int64_t t, int tokens, int pos, int seq, int item, Team &team) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, hd = (int)p.c.head_dim, hkv = (int)p.c.kv_heads, per_row = hd / 8, abreast = 64 / per_row;
    const int slot = lane / per_row, i = lane % per_row, held = HELD * abreast;
    const int from = TEAM ? wave * held : 0, step = TEAM ? kWaves * held : held;  // this wavefront's rows
    const bool keys = item < hkv, there = slot < abreast;
    const int64_t h = keys ? item : item - hkv, pitch = keys ? p.d.k_row_stride : p.d.v_row_stride;
    const float *src = keys ? p.k + t * pitch + h * p.d.k_head_stride : p.v + t * pitch + h * p.d.v_head_stride;
    const bool turns = keys && p.d.rotary_dim > 0;
    const Chunks at = chunks_of<INTER>(i, hd, (int)p.d.rotary_dim, turns);
    // rows that have an angle (the others have no place either, and are not stored)
    const int64_t angles = pos < 0 ? 0 : p.d.max_pos - pos;
    const int to_turn = !turns || angles < 0 ? 0 : angles < tokens ? (int)angles : tokens;
    F4 x[HELD], y[HELD];
    auto fetch = [&](int row0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int row = row0 + j * abreast + slot;
            x[j] = y[j] = F4{0.f, 0.f, 0.f, 0.f};
            if (there && row < tokens) {
                x[j] = load4<NT>(src + row * pitch + at.a);
                y[j] = load4<NT>(src + row * pitch + at.b);
            }
        }
    };
    auto turn_all = [&](int row0) __attribute__((always_inline)) {
        if (!turns) return;
        constexpr int AT_ONCE = INTER ? HELD / 2 : HELD;  // (registers)
#pragma unroll
        for (int j0 = 0; j0 < HELD; j0 += AT_ONCE) {
            Angles g[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int row = row0 + (j0 + j) * abreast + slot;
                if (there && row < to_turn) g[j] = angles_at<INTER>(p, pos + row, i, at);
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
                if (there && row0 + (j0 + j) * abreast + slot < to_turn) turn<INTER>(x[j0 + j], y[j0 + j], g[j], at);
            if (INTER) __builtin_amdgcn_sched_barrier(0);
        }
    };
    fetch(from);
    int page = 0, row = 0;
    const bool placed = find_row(p, seq, pos, &page, &row);
    const int first = placed ? (int)p.by_block((uint32_t)row) * (int)p.sc.block : 0;
    float *scale = (keys ? p.k_scales : p.v_scales) + (placed ? page : 0) * p.sc.page_stride + h * p.sc.head_stride + (int)p.by_block((uint32_t)first);
    float had = placed && row > first && (!TEAM || wave == 0) ? *scale : 0.f;
    turn_all(from);
    if (!placed) {
        if (item == 0 && threadIdx.x % (TEAM ? 64 * kWaves : 64) == 0) fth::report_bad_entry(p.bad, t);
        return;
    }
    if (p.d.rotary_dim > 0 && pos + (int64_t)tokens > p.d.max_pos) {  // its last tokens have no place
        const int rest = (int)(p.d.max_pos - pos);
        if (item == 0 && threadIdx.x % (TEAM ? 64 * kWaves : 64) == 0) fth::report_bad_entry(p.bad, t + rest);
        tokens = rest;
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if (from + j * abreast + slot >= tokens) x[j] = y[j] = F4{0.f, 0.f, 0.f, 0.f};
    }
    uint32_t largest = 0;
#pragma unroll
    for (int j = 0; j < HELD; ++j) largest = largest_of(x[j], y[j], largest);
    for (int row0 = from + step; row0 < tokens; row0 += step) {
        fetch(row0);
        turn_all(row0);
#pragma unroll
        for (int j = 0; j < HELD; ++j) largest = largest_of(x[j], y[j], largest);
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const uint32_t other = __shfl_xor(largest, m);
        largest = other > largest ? other : largest;
    }
    if constexpr (TEAM) {
        __syncthreads();  // what an earlier run left has been read
        if (lane == 0) {
            team.largest[wave] = largest;
            if (wave == 0) team.had = had;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) largest = team.largest[w] > largest ? team.largest[w] : largest;
        had = team.had;
    }
    const float now = larger_scale(had, scale_for<T>(__uint_as_float(largest))), per = per_scale(now);
    uint8_t *dst = static_cast<uint8_t *>(keys ? p.k_cache : p.v_cache) + page * p.c.page_stride + h * p.c.head_stride;
    if (row == first || now != had) {
        const float shrink = had * per;
        for (int old = first + slot + (TEAM ? wave * abreast : 0); there && old < row; old += abreast * (TEAM ? kWaves : 1)) {
            uint32_t *w = reinterpret_cast<uint32_t *>(dst + old * p.c.row_stride + 8 * i);
            const uint32_t u = w[0], v = w[1];
            w[0] = now == now ? codes4<T>(values4<T>(u) * shrink) : 0u;
            w[1] = now == now ? codes4<T>(values4<T>(v) * shrink) : 0u;
        }
        if (lane == 0 && (!TEAM || wave == 0)) *scale = now;
    }
    for (int row0 = from; row0 < tokens; row0 += step) {
        if (tokens > step) {
            fetch(row0);
            turn_all(row0);
        }
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int in_run = row0 + j * abreast + slot;
            if (!there || in_run >= tokens) continue;
            uint8_t *to = dst + (row + in_run) * p.c.row_stride;
            *reinterpret_cast<uint32_t *>(to + at.a) = now == now ? codes4<T>(x[j] * per) : 0u;
            *reinterpret_cast<uint32_t *>(to + at.b) = now == now ? codes4<T>(y[j] * per) : 0u;
        }
    }
}

// The rows of one token: its queries, and with blocks of one position (ONE) its keys and values, each row with a scale of its own.
template <typename T, bool INTER, bool NT, bool ONE> __device__ __forceinline__ void store_token(const Args &p, int64_t t, int part) {
    constexpr int HELD = 4;
    const int lane = threadIdx.x & 63, hd = (int)p.c.head_dim, hq = (int)p.d.q_heads, hkv = ONE ? (int)p.c.kv_heads : 0, per_row = hd / 8, abreast = 64 / per_row;
    const int slot = lane / per_row, i = lane % per_row, h0 = part * HELD * abreast + slot, rows = hq + 2 * hkv;
    const int pos = p.positions[t], seq = p.seq_ids[t];
    const bool there = slot < abreast;
    const Chunks turned_at = chunks_of<INTER>(i, hd, (int)p.d.rotary_dim, p.d.rotary_dim > 0), plain_at = chunks_of<INTER>(i, hd, 0, false);
    F4 x[HELD], y[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int h = h0 + j * abreast;
        x[j] = y[j] = F4{0.f, 0.f, 0.f, 0.f};
        if (!there || h >= rows) continue;
        const float *src = h < hq ? p.q + t * p.d.q_row_stride + h * p.d.q_head_stride
                           : h < hq + hkv ? p.k + t * p.d.k_row_stride + (h - hq) * p.d.k_head_stride
                                          : p.v + t * p.d.v_row_stride + (h - hq - hkv) * p.d.v_head_stride;
        const Chunks &at = h < hq + hkv ? turned_at : plain_at;
        x[j] = load4<NT>(src + at.a);
        y[j] = load4<NT>(src + at.b);
    }
    if (pos == -1) return;
    int page = 0, row = 0;
    if (!find_row(p, seq, pos, &page, &row)) {
        if (ONE && part == 0 && lane == 0) fth::report_bad_entry(p.bad, t);
        return;
    }
    const bool again = ONE && t > 0 && p.positions[t - 1] == pos && p.seq_ids[t - 1] == seq;  // once more the same place
    if (again && part == 0 && lane == 0) fth::report_bad_entry(p.bad, t);
    if (p.d.rotary_dim > 0) {
        const Angles g = angles_at<INTER>(p, pos, i, turned_at);
#pragma unroll
        for (int j = 0; j < HELD; ++j)
            if (h0 + j * abreast < hq + hkv) turn<INTER>(x[j], y[j], g, turned_at);
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int h = h0 + j * abreast;
        const bool mine = there && h < rows;
        if (mine && h < hq) {
            float *dst = p.q_out + t * p.d.out_row_stride + h * p.d.out_head_stride;
            if constexpr (NT) {
                __builtin_nontemporal_store(x[j], reinterpret_cast<F4 *>(dst + turned_at.a));
                __builtin_nontemporal_store(y[j], reinterpret_cast<F4 *>(dst + turned_at.b));
            } else {
                *reinterpret_cast<F4 *>(dst + turned_at.a) = x[j];
                *reinterpret_cast<F4 *>(dst + turned_at.b) = y[j];
            }
        }
        if constexpr (ONE) {
            uint32_t largest = largest_of(x[j], y[j], 0);
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {  // to the first lane of the row, which need not be a power of two long
                const uint32_t other = __shfl_down(largest, m);
                largest = i + m < per_row && other > largest ? other : largest;
            }
            largest = __shfl(largest, slot * per_row);
            if (!mine || h < hq || again) continue;
            const bool keys = h < hq + hkv;
            const int64_t hk = keys ? h - hq : h - hq - hkv;
            const Chunks &at = keys ? turned_at : plain_at;
            const float now = scale_for<T>(__uint_as_float(largest)), per = per_scale(now);
            uint8_t *to = static_cast<uint8_t *>(keys ? p.k_cache : p.v_cache) + page * p.c.page_stride + hk * p.c.head_stride + row * p.c.row_stride;
            *reinterpret_cast<uint32_t *>(to + at.a) = now == now ? codes4<T>(x[j] * per) : 0u;
            *reinterpret_cast<uint32_t *>(to + at.b) = now == now ? codes4<T>(y[j] * per) : 0u;
            if (i == 0) (keys ? p.k_scales : p.v_scales)[page * p.sc.page_stride + hk * p.sc.head_stride + row] = now;
        }
    }
}

// What a wavefront takes: one token's rows alone (RUNS none, blocks of one position); or the runs that begin in `chunk` tokens, for one head (one), and so
// all wavefronts of the workgroup together (team). Workgroups with rows of tokens stand between those with runs, which wait for loads that depend on each
// other.
enum class Runs { none, one, team };

struct Cut {
    uint32_t share;      // of the first b workgroups, b share / 2^32 have runs (0: all)
    int chunk, runs;     // tokens; items of a chunk and a head
    int parts;           // wavefronts for the rows of a token
    fth::Divisor by_heads, by_parts;
};

template <typename T, bool INTER, bool NT, Runs RUNS, int HELD> __global__ __launch_bounds__(64 * kWaves, HELD == 2 ? 5 : 4) void append_scaled_vec_kernel(const Args p, const Cut cut) {
    constexpr bool TEAM = RUNS == Runs::team;
    __shared__ Team team;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = 2 * (int)p.c.kv_heads;
    auto with_runs = [&](uint32_t b) { return RUNS == Runs::none ? 0 : cut.share ? (int)__umulhi(b, cut.share) : (int)b; };
    const int before = with_runs(blockIdx.x), upto = with_runs(blockIdx.x + 1);
    if (before == upto) {
        const int work = ((int)blockIdx.x - before) * kWaves + wave, t = (int)cut.by_parts((uint32_t)work);
        if (t < p.d.tokens) store_token<T, INTER, NT, RUNS == Runs::none>(p, t, work - t * cut.parts);
        return;
    }
    if constexpr (RUNS != Runs::none) {
        const int work = TEAM ? before : before * kWaves + wave;
        if (work >= cut.runs) return;
        const int group = (int)cut.by_heads((uint32_t)work), item = work - group * heads, chunk = cut.chunk, block = (int)p.sc.block;
        const int64_t t0 = (int64_t)group * chunk, t = t0 + lane;
        const bool there = t < p.d.tokens;
        const int pos = there ? p.positions[t] : -1, seq = there ? p.seq_ids[t] : -1;
        int pos_before = __shfl_up(pos, 1), seq_before = __shfl_up(seq, 1);
        if (lane == 0 && t0 > 0) pos_before = p.positions[t0 - 1], seq_before = p.seq_ids[t0 - 1];
        const bool known = t > 0 && pos >= 0 && pos_before >= 0 && seq == seq_before;
        const int start = pos >= 0 ? (int)p.by_block((uint32_t)pos) * block : 0;  // of its block (pages are whole blocks)
        const bool inside = known && pos_before >= start && pos_before - start < block, goes_on = inside && pos_before == pos - 1;
        const uint64_t on = __ballot(goes_on);
        if (item == 0 && lane < chunk && inside && !goes_on) fth::report_bad_entry(p.bad, t);
        for (uint64_t begins = __ballot(lane < chunk && there && pos != -1 && !inside); begins; begins &= begins - 1) {
            const int at = __builtin_ctzll(begins);
            const int first_pos = __builtin_amdgcn_readlane(pos, at), first_seq = __builtin_amdgcn_readlane(seq, at);
            const uint64_t others = ~(at < 63 ? on >> (at + 1) : 0);
            int n = 1 + (others ? __builtin_ctzll(others) : 64);
            // (a block that reaches past these 64 tokens)
            if (at + n >= 64) {
                n = 64 - at;
                const int most = first_pos < 0 ? n : block - (first_pos - (int)p.by_block((uint32_t)first_pos) * block);
                for (;;) {
                    const int64_t next = t0 + at + n + lane;
                    const bool more = n + lane < most && next < p.d.tokens && p.positions[next] == first_pos + n + lane && p.seq_ids[next] == first_seq;
                    const uint64_t every = __ballot(more);
                    n += ~every ? __builtin_ctzll(~every) : 64;
                    if (~every) break;
                }
            }
            store_run<T, INTER, NT, TEAM, HELD>(p, t0 + at, n, first_pos, first_seq, item, team);
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
        const bool one = a.sc.block == 1;
        // Tokens that a wavefront looks through for runs (the host does not know whether they make a few long ones or each its own). us for 1 / 4 / 32 of them,
        // 16 heads of 128: steps of 64 sequences 5.6 / 10.7 / 33, of 256 9.0 / 12.4 / 35, of 700 18.0 / 18.5 / 40, of 2000 43 / 38 / 57; 3 prompts of up to
        // 150 tokens, blocks of 48, 16.3 / 9.0 / 10.7, of up to 300 19.7 / 11.7 / 12.2, of 1000 37 / 28 / 23, of 7001 184 / 157 / 117; 8 of up
        // to 1024, 24 heads of 64, 53 / 18.6 / 12.6.
        const int most = a.d.tokens * heads <= 8192 ? 1 : a.d.tokens * heads <= 32768 ? 4 : 32, chunk = (int)(a.sc.block < most ? a.sc.block : most);
        const int64_t run_items = one ? 0 : fth::ceil_div(a.d.tokens, chunk) * heads, parts = fth::ceil_div(a.d.q_heads + (one ? heads : 0), abreast * 4);
        // Four wavefronts for a run that one would read twice (us, one / four: 3 prompts of up to 7001, blocks of 32 137 / 124, of 64 156 / 119; against it 8 of up
        // to 1024, heads of 64, blocks of 64 14.6 / 19).
        const bool team = a.sc.block > kHeld * abreast && chunk > 1;
        const int64_t run_blocks = team ? run_items : fth::ceil_div(run_items, kWaves), blocks = run_blocks + fth::ceil_div(a.d.tokens * parts, kWaves);
        FTH_ARG(run_items <= 2147483600LL && a.d.tokens * parts <= 2147483600LL && blocks <= 2147483647LL, "paged_append_scaled: too many tokens for one launch");
        // Nontemporal where rows and queries are more than the 256 MB last-level cache has (us, without / with: 3 prompts of up to 7001, 680 MB, 126 / 117, of
        // 4000 78 / 71, of 3000 61 / 55; of 2000, 190 MB, 42 / 38, but what comes next finds its queries there; 8 of up to 1024 12.6 / 12.9).
        const bool nt = (double)a.d.tokens * a.c.head_dim * (8.0 * a.d.q_heads + 10.0 * a.c.kv_heads) > 0x1p28;
        Cut cut;
        cut.chunk = chunk; cut.runs = (int)run_items; cut.parts = (int)(parts ? parts : 1);
        cut.share = run_blocks == blocks ? 0u : (uint32_t)((((uint64_t)run_blocks << 32) + (uint64_t)blocks - 1) / (uint64_t)blocks);  // rounded up: of all, run_blocks have them
        cut.by_heads = fth::Divisor((uint32_t)heads);
        cut.by_parts = fth::Divisor((uint32_t)cut.parts);
        auto go = [&](auto kernel) { kernel<<<dim3((unsigned)blocks), dim3(64 * kWaves), 0, st>>>(a, cut); };
        auto pick = [&](auto inter, auto past) {
            constexpr bool I = decltype(inter)::value, N = decltype(past)::value;
            // Rows that blocks do not have cost wavefronts (us, 4 / 2 rows a lane: heads of 64, blocks of 16 14.2 / 12.6, of 8 20.8 / 17.2; heads of 128, of 16 113 / 137, of
            // 8 121 / 117, of 4 135 / 124).
            if (one) go(append_scaled_vec_kernel<T, I, N, Runs::none, kHeld>);
            else if (team) go(append_scaled_vec_kernel<T, I, N, Runs::team, kHeld>);
            else if (a.sc.block > 2 * abreast) go(append_scaled_vec_kernel<T, I, N, Runs::one, kHeld>);
            else go(append_scaled_vec_kernel<T, I, N, Runs::one, 2>);
        };
        const bool inter = a.d.interleaved && a.d.rotary_dim > 0;
        if (inter) nt ? pick(std::true_type(), std::true_type()) : pick(std::true_type(), std::false_type());
        else nt ? pick(std::false_type(), std::true_type()) : pick(std::false_type(), std::false_type());
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
