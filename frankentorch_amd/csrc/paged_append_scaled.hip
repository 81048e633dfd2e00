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

template <typename T> int32_t launch(const Args &a, hipStream_t st) {
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
