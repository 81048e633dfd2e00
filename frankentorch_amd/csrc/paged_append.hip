// Keys and values of new tokens into a paged cache, with the position rotation of keys and queries on the way.
//
// HBM-bound: one pass over the packed projection, every K, V and query element read once and written once. A thread owns pairs of
// a rotation (both elements of each, so queries may be rotated in place) or the same number of elements that are only copied; no
// two threads touch one element. -ffp-contract=off rounds a c, b s and their difference one by one.
// What 128-bit accesses cannot take goes element by element.
//
// Measured: three prompts of up to 7001 tokens, 32 query and 8 K/V heads of 128, f16 (712 MB) 109 us, 6.5 TB/s, what a copy of that
// size reaches (through the caches 134; element by element 447); eight of up to 1024 tokens, 12 heads of 64, fp32 (68 MB) 13 us
// (50); a step of 64 sequences 3.8 us. Four tokens a workgroup where it holds all heads of one are slower (22 us for the eight
// prompts: registers), and so is a workgroup that looks the next token up while this one's rows are on their way (145 us for the three).

#include <type_traits>

#include "paged.hpp"

namespace {

constexpr int kBlock = 256;

struct AppendArgs {
    fth_paged_cache c;
    fth_paged_append_desc d;
    const float *q, *k, *v, *cosines, *sines;
    const int32_t *table, *seq_ids, *positions;
    float *q_out;
    void *k_cache, *v_cache;
    int64_t *bad;
    fth::Divisor by_page;
    int kv_heads;           // 0: queries only
    int pair_units, units;  // of a rotated head, pairs first; of a token
};

// Where token t goes in the cache (nowhere without keys); false when there is no such place.
__device__ __forceinline__ bool find_slot(const AppendArgs &p, int64_t t, int pos, int64_t *slot) {
    if (pos < 0 || (p.d.rotary_dim > 0 && pos >= p.d.max_pos)) return false;
    if (p.kv_heads == 0) return true;
    const int seq = p.seq_ids[t];
    if (seq < 0 || seq >= p.c.num_seqs || pos >= p.c.max_pages * p.c.page_size) return false;
    const int index = (int)p.by_page((uint32_t)pos);
    const int page = p.table[(int64_t)seq * p.c.table_stride + index];
    if (page < 0 || page >= p.c.num_pages) return false;
    *slot = (int64_t)page * p.c.page_stride + (int64_t)(pos - index * (int)p.c.page_size) * p.c.row_stride;
    return true;
}

__device__ __forceinline__ void store_as(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_as(fth::f16 *p, float x) { *p = (fth::f16)x; }
__device__ __forceinline__ void store_as(fth::bf16 *p, float x) { *reinterpret_cast<__bf16 *>(p) = (__bf16)x; }

// Unit u of one head's row: a pair while u < pairs, one element that is copied from there on.
template <typename T> __device__ __forceinline__ void head_unit(const float *src, T *dst, int u, int pairs, bool interleaved, const float *c, const float *s) {
    if (u >= pairs) {
        store_as(dst + pairs + u, src[pairs + u]);
        return;
    }
    const int ia = interleaved ? 2 * u : u, ib = interleaved ? 2 * u + 1 : u + pairs;
    const float a = src[ia], b = src[ib], cc = c[u], ss = s[u];
    store_as(dst + ia, a * cc - b * ss);
    store_as(dst + ib, b * cc + a * ss);
}

template <typename T> __global__ __launch_bounds__(kBlock) void paged_append_kernel(const AppendArgs p, int blocks_per_token) {
    const int64_t t = blockIdx.x / blocks_per_token;
    const int part = (int)(blockIdx.x % blocks_per_token);
    const int pos = p.positions[t];
    if (pos == -1) return;
    int64_t slot = 0;
    if (!find_slot(p, t, pos, &slot)) {
        if (part == 0 && threadIdx.x == 0) fth::report_bad_entry(p.bad, t);
        return;
    }
    const int pairs = (int)p.d.rotary_dim / 2, hd = (int)p.c.head_dim, hq = (int)p.d.q_heads, hkv = p.kv_heads;
    const float *c = p.cosines + (int64_t)pos * pairs, *s = p.sines + (int64_t)pos * pairs;
    const bool inter = p.d.interleaved != 0;
    const int rotated = (hq + hkv) * p.pair_units;
    for (int u = part * kBlock + threadIdx.x; u < p.units; u += blocks_per_token * kBlock) {
        if (u < rotated) {
            const int h = u / p.pair_units, i = u % p.pair_units;
            if (h < hq) {
                head_unit(p.q + t * p.d.q_row_stride + h * p.d.q_head_stride, p.q_out + t * p.d.out_row_stride + h * p.d.out_head_stride, i, pairs, inter, c, s);
            } else {
                head_unit(p.k + t * p.d.k_row_stride + (h - hq) * p.d.k_head_stride, static_cast<T *>(p.k_cache) + slot + (h - hq) * p.c.head_stride, i, pairs, inter, c, s);
            }
        } else {
            const int h = (u - rotated) / hd, i = (u - rotated) % hd;
            head_unit(p.v + t * p.d.v_row_stride + h * p.d.v_head_stride, static_cast<T *>(p.v_cache) + slot + h * p.c.head_stride, i, 0, false, c, s);
        }
    }
}

using F4 = float __attribute__((ext_vector_type(4)));

template <bool NT> __device__ __forceinline__ F4 load4(const float *p) {
    const F4 *v = reinterpret_cast<const F4 *>(p);
    return NT ? __builtin_nontemporal_load(v) : *v;
}
// Two adjacent pairs.
__device__ __forceinline__ F4 turned(F4 v, float c0, float s0, float c1, float s1) {
    return F4{v[0] * c0 - v[1] * s0, v[1] * c0 + v[0] * s0, v[2] * c1 - v[3] * s1, v[3] * c1 + v[2] * s1};
}
// Eight elements as they are stored: four at `a` and four at `b`, which are the next four when `adjacent`.
template <bool NT> __device__ __forceinline__ void store8(float *a, float *b, F4 x, F4 y, bool) {
    if constexpr (NT) {
        __builtin_nontemporal_store(x, reinterpret_cast<F4 *>(a));
        __builtin_nontemporal_store(y, reinterpret_cast<F4 *>(b));
    } else {
        *reinterpret_cast<F4 *>(a) = x;
        *reinterpret_cast<F4 *>(b) = y;
    }
}
template <bool NT, typename T> __device__ __forceinline__ void store8(T *a, T *b, F4 x, F4 y, bool adjacent) {
    using E = typename std::conditional<std::is_same<T, fth::bf16>::value, __bf16, _Float16>::type;
    using E4 = E __attribute__((ext_vector_type(4)));
    using E8 = E __attribute__((ext_vector_type(8)));
    const E4 u = __builtin_convertvector(x, E4), v = __builtin_convertvector(y, E4);
    if (adjacent) {
        *reinterpret_cast<E8 *>(a) = __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        *reinterpret_cast<E4 *>(a) = u;
        *reinterpret_cast<E4 *>(b) = v;
    }
}

// Whole vectors: a thread owns two chunks of four elements at one place of the row and takes them from several heads, so that the
// tables' entries are read once; kHeads rows are in flight per thread. The chunks are the two sides of four pairs
// (i, i + rotary_dim / 2), else neighbours, which a 16-bit cache takes in one store.
// STREAM, for what the caches cannot hold: operands and rotated queries go past them, and then every access has to cover whole lines,
// so chunks that are no pairs come from the two halves of what they cover (an fp32 cache is stored the same way; 16-bit ones, whose
// rows are then stored by half lines, go through the caches).
constexpr int kHeads = 4;
template <typename T, bool INTER, bool STREAM> __global__ __launch_bounds__(kBlock) void paged_append_vec_kernel(const AppendArgs p, int blocks_per_token) {
    const int64_t t = blockIdx.x / (unsigned)blocks_per_token;
    const int part = (int)(blockIdx.x % (unsigned)blocks_per_token);
    const int pos = p.positions[t];
    if (pos == -1) return;
    const int hd = (int)p.c.head_dim, per_row = hd / 8, slots = kBlock / per_row;
    int64_t at = 0;
    if (!find_slot(p, t, pos, &at)) {
        if (part == 0 && threadIdx.x == 0) fth::report_bad_entry(p.bad, t);
        return;
    }
    const int slot = (int)threadIdx.x / per_row, i = (int)threadIdx.x % per_row;
    if (slot >= slots) return;
    const int rotary = (int)p.d.rotary_dim, hq = (int)p.d.q_heads, hkv = p.kv_heads, heads = hq + 2 * hkv;
    const int va = STREAM ? 4 * i : 8 * i, vb = STREAM ? hd / 2 + 4 * i : 8 * i + 4;  // chunks of a row that is only copied
    int ra = va, rb = vb;                                                           // of one that is rotated
    bool turn_a = va < rotary, turn_b = vb < rotary;
    F4 c = {1.f, 1.f, 1.f, 1.f}, s = {0.f, 0.f, 0.f, 0.f};
    const float *cosines = p.cosines + (int64_t)pos * (rotary / 2), *sines = p.sines + (int64_t)pos * (rotary / 2);
    if constexpr (INTER) {  // two pairs a chunk
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (turn_a) c[e] = cosines[va / 2 + e], s[e] = sines[va / 2 + e];
            if (turn_b) c[2 + e] = cosines[vb / 2 + e], s[2 + e] = sines[vb / 2 + e];
        }
    } else {
        turn_a = turn_b = 8 * i < rotary;
        if (turn_a) {
            ra = 4 * i;
            rb = rotary / 2 + 4 * i;
            c = load4<false>(cosines + 4 * i);
            s = load4<false>(sines + 4 * i);
        } else if (STREAM) {
            ra = rotary + 4 * (i - rotary / 8);
            rb = ra + (hd - rotary) / 2;
        }
    }
    const int stride = slots * blocks_per_token;
    for (int h0 = part * slots + slot; h0 < heads; h0 += kHeads * stride) {
        F4 a[kHeads], b[kHeads];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = h0 + j * stride;
            if (h >= heads) continue;
            const float *src = h < hq ? p.q + t * p.d.q_row_stride + h * p.d.q_head_stride
                               : h < hq + hkv ? p.k + t * p.d.k_row_stride + (h - hq) * p.d.k_head_stride
                                              : p.v + t * p.d.v_row_stride + (h - hq - hkv) * p.d.v_head_stride;
            a[j] = load4<STREAM>(src + (h < hq + hkv ? ra : va));
            b[j] = load4<STREAM>(src + (h < hq + hkv ? rb : vb));
        }
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            const int h = h0 + j * stride;
            if (h >= heads) continue;
            const bool turns = h < hq + hkv;
            F4 x = a[j], y = b[j];
            if constexpr (INTER) {
                if (turns && turn_a) x = turned(x, c[0], s[0], c[1], s[1]);
                if (turns && turn_b) y = turned(y, c[2], s[2], c[3], s[3]);
            } else if (turns && turn_a) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = a[j][e] * c[e] - b[j][e] * s[e];
                    y[e] = b[j][e] * c[e] + a[j][e] * s[e];
                }
            }
            const int xa = turns ? ra : va, xb = turns ? rb : vb;
            if (h < hq) {
                float *dst = p.q_out + t * p.d.out_row_stride + h * p.d.out_head_stride;
                store8<STREAM>(dst + xa, dst + xb, x, y, false);
            } else {
                T *dst = turns ? static_cast<T *>(p.k_cache) + at + (h - hq) * p.c.head_stride : static_cast<T *>(p.v_cache) + at + (h - hq - hkv) * p.c.head_stride;
                store8<STREAM>(dst + xa, dst + xb, x, y, !STREAM && (INTER || !turns || !turn_a));
            }
        }
    }
}

bool aligned(const void *p, int64_t row_stride, int64_t head_stride, int64_t elems) {
    return ((uintptr_t)p & 15u) == 0 && row_stride % elems == 0 && head_stride % elems == 0;
}

// Rows, pairs and strides that 128-bit accesses take.
template <typename T> bool takes_vectors(const AppendArgs &a) {
    const int64_t ch = 16 / (int64_t)sizeof(T);
    const bool cache = a.kv_heads == 0 || (a.c.page_stride % ch == 0 && aligned(a.k_cache, a.c.row_stride, a.c.head_stride, ch) &&
                                           aligned(a.v_cache, a.c.row_stride, a.c.head_stride, ch) && aligned(a.k, a.d.k_row_stride, a.d.k_head_stride, 4) &&
                                           aligned(a.v, a.d.v_row_stride, a.d.v_head_stride, 4));
    const bool rows = a.c.head_dim % 8 == 0 && a.d.rotary_dim % 8 == 0 &&
                      (a.d.q_heads == 0 || (aligned(a.q, a.d.q_row_stride, a.d.q_head_stride, 4) && aligned(a.q_out, a.d.out_row_stride, a.d.out_head_stride, 4)));
    return cache && rows && (a.d.rotary_dim == 0 || (((uintptr_t)a.cosines | (uintptr_t)a.sines) & 15u) == 0);
}

template <typename T> int32_t launch(const AppendArgs &a, hipStream_t st) {
    if (takes_vectors<T>(a)) {
        const int64_t slots = kBlock / (a.c.head_dim / 8), heads = a.d.q_heads + 2 * a.kv_heads;
        // A workgroup a token and four rows a thread; one row a thread where tokens are few (64 of 48 heads of 128: 4.5 -> 3.7 us).
        const int64_t blocks_per_token = fth::ceil_div(heads, a.d.tokens < 1024 ? slots : slots * kHeads);
        FTH_ARG(a.d.tokens * blocks_per_token <= 2147483647LL, "paged_append: too many tokens for one launch");
        // past the caches from their 256 MB on (us, with / without: 712 MB, f16 cache 112 / 134, 789 MB, fp32 cache 132 / 150, 271 MB,
        // fp32 cache 54 / 59; 325 MB level; 68 MB 17.2 / 16.2)
        const double bytes = (double)a.d.tokens * a.c.head_dim * (8.0 * a.d.q_heads + 2.0 * a.kv_heads * (4 + sizeof(T)));
        const bool stream = bytes > 0x1p28;
        auto go = [&](auto k) { k<<<dim3((unsigned)(a.d.tokens * blocks_per_token)), dim3(kBlock), 0, st>>>(a, (int)blocks_per_token); };
        if (a.d.interleaved && a.d.rotary_dim > 0) go(stream ? paged_append_vec_kernel<T, true, true> : paged_append_vec_kernel<T, true, false>);
        else go(stream ? paged_append_vec_kernel<T, false, true> : paged_append_vec_kernel<T, false, false>);
        FTH_CHECK_LAUNCH("paged_append");
        return FTH_OK;
    }
    const int64_t per_token = fth::ceil_div(a.units, kBlock);
    FTH_ARG(a.d.tokens * per_token <= 2147483647LL, "paged_append: too many tokens for one launch");
    paged_append_kernel<T><<<dim3((unsigned)(a.d.tokens * per_token)), dim3(kBlock), 0, st>>>(a, (int)per_token);
    FTH_CHECK_LAUNCH("paged_append");
    return FTH_OK;
}

}  // namespace

extern "C" {

void fth_dev_paged_cache_contiguous(fth_paged_cache *c, int64_t num_pages, int64_t page_size, int64_t kv_heads, int64_t head_dim, int64_t num_seqs, int64_t max_pages,
                                int32_t dtype) {
    if (!c) return;
    std::memset(c, 0, sizeof *c);
    c->num_pages = num_pages;
    c->page_size = page_size;
    c->kv_heads = kv_heads;
    c->head_dim = head_dim;
    c->row_stride = head_dim;
    // wrapped products of sizes that no memory holds; the calls refuse such caches
    c->head_stride = (int64_t)((uint64_t)page_size * (uint64_t)head_dim);
    c->page_stride = (int64_t)((uint64_t)kv_heads * (uint64_t)c->head_stride);
    c->num_seqs = num_seqs;
    c->max_pages = c->table_stride = max_pages;
    c->dtype = dtype;
}

int32_t fth_dev_paged_append_f32(const fth_paged_cache *c, const fth_paged_append_desc *d, const float *q, const float *k, const float *v, const float *cosines,
                                 const float *sines, const int32_t *block_table, const int32_t *seq_ids, const int32_t *positions, float *q_out, void *k_cache,
                                 void *v_cache, int64_t *bad_index, fth_stream s) {
    if (int32_t rc = fth::check_paged_cache(c, "paged_append")) return rc;
    FTH_ARG(d, "paged_append: NULL descriptor");
    FTH_ARG(d->tokens >= 0 && d->q_heads >= 0, "paged_append: negative extent");
    FTH_ARG(d->rotary_dim >= 0 && d->rotary_dim % 2 == 0 && d->rotary_dim <= c->head_dim, "paged_append: rotary_dim %lld is odd or outside 0..head_dim",
            (long long)d->rotary_dim);
    FTH_ARG(d->rotary_dim == 0 || d->max_pos >= 0, "paged_append: negative max_pos");
    for (int64_t x : {d->q_row_stride, d->q_head_stride, d->k_row_stride, d->k_head_stride, d->v_row_stride, d->v_head_stride, d->out_row_stride, d->out_head_stride})
        FTH_ARG(fth::stride_in_range(x), "paged_append: a stride is negative or over 2^40");
    if (d->q_heads > (1 << 20) || d->q_heads + c->kv_heads > (1 << 20) || d->tokens > 2147483647LL) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "paged_append: extents overflow");
    if (d->tokens > 0) {
        FTH_ARG(positions && (k != nullptr) == (v != nullptr) && (k || d->q_heads > 0), "paged_append: NULL operand");
        FTH_ARG(!k || (seq_ids && (block_table || c->max_pages == 0) && ((k_cache && v_cache) || c->num_pages == 0)), "paged_append: NULL cache, table or sequences");
        FTH_ARG(d->q_heads == 0 || (q && q_out), "paged_append: NULL queries");
        FTH_ARG(d->rotary_dim == 0 || (cosines && sines), "paged_append: NULL rotation tables");
        FTH_ARG(q != q_out || d->q_heads == 0 || (d->q_row_stride == d->out_row_stride && d->q_head_stride == d->out_head_stride),
                "paged_append: queries rotated in place need the strides they have");
    }
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("paged_append(bad_index reset)");
    }
    if (d->tokens == 0) return FTH_OK;
    AppendArgs a;
    a.c = *c;
    a.d = *d;
    a.q = q; a.k = k; a.v = v; a.cosines = cosines; a.sines = sines;
    a.table = block_table; a.seq_ids = seq_ids; a.positions = positions;
    a.q_out = q_out; a.k_cache = k_cache; a.v_cache = v_cache; a.bad = bad_index;
    a.by_page = fth::Divisor((uint32_t)c->page_size);
    a.pair_units = (int)(c->head_dim - d->rotary_dim / 2);
    a.kv_heads = k ? (int)c->kv_heads : 0;
    a.units = (int)((d->q_heads + a.kv_heads) * a.pair_units + a.kv_heads * c->head_dim);
    switch (c->dtype) {
        case FTH_DTYPE_F32: return launch<float>(a, st);
        case FTH_DTYPE_F16: return launch<fth::f16>(a, st);
        default: return launch<fth::bf16>(a, st);
    }
}

}  // extern "C"
