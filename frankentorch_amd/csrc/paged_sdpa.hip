// Attention of the last one to eight tokens of every sequence over a paged K/V cache.
//
//   out[s, i, h] = sum_j w_j v_j / sum_j w_j,   w_j = exp(x_j - max x),   x_j = scale q . k_j,   j < lens[s] - new_tokens + i + 1
//
// One wavefront a query row: 64 keys at a time, a key per lane for the scores, columns over the lanes for the outputs, a
// running maximum and sum (fp32) in between. Bound by reading the cache; every query head of a group reads its K/V head again.

#include "paged.hpp"

namespace {

constexpr float kLog2e = 1.44269502162933349609375f;

struct PagedArgs {
    fth_paged_cache c;
    fth_paged_sdpa_desc d;
    const float *q;
    const void *k, *v;
    const int32_t *table, *lens;
    float *out;
    int64_t *bad;
    float scale;
};

template <typename F> __device__ __forceinline__ float wave_reduce(float x, F op) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    return x;
}

template <typename T> __global__ __launch_bounds__(64) void paged_sdpa_rows_kernel(const PagedArgs p) {
    __shared__ float qs[256], ps[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x, hd = (int)p.c.head_dim, page_size = (int)p.c.page_size;
    const int64_t row = blockIdx.x;  // (sequence * new_tokens + i) * q_heads + h
    const int h = (int)(row % p.d.q_heads), i = (int)(row / p.d.q_heads % p.d.new_tokens);
    const int64_t seq = row / p.d.q_heads / p.d.new_tokens;
    const int64_t hk = h / (p.d.q_heads / p.c.kv_heads);
    const T *K = static_cast<const T *>(p.k) + hk * p.c.head_stride, *V = static_cast<const T *>(p.v) + hk * p.c.head_stride;
    const int64_t most = p.c.max_pages * p.c.page_size < p.d.max_len ? p.c.max_pages * p.c.page_size : p.d.max_len;
    const int len = p.lens[seq];
    bool bad = len < 0 || len > most;
    const int sees = bad ? 0 : len - (int)p.d.new_tokens + i + 1;
    const float *q = p.q + seq * p.d.q_seq_stride + i * p.d.q_row_stride + h * p.d.q_head_stride;
    for (int c = lane; c < hd; c += 64) qs[c] = q[c];
    __syncthreads();
    float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -__builtin_inff(), l = 0.f;
    for (int key0 = 0; key0 < sees; key0 += 64) {
        const int key = key0 + lane, n = sees - key0 < 64 ? sees - key0 : 64;
        float x = -__builtin_inff();
        if (lane < n) {
            int page = p.table[seq * p.c.table_stride + key / page_size];
            if (page < 0 || page >= p.c.num_pages) {
                bad = true;
                page = -1;
            }
            const int64_t off = page < 0 ? -1 : (int64_t)page * p.c.page_stride + (int64_t)(key % page_size) * p.c.row_stride;
            at[lane] = off;
            if (page >= 0) {
                float dot = 0.f;
                for (int c = 0; c < hd; ++c) dot = __builtin_fmaf(qs[c], fth::to_f32(K[off + c]), dot);
                x = dot * p.scale;
            }
        }
        const float m_new = fmaxf(m, wave_reduce(x, [](float a, float b) { return fmaxf(a, b); }));
        const float ref = m_new == -__builtin_inff() ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f((m - ref) * kLog2e), w = lane < n ? __builtin_amdgcn_exp2f((x - ref) * kLog2e) : 0.f;
        m = m_new;
        l = l * alpha + wave_reduce(w, [](float a, float b) { return a + b; });
        ps[lane] = w;
        __syncthreads();
        for (int j = 0; j < 4; ++j) {
            const int c = lane + 64 * j;
            if (c >= hd) break;
            float acc = o[j] * alpha;
            for (int r = 0; r < n; ++r)
                if (at[r] >= 0) acc = __builtin_fmaf(ps[r], fth::to_f32(V[at[r] + c]), acc);
            o[j] = acc;
        }
        __syncthreads();
    }
    bad = __any(bad);
    if (bad && lane == 0) fth::report_bad_entry(p.bad, seq);
    float *out = p.out + seq * p.d.o_seq_stride + i * p.d.o_row_stride + h * p.d.o_head_stride;
    for (int j = 0; j < 4; ++j) {
        const int c = lane + 64 * j;
        if (c < hd) out[c] = bad ? __builtin_nanf("") : sees <= 0 ? 0.f : o[j] / l;
    }
}

template <typename T> int32_t launch(const PagedArgs &a, hipStream_t st) {
    paged_sdpa_rows_kernel<T><<<dim3((unsigned)(a.c.num_seqs * a.d.new_tokens * a.d.q_heads)), dim3(64), 0, st>>>(a);
    FTH_CHECK_LAUNCH("paged_sdpa");
    return FTH_OK;
}

int32_t check(const fth_paged_cache *c, const fth_paged_sdpa_desc *d) {
    if (int32_t rc = fth::check_paged_cache(c, "paged_sdpa", nullptr)) return rc;
    FTH_ARG(d, "paged_sdpa: NULL descriptor");
    FTH_ARG(d->q_heads >= 1 && d->q_heads % c->kv_heads == 0, "paged_sdpa: %lld query heads on %lld K/V heads", (long long)d->q_heads, (long long)c->kv_heads);
    FTH_ARG(d->new_tokens >= 1 && d->new_tokens <= 8, "paged_sdpa: new_tokens %lld is outside 1..8", (long long)d->new_tokens);
    FTH_ARG(d->max_len >= 0 && d->max_len <= 2147483647LL, "paged_sdpa: max_len %lld is outside 0..2^31 - 1", (long long)d->max_len);
    for (int64_t x : {d->q_seq_stride, d->q_row_stride, d->q_head_stride, d->o_seq_stride, d->o_row_stride, d->o_head_stride})
        FTH_ARG(fth::stride_in_range(x), "paged_sdpa: a stride is negative or over 2^40");
    int64_t rows = 0;
    if (__builtin_mul_overflow(c->num_seqs * d->new_tokens, d->q_heads, &rows) || rows > 2147483647LL)
        return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "paged_sdpa: too many query rows for one launch");
    return FTH_OK;
}

}  // namespace

extern "C" {

size_t fth_dev_paged_sdpa_workspace_bytes(const fth_paged_cache *c, const fth_paged_sdpa_desc *d) {
    return check(c, d) == FTH_OK ? 0 : 0;
}

int32_t fth_dev_paged_sdpa_f32(const fth_paged_cache *c, const fth_paged_sdpa_desc *d, float scale, const float *q, const void *k_cache, const void *v_cache,
                               const int32_t *block_table, const int32_t *lens, float *out, int64_t *bad_index, void *workspace, size_t workspace_bytes,
                               fth_stream s) {
    if (int32_t rc = check(c, d)) return rc;
    FTH_ARG(c->num_seqs == 0 || (q && lens && out && (block_table || c->max_pages == 0) && ((k_cache && v_cache) || c->num_pages == 0)), "paged_sdpa: NULL operand");
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("paged_sdpa(bad_index reset)");
    }
    if (c->num_seqs == 0) return FTH_OK;
    (void)workspace;
    (void)workspace_bytes;
    PagedArgs a;
    a.c = *c;
    a.d = *d;
    a.q = q; a.k = k_cache; a.v = v_cache; a.table = block_table; a.lens = lens; a.out = out; a.bad = bad_index;
    a.scale = scale;
    switch (c->dtype) {
        case FTH_DTYPE_F32: return launch<float>(a, st);
        case FTH_DTYPE_F16: return launch<fth::f16>(a, st);
        default: return launch<fth::bf16>(a, st);
    }
}

}  // extern "C"
