// What the operators on the paged K/V cache share: checks of the descriptor, the report of invalid entries, the storage types.
#pragma once

#include "common.hpp"

namespace fth {

using f16 = _Float16;
struct bf16 {
    uint16_t bits;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(f16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }

// bad_index starts at -1, the largest unsigned number; the minimum over all reports does not depend on their order.
static __global__ void reset_bad_kernel(int64_t *bad) { *bad = -1; }
__device__ __forceinline__ void report_bad_entry(int64_t *bad, int64_t at) {
    if (bad) atomicMin(reinterpret_cast<unsigned long long *>(bad), (unsigned long long)at);
}

inline int32_t check_paged_cache(const fth_paged_cache *c, const char *who) {
    FTH_ARG(c, "%s: NULL cache descriptor", who);
    FTH_ARG(c->dtype == FTH_DTYPE_F32 || c->dtype == FTH_DTYPE_F16 || c->dtype == FTH_DTYPE_BF16, "%s: a cache holds F32, F16 or BF16, not dtype %d", who, c->dtype);
    FTH_ARG(c->num_pages >= 0 && c->num_seqs >= 0 && c->max_pages >= 0, "%s: negative extent", who);
    FTH_ARG(c->kv_heads >= 1 && c->page_size >= 1, "%s: a page has at least one head and one row", who);
    FTH_ARG(c->head_dim >= 1 && c->head_dim <= 256, "%s: head_dim %lld is outside 1..256", who, (long long)c->head_dim);
    FTH_ARG(c->page_stride >= c->head_dim && c->head_stride >= c->head_dim && c->row_stride >= c->head_dim, "%s: a stride of the cache is below head_dim", who);
    FTH_ARG(c->table_stride >= c->max_pages, "%s: table_stride is below max_pages", who);
    // page numbers, positions, sequences and heads are 32-bit numbers in the kernels, and so is the divisor of positions
    const int64_t most = 2147483647LL;
    int64_t positions = 0, pages = 0, heads = 0, rows = 0, table = 0;
    bool over = c->num_pages > most || c->num_seqs > most || c->kv_heads > most || c->page_size > most || __builtin_mul_overflow(c->max_pages, c->page_size, &positions) || positions > most;
    over = over || __builtin_mul_overflow(c->num_pages, c->page_stride, &pages) || __builtin_mul_overflow(c->kv_heads, c->head_stride, &heads) ||
           __builtin_mul_overflow(c->page_size, c->row_stride, &rows) || __builtin_mul_overflow(c->num_seqs, c->table_stride, &table);
    const int64_t half = (int64_t)1 << 58;  // bytes of every offset fit 62 bits
    if (over || pages > half || heads > half || rows > half || table > half) return set_error(FTH_ERR_SIZE_OVERFLOW, "%s: the cache's extents overflow", who);
    return FTH_OK;
}

// n / d for 0 <= n < 2^31 by a multiplication: shift = ceil(log2 d), mul = ceil(2^(32 + shift) / d) - 2^32.
struct Divisor {
    uint32_t mul = 1, shift = 0;
    Divisor() = default;
    explicit Divisor(uint32_t d) {
        shift = d > 1 ? 32 - (uint32_t)__builtin_clz(d - 1) : 0;
        mul = (uint32_t)(((((uint64_t)1 << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)(((uint64_t)__umulhi(n, mul) + n) >> shift); }
};

inline bool stride_in_range(int64_t s) { return s >= 0 && s <= ((int64_t)1 << 40); }

}  // namespace fth
