// The next token of each row of logits from a given number: temperature, top-k, top-p, min-p.
//
// Weights are whole numbers W = round(2^kS exp((x - max) / T)): their sums do not depend on the order, so neither does the token. Tokens are
// ordered by a code of 64 bits, the complement of the logit's ordered bits above the index: smaller codes come first. Every
// filter keeps a prefix of that order, so the kept tokens are those up to a last code (and above min-p).

#include "devmath.hpp"
#include "paged.hpp"

namespace {

constexpr int kThreads = 1024;

struct SampleArgs {
    fth_sample_desc d;
    const float *logits, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    const double *uniform;
    int32_t *tokens;
    float *logprobs;
    int64_t *bad;
    double magic;  // 1.5 * 2^(52 - S): added to a weight in [0, 1], leaves round(2^S weight) in the low bits
};

__device__ __forceinline__ uint64_t code_of(float x, uint32_t v) {
    x = x == 0.f ? 0.f : x;  // -0 is 0
    const uint32_t b = __float_as_uint(x);
    return (uint64_t)((b & 0x80000000u) ? b : b ^ 0x7fffffffu) << 32 | v;
}

template <typename T, typename F> __device__ __forceinline__ T block_reduce(T x, T *lds, F op) {
    for (int m = 32; m > 0; m >>= 1) x = op(x, (T)__shfl_xor(x, m));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
    for (int w = 1; w < kThreads / 64; ++w) x = op(x, lds[w]);
    return x;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs p) {
    __shared__ uint64_t lds[kThreads / 64], weight[256];
    __shared__ uint32_t count[256];
    __shared__ float ldsf[kThreads / 64];
    __shared__ uint64_t found, above;
    __shared__ int token;
    const int64_t r = blockIdx.x;
    const int vocab = (int)p.d.vocab, t = threadIdx.x;
    const float *x = p.logits + r * p.d.logits_stride;
    const float temp = p.temperature ? p.temperature[r] : 1.f, top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f;
    int top_k = p.top_k ? p.top_k[r] : 0;
    const double u = p.uniform[r];
    bool bad = !(temp >= 0.f && temp < __builtin_inff()) || !(top_p >= 0.f) || !(min_p >= 0.f && min_p <= 1.f) || top_k < 0 || !(u >= 0.0 && u < 1.0);
    float big = -__builtin_inff();
    for (int v = t; v < vocab; v += kThreads) {
        const float z = x[v];
        bad |= !(z < __builtin_inff());
        big = fmaxf(big, z);
    }
    bad = __syncthreads_or(bad);
    big = block_reduce(big, ldsf, [](float a, float b) { return fmaxf(a, b); });
    if (bad || big == -__builtin_inff()) {
        if (t == 0) {
            p.tokens[r] = -1;
            if (p.logprobs) p.logprobs[r] = __builtin_nanf("");
            fth::report_bad_entry(p.bad, r);
        }
        return;
    }
    if (temp == 0.f) top_k = 1;
    const double rate = 1.4426950408889634074 / (temp == 0.f ? 1.0 : (double)temp);
    auto weight_of = [&](float z, double *w) {
        *w = fth::exp2_softmax(((double)z - (double)big) * rate);
        return (uint64_t)__builtin_bit_cast(int64_t, *w + p.magic) - (uint64_t)__builtin_bit_cast(int64_t, p.magic);
    };
    uint64_t last = ~0ull;  // the last code that is kept
    // The smallest code c <= last for which the tokens up to c are `k` at least (k > 0) or have a weight of `need`.
    auto boundary = [&](uint32_t k, uint64_t need) {
        uint64_t prefix = 0, had = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            if (t < 256) {
                weight[t] = 0;
                count[t] = 0;
            }
            __syncthreads();
            for (int v = t; v < vocab; v += kThreads) {
                const uint64_t c = code_of(x[v], v);
                if (c > last || (shift < 56 && c >> (shift + 8) != prefix)) continue;
                double w;
                const int at = (int)(c >> shift) & 255;
                if (k) atomicAdd(&count[at], 1u);
                else atomicAdd(reinterpret_cast<unsigned long long *>(&weight[at]), (unsigned long long)weight_of(x[v], &w));
            }
            __syncthreads();
            if (t == 0) {
                uint64_t upto = had;
                int at = 0;
                for (;; ++at) {
                    const uint64_t here = k ? count[at] : weight[at];
                    if (upto + here >= (k ? k : need) || at == 255) break;
                    upto += here;
                }
                found = prefix << 8 | at;
                above = upto;
            }
            __syncthreads();
            prefix = found;
            had = above;
        }
        return prefix;
    };
    auto sum_kept = [&](bool floor) {
        uint64_t sum = 0;
        for (int v = t; v < vocab; v += kThreads) {
            double w;
            if (code_of(x[v], v) > last) continue;
            const uint64_t whole = weight_of(x[v], &w);
            if (!floor || w >= (double)min_p) sum += whole;
        }
        return block_reduce(sum, lds, [](uint64_t a, uint64_t b) { return a + b; });
    };
    if (top_k > 0 && top_k < vocab) last = boundary(top_k, 0);
    if (top_p < 1.f) {
        const double need = (double)sum_kept(false) * (double)top_p;
        const uint64_t whole = (uint64_t)__builtin_ceil(need);
        last = boundary(0, whole < 1 ? 1 : whole);
    }
    const uint64_t total = sum_kept(true);
    uint64_t target = (uint64_t)((double)total * u);
    target = target < total ? target : total - 1;
    // in the order of the vocabulary
    uint64_t upto = 0;
    for (int v0 = 0; v0 < vocab; v0 += kThreads) {
        const int v = v0 + t;
        uint64_t whole = 0;
        if (v < vocab && code_of(x[v], v) <= last) {
            double w;
            whole = weight_of(x[v], &w);
            if (w < (double)min_p) whole = 0;
        }
        uint64_t here = whole;
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t other = __shfl_up(here, m);
            here += (t & 63) >= m ? other : 0;
        }
        __syncthreads();
        if ((t & 63) == 63) lds[t >> 6] = here;
        __syncthreads();
        uint64_t before = upto;
        for (int w = 0; w < kThreads / 64; ++w) {
            if (w < t >> 6) before += lds[w];
            upto += lds[w];
        }
        if (whole > 0 && before + here > target && before + here - whole <= target) {
            p.tokens[r] = v;
            if (p.logprobs) p.logprobs[r] = (float)log((double)whole / (double)total);
        }
        if (upto > target) return;
    }
}

int32_t check(const fth_sample_desc *d) {
    FTH_ARG(d, "sample: NULL descriptor");
    FTH_ARG(d->rows >= 0 && d->vocab >= 0, "sample: negative extent");
    FTH_ARG(d->logits_stride >= d->vocab, "sample: the row stride is below the vocabulary");
    if (d->logits_stride > ((int64_t)1 << 40) || d->vocab > 2147483647LL || d->rows > ((int64_t)1 << 20)) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "sample: extents overflow");
    FTH_ARG(d->rows == 0 || d->vocab > 0, "sample: no token to choose from");
    return FTH_OK;
}

}  // namespace

extern "C" {

size_t fth_dev_sample_workspace_bytes(const fth_sample_desc *d) { return check(d) == FTH_OK ? 0 : 0; }

int32_t fth_dev_sample_f32(const fth_sample_desc *d, const float *logits, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                           const double *uniform, int32_t *tokens, float *logprobs, int64_t *bad_index, void *workspace, size_t workspace_bytes, fth_stream s) {
    if (int32_t rc = check(d)) return rc;
    FTH_ARG(d->rows == 0 || (logits && uniform && tokens), "sample: NULL operand");
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("sample(bad_index reset)");
    }
    if (d->rows == 0) return FTH_OK;
    SampleArgs a;
    a.d = *d;
    a.logits = logits; a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.uniform = uniform;
    a.tokens = tokens; a.logprobs = logprobs; a.bad = bad_index;
    int bits = 0;
    while (((int64_t)1 << bits) < d->vocab) ++bits;
    const int s_bits = 62 - bits < 45 ? 62 - bits : 45;
    a.magic = __builtin_ldexp(1.5, 52 - s_bits);
    sample_kernel<<<dim3((unsigned)d->rows), dim3(kThreads), 0, st>>>(a);
    FTH_CHECK_LAUNCH("sample");
    return FTH_OK;
}

}  // extern "C"
