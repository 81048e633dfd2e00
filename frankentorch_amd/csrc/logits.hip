// Penalties for repeated tokens, a bias and a mask of allowed tokens on the logits of a generation step.
//
// A workgroup owns one row's logits over a stretch of the vocabulary. It counts the history's tokens that fall into its stretch
// in LDS (integer atomics: the counts do not depend on their order), then makes one pass over the logits. Each workgroup of a row
// scans the whole history, which comes from L2; in return nothing is handed from one launch to another.

#include "paged.hpp"

namespace {

constexpr int kBlock = 256, kStretch = 4096;
constexpr uint32_t kGiven = 0x80000000u;  // bit 31: among the given tokens; below it: times generated

struct LogitsArgs {
    fth_logits_desc d;
    const float *logits, *repetition, *frequency, *presence, *bias;
    const int32_t *history, *history_len, *prompt_len;
    const uint32_t *mask;
    float *out;
    int64_t *bad;
    int stretches;
};

__global__ __launch_bounds__(kBlock) void logits_process_kernel(const LogitsArgs p) {
    __shared__ uint32_t seen[kStretch];
    const int64_t r = blockIdx.x / p.stretches;
    const int64_t v0 = (int64_t)(blockIdx.x % p.stretches) * kStretch;
    const int n = (int)(p.d.vocab - v0 < kStretch ? p.d.vocab - v0 : kStretch);
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (p.history) {
        for (int i = threadIdx.x; i < n; i += kBlock) seen[i] = 0;
        __syncthreads();
        const int len = p.history_len[r], prompt = p.prompt_len[r];
        bool bad = len < 0 || len > p.d.history_stride || prompt < 0 || prompt > len;
        for (int i = threadIdx.x; i < (bad ? 0 : len); i += kBlock) {
            const int64_t id = p.history[r * p.d.history_stride + i];
            if (id < 0 || id >= p.d.vocab) bad = true;
            else if (id >= v0 && id < v0 + n) {
                if (i < prompt) atomicOr(&seen[id - v0], kGiven);
                else atomicAdd(&seen[id - v0], 1u);
            }
        }
        if (__syncthreads_or(bad)) {
            if (threadIdx.x == 0 && v0 == 0) fth::report_bad_entry(p.bad, r);
            return;
        }
        if (p.repetition) rep = p.repetition[r];
        if (p.frequency) freq = p.frequency[r];
        if (p.presence) pres = p.presence[r];
    }
    const float *x = p.logits + r * p.d.logits_stride + v0, *bias = p.bias ? p.bias + r * p.d.bias_stride + v0 : nullptr;
    const uint32_t *mask = p.mask ? p.mask + r * p.d.mask_stride + v0 / 32 : nullptr;
    float *y = p.out + r * p.d.out_stride + v0;
    for (int i = threadIdx.x; i < n; i += kBlock) {
        float z = x[i];
        if (p.history) {
            const uint32_t c = seen[i];
            if (c) {
                if (p.repetition) z = z > 0.f ? z / rep : z * rep;
                if (c & ~kGiven) {
                    if (p.frequency) z = z - freq * (float)(c & ~kGiven);
                    if (p.presence) z = z - pres;
                }
            }
        }
        if (bias) z = z + bias[i];
        if (mask && !((mask[i / 32] >> (i % 32)) & 1u)) z = -__builtin_inff();
        y[i] = z;
    }
}

}  // namespace

extern "C" int32_t fth_dev_logits_process_f32(const fth_logits_desc *d, const float *logits, const int32_t *history, const int32_t *history_len,
                                              const int32_t *prompt_len, const float *repetition, const float *frequency, const float *presence, const float *bias,
                                              const uint32_t *mask, float *out, int64_t *bad_index, fth_stream s) {
    FTH_ARG(d, "logits_process: NULL descriptor");
    FTH_ARG(d->rows >= 0 && d->vocab >= 0, "logits_process: negative extent");
    FTH_ARG(d->logits_stride >= d->vocab && d->out_stride >= d->vocab, "logits_process: a row stride is below the vocabulary");
    FTH_ARG(!history || d->history_stride >= 0, "logits_process: negative history_stride");
    FTH_ARG(!bias || d->bias_stride == 0 || d->bias_stride >= d->vocab, "logits_process: bias_stride is neither 0 nor a row");
    FTH_ARG(!mask || d->mask_stride >= fth::ceil_div(d->vocab, 32), "logits_process: mask_stride is below the words of a row");
    const int64_t most = (int64_t)1 << 40;
    for (int64_t x : {d->logits_stride, d->out_stride, history ? d->history_stride : 0, bias ? d->bias_stride : 0, mask ? d->mask_stride : 0})
        if (x > most || d->vocab > 2147483647LL || d->rows > ((int64_t)1 << 20)) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "logits_process: extents overflow");
    if (d->rows > 0 && d->vocab > 0) {
        FTH_ARG(logits && out, "logits_process: NULL operand");
        FTH_ARG(!history || (history_len && prompt_len), "logits_process: a history without its lengths");
        FTH_ARG(logits != out || d->logits_stride == d->out_stride, "logits_process: in place needs one stride");
    }
    FTH_REQUIRE_DEVICE();
    hipStream_t st = fth::resolve_stream(s);
    if (bad_index) {
        fth::reset_bad_kernel<<<1, 1, 0, st>>>(bad_index);
        FTH_CHECK_LAUNCH("logits_process(bad_index reset)");
    }
    if (d->rows == 0 || d->vocab == 0) return FTH_OK;
    LogitsArgs a;
    a.d = *d;
    a.logits = logits;
    a.history = repetition || frequency || presence ? history : nullptr;
    a.history_len = history_len; a.prompt_len = prompt_len;
    a.repetition = repetition; a.frequency = frequency; a.presence = presence;
    a.bias = bias; a.mask = mask; a.out = out; a.bad = bad_index;
    a.stretches = (int)fth::ceil_div(d->vocab, kStretch);
    FTH_ARG(d->rows * a.stretches <= 2147483647LL, "logits_process: too many rows for one launch");
    logits_process_kernel<<<dim3((unsigned)(d->rows * a.stretches)), dim3(kBlock), 0, st>>>(a);
    FTH_CHECK_LAUNCH("logits_process");
    return FTH_OK;
}
