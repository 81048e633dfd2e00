// Penalties for repeated tokens, a bias and a mask of allowed tokens on the logits of a generation step.
//
// A workgroup owns one row's logits over a stretch of the vocabulary. It counts the history's tokens that fall into its stretch
// in LDS (integer atomics: the counts do not depend on their order), then makes one pass over the logits. Each workgroup of a row
// scans the whole history, which comes from L2; in return nothing is handed from one launch to another. HBM-bound: every logit
// is read and written once, a row's own bias read once.
//   * A scan costs about eight instructions an id and is repeated by every stretch of the row: with 2048 steps of 4096 logits and
//     more, a stretch is two of them (200 rows of 131071, up to 8000 tokens before: 67 -> 60 us; four steps leave too few
//     workgroups: 64). The loads of a step go out before the one before it is finished, those of the first before the scan.
//   * What a thread loads and stores is 128 bits at 4-byte alignment, since rows of an odd vocabulary start anywhere (65 us where
//     131072 takes 61).
//   * A bias of the row's own is loaded past the caches, where it would push out logits (64.5 -> 60 us); one for all rows is not
//     (64 rows of 50257: 9.9 us, past the caches 11.5). Outputs over 8 MiB are stored past them (200 rows 72 -> 60 us; 64 rows
//     11.1 -> 9.5, and the argmax after it as fast as before in all: 27 us; 8 rows lose 1.2 of 22 us with the argmax).
//
// Measured: 200 rows of 131071, a bias each, a mask, up to 8000 tokens before 57 us (322 MB, 5.6 TB/s; one entry a thread and
// stretches of 4096: 143); 64 rows of 50257, one bias, a mask 7.7 us (27 MB; 17.3); one row 4.0 us.

#include <type_traits>

#include "paged.hpp"

namespace {

constexpr int kThreads = 512, kVecs = 2, kStep = kThreads * kVecs * 4, kMostSteps = 2;

struct LogitsArgs {
    fth_logits_desc d;
    const float *logits, *repetition, *frequency, *presence, *bias;
    const int32_t *history, *history_len, *prompt_len;
    const uint32_t *mask;
    float *out;
    int64_t *bad;
    int stretches, steps;  // stretches of a row, steps of a stretch
};

using F4u = float __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere
using I4u = int32_t __attribute__((ext_vector_type(4), aligned(4)));

constexpr uint32_t kGiven = 0x80000000u;  // bit 31: among the given tokens; below it: times generated

struct Step {  // one step's inputs of a thread
    F4u z[kVecs], b[kVecs];
    uint32_t bits[kVecs];
};

// NTB: a bias that no other row reads; NTS: more output than the caches hold.
template <bool NTB, bool NTS> __global__ __launch_bounds__(kThreads) void logits_process_kernel(const LogitsArgs p) {
    __shared__ __attribute__((aligned(16))) uint32_t seen[kMostSteps * kStep];
    const int64_t r = blockIdx.x / (unsigned)p.stretches;
    const int64_t v0 = (int64_t)(blockIdx.x % (unsigned)p.stretches) * (p.steps * kStep);
    const int n = (int)(p.d.vocab - v0 < p.steps * kStep ? p.d.vocab - v0 : p.steps * kStep);
    const float *x = p.logits + r * p.d.logits_stride + v0, *bias = p.bias ? p.bias + r * p.d.bias_stride + v0 : nullptr;
    const uint32_t *mask = p.mask ? p.mask + r * p.d.mask_stride + v0 / 32 : nullptr;
    auto place = [&](int step, int j) { return step * kStep + (j * kThreads + (int)threadIdx.x) * 4; };
    auto load4 = [&](const float *src, int i, auto nt) __attribute__((always_inline)) {
        F4u v = {0.f, 0.f, 0.f, 0.f};
        if (i + 4 <= n) v = nt ? __builtin_nontemporal_load(reinterpret_cast<const F4u *>(src + i)) : *reinterpret_cast<const F4u *>(src + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) v[e] = src[i + e];
        return v;
    };
    auto load = [&](int step) __attribute__((always_inline)) {
        Step s;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int i = place(step, j);
            s.z[j] = load4(x, i, std::false_type());
            if (bias) s.b[j] = load4(bias, i, std::bool_constant<NTB>());
            s.bits[j] = mask && i < n ? mask[i / 32] >> (i % 32) : 15u;
        }
        return s;
    };

    Step now = load(0);
    float rep = 1.f, freq = 0.f, pres = 0.f;
    bool counted = false;
    if (p.history) {
        const int len = p.history_len[r], prompt = p.prompt_len[r];
        const int32_t *history = p.history + r * p.d.history_stride;
        const bool bad = len < 0 || len > p.d.history_stride || prompt < 0 || prompt > len;
        const int count = bad ? 0 : len;
        uint32_t largest = 0;  // as unsigned numbers, negative ids are beyond every vocabulary
        counted = count > 0;
        if (counted) {
            for (int i = (int)threadIdx.x * 4; i < n; i += kThreads * 4) *reinterpret_cast<uint4 *>(&seen[i]) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            auto note = [&](int32_t id, int i) __attribute__((always_inline)) {
                largest = (uint32_t)id > largest ? (uint32_t)id : largest;
                const uint32_t at = (uint32_t)id - (uint32_t)v0;
                if (at < (uint32_t)n) {
                    if (i < prompt) atomicOr(&seen[at], kGiven);
                    else atomicAdd(&seen[at], 1u);
                }
            };
            // (unsigned: the step past the end of 2^31 - 1 tokens is a number too)
            for (uint32_t i = threadIdx.x * 4; i < (uint32_t)count; i += kThreads * 4) {
                if (i + 4 <= (uint32_t)count) {
                    const I4u ids = *reinterpret_cast<const I4u *>(history + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) note(ids[e], (int)i + e);
                } else {
                    for (int e = (int)i; e < count; ++e) note(history[e], e);
                }
            }
        }
        if (p.repetition) rep = p.repetition[r];
        if (p.frequency) freq = p.frequency[r];
        if (p.presence) pres = p.presence[r];
        if (__syncthreads_or(bad || (counted && largest >= (uint32_t)p.d.vocab))) {
            if (threadIdx.x == 0 && v0 == 0) fth::report_bad_entry(p.bad, r);
            return;
        }
    }
    float *y = p.out + r * p.d.out_stride + v0;
    auto finish = [&](float t, uint32_t c, float b, bool allowed) __attribute__((always_inline)) {
        if (c) {
            if (p.repetition) t = t > 0.f ? t / rep : t * rep;
            if (c & ~kGiven) {
                if (p.frequency) t = t - freq * (float)(c & ~kGiven);
                if (p.presence) t = t - pres;
            }
        }
        if (bias) t = t + b;
        return allowed ? t : -__builtin_inff();
    };
    for (int step = 0; step < p.steps && step * kStep < n; ++step) {
        Step next;
        if (step + 1 < p.steps) next = load(step + 1);
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int i = place(step, j);
            if (i >= n) break;
            const uint4 counts = counted ? *reinterpret_cast<const uint4 *>(&seen[i]) : make_uint4(0, 0, 0, 0);
            const uint32_t c[4] = {counts.x, counts.y, counts.z, counts.w};
            F4u t;
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = finish(now.z[j][e], c[e], now.b[j][e], (now.bits[j] >> e) & 1u);
            if (i + 4 <= n) {
                if constexpr (NTS) __builtin_nontemporal_store(t, reinterpret_cast<F4u *>(y + i));
                else *reinterpret_cast<F4u *>(y + i) = t;
            } else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < n) y[i + e] = t[e];
        }
        now = next;
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
    a.repetition = a.history ? repetition : nullptr; a.frequency = a.history ? frequency : nullptr; a.presence = a.history ? presence : nullptr;
    a.bias = bias; a.mask = mask; a.out = out; a.bad = bad_index;
    const int64_t steps = fth::ceil_div(d->vocab, kStep);
    a.steps = a.history && d->rows * steps >= 2048 ? kMostSteps : 1;
    a.stretches = (int)fth::ceil_div(steps, a.steps);
    FTH_ARG(d->rows * a.stretches <= 2147483647LL, "logits_process: too many rows for one launch");
    const bool ntb = bias && d->bias_stride != 0, nts = d->rows * d->vocab > (2 << 20);
    auto go = [&](auto kernel) { kernel<<<dim3((unsigned)(d->rows * a.stretches)), dim3(kThreads), 0, st>>>(a); };
    if (ntb) go(nts ? logits_process_kernel<true, true> : logits_process_kernel<true, false>);
    else go(nts ? logits_process_kernel<false, true> : logits_process_kernel<false, false>);
    FTH_CHECK_LAUNCH("logits_process");
    return FTH_OK;
}
