// The next token of each row of logits from a given number: temperature, top-k, top-p, min-p.
//
// Tokens are ordered by a code of 64 bits, the complement of the logit's ordered bits above the index: smaller codes come first. Every
// filter keeps a prefix of that order, so the kept tokens are those up to a last code (and above min-p). Weights are fp64 exponentials (which side of a
// border a sum lies on decides the token); where sums of them are collected by atomics they are whole numbers W = round(2^S w), S = 45 up to 2^17 tokens,
// whose sums are exact and do not depend on the order: a weight under 2^-46 of the largest counts as none there. That
// is so where the border of top-p is looked for; the token is drawn with the fp64 weights, summed in a fixed order. Two launches:
//   * pieces: one wavefront for 2048 logits, which it holds. It finds their maximum; where all of the row count (no top-k) the sum of their
//     weights relative to that maximum; and where there is a filter it writes down the largest of them, in the order of the vocabulary: at least
//     `want`, by a bisection of the lanes' maxima, which costs a comparison of one register a step.
//   * choice: one workgroup for a row. Without a filter the sums of the pieces give the piece, and its logits the token. With one, the
//     candidates of all pieces are gathered in LDS, and a histogram over max - x and the ranks inside one of its bins find the last code. It holds if no piece
//     has left out what could lie before it; otherwise the same is done over the whole row.
//
// Bound by latency, then by reading: 200 rows of 131071, top-k 1000 and top-p 0.98, 38.8 us = 23.6 for the pieces (4.4 TB/s; reading and the maxima
// alone 19.8) + 15.7 for the choice (eight passes of a radix selection a row, the simplest form, took 1171). Without filters 40 us, as each logit needs an fp64
// exponential (31 + 8.3). 64 rows of 50257 17.4 (9.4 + 8.7: 4.4 for reading, 3 for exponentials, 2.4 for the candidates), 16 10.6, 1 13.3. Slower were: pieces of 1024 logits (twice the
// candidates), wavefronts that take several pieces with the next one's loads ahead and bounds of 72 or 64 registers, the last three by spills (87, 80 and
// 90 us for the pieces); candidates straight to memory, a branch each (25.9); one thread to rank each member of a bin (the choice 17.1). Level: eight wavefronts a SIMD instead of six. The choice by 512 threads 20.9, 256 32.3 us.
// Rows that the candidates do not decide (a nucleus of tens of thousands, top-k 20000) are read again by one workgroup: once for the bins, once for each
// border (top-k, top-p) or eight times where the border's bin has more than kList members, once for the draw, each time with an fp64 exponential a logit
// and atomics in LDS. 131071 normal logits 156 to 193 us, 50257 90 to 108, 200 rows of 131071 192 to 237; 131071 equal logits 1730 us with one border, 3180
// with two, 50257 730 and 1330 (of two values half of that). Vocabularies above kPlaces pieces, 2^20 tokens, are always read so.

#include <type_traits>

#include "devmath.hpp"
#include "paged.hpp"

namespace {

constexpr int kPiece = 2048, kEntries = 128, kWaves = 4;         // logits of a piece, candidates that it may write down, pieces of a workgroup
constexpr int kThreads = 1024, kBins = 2048, kList = 7168, kRanked = 256;   // the choice: bins, candidates in LDS, members of a bin that are ranked
constexpr int kAtOnce = 8;  // logits that a thread asks for at once in passes over the row (4 / 8 / 16: 501 / 475 / 473 us before members went digit by digit)
constexpr int kPlaces = 512, kAhead = 4, kGroups = kPiece / kThreads, kMyBins = kBins / kThreads;                            // pieces of a row whose candidates are listed; of a wavefront, fetched at once

struct Piece {
    float max, limit;  // of what is not written down, every logit is below `limit` (-inf: all is written down)
    uint32_t count, bad;
    double sum;        // of exp((x - max) / temperature), where the row asks for it
};
struct Entry {
    float x;
    uint32_t v;
};

struct SampleArgs {
    fth_sample_desc d;
    const float *logits, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    const double *uniform;
    int32_t *tokens;
    float *logprobs;
    int64_t *bad;
    Piece *pieces;
    Entry *entries;
    int per_row;  // pieces of a row
    int want_p;   // lanes of a piece that write something down for top-p and min-p
    double magic; // 1.5 * 2^(52 - S): added to a weight in [0, 1], leaves round(2^S weight) in the low bits
    double unit;  // 2^S
    fth::Divisor by_pieces;  // by per_row
};

constexpr int kVecs = kPiece / 256;
using F4u = float __attribute__((ext_vector_type(4), aligned(4)));  // rows start anywhere

// A row's settings as they are used.
struct Settings {
    double rate;  // log2(e) / temperature
    float top_p, min_p;
    int top_k;    // 0: all
    bool bad;
    __device__ __forceinline__ Settings(const SampleArgs &p, int64_t r) {
        const float t = p.temperature ? p.temperature[r] : 1.f;
        top_p = p.top_p ? p.top_p[r] : 1.f;
        min_p = p.min_p ? p.min_p[r] : 0.f;
        top_k = p.top_k ? p.top_k[r] : 0;
        bad = !(t >= 0.f && t < __builtin_inff()) || !(top_p >= 0.f) || !(min_p >= 0.f && min_p <= 1.f) || top_k < 0;
        if (t == 0.f) top_k = 1;
        if (top_k >= p.d.vocab) top_k = 0;
        rate = 1.4426950408889634074 / (t == 0.f ? 1.0 : (double)t);
    }
    __device__ __forceinline__ bool filters() const { return top_k > 0 || top_p < 1.f || min_p > 0.f; }
};

// 32 bits in the order of floats, largest first; -0 is 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return (b & 0x80000000u) ? b : b ^ 0x7fffffffu;
}
__device__ __forceinline__ uint64_t code_of(float x, uint32_t v) { return (uint64_t)order_of(x) << 32 | v; }

// Across a wavefront by data-parallel moves (a shuffle through LDS costs five times as much): a lane without a source gets `old`.
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T moved(T old, T x) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
    } else {
        const uint64_t o = __builtin_bit_cast(uint64_t, old), v = __builtin_bit_cast(uint64_t, x);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)o, (int)v, CTRL, ROWS, 0xf, false);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(o >> 32), (int)(v >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    }
}
template <typename T> __device__ __forceinline__ T lane_value(T x, int lane) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
    } else {
        const uint64_t v = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
    }
}
// op over the lanes up to each one: within rows of 16, then the last of a row into the next, then of the first half into the second. NEUTRAL is
// its neutral element.
template <typename T, typename F> __device__ __forceinline__ T wave_scan(T x, T neutral, F op) {
    x = op(moved<0x111, 0xf>(neutral, x), x);
    x = op(moved<0x112, 0xf>(neutral, x), x);
    x = op(moved<0x114, 0xf>(neutral, x), x);
    x = op(moved<0x118, 0xf>(neutral, x), x);
    x = op(moved<0x142, 0xa>(neutral, x), x);
    return op(moved<0x143, 0xc>(neutral, x), x);
}
struct MaxOp { template <typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; } };
struct AddOp { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };
// The sum over 4 or 16 neighbouring lanes, in each of them: pairs and pairs of pairs of a quad, then mirror images.
template <int N, typename T> __device__ __forceinline__ T neighbours_sum(T x) {
    static_assert(N == 4 || N == 16, "a quad or a row");
    x += moved<0xb1, 0xf>(x, x);
    x += moved<0x4e, 0xf>(x, x);
    if constexpr (N == 16) {
        x += moved<0x141, 0xf>(x, x);
        x += moved<0x140, 0xf>(x, x);
    }
    return x;
}
template <typename T> __device__ __forceinline__ T wave_sum(T x) { return lane_value(wave_scan(x, (T)0, AddOp()), 63); }
__device__ __forceinline__ float wave_max(float x) { return lane_value(wave_scan(x, -__builtin_inff(), MaxOp()), 63); }

// ---- pieces -----------------------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(64 * kWaves) void sample_pieces_kernel(const SampleArgs p) {
    __shared__ Entry found[kWaves][kEntries + 64];  // of each wavefront, and a place for each lane that has none to write
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int piece32 = (int)blockIdx.x * kWaves + wave, row32 = (int)p.by_pieces((uint32_t)piece32);
    const int64_t piece = piece32, r = row32;
    if (r >= p.d.rows) return;
    const int64_t v0 = (int64_t)(piece32 - row32 * p.per_row) * kPiece;
    const int n = (int)(p.d.vocab - v0 < kPiece ? p.d.vocab - v0 : kPiece);
    const float *x = p.logits + r * p.d.logits_stride + v0;
    F4u z[kVecs];  // logit 256 s + 4 lane + e of the piece
    if (n == kPiece) {
#pragma unroll
        for (int s = 0; s < kVecs; ++s) z[s] = *reinterpret_cast<const F4u *>(x + 256 * s + 4 * lane);
    } else {
#pragma unroll
        for (int s = 0; s < kVecs; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[s][e] = 256 * s + 4 * lane + e < n ? x[256 * s + 4 * lane + e] : -__builtin_inff();
    }
    const Settings set(p, r);
    float mine = -__builtin_inff();
    int up = 0;          // +inf and positive NaN are the largest numbers as signed integers,
    uint32_t down = 0u;  // negative NaN as unsigned ones
#pragma unroll
    for (int s = 0; s < kVecs; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t bits = __float_as_uint(z[s][e]);
            mine = fmaxf(mine, z[s][e]);
            up = (int)bits > up ? (int)bits : up;
            down = bits > down ? bits : down;
        }
    const bool bad = __any(up >= 0x7f800000 || down > 0xff800000u);
    Piece out = {wave_max(mine), -__builtin_inff(), 0u, bad ? 1u : 0u, 0.0};
    if (!bad && !set.bad && out.max > -__builtin_inff()) {
        if (set.top_k == 0) {
            double sum = 0.0;
#pragma unroll
            for (int s = 0; s < kVecs; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum += fth::exp2_softmax(((double)z[s][e] - (double)out.max) * set.rate);
                    if (e & 1) __builtin_amdgcn_sched_barrier(0);  // two at a time, for the registers' sake
                }
            out.sum = wave_sum(sum);
        }
        if (set.filters()) {
            // How many lanes shall write something down (tokens of a vocabulary in order of frequency have their largest logits side by side: 36 at
            // least, though spread evenly 16 would do; us for 200 x 131071, top-k 50, 16 / 36 / 52 of them: the choice 12.8 / 12.8 / 14.8),
            // and what cannot be kept, as far as the piece by itself can tell (no more than a hint: `limit` says what was left out).
            int want = p.want_p;
            float hint = -3.402823466e38f;
            if (set.top_k > 0) {
                const int share = 2 * (int)p.by_pieces((uint32_t)((set.top_k < 1 << 30 ? set.top_k : 1 << 30) + p.per_row - 1)) + 14;
                want = share < 36 ? 36 : share < 52 ? share : 52;
                want = want < set.top_k ? want : set.top_k;
            } else {
                const float part = set.top_p < 1.f ? (1.f - set.top_p) * (float)out.sum * (1.f / kPiece) : 0.f, far = fmaxf(part, set.min_p * 0.999f);
                if (far > 0.f) hint = fmaxf(hint, out.max + __builtin_amdgcn_logf(far) / (float)set.rate);
            }
            const uint32_t key = order_of(mine);
            // Written down is what reaches `least`: all that the hint leaves, if few lanes have any of it; else what reaches the number of 16 bits that
            // `want` lanes reach, or fewer lanes where that would be too much.
            float least = hint;
            if (least > -3.402823466e38f) out.limit = least;
            int tries = 0;
            bool first = __popcll(__ballot(mine >= least)) > want;
            for (;;) {
                if (!first) {
                    uint32_t at = 0, v = (uint32_t)v0 + 4 * lane;
                    asm volatile("" : "+v"(v));  // (32 token numbers need not stay in registers from here on)
#pragma unroll
                    for (int s = 0; s < kVecs; ++s) {
                        uint32_t before = at;
                        uint64_t in[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            in[e] = __ballot(z[s][e] >= least);
                            before = __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], before));
                            at += __popcll(in[e]);
                        }
                        if (at > kEntries) continue;  // too many: once more with fewer
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool mine = z[s][e] >= least;
                            Entry &to = found[wave][mine ? before : kEntries + lane];
                            to.x = z[s][e];
                            to.v = v + 256 * s + e;
                            before += mine;
                        }
                        __builtin_amdgcn_sched_barrier(0);  // for the registers' sake
                    }
                    if (at <= kEntries) {
                        out.count = at;
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                        for (int h = 0; h < kEntries / 64; ++h)
                            if (64 * h + lane < (int)at) p.entries[piece * kEntries + 64 * h + lane] = found[wave][64 * h + lane];
                        break;
                    }
                    if (want == 0) {
                        out.limit = __builtin_inff();
                        break;
                    }
                }
                first = false;
                uint32_t c = 0;  // the smallest for which `want` lanes have key < (c + 1) << 16
#pragma unroll
                for (int b = 15; b >= 0; --b) {
                    const uint32_t c1 = c | (1u << b);
                    if (__popcll(__ballot(key < c1 << 16)) < want) c = c1;
                }
                const uint32_t end = c << 16 | 0xffffu;  // the order of `least`
                const float reached = __uint_as_float((end & 0x80000000u) ? end : end ^ 0x7fffffffu);
                if (reached > least) least = out.limit = reached;  // (else fewer lanes than that have anything)
                want = tries++ < 3 ? want - want / 8 : want >> 1;  // (the first time it goes down after too many; ties would go down far)
            }
        }
    }
    if (lane == 0) p.pieces[piece] = out;
}

// ---- the choice ---------------------------------------------------------------------------------------------------------------

struct Member {
    uint64_t code, weight;
};
struct Found {  // what the threads of a boundary() tell each other
    uint64_t code, weight;
    uint32_t members;
    int at;
};
struct Shared {
    uint64_t weight[kBins];  // of the bins
    uint32_t count[kBins];
    Entry list[kList];       // the candidates, in the order of the vocabulary
    double weigh[kList];     // their weights
    Member few[kRanked];     // the members of a bin, or bins of digits, or the sums of ranges
    uint64_t sums[2][32];
    Found finds[2];
    uint32_t places[kPlaces + 1];  // where the candidates of each piece stand in the list
};

// op over the lanes of a row of 16 up to each one.
template <typename T, typename F> __device__ __forceinline__ T row_scan(T x, T neutral, F op) {
    x = op(moved<0x111, 0xf>(neutral, x), x);
    x = op(moved<0x112, 0xf>(neutral, x), x);
    x = op(moved<0x114, 0xf>(neutral, x), x);
    return op(moved<0x118, 0xf>(neutral, x), x);
}
// The sum over the threads before this one, and over all. One barrier before `lds` is written, one after.
template <typename T> struct BlockScan {
    static constexpr int W = kThreads / 64;
    static_assert(W == 16, "the wavefronts' sums are a row of lanes");
    T x, upto, *lds;
    int wave;
    __device__ __forceinline__ BlockScan(T x, T *lds) : x(x), upto(wave_scan(x, (T)0, AddOp())), lds(lds), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {}
    __device__ __forceinline__ void write() const {
        if ((threadIdx.x & 63) == 63) lds[wave] = upto;
    }
    __device__ __forceinline__ T read(T *all) const {
        const T t = row_scan(lds[threadIdx.x & (W - 1)], (T)0, AddOp());
        *all = lane_value(t, W - 1);
        return upto - x + (wave ? lane_value(t, wave ? wave - 1 : 0) : (T)0);
    }
    __device__ __forceinline__ T read_upto(T *all) const {  // with this thread's
        const T t = row_scan(lds[threadIdx.x & (W - 1)], (T)0, AddOp());
        *all = lane_value(t, W - 1);
        return upto + (wave ? lane_value(t, wave ? wave - 1 : 0) : (T)0);
    }
};
template <typename T> __device__ __forceinline__ T block_scan(T x, T *lds, T *all) {
    const BlockScan<T> scan(x, lds);
    __syncthreads();
    scan.write();
    __syncthreads();
    return scan.read(all);
}

struct Row {
    const SampleArgs &p;
    const Settings &set;
    Shared &s;
    const float *x;
    float big;
    double u;
    int64_t r;

    __device__ __forceinline__ double weight_of(float z) const { return fth::exp2_softmax(((double)z - (double)big) * set.rate); }
    __device__ __forceinline__ uint64_t whole(double w) const {
        return (uint64_t)__builtin_bit_cast(int64_t, w + p.magic) - (uint64_t)__builtin_bit_cast(int64_t, p.magic);
    }
    // Distances from the maximum in steps of 1/64 of their size, from 2^-16 to 2^16: they grow with the order.
    __device__ __forceinline__ int bin_of(float z) const {
        const int b = (int)(__float_as_uint(big - z) >> 17) - ((127 - 16) << 6);
        return b < 0 ? 0 : b >= kBins ? kBins - 1 : b;
    }
    // f(logit, token, weight) of every candidate (of the row: of every token that is allowed), by this workgroup's threads.
    template <bool LIST, typename F> __device__ __forceinline__ void each(int n, F f) const {
        if constexpr (LIST) {
            for (int i = threadIdx.x; i < n; i += kThreads) f(s.list[i].x, s.list[i].v, s.weigh[i]);
        } else {
            for (int i = threadIdx.x; i < n; i += kAtOnce * kThreads) {
                float z[kAtOnce];
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e) z[e] = i + e * kThreads < n ? x[i + e * kThreads] : -__builtin_inff();
#pragma unroll
                for (int e = 0; e < kAtOnce; ++e)
                    if (z[e] > -__builtin_inff()) f(z[e], (uint32_t)(i + e * kThreads), weight_of(z[e]));
            }
        }
    }
    __device__ __forceinline__ void write(int token, double share) const {
        p.tokens[r] = token;
        if (p.logprobs) p.logprobs[r] = (float)log(share);
    }
    __device__ __forceinline__ void clear_bins() const {
        if (threadIdx.x < 2) s.finds[threadIdx.x] = Found{0, 0, 0, -1};
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            s.weight[b] = 0;
            s.count[b] = 0;
        }
    }
    __device__ __forceinline__ void to_bin(float z, double weight) const {
        const int b = bin_of(z);
        const uint64_t w = whole(weight);
        atomicAdd(&s.count[b], 1u);
        if (w) atomicAdd(reinterpret_cast<unsigned long long *>(&s.weight[b]), (unsigned long long)w);
    }

    // What comes before a thread's first bin.
    struct Prefix {
        uint32_t count;
        uint64_t weight;
    };
    __device__ __forceinline__ Prefix scan_bins(bool counts, bool weights, uint64_t *all) const {
        Prefix at = {0, 0};
#pragma unroll
        for (int b = 0; b < kMyBins; ++b) {
            at.count += s.count[kMyBins * threadIdx.x + b];
            at.weight += s.weight[kMyBins * threadIdx.x + b];
        }
        uint32_t unused;
        if (counts && weights) {  // between the same barriers
            const BlockScan<uint32_t> count(at.count, reinterpret_cast<uint32_t *>(s.sums[1]));
            const BlockScan<uint64_t> weight(at.weight, s.sums[0]);
            __syncthreads();
            count.write();
            weight.write();
            __syncthreads();
            return Prefix{count.read(&unused), weight.read(all)};
        }
        if (counts) at.count = block_scan(at.count, reinterpret_cast<uint32_t *>(s.sums[1]), &unused);
        if (weights) at.weight = block_scan(at.weight, s.sums[0], all);
        return at;
    }

    // The smallest code for which the tokens up to it are `k` at least (k > 0) or weigh `need`, by the bins: the bin, then the ranks of its
    // members; where it has too many (ties, wide nuclei) digit by digit. All ones if there is none. *weight: what they weigh. `call`: 0, then 1.
    template <bool LIST> __device__ __forceinline__ uint64_t boundary(int n, const Prefix &at, uint32_t k, uint64_t need, int call, uint64_t *weight) const {
        const int t = threadIdx.x;
        Found &f = s.finds[call];
        const uint64_t goal = k ? k : need;
        uint64_t before = k ? (uint64_t)at.count : at.weight, weighed = at.weight;
        if (before < goal)
#pragma unroll
            for (int b = 0; b < kMyBins; ++b) {
                const uint64_t w = s.weight[kMyBins * t + b], here = k ? (uint64_t)s.count[kMyBins * t + b] : w;
                if (before < goal && before + here >= goal) {
                    f.at = kMyBins * t + b;
                    f.code = weighed;
                    f.weight = before;
                }
                before += here;
                weighed += w;
            }
        __syncthreads();
        const int bin = f.at;
        if (bin < 0) return ~0ull;
        uint64_t weighs = f.code, had = f.weight;
        const uint32_t members = s.count[bin];
        if (members <= kRanked) {
            each<LIST>(n, [&](float z, uint32_t v, double w) {
                if (bin_of(z) == bin) s.few[atomicAdd(&f.members, 1u)] = Member{code_of(z, v), whole(w)};
            });
            __syncthreads();
            // ranks, in whatever order the members stand: PARTS neighbouring threads for one
            auto rank = [&](auto parts) {
                constexpr int PARTS = decltype(parts)::value;
                const int m = t / PARTS;
                if (m >= (int)members) return;
                const Member mine = s.few[m];
                uint32_t count = 0;
                uint64_t sum = 0;
#pragma unroll 4
                for (uint32_t i = t % PARTS; i < members; i += PARTS) {
                    const Member other = s.few[i];
                    const bool before = other.code < mine.code;
                    count += before;
                    sum += before ? other.weight : 0;
                }
                if constexpr (PARTS > 1) {
                    count = neighbours_sum<PARTS>(count);
                    sum = neighbours_sum<PARTS>(sum);
                }
                const uint64_t upto = had + (k ? count : sum), here = k ? 1 : mine.weight;
                if (t % PARTS == 0 && upto < goal && upto + here >= goal) {
                    f.code = mine.code;
                    f.weight = weighs + sum + mine.weight;
                }
            };
            if (members <= 16) rank(std::integral_constant<int, 1>());
            else if (members <= kThreads / 16) rank(std::integral_constant<int, 16>());
            else rank(std::integral_constant<int, kThreads / kRanked>());
            __syncthreads();
            *weight = f.weight;
            return f.code;
        }
        // Digit by digit (the bins of digits stand where the members would); of the row the members alone, if the list has room for them.
        if constexpr (!LIST) {
            if (members <= kList) {
                each<false>(n, [&](float z, uint32_t v, double w) {
                    if (bin_of(z) != bin) return;
                    const uint32_t at_member = atomicAdd(&f.members, 1u);
                    s.list[at_member] = Entry{z, v};
                    s.weigh[at_member] = w;
                });
                return digits<true>((int)members, bin, k != 0, goal, had, weighs, f, weight);
            }
        }
        return digits<LIST>(n, bin, k != 0, goal, had, weighs, f, weight);
    }
    // Among the candidates in `bin`, before which there are `had` (tokens, or their weights) and the weights `weighs`.
    template <bool LIST> __device__ __forceinline__ uint64_t digits(int n, int bin, bool counts, uint64_t goal, uint64_t had, uint64_t weighs, Found &f, uint64_t *weight) const {
        static_assert(kRanked >= 192, "256 weights and 256 counts");
        uint64_t *digit_weight = &s.few[0].code;
        uint32_t *digit_count = reinterpret_cast<uint32_t *>(&s.few[128]);
        uint64_t prefix = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int d = threadIdx.x; d < 256; d += kThreads) {
                digit_weight[d] = 0;
                digit_count[d] = 0;
            }
            __syncthreads();
            each<LIST>(n, [&](float z, uint32_t v, double w) {
                const uint64_t c = code_of(z, v);
                if (bin_of(z) != bin || (shift < 56 && c >> (shift + 8) != prefix)) return;
                const int at_digit = (int)(c >> shift) & 255;
                atomicAdd(&digit_count[at_digit], 1u);
                atomicAdd(reinterpret_cast<unsigned long long *>(&digit_weight[at_digit]), (unsigned long long)whole(w));
            });
            __syncthreads();
            if (threadIdx.x < 64) {  // four digits a lane
                const int lane = threadIdx.x;
                uint64_t here[4], heavy[4], all = 0, all_heavy = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    heavy[e] = digit_weight[4 * lane + e];
                    here[e] = counts ? digit_count[4 * lane + e] : heavy[e];
                    all += here[e];
                    all_heavy += heavy[e];
                }
                const uint64_t upto = wave_scan(all, (uint64_t)0, AddOp()), upto_heavy = wave_scan(all_heavy, (uint64_t)0, AddOp());
                const uint64_t over = __ballot(had + upto >= goal);
                if (lane == (over ? __builtin_ctzll(over) : 63)) {
                    uint64_t before = had + upto - all, before_heavy = weighs + upto_heavy - all_heavy;
                    bool found = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (found) continue;
                        if (before + here[e] >= goal || e == 3) {
                            f.code = prefix << 8 | (uint32_t)(4 * lane + e);
                            f.weight = before;
                            s.sums[0][0] = before_heavy + heavy[e];
                            s.sums[0][1] = before_heavy;
                            found = true;
                        }
                        before += here[e];
                        before_heavy += heavy[e];
                    }
                }
            }
            __syncthreads();
            prefix = f.code;
            had = f.weight;
            *weight = s.sums[0][0];
            weighs = s.sums[0][1];
        }
        return prefix;
    }

    // The last code that the filters keep; 0: the candidates do not say. `limit`: what is not among them is below it. `sum`: of all
    // weights. The bins hold all candidates.
    template <bool LIST> __device__ __forceinline__ uint64_t filter(int n, double sum, float limit) const {
        const bool whole_row = !LIST || limit == -__builtin_inff();
        // whether nothing that was left out could stand before a code
        auto sure = [&](uint64_t code) { return whole_row || (code != ~0ull && (uint32_t)(code >> 32) <= order_of(limit)); };
        // whether min-p leaves out what was left out, and so all that other filters are not sure of
        const bool below = !whole_row && set.min_p > 0.f && fth::exp2_softmax(((double)limit - (double)big) * set.rate) < (double)set.min_p;
        uint64_t last = ~0ull, weight = 0, all = 0;
        if (set.top_k == 0 && !(set.top_p < 1.f)) return whole_row || below ? last : 0;
        const Prefix at = scan_bins(set.top_k > 0, set.top_p < 1.f, &all);
        if (set.top_k > 0) {
            last = boundary<LIST>(n, at, (uint32_t)set.top_k, 0, 0, &weight);
            if (!sure(last) && (set.top_p < 1.f || !below)) return 0;
            sum = (double)(last == ~0ull ? all : weight);  // (fewer tokens are allowed)
        }
        if (set.top_p < 1.f) {
            const double need = __builtin_ceil(sum * (double)set.top_p);
            const uint64_t code = boundary<LIST>(n, at, 0, need < 1.0 ? 1 : (uint64_t)need, 1, &weight);
            if (code < last) last = code;  // (none: rounded weights fall short of it, or the candidates do)
            if (!sure(last) && (set.top_k > 0 || !below)) return 0;
        }
        return last;
    }

    // Which thread's `mine` the number leads to: the first whose sums reach over it, or where rounding at the very end leaves none, the last that has
    // anything. (Sums in floating point need not ascend from thread to thread: their comparison alone could name two threads or none.)
    struct Drawn {
        int who;
        double left, total;  // of the number, once what is before the thread is gone (in that thread alone); of all threads
    };
    __device__ __forceinline__ Drawn draw(double mine) const {
        const BlockScan<double> scan(mine, reinterpret_cast<double *>(s.sums[0]));
        __syncthreads();
        scan.write();
        if (threadIdx.x == 0) {
            s.finds[0].at = kThreads;
            s.finds[1].at = -1;
        }
        __syncthreads();
        Drawn d;
        const double upto = scan.read_upto(&d.total), target = d.total * u;
        const uint64_t over = __ballot(mine > 0.0 && upto > target), some = __ballot(mine > 0.0);
        const int first = threadIdx.x & ~63;
        if (threadIdx.x == first) {
            if (over) atomicMin(&s.finds[0].at, first + __builtin_ctzll(over));
            if (some) atomicMax(&s.finds[1].at, first + 63 - __builtin_clzll(some));
        }
        __syncthreads();
        d.who = s.finds[0].at;
        d.left = target - (upto - mine);
        if (d.who == kThreads) {
            d.who = s.finds[1].at;
            d.left = 1e300;
        }
        return d;
    }

    // The token among the candidates up to `last` and above min-p.
    __device__ __forceinline__ void draw_list(int n, uint64_t last) const {
        const int t = threadIdx.x, each_has = (n + kThreads - 1) / kThreads, from = t * each_has, to = from + each_has < n ? from + each_has : n;
        auto kept = [&](int i) {
            const double w = s.weigh[i];
            return code_of(s.list[i].x, s.list[i].v) > last || w < (double)set.min_p ? 0.0 : w;
        };
        double mine = 0.0;
        for (int i = from; i < to; ++i) mine += kept(i);
        const Drawn d = draw(mine);
        if (t != d.who) return;
        double left = d.left, share = 0.0;
        int token = 0;
        for (int i = from; i < to; ++i) {
            const double w = kept(i);
            if (!(w > 0.0)) continue;
            token = (int)s.list[i].v;
            share = w;
            if (w > left) break;
            left -= w;
        }
        write(token, share / d.total);
    }

    // The same from the whole row: cut into 256 ranges, whose sums give the range; a wavefront finds the token in it.
    __device__ __forceinline__ void draw_row(int n, uint64_t last) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, length = ((n + 255) / 256 + 63) & ~63;
        double *ranges = reinterpret_cast<double *>(s.few);
        auto logit = [&](int64_t i) { return i < n ? x[i] : -__builtin_inff(); };
        auto kept = [&](int64_t i, float z) {
            if (!(z > -__builtin_inff()) || code_of(z, (uint32_t)i) > last) return 0.0;
            const double w = weight_of(z);
            return w < (double)set.min_p ? 0.0 : w;
        };
        __syncthreads();
        for (int g = wave; g < 256; g += kThreads / 64) {
            double sum = 0.0;
            const int64_t end = (g + 1) * (int64_t)length;
            if (end - length < n)
                for (int64_t i = end - length + lane; i < end; i += kAtOnce * 64) {
                    float z[kAtOnce];
#pragma unroll
                    for (int e = 0; e < kAtOnce; ++e) z[e] = i + 64 * e < end ? logit(i + 64 * e) : -__builtin_inff();
#pragma unroll
                    for (int e = 0; e < kAtOnce; ++e) sum += kept(i + 64 * e, z[e]);
                }
            sum = wave_sum(sum);
            if (lane == 0) ranges[g] = sum;
        }
        __syncthreads();
        static_assert(kThreads >= 256, "a thread for each range");
        const Drawn d = draw(threadIdx.x < 256 ? ranges[threadIdx.x] : 0.0);
        if ((int)threadIdx.x == d.who) s.finds[0].code = __builtin_bit_cast(uint64_t, d.left);
        __syncthreads();
        if (wave != 0) return;
        double left = __builtin_bit_cast(double, s.finds[0].code), share = 0.0;
        int token = 0;
        for (int i0 = 0; i0 < length; i0 += 64) {
            const int64_t i = (int64_t)d.who * length + i0 + lane;
            const double here = kept(i, logit(i)), upto = wave_scan(here, 0.0, AddOp());
            const uint64_t over = __ballot(here > 0.0 && upto > left), some = __ballot(here > 0.0);
            if (!some) continue;
            const int which = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
            token = (int)((int64_t)d.who * length + i0 + which);
            share = lane_value(here, which);
            if (over) break;
            left -= lane_value(upto, 63);
        }
        if (lane == 0) write(token, share / d.total);
    }

    // Without a filter: the token that `left` of the weight before it leads to, in piece `at`. Where rounding leads past the piece's end, its
    // last. The piece has weight: its largest token is above 2^-1000 of the row's. Each wavefront has two groups of 64 neighbouring tokens.
    __device__ __forceinline__ void draw_piece(int at, double left, double total) const {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int64_t v0 = (int64_t)at * kPiece + kGroups * 64 * wave;
        double *sums = reinterpret_cast<double *>(s.sums);
        double w[kGroups], upto[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const float z = v0 + 64 * g + lane < p.d.vocab ? x[v0 + 64 * g + lane] : -__builtin_inff();
            w[g] = z > -__builtin_inff() ? fth::exp2_softmax(((double)z - (double)big) * set.rate) : 0.0;
            upto[g] = wave_scan(w[g], 0.0, AddOp());
            if (lane == 63) sums[kGroups * wave + g] = upto[g];
        }
        __syncthreads();
        static_assert(kPiece == 64 * kGroups * (kThreads / 64) && kPiece / 64 <= 64, "a lane for each group");
        const double here = lane < kPiece / 64 ? sums[lane] : 0.0, through = wave_scan(here, 0.0, AddOp());
        const uint64_t over = __ballot(here > 0.0 && through > left), some = __ballot(here > 0.0);
        const int group = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
        if (group / kGroups != wave) return;
        left -= lane_value(through - here, group);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            if (g != group % kGroups) continue;
            const uint64_t past = __ballot(w[g] > 0.0 && upto[g] > left), any = __ballot(w[g] > 0.0);
            const int which = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
            if (lane == which) write((int)v0 + 64 * g + lane, w[g] / total);
        }
    }
};

__global__ __launch_bounds__(kThreads) void sample_choice_kernel(const SampleArgs p) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const Piece *pieces = p.pieces + r * p.per_row;
    // The candidates of the first pieces, before it is known how many there are.
    Entry ahead[kAhead][kEntries / 64];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = wave + j * (kThreads / 64);
#pragma unroll
        for (int h = 0; h < kEntries / 64; ++h) ahead[j][h] = p.entries[(r * p.per_row + (i < p.per_row ? i : 0)) * kEntries + 64 * h + lane];
    }
    const Settings set(p, r);
    const double u = p.uniform[r];
    // Every wavefront looks at all pieces, a lane at neighbouring ones, so that nothing has to be handed round.
    const int each = (p.per_row + 63) / 64, from = lane * each, to = from + each < p.per_row ? from + each : p.per_row;
    bool bad = set.bad || !(u >= 0.0 && u < 1.0);
    float big = -__builtin_inff(), limit = -__builtin_inff();
    uint32_t count = 0;
    for (int i = from; i < to; ++i) {
        const Piece one = pieces[i];
        bad |= one.bad != 0;
        big = fmaxf(big, one.max);
        limit = fmaxf(limit, one.limit);
        count += one.count;
    }
    big = wave_max(big) + 0.f;  // (0 - -0 is 0, -0 - 0 would be -0)
    if (__any(bad) || big == -__builtin_inff()) {
        if (t == 0) {
            p.tokens[r] = -1;
            if (p.logprobs) p.logprobs[r] = __builtin_nanf("");
            fth::report_bad_entry(p.bad, r);
        }
        return;
    }
    const Row row = {p, set, s, p.logits + r * p.d.logits_stride, big, u, r};
    auto sum_of = [&](int i) {  // (0 where the weights of its tokens could be)
        const double far = ((double)pieces[i].max - (double)big) * set.rate;
        return far > -1000.0 ? pieces[i].sum * fth::exp2_softmax(far) : 0.0;
    };
    double mine = 0.0, upto = 0.0, total = 0.0;
    if (set.top_k == 0) {
        for (int i = from; i < to; ++i) mine += sum_of(i);
        upto = wave_scan(mine, 0.0, AddOp());
        total = lane_value(upto, 63);
    }
    if (!set.filters()) {
        // the first lane over the number (none, by rounding at the very end: the last that has something)
        const double target = total * u;
        const uint64_t over = __ballot(mine > 0.0 && upto > target), some = __ballot(mine > 0.0);
        const int who = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
        int at = from, last = from;
        double left = target - (upto - mine);
        for (; at < to; ++at) {
            const double here = sum_of(at);  // (`left` may be just below 0 by the scan's rounding: a piece without weight is never it)
            if (here > 0.0) {
                if (here > left) break;
                last = at;
            }
            left -= here;
        }
        if (at == to) {
            at = last;
            left = 1e300;
        }
        row.draw_piece(lane_value(at, who), lane_value(left, who), total);
        return;
    }

    limit = wave_max(limit);
    const uint32_t upto_count = wave_scan(count, 0u, AddOp()), listed = lane_value(upto_count, 63);
    uint64_t last = 0;
    row.clear_bins();
    if (listed <= kList && p.per_row <= kPlaces) {
        if (wave == 0) {
            uint32_t place = upto_count - count;
            for (int i = from; i < to; ++i) {
                s.places[i] = place;
                place += pieces[i].count;
            }
            if (lane == 0) s.places[p.per_row] = listed;
        }
        __syncthreads();
        auto put = [&](int i, int h, Entry one) {
            const uint32_t place = s.places[i] + 64 * h;
            if (place + lane >= s.places[i + 1]) return;
            const double w = row.weight_of(one.x);
            s.list[place + lane] = one;
            s.weigh[place + lane] = w;
            row.to_bin(one.x, w);
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (wave + j * (kThreads / 64) < p.per_row)
#pragma unroll
                for (int h = 0; h < kEntries / 64; ++h) put(wave + j * (kThreads / 64), h, ahead[j][h]);
        for (int i = wave + kAhead * (kThreads / 64); i < p.per_row; i += kThreads / 64)
            for (int h = 0; h < kEntries / 64; ++h) put(i, h, p.entries[(r * p.per_row + i) * kEntries + 64 * h + lane]);
        __syncthreads();
        last = row.filter<true>((int)listed, total * p.unit, limit);
        if (last) {
            row.draw_list((int)listed, last);
            return;
        }
        __syncthreads();
        row.clear_bins();
    }
    __syncthreads();
    row.each<false>((int)p.d.vocab, [&](float z, uint32_t, double w) { row.to_bin(z, w); });
    __syncthreads();
    last = row.filter<false>((int)p.d.vocab, total * p.unit, limit);
    row.draw_row((int)p.d.vocab, last);
}

int64_t pieces_of(const fth_sample_desc &d) { return d.rows * fth::ceil_div(d.vocab, kPiece); }

int32_t check(const fth_sample_desc *d) {
    FTH_ARG(d, "sample: NULL descriptor");
    FTH_ARG(d->rows >= 0 && d->vocab >= 0, "sample: negative extent");
    FTH_ARG(d->logits_stride >= d->vocab, "sample: the row stride is below the vocabulary");
    if (d->logits_stride > ((int64_t)1 << 40) || d->vocab > ((int64_t)1 << 30) || d->rows > ((int64_t)1 << 20)) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "sample: extents overflow");
    FTH_ARG(d->rows == 0 || d->vocab > 0, "sample: no token to choose from");
    if (pieces_of(*d) > 2147483640LL) return fth::set_error(FTH_ERR_SIZE_OVERFLOW, "sample: more than 2^42 logits");
    return FTH_OK;
}

}  // namespace

extern "C" {

size_t fth_dev_sample_workspace_bytes(const fth_sample_desc *d) { return check(d) == FTH_OK ? (size_t)pieces_of(*d) * (sizeof(Piece) + kEntries * sizeof(Entry)) : 0; }

int32_t fth_dev_sample_f32(const fth_sample_desc *d, const float *logits, const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                           const double *uniform, int32_t *tokens, float *logprobs, int64_t *bad_index, void *workspace, size_t workspace_bytes, fth_stream s) {
    if (int32_t rc = check(d)) return rc;
    FTH_ARG(d->rows == 0 || (logits && uniform && tokens), "sample: NULL operand");
    const size_t need = fth_dev_sample_workspace_bytes(d);
    FTH_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15u) == 0), "sample: needs a workspace of %zu bytes, 16-byte aligned", need);
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
    const int64_t pieces = pieces_of(*d);
    a.pieces = static_cast<Piece *>(workspace);
    a.entries = reinterpret_cast<Entry *>(a.pieces + pieces);
    a.per_row = (int)fth::ceil_div(d->vocab, kPiece);
    a.by_pieces = fth::Divisor((uint32_t)a.per_row);
    a.want_p = 48;  // (us for 200 x 131071, top-p 0.9, 24 / 48 / 63: 37.3 + 11.4 / 38.2 + 13.9 / 40.9 + 12.5 in all; fewer send more rows to the pass over all)
    int bits = 0;
    while (((int64_t)1 << bits) < d->vocab) ++bits;
    const int s_bits = 62 - bits < 45 ? 62 - bits : 45;
    a.magic = __builtin_ldexp(1.5, 52 - s_bits);
    a.unit = __builtin_ldexp(1.0, s_bits);
    const int64_t blocks = fth::ceil_div(pieces, kWaves);
    sample_pieces_kernel<<<dim3((unsigned)blocks), dim3(64 * kWaves), 0, st>>>(a);
    FTH_CHECK_LAUNCH("sample_pieces");
    sample_choice_kernel<<<dim3((unsigned)d->rows), dim3(kThreads), 0, st>>>(a);
    FTH_CHECK_LAUNCH("sample_choice");
    return FTH_OK;
}

}  // extern "C"
