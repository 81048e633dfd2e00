// The next token of each row of logits from a given number: temperature, top-k, top-p, min-p.
//
// Tokens are ordered by a code of 64 bits, the complement of the logit's ordered bits above the index: smaller codes come first. Every
// filter keeps a prefix of that order, so the kept tokens are those up to a last code (and above min-p). Weights are fp64 exponentials; where sums of
// them are collected by atomics they are whole numbers W = round(2^S w), whose sums do not depend on the order. Two launches:
//   * pieces: one wavefront for 1024 logits, which it holds. It finds their maximum; where all of the row count (no top-k) the sum of their
//     weights relative to that maximum; and where there is a filter it writes down the largest of them, in the order of the vocabulary: at least
//     `want`, by a bisection of the lanes' maxima, which costs a comparison of one register a step.
//   * choice: one workgroup for a row. Without a filter the sums of the pieces give the piece, and its logits the token. With one, the
//     candidates of all pieces are gathered in LDS, and a histogram over max - x and the ranks inside one of its bins find the last code. It holds if no piece
//     has left out what could lie before it; otherwise the same is done over the whole row.

#include "devmath.hpp"
#include "paged.hpp"

namespace {

constexpr int kPiece = 1024, kEntries = 64, kWaves = 4;          // logits of a piece, candidates that it may write down, pieces of a workgroup
constexpr int kThreads = 1024, kBins = 2048, kList = 8192, kFew = 1024;  // the choice: bins, candidates in LDS, members of a bin that are ranked

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
    int want_p;   // candidates of a piece for top-p and min-p
    double magic; // 1.5 * 2^(52 - S): added to a weight in [0, 1], leaves round(2^S weight) in the low bits
    double unit;  // 2^S
};

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

template <typename T, typename F> __device__ __forceinline__ T wave_reduce(T x, F op) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) x = op(x, (T)__shfl_xor(x, m));
    return x;
}
struct MaxOp { template <typename T> __device__ T operator()(T a, T b) const { return a > b ? a : b; } };
struct AddOp { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };

// ---- pieces -----------------------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(64 * kWaves) void sample_pieces_kernel(const SampleArgs p) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t piece = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t r = piece / p.per_row;
    if (r >= p.d.rows) return;
    const int64_t v0 = (piece - r * p.per_row) * kPiece;
    const int n = (int)(p.d.vocab - v0 < kPiece ? p.d.vocab - v0 : kPiece);
    const float *x = p.logits + r * p.d.logits_stride + v0;
    F4u z[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int i = 256 * s + 4 * lane;
        z[s] = F4u{-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        if (i + 4 <= n) z[s] = *reinterpret_cast<const F4u *>(x + i);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < n) z[s][e] = x[i + e];
    }
    const Settings set(p, r);
    float mine = -__builtin_inff();
    bool bad = false;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bad |= !(z[s][e] < __builtin_inff());
            mine = fmaxf(mine, z[s][e]);
        }
    bad = __any(bad);
    Piece out = {wave_reduce(mine, MaxOp()), -__builtin_inff(), 0u, bad ? 1u : 0u, 0.0};
    if (!bad && !set.bad && out.max > -__builtin_inff()) {
        if (set.top_k == 0) {
            double sum = 0.0;
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += fth::exp2_softmax(((double)z[s][e] - (double)out.max) * set.rate);
            out.sum = wave_reduce(sum, AddOp());
        }
        if (set.filters()) {
            // The largest power-of-two-spaced number that `want` lanes reach; fewer where they would write down too much.
            int want = p.want_p;
            if (set.top_k > 0) {
                const int share = 2 * ((set.top_k + p.per_row - 1) / p.per_row) + 14;
                want = share < 40 ? share : 40;
                want = want < set.top_k ? want : set.top_k;
            }
            const uint32_t key = order_of(mine);
            Entry *to = p.entries + piece * kEntries;
            for (; want > 0; want >>= 1) {
                // the smallest c (16 bits) for which `want` lanes have key < (c + 1) << 16
                uint32_t c = 0;
#pragma unroll
                for (int b = 15; b >= 0; --b) {
                    const uint32_t c1 = c | (1u << b);
                    if (__popcll(__ballot(key < c1 << 16)) < want) c = c1;
                }
                const uint32_t end = c << 16 | 0xffffu;  // written down: what has an order up to `end`
                uint32_t at = 0;
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) at += __popcll(__ballot(order_of(z[s][e]) <= end && z[s][e] > -__builtin_inff()));
                if (at > kEntries) continue;
                out.count = at;
                at = 0;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint64_t in[4];
                    uint32_t before = at;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        in[e] = __ballot(order_of(z[s][e]) <= end && z[s][e] > -__builtin_inff());
                        before += __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0));
                        at += __popcll(in[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (in[e] >> lane & 1) to[before++] = Entry{z[s][e], (uint32_t)(v0 + 256 * s + 4 * lane + e)};
                }
                // the number whose order is `end`: what is left is below it
                out.limit = end == ~0u ? -__builtin_inff() : __uint_as_float((end & 0x80000000u) ? end : end ^ 0x7fffffffu);
                bool left = false;
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) left |= order_of(z[s][e]) > end && z[s][e] > -__builtin_inff();
                if (!__any(left)) out.limit = -__builtin_inff();
                break;
            }
            if (want == 0) out.limit = __builtin_inff();
        }
    }
    if (lane == 0) p.pieces[piece] = out;
}

// ---- the choice ---------------------------------------------------------------------------------------------------------------

struct Shared {
    uint64_t sums[kThreads / 64];
    uint64_t ranges[256];
    uint64_t weight[kBins];
    uint32_t count[kBins];
    Entry list[kList];
    Entry few[kFew];
    float maxima[kThreads / 64];
    uint64_t found, above;
    uint32_t members;
    int at;
};

template <typename T, typename F> __device__ __forceinline__ T block_reduce(T x, T *lds, F op) {
    x = wave_reduce(x, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
    for (int w = 1; w < kThreads / 64; ++w) x = op(x, lds[w]);
    return x;
}
// The sum over the threads before this one; *total: over all.
template <typename T> __device__ __forceinline__ T block_scan(T x, T *lds, T *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T upto = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const T other = (T)__shfl_up(upto, m);
        upto += lane >= m ? other : (T)0;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += lds[w];
        all += lds[w];
    }
    *total = all;
    return before + upto - x;
}

struct Row {
    const SampleArgs &p;
    const Settings &set;
    Shared &s;
    const float *x;
    float big;
    double u;
    int64_t r;

    __device__ __forceinline__ uint64_t whole(float z, double *w) const {
        *w = fth::exp2_softmax(((double)z - (double)big) * set.rate);
        return (uint64_t)__builtin_bit_cast(int64_t, *w + p.magic) - (uint64_t)__builtin_bit_cast(int64_t, p.magic);
    }
    __device__ __forceinline__ uint64_t whole(float z) const {
        double w;
        return whole(z, &w);
    }
    // Distances from the maximum in steps of 1/64 of their size, from 2^-16 to 2^16: they grow with the order.
    __device__ __forceinline__ int bin_of(float z) const {
        const int b = (int)(__float_as_uint(big - z) >> 17) - ((127 - 16) << 6);
        return b < 0 ? 0 : b >= kBins ? kBins - 1 : b;
    }
    template <bool LIST, typename F> __device__ __forceinline__ void each(int n, F f) const {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            if constexpr (LIST) f(s.list[i].x, s.list[i].v);
            else f(x[i], (uint32_t)i);
        }
    }
    __device__ __forceinline__ void write(int token, double share) const {
        p.tokens[r] = token;
        if (p.logprobs) p.logprobs[r] = (float)log(share);
    }

    // The smallest code for which the tokens up to it are `k` at least (k > 0) or weigh `need`, among those up to `last` of the n of the list
    // (of the row); all ones if there is none. *weight: what they weigh (k > 0). Bins first, then ranks in one of them; where a bin has
    // too many members (ties) digit by digit.
    template <bool LIST> __device__ __forceinline__ uint64_t boundary(int n, uint64_t last, uint32_t k, uint64_t need, uint64_t *weight) const {
        const int t = threadIdx.x;
        __syncthreads();
        for (int b = t; b < kBins; b += kThreads) {
            s.weight[b] = 0;
            s.count[b] = 0;
        }
        if (t == 0) {
            s.members = 0;
            s.at = -1;
        }
        __syncthreads();
        each<LIST>(n, [&](float z, uint32_t v) {
            if (!(z > -__builtin_inff()) || code_of(z, v) > last) return;
            const int b = bin_of(z);
            const uint64_t w = whole(z);
            atomicAdd(&s.count[b], 1u);
            if (w) atomicAdd(reinterpret_cast<unsigned long long *>(&s.weight[b]), (unsigned long long)w);
        });
        __syncthreads();
        uint64_t total;
        const uint64_t c0 = s.count[2 * t], c1 = s.count[2 * t + 1], w0 = s.weight[2 * t], w1 = s.weight[2 * t + 1];
        const uint64_t wb = block_scan(w0 + w1, s.sums, &total), cb = block_scan(c0 + c1, s.sums, &total);
        const uint64_t goal = k ? k : need, b0 = k ? cb : wb, m0 = b0 + (k ? c0 : w0), e0 = m0 + (k ? c1 : w1);
        if (b0 < goal && e0 >= goal) {
            const bool second = m0 < goal;
            s.at = 2 * t + second;
            s.found = wb + (second ? w0 : 0);
            s.above = second ? m0 : b0;
        }
        __syncthreads();
        const int bin = s.at;
        if (bin < 0) return ~0ull;
        uint64_t weighs = s.found, had = s.above;
        const uint32_t members = s.count[bin];
        if (members <= kFew) {
            each<LIST>(n, [&](float z, uint32_t v) {
                if (z > -__builtin_inff() && code_of(z, v) <= last && bin_of(z) == bin) s.few[atomicAdd(&s.members, 1u)] = Entry{z, v};
            });
            __syncthreads();
            if (t < (int)members) {  // ranks: in whatever order the members stand
                const uint64_t mine = code_of(s.few[t].x, s.few[t].v);
                uint64_t count = 0, sum = 0;
                for (uint32_t i = 0; i < members; ++i) {
                    const bool before = code_of(s.few[i].x, s.few[i].v) < mine;
                    count += before;
                    if (before) sum += whole(s.few[i].x);
                }
                const uint64_t w = whole(s.few[t].x), upto = had + (k ? count : sum), here = k ? 1 : w;
                if (upto < goal && upto + here >= goal) {
                    s.found = mine;
                    s.above = weighs + sum + w;
                }
            }
            __syncthreads();
            *weight = s.above;
            return s.found;
        }
        uint64_t prefix = 0;
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            if (t < 256) {
                s.weight[t] = 0;
                s.count[t] = 0;
            }
            __syncthreads();
            each<LIST>(n, [&](float z, uint32_t v) {
                const uint64_t c = code_of(z, v);
                if (!(z > -__builtin_inff()) || c > last || bin_of(z) != bin || (shift < 56 && c >> (shift + 8) != prefix)) return;
                const int at = (int)(c >> shift) & 255;
                atomicAdd(&s.count[at], 1u);
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.weight[at]), (unsigned long long)whole(z));
            });
            __syncthreads();
            if (t == 0) {
                int at = 0;
                for (;; ++at) {
                    const uint64_t here = k ? s.count[at] : s.weight[at];
                    if (had + here >= goal || at == 255) break;
                    had += here;
                    weighs += s.weight[at];
                }
                s.found = prefix << 8 | at;
                s.above = had;
                s.sums[0] = weighs + s.weight[at];
                s.sums[1] = weighs;
            }
            __syncthreads();
            prefix = s.found;
            had = s.above;
            *weight = s.sums[0];
            weighs = s.sums[1];
        }
        return prefix;
    }

    // The token among those up to `last` and above min-p, from the n of the list (of the row), which stand in the order of the vocabulary: they
    // are cut into 256 ranges; the sums of all give the range, the wavefront that has it the token.
    template <bool LIST> __device__ __forceinline__ void draw(int n, uint64_t last) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, length = ((n + 255) / 256 + 63) & ~63;  // of a range
        auto weigh = [&](int64_t i, uint32_t *v) {
            if (i >= n) return (uint64_t)0;
            const float z = LIST ? s.list[i].x : x[i];
            *v = LIST ? s.list[i].v : (uint32_t)i;
            if (!(z > -__builtin_inff()) || code_of(z, *v) > last) return (uint64_t)0;
            double w;
            const uint64_t all = whole(z, &w);
            return w >= (double)set.min_p ? all : (uint64_t)0;
        };
        uint32_t v;
        __syncthreads();
        for (int g = wave; g < 256; g += kThreads / 64) {
            uint64_t sum = 0;
            if (g * (int64_t)length < n)
                for (int i = lane; i < length; i += 64) sum += weigh((int64_t)g * length + i, &v);
            sum = wave_reduce(sum, AddOp());
            if (lane == 0) s.ranges[g] = sum;
        }
        __syncthreads();
        uint64_t total;
        const uint64_t mine = threadIdx.x < 256 ? s.ranges[threadIdx.x] : 0, before = block_scan(mine, s.sums, &total);
        uint64_t target = (uint64_t)((double)total * u);
        target = target < total ? target : total - 1;
        if (mine > 0 && before <= target && before + mine > target) {
            s.at = threadIdx.x;
            s.found = target - before;
        }
        __syncthreads();
        if (wave != 0) return;
        uint64_t left = s.found;
        const int g = s.at;
        for (int i0 = 0; i0 < length; i0 += 64) {
            const uint64_t here = i0 + lane < length ? weigh((int64_t)g * length + i0 + lane, &v) : 0;
            uint64_t upto = here;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint64_t other = __shfl_up(upto, m);
                upto += lane >= m ? other : 0;
            }
            if (here > 0 && upto > left && upto - here <= left) write((int)v, (double)here / (double)total);
            const uint64_t all = __shfl(upto, 63);
            if (all > left) return;
            left -= all;
        }
    }

    // The last code that the filters keep; 0: the candidates do not say. `limit`: what is not among them is below it. `sum`: of all weights.
    template <bool LIST> __device__ __forceinline__ uint64_t filter(int n, double sum, float limit) const {
        const bool whole_row = !LIST || limit == -__builtin_inff();
        // whether nothing that was left out could stand before a code
        auto sure = [&](uint64_t code) { return whole_row || (code != ~0ull && (uint32_t)(code >> 32) <= order_of(limit)); };
        // whether min-p leaves out what was left out, and so all that other filters are not sure of
        const bool below = !whole_row && set.min_p > 0.f && fth::exp2_softmax(((double)limit - (double)big) * set.rate) < (double)set.min_p;
        uint64_t last = ~0ull, weight = 0;
        if (set.top_k > 0) {
            last = boundary<LIST>(n, last, (uint32_t)set.top_k, 0, &weight);
            if (!sure(last) && (set.top_p < 1.f || !below)) return 0;
            if (last == ~0ull) {  // fewer tokens are allowed
                uint64_t all = 0;
                each<LIST>(n, [&](float z, uint32_t) { all += whole(z); });
                weight = block_reduce(all, s.sums, AddOp());
            }
            sum = (double)weight;
        }
        if (set.top_p < 1.f) {
            const double need = __builtin_ceil(sum * (double)set.top_p);
            const uint64_t code = boundary<LIST>(n, last, 0, need < 1.0 ? 1 : (uint64_t)need, &weight);
            if (code != ~0ull) last = code;  // (else rounded weights fall short of it, or the candidates do)
            if (!sure(last) && (set.top_k > 0 || !below)) return 0;
        } else if (set.top_k == 0 && !whole_row && !below) {
            return 0;
        }
        return last;
    }
};

__global__ __launch_bounds__(kThreads) void sample_choice_kernel(const SampleArgs p) {
    __shared__ Shared s;
    const int64_t r = blockIdx.x;
    const int t = threadIdx.x;
    const Settings set(p, r);
    const double u = p.uniform[r];
    const Piece *pieces = p.pieces + r * p.per_row;
    bool bad = set.bad || !(u >= 0.0 && u < 1.0);
    float big = -__builtin_inff(), limit = -__builtin_inff();
    uint32_t count = 0;
    for (int i = t; i < p.per_row; i += kThreads) {
        const Piece one = pieces[i];
        bad |= one.bad != 0;
        big = fmaxf(big, one.max);
        limit = fmaxf(limit, one.limit);
        count += one.count;
    }
    bad = __syncthreads_or(bad);
    big = block_reduce(big, s.maxima, MaxOp());
    if (bad || big == -__builtin_inff()) {
        if (t == 0) {
            p.tokens[r] = -1;
            if (p.logprobs) p.logprobs[r] = __builtin_nanf("");
            fth::report_bad_entry(p.bad, r);
        }
        return;
    }
    const Row row = {p, set, s, p.logits + r * p.d.logits_stride, big, u, r};
    // the sums of the pieces, in their order: a thread has neighbouring ones
    const int each = (p.per_row + kThreads - 1) / kThreads, from = t * each, to = from + each < p.per_row ? from + each : p.per_row;
    auto sum_of = [&](int i) {  // (0 where the weights of its tokens could be)
        const double t = ((double)pieces[i].max - (double)big) * set.rate;
        return t > -1000.0 ? pieces[i].sum * fth::exp2_softmax(t) : 0.0;
    };
    double mine = 0.0, total = 0.0, before = 0.0;
    if (set.top_k == 0) {
        for (int i = from; i < to; ++i) mine += sum_of(i);
        before = block_scan(mine, reinterpret_cast<double *>(s.sums), &total);
    }
    if (!set.filters()) {
        const double target = total * u;
        if (t == 0) s.at = -1;
        __syncthreads();
        // (several threads, where rounding lets their stretches overlap: the first; none at the very end: the last that has something)
        if (mine > 0.0 && before + mine > target) atomicMin(reinterpret_cast<unsigned *>(&s.at), (unsigned)t);
        __syncthreads();
        int who = s.at;
        if (who < 0) {
            __syncthreads();
            if (mine > 0.0) atomicMax(&s.at, t);
            __syncthreads();
            who = s.at;
        }
        if (t != who && (t >> 6) != (who >> 6)) return;
        // the wavefront of that thread: its piece, and the token in it
        int at = 0;
        double left = 0.0;
        if (t == who) {
            left = target - before;
            int last = from;
            for (at = from; at < to; ++at) {
                const double here = sum_of(at);
                if (here > left) break;
                if (here > 0.0) last = at;
                left -= here;
            }
            if (at == to) {
                at = last;
                left = 1e300;
            }
        }
        at = __shfl(at, who & 63);
        left = __shfl(left, who & 63);
        const int lane = t & 63, n = (int)(p.d.vocab - (int64_t)at * kPiece < kPiece ? p.d.vocab - (int64_t)at * kPiece : kPiece);
        int token = -1;
        double share = 0.0;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const float z = i0 + lane < n ? row.x[(int64_t)at * kPiece + i0 + lane] : -__builtin_inff();
            const double w = z > -__builtin_inff() ? fth::exp2_softmax(((double)z - (double)big) * set.rate) : 0.0;
            double upto = w;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const double other = __shfl_up(upto, m);
                upto += lane >= m ? other : 0.0;
            }
            const uint64_t over = __ballot(w > 0.0 && upto > left), some = __ballot(w > 0.0);
            if (some) {  // the first that is over, else the last so far
                const int lane_of = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
                token = at * kPiece + i0 + lane_of;
                share = __shfl(w, lane_of);
            }
            if (over) break;
            left -= __shfl(upto, 63);
        }
        if (lane == 0) row.write(token, share / total);
        return;
    }

    limit = block_reduce(limit, s.maxima, MaxOp());
    count = 0;
    for (int i = from; i < to; ++i) count += pieces[i].count;
    uint32_t listed;
    uint32_t place = block_scan(count, reinterpret_cast<uint32_t *>(s.sums), &listed);
    uint64_t last = 0;
    if (listed <= kList) {
        __syncthreads();
        if (p.per_row <= kThreads) {  // a wavefront for a piece
            s.count[t] = count;
            s.members = 0;
            reinterpret_cast<uint32_t *>(s.weight)[t] = place;
            __syncthreads();
#pragma unroll 4
            for (int i = t >> 6; i < p.per_row; i += kThreads / 64)
                if ((uint32_t)(t & 63) < s.count[i]) s.list[reinterpret_cast<uint32_t *>(s.weight)[i] + (t & 63)] = p.entries[(r * p.per_row + i) * kEntries + (t & 63)];
        } else {
            for (int i = from; i < to; ++i)
                for (uint32_t e = 0; e < pieces[i].count; ++e) s.list[place++] = p.entries[(r * p.per_row + i) * kEntries + e];
        }
        __syncthreads();
        last = row.filter<true>((int)listed, total * p.unit, limit);
    }
    if (last) {
        row.draw<true>((int)listed, last);
    } else {
        last = row.filter<false>((int)p.d.vocab, total * p.unit, limit);
        row.draw<false>((int)p.d.vocab, last);
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

int64_t pieces_of(const fth_sample_desc &d) { return d.rows * fth::ceil_div(d.vocab, kPiece); }

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
    a.want_p = 32;
    int bits = 0;
    while (((int64_t)1 << bits) < d->vocab) ++bits;
    const int s_bits = 62 - bits < 45 ? 62 - bits : 45;
    a.magic = __builtin_ldexp(1.5, 52 - s_bits);
    a.unit = __builtin_ldexp(1.0, s_bits);
    const int64_t blocks = fth::ceil_div(pieces, kWaves);
    FTH_ARG(blocks <= 2147483647LL, "sample: too many rows for one launch");
    sample_pieces_kernel<<<dim3((unsigned)blocks), dim3(64 * kWaves), 0, st>>>(a);
    FTH_CHECK_LAUNCH("sample_pieces");
    sample_choice_kernel<<<dim3((unsigned)d->rows), dim3(kThreads), 0, st>>>(a);
    FTH_CHECK_LAUNCH("sample_choice");
    return FTH_OK;
}

}  // extern "C"
