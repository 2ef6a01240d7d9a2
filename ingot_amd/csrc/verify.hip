// Verification of drafted tokens: which of them are kept, and the token that
// follows.
//
// With p the target's probabilities after a node (its logits over the
// temperature, softmax) the node's children come in turn:
//   candidates that were given (trees): token t is kept where u·(1 − R) < p(t), R
//     the mass of the children turned down before it; where none is kept the next
//     token is drawn from p without those tokens;
//   tokens drawn from a draft's probabilities q (chains): kept where u·q(t) < p(t);
//     turned down, the next token is drawn from max(p − q, 0).
// A token that nobody proposed after the last one kept is drawn from p. All three
// leave the next tokens distributed as the target alone would draw them.
//
// Three launches, one more with q and one more for many sequences. The first reads
// all logits once and leaves each row's maximum and sum of exponentials in chunks:
// bound by the bytes, 64 trees of up to 16 nodes over 128000 bf16 logits (197 MB) in
// 39 µs, 5 TB/s. Then a wave walks the tree of a sequence: the decisions of 64 nodes
// need only their parents' statistics and one logit each, which lanes ask for
// together; the walk moves lane values. A decision nearer to its border than statistics
// in 32 bits can tell is made again with sums in 64 bits, so all of them are those of
// the definition in 64 bits (calls without such a one take 0.1 to 0.8 µs more for it).
// The last node's weights are summed by pieces, and the last launch finds the piece and
// the token at which the running sum passes u times the whole. Each of these launches
// is a chain of three or four dependent reads: walk 8 to 9 µs, sums 5 to 11.5, what a
// draft leaves 4.5, the draw 7 to 8.6.
// The weights that are drawn from are computed and summed in 64 bits: with 10^5 tokens
// a sum in 32 bits would move a border by more than many of them weigh.
//
// Times: one token of 32000 f32 logits 14 µs, 8 trees of up to 24 nodes over 50001
// bf16 25, 32 chains of up to 6 over 131072 f32 with their draft's (151 MB) 50, 64
// trees of up to 16 over 128000 bf16 65.

#include <algorithm>

#include "decoder.hpp"
#include "launch_bound.hpp"

namespace ingot {

namespace {

constexpr int PIECE = 2048;  // tokens a workgroup sums
constexpr int PER = PIECE / 256;
constexpr int FIND = 512;  // threads that look through a piece
constexpr int EACH = PIECE / FIND;

__device__ __forceinline__ double shfl_xor_f64(double v, int off, int lane) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = xor_partner_bits((int)(uint32_t)u, off, lane), hi = xor_partner_bits((int)(u >> 32), off, lane);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double wave_sum(double v, int lane) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v += shfl_xor_f64(v, off, lane);
    return v;
}
__device__ __forceinline__ double lane_f64(double v, int from) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, from), hi = __builtin_amdgcn_readlane((int)(u >> 32), from);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// ln(2)^k / k!, k = 0 .. 11.
struct Exp2Terms {
    double of[12];
    constexpr Exp2Terms() : of() {
        of[0] = 1.0;
        for (int k = 1; k < 12; ++k) of[k] = of[k - 1] * 0.693147180559945309417232 / k;
    }
};

// 2^y for y <= 0; 0 below 2^-1000 (and for −Inf). The whole part n goes into the
// exponent's bits (added to 1.5·2^52 it stands in the lower word), the rest, at most
// a half, through the series of 2^f up to f^11 (6e-15 of the value): of 64-bit
// instructions only sums and products, which run at the full rate.
__device__ __forceinline__ double exp2_f64(double y) {
    constexpr Exp2Terms terms;
    const double t = fmax(y, -1000.0) + 0x1.8p52, f = fmax(y, -1000.0) - (t - 0x1.8p52);
    double r = terms.of[11];
#pragma unroll
    for (int k = 10; k >= 0; --k) r = fma(r, f, terms.of[k]);
    const int64_t bits = __double_as_longlong(r) + ((int64_t)(int32_t)__double_as_longlong(t) << 52);
    return y > -1000.0 ? __longlong_as_double(bits) : 0.0;
}

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit<float>(float v) { return v; }
template <> __device__ __forceinline__ float logit<uint16_t>(uint16_t v) { return bf16_to_f32(v); }

constexpr double LOG2E = 1.4426950408889634, LARGEST = 3.4028234663852886e38;

// 0 is greedy.
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int b) { return a.temperature ? a.temperature[b] : 0.f; }

// The sequence that row t belongs to: as many end at or before it.
__device__ __forceinline__ int sequence_of(const VerifyArgs& a, int t) {
    return min(count_at_most(a.starts + 1, a.batch, t), a.batch - 1);
}

// 256·E logits of a row in a workgroup's registers, as they lie in memory: a thread
// has E / VEC accesses of 16 bytes, 256 of them apart.
template <typename T, int E>
struct Logits {
    static constexpr int VEC = 16 / sizeof(T), N = E / VEC;
    T raw[N][VEC];
    __device__ __forceinline__ static int place(int n) { return (n * 256 + (int)threadIdx.x) * VEC; }
    // From `base` on; what lies past the vocabulary is not read.
    __device__ __forceinline__ void load(const T* row, int base, int vocab) {
        if (base + 256 * E <= vocab) {
#pragma unroll
            for (int n = 0; n < N; ++n) __builtin_memcpy(raw[n], row + base + place(n), 16);
            return;
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int at = base + place(n);
            if (at + VEC <= vocab) {
                __builtin_memcpy(raw[n], row + at, 16);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    raw[n][i] = sizeof(T) == 2 ? (T)0xFF80 : (T)-__builtin_inff();
                    if (at + i < vocab) raw[n][i] = row[at + i];
                }
            }
        }
    }
    __device__ __forceinline__ float get(int n, int i) const { return logit<T>(raw[n][i]); }
};

// A workgroup takes 256·E logits of a row, all of them in registers at once: their
// maximum, then the sum of exp((x − maximum) / temperature), or for a greedy
// sequence the first place of the maximum. A weight 2^y is off by up to (2y + 2)·2^-24
// of itself (y is rounded three times: difference, factor, product), so the sum by
// as much for the y at which most of it lies: 2^-22 for a few likely tokens, 2^-19 for
// 10^5 of a thousandth of the largest. It takes part in acceptance alone, and where that
// is too near to tell the row is summed again (kept_exactly); 64-bit powers here would
// take as long as the bytes again.
// A NaN in the chunk leaves a NaN sum.
template <typename T, int E>
__global__ void __launch_bounds__(256) verify_stats_kernel(VerifyArgs a, FastDiv by_chunks) {
    using Chunk = Logits<T, E>;
    __shared__ float tops[4];
    __shared__ int firsts[4];
    __shared__ double sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = by_chunks.div((int)blockIdx.x), chunk = (int)blockIdx.x - t * by_chunks.d, base = chunk * 256 * E;
    const bool of_draft = blockIdx.y;
    Chunk x;
    x.load((const T*)(of_draft ? a.draft : a.logits) + t * (of_draft ? a.draft_ld : a.logits_ld), base, a.vocab);
    const float temp = temperature_of(a, sequence_of(a, t));
    float top = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < Chunk::N; ++n)
#pragma unroll
        for (int i = 0; i < Chunk::VEC; ++i) top = fmaxf(top, x.get(n, i));
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0.0;
    int first = 0x7FFFFFFF;
    if (temp == 0.f) {
        bool nan = false;
#pragma unroll
        for (int n = 0; n < Chunk::N; ++n)
#pragma unroll
            for (int i = 0; i < Chunk::VEC; ++i) {
                const float v = x.get(n, i);
                if (v == top) first = min(first, base + Chunk::place(n) + i);
                nan = nan || v != v;
            }
#pragma unroll
        for (int off = 32; off; off >>= 1) first = min(first, xor_partner_bits(first, off, lane));
        sum = __any(nan) ? __builtin_nan("") : 0.0;
    } else {
        // log2(e) / temperature, the largest f32 where it is more
        const float rate = (float)fmin(LOG2E / (double)temp, LARGEST);
        const float mu = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int n = 0; n < Chunk::N; ++n) {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < Chunk::VEC; ++i) part += __builtin_amdgcn_exp2f((x.get(n, i) - mu) * rate);
            sum += (double)part;
        }
        sum = wave_sum(sum, lane);
    }
    if (lane == 0) sums[wave] = sum, firsts[wave] = first;
    __syncthreads();
    if (threadIdx.x == 0) {
        VerifyStats s;
        s.top = top;
        s.first = min(min(firsts[0], firsts[1]), min(firsts[2], firsts[3]));
        s.sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        (of_draft ? a.draft_stats : a.stats)[(int64_t)t * a.chunks + chunk] = s;
    }
}

// What a sum over the maximum `from` counts over the maximum `to`; rate is
// log2(e) / temperature (the largest f32 where it is more), 0 for a greedy sequence.
__device__ __forceinline__ double decay(float from, float to, float rate) {
    // a finite difference, where both are −Inf or the rate is 0 too
    return (double)__builtin_amdgcn_exp2f(fmaxf(from - to, -(float)LARGEST) * rate);
}
// Joins the statistics of later places to r.
__device__ __forceinline__ void join(VerifyStats& r, const VerifyStats& s, float rate) {
    const bool rise = s.top > r.top;
    const double scale = rise ? decay(r.top, s.top, rate) : decay(s.top, r.top, rate);
    r.sum = rise ? r.sum * scale + s.sum : r.sum + s.sum * scale;
    if (rise) r.top = s.top, r.first = s.first;
}
// The maximum of a row that cannot be used (a NaN in it, or a maximum that is not
// finite) is NaN.
__device__ __forceinline__ void mark_unusable(VerifyStats& r) {
    if (!(fabsf(r.top) < __builtin_inff()) || r.sum != r.sum) r.top = __builtin_nanf("");
}
// A row's statistics from its chunks', each lane a row of its own, eight asked for
// at a time.
__device__ __forceinline__ VerifyStats row_stats(const VerifyStats* of, int chunks, float rate) {
    VerifyStats r = {-__builtin_inff(), 0, 0.0};
    for (int c = 0; c < chunks; c += 8) {
        VerifyStats s[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = of[min(c + k, chunks - 1)];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k < chunks) join(r, s[k], rate);
    }
    mark_unusable(r);
    return r;
}
// The same of one row, its chunks spread over the lanes.
__device__ __forceinline__ VerifyStats row_stats_together(const VerifyStats* of, int chunks, float rate, int lane) {
    VerifyStats r = {-__builtin_inff(), 0, 0.0};
    const int each = (chunks + 63) / 64;  // neighbours to a lane
    for (int c = lane * each; c < min(chunks, (lane + 1) * each); ++c) join(r, of[c], rate);
    float top = r.top;
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    r.sum *= decay(r.top, top, rate);
    r.sum = wave_sum(r.sum, lane);
    const uint64_t has = __ballot(r.top == top);
    r.first = has ? __builtin_amdgcn_readlane(r.first, __builtin_ctzll(has)) : 0;
    r.top = top;
    mark_unusable(r);
    return r;
}

// Weight of logit x in 64 bits; 0 for −Inf.
__device__ __forceinline__ double weight(float x, float top, double rate) {
    return exp2_f64(((double)x - (double)top) * rate);
}

// The token of the i-th node after the last one kept if it is a child of that.
__device__ __forceinline__ int child_token(const VerifyArgs& a, const VerifyEnd& e, int i) {
    i += e.node + 1;
    if (e.mode != VERIFY_WITHOUT || i >= e.nodes) return -1;
    const int token = a.draft_tokens[e.start + i];
    return (a.parents ? a.parents[e.start + i] : i - 1) == e.node ? token : -1;
}
// Tokens of a piece that the children of the last node had, as bits.
struct Rejected {
    static constexpr int WORDS = PIECE / 32 + 1;  // the last says whether there is any
    uint32_t* bits;
    __device__ __forceinline__ void mark(int token, int piece) const {
        if (token >= 0 && token / PIECE == piece) {
            atomicOr(&bits[token % PIECE / 32], 1u << (token % 32));
            bits[WORDS - 1] = 1;
        }
    }
    // All of a workgroup call it. `early`: the thread's first child_token, which may be
    // asked for before the piece is known.
    __device__ __forceinline__ void collect(const VerifyArgs& a, const VerifyEnd& e, int piece, int early) const {
        for (int i = threadIdx.x; i < WORDS; i += (int)blockDim.x) bits[i] = 0;
        __syncthreads();
        mark(early, piece);
        for (int i = (int)(threadIdx.x + blockDim.x); i < e.nodes - e.node - 1; i += (int)blockDim.x) mark(child_token(a, e, i), piece);
        __syncthreads();
    }
    // By one wave, of the children of node cur before `child`.
    __device__ __forceinline__ void collect(const VerifyArgs& a, int start, int cur, int child, int piece) const {
        const auto order = [] {  // lanes read what other lanes wrote
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
        const int lane = threadIdx.x & 63;
        order();
        for (int i = lane; i < WORDS; i += 64) bits[i] = 0;
        order();
        for (int c = cur + 1 + lane; c < child; c += 64)
            if ((a.parents ? a.parents[start + c] : c - 1) == cur) mark(a.draft_tokens[start + c], piece);
        order();
    }
    __device__ __forceinline__ bool operator[](int in) const { return (bits[in / 32] >> (in % 32)) & 1; }
    __device__ __forceinline__ bool any() const { return bits[WORDS - 1] != 0; }
};

__device__ __forceinline__ float logit_at(const VerifyArgs& a, const void* of, int64_t at) {
    return a.bf16 ? bf16_to_f32(((const uint16_t*)of)[at]) : ((const float*)of)[at];
}

// The weights of a row in 64 bits, summed by a wave: of all tokens but those that the
// children of node cur before `child` had (cur + 1: of all).
__device__ __forceinline__ double weights_left(const VerifyArgs& a, const Rejected& gone, const void* of, int64_t row, float top,
                                               double rate, int start, int cur, int child) {
    constexpr int AT_ONCE = 8;
    const int lane = threadIdx.x & 63;
    const bool some = child > cur + 1;
    double sum = 0.0;
    for (int piece = 0; piece < a.pieces; ++piece) {
        if (some) gone.collect(a, start, cur, child, piece);
        for (int in0 = lane; in0 < PIECE; in0 += 64 * AT_ONCE) {
            const int token = piece * PIECE + in0;
            float x[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) x[k] = logit_at(a, of, row + min(token + 64 * k, a.vocab - 1));
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const bool counts = token + 64 * k < a.vocab && !(some && gone[in0 + 64 * k]);
                sum += counts ? weight(x[k], top, rate) : 0.0;
            }
        }
    }
    return wave_sum(sum, lane);
}

// Whether a child of node cur is kept, with sums in 64 bits. What its predecessors left
// is summed and not taken as a difference, so the last candidate with a weight is
// compared with itself and kept by every number below 1. A wave reads the row (and
// the draft's) for this, 32000 f32 logits in 76 µs, 128000 bf16 in 450; numbers come so
// near to a border once in 2^16 decisions.
__device__ __forceinline__ bool kept_exactly(const VerifyArgs& a, const Rejected& gone, int start, int cur, int child, double u,
                                             double rate, float rate32) {
    const int lane = threadIdx.x & 63, row = start + cur, token = a.draft_tokens[start + child];
    const auto of_token = [&](const void* of, int64_t ld, const VerifyStats* stats, int until, double* whole) {
        const float top = row_stats_together(stats + (int64_t)row * a.chunks, a.chunks, rate32, lane).top;
        *whole = weights_left(a, gone, of, row * ld, top, rate, start, cur, until);
        return weight(logit_at(a, of, row * ld + token), top, rate);
    };
    double left, whole;
    const double p = of_token(a.logits, a.logits_ld, a.stats, a.draft ? cur + 1 : child, &left);
    if (!a.draft) return u * left < p;
    const double q = of_token(a.draft, a.draft_ld, a.draft_stats, cur + 1, &whole);
    return u * q * left < p * whole;
}

// A decision is made again with sums in 64 bits where its sides, each off by the error
// of a row's sum of f32 powers, are nearer than this part of them. The error of
// a weight 2^y (see verify_stats_kernel) with that of its sum over a thread's access,
// and y at most 24 where 2^24 tokens share the mass: below 2^-18.
constexpr double NEAR = 0x1p-17;
// Temperatures at which a sum in f32 has no such bound: a factor past f32, or
// differences past it that still have a weight.
constexpr double LEAST_RATE = 0x1p-110;

// Walks the tree of sequence b, a wave; one of those that do writes what it finds.
__device__ __forceinline__ VerifyEnd walk(const VerifyArgs& a, const Rejected& rejected, int b, bool write) {
    const int lane = threadIdx.x & 63;
    const int start = a.starts[b], stop = min(a.starts[b + 1], a.tokens);
    const int n = start < 0 ? 0 : max(stop - start, 0);
    const float temp = temperature_of(a, b);
    const bool ok = temp >= 0.f && temp < __builtin_inff(), greedy = temp == 0.f;
    const double rate = greedy || !ok ? 0.0 : LOG2E / (double)temp;
    const float rate32 = (float)fmin(rate, LARGEST);
    int32_t* out = a.accepted + (int64_t)b * a.max_accept;
    int cur = 0, count = n > 0, last = 0;  // nodes up to `last` have been looked at
    bool failed = false;
    double gone = 0.0;  // mass of the children of cur that were turned down
    if (write && lane == 0 && n > 0) out[0] = 0;
    const double near = rate >= LEAST_RATE && rate <= LARGEST ? NEAR : __builtin_inf();
    for (int base = 0; ok && base < n && count < a.max_accept && (a.parents || !failed); base += 64) {
        const int i = base + lane;
        int parent = -1, token = -1;
        if (i > 0 && i < n) {
            parent = a.parents ? a.parents[start + i] : i - 1;
            token = a.draft_tokens[start + i];
            if (parent >= i) parent = -1;
        }
        double p = 0.0, q = 0.0, u = 0.0;
        if (parent >= 0 && token >= 0 && token < a.vocab) {
            const int row = start + parent;
            if (greedy) {
                const VerifyStats s = row_stats(a.stats + (int64_t)row * a.chunks, a.chunks, 0.f);
                p = s.top == s.top && s.first == token ? 1.0 : 0.0;
            } else {
                const float x = logit_at(a, a.logits, row * a.logits_ld + token);
                const float y = a.draft ? logit_at(a, a.draft, row * a.draft_ld + token) : 0.f;
                u = (double)a.accept_u[start + i];
                if (u < 0.0) u = 0.0;
                const VerifyStats s = row_stats(a.stats + (int64_t)row * a.chunks, a.chunks, rate32);
                p = s.top == s.top ? exp2_f64(((double)x - (double)s.top) * rate) / s.sum : __builtin_nan("");
                if (a.draft) {
                    const VerifyStats d = row_stats(a.draft_stats + (int64_t)row * a.chunks, a.chunks, rate32);
                    q = d.top == d.top ? exp2_f64(((double)y - (double)d.top) * rate) / d.sum : __builtin_nan("");
                }
            }
        }
        while (count < a.max_accept) {
            const uint64_t next = __ballot(parent == cur && i > last);
            if (!next) break;
            const int at = __builtin_ctzll(next), child = base + at;
            last = child;
            double pc = lane_f64(p, at);
            bool keep;
            if (greedy) {
                keep = pc == 1.0;
            } else {
                const double uc = lane_f64(u, at);
                double side, size;  // what p is compared with; the errors are parts of size
                if (a.draft) {
                    side = uc * lane_f64(q, at);
                    size = side + pc;
                } else {
                    // a token that an earlier child of cur had has nothing left
                    const int tc = __builtin_amdgcn_readlane(token, at);
                    bool again = __ballot(parent == cur && token == tc && i < child) != 0;
                    for (int c = cur / 64 * 64; !again && c < base; c += 64) {
                        const int j = c + lane;
                        const bool sibling = j > cur && (a.parents ? a.parents[start + j] : j - 1) == cur;
                        again = __ballot(sibling && a.draft_tokens[start + j] == tc) != 0;
                    }
                    if (again) pc = 0.0;
                    side = uc * fmax(1.0 - gone, 0.0);
                    size = uc + pc;
                }
                const double over = pc - side, error = near * size;
                keep = over > error;
                if (__builtin_expect(!keep && !(over < -error), 0))  // a NaN comes here too
                    keep = pc > 0.0 && kept_exactly(a, rejected, start, cur, child, uc, rate, rate32);
            }
            if (keep) {
                if (write && lane == 0) out[count] = child;
                cur = child;
                ++count;
                gone = 0.0;
                failed = false;
            } else {
                gone += pc;
                failed = true;
            }
        }
    }
    if (write)
        for (int i = count + lane; i < a.max_accept; i += 64) out[i] = -1;
    VerifyEnd e = {};
    e.node = cur;
    e.nodes = n;
    e.start = start;
    e.rate = rate;
    e.mode = VERIFY_NONE;
    if (n > 0 && ok) {
        const VerifyStats s = row_stats_together(a.stats + (int64_t)(start + cur) * a.chunks, a.chunks, rate32, lane);
        e.top = s.top;
        e.first = s.first;
        if (s.top == s.top) e.mode = greedy ? VERIFY_FIRST : failed ? VERIFY_WITHOUT : VERIFY_DRAW;
        if (e.mode == VERIFY_WITHOUT && a.draft) {
            const VerifyStats d = row_stats_together(a.draft_stats + (int64_t)(start + cur) * a.chunks, a.chunks, rate32, lane);
            e.draft_top = d.top;
            e.mode = d.top == d.top ? VERIFY_REST : VERIFY_NONE;
        }
    }
    if (write && lane == 0) {
        a.counts[b] = count;
        a.ends[b] = e;
        if (e.mode < VERIFY_DRAW) a.next[b] = e.mode == VERIFY_FIRST ? e.first : -1;
    }
    return e;
}

__global__ void __launch_bounds__(64) verify_walk_kernel(VerifyArgs a) {
    __shared__ uint32_t words[Rejected::WORDS];
    walk(a, {words}, blockIdx.x, true);
}

__device__ __forceinline__ double block_sum(double v, double* part, int lane, int wave) {
    v = wave_sum(v, lane);
    if (lane == 0) part[wave] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return v;
}

template <typename T>
__device__ __forceinline__ const T* end_row(const void* of, int64_t ld, const VerifyEnd& e) {
    return (const T*)of + (int64_t)(e.start + e.node) * ld;
}

// Sums the weights of a piece of the sequence's last node; where what a draft leaves
// is drawn from, those of the draft's row too. WALK: every workgroup of a sequence
// walks its tree for itself, one launch less.
template <typename T, bool WALK>
__global__ void __launch_bounds__(256) verify_sum_kernel(VerifyArgs a, FastDiv by_pieces) {
    using Piece = Logits<T, PER>;
    __shared__ uint32_t words[Rejected::WORDS];
    __shared__ double part[4];
    __shared__ VerifyEnd end;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = by_pieces.div((int)blockIdx.x), piece = (int)blockIdx.x - b * a.pieces;
    if (WALK) {
        if (wave == 0) {
            const VerifyEnd e = walk(a, {words}, b, piece == 0);
            if (lane == 0) end = e;
        }
        __syncthreads();
    }
    const VerifyEnd e = WALK ? end : a.ends[b];
    if (e.mode < VERIFY_DRAW) return;
    Piece x;
    x.load(end_row<T>(a.logits, a.logits_ld, e), piece * PIECE, a.vocab);
    const Rejected rejected = {words};
    rejected.collect(a, e, piece, child_token(a, e, (int)threadIdx.x));
    const bool some = rejected.any();
    double sum = 0.0;
#pragma unroll
    for (int n = 0; n < Piece::N; ++n)
#pragma unroll
        for (int i = 0; i < Piece::VEC; ++i) {
            const double w = weight(x.get(n, i), e.top, e.rate);
            sum += some && rejected[Piece::place(n) + i] ? 0.0 : w;
        }
    sum = block_sum(sum, part, lane, wave);
    if (threadIdx.x == 0) a.sums[(int64_t)b * a.pieces + piece] = sum;
    if (e.mode != VERIFY_REST) return;
    x.load(end_row<T>(a.draft, a.draft_ld, e), piece * PIECE, a.vocab);
    sum = 0.0;
#pragma unroll
    for (int n = 0; n < Piece::N; ++n)
#pragma unroll
        for (int i = 0; i < Piece::VEC; ++i) sum += weight(x.get(n, i), e.draft_top, e.rate);
    sum = block_sum(sum, part, lane, wave);
    if (threadIdx.x == 0) a.sums[((int64_t)a.batch + b) * a.pieces + piece] = sum;
}

// The whole of a row of sums.
__device__ __forceinline__ double whole_sum(const VerifyArgs& a, int64_t row, int lane) {
    double v = 0.0;
    for (int p = lane; p < a.pieces; p += 64) v += a.sums[row * a.pieces + p];
    return wave_sum(v, lane);
}

// max(p − q, 0), of weights and their sums' reciprocals: without a fused product, which
// would leave the rounding of one of two equal ones.
__device__ __forceinline__ double above(double p, double ip, double q, double iq) {
#pragma clang fp contract(off)
    return fmax(p * ip - q * iq, 0.0);
}

// Sums max(p − q, 0) by pieces.
template <typename T>
__global__ void __launch_bounds__(256) verify_rest_kernel(VerifyArgs a, FastDiv by_pieces) {
    using Piece = Logits<T, PER>;
    __shared__ double part[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = by_pieces.div((int)blockIdx.x), piece = (int)blockIdx.x - b * a.pieces;
    const VerifyEnd e = a.ends[b];
    if (e.mode != VERIFY_REST) return;
    Piece x, y;
    x.load(end_row<T>(a.logits, a.logits_ld, e), piece * PIECE, a.vocab);
    y.load(end_row<T>(a.draft, a.draft_ld, e), piece * PIECE, a.vocab);
    const double ip = 1.0 / whole_sum(a, b, lane), iq = 1.0 / whole_sum(a, (int64_t)a.batch + b, lane);
    double sum = 0.0;
#pragma unroll
    for (int n = 0; n < Piece::N; ++n)
#pragma unroll
        for (int i = 0; i < Piece::VEC; ++i)
            sum += above(weight(x.get(n, i), e.top, e.rate), ip, weight(y.get(n, i), e.draft_top, e.rate), iq);
    sum = block_sum(sum, part, lane, wave);
    if (threadIdx.x == 0) a.sums[((int64_t)2 * a.batch + b) * a.pieces + piece] = sum;
}

// v added up over the lanes up to this one, moved by lane permutes of the VALU: by 1,
// 2, 4 and 8 lanes within rows of 16, then the last lane of a row (of 32 lanes) to
// the whole of the next.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_moved(double v) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xF, true);
    return v + __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));  // + 0.0 where nothing comes
}
__device__ __forceinline__ double running_sum(double v) {
    v = add_moved<0x111, 0xF>(v);  // row_shr:1
    v = add_moved<0x112, 0xF>(v);
    v = add_moved<0x114, 0xF>(v);
    v = add_moved<0x118, 0xF>(v);
    v = add_moved<0x142, 0xA>(v);  // row_bcast:15 to rows 1 and 3
    return add_moved<0x143, 0xC>(v);  // row_bcast:31 to rows 2 and 3
}

// Finds the next token of sequence b: the first with a weight at which the running
// sum passes u times the whole one, or the last with a weight. Where p is nowhere above
// q (they are the same to 64 bits) it is drawn from p.
template <typename T>
__global__ void __launch_bounds__(FIND) verify_next_kernel(VerifyArgs a) {
    __shared__ uint32_t words[Rejected::WORDS];
    __shared__ double part[FIND / 64];
    __shared__ int found[2];  // the least token that passes, the last with a weight
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.x;
    const VerifyEnd e = a.ends[b];
    if (e.mode < VERIFY_DRAW) return;  // the walk has written it
    bool rest = e.mode == VERIFY_REST;
    const int early = child_token(a, e, (int)threadIdx.x);
    const double u = (double)a.sample_u[b];
    double ip = 1.0, iq = 1.0;
    if (rest) ip = 1.0 / whole_sum(a, b, lane), iq = 1.0 / whole_sum(a, (int64_t)a.batch + b, lane);
    // the lane with the piece (neighbours to a lane), then the piece, and what lies before it
    const int each = (a.pieces + 63) / 64, from = lane * each, to = min(a.pieces, from + each);
    const double* sums = a.sums + (rest ? (int64_t)2 * a.batch + b : b) * a.pieces;
    double own = 0.0;
    for (int p = from; p < to; ++p) own += sums[p];
    uint64_t some = __ballot(own > 0.0);
    if (rest && !some) {
        rest = false;
        sums = a.sums + (int64_t)b * a.pieces;
        own = 0.0;
        for (int p = from; p < to; ++p) own += sums[p];
        some = __ballot(own > 0.0);
    }
    const double upto = running_sum(own);
    const double target = u * lane_f64(upto, 63);
    const uint64_t passed = __ballot(own > 0.0 && upto > target);
    if (!some) {  // nothing is left
        if (threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    const int at = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
    double before = lane_f64(upto - own, at);
    int piece = at * each;
    if (each > 1) {
        double run = before;
        piece = -1;
        for (int p = at * each; p < min(a.pieces, (at + 1) * each); ++p) {
            const double v = sums[p];
            if (v > 0.0) piece = p, before = run;
            run += v;
            if (v > 0.0 && run > target) break;
        }
    }
    const Rejected rejected = {words};
    if (threadIdx.x == 0) found[0] = 0x7FFFFFFF, found[1] = -1;
    rejected.collect(a, e, piece, early);
    // each thread has EACH neighbours, so threads follow each other as tokens do
    const int in0 = (int)threadIdx.x * EACH, at0 = piece * PIECE + in0;
    const T *xs = end_row<T>(a.logits, a.logits_ld, e) + at0, *ys = end_row<T>(a.draft, a.draft_ld, e) + at0;
    T x[EACH], y[EACH];
    if (at0 + EACH <= a.vocab) {
        __builtin_memcpy(x, xs, sizeof(x));
        if (rest) __builtin_memcpy(y, ys, sizeof(y));
    } else {
#pragma unroll
        for (int k = 0; k < EACH; ++k)
            if (at0 + k < a.vocab) {
                x[k] = xs[k];
                if (rest) y[k] = ys[k];
            }
    }
    double w[EACH], mine = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        w[k] = weight(logit<T>(x[k]), e.top, e.rate);
        if (rest) w[k] = above(w[k], ip, weight(logit<T>(y[k]), e.draft_top, e.rate), iq);
        if (at0 + k >= a.vocab || rejected[in0 + k]) w[k] = 0.0;
        mine += w[k];
    }
    const double up = running_sum(mine);
    if (lane == 63) part[wave] = up;
    __syncthreads();
    double run = before + (up - mine);
    for (int k = 0; k < wave; ++k) run += part[k];
    int pass = 0x7FFFFFFF, held = -1;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
        run += w[k];
        if (w[k] > 0.0) {
            held = at0 + k;
            if (run > target) pass = min(pass, at0 + k);
        }
    }
    if (pass != 0x7FFFFFFF) atomicMin(&found[0], pass);
    if (held >= 0) atomicMax(&found[1], held);
    __syncthreads();
    if (threadIdx.x == 0) a.next[b] = found[0] != 0x7FFFFFFF ? found[0] : found[1];
}

template <typename T, int E>
hipError_t launch_stats(const VerifyArgs& a, hipStream_t st) {
    if (!a.tokens) return hipSuccess;
    verify_stats_kernel<T, E><<<dim3((unsigned)((int64_t)a.tokens * a.chunks), a.draft ? 2 : 1), 256, 0, st>>>(a, FastDiv(a.chunks));
    return hipGetLastError();
}

template <typename T>
hipError_t launch(const VerifyArgs& a, hipStream_t st) {
    hipError_t e = a.chunk == 8192   ? launch_stats<T, 32>(a, st)
                   : a.chunk == 4096 ? launch_stats<T, 16>(a, st)
                                     : launch_stats<T, 8>(a, st);
    if (e != hipSuccess) return e;
    // Walks in the sums' workgroups take one token of 32000 (16 pieces) from 16.6 µs to
    // 15.0 and 8 trees over 50001 (200 pieces) from 26.5 to 23.8; past about four
    // workgroups a CU they would take places from the sums (64 trees over 128000, 4032
    // pieces: a launch of its own takes 8 µs, the sums after it 11.5).
    const unsigned grid = (unsigned)((int64_t)a.batch * a.pieces);
    if (a.temperature && grid <= 1024) {
        verify_sum_kernel<T, true><<<grid, 256, 0, st>>>(a, FastDiv(a.pieces));
    } else {
        verify_walk_kernel<<<(unsigned)a.batch, 64, 0, st>>>(a);
        if ((e = hipGetLastError()) != hipSuccess || !a.temperature) return e;
        verify_sum_kernel<T, false><<<grid, 256, 0, st>>>(a, FastDiv(a.pieces));
    }
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (a.draft) {
        verify_rest_kernel<T><<<grid, 256, 0, st>>>(a, FastDiv(a.pieces));
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    verify_next_kernel<T><<<(unsigned)a.batch, FIND, 0, st>>>(a);
    return hipGetLastError();
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t plan_verify(VerifyArgs& a) {
    // the largest chunk that still gives every compute unit four workgroups
    const auto chunks = [&](int size) { return ((int64_t)a.vocab + size - 1) / size; };
    a.chunk = 8192;
    while (a.chunk > 2048 && a.tokens * chunks(a.chunk) < 1024) a.chunk /= 2;
    a.pieces = (int32_t)chunks(PIECE);
    const int64_t n = chunks(a.chunk);
    constexpr int64_t most = kLaunchWorkgroups * kWorkgroupThreads / FIND;  // workgroups of the last launch
    if (a.tokens * n > kLaunchWorkgroups || (int64_t)a.batch * a.pieces > kLaunchWorkgroups || a.batch > most) return 0;
    a.chunks = (int32_t)n;
    const size_t stats = align16((size_t)a.tokens * n * sizeof(VerifyStats));
    return stats * (a.draft ? 2 : 1) + align16((size_t)a.batch * sizeof(VerifyEnd)) +
           (size_t)a.batch * a.pieces * sizeof(double) * (a.draft ? 3 : 1);
}

void place_verify(VerifyArgs& a, void* ws) {
    char* p = (char*)ws;
    const size_t stats = align16((size_t)a.tokens * a.chunks * sizeof(VerifyStats));
    a.stats = (VerifyStats*)p;
    p += stats;
    if (a.draft) {
        a.draft_stats = (VerifyStats*)p;
        p += stats;
    }
    a.ends = (VerifyEnd*)p;
    p += align16((size_t)a.batch * sizeof(VerifyEnd));
    a.sums = (double*)p;
}

hipError_t launch_verify(const VerifyArgs& a, hipStream_t st) {
    return a.bf16 ? launch<uint16_t>(a, st) : launch<float>(a, st);
}

}  // namespace ingot
