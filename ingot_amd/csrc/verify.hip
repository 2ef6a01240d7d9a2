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
// Three launches (four with q). The first reads all logits once and leaves each
// row's maximum and sum of exponentials in chunks. The second walks the tree, every
// workgroup of a sequence for itself (the decisions of 64 nodes need only their
// parents' statistics and one logit each, which lanes ask for together; the walk
// then moves lane values), and sums the last node's weights by pieces. The third
// finds the piece and the token at which the running sum passes u times the whole.
// The weights that are drawn from are computed and summed in 64 bits: with 10^5
// tokens a sum in 32 bits would move a border by more than many of them weigh.

#include <algorithm>

#include "decoder.hpp"
#include "launch_bound.hpp"

namespace ingot {

namespace {

constexpr int PIECE = 4096;  // tokens a workgroup of the second launch sums
constexpr int PER = PIECE / 256;

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

template <typename T> __device__ __forceinline__ float logit(T v);
template <> __device__ __forceinline__ float logit<float>(float v) { return v; }
template <> __device__ __forceinline__ float logit<uint16_t>(uint16_t v) { return bf16_to_f32(v); }

// Whether a temperature can be used; 0 is greedy.
__device__ __forceinline__ bool usable(float t) { return t >= 0.f && t < __builtin_inff(); }
__device__ __forceinline__ float temperature_of(const VerifyArgs& a, int b) { return a.temperature ? a.temperature[b] : 0.f; }

// The sequence that row t belongs to: how many of them end at or before it.
__device__ __forceinline__ int sequence_of(const VerifyArgs& a, int t, int lane) {
    int n = 0;
    for (int b = 0; b < a.batch; b += 64) n += __builtin_popcountll(__ballot(b + lane < a.batch && a.starts[b + lane + 1] <= t));
    return min(n, a.batch - 1);
}

// A workgroup takes 256·E logits of a row, all of them in registers at once: their
// maximum, then the sum of exp((x − maximum) / temperature), or for a greedy
// sequence the first place of the maximum. The product with log2(e) / temperature
// is carried in two parts, so that a weight is off by a few 2^-24 of itself.
// A NaN in the chunk leaves a NaN sum.
template <typename T, int E>
__global__ void __launch_bounds__(256) verify_stats_kernel(VerifyArgs a, FastDiv by_chunks) {
    constexpr int VEC = 16 / sizeof(T), N = E / VEC;
    __shared__ float tops[4];
    __shared__ int firsts[4];
    __shared__ double sums[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t = by_chunks.div((int)blockIdx.x), chunk = (int)blockIdx.x - t * by_chunks.d;
    const bool of_draft = blockIdx.y;
    const T* row = (const T*)(of_draft ? a.draft : a.logits) + t * (of_draft ? a.draft_ld : a.logits_ld);
    const int base = chunk * 256 * E;
    T raw[N][VEC];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int at = base + (n * 256 + (int)threadIdx.x) * VEC;
        if (at + VEC <= a.vocab) {
            __builtin_memcpy(raw[n], row + at, 16);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (at + i < a.vocab) raw[n][i] = row[at + i];
        }
    }
    const int b = sequence_of(a, t, lane);
    const float temp = temperature_of(a, b);
    const bool greedy = temp == 0.f;
    float x[N][VEC], top = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int at = base + (n * 256 + (int)threadIdx.x) * VEC + i;
            x[n][i] = at < a.vocab ? logit<T>(raw[n][i]) : -__builtin_inff();
            top = fmaxf(top, x[n][i]);
        }
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0.0;
    int first = 0x7FFFFFFF;
    if (greedy) {
        bool nan = false;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int at = base + (n * 256 + (int)threadIdx.x) * VEC + i;
                if (x[n][i] == top && at < a.vocab) first = min(first, at);
                nan = nan || x[n][i] != x[n][i];
            }
#pragma unroll
        for (int off = 32; off; off >>= 1) first = min(first, xor_partner_bits(first, off, lane));
        sum = __any(nan) ? __builtin_nan("") : 0.0;
    } else {
        // 1 / temperature · log2(e) as the sum of two f32; the largest f32 where it is more
        const double rate = fmin(1.4426950408889634 / (double)temp, 3.4028234663852886e38);
        const float hi = (float)rate, lo = (float)(rate - (double)hi);
        const float mu = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = x[n][i] - mu, y = d * hi;
                const float rest = fmaf(d, hi, -y) + d * lo;
                const float e = __builtin_amdgcn_exp2f(y);
                part += y > -150.f ? fmaf(e, rest * 0.69314718f, e) : e;
            }
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

// A row's statistics from its chunks': the maximum (NaN where the row cannot be
// used: a NaN in it, or a maximum that is not finite), its first place, the sum.
__device__ __forceinline__ VerifyStats row_stats(const VerifyStats* of, int chunks, double rate) {
    VerifyStats r = of[0];
    for (int c = 1; c < chunks; ++c) {
        const VerifyStats s = of[c];
        if (s.top > r.top) r.top = s.top, r.first = s.first;  // chunks rise: a tie stays with the first
    }
    double sum = 0.0;
    for (int c = 0; c < chunks; ++c) {
        const VerifyStats s = of[c];
        if (rate > 0.0) sum += s.sum == 0.0 ? 0.0 : s.sum * exp(((double)s.top - (double)r.top) * rate);
        else sum += s.sum;
    }
    r.sum = sum;
    if (!(fabsf(r.top) < __builtin_inff()) || sum != sum) r.top = __builtin_nanf("");
    return r;
}

// The walk of sequence b, by one wave. With `write` it also leaves the accepted
// nodes and their count.
__device__ __forceinline__ VerifyEnd walk(const VerifyArgs& a, int b, bool write) {
    const int lane = threadIdx.x & 63;
    const int start = a.starts[b], stop = min(a.starts[b + 1], a.tokens);
    const int n = start < 0 ? 0 : max(stop - start, 0);
    const float temp = temperature_of(a, b);
    const bool ok = usable(temp), greedy = temp == 0.f;
    const double rate = greedy || !ok ? 0.0 : 1.0 / (double)temp;
    int32_t* out = a.accepted + (int64_t)b * a.max_accept;
    int cur = 0, count = n > 0, last = 0;  // nodes up to `last` have been looked at
    bool failed = false;
    double gone = 0.0;  // mass of the children of cur that were turned down
    if (write && lane == 0 && n > 0) out[0] = 0;
    const auto load = [&](const void* of, int64_t ld, int row, int token) {
        const int64_t at = (int64_t)row * ld + token;
        return a.bf16 ? bf16_to_f32(((const uint16_t*)of)[at]) : ((const float*)of)[at];
    };
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
            const VerifyStats s = row_stats(a.stats + (int64_t)(start + parent) * a.chunks, a.chunks, rate);
            if (greedy) {
                p = s.top == s.top && s.first == token ? 1.0 : 0.0;
            } else {
                p = exp(((double)load(a.logits, a.logits_ld, start + parent, token) - (double)s.top) * rate) / s.sum;
                if (a.draft) {
                    const VerifyStats d = row_stats(a.draft_stats + (int64_t)(start + parent) * a.chunks, a.chunks, rate);
                    q = exp(((double)load(a.draft, a.draft_ld, start + parent, token) - (double)d.top) * rate) / d.sum;
                }
                u = (double)a.accept_u[start + i];
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
            } else if (a.draft) {
                keep = lane_f64(u, at) * lane_f64(q, at) < pc;
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
                keep = lane_f64(u, at) * (1.0 - gone) < pc;
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
    if (write) {
        for (int i = count + lane; i < a.max_accept; i += 64) out[i] = -1;
        if (lane == 0) a.counts[b] = count;
    }
    VerifyEnd e = {};
    e.node = cur;
    e.nodes = n;
    e.start = start;
    e.rate = rate;
    e.mode = VERIFY_NONE;
    if (n > 0 && ok) {
        const VerifyStats s = row_stats(a.stats + (int64_t)(start + cur) * a.chunks, a.chunks, rate);
        e.top = s.top;
        e.first = s.first;
        if (s.top == s.top) e.mode = greedy ? VERIFY_FIRST : VERIFY_DRAW;
        if (e.mode == VERIFY_DRAW && failed) {
            e.mode = VERIFY_WITHOUT;
            if (a.draft) {
                const VerifyStats d = row_stats(a.draft_stats + (int64_t)(start + cur) * a.chunks, a.chunks, rate);
                e.draft_top = d.top;
                e.mode = d.top == d.top ? VERIFY_REST : VERIFY_NONE;
            }
        }
    }
    return e;
}

// Weight of logit x in 64 bits; 0 for −Inf.
__device__ __forceinline__ double weight(float x, float top, double rate) { return exp(((double)x - (double)top) * rate); }

// Marks the tokens of piece `piece` that the children of the last node had.
__device__ __forceinline__ void mark_rejected(const VerifyArgs& a, const VerifyEnd& e, int piece, uint32_t* bits) {
    if (threadIdx.x < PIECE / 32) bits[threadIdx.x] = 0;
    __syncthreads();
    if (e.mode == VERIFY_WITHOUT)
        for (int i = e.node + 1 + (int)threadIdx.x; i < e.nodes; i += 256) {
            const int token = (a.parents ? a.parents[e.start + i] : i - 1) == e.node ? a.draft_tokens[e.start + i] : -1;
            if (token >= 0 && token / PIECE == piece) atomicOr(&bits[token % PIECE / 32], 1u << (token % 32));
        }
    __syncthreads();
}

template <typename T>
__device__ __forceinline__ float read_logit(const void* of, int64_t ld, int row, int at) {
    return logit<T>(((const T*)of)[row * ld + at]);
}

__device__ __forceinline__ double block_sum(double v, double* part, int lane, int wave) {
    v = wave_sum(v, lane);
    if (lane == 0) part[wave] = v;
    __syncthreads();
    v = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
    return v;
}

// Walks sequence b (blockIdx.y) and sums the weights of piece blockIdx.x of its
// last node; with a draft those of the draft's row too.
template <typename T>
__global__ void __launch_bounds__(256) verify_walk_kernel(VerifyArgs a) {
    __shared__ VerifyEnd end;
    __shared__ uint32_t bits[PIECE / 32];
    __shared__ double part[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = (int)blockIdx.x / a.pieces, piece = (int)blockIdx.x - b * a.pieces;
    if (wave == 0) {
        const VerifyEnd e = walk(a, b, piece == 0);
        if (lane == 0) {
            end = e;
            if (piece == 0) a.ends[b] = e;
        }
    }
    __syncthreads();
    const VerifyEnd e = end;
    if (e.mode < VERIFY_DRAW) return;
    mark_rejected(a, e, piece, bits);
    double sum = 0.0, drafted = 0.0;
#pragma unroll 4
    for (int k = 0; k < PER; ++k) {
        const int in = k * 256 + (int)threadIdx.x, at = piece * PIECE + in;
        if (at >= a.vocab) break;
        if (!((bits[in / 32] >> (in % 32)) & 1)) sum += weight(read_logit<T>(a.logits, a.logits_ld, e.start + e.node, at), e.top, e.rate);
        if (e.mode == VERIFY_REST)
            drafted += weight(read_logit<T>(a.draft, a.draft_ld, e.start + e.node, at), e.draft_top, e.rate);
    }
    sum = block_sum(sum, part, lane, wave);
    drafted = block_sum(drafted, part, lane, wave);
    if (threadIdx.x == 0) {
        a.sums[(int64_t)b * a.pieces + piece] = sum;
        if (a.draft) a.sums[((int64_t)a.batch + b) * a.pieces + piece] = drafted;
    }
}

// The whole sums of a sequence's weights and of its draft's.
__device__ __forceinline__ double whole_sum(const VerifyArgs& a, int64_t row, int lane) {
    double v = 0.0;
    for (int p = lane; p < a.pieces; p += 64) v += a.sums[row * a.pieces + p];
    return wave_sum(v, lane);
}

__device__ __forceinline__ double left_over(double p, double q) { return p > q ? p - q : p == p && q == q ? 0.0 : p - q; }

// Sums max(p − q, 0) by pieces.
template <typename T>
__global__ void __launch_bounds__(256) verify_rest_kernel(VerifyArgs a) {
    __shared__ double part[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int b = (int)blockIdx.x / a.pieces, piece = (int)blockIdx.x - b * a.pieces;
    const VerifyEnd e = a.ends[b];
    if (e.mode != VERIFY_REST) return;
    const double ip = 1.0 / whole_sum(a, b, lane), iq = 1.0 / whole_sum(a, (int64_t)a.batch + b, lane);
    double sum = 0.0;
#pragma unroll 4
    for (int k = 0; k < PER; ++k) {
        const int at = piece * PIECE + k * 256 + (int)threadIdx.x;
        if (at >= a.vocab) break;
        sum += left_over(weight(read_logit<T>(a.logits, a.logits_ld, e.start + e.node, at), e.top, e.rate) * ip,
                         weight(read_logit<T>(a.draft, a.draft_ld, e.start + e.node, at), e.draft_top, e.rate) * iq);
    }
    sum = block_sum(sum, part, lane, wave);
    if (threadIdx.x == 0) a.sums[((int64_t)2 * a.batch + b) * a.pieces + piece] = sum;
}

// Finds the next token of sequence b: the first with a weight at which the running
// sum passes u times the whole one, or the last with a weight.
template <typename T>
__global__ void __launch_bounds__(256) verify_next_kernel(VerifyArgs a) {
    __shared__ uint32_t bits[PIECE / 32];
    __shared__ double part[4];
    __shared__ int found[2];  // piece; the least token that passes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.x;
    const VerifyEnd e = a.ends[b];
    if (e.mode < VERIFY_DRAW) {
        if (threadIdx.x == 0) a.next[b] = e.mode == VERIFY_FIRST ? e.first : -1;
        return;
    }
    const int64_t row = e.mode == VERIFY_REST ? (int64_t)2 * a.batch + b : b;
    const double whole = whole_sum(a, row, lane), target = (double)a.sample_u[b] * whole;
    double ip = 1.0, iq = 1.0;
    if (e.mode == VERIFY_REST) ip = 1.0 / whole_sum(a, b, lane), iq = 1.0 / whole_sum(a, (int64_t)a.batch + b, lane);
    // the piece, and what lies before it
    double before = 0.0, base = 0.0;
    int piece = -1;
    for (int p0 = 0; p0 < a.pieces; p0 += 64) {
        const int p = p0 + lane;
        const double own = p < a.pieces ? a.sums[row * a.pieces + p] : 0.0;
        double upto = own;
        for (int off = 1; off < 64; off <<= 1) {
            const double v = __shfl_up(upto, off);
            if (lane >= off) upto += v;
        }
        const uint64_t some = __ballot(own > 0.0), passed = __ballot(own > 0.0 && base + upto > target);
        if (some) {
            const int at = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
            piece = p0 + at;
            before = base + lane_f64(upto - own, at);
        }
        if (passed) break;
        base += lane_f64(upto, 63);
    }
    if (piece < 0) {  // nothing is left, or the sum is no number
        if (threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    mark_rejected(a, e, piece, bits);
    if (threadIdx.x == 0) found[0] = 0x7FFFFFFF, found[1] = -1;
    // each thread has PER neighbours, so threads follow each other as tokens do
    double w[PER], own = 0.0;
    const int in0 = (int)threadIdx.x * PER, at0 = piece * PIECE + in0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        w[k] = 0.0;
        if (at0 + k < a.vocab && !((bits[(in0 + k) / 32] >> ((in0 + k) % 32)) & 1)) {
            w[k] = weight(read_logit<T>(a.logits, a.logits_ld, e.start + e.node, at0 + k), e.top, e.rate);
            if (e.mode == VERIFY_REST)
                w[k] = left_over(w[k] * ip, weight(read_logit<T>(a.draft, a.draft_ld, e.start + e.node, at0 + k), e.draft_top, e.rate) * iq);
        }
        own += w[k];
    }
    double upto = own;
    for (int off = 1; off < 64; off <<= 1) {
        const double v = __shfl_up(upto, off);
        if (lane >= off) upto += v;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    double run = before + (upto - own);
    for (int k = 0; k < wave; ++k) run += part[k];
    int pass = 0x7FFFFFFF, some = -1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        run += w[k];
        if (w[k] > 0.0) {
            some = at0 + k;
            if (run > target) pass = min(pass, at0 + k);
        }
    }
    if (pass != 0x7FFFFFFF) atomicMin(&found[0], pass);
    if (some >= 0) atomicMax(&found[1], some);
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
    const unsigned grid = (unsigned)((int64_t)a.batch * a.pieces);
    verify_walk_kernel<T><<<grid, 256, 0, st>>>(a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (a.draft) {
        verify_rest_kernel<T><<<grid, 256, 0, st>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    verify_next_kernel<T><<<(unsigned)a.batch, 256, 0, st>>>(a);
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
    if (a.tokens * n > kLaunchWorkgroups || (int64_t)a.batch * a.pieces > kLaunchWorkgroups) return 0;
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
