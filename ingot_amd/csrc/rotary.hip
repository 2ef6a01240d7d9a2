// Rotary positions: the tables of angles, the rotation of heads, the rotation
// fused with the append of keys and values to cache pages, and both with a norm
// of each head before the rotation.

#include <algorithm>

#include "decoder.hpp"
#include "launch_bound.hpp"

namespace ingot {

namespace {

// One angle per thread in 64 bits: with positions up to 2^31 the product p·f
// needs more than the 24 bits of f32 before it is reduced to one turn (at
// p = 10^5 an f32 product is off by up to 0.004 rad). Runs when a model is
// loaded; the transcendental functions bound it.
__global__ void rotary_table_kernel(ingot_rocm_rotary_table_args a, double base, int64_t from) {
    const int half = a.rot_dim / 2;
    const int64_t i = from + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.rows * half) return;
    const int64_t row = i / half;
    const int j = (int)(i - row * half);
    double f = pow(base, -2.0 * j / a.rot_dim);
    if (a.scaling == INGOT_ROTARY_LINEAR) {
        f /= a.factor;
    } else if (a.scaling == INGOT_ROTARY_BY_PARTS) {
        const double turns = a.trained * f / 6.283185307179586;
        const double g = fmin(fmax((turns - a.low) / (a.high - a.low), 0.0), 1.0);
        f = (1.0 - g) * f / a.factor + g * f;
    }
    double s, c;
    sincos((double)(a.first + row) * f, &s, &c);
    a.d_cos[i] = (float)(c * a.amplitude);
    a.d_sin[i] = (float)(s * a.amplitude);
}

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<uint16_t>(uint16_t v) { return bf16_to_f32(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ uint16_t narrow<uint16_t>(float v) { return f32_to_bf16(v); }

// V elements moved by one access of V·sizeof(T) bytes (V = 1: no alignment).
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, float (&v)[V]) {
    T t[V];
    __builtin_memcpy(t, __builtin_assume_aligned(p, V * sizeof(T) > 16 ? 16 : V * sizeof(T)), V * sizeof(T));
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = widen<T>(t[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_f32(T* p, const float (&v)[V]) {
    T t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = narrow<T>(v[i]);
    __builtin_memcpy(__builtin_assume_aligned(p, V * sizeof(T) > 16 ? 16 : V * sizeof(T)), t, V * sizeof(T));
}

// One unit: 2V elements of a head, read before any of them is written, so that
// y may be x. Units 0 .. half/V − 1 hold V pairs each; the units after them the
// dimensions past rot_dim, V at a time in two pieces.
template <typename X, typename Y, int V>
__device__ __forceinline__ void turn_unit(const X* x, Y* y, int u, int pairs, int half, int dim, bool rotate,
                                          bool interleaved, const float* cos, const float* sin, float sign,
                                          bool in_table) {
    float a[V], b[V];
    if (rotate && u < pairs) {
        float c[V], s[V];
        if (in_table) {
            load_f32<float, V>(cos + u * V, c);
            load_f32<float, V>(sin + u * V, s);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = s[i] = __builtin_nanf("");
        }
        if (interleaved) {
            float p[2 * V];
            load_f32<X, V>(x + 2 * u * V, a);
            load_f32<X, V>(x + 2 * u * V + V, b);
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] = a[i], p[V + i] = b[i];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float e = p[2 * i], o = p[2 * i + 1];
                const float n = e * c[i] - o * sign * s[i], m = o * c[i] + e * sign * s[i];
                if (2 * i < V) a[2 * i] = n; else b[2 * i - V] = n;
                if (2 * i + 1 < V) a[2 * i + 1] = m; else b[2 * i + 1 - V] = m;
            }
            store_f32<Y, V>(y + 2 * u * V, a);
            store_f32<Y, V>(y + 2 * u * V + V, b);
        } else {
            load_f32<X, V>(x + u * V, a);
            load_f32<X, V>(x + half + u * V, b);
            float n[V], m[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                n[i] = a[i] * c[i] - b[i] * sign * s[i];
                m[i] = b[i] * c[i] + a[i] * sign * s[i];
            }
            store_f32<Y, V>(y + u * V, n);
            store_f32<Y, V>(y + half + u * V, m);
        }
        return;
    }
    const int at = (rotate ? 2 * half + (u - pairs) * 2 * V : u * 2 * V);
    const bool two = at + V < dim;
    if (at >= dim) return;
    load_f32<X, V>(x + at, a);
    if (two) load_f32<X, V>(x + at + V, b);
    store_f32<Y, V>(y + at, a);
    if (two) store_f32<Y, V>(y + at + V, b);
}

// Elements from the cache's first to head 0 of token t's slot, -1 where the
// token's row or page is not there.
__device__ __forceinline__ int64_t slot_of(const KvView& kv, int64_t t) {
    // the token's sequence: the last b with starts[b] <= t
    int lo = 0, hi = kv.batch;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (kv.starts[mid] <= t) lo = mid; else hi = mid;
    }
    const int start = kv.starts[lo];
    const int r = kv.row_of(lo);
    if (r < 0 || t < start || t >= kv.starts[lo + 1]) return -1;
    const int64_t at = (int64_t)kv.len[r] + (t - start);
    const int page = kv.page_of(r, at);
    if (page < 0) return -1;
    const int slot = (int)at - kv.by_page.div((int)at) * kv.page_size;
    return page * kv.stride_page + slot * kv.stride_slot;
}

// A thread takes one unit of one head of one token; heads are the query heads,
// then the key heads, then the value heads. Six operations a pair against 16
// bytes or more moved: bound by the bytes, and for few tokens by the launch. A
// unit is 2V elements so that each half of its pairs is one 16-byte access.
// 8191 tokens of 32 f32 heads of 128 take 48 µs (273 MB, 5.7 TB/s), 512 tokens of
// 32 + 8 + 8 bf16 heads with their append 6.0, one token 4.0 to 4.8.
template <typename X, typename C, int V, bool APPEND>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a, FastDiv by_token, FastDiv by_head, int64_t first,
                                                     int count) {
    const int idx = blockIdx.x * 256 + threadIdx.x;
    if (idx >= count) return;
    const int dt = by_token.div(idx), in_token = idx - dt * by_token.d;
    const int64_t t = first + dt;
    int h = by_head.div(in_token);
    const int u = in_token - h * by_head.d;
    const int half = a.rot.half, pairs = half / V;
    const float sign = a.rot.inverse ? -1.f : 1.f;
    const int pos = half ? a.rot.positions[t] : 0;
    const bool in_table = pos >= 0 && pos < a.rot.rows;
    const float *cos = a.rot.cos + (int64_t)pos * half, *sin = a.rot.sin + (int64_t)pos * half;
    if (!APPEND || h < a.heads) {
        const X* x = (const X*)a.x.data + t * a.x.token + h * a.x.head;
        X* y = (X*)a.y.data + t * a.y.token + h * a.y.head;
        turn_unit<X, X, V>(x, y, u, pairs, half, a.dim, true, a.rot.interleaved, cos, sin, sign, in_table);
        return;
    }
    if constexpr (APPEND) {
        h -= a.heads;
        const bool is_v = h >= a.kv_heads;
        if (is_v) h -= a.kv_heads;
        const int64_t at_slot = slot_of(a.kv, t);
        if (at_slot < 0) return;
        const int64_t off = at_slot + h * a.kv.stride_head;
        const HeadsView& src = is_v ? a.v : a.k;
        turn_unit<X, C, V>((const X*)src.data + t * src.token + h * src.head, (C*)(is_v ? a.kv.v : a.kv.k) + off, u,
                           pairs, half, a.dim, !is_v, a.rot.interleaved, cos, sin, sign, in_table);
    }
}

template <typename X, typename C, int V, bool APPEND>
hipError_t launch(const RotaryArgs& a, hipStream_t st) {
    // a value head has dim / 2V units, no more than a rotated one
    const int half = a.rot.half, units = half / V + (a.dim - 2 * half + 2 * V - 1) / (2 * V);
    const int unit_max = std::max(units, (a.dim + 2 * V - 1) / (2 * V));
    const int64_t per_token = (int64_t)(a.heads + 2 * (APPEND ? a.kv_heads : 0)) * unit_max;
    const int64_t step = std::max<int64_t>(1, (((int64_t)1 << 30) / per_token));
    for (int64_t first = 0; first < a.tokens; first += step) {
        const int64_t n = std::min(step, a.tokens - first) * per_token;
        rotary_kernel<X, C, V, APPEND><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
            a, FastDiv((int32_t)per_token), FastDiv(unit_max), first, (int)n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// V elements stored by one access, bf16 rounded (RNE) by the hardware's conversion.
template <typename T, int V>
__device__ __forceinline__ void store_rounded(T* p, const float (&v)[V]) {
    if constexpr (sizeof(T) == 4) {
        store_f32<T, V>(p, v);
    } else {
        __bf16 t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = (__bf16)v[i];
        __builtin_memcpy(__builtin_assume_aligned(p, V * sizeof(T)), t, V * sizeof(T));
    }
}

// Where the two pieces of a head's unit u lie, in elements: the halves or the
// neighbours of its pairs, or two pieces past rot_dim. A piece past the head is
// read from its beginning and not used.
template <int V, bool INTER>
struct UnitPlace {
    int ia, ib;
    bool turned, has_a, has_b;
    __device__ __forceinline__ UnitPlace(int u, int units, int half, int dim) {
        const int pairs = half / V;
        turned = u < pairs;
        ia = turned ? (INTER ? 2 * u * V : u * V) : 2 * half + (u - pairs) * 2 * V;
        ib = turned && !INTER ? ia + half : ia + V;
        has_a = u < units && ia < dim;
        has_b = u < units && ib < dim;
        if (!has_a) ia = 0;
        if (!has_b) ib = 0;
    }
};

// The pairs of two pieces turned.
template <int V, bool INTER>
__device__ __forceinline__ void turn_pieces(float (&a)[V], float (&b)[V], const float (&c)[V], const float (&s)[V]) {
    if constexpr (!INTER || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float n = a[i] * c[i] - b[i] * s[i];
            b[i] = b[i] * c[i] + a[i] * s[i];
            a[i] = n;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float n = a[2 * i] * c[i] - a[2 * i + 1] * s[i];
            a[2 * i + 1] = a[2 * i + 1] * c[i] + a[2 * i] * s[i];
            a[2 * i] = n;
            const float m = b[2 * i] * c[V / 2 + i] - b[2 * i + 1] * s[V / 2 + i];
            b[2 * i + 1] = b[2 * i + 1] * c[V / 2 + i] + b[2 * i] * s[V / 2 + i];
            b[2 * i] = m;
        }
    }
}

// V elements as they lie in memory, asked for now and widened where they are used.
template <typename T, int V>
struct Raw {
    T t[V];
    __device__ __forceinline__ void load(const T* p) {
        __builtin_memcpy(t, __builtin_assume_aligned(p, V * sizeof(T) > 16 ? 16 : V * sizeof(T)), V * sizeof(T));
    }
    __device__ __forceinline__ void get(float (&v)[V], bool there) const {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = there ? widen<T>(t[i]) : 0.f;
    }
};

// Weights of heads that have none.
__device__ __attribute__((aligned(32))) const float unit_weights[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};

// 1 / sqrt(v) for v >= 0 by the hardware's reciprocal root, which is off by at
// most one step (2^-23 of the value) and takes values below the smallest normal
// number for 0: those are scaled first.
__device__ __forceinline__ float inverse_root(float v) {
    const bool tiny = v < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p64f : v) * (tiny ? 0x1p32f : 1.f);
}

// y = turned(w · x / sqrt(mean(x²) + eps)) for query and key heads, values as they
// are. 2^lanes_log lanes take a head of a token, a unit of it each: it is read
// whole before anything is written (so y may be x), all loads before the first use
// (a branch around one would wait for it inside: 8191 tokens of 32 bf16 heads of
// 128 took 45 µs so, and take 28 to 30), and the sums of squares are added over
// the lanes by permutes. Bound by the bytes: 138 MB, 4.7 TB/s, where a copy of them
// takes 26 µs; lanes that keep their angles for two or four heads take 30 and 31.
// One token 3.7 to 3.9, 512 tokens of 32 + 8 + 8 bf16 heads of 80 with their append
// 5.2. WIDE: heads of more than 64 units, whose lanes go over their units twice.
// Sums and products are f32, rounded once at the store.
template <typename X, typename C, int V, bool APPEND, bool WIDE, bool INTER>
__global__ void __launch_bounds__(256) norm_rotary_kernel(NormRotaryArgs a, FastDiv by_token, int lanes_log, int units,
                                                          int64_t first, int count) {
    using Place = UnitPlace<V, INTER>;
    const int lane = threadIdx.x & 63, lanes = 1 << lanes_log, u0 = lane & (lanes - 1);
    const int number = (int)((blockIdx.x * 256 + threadIdx.x) >> lanes_log);
    const bool there = number < count;  // all lanes take part in the sums
    const int dt = by_token.div(there ? number : 0);
    const int64_t t = first + dt;
    int h = (there ? number : 0) - dt * by_token.d, kind = 0;  // 0 query, 1 key, 2 value
    const int half = a.rot.half;
    const int pos = half ? a.rot.positions[t] : 0;
    const bool in_table = pos >= 0 && pos < a.rot.rows;

    // source and weights of the head
    const X* x;
    const float* w;
    if (APPEND && h >= a.heads) {
        h -= a.heads;
        kind = h >= a.kv_heads ? 2 : 1;
        if (kind == 2) h -= a.kv_heads;
        const HeadsView& src = kind == 2 ? a.v : a.k;
        x = (const X*)src.data + t * src.token + h * src.head;
        w = kind == 2 || !a.weight_k ? nullptr : a.weight_k + h * a.weight_k_head;
    } else {
        x = (const X*)a.x.data + t * a.x.token + h * a.x.head;
        w = a.weight_q ? a.weight_q + h * a.weight_q_head : nullptr;
    }

    const auto angles = [&](int u, bool turned, float (&c)[V], float (&s)[V]) {
        if (half && a.rot.rows) {  // the same for all lanes
            const int64_t at = (int64_t)(in_table ? pos : 0) * half + (turned ? u * V : 0);
            load_f32<float, V>(a.rot.cos + at, c);
            load_f32<float, V>(a.rot.sin + at, s);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            c[i] = in_table ? c[i] : __builtin_nanf("");
            s[i] = in_table ? s[i] : __builtin_nanf("");
        }
    };
    const auto weights = [&](const Place& p, float (&e)[V], float (&f)[V]) {
        load_f32<float, V>(w ? w + p.ia : unit_weights, e);
        load_f32<float, V>(w ? w + p.ib : unit_weights, f);
    };

    const Place place(u0, units, half, a.dim);
    float sum = 0.f, c[V] = {}, s[V] = {}, p[V], q[V], we[V], wf[V];
    {
        Raw<X, V> ra, rb;
        ra.load(x + place.ia), rb.load(x + place.ib);
        angles(u0, place.turned, c, s);
        weights(place, we, wf);
        ra.get(p, place.has_a), rb.get(q, place.has_b);
#pragma unroll
        for (int i = 0; i < V; ++i) sum = fmaf(p[i], p[i], fmaf(q[i], q[i], sum));
    }
    const int64_t at_slot = APPEND && kind ? slot_of(a.kv, t) : 0;
    if constexpr (WIDE) {
        for (int u = u0 + 64; u < units; u += 64) {
            const Place at(u, units, half, a.dim);
            Raw<X, V> ra, rb;
            float e[V], f[V];
            ra.load(x + at.ia), rb.load(x + at.ib);
            ra.get(e, at.has_a), rb.get(f, at.has_b);
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(e[i], e[i], fmaf(f[i], f[i], sum));
        }
    }
#pragma unroll
    for (int off = 32; off; off >>= 1)
        if (off < lanes) sum += xor_partner(sum, off, lane);
    if (!there) return;

    const bool normed = kind == 0 ? a.norm_q : kind == 1 && a.norm_k;
    const float inv = normed ? inverse_root(fmaf(sum, a.inv_dim, kind ? a.eps_k : a.eps_q)) : 1.f;
    const auto put = [&](const Place& at) {
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = p[i] * inv * we[i], q[i] = q[i] * inv * wf[i];
        if (at.turned && kind < 2) turn_pieces<V, INTER>(p, q, c, s);
        if (!APPEND || kind == 0) {
            X* y = (X*)a.y.data + t * a.y.token + h * a.y.head;
            if (at.has_a) store_rounded<X, V>(y + at.ia, p);
            if (at.has_b) store_rounded<X, V>(y + at.ib, q);
        } else if (at_slot >= 0) {
            C* y = (C*)(kind == 2 ? a.kv.v : a.kv.k) + at_slot + h * a.kv.stride_head;
            if (at.has_a) store_rounded<C, V>(y + at.ia, p);
            if (at.has_b) store_rounded<C, V>(y + at.ib, q);
        }
    };
    put(place);
    if constexpr (WIDE) {
        // each lane reads again only what it then writes
        for (int u = u0 + 64; u < units; u += 64) {
            const Place at(u, units, half, a.dim);
            Raw<X, V> ra, rb;
            ra.load(x + at.ia), rb.load(x + at.ib);
            ra.get(p, at.has_a), rb.get(q, at.has_b);
            angles(u, at.turned, c, s);
            weights(at, we, wf);
            put(at);
        }
    }
}

// The widest accesses, up to V elements, at which every address is a multiple of
// its own size: the rotated half, the head and all strides are multiples of them.
// 5162 tokens of 48 bf16 heads of 80, 20 of them rotated (halves of 10): 28 µs
// with 2 elements an access, 42 with 1.
int widest(const RotaryArgs& a, int v, int esz, bool append) {
    const auto fits = [&](const HeadsView& h) {
        return (uintptr_t)h.data % std::min(16, v * esz) == 0 && h.token % v == 0 && h.head % v == 0;
    };
    const auto tables = [&]() { return ((uintptr_t)a.rot.cos | (uintptr_t)a.rot.sin) % std::min(16, v * 4) == 0; };
    for (; v > 1; v /= 2)
        if (a.rot.half % v == 0 && a.dim % v == 0 && tables() && fits(a.x) && fits(a.y) &&
            (!append || (fits(a.k) && fits(a.v))))
            return v;  // the cache's own alignment is checked by the entry point
    return 1;
}

template <typename X, typename C, int V, bool APPEND, bool INTER>
hipError_t launch_norm(const NormRotaryArgs& a, hipStream_t st) {
    const int half = a.rot.half, units = half / V + (a.dim - 2 * half + 2 * V - 1) / (2 * V);
    int log = 0;
    while (log < 6 && (1 << log) < units) ++log;
    const auto kernel = units > 64 ? norm_rotary_kernel<X, C, V, APPEND, true, INTER>
                                   : norm_rotary_kernel<X, C, V, APPEND, false, INTER>;
    const int64_t per_token = a.heads + 2 * (APPEND ? a.kv_heads : 0);
    const int64_t step = std::max<int64_t>(1, (((int64_t)1 << 30) >> log) / per_token);
    for (int64_t first = 0; first < a.tokens; first += step) {
        const int64_t n = std::min(step, a.tokens - first) * per_token;
        kernel<<<(unsigned)(((n << log) + 255) / 256), 256, 0, st>>>(a, FastDiv((int32_t)per_token), log, units, first,
                                                                     (int)n);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <typename X, typename C, int V>
hipError_t pick_norm(const NormRotaryArgs& a, int v, bool append, hipStream_t st) {
    if constexpr (V > 1)
        if (v < V) return pick_norm<X, C, V / 2>(a, v, append, st);
    if (a.rot.interleaved) return append ? launch_norm<X, C, V, true, true>(a, st) : launch_norm<X, X, V, false, true>(a, st);
    return append ? launch_norm<X, C, V, true, false>(a, st) : launch_norm<X, X, V, false, false>(a, st);
}

template <typename X, typename C, int V>
hipError_t pick(const RotaryArgs& a, int v, bool append, hipStream_t st) {
    if constexpr (V > 1)
        if (v < V) return pick<X, C, V / 2>(a, v, append, st);
    return append ? launch<X, C, V, true>(a, st) : launch<X, X, V, false>(a, st);
}

}  // namespace

hipError_t launch_rotary_table(const ingot_rocm_rotary_table_args& a, hipStream_t st) {
    const int64_t n = a.rows * (a.rot_dim / 2);
    double base = a.base;
    if (a.scaling == INGOT_ROTARY_BASE && a.rot_dim > 2) base *= pow(a.factor, (double)a.rot_dim / (a.rot_dim - 2));
    constexpr int64_t step = kLaunchWorkgroups * kWorkgroupThreads;
    for (int64_t from = 0; from < n; from += step) {
        const int64_t m = std::min(step, n - from);
        rotary_table_kernel<<<(unsigned)((m + 255) / 256), 256, 0, st>>>(a, base, from);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_rotary(const RotaryArgs& a, int dtype, int cache_dtype, hipStream_t st) {
    const bool append = a.kv_heads > 0;
    if (dtype == INGOT_DT_BF16) {
        const int v = widest(a, 8, 2, append);
        if (cache_dtype == INGOT_DT_F32) return pick<uint16_t, float, 8>(a, v, append, st);
        return pick<uint16_t, uint16_t, 8>(a, v, append, st);
    }
    const int v = widest(a, 4, 4, append);
    if (cache_dtype == INGOT_DT_BF16) return pick<float, uint16_t, 4>(a, v, append, st);
    return pick<float, float, 4>(a, v, append, st);
}

hipError_t launch_norm_rotary(const NormRotaryArgs& a, int dtype, int cache_dtype, hipStream_t st) {
    const bool append = a.kv_heads > 0;
    const auto narrowed = [&](int v) {  // weights are read by the same accesses
        const auto fits = [&](const float* w, int64_t head) {
            return (uintptr_t)w % std::min(16, v * 4) == 0 && head % v == 0;
        };
        while (v > 1 && !(fits(a.weight_q, a.weight_q_head) && fits(a.weight_k, a.weight_k_head))) v /= 2;
        return v;
    };
    if (dtype == INGOT_DT_BF16) {
        const int v = narrowed(widest(a, 8, 2, append));
        if (cache_dtype == INGOT_DT_F32) return pick_norm<uint16_t, float, 8>(a, v, append, st);
        return pick_norm<uint16_t, uint16_t, 8>(a, v, append, st);
    }
    const int v = narrowed(widest(a, 4, 4, append));
    if (cache_dtype == INGOT_DT_BF16) return pick_norm<float, uint16_t, 4>(a, v, append, st);
    return pick_norm<float, float, 4>(a, v, append, st);
}

}  // namespace ingot
