// Rotary positions: the tables of angles, the rotation of heads, and the
// rotation fused with the append of keys and values to cache pages.

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
        // the token's sequence: the last b with starts[b] <= t
        int lo = 0, hi = a.kv.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.kv.starts[mid] <= t) lo = mid; else hi = mid;
        }
        const int start = a.kv.starts[lo];
        const int r = a.kv.row_of(lo);
        if (r < 0 || t < start || t >= a.kv.starts[lo + 1]) return;
        const int64_t at = (int64_t)a.kv.len[r] + (t - start);
        const int page = a.kv.page_of(r, at);
        if (page < 0) return;
        const int slot = (int)at - a.kv.by_page.div((int)at) * a.kv.page_size;
        const int64_t off = page * a.kv.stride_page + h * a.kv.stride_head + slot * a.kv.stride_slot;
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

}  // namespace ingot
