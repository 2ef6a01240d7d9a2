// Attention of new (drafted) tokens over a paged key/value cache.
//
// The rows of a sequence's key head are its (node, query head of the group)
// pairs: they all read the same keys, so a workgroup takes up to 16·RT of them
// at once and each key and value is fetched once per row tile. Its four waves
// take blocks of KB positions in turn, each with its own running maximum, sum
// and output (one pass, online softmax), and join at the end; where there are
// few rows the positions are cut over workgroups too, and a second launch joins
// the pieces.
//
// Per block the scores are computed transposed, Sᵀ[key][row] = K·Qᵀ, by 16 × 16
// MFMA tiles: a lane then holds 4 consecutive keys of one row, which is the form
// in which the next product, Oᵀ[d][row] += Vᵀ·Pᵀ, takes its second operand
// (over a bf16 cache with the keys of two tiles interleaved, the same order on
// both sides). So the probabilities never leave the registers, and a lane's
// output column is the row whose maximum and sum it keeps: rescaling needs no
// exchange. Keys are read from memory in fragment form. bf16 values go through
// LDS, each wave its own part (no barrier in the loop), and come back by
// transposing reads; f32 values are read as fragments too.
//
// Bound by the bytes of the cache for one or few rows.

#include <algorithm>

#include "decoder.hpp"

namespace ingot {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr int TAB = 1024;  // pages whose offsets are held in LDS at a time
constexpr int STEP = 128;  // positions a workgroup's waves take together (the finest cut of them)

__device__ __forceinline__ bool nonfinite(float v) { return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u; }

// Row bounds of one (sequence, row tile): shared by the kernel and the join.
struct TileSpan {
    int row;         // of the table, -1: none
    int start;       // first token
    int rows;        // rows of the sequence's key head
    int len;         // committed tokens
    int end;         // positions the tile's rows may see
    int full_end;    // positions all of them see
};
template <int BR>
__device__ __forceinline__ TileSpan tile_span(const TreeAttnArgs& a, int b, int tile) {
    TileSpan s;
    s.start = a.kv.starts[b];
    const int last = min(a.kv.starts[b + 1], a.kv.tokens);
    const int n = s.start < 0 ? 0 : min(max(last - s.start, 0), a.max_nodes);
    s.rows = n * a.group;
    s.row = a.kv.row_of(b);
    s.len = s.row < 0 ? 0 : max(0, a.kv.len[s.row]);
    const int64_t all = s.row < 0 ? 0 : min((int64_t)s.len + n, (int64_t)a.max_tokens);
    const int r0 = tile * BR;
    if (a.mask) {
        s.end = (int)all;
        s.full_end = (int)min((int64_t)s.len, all);
    } else {
        const int first = a.by_group.div(r0), final = a.by_group.div(max(0, min(s.rows, r0 + BR) - 1));
        s.end = (int)min(all, (int64_t)s.len + final + 1);
        s.full_end = (int)min(all, (int64_t)s.len + first + 1);
    }
    return s;
}

// 4 consecutive elements of a row of q as f32, zero from dimension `dim` on.
__device__ __forceinline__ f32x4_t load_q4(const TreeAttnArgs& a, const char* row, int d) {
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (!row || d >= a.dim) return v;  // dim is a multiple of 8
    if (a.q_bf16) {
        const uint16_t* p = (const uint16_t*)row + d;
        uint16_t t[4];
        if (a.q_vec) __builtin_memcpy(t, __builtin_assume_aligned(p, 8), 8);
        else for (int i = 0; i < 4; ++i) t[i] = p[i];
        for (int i = 0; i < 4; ++i) v[i] = bf16_to_f32(t[i]);
    } else {
        const float* p = (const float*)row + d;
        if (a.q_vec) v = *(const f32x4_t*)p;
        else for (int i = 0; i < 4; ++i) v[i] = p[i];
    }
    return v;
}

constexpr float TINY = 0x1p-126f;

// x as QT bf16 terms: rounded where there is one; the three whose sum is x
// where there are three (each cuts off the next 8 bits, so no term is rounded).
// The terms have x's sign, ±TINY in place of zeros unless x is zero: an infinite
// factor then gives ±Inf as x itself would, where a zero term would give NaN.
template <int QT>
__device__ __forceinline__ void terms_of(float x, float (&t)[QT]) {
    if constexpr (QT == 1) {
        t[0] = x;
    } else {
        const float tiny = copysignf(fminf(fabsf(x), TINY), x);
        const auto cut = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); };
        t[0] = cut(x);
        const float r = x - t[0];
        t[1] = cut(r);
        t[2] = cut(r - t[1]);
        if (fabsf(t[1]) < TINY) t[1] = tiny;
        if (fabsf(t[2]) < TINY) t[2] = tiny;
    }
}
// terms_of for a query, which may not be finite: carried by the first term.
template <int QT>
__device__ __forceinline__ void query_terms(float x, uint16_t (&t)[QT]) {
    float f[QT];
    terms_of<QT>(x, f);
    if (QT > 1 && nonfinite(x)) {
        f[0] = x;
        f[1] = f[QT - 1] = copysignf(TINY, x);
    }
#pragma unroll
    for (int q = 0; q < QT; ++q) t[q] = f32_to_bf16(f[q]);
}

// Position of 16-byte chunk c of value row `key` in a wave's LDS part: rows are
// DP·2 bytes; pairs of chunks are exchanged so that the four rows a lane group
// reads together, and those of the other groups, lie in different banks.
template <int DP>
__device__ __forceinline__ int v_chunk(int key, int c) {
    const int x = DP >= 128 ? (key & 7) : ((key >> 1) & 3);
    return key * (DP / 8) + (c ^ (2 * x));
}

template <typename T, int DP, int RT, int QT>
__global__ void __launch_bounds__(256) tree_attention_kernel(TreeAttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int BR = 16 * RT, NT = DP / 16;
    constexpr int KB = F32 ? 16 : 32, KTN = KB / 16;  // positions of a wave's block, key tiles
    constexpr int EPC = 16 / sizeof(T);               // elements of a 16-byte chunk
    constexpr int NC = DP / (4 * EPC);                // chunks a lane takes of a key row
    constexpr int ROW_CHUNKS = DP / EPC, VROWS = 64 / ROW_CHUNKS;  // bf16: value rows of one wave-wide load
    constexpr int NV = F32 ? 4 * (DP / 64) : KB / VROWS;
    __shared__ __align__(16) char buf[WAVES * 64 * DP];  // values, then the join's output tiles
    __shared__ int64_t tab[TAB];
    __shared__ float ml[2][WAVES][BR];

    const int pid = ((int)blockIdx.x & 7) * a.per_xcd + ((int)blockIdx.x >> 3);
    if (pid >= a.items) return;
    const int tile = pid % a.row_tiles, ps = pid / a.row_tiles, split = ps % a.splits, bh = ps / a.splits;
    const int b = bh / a.kv.kv_heads, h = bh - b * a.kv.kv_heads;
    const TileSpan sp = tile_span<BR>(a, b, tile);
    const int r0 = tile * BR;
    if (r0 >= sp.rows) return;
    const int64_t begin = (int64_t)split * a.chunk;
    if (split > 0 && begin >= sp.end) return;
    const int stop = (int)min((int64_t)sp.end, begin + a.chunk);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int esz = sizeof(T);

    // the rows' queries, second operand of K·Qᵀ
    i32x4_t qf[QT][RT][NC];
    int node[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + 16 * rt + col;
        const bool in = r < sp.rows;
        const int i = a.by_group.div(in ? r : 0), head = h * a.group + (in ? r : 0) - i * a.group;
        node[rt] = in ? i : -1;
        const char* row = in ? a.q.data + ((sp.start + i) * a.q.token + head * a.q.head) * (a.q_bf16 ? 2 : 4) : nullptr;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = (4 * c + g) * EPC;
            if constexpr (F32) {
                qf[0][rt][c] = __builtin_bit_cast(i32x4_t, load_q4(a, row, d));
            } else {
                const f32x4_t lo = load_q4(a, row, d), hi = load_q4(a, row, d + 4);
                uint16_t t[QT][8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint16_t w[QT];
                    query_terms<QT>(e < 4 ? lo[e & 3] : hi[e & 3], w);
#pragma unroll
                    for (int q = 0; q < QT; ++q) t[q][e] = w[q];
                }
#pragma unroll
                for (int q = 0; q < QT; ++q) __builtin_memcpy(&qf[q][rt][c], t[q], 16);
            }
        }
    }

    f32x4_t o[RT][NT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff();
        l[rt] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) o[rt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }

    char* const vbuf = buf + wave * 64 * DP;
    const int64_t slot_bytes = a.kv.stride_slot * esz;
    for (int ws = (int)begin; ws < stop;) {
        // the offsets of the next pages: those of up to TAB, in whole steps of the waves
        const int p0 = a.kv.by_page.div(ws);
        const int64_t room = (int64_t)(p0 + (int64_t)TAB) * a.kv.page_size;
        const int we = room >= stop ? stop : ws + (((int)room - ws) & ~(STEP - 1));
        const int count = a.kv.by_page.div(we - 1) - p0 + 1;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += 256) {
            int id = -1;
            if (p0 + i < a.kv.max_pages) id = a.kv.pages[(int64_t)sp.row * a.kv.max_pages + p0 + i];
            tab[i] = id >= 0 && id < a.kv.num_pages ? (id * a.kv.stride_page + h * a.kv.stride_head) * esz : -1;
        }
        __syncthreads();
        // byte offset of a position's row, -1 where there is none (then row 0 is read, and hidden)
        const auto place = [&](int pos) -> int64_t {
            if (pos >= we) return -1;
            const int p = a.kv.by_page.div(pos);
            const int64_t base = tab[p - p0];
            return base < 0 ? -1 : base + (pos - p * a.kv.page_size) * slot_bytes;
        };
        for (int kb = ws + wave * KB; kb < we; kb += WAVES * KB) {
            // ---- loads ----
            i32x4_t kf[KTN][NC], vf[NV];
            uint32_t holes = 0;  // keys of the block that are not there
#pragma unroll
            for (int kt = 0; kt < KTN; ++kt) {
                const int64_t off = place(kb + 16 * kt + col);
                holes |= ((uint32_t)__ballot(off < 0) & 0xFFFFu) << (16 * kt);
                const char* p = a.kv.k + (off < 0 ? 0 : off);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const int d = (4 * c + g) * EPC;
                    kf[kt][c] = *(const i32x4_t*)(p + (d < a.dim ? d * esz : 0));
                    // q is zero there, but 0 · Inf is not
                    if (a.dim < DP && d >= a.dim) kf[kt][c] = i32x4_t{0, 0, 0, 0};
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t off = place(kb + 4 * g + i);
                    const char* p = a.kv.v + (off < 0 ? 0 : off);
#pragma unroll
                    for (int u = 0; u < DP / 64; ++u) {
                        const int d = 64 * u + 4 * col;
                        vf[i * (DP / 64) + u] = *(const i32x4_t*)(p + (d < a.dim ? d * 4 : 0));
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int64_t off = place(kb + j * VROWS + lane / ROW_CHUNKS);
                    const int c = lane % ROW_CHUNKS;
                    vf[j] = *(const i32x4_t*)(a.kv.v + (off < 0 ? 0 : off) + (c * EPC < a.dim ? c * 16 : 0));
                }
            }
            // ---- scores ----
            f32x4_t s[RT][KTN];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int kt = 0; kt < KTN; ++kt) {
                    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        if constexpr (F32) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __builtin_bit_cast(f32x4_t, kf[kt][c])[e],
                                    __builtin_bit_cast(f32x4_t, qf[0][rt][c])[e], acc, 0, 0, 0);
                        } else {
#pragma unroll
                            for (int q = 0; q < QT; ++q)
                                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[kt][c]),
                                                                              __builtin_bit_cast(bf16x8_t, qf[q][rt][c]),
                                                                              acc, 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] *= a.scale;
                    s[rt][kt] = acc;
                }
            // ---- who sees what: most blocks are seen whole by every row ----
            const bool whole = kb + KB <= sp.full_end && !holes;
            uint32_t vis[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) vis[rt] = 0xFFu;
            if (!whole) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    vis[rt] = 0;
                    const uint32_t* words = a.mask ? a.mask + (int64_t)(sp.start + max(node[rt], 0)) * a.mask_words : nullptr;
#pragma unroll
                    for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = 16 * kt + 4 * g + i, n = kb + key - sp.len;
                            bool see = node[rt] >= 0 && !((holes >> key) & 1u);
                            if (see && n >= 0)
                                see = words ? (n >> 5) < a.mask_words && ((words[n >> 5] >> (n & 31)) & 1u) : n <= node[rt];
                            if (see) vis[rt] |= 1u << (4 * kt + i);
                            else s[rt][kt][i] = -__builtin_inff();
                        }
                }
            }
            // ---- running maximum and sum ----
            float p[RT][KTN][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float mx = s[rt][0][0];
#pragma unroll
                for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][kt][i]);
                mx = fmaxf(mx, xor_partner(mx, 32, lane));
                mx = fmaxf(mx, xor_partner(mx, 16, lane));
                const float mn = fmaxf(m[rt], mx), mu = mn == -__builtin_inff() ? 0.f : mn;
                const float keep = __builtin_amdgcn_exp2f(m[rt] - mu);
                m[rt] = mn;
                l[rt] *= keep;
#pragma unroll
                for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[rt][kt][i] = __builtin_amdgcn_exp2f(s[rt][kt][i] - mu);
                        l[rt] += p[rt][kt][i];
                    }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[rt][t][i] *= keep;
            }
            // ---- output ----
            bool strange = false;  // a value that is not finite where not every row sees it
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < DP / 64; ++u) {
                        f32x4_t v = __builtin_bit_cast(f32x4_t, vf[i * (DP / 64) + u]);
                        if (!whole) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (nonfinite(v[e])) v[e] = 0.f, strange = true;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt)
                                o[rt][4 * u + e] =
                                    __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], p[rt][0][i], o[rt][4 * u + e], 0, 0, 0);
                    }
            } else {
                bf16x8_t pf[QT][RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float x[QT];
                        terms_of<QT>(p[rt][e >> 2][e & 3], x);
#pragma unroll
                        for (int q = 0; q < QT; ++q) pf[q][rt][e] = (__bf16)x[q];
                    }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int key = j * VROWS + lane / ROW_CHUNKS;
                    *(i32x4_t*)(vbuf + v_chunk<DP>(key, lane % ROW_CHUNKS) * 16) = vf[j];
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint32_t w[4];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int key = 16 * half + 4 * g + (col >> 2);
                        const char* at = vbuf + v_chunk<DP>(key, 2 * t + ((col & 3) >> 1)) * 16 + 8 * (col & 1);
                        const s16x4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4_t*)at);
                        __builtin_memcpy(&w[2 * half], &r, 8);
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u, strange = true;
                            if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0xFFFFu, strange = true;
                        }
                    }
                    bf16x8_t v;
                    __builtin_memcpy(&v, w, 16);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int q = 0; q < QT; ++q)
                            o[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pf[q][rt], o[rt][t], 0, 0, 0);
                }
            }
            // The products above took such values as zeros; add them where they are seen (0 · Inf included).
            if (!whole && __any(strange)) {
                for (int gk = 0; gk < 4; ++gk) {
#pragma unroll
                    for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                        for (int ik = 0; ik < 4; ++ik)
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
                                const float pk = __shfl(p[rt][kt][ik], 16 * gk + col);
                                const bool see = (__shfl((int)vis[rt], 16 * gk + col) >> (4 * kt + ik)) & 1;
#pragma unroll
                                for (int t = 0; t < NT; ++t)
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        float v;
                                        if constexpr (F32) {
                                            const f32x4_t own = __builtin_bit_cast(f32x4_t, vf[ik * (DP / 64) + t / 4]);
                                            v = __shfl(own[t & 3], 16 * gk + 4 * g + i);
                                        } else {
                                            const int d = 16 * t + 4 * g + i;
                                            v = bf16_to_f32(((const uint16_t*)(vbuf + v_chunk<DP>(16 * kt + 4 * gk + ik, d >> 3) * 16))[d & 7]);
                                        }
                                        if (see && nonfinite(v)) o[rt][t][i] += pk * v;
                                    }
                            }
                }
            }
        }
        ws = we;
    }

    // ---- the waves join ----
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] += xor_partner(l[rt], 32, lane);
        l[rt] += xor_partner(l[rt], 16, lane);
        if (g == 0) {
            ml[0][wave][16 * rt + col] = m[rt];
            ml[1][wave][16 * rt + col] = l[rt];
        }
    }
    __syncthreads();
    const int64_t part = ((int64_t)bh * a.row_tiles + tile) * a.splits + split;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float top = ml[0][0][16 * rt + col];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, ml[0][w][16 * rt + col]);
        const float tu = top == -__builtin_inff() ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
            sum += ml[1][w][16 * rt + col] * __builtin_amdgcn_exp2f(ml[0][w][16 * rt + col] - tu);
        const float mine = __builtin_amdgcn_exp2f(m[rt] - tu);
        if (rt) __syncthreads();  // the last tile's readers are done
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f32x4_t v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = o[rt][t][i] * mine;
            *(f32x4_t*)(vbuf + (t * 64 + lane) * 16) = v;
        }
        __syncthreads();
        const int r = r0 + 16 * rt + col;
        if (a.splits > 1 && wave == 0 && g == 0 && r < sp.rows) a.part_ml[part * BR + 16 * rt + col] = make_float2(top, sum);
#pragma unroll
        for (int k = 0; k < NT / WAVES; ++k) {
            const int t = wave * (NT / WAVES) + k;
            f32x4_t v = *(const f32x4_t*)(buf + (t * 64 + lane) * 16);
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                const f32x4_t x = *(const f32x4_t*)(buf + w * 64 * DP + (t * 64 + lane) * 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += x[i];
            }
            if (r >= sp.rows) continue;
            // dimensions of v[0..3]: 4 neighbours, or (f32 tiles) 4 apart
            const int d0 = F32 ? 64 * (t / 4) + 16 * g + (t & 3) : 16 * t + 4 * g;
            constexpr int ds = F32 ? 4 : 1;
            if (a.splits > 1) {
                float* dst = a.part_o + (part * BR + 16 * rt + col) * a.dim;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d0 + ds * i < a.dim) dst[d0 + ds * i] = v[i];
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = sum == 0.f ? 0.f : v[i] / sum;
            const int i_node = a.by_group.div(r), head = h * a.group + r - i_node * a.group;
            const int64_t at = (sp.start + i_node) * a.y.token + head * a.y.head;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d0 + ds * i < a.dim) {
                    if (a.q_bf16) ((uint16_t*)a.y.data)[at + d0 + ds * i] = f32_to_bf16(v[i]);
                    else ((float*)a.y.data)[at + d0 + ds * i] = v[i];
                }
        }
    }
}

// Joins the pieces of a row tile, a wave per row: lanes hold 4 dimensions each,
// and where that leaves lanes over, groups of lanes take the pieces in turn.
template <int BR>
__global__ void __launch_bounds__(256) tree_attention_join_kernel(TreeAttnArgs a) {
    const int tile = (int)blockIdx.x % a.row_tiles, bh = (int)blockIdx.x / a.row_tiles;
    const int b = bh / a.kv.kv_heads, h = bh - b * a.kv.kv_heads;
    const int lane = threadIdx.x & 63, rr = blockIdx.y * WAVES + (threadIdx.x >> 6);
    const TileSpan sp = tile_span<BR>(a, b, tile);
    const int r = tile * BR + rr;
    if (r >= sp.rows) return;
    const int pieces = max(1, (int)(((int64_t)sp.end + a.chunk - 1) / a.chunk));
    const int64_t first = ((int64_t)bh * a.row_tiles + tile) * a.splits;
    const int lanes = a.dim <= 64 ? 16 : a.dim <= 128 ? 32 : 64, groups = 64 / lanes;
    const int d = (lane % lanes) * 4, mine = lane / lanes;
    float top = -__builtin_inff();
    for (int s = 0; s < pieces; ++s) top = fmaxf(top, a.part_ml[(first + s) * BR + rr].x);
    const float tu = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = mine; s < pieces; s += groups) {
        const float2 x = a.part_ml[(first + s) * BR + rr];
        const float w = __builtin_amdgcn_exp2f(x.x - tu);
        sum += w * x.y;
        if (d < a.dim) {
            const f32x4_t v = *(const f32x4_t*)(a.part_o + ((first + s) * BR + rr) * a.dim + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += w * v[i];
        }
    }
    for (int off = lanes; off < 64; off <<= 1) {
        sum += xor_partner(sum, off, lane);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += xor_partner(acc[i], off, lane);
    }
    if (mine || d >= a.dim) return;
    const int i_node = a.by_group.div(r), head = h * a.group + r - i_node * a.group;
    const int64_t at = (sp.start + i_node) * a.y.token + head * a.y.head + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = sum == 0.f ? 0.f : acc[i] / sum;
    if (a.q_bf16) {
        uint16_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = f32_to_bf16(acc[i]);
        uint16_t* p = (uint16_t*)a.y.data + at;
        if (a.y_vec) __builtin_memcpy(__builtin_assume_aligned(p, 8), t, 8);
        else for (int i = 0; i < 4; ++i) p[i] = t[i];
    } else {
        float* p = (float*)a.y.data + at;
        if (a.y_vec) *(f32x4_t*)p = acc;
        else for (int i = 0; i < 4; ++i) p[i] = acc[i];
    }
}

// Row tiles of a wave: as many as the rows fill and the registers hold.
int row_tiles_of(const TreeAttnArgs& a, int cache_dtype) {
    const int rows = a.max_nodes * a.group;
    const bool f32 = cache_dtype == INGOT_DT_F32, three = !f32 && !a.q_bf16;
    const int most = a.dim > 128 ? (f32 || three ? 1 : 2) : (f32 || three ? 2 : 4);
    return std::min(most, rows <= 16 ? 1 : rows <= 32 ? 2 : 4);
}

template <typename T, int DP, int RT, int QT>
hipError_t launch(const TreeAttnArgs& a, hipStream_t st) {
    tree_attention_kernel<T, DP, RT, QT><<<(unsigned)(a.per_xcd * 8), 256, 0, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    const unsigned tiles = (unsigned)(a.items / a.splits);
    tree_attention_join_kernel<16 * RT><<<dim3(tiles, 16 * RT / WAVES), 256, 0, st>>>(a);
    return hipGetLastError();
}

template <typename T, int DP, int QT>
hipError_t launch_rows(const TreeAttnArgs& a, int rt, hipStream_t st) {
    constexpr bool WIDE = sizeof(T) == 4 || QT > 1;
    if constexpr (DP <= 128 && !WIDE)
        if (rt == 4) return launch<T, DP, 4, QT>(a, st);
    if constexpr (DP <= 128 || !WIDE)
        if (rt == 2) return launch<T, DP, 2, QT>(a, st);
    return launch<T, DP, 1, QT>(a, st);
}

}  // namespace

size_t plan_tree_attention(TreeAttnArgs& a, int cache_dtype, int num_cus) {
    const int br = 16 * row_tiles_of(a, cache_dtype);
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const int64_t tiles = (rows + br - 1) / br, base = tiles * a.kv.batch * a.kv.kv_heads;
    a.items = 0;
    if (base > (1 << 24)) return 0;
    a.row_tiles = (int32_t)tiles;
    const int64_t most = std::max<int64_t>(1, (a.max_tokens + 2 * STEP - 1) / (2 * STEP));
    const int64_t splits = std::min<int64_t>(most, std::max<int64_t>(1, 2 * num_cus / base));
    a.chunk = (int32_t)std::min<int64_t>(0x7FFFFF80, (((a.max_tokens + splits - 1) / splits) + STEP - 1) / STEP * STEP);
    a.splits = (int32_t)std::max<int64_t>(1, ((int64_t)a.max_tokens + a.chunk - 1) / a.chunk);
    a.items = (int32_t)(base * a.splits);
    a.per_xcd = (a.items + 7) / 8;
    return a.splits == 1 ? 0 : (size_t)a.items * br * (a.dim + 2) * sizeof(float);
}

hipError_t launch_tree_attention(const TreeAttnArgs& a, int cache_dtype, hipStream_t st) {
    const int rt = row_tiles_of(a, cache_dtype);
    const auto by_dim = [&](auto type, auto qt) {
        using T = decltype(type);
        constexpr int QT = decltype(qt)::value;
        if (a.dim <= 64) return launch_rows<T, 64, QT>(a, rt, st);
        if (a.dim <= 128) return launch_rows<T, 128, QT>(a, rt, st);
        return launch_rows<T, 256, QT>(a, rt, st);
    };
    if (cache_dtype == INGOT_DT_F32) return by_dim(float{}, std::integral_constant<int, 1>{});
    if (a.q_bf16) return by_dim(uint16_t{}, std::integral_constant<int, 1>{});
    return by_dim(uint16_t{}, std::integral_constant<int, 3>{});
}

}  // namespace ingot
