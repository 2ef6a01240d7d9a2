// Attention of new (drafted) tokens over a paged key/value cache.
//
// The rows of a sequence's key head are its (node, query head of the group)
// pairs: they all read the same keys, so a workgroup takes a tile of them at
// once and each key and value is fetched once per tile. One pass over the
// positions, with the running maximum m and sum l of the softmax (online): where
// a row's maximum rises from m to m', its sum and output are multiplied by
// exp(m − m'). exp is taken as 2^x, 1/ln 2 being part of the scale.
//
// Per block of 32 positions the scores are computed transposed, Sᵀ[key][row] =
// K·Qᵀ, by MFMA tiles: a lane then holds keys of one row in the order in which
// the next product, Oᵀ[d][row] += Vᵀ·Pᵀ, takes its second operand (the keys of
// V are read in the same order). So the probabilities never leave the registers,
// and a lane's output column is the row whose maximum and sum it keeps:
// rescaling needs no exchange.
//
// Two forms. With up to 16 rows, or an f32 cache, the four waves of a workgroup
// share the rows and take blocks of positions in turn, each with its own m, l
// and output, which they join at the end. With more rows over a bf16 cache each
// wave has rows of its own and all waves the same positions, which go through a
// ring in LDS. In both, where there are too few workgroups for the card the
// positions are cut over several, and a second launch joins their pieces.
//
// Precision: sums, statistics and outputs are f32. Over a bf16 cache f32 queries
// and their probabilities enter the products as three bf16 terms of 8 bits (the
// products are then exact in f32 but for the sum's own roundings: errors of 3e-7
// of the result at 2000 positions, where f32 arithmetic has 5e-7). bf16 queries
// are one term, and their probabilities are rounded to bf16 once: 2^-9 of each
// and without a common sign, below the rounding of the bf16 result (measured
// together 0.0022 of the result's size, the result's rounding alone 0.0017), for a
// third of the products.
//
// Times in these comments: two of one choice were taken side by side on one card,
// over three inputs in turn; cards differ by up to 10%. The same input again takes
// less where much of it stays in the memory-side cache.

#include <algorithm>
#include <type_traits>

#include "decoder.hpp"
#include "launch_bound.hpp"

namespace ingot {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));

constexpr int WAVES = 4;
constexpr int TAB = 1024;  // pages whose offsets are held in LDS at a time
constexpr int LONG = 512;  // pieces cut by lengths are no shorter than this
constexpr int STEP = 128;  // positions a workgroup's waves take together (the finest cut of them)

__device__ __forceinline__ bool nonfinite(float v) { return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u; }

// What a workgroup does: piece `split` (positions split·chunk on) of a row tile.
// Its partial results are number part, of `pieces`.
struct WorkItem {
    int tile, split, bh, chunk, pieces, part;
};

// The cut of up to 64 sequences, worked out by every wave from their lengths, a
// lane each: pieces of a length that is the same for all but for rounding, as
// short as the workgroups that the card holds at once (a.slots) allow, so that
// all of them are at work and none waits for a place, in multiples of CUT, the
// positions of a workgroup's step. Pieces are numbered by
// sequence, piece, key head and row tile and go to the 8 XCDs in runs: row tiles
// that read the same keys share an L2.
template <int BR, int CUT>
__device__ __forceinline__ WorkItem cut_item(const TreeAttnArgs& a) {
    const int lane = threadIdx.x & 63, heads = a.kv.kv_heads;
    int tiles = 0, all = 0;
    if (lane < a.kv.batch) {
        const int start = a.kv.starts[lane], last = min(a.kv.starts[lane + 1], a.kv.tokens), row = a.kv.row_of(lane);
        const int len = a.kv.len[max(row, 0)];
        const int n = start < 0 ? 0 : min(max(last - start, 0), a.max_nodes);
        tiles = (n * a.group + BR - 1) / BR;
        all = row < 0 ? 0 : (int)min((int64_t)max(0, len) + n, (int64_t)a.max_tokens);
    }
    const int weight = tiles * heads;
    const float span = (float)(all - 1);
    float work = (float)weight * (float)all, held = (float)weight;
#pragma unroll
    for (int off = 32; off; off >>= 1) work += xor_partner(work, off, lane), held += xor_partner(held, off, lane);
    // Each lane tries a length, from the shortest there could be to one at which
    // the pieces, at most work / length + held, are few enough in any case (the
    // host sees to it that held is at most half of a.slots).
    const float slots = (float)a.slots, low = fmaxf((float)a.chunk, work / slots);
    const float high = fmaxf(low, 1.001f * work / (slots - held));
    const float per = 1.f / (low + (high - low) * (float)lane * (1.f / 63.f));
    int sum = 0;
    for (int b = 0; b < a.kv.batch; ++b) {
        const float b_span = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(span), b));
        sum += __builtin_amdgcn_readlane(weight, b) * ((int)(b_span * per) + 1);
    }
    const uint64_t fits = __ballot(sum <= a.slots);
    const float chosen =
        fits ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(per), __builtin_ctzll(fits))) : 0.f;
    const int pieces = (int)(span * chosen) + 1, count = weight * pieces;
    int upto = count;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(upto, off);
        if (lane >= off) upto += v;
    }
    const int total = __builtin_amdgcn_readlane(upto, 63);
    const int per_xcd = (total + 7) >> 3, item = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    const uint64_t past = __ballot(upto > item);
    if (((int)blockIdx.x >> 3) >= per_xcd || !past) return {-1, 0, 0, 0, 1, 0};
    const int b = __builtin_ctzll(past);
    const int first = __builtin_amdgcn_readlane(upto - count, b), n = item - first;
    const int b_tiles = __builtin_amdgcn_readlane(tiles, b), b_all = __builtin_amdgcn_readlane(all, b);
    const int b_pieces = __builtin_amdgcn_readlane(pieces, b), step = b_tiles * heads;
    const auto quotient = [](int x, int y) { return __builtin_amdgcn_readfirstlane(x / y); };
    const int split = quotient(n, step), in_piece = n - split * step;
    const int h = quotient(in_piece, b_tiles), tile = in_piece - h * b_tiles;
    const int bh = b * heads + h;
    if (split == 0 && threadIdx.x == 0) a.cuts[bh * a.row_tiles + tile] = make_int4(item, b_pieces, step, 0);
    const int even = (quotient(b_all + b_pieces - 1, b_pieces) + CUT - 1) / CUT * CUT;  // b_all <= 2^30
    return {tile, split, bh, even, b_pieces, item};
}

// Without a cut by lengths, workgroups go to the 8 XCDs in turn: the row tiles of
// one piece, which read the same keys, follow each other on one XCD (and find
// them in its L2), and the pieces go round the XCDs, first pieces of all
// sequences first, so that long sequences burden all XCDs alike.
template <int BR, int CUT>
__device__ __forceinline__ WorkItem work_item(const TreeAttnArgs& a) {
    if (a.slots) return cut_item<BR, CUT>(a);
    const int idx = (int)blockIdx.x >> 3, turn = idx / a.row_tiles, piece = turn * 8 + ((int)blockIdx.x & 7);
    const int heads = a.kv.batch * a.kv.kv_heads, split = piece / heads, bh = piece - split * heads;
    const int tile = idx - turn * a.row_tiles;
    return {split < a.splits ? tile : -1, split, bh, a.chunk, a.splits, (bh * a.row_tiles + tile) * a.splits + split};
}

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
__device__ __forceinline__ TileSpan tile_span(const TreeAttnArgs& a, int b, int tile, int row) {
    TileSpan s;
    s.start = a.kv.starts[b];
    const int last = min(a.kv.starts[b + 1], a.kv.tokens);
    const int n = s.start < 0 ? 0 : min(max(last - s.start, 0), a.max_nodes);
    s.rows = n * a.group;
    s.row = row;
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

// N consecutive elements of a row of q as f32 (N = 4 or 8), bf16 (QB) or f32,
// by 16-byte loads where they are aligned (VEC; 8 bytes for 4 bf16).
template <int N, bool QB, bool VEC>
__device__ __forceinline__ void load_query(const char* row, int d, float (&v)[N]) {
    if constexpr (QB) {
        uint16_t t[N];
        const uint16_t* p = (const uint16_t*)row + d;
        if constexpr (VEC) {
            __builtin_memcpy(t, __builtin_assume_aligned(p, 2 * N), 2 * N);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) t[i] = p[i];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = bf16_to_f32(t[i]);
    } else {
        const float* p = (const float*)row + d;
        if constexpr (VEC) {
            __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 4 * N);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = p[i];
        }
    }
}

constexpr float TINY = 0x1p-126f;

// x as three bf16 terms whose sum is x: each cuts off the next 8 bits, so no
// term is rounded. The terms have x's sign, ±TINY in place of zeros unless x is
// zero: an infinite factor then gives ±Inf as x itself would, where a zero term
// would give NaN. An infinite or NaN x is carried by the first term; a NaN made
// quiet, since one whose payload is in the lower half alone would leave an
// infinity in the upper. POSITIVE: x is not negative (a probability: no input, so
// a NaN among them is quiet), so neither are the remainders. The lower halves of
// the terms are left as they are: fragments() takes the upper ones.
template <bool POSITIVE>
__device__ __forceinline__ void three_terms(float x, float (&t)[3]) {
    const auto cut = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); };
    t[0] = x;
    const float r = x - cut(x), rest = r - cut(r);
    if constexpr (POSITIVE) {
        const float tiny = fminf(x, TINY);
        t[1] = fmaxf(r, tiny);
        t[2] = fmaxf(rest, tiny);
        return;
    }
    const uint32_t bits = __float_as_uint(x);
    if ((bits & 0x7FFFFFFFu) > 0x7F800000u) t[0] = __uint_as_float(bits | 0x00400000u);
    const float tiny = copysignf(fminf(fabsf(x), TINY), x);
    t[1] = r;
    t[2] = rest;
    if (!(fabsf(t[1]) >= TINY)) t[1] = tiny;
    if (!(fabsf(t[2]) >= TINY)) t[2] = tiny;
}
// 8 values as QT fragments of 8 bf16: the terms, or one rounding.
template <int QT, bool POSITIVE = false>
__device__ __forceinline__ void fragments(const float (&x)[8], i32x4_t (&f)[QT]) {
    if constexpr (QT == 1) {
        bf16x8_t v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (__bf16)x[e];
        f[0] = __builtin_bit_cast(i32x4_t, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float a[3], b[3];
            three_terms<POSITIVE>(x[e], a);
            three_terms<POSITIVE>(x[e + 1], b);
#pragma unroll
            for (int q = 0; q < 3; ++q)  // the upper halves of both
                f[q][e / 2] = (int)__builtin_amdgcn_perm(__float_as_uint(b[q]), __float_as_uint(a[q]), 0x07060302u);
        }
    }
}

// What the lanes past head_dim are pointed at: the padding of a key has to be
// zeros (the query's is, but 0 · Inf is not 0), that of a value may be anything.
__device__ const i32x4_t zero_chunk = {0, 0, 0, 0};

// Byte offsets (of head h in layer) of the pages of positions ws .. we − 1 in
// LDS, at most TAB of them; entry 1 marks one that is not there (offsets are
// multiples of 16; then page 0 is read, and hidden). One of the two words after
// them, in turn from window to window, says whether there is such an entry.
struct PageWindow {
    const int64_t* tab;
    int p0, we;
    uint32_t slot_bytes;
    bool missing;  // some page is not there
    __device__ __forceinline__ int64_t entry(const TreeAttnArgs& a, int pos, int* slot) const {
        const int p = a.kv.by_page.div(pos);
        *slot = pos - p * a.kv.page_size;
        return tab[p - p0];
    }
    // Of position pos, or of the last one where pos is past it.
    __device__ __forceinline__ int64_t offset(const TreeAttnArgs& a, int pos) const {
        int slot;
        const int64_t base = entry(a, min(pos, we - 1), &slot);
        return (base & ~(int64_t)1) + (uint64_t)slot_bytes * (uint32_t)slot;
    }
    // Keys of a block of KB at kb that are not there, as bits.
    template <int KB>
    __device__ __forceinline__ uint32_t holes(const TreeAttnArgs& a, int kb, int lane) const {
        const int have = we - kb;
        uint32_t h = have >= KB ? 0u : have <= 0 ? ~0u : ~0u << have;
        if (missing) {
            int slot;
            h |= (uint32_t)__ballot(entry(a, min(kb + (lane & (KB - 1)), we - 1), &slot) & 1);
        }
        return KB == 32 ? h : h & 0xFFFFu;
    }
};
// The thread's entry of a piece's first pages, asked for before it is known how
// many the row needs: the table and the lengths come back together.
__device__ __forceinline__ int first_pages(const TreeAttnArgs& a, int row, int64_t begin) {
    const int64_t at = (begin > 0x7FFFFFFF ? a.kv.max_pages : a.kv.by_page.div((int)begin)) + (int)threadIdx.x;
    return row >= 0 && at < a.kv.max_pages ? a.kv.pages[(int64_t)row * a.kv.max_pages + at] : -1;
}
// Fills the table for as many positions from ws on, up to stop, as it holds (in
// whole steps of the waves). The whole workgroup calls it.
// `early` is what first_pages read for this thread, which window 0 takes. The flag
// of a window is cleared in the one before, after its second barrier: by then every
// wave has read it for the window before that, and nobody sets it before the next
// first barrier. (Cleared at the window's own beginning it could be cleared under
// a wave that has still to read it: no barrier need lie between two windows.)
__device__ __forceinline__ PageWindow page_window(const TreeAttnArgs& a, const TileSpan& sp, int h, int esz, int ws,
                                                  int stop, int64_t* tab, int early, int window) {
    PageWindow w;
    int64_t* const flag = tab + TAB + (window & 1);
    w.tab = tab;
    w.p0 = a.kv.by_page.div(ws);
    const int64_t room = ((int64_t)w.p0 + TAB) * a.kv.page_size;
    w.we = room >= stop ? stop : ws + (((int)room - ws) & ~(STEP - 1));
    w.slot_bytes = (uint32_t)(a.kv.stride_slot * esz);
    const int count = a.kv.by_page.div(w.we - 1) - w.p0 + 1;
    if (window == 0 && threadIdx.x == 0) *flag = 0;
    __syncthreads();  // the last window's readers of the table are done
    bool lost = false;
    for (int i = threadIdx.x; i < count; i += 256) {
        int id = early;
        if (window || i >= 256) {
            id = -1;
            if (w.p0 + i < a.kv.max_pages) id = a.kv.pages[(int64_t)sp.row * a.kv.max_pages + w.p0 + i];
        }
        const bool there = id >= 0 && id < a.kv.num_pages;
        lost = lost || !there;
        tab[i] = there ? (id * a.kv.stride_page + h * a.kv.stride_head) * esz : 1;
    }
    if (lost) *flag = 1;  // the same value from whoever writes
    __syncthreads();
    w.missing = *flag != 0;
    if (threadIdx.x == 0) tab[TAB + (~window & 1)] = 0;  // the next window's
    return w;
}

// Chunk places within a row of an LDS tile: lanes that read one chunk of 16 rows
// (keys), or a pair of chunks of 8 rows or two pairs of 4 (values), meet
// different banks. The same for rows 8 apart.
template <int DP> __device__ __forceinline__ int key_swizzle(int key) { return DP == 64 ? (key >> 1) & 7 : key & 15; }
template <int DP> __device__ __forceinline__ int value_swizzle(int key) {
    return DP >= 128 ? 4 * (key & 3) + 2 * ((key >> 2) & 1) : 4 * ((key >> 1) & 1) + 2 * ((key >> 2) & 1);
}

template <int DP>
__device__ __forceinline__ int v_chunk(int key, int c) { return key * (DP / 8) + (c ^ value_swizzle<DP>(key)); }

// Vᵀ's fragment of dimensions 16t .. 16t + 15 over a wave's 32 values: lane
// (g, col) gets dimension 16t + col of keys 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3
// (the read gives a lane of a group of 16 element i of each of 4 rows, the rows
// being addressed by the lanes' quarters, 4 elements a lane).
template <int DP>
__device__ __forceinline__ void value_fragment(const char* vbuf, int t, int g, int col, uint32_t (&w)[4]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int key = 16 * half + 4 * g + (col >> 2);
        const char* at = vbuf + v_chunk<DP>(key, 2 * t + ((col & 3) >> 1)) * 16 + 8 * (col & 1);
        const s16x4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)at);
        __builtin_memcpy(&w[2 * half], &r, 8);
    }
}

// Waits until at most `stages` stages of NI loads are on their way (<= MOST).
template <int NI, int MOST>
__device__ __forceinline__ void wait_stages(int stages) {
    static_assert(NI * MOST < 64, "vmcnt is 6 bits");
    constexpr auto code = [](int v) { return (v & 15) | ((v >> 4) << 14) | 0xF70; };
    if constexpr (MOST > 0) {
        if (stages >= MOST) {
            __builtin_amdgcn_s_waitcnt(code(NI * MOST));
            return;
        }
        wait_stages<NI, MOST - 1>(stages);
    } else {
        __builtin_amdgcn_s_waitcnt(code(0));
    }
}

// The mask of a row over N blocks of 32 keys from node number `base` on (negative
// numbers are committed tokens, which all rows see): N + 1 words from the one
// that holds `base`, asked for with the block's keys.
template <int N>
struct MaskWords {
    uint32_t w[N + 1];
    __device__ __forceinline__ void load(const TreeAttnArgs& a, const TileSpan& sp, int node, int base) {
        if (!a.mask) return;
        const uint32_t* words = a.mask + (int64_t)(sp.start + max(node, 0)) * a.mask_words;
        const int most = (int)a.mask_words - 1, first = base >> 5;
#pragma unroll
        for (int i = 0; i <= N; ++i) w[i] = words[min(max(first + i, 0), most)];
    }
    // Which keys of block n a row of node `node` sees, as bits (node < 0: an unused row).
    __device__ __forceinline__ uint32_t seen(const TreeAttnArgs& a, int node, int base, int n) const {
        uint32_t see;
        if (a.mask) {
            const int most = (int)a.mask_words - 1, first = (base >> 5) + n;
            const uint32_t lo = first < 0 ? ~0u : first > most ? 0u : w[n];
            const uint32_t hi = first + 1 < 0 ? ~0u : first + 1 > most ? 0u : w[n + 1];
            see = (uint32_t)((((uint64_t)hi << 32) | lo) >> (base & 31));
        } else {
            const int k = node + 1 - base - 32 * n;  // keys up to the node itself
            see = k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1u;
        }
        return node < 0 ? 0u : see;
    }
};

// Whether any of 8·N bf16 values is not finite: the largest of them without its
// sign is.
template <int N>
__device__ __forceinline__ bool any_nonfinite(const uint32_t (&w)[N][4]) {
    typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t top = {0, 0};
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, w[k][i] & 0x7FFF7FFFu));
    return max(top[0], top[1]) >= 0x7F80u;
}

// Values of a fragment that are not finite become 0.
__device__ __forceinline__ void zero_nonfinite(uint32_t (&w)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7F80u) == 0x7F80u) w[i] &= 0xFFFF0000u;
        if ((w[i] & 0x7F800000u) == 0x7F800000u) w[i] &= 0xFFFFu;
    }
}

// 1 in place of +Inf and NaN (sign: of −Inf and NaN), 0 in place of the others.
__device__ __forceinline__ void infinite_or_nan(uint32_t (&w)[4], int sign) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t out = 0;
#pragma unroll
        for (int sh = 0; sh < 32; sh += 16) {
            const uint32_t v = (w[i] >> sh) & 0xFFFFu, abs = v & 0x7FFFu;
            if (abs > 0x7F80u || v == (sign ? 0xFF80u : 0x7F80u)) out |= 0x3F80u << sh;
        }
        w[i] = out;
    }
}

// Products took the values that are not finite of a block that not every row
// sees as zeros. Where a row sees one its sum is the infinity, or NaN of both:
// products of 0/1 matrices count, per row and dimension, the seen +Inf or NaN
// and the seen −Inf or NaN.
template <int DP, int RT>
__device__ __forceinline__ void add_nonfinite(const char* values, const uint32_t (&see)[RT], int g, int col,
                                              f32x4_t (&o)[RT][DP / 16]) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        bf16x8_t who;
#pragma unroll
        for (int e = 0; e < 8; ++e) who[e] = (__bf16)((see[rt] >> (16 * (e >> 2) + 4 * g + (e & 3))) & 1u ? 1.f : 0.f);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            uint32_t w[4], up[4], dn[4];
            value_fragment<DP>(values, t, g, col, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                up[i] = dn[i] = 0;
#pragma unroll
                for (int sh = 0; sh < 32; sh += 16) {
                    const float v = bf16_to_f32((uint16_t)(w[i] >> sh));
                    if (nonfinite(v) && !(v < 0.f)) up[i] |= 0x3F80u << sh;
                    if (nonfinite(v) && !(v > 0.f)) dn[i] |= 0x3F80u << sh;
                }
            }
            bf16x8_t u8, d8;
            __builtin_memcpy(&u8, up, 16);
            __builtin_memcpy(&d8, dn, 16);
            const f32x4_t none = {0.f, 0.f, 0.f, 0.f};
            const f32x4_t plus = __builtin_amdgcn_mfma_f32_16x16x32_bf16(u8, who, none, 0, 0, 0);
            const f32x4_t minus = __builtin_amdgcn_mfma_f32_16x16x32_bf16(d8, who, none, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (plus[i] > 0.f) o[rt][t][i] += __builtin_inff();
                if (minus[i] > 0.f) o[rt][t][i] -= __builtin_inff();
            }
        }
    }
}

// 4 neighbouring results at element `at` of y.
__device__ __forceinline__ void store_y4(const TreeAttnArgs& a, int64_t at, const f32x4_t& v) {
    if (a.q_bf16) {
        uint16_t t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = f32_to_bf16(v[i]);
        uint16_t* p = (uint16_t*)a.y.data + at;
        if (a.y_vec) {
            __builtin_memcpy(__builtin_assume_aligned(p, 8), t, 8);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = t[i];
        }
    } else {
        float* p = (float*)a.y.data + at;
        if (a.y_vec) {
            *(f32x4_t*)p = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = v[i];
        }
    }
}

// The form for few rows: 16·RT of them, four waves that take blocks of KB
// positions in turn. Keys are read from memory in fragment form, the next block's
// while this one is worked on; bf16 values go through LDS, each wave its own part
// (no barrier in the loop), and come back by transposing reads; f32 values are
// read as fragments too. Bound by the bytes of the cache: 64 sequences of one
// token, 4 query heads to a key head, about 1500 positions: 396 MB in 82 to 84 µs
// (4.7 to 4.8 TB/s). A single token over 517 positions (16 heads) takes 10.7 µs, of
// which the join is 3: a chain of dependent reads (sequence, length, pages, keys)
// in 5 pieces. 16 × 16 tiles and not 32 × 32, which a few
// rows would leave empty. f32 products (16 × 16 × 4) take 8 times as long as
// bf16's: 3 × 7 tokens, 12 heads of 80, about 800 positions 16 µs. An f32 cache of
// 128 dimensions with 32 rows (392 registers) and all caches of more dimensions (404
// to 512; LDS) leave a CU one workgroup; f32 queries over 256 bf16 dimensions spill 4
// registers (20 bytes a lane): 64 sequences as above of 256 dimensions take 177 µs,
// bf16 queries, without spills, 165 (792 MB).
template <typename T, int DP, int RT, int QT>
__global__ void __launch_bounds__(256, (RT == 1 && DP <= 128) || DP == 64 ? 2 : 1) tree_attention_kernel(TreeAttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int BR = 16 * RT, NT = DP / 16;
    constexpr int KB = F32 ? 16 : 32, KTN = KB / 16;  // positions of a wave's block, key tiles
    constexpr int EPC = 16 / sizeof(T);               // elements of a 16-byte chunk
    constexpr int NC = DP / (4 * EPC);                // chunks a lane takes of a key row
    constexpr int ROW_CHUNKS = DP / EPC, VROWS = 64 / ROW_CHUNKS;  // bf16: value rows of one wave-wide load
    constexpr int NV = F32 ? 4 * (DP / 64) : KB / VROWS;
    __shared__ __align__(16) char qbuf[QT * RT * NC * 1024];
    __shared__ __align__(16) char buf[WAVES * 64 * DP];  // values, then the join's output tiles
    __shared__ int64_t tab[TAB + 2];
    __shared__ float ml[2][WAVES][BR];

    const WorkItem wi = work_item<BR, STEP>(a);
    if (wi.tile < 0) return;
    const int tile = wi.tile, split = wi.split, bh = wi.bh, b = bh / a.kv.kv_heads, h = bh - b * a.kv.kv_heads;
    const int64_t begin = (int64_t)split * wi.chunk;
    const int table_row = a.kv.row_of(b), early = first_pages(a, table_row, begin);
    const TileSpan sp = tile_span<BR>(a, b, tile, table_row);
    const int r0 = tile * BR;
    if (r0 >= sp.rows) return;
    const int64_t part = wi.part;
    if (split > 0 && begin >= sp.end) {
        if ((int)threadIdx.x < BR) a.part_ml[part * BR + threadIdx.x] = make_float2(-__builtin_inff(), 0.f);  // nothing to join
        return;
    }
    const int stop = (int)min((int64_t)sp.end, begin + wi.chunk);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, col = lane & 15;
    const int esz = sizeof(T);

    // The rows' queries, second operand of K·Qᵀ: each wave takes a quarter from
    // memory (and splits it), all of them read the whole back from LDS. Asked for
    // here, needed when the first keys are on their way.
    constexpr int NW = (NC + WAVES - 1) / WAVES;  // fragments of a row tile that a wave takes
    i32x4_t qf[QT][RT][NC];
    int node[RT];
    float x[RT][NW][EPC];
    {
        const char* row[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int r = r0 + 16 * rt + col, in = r < sp.rows;
            const int rr = in ? r : r0, i = a.by_group.div(rr), head = h * a.group + rr - i * a.group;
            node[rt] = in ? i : -1;
            row[rt] = a.q.data + ((sp.start + i) * a.q.token + head * a.q.head) * (a.q_bf16 ? 2 : 4);
        }
        const auto fetch = [&](auto qb, auto vec) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int k = 0; k < NW; ++k) {
                    const int d = (4 * (k * WAVES + wave) + g) * EPC;
                    load_query<EPC, decltype(qb)::value, decltype(vec)::value>(row[rt], d < a.dim ? d : 0, x[rt][k]);
                }
        };
        const std::true_type yes;
        const std::false_type no;
        if (a.q_vec) a.q_bf16 ? fetch(yes, yes) : fetch(no, yes);
        else a.q_bf16 ? fetch(yes, no) : fetch(no, no);
    }
    const auto share_queries = [&]() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int k = 0; k < NW; ++k) {
                const int c = k * WAVES + wave;
                if (NC % WAVES && c >= NC) break;
                const bool in = node[rt] >= 0 && (4 * c + g) * EPC < a.dim;
                i32x4_t* dst = (i32x4_t*)qbuf + (rt * NC + c) * QT * 64 + lane;
#pragma unroll
                for (int e = 0; e < EPC; ++e) x[rt][k][e] = !in ? 0.f : a.flip ? -x[rt][k][e] : x[rt][k][e];
                if constexpr (F32) {
                    __builtin_memcpy(dst, x[rt][k], 16);
                } else {
                    i32x4_t f[QT];
                    fragments<QT>(x[rt][k], f);
#pragma unroll
                    for (int q = 0; q < QT; ++q) dst[q * 64] = f[q];
                }
            }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int q = 0; q < QT; ++q) qf[q][rt][c] = ((const i32x4_t*)qbuf)[((rt * NC + c) * QT + q) * 64 + lane];
    };

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
    for (int ws = (int)begin, window = 0; ws < stop; ++window) {
        const PageWindow win = page_window(a, sp, h, esz, ws, stop, tab, early, window);
        const int we = win.we;
        // keys and values of the block at kb
        i32x4_t kf[KTN][NC], vf[NV];
        const auto load_keys = [&](int kb) {
#pragma unroll
            for (int kt = 0; kt < KTN; ++kt) {
                const char* p = a.kv.k + win.offset(a, kb + 16 * kt + col) + g * 16;
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    kf[kt][c] = *(const i32x4_t*)((4 * c + g) * EPC < a.dim ? p + c * 64 : (const char*)&zero_chunk);
            }
        };
        const auto load_values = [&](int kb) {
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const char* p = a.kv.v + win.offset(a, kb + 4 * g + i);
#pragma unroll
                    for (int u = 0; u < DP / 64; ++u) {
                        const int d = 64 * u + 4 * col;
                        vf[i * (DP / 64) + u] = *(const i32x4_t*)(p + (d < a.dim ? d * 4 : 0));
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = lane % ROW_CHUNKS;
                    vf[j] = *(const i32x4_t*)(a.kv.v + win.offset(a, kb + j * VROWS + lane / ROW_CHUNKS) + (c * EPC < a.dim ? c * 16 : 0));
                }
            }
        };
        MaskWords<1> mask[RT];
        const auto load_mask = [&](int kb) {
            if (kb + KB > sp.full_end)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) mask[rt].load(a, sp, node[rt], kb - sp.len);
        };
        const int first = ws + wave * KB;
        if (first < we) load_mask(first), load_keys(first), load_values(first);
        if (window == 0) share_queries();
        for (int kb = first; kb < we; kb += WAVES * KB) {
            const int next = kb + WAVES * KB;
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
                    s[rt][kt] = acc;
                }
            // ---- who sees what: most blocks are seen whole by every row ----
            const uint32_t holes = win.holes<KB>(a, kb, lane);
            const bool whole = kb + KB <= sp.full_end && !holes;
            uint32_t see[RT];  // keys of the block a row sees, as bits
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) see[rt] = ~0u;
            if (!whole) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    see[rt] = mask[rt].seen(a, node[rt], kb - sp.len, 0) & ~holes;
#pragma unroll
                    for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!((see[rt] >> (16 * kt + 4 * g + i)) & 1u)) s[rt][kt][i] = -__builtin_inff();
                }
            }
            if (next < we) load_mask(next), load_keys(next);
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
                mx = fmaxf(mx, xor_partner(mx, 16, lane)) * a.scale;
                if (__any(mx > m[rt])) {
                    const float mn = fmaxf(m[rt], mx);
                    const float keep = __builtin_amdgcn_exp2f(m[rt] - (mn == -__builtin_inff() ? 0.f : mn));
                    m[rt] = mn;
                    l[rt] *= keep;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[rt][t][i] *= keep;
                }
                const float mu = m[rt] == -__builtin_inff() ? 0.f : -m[rt];
#pragma unroll
                for (int kt = 0; kt < KTN; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        p[rt][kt][i] = __builtin_amdgcn_exp2f(fmaf(s[rt][kt][i], a.scale, mu));
                        l[rt] += p[rt][kt][i];
                    }
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
                i32x4_t pf[RT][QT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = p[rt][e >> 2][e & 3];
                    fragments<QT, true>(x, pf[rt]);
                }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int key = j * VROWS + lane / ROW_CHUNKS;
                    *(i32x4_t*)(vbuf + v_chunk<DP>(key, lane % ROW_CHUNKS) * 16) = vf[j];
                }
                if (!whole) {
                    uint32_t w[NV][4];
                    __builtin_memcpy(w, vf, sizeof(vf));
                    strange = __any(any_nonfinite(w));
                }
                if (next < we) load_values(next);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint32_t w[4];
                    value_fragment<DP>(vbuf, t, g, col, w);
                    if (strange) zero_nonfinite(w);
                    bf16x8_t v;
                    __builtin_memcpy(&v, w, 16);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int q = 0; q < QT; ++q)
                            o[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8_t, pf[rt][q]), o[rt][t], 0, 0, 0);
                }
            }
            if (!whole && __any(strange)) {
                if constexpr (!F32) {
                    add_nonfinite<DP, RT>(vbuf, see, g, col, o);
                } else {  // add_nonfinite with the fragments at hand
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            f32x4_t plus = {0.f, 0.f, 0.f, 0.f}, minus = plus;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float v = __builtin_bit_cast(f32x4_t, vf[i * (DP / 64) + t / 4])[t & 3];
                                const float who = (see[rt] >> (4 * g + i)) & 1u ? 1.f : 0.f;
                                plus = __builtin_amdgcn_mfma_f32_16x16x4f32(nonfinite(v) && !(v < 0.f) ? 1.f : 0.f, who, plus, 0, 0, 0);
                                minus = __builtin_amdgcn_mfma_f32_16x16x4f32(nonfinite(v) && !(v > 0.f) ? 1.f : 0.f, who, minus, 0, 0, 0);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (plus[i] > 0.f) o[rt][t][i] += __builtin_inff();
                                if (minus[i] > 0.f) o[rt][t][i] -= __builtin_inff();
                            }
                        }
                }
            }
            if constexpr (F32)
                if (next < we) load_values(next);
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
        if (wi.pieces > 1 && wave == 0 && g == 0 && r < sp.rows) a.part_ml[part * BR + 16 * rt + col] = make_float2(top, sum);
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
            if (wi.pieces > 1) {
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

// The MFMA shapes of the ring form, M × M tiles of Sᵀ (keys × rows) and Oᵀ
// (dimensions × rows): a lane's column is its row, group lane / M.
template <int M> struct Shape;
template <> struct Shape<16> {
    typedef f32x4_t Acc;
    static constexpr int STEP_K = 32, REGS = 4;
    static __device__ __forceinline__ Acc mma(bf16x8_t x, bf16x8_t y, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
};
template <> struct Shape<32> {
    typedef float Acc __attribute__((ext_vector_type(16)));
    static constexpr int STEP_K = 16, REGS = 16;
    static __device__ __forceinline__ Acc mma(bf16x8_t x, bf16x8_t y, Acc c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }
};
// Row (of the tile) that register i of group g holds: 4 in a row, the groups
// in turn.
template <int M> __device__ __forceinline__ int acc_row(int g, int i) { return (256 / M) * (i >> 2) + 4 * g + (i & 3); }

// The wave's maximum, or sum, over the lanes of a column.
template <int M, typename F>
__device__ __forceinline__ float over_column(float x, F f) {
    const int u = __float_as_int(x);
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // each lane: both halves' values
    x = f(__int_as_float((int)s[0]), __int_as_float((int)s[1]));
    if constexpr (M == 16) {
        const int v = __float_as_int(x);
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        x = f(__int_as_float((int)r[0]), __int_as_float((int)r[1]));
    }
    return x;
}

// Second operands of Vᵀ·P: fragment (t, step) holds, in lane (g, col), dimension
// M·t + col of the keys whose probabilities the lane holds in that step. A
// transposing read gives a lane of a group of 16 element i of each of 4 rows,
// which the lanes' quarters address, 4 elements a lane. Eight reads a statement,
// which waits for them itself: before such a read the compiler's own wait would
// be for all DMA.
template <int DP, int M, int NF>
__device__ __forceinline__ void value_fragments(const char* vbuf, int t0, int lane, uint32_t (&w)[NF][4]) {
    typedef int i32x2_t __attribute__((ext_vector_type(2)));
    static_assert(NF == 4, "eight reads");
    constexpr int ROW = DP * 2;
    const int sub = lane & 15, q = (sub & 3) >> 1, half = 8 * (sub & 1);
    i32x2_t r[8];
    if constexpr (M == 16) {
        const int key = 4 * (lane >> 4) + (sub >> 2);
        uint32_t at[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            at[k] = (uint32_t)(uintptr_t)LDS_AS(vbuf + key * ROW + ((2 * (t0 + k) + q) ^ value_swizzle<DP>(key)) * 16 + half);
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
            "ds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
            "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
            "ds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
            : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(16 * ROW)
            : "memory");
    } else {
        const int key = 4 * (lane >> 5) + (sub >> 2);
        uint32_t at[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = 4 * (t0 + k) + 2 * ((lane >> 4) & 1) + q;
            at[k] = (uint32_t)(uintptr_t)LDS_AS(vbuf + key * ROW + (c ^ value_swizzle<DP>(key)) * 16 + half);
        }
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
            "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
            "ds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
            "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
            : "v"(at[0]), "v"(at[1]), "n"(8 * ROW), "n"(16 * ROW), "n"(24 * ROW)
            : "memory");
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        w[k][0] = (uint32_t)r[2 * k][0], w[k][1] = (uint32_t)r[2 * k][1];
        w[k][2] = (uint32_t)r[2 * k + 1][0], w[k][3] = (uint32_t)r[2 * k + 1][1];
    }
}

// Schedule of NC steps of ND reads of LDS and NM matrix instructions: the reads
// stay AHEAD steps in front (left alone, the compiler reads into few registers
// and waits for every pair).
template <int ND, int NM, int NC, int AHEAD, int C = 0>
__device__ __forceinline__ void read_ahead() {
    if constexpr (C == 0) __builtin_amdgcn_sched_group_barrier(0x100, ND * (AHEAD < NC ? AHEAD : NC), 0);
    if constexpr (C < NC) {
        __builtin_amdgcn_sched_group_barrier(0x008, NM, 0);
        if constexpr (C + AHEAD < NC) __builtin_amdgcn_sched_group_barrier(0x100, ND, 0);
        read_ahead<ND, NM, NC, AHEAD, C + 1>();
    }
}

// The form over a bf16 cache for more than 16 rows: the waves take M rows each,
// and all of them the same keys, which go through an LDS ring by DMA: S stages of
// 32·SUB positions, S − 1 of them on their way while one is used, one barrier a
// stage. No wave has anything to join with another.
// 4 sequences of up to 64 tokens × 4 query heads, 8 key heads, 16384 to 32768
// positions (77 GFLOP, 407 MB): 165 to 184 µs, 420 to 470 TFLOP/s, of which the join
// is 12; the same input again 155 to 160. 2 × 500 prompt tokens, 4 query heads to
// each of 4 key heads, over 1750 to 4000 positions (17 GFLOP) 56 to 62. With two
// workgroups a CU a stage of 64 positions × 128 rows takes 2.0 to 2.4 µs, 900
// TFLOP/s over the card; alone 1.4: each wave's chain of reads, products and
// exponentials, with two waves a SIMD (242 registers a lane; three would have 168). LDS has no conflicts. Besides, 4 to 6 µs pass before the first stage.
// SUB = 2, a barrier for 64 positions, takes 59 for the second and 22.4 for 8 × 64
// rows over 1024 to 2048; SUB = 1 63 and 25.8. No faster were 8 waves with 4 stages
// and one workgroup a CU (63 where 4 waves took 61), the probabilities of one block
// taken up between the products of the other (65, spills), page numbers looked up a
// stage ahead or once for a wave (level).
template <int DP, int M, int QT, int SUB>
__global__ void __launch_bounds__(256, DP == 256 && QT > 1 ? 1 : 2) tree_attention_ring_kernel(TreeAttnArgs a) {
    using Sh = Shape<M>;
    using Acc = typename Sh::Acc;
    constexpr int BR = M * WAVES, NC = DP / Sh::STEP_K, NT = DP / M;
    constexpr int KT = 32 / M, STEPS = 32 / Sh::STEP_K;          // key tiles, steps of P over a stage
    constexpr int E = M == 16 ? 8 : 16;                          // probabilities a lane holds of a stage
    constexpr int TF = 4 / STEPS;                                // dimension tiles of one value_fragments
    constexpr int ROW_CHUNKS = DP / 8, LROWS = 64 / ROW_CHUNKS;  // rows of one wave-wide load
    constexpr int KEYS = 32 * SUB;                               // positions of a stage: SUB blocks of 32
    constexpr int TILE = 32 * DP * 2, BLOCK = 2 * TILE;          // bytes of a block's keys; keys and values
    constexpr int NB = (64 << 10) / BLOCK;                       // blocks the ring holds
    constexpr int S = NB / SUB;
    constexpr int NI = 2 * 32 / LROWS / WAVES;                   // loads of a wave per block
    constexpr int AHEAD = 3;                                     // chunks of the keys read before their products
    // One array, and no library call that has its own (__syncthreads_or): with several
    // the compiler tracks which the DMA writes, and waits for all of it at every read;
    // with one it leaves the waits to wait_stages.
    __shared__ __align__(16) char ring[NB * BLOCK + (TAB + 2) * 8];
    int64_t* const tab = (int64_t*)(ring + NB * BLOCK);

    const WorkItem wi = work_item<BR, KEYS>(a);
    if (wi.tile < 0) return;
    const int tile = wi.tile, split = wi.split, bh = wi.bh, b = bh / a.kv.kv_heads, h = bh - b * a.kv.kv_heads;
    const int64_t begin = (int64_t)split * wi.chunk;
    const int table_row = a.kv.row_of(b), early = first_pages(a, table_row, begin);
    const TileSpan sp = tile_span<BR>(a, b, tile, table_row);
    if (tile * BR >= sp.rows) return;
    const int64_t part = wi.part;
    if (split > 0 && begin >= sp.end) {
        if ((int)threadIdx.x < BR) a.part_ml[part * BR + threadIdx.x] = make_float2(-__builtin_inff(), 0.f);  // nothing to join
        return;
    }
    const int stop = (int)min((int64_t)sp.end, begin + wi.chunk);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane / M, col = lane % M;
    const int r0 = tile * BR + wave * M;
    const bool active = r0 < sp.rows;  // a wave without rows only loads
    const bool in = r0 + col < sp.rows;
    const int r = in ? r0 + col : tile * BR, i_node = a.by_group.div(r), head = h * a.group + r - i_node * a.group;
    const int node = in ? i_node : -1;

    // The row's query, second operand of K·Qᵀ, is asked for before the first page
    // numbers, and taken when both are there. One term is a bf16 query as it is,
    // three are an f32 one's.
    i32x4_t qf[QT][NC];
    PageWindow win = {};
    {
        const auto have = [&](int c) { return in && c * Sh::STEP_K + 8 * g < a.dim; };
        const int64_t at = (sp.start + i_node) * a.q.token + head * a.q.head;
        float x[QT == 1 ? 1 : NC][8];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = have(c) ? c * Sh::STEP_K + 8 * g : 0;
            if constexpr (QT == 1) {
                const uint16_t* p = (const uint16_t*)a.q.data + at + d;
                if (a.q_vec) {
                    qf[0][c] = *(const i32x4_t*)p;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) qf[0][c][e] = p[2 * e] | (p[2 * e + 1] << 16);
                }
            } else {
                const char* row = a.q.data + at * 4;
                if (a.q_vec) load_query<8, false, true>(row, d, x[c]);
                else load_query<8, false, false>(row, d, x[c]);
            }
        }
        if (begin < stop) win = page_window(a, sp, h, 2, (int)begin, stop, tab, early, 0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if constexpr (QT == 1) {
                const int sign = a.flip ? (int)0x80008000u : 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) qf[0][c][e] = have(c) ? qf[0][c][e] ^ sign : 0;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[c][e] = !have(c) ? 0.f : a.flip ? -x[c][e] : x[c][e];
                i32x4_t f[QT];
                fragments<QT>(x[c], f);
#pragma unroll
                for (int q = 0; q < QT; ++q) qf[q][c] = f[q];
            }
        }
    }

    Acc o[NT];
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < Sh::REGS; ++i) o[t][i] = 0.f;

    const int lrow = lane / ROW_CHUNKS, lpos = lane % ROW_CHUNKS;
    const float scale = a.scale;
    for (int ws = (int)begin, window = 0; ws < stop; ++window) {
        if (window) win = page_window(a, sp, h, 2, ws, stop, tab, early, window);
        const int we = win.we;
        const int stages = (we - ws + KEYS - 1) / KEYS;
        // keys, then values of block j: rows of 16-byte chunks, exchanged within a row
        // (the lane that fills a place fetches the chunk that belongs there)
        const auto look_up = [&](int j, int64_t (&off)[NI / 2]) {
#pragma unroll
            for (int n = 0; n < NI / 2; ++n) off[n] = win.offset(a, ws + 32 * j + (n * WAVES + wave) * LROWS + lrow);
        };
        const auto issue = [&](int j, const int64_t (&off)[NI / 2]) {
            char* const st = ring + (j % NB) * BLOCK;
#pragma unroll
            for (int n = 0; n < NI / 2; ++n) {
                const int first = (n * WAVES + wave) * LROWS, key = first + lrow;
                const int ck = lpos ^ key_swizzle<DP>(key), cv = lpos ^ value_swizzle<DP>(key);
                const char* const kp = ck * 8 < a.dim ? a.kv.k + off[n] + ck * 16 : (const char*)&zero_chunk;
                const char* const vp = a.kv.v + off[n] + (cv * 8 < a.dim ? cv * 16 : 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)kp,
                                                 LDS_AS(st + first * DP * 2), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)vp,
                                                 LDS_AS(st + TILE + first * DP * 2), 16, 0, 0);
            }
        };
        // all looked up before the first DMA: the compiler lets a later read of LDS wait for that
        int64_t off[SUB][NI / 2];
#pragma unroll
        for (int j = 0; j < S - 1; ++j)
            if (j < stages) {
#pragma unroll
                for (int n = 0; n < SUB; ++n) look_up(j * SUB + n, off[n]);
#pragma unroll
                for (int n = 0; n < SUB; ++n) issue(j * SUB + n, off[n]);
            }
        MaskWords<SUB> mask = {};
        if (ws + KEYS > sp.full_end) mask.load(a, sp, node, ws - sp.len);
        for (int j = 0; j < stages; ++j) {
            const int kb = ws + KEYS * j;
            // stage j has landed for every wave, and every wave is done with stage j − 1
            wait_stages<NI * SUB, S - 2>(min(S - 2, stages - 1 - j));
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const MaskWords<SUB> mask_now = mask;
            if (kb + 2 * KEYS > sp.full_end) mask.load(a, sp, node, kb + KEYS - sp.len);  // the next stage's
            if (j + S - 1 < stages) {
#pragma unroll
                for (int n = 0; n < SUB; ++n) look_up((j + S - 1) * SUB + n, off[n]);
#pragma unroll
                for (int n = 0; n < SUB; ++n) issue((j + S - 1) * SUB + n, off[n]);
            }
            if (!active) continue;
            const char* const k_lds = ring + (j % S) * (SUB * BLOCK);
            const char* const v_lds = k_lds + TILE;
            // ---- scores ----
            Acc s[SUB][KT];
#pragma unroll
            for (int n = 0; n < SUB * KT; ++n)
#pragma unroll
                for (int i = 0; i < Sh::REGS; ++i) s[n / KT][n % KT][i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int n = 0; n < SUB * KT; ++n) {
                    const int key = M * (n % KT) + col, chunk = c * (Sh::STEP_K / 8) + g;
                    const i32x4_t kf = *(const i32x4_t*)(k_lds + (n / KT) * BLOCK + key * DP * 2 + ((chunk ^ key_swizzle<DP>(key)) * 16));
                    Acc& d = s[n / KT][n % KT];
#pragma unroll
                    for (int q = 0; q < QT; ++q)
                        d = Sh::mma(__builtin_bit_cast(bf16x8_t, kf), __builtin_bit_cast(bf16x8_t, qf[q][c]), d);
                }
            read_ahead<SUB * KT, SUB * KT * QT, NC, AHEAD>();
            float x[SUB][E];  // score, then probability, of key M·(e / REGS) + acc_row(g, e % REGS) of a block
#pragma unroll
            for (int n = 0; n < SUB; ++n)
#pragma unroll
                for (int e = 0; e < E; ++e) x[n][e] = s[n][e / Sh::REGS][e % Sh::REGS];
            // ---- who sees what: most blocks are seen whole by every row ----
            const bool whole = kb + KEYS <= min(we, sp.full_end) && !win.missing;
            uint32_t see[SUB];
#pragma unroll
            for (int n = 0; n < SUB; ++n) {
                see[n] = ~0u;
                if (!whole) {
                    see[n] = mask_now.seen(a, node, kb - sp.len, n) & ~win.holes<32>(a, kb + 32 * n, lane);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (!((see[n] >> (M * (e / Sh::REGS) + acc_row<M>(g, e % Sh::REGS))) & 1u)) x[n][e] = -__builtin_inff();
                }
            }
            // ---- running maximum and sum ----
            float mx = x[0][0];
#pragma unroll
            for (int n = 0; n < SUB; ++n)
#pragma unroll
                for (int e = 0; e < E; ++e) mx = fmaxf(mx, x[n][e]);
            mx = over_column<M>(mx, [](float u, float v) { return fmaxf(u, v); }) * scale;
            if (__any(mx > m)) {
                const float mn = fmaxf(m, mx);
                const float keep = __builtin_amdgcn_exp2f(m - (mn == -__builtin_inff() ? 0.f : mn));
                m = mn;
                l *= keep;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < Sh::REGS; ++i) o[t][i] *= keep;
            }
            const float mu = m == -__builtin_inff() ? 0.f : -m;
            i32x4_t pf[SUB][STEPS][QT];
#pragma unroll
            for (int n = 0; n < SUB; ++n)
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        y[e] = __builtin_amdgcn_exp2f(fmaf(x[n][8 * st + e], scale, mu));
                        l += y[e];
                    }
                    fragments<QT, true>(y, pf[n][st]);
                }
            // ---- output ----
            bool strange = false;
#pragma unroll
            for (int n = 0; n < SUB; ++n)
#pragma unroll
                for (int t = 0; t < NT; t += TF) {
                    uint32_t w[4][4];
                    value_fragments<DP, M>(v_lds + n * BLOCK, t, lane, w);
                    if (!whole && __any(any_nonfinite(w))) {
                        strange = true;
#pragma unroll
                        for (int k = 0; k < 4; ++k) zero_nonfinite(w[k]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        bf16x8_t v;
                        __builtin_memcpy(&v, w[k], 16);
#pragma unroll
                        for (int q = 0; q < QT; ++q)
                            o[t + k / STEPS] = Sh::mma(v, __builtin_bit_cast(bf16x8_t, pf[n][k % STEPS][q]), o[t + k / STEPS]);
                    }
                }
            if (!whole && __any(strange)) {
                // Products took the values that are not finite as zeros. Where a row sees one
                // its sum is the infinity, or NaN of both: products of 0/1 matrices count, per
                // row and dimension, the seen +Inf or NaN and the seen −Inf or NaN.
#pragma unroll
                for (int n = 0; n < SUB; ++n) {
                    bf16x8_t who[STEPS];
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        who[e / 8][e % 8] = (__bf16)((see[n] >> (M * (e / Sh::REGS) + acc_row<M>(g, e % Sh::REGS))) & 1u ? 1.f : 0.f);
#pragma unroll 1
                    for (int sign = 0; sign < 2; ++sign) {
#pragma unroll
                        for (int t = 0; t < NT; t += TF) {
                            uint32_t w[4][4];
                            value_fragments<DP, M>(v_lds + n * BLOCK, t, lane, w);
#pragma unroll
                            for (int u = 0; u < TF; ++u) {
                                Acc count;
#pragma unroll
                                for (int i = 0; i < Sh::REGS; ++i) count[i] = 0.f;
#pragma unroll
                                for (int st = 0; st < STEPS; ++st) {
                                    bf16x8_t v;
                                    infinite_or_nan(w[u * STEPS + st], sign);
                                    __builtin_memcpy(&v, w[u * STEPS + st], 16);
                                    count = Sh::mma(v, who[st], count);
                                }
#pragma unroll
                                for (int i = 0; i < Sh::REGS; ++i)
                                    if (count[i] > 0.f) o[t + u][i] += sign ? -__builtin_inff() : __builtin_inff();
                            }
                        }
                    }
                }
            }
        }
        ws = we;
    }
    if (!active) return;

    l = over_column<M>(l, [](float u, float v) { return u + v; });
    if (!in) return;
    float* po = nullptr;
    int64_t at = 0;
    if (wi.pieces > 1) {
        const int64_t at_row = part * BR + (r - tile * BR);
        if (g == 0) a.part_ml[at_row] = make_float2(m, l);
        po = a.part_o + at_row * a.dim;
    } else {
        at = (sp.start + i_node) * a.y.token + head * a.y.head;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < Sh::REGS; i += 4) {
            const int d = M * t + acc_row<M>(g, i);
            f32x4_t v;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = o[t][i + k];
            if (d >= a.dim) continue;
            if (po) {
                *(f32x4_t*)(po + d) = v;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = l == 0.f ? 0.f : v[k] * inv;
                store_y4(a, at + d, v);
            }
        }
}

// Joins the pieces of a row tile, a wave per row: lanes hold 4 dimensions each,
// and where that leaves lanes over, groups of lanes take the pieces in turn.
// The pieces' maxima and sums come at once, a lane each, and what they weigh is
// asked for 4 at a time. The order of the sum is that of the pieces. Few rows: a
// few dependent reads bound it, 3 µs; many rows: the bytes, 8192 rows of 8 pieces (34 MB) 9 µs.
template <int BR>
__global__ void __launch_bounds__(256) tree_attention_join_kernel(TreeAttnArgs a) {
    const int tile = (int)blockIdx.x % a.row_tiles, bh = (int)blockIdx.x / a.row_tiles;
    const int b = bh / a.kv.kv_heads, h = bh - b * a.kv.kv_heads;
    const int lane = threadIdx.x & 63, rr = blockIdx.y * WAVES + (threadIdx.x >> 6), r = tile * BR + rr;
    const int at_cut = bh * a.row_tiles + tile;
    int4 cut = {at_cut * a.splits, a.splits, 1, 0};
    if (a.slots) cut = a.cuts[at_cut];  // not written for tiles without rows
    const int splits = cut.y;
    const int64_t first = (int64_t)cut.x * BR + rr, step = (int64_t)cut.z * BR;
    float2 own = make_float2(-__builtin_inff(), 0.f);
    if (!a.slots && lane < splits) own = a.part_ml[first + lane * step];
    const int start = a.kv.starts[b], last = min(a.kv.starts[b + 1], a.kv.tokens);
    const int rows = (start < 0 ? 0 : min(max(last - start, 0), a.max_nodes)) * a.group;
    if (r >= rows || splits == 1) return;
    if (a.slots && lane < splits) own = a.part_ml[first + lane * step];
    float top = own.x;
    for (int s = lane + 64; s < splits; s += 64) top = fmaxf(top, a.part_ml[first + s * step].x);
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    const float tu = top == -__builtin_inff() ? 0.f : top;
    const int lanes = a.dim <= 64 ? 16 : a.dim <= 128 ? 32 : 64, groups = 64 / lanes;
    const int d = (lane % lanes) * 4, mine = lane / lanes, dd = d < a.dim ? d : 0;
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 64) {
        if (s0) {
            own = make_float2(-__builtin_inff(), 0.f);
            if (s0 + lane < splits) own = a.part_ml[first + (s0 + lane) * step];
        }
        const float weight = __builtin_amdgcn_exp2f(own.x - tu);
        // NaN counts: a piece is passed over only where it is empty
        const uint64_t some = __ballot(!(own.x == -__builtin_inff() && own.y == 0.f));
        sum += weight * own.y;
        const int n = 64 - (some ? __builtin_clzll(some) : 64);  // pieces up to the last that is not empty
        for (int s = 0; s < n; s += 4 * groups) {
            f32x4_t v[4];
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = s + k * groups + mine;
                const bool take = p < n && ((some >> (p & 63)) & 1);
                w[k] = __shfl(weight, p & 63);
                v[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (take) v[k] = *(const f32x4_t*)(a.part_o + (first + (s0 + p) * step) * a.dim + dd);
                else w[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] += w[k] * v[k][i];
        }
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) sum += xor_partner(sum, off, lane);
    for (int off = lanes; off < 64; off <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += xor_partner(acc[i], off, lane);
    if (mine || d >= a.dim) return;
    const int i_node = a.by_group.div(r), head = h * a.group + r - i_node * a.group;
    const int64_t at = (start + i_node) * a.y.token + head * a.y.head + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = sum == 0.f ? 0.f : acc[i] / sum;
    store_y4(a, at, acc);
}

// How the rows of a key head are laid out: `tile` of them to each wave of a ring
// workgroup, or `tile` that all waves share.
struct Form {
    bool ring;
    int tile;
    int rows() const { return tile * (ring ? WAVES : 1); }
};
// Up to 16 rows share the waves' keys: 64 sequences of 4 rows over 1000 to 2000
// positions take 82 µs, in the ring form (three idle waves) 87; one of 1 row over
// 517 takes 10.6 and 19.0. Up to 64 rows 16 to a wave, more 32: 4 × 256 rows over
// 16384 to 32768 positions take 175 to 179 µs with 32 and 216 with 16, 2 × 2000
// rows over 1750 to 4000 59 and 66. Not so with three-term queries, which do not
// fit the registers beside 32 rows of output (630 rows over 17280 positions: 74 µs
// with 16, 105 with 32), nor with heads past 128. f32 products are bound by the
// matrix units: 32 rows to fetch the keys half as often.
Form form_of(const TreeAttnArgs& a, int cache_dtype) {
    const int rows = a.max_nodes * a.group;
    if (cache_dtype == INGOT_DT_F32) return {false, a.dim > 128 || rows <= 16 ? 16 : 32};
    if (rows <= 16) return {false, 16};
    return {true, !a.q_bf16 || a.dim > 128 || rows <= 16 * WAVES ? 16 : 32};
}

template <int BR>
hipError_t join(const TreeAttnArgs& a, hipStream_t st) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    const int groups = a.kv.batch * a.kv.kv_heads;
    tree_attention_join_kernel<BR><<<dim3((unsigned)(groups * a.row_tiles), BR / WAVES), 256, 0, st>>>(a);
    return hipGetLastError();
}

// Workgroups of the attention: the device-side cut's places, or the items, whole
// rounds over the XCDs in both.
int64_t grid_of(const TreeAttnArgs& a) {
    if (a.slots) return (a.slots + 7) / 8 * 8;
    return (a.items / a.row_tiles + 7) / 8 * 8 * (int64_t)a.row_tiles;
}

template <typename T, int DP, int QT>
hipError_t launch(const TreeAttnArgs& a, const Form& f, hipStream_t st) {
    const unsigned grid = (unsigned)grid_of(a);
    if constexpr (sizeof(T) == 2) {
        if (f.ring) {
            if constexpr (DP <= 128 && QT == 1)
                if (f.tile == 32) {
                    tree_attention_ring_kernel<DP, 32, QT, 2><<<grid, 256, 0, st>>>(a);
                    return join<32 * WAVES>(a, st);
                }
            tree_attention_ring_kernel<DP, 16, QT, DP <= 128 ? 2 : 1><<<grid, 256, 0, st>>>(a);
            return join<16 * WAVES>(a, st);
        }
    } else if constexpr (DP <= 128) {
        if (f.tile == 32) {
            tree_attention_kernel<T, DP, 2, QT><<<grid, 256, 0, st>>>(a);
            return join<32>(a, st);
        }
    }
    tree_attention_kernel<T, DP, 1, QT><<<grid, 256, 0, st>>>(a);
    return join<16>(a, st);
}

size_t cuts_bytes(const TreeAttnArgs& a) {
    return a.slots ? (size_t)a.kv.batch * a.kv.kv_heads * a.row_tiles * sizeof(int4) : 0;
}

}  // namespace

size_t plan_tree_attention(TreeAttnArgs& a, int cache_dtype, int num_cus) {
    const Form f = form_of(a, cache_dtype);
    const int br = f.rows();
    const int64_t rows = (int64_t)a.max_nodes * a.group;
    const int64_t tiles = (rows + br - 1) / br, base = tiles * a.kv.batch * a.kv.kv_heads;
    a.items = 0;
    if (base > kLaunchWorkgroups) return 0;
    a.row_tiles = (int32_t)tiles;
    // Two workgroups a CU are what the card holds at once of the forms of up to 128
    // dimensions (but f32 keys with 32 rows) and of the ring of bf16 queries past that:
    // 4 × 256 rows over 16384 to 32768 positions take 175 to 179 µs in so many pieces,
    // 203 in half as many, 189 in twice as many; 2 × 2000 rows over 1750 to 4000 59, 64
    // and 68. The others hold one, and their pieces run in twice the rounds counted here.
    const int64_t slots = 2 * (int64_t)num_cus;
    // The shortest piece worth its partial results and its start: 128 positions for
    // shared rows (one token over 517: 10.6 µs, with 256 12.3), 8 to a row in the ring
    // form (8 × 64 rows over 1024 to 2048: 512; 256 take as long and join twice the parts).
    const int64_t least = f.ring ? 8 * br : STEP;
    const int64_t most = (a.max_tokens + least - 1) / least;
    // Pieces for one to four rounds of places, whichever takes least: a round costs a
    // piece's positions, a start of about 256 and the part's bytes (3 positions a
    // row); half a round or less, one workgroup a CU, 0.65 of that. 692 f32 rows
    // over 15617 positions of an f32 cache (176 tiles): 208 µs, in one round 265;
    // 9 × 512 rows over 8192 (288 tiles) 203 and 223.
    const auto cost = [&](int64_t n) {
        const int64_t rest = base * n % slots, rounds = base * n / slots * 20 + (!rest ? 0 : 2 * rest <= slots ? 13 : 20);
        return rounds * (256 + (n > 1 ? 3 * br : 0) + a.max_tokens / n);
    };
    int64_t splits = 1;
    for (int rounds = 1; rounds <= 4; ++rounds) {
        const int64_t n = std::min(most, rounds * slots / base);
        if (n > 1 && cost(n) < cost(splits)) splits = n;
    }
    a.chunk = (int32_t)std::min<int64_t>(0x3FFFFF80, ((a.max_tokens + splits - 1) / splits + STEP - 1) / STEP * STEP);
    a.splits = (int32_t)std::max<int64_t>(1, ((int64_t)a.max_tokens + a.chunk - 1) / a.chunk);
    a.items = (int32_t)(base * a.splits);
    // Long pieces of several sequences (a lane each) are cut by the lengths, which the
    // device knows: 4 × 256 rows over 16384 to 32768 positions 175 to 179 µs, by
    // max_tokens 191; 2 × 2000 rows over 1750 to 4000 level. It takes a workgroup 1 to
    // 2 µs, as long as a block of positions, so pieces up to 512 stay as they are;
    // and it counts on half the places being enough for the tiles.
    a.slots = 0;
    if (a.splits > 1 && 2 * base <= slots && a.kv.batch > 1 && a.kv.batch <= 64 && a.chunk > LONG) {
        a.slots = a.items = (int32_t)slots;
        a.chunk = LONG;
    }
    if (grid_of(a) > kLaunchWorkgroups) {
        a.items = 0;
        return 0;
    }
    return a.splits == 1 ? 0 : cuts_bytes(a) + (size_t)a.items * br * (a.dim + 2) * sizeof(float);
}

void place_tree_attention(TreeAttnArgs& a, int cache_dtype, void* ws) {
    a.cuts = (int4*)ws;
    a.part_o = (float*)((char*)ws + cuts_bytes(a));
    a.part_ml = (float2*)(a.part_o + (size_t)a.items * form_of(a, cache_dtype).rows() * a.dim);
}

hipError_t launch_tree_attention(const TreeAttnArgs& a, int cache_dtype, hipStream_t st) {
    const Form f = form_of(a, cache_dtype);
    const auto by_dim = [&](auto type, auto qt) {
        using T = decltype(type);
        constexpr int QT = decltype(qt)::value;
        if (a.dim <= 64) return launch<T, 64, QT>(a, f, st);
        if (a.dim <= 128) return launch<T, 128, QT>(a, f, st);
        return launch<T, 256, QT>(a, f, st);
    };
    if (cache_dtype == INGOT_DT_F32) return by_dim(float{}, std::integral_constant<int, 1>{});
    if (a.q_bf16) return by_dim(uint16_t{}, std::integral_constant<int, 1>{});
    return by_dim(uint16_t{}, std::integral_constant<int, 3>{});
}

}  // namespace ingot
