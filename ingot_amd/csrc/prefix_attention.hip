// Attention of sequences that share a prefix: the prefix' keys and values are read
// once for all new tokens of a group, the rest of each sequence as ever, and the
// two are joined.
//
// A softmax over two sets of positions is that of each with its maximum m and sum l
// kept, weighed together: with o the sums of p·v, the whole is
//   (e^(m1 − m)·o1 + e^(m2 − m)·o2) / (e^(m1 − m)·l1 + e^(m2 − m)·l2).
// So the tokens of a group (they follow each other in the call) are one run of rows
// over the prefix, with the kernels of tree_attention.hpp; with 32 sequences of 4
// query heads a tile of 128 rows reads each key once where each sequence alone would
// read it for 4. Probabilities of bf16 queries are rounded to bf16 as in
// tree_attention.hpp, once in each of the two sets.
//
// Launches: one workgroup works out the spans (a group and its prefix, a sequence
// and its rest) and cuts them into pieces by their lengths, which only the device
// knows; the attention over all of them, prefixes first, by whichever form of the
// kernel suits the rows of each; the join.
//
// Times: 32 single bf16 tokens over up to 4096 shared and 300 own positions, 32 heads
// on 8 of 128 (43 MB) 27 µs, of which the plan is 4 and the join 5 to 6 (each alone 49);
// 128 in two groups over up to 32768 and 600 (440 MB, 52 GFLOP) 120 to 136 µs, the
// attention 126 under the profiler, 3.5 TB/s of what it needs, where a copy moves 4.7
// (each alone 954).

#include <cmath>

#include "tree_attention.hpp"

namespace ingot {

namespace {

constexpr int PLAN = 512;     // threads of the planning workgroup
constexpr int PLANW = PLAN / 64;

// Exclusive sums of two counts (see counted) over the workgroup's threads, each at most
// 64 + PLANW of them, and the wholes as counts.
__device__ __forceinline__ int2 block_scan(int2 v, int2 room, int2* part, int2* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int2 upto = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int x = __shfl_up(upto.x, off), y = __shfl_up(upto.y, off);
        if (lane >= off) upto.x += x, upto.y += y;
    }
    if (lane == 63) part[wave] = make_int2(counted(upto.x, room.x), counted(upto.y, room.y));
    __syncthreads();
    int2 before = {0, 0}, sum = {0, 0};
#pragma unroll
    for (int w = 0; w < PLANW; ++w) {
        if (w < wave) before.x += part[w].x, before.y += part[w].y;
        sum.x += part[w].x, sum.y += part[w].y;
    }
    __syncthreads();
    *all = make_int2(counted(sum.x, room.x), counted(sum.y, room.y));
    return make_int2(before.x + upto.x - v.x, before.y + upto.y - v.y);
}

// The spans of a call and their cut into pieces of one length but for rounding. A
// chain of four dependent reads and as many barriers: 4 to 6 µs. Up to PLAN spans
// stay in LDS.
__global__ void __launch_bounds__(PLAN) prefix_plan_kernel(PrefixArgs a) {
    __shared__ int firsts[PLAN + 1];
    __shared__ AttnSpan held[PLAN];
    __shared__ float sums[PLANW][64];
    __shared__ float2 totals[PLANW];
    __shared__ int2 part[PLANW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int seqs = a.t.kv.batch, groups = a.prefix.count, all = groups + seqs, heads = a.t.kv.kv_heads;
    const bool fits = all <= PLAN;
    AttnSpan* const spans = fits ? held : a.prefix.spans;  // the rests' follow the prefixes'
    const int* const first = fits ? firsts : a.first;
    if (fits) {
        if (tid <= groups) firsts[tid] = a.first[tid];
        __syncthreads();
    }
    const auto tokens_of = [&](int from, int to, int most, int* start) {
        *start = a.t.kv.starts[from];
        const int last = min(a.t.kv.starts[to], a.t.kv.tokens);
        return *start < 0 ? 0 : min(max(last - *start, 0), most);
    };
    const auto weight_of = [&](const AttnSpan& s, int* len) {  // workgroups to a piece, and the positions
        *len = max(s.end - s.begin, 0);
        return *len ? s.tiles * heads : 0;
    };
    float2 sum = {0.f, 0.f};  // work, weights
    for (int i = tid; i < all; i += PLAN) {
        AttnSpan s = {};
        s.group = -1;
        if (i < groups) {
            const int s0 = min(max(first[i], 0), seqs), s1 = min(max(first[i + 1], 0), seqs);
            if (s0 < s1) {
                s.rows = tokens_of(s0, s1, a.t.kv.tokens, &s.start) * a.t.group;
                const int common = min(max(a.shared[i], 0), a.max_shared);
                // the first row that holds them: sequences that have ended may lead the group
                s.row = -1;
                for (int b = s0; b < s1 && s.row < 0; ++b) {
                    const int row = a.t.kv.row_of(b);
                    if (row >= 0 && a.t.kv.len[row] >= common) s.row = row;
                }
                s.end = s.len = s.row < 0 ? 0 : common;
            }
            s.tiles = (int)(((int64_t)s.rows + (1 << a.prefix.rows_log) - 1) >> a.prefix.rows_log);
        } else {
            const int b = i - groups;
            const int n = tokens_of(b, b + 1, a.t.max_nodes, &s.start);
            s.row = a.t.kv.row_of(b);
            s.rows = n * a.t.group;
            s.len = s.row < 0 ? 0 : max(0, a.t.kv.len[s.row]);
            s.end = s.row < 0 ? 0 : (int)min((int64_t)s.len + n, (int64_t)a.t.max_tokens);
            s.tiles = (int)(((int64_t)s.rows + (1 << a.rest.rows_log) - 1) >> a.rest.rows_log);
            // the group: the last with first[g] <= b, if b is in it; tokens without a row of the
            // table see nothing, no prefix either
            int lo = 0, hi = groups;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= b) lo = mid; else hi = mid;
            }
            if (s.row >= 0 && first[lo] >= 0 && first[lo] <= b && b < first[lo + 1]) {
                s.group = lo;
                s.begin = min(max(a.shared[lo], 0), a.max_shared);
                if (s.begin > min(s.len, s.end)) s.begin = s.end;  // the row holds less: nothing of its own
            }
        }
        int len;
        const int w = weight_of(s, &len);
        sum.x += (float)w * (float)len;
        sum.y += (float)w;
        spans[i] = s;
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) sum.x += xor_partner(sum.x, off, lane), sum.y += xor_partner(sum.y, off, lane);
    if (lane == 0) totals[wave] = sum;
    __syncthreads();
    sum = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < PLANW; ++w) sum.x += totals[w].x, sum.y += totals[w].y;
    const float slots = (float)a.slots, low = fmaxf((float)a.least, sum.x / slots);
    float per = 1.f / low;  // pieces to a position
    if (2.f * sum.y <= slots) {
        // each lane tries a length, from the shortest there could be to one at which the
        // pieces, at most work / length + weights, are few enough in any case
        const float high = fmaxf(low, 1.001f * sum.x / (slots - sum.y));
        const float mine = 1.f / (low + (high - low) * (float)lane * (1.f / 63.f));
        float n = 0.f;
        for (int i = wave; i < all; i += PLANW) {
            int len;
            const int w = weight_of(spans[i], &len);
            n += (float)w * (float)((int)((float)max(len - 1, 0) * mine) + 1);
        }
        sums[wave][lane] = n;
        __syncthreads();
        n = 0.f;
#pragma unroll
        for (int w = 0; w < PLANW; ++w) n += sums[w][lane];
        const uint64_t few = __ballot(n <= slots);
        per = few ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), __builtin_ctzll(few))) : 0.f;
    }
    const int2 room = make_int2(a.prefix.room, a.rest.room);
    int2 base = {0, 0};
    for (int i0 = 0; i0 < all; i0 += PLAN) {
        const int i = i0 + tid;
        AttnSpan s = {};
        if (i < all) s = spans[i];
        int len;
        const int w = weight_of(s, &len);
        if (w) {
            s.pieces = (int)((float)(len - 1) * per) + 1;
            s.chunk = ((len + s.pieces - 1) / s.pieces + a.step - 1) / a.step * a.step;
            s.pieces = (len + s.chunk - 1) / s.chunk;
        }
        const int items = counted((int64_t)w * s.pieces, i < groups ? room.x : room.y);
        int2 whole;
        const int2 before = block_scan(i < groups ? make_int2(items, 0) : make_int2(0, items), room, part, &whole);
        s.item0 = i < groups ? base.x + before.x : base.y + before.y;
        if (i < all) {
            // spans past the room for parts (only starts or groups that do not rise make such)
            // get none; their first items, and all after them, are past it too
            if (s.item0 + items > (i < groups ? room.x : room.y)) s.pieces = s.rows = 0;
            a.prefix.spans[i] = s;
            a.prefix.item0[i] = s.item0;
        }
        base.x = counted(base.x + whole.x, room.x);
        base.y = counted(base.y + whole.y, room.y);
    }
    if (tid == 0) a.totals[0] = min(base.x, room.x), a.totals[1] = min(base.y, room.y);
}

// The first 64 spans' first items, a lane each, asked for before the item is known.
__device__ __forceinline__ int early_items(const PrefixList& l) {
    const int lane = threadIdx.x & 63;
    return lane < l.count ? l.item0[lane] : 0x7FFFFFFF;
}
// The span of an item of a list: the last whose items begin at or before it.
__device__ __forceinline__ int span_of(const PrefixList& l, int item, int early) {
    const int n = l.count <= 64 ? __builtin_popcountll(__ballot(early <= item)) : count_at_most(l.item0, l.count, item);
    return __builtin_amdgcn_readfirstlane(n - 1);
}

// Items of the prefixes, then of the rests, each list going to the 8 XCDs in runs
// (items are numbered by span, piece, key head and row tile, so row tiles that read
// the same keys share an L2). Prefixes are work for the matrix units, rests for the
// memory: in one launch they run beside each other.
template <typename P, typename R>
__global__ void __launch_bounds__(256, (P::WGS < R::WGS ? P::WGS : R::WGS)) prefix_attention_kernel(PrefixArgs a) {
    __shared__ __align__(16) char lds[P::LDS > R::LDS ? P::LDS : R::LDS];
    const int xcd = blockIdx.x & 7, turn = blockIdx.x >> 3;
    const int early_prefix = early_items(a.prefix), early_rest = early_items(a.rest);
    const int of_prefix = a.totals[0], of_rest = a.totals[1], turns = (of_prefix + 7) >> 3, rest_turns = (of_rest + 7) >> 3;
    if (turn < turns) {
        const int item = xcd * turns + turn;
        if (item >= of_prefix) return;
        TreeAttnArgs t = a.t;
        t.mask = nullptr;  // every row sees all of its prefix
        t.part_o = a.prefix.part_o;
        t.part_ml = a.prefix.part_ml;
        const Piece pc = piece_of_span<P::BR>(t, a.prefix.spans[span_of(a.prefix, item, early_prefix)], item);
        P::run(t, pc, lds);
        return;
    }
    const int item = xcd * rest_turns + turn - turns;
    if (turn - turns >= rest_turns || item >= of_rest) return;
    TreeAttnArgs t = a.t;
    t.part_o = a.rest.part_o;
    t.part_ml = a.rest.part_ml;
    const Piece pc = piece_of_span<R::BR>(t, a.rest.spans[span_of(a.rest, item, early_rest)], item);
    R::run(t, pc, lds);
}

// Joins the pieces of a row's prefix and rest, a wave to a row (a token's head):
// lanes hold 4 dimensions each, and where that leaves lanes over, groups of lanes
// take the pieces in turn; the pieces' maxima and sums come at once, a lane each.
// Few rows: a chain of dependent reads (starts, spans, sums, parts), 4 to 5 µs; 4096
// rows of 11 pieces (25 MB) 9 µs.
__global__ void __launch_bounds__(256) prefix_join_kernel(PrefixArgs a, FastDiv by_heads, int rows) {
    const int lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6);
    const TreeAttnArgs& y = a.t;
    const int t = by_heads.div(min(at, rows - 1)), head = min(at, rows - 1) - t * by_heads.d;
    const int b = count_at_most(y.kv.starts + 1, y.kv.batch, t);
    if (at >= rows || b >= y.kv.batch) return;
    const AttnSpan& rest = a.rest.spans[__builtin_amdgcn_readfirstlane(b)];
    const int h = y.by_group.div(head), in_group = head - h * y.group;
    const int64_t r = (int64_t)(t - rest.start) * y.group + in_group;
    if (t < rest.start || r >= rest.rows) return;
    // piece p of the row is at p steps from these, the prefix' pieces first
    const int64_t rest_step = (int64_t)(rest.tiles * y.kv.kv_heads) << a.rest.rows_log;
    const int64_t rest_at = ((int64_t)(rest.item0 + h * rest.tiles) << a.rest.rows_log) + r;
    int64_t step = 0, from = 0;
    int before = 0;
    if (rest.group >= 0) {
        const AttnSpan& prefix = a.prefix.spans[rest.group];
        const int64_t rp = (int64_t)(t - prefix.start) * y.group + in_group;
        if (t >= prefix.start && rp < prefix.rows) before = prefix.pieces;
        step = (int64_t)(prefix.tiles * y.kv.kv_heads) << a.prefix.rows_log;
        from = ((int64_t)(prefix.item0 + h * prefix.tiles) << a.prefix.rows_log) + rp;
    }
    const int pieces = before + rest.pieces;
    const auto place = [&](int p) { return p < before ? from + p * step : rest_at + (p - before) * rest_step; };
    const auto ml = [&](int p) { return (p < before ? a.prefix.part_ml : a.rest.part_ml)[place(p)]; };
    const int lanes = y.dim <= 64 ? 16 : y.dim <= 128 ? 32 : 64, turns = 64 / lanes;
    const int d = (lane % lanes) * 4, mine = lane / lanes, dd = d < y.dim ? d : 0;
    float2 own = make_float2(-__builtin_inff(), 0.f);
    if (lane < pieces) own = ml(lane);
    float top = own.x;
    for (int p = lane + 64; p < pieces; p += 64) top = fmaxf(top, ml(p).x);
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    const float tu = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < pieces; p0 += 64) {
        if (p0) {
            own = make_float2(-__builtin_inff(), 0.f);
            if (p0 + lane < pieces) own = ml(p0 + lane);
        }
        const float weight = __builtin_amdgcn_exp2f(own.x - tu);
        // NaN counts: a piece is passed over only where it is empty
        const uint64_t some = __ballot(!(own.x == -__builtin_inff() && own.y == 0.f));
        sum += weight * own.y;
        const int n = 64 - (some ? __builtin_clzll(some) : 64);
        for (int s = 0; s < n; s += 4 * turns) {
            f32x4_t v[4];
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = s + k * turns + mine;
                const bool take = p < n && ((some >> (p & 63)) & 1);
                w[k] = __shfl(weight, p & 63);
                v[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (take) v[k] = *(const f32x4_t*)((p0 + p < before ? a.prefix.part_o : a.rest.part_o) + place(p0 + p) * y.dim + dd);
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
    if (mine || d >= y.dim) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = sum == 0.f ? 0.f : acc[i] / sum;
    store_y4(y, (int64_t)t * y.y.token + (int64_t)head * y.y.head + d, acc);
}

size_t align16(size_t n) { return (n + 15) & ~(size_t)15; }

// Forms of the two lists: the rows of a group by its share of the tokens, and no
// smaller tiles than the rests have.
struct Forms {
    Form prefix, rest;
};
Forms forms_of(const PrefixArgs& a, int cache_dtype) {
    TreeAttnArgs t = a.t;
    const Form rest = form_of(t, cache_dtype);
    t.max_nodes = (t.kv.tokens + a.prefix.count - 1) / a.prefix.count;
    const Form prefix = form_of(t, cache_dtype);
    return {prefix.rows() < rest.rows() ? rest : prefix, rest};
}

}  // namespace

// Reading a prefix once saves bytes, and products where the rows of one sequence leave
// tiles empty, and costs two more dependent launches. Expected µs: alone 10 and the
// bytes at 7 TB/s (sequences that read the same pages partly find them in the caches),
// with prefixes 19 and the bytes at 4.7; or the products' time, if that is longer.
// Taken where it is a tenth less, and not asked where the host does not know how much is
// shared at most. Every sequence is taken to be in a group. Alone and with prefixes,
// single bf16 tokens of 200 positions of their own, 32 heads on 8 of 128: 4 sequences over 4096 17 and 22, 8 28
// and 22, 16 38 and 24, 32 48 and 27; 16 over 1024 17 and 21, 32 25 and 25. 9 × 3
// tokens on an f32 cache (3 groups of 1500, 12 heads of 80) 31 and 26; 24 trees of 16
// f32 tokens over bf16 (5 groups of 3000), bound by the products, 70 and 80.
bool prefix_pays(const PrefixArgs& a, int cache_dtype) {
    const TreeAttnArgs& t = a.t;
    const bool f32 = cache_dtype == INGOT_DT_F32;
    const double own = std::max(t.max_tokens - a.max_shared, 0), groups = a.prefix.count, batch = t.kv.batch;
    const double position = 2.0 * t.kv.kv_heads * t.dim * (f32 ? 4 : 2);  // bytes
    const auto padded = [](double rows) { return 16.0 * std::ceil(rows / 16.0); };
    const double rows = batch * padded((double)t.max_nodes * t.group);
    const double rows_once = groups * padded((double)t.kv.tokens * t.group / groups);
    const double width = t.dim <= 64 ? 64 : t.dim <= 128 ? 128 : 256;
    const double per_row = 4.0 * t.kv.kv_heads * width / (f32 ? 60e6 : t.q_bf16 ? 900e6 : 300e6);  // µs a position
    const double alone = 10.0 + std::max(batch * t.max_tokens * position / 7e6, rows * t.max_tokens * per_row);
    const double once = 19.0 + std::max((groups * a.max_shared + batch * own) * position / 4.7e6,
                                        (rows_once * a.max_shared + rows * own) * per_row);
    return once < 0.9 * alone;
}

size_t plan_prefix_attention(PrefixArgs& a, int cache_dtype, int num_cus) {
    const Forms f = forms_of(a, cache_dtype);
    const int64_t rows = (int64_t)a.t.kv.tokens * a.t.group;
    // what the card holds at once of most forms; of f32 keys with 32 rows, and past 128
    // dimensions of the few-rows form and the ring of three terms, it holds one workgroup a
    // CU, and their pieces run in two rounds
    a.slots = 2 * num_cus;
    a.rest.count = a.t.kv.batch;
    a.step = f.prefix.ring && f.rest.ring ? 64 : STEP;
    a.least = f.prefix.ring ? 256 : STEP;
    int64_t grid = 0;
    const auto fill = [&](PrefixList& l, const Form& form) {
        l.rows_log = 0;
        while ((1 << l.rows_log) < form.rows()) ++l.rows_log;
        // pieces of at least work / slots positions are at most a piece a tile and `slots`
        // more (and a few for the roundings of f32 sums)
        const int64_t tiles = (rows / form.rows() + l.count) * a.t.kv.kv_heads, room = tiles + a.slots + 64;
        grid += room + 8;
        l.room = (int32_t)std::min<int64_t>(room, kLaunchWorkgroups);
    };
    fill(a.prefix, f.prefix);
    fill(a.rest, f.rest);
    if (grid > kLaunchWorkgroups - 8 || rows > (1 << 28) || (int64_t)a.t.kv.tokens * a.t.heads > 4 * kLaunchWorkgroups) return 0;
    const size_t spans = (size_t)a.prefix.count + a.rest.count;
    const auto parts = [&](const PrefixList& l) { return align16(((size_t)l.room << l.rows_log) * (a.t.dim + 2) * sizeof(float)); };
    return 16 + align16(spans * sizeof(AttnSpan)) + align16(spans * sizeof(int32_t)) + parts(a.prefix) + parts(a.rest);
}

hipError_t launch_prefix_attention(PrefixArgs& a, int cache_dtype, void* ws, hipStream_t st) {
    char* p = (char*)ws;
    const size_t spans = (size_t)a.prefix.count + a.rest.count;
    a.totals = (int32_t*)p;
    p += 16;
    a.prefix.spans = (AttnSpan*)p;
    a.rest.spans = a.prefix.spans + a.prefix.count;
    p += align16(spans * sizeof(AttnSpan));
    a.prefix.item0 = (int32_t*)p;
    a.rest.item0 = a.prefix.item0 + a.prefix.count;
    p += align16(spans * sizeof(int32_t));
    for (PrefixList* l : {&a.prefix, &a.rest}) {
        l->part_o = (float*)p;
        l->part_ml = (float2*)(l->part_o + ((size_t)l->room << l->rows_log) * a.t.dim);
        p += align16(((size_t)l->room << l->rows_log) * (a.t.dim + 2) * sizeof(float));
    }
    prefix_plan_kernel<<<1, PLAN, 0, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const Forms f = forms_of(a, cache_dtype);
    const unsigned grid = (unsigned)(((int64_t)a.prefix.room + 7) / 8 * 8 + ((int64_t)a.rest.room + 7) / 8 * 8);
    e = by_types(a.t, cache_dtype, [&](auto type, auto dim, auto qt) {
        using T = decltype(type);
        constexpr int DP = decltype(dim)::value, QT = decltype(qt)::value;
        using Few = FewRows<T, DP, 1, QT>;
        if constexpr (sizeof(T) == 2) {
            using Ring = RingRows<DP, 16, QT, DP <= 128 ? 2 : 1>;
            if constexpr (DP <= 128 && QT == 1) {
                using Wide = RingRows<DP, 32, QT, 2>;
                if (f.prefix.tile == 32) {
                    if (!f.rest.ring) prefix_attention_kernel<Wide, Few><<<grid, 256, 0, st>>>(a);
                    else if (f.rest.tile == 16) prefix_attention_kernel<Wide, Ring><<<grid, 256, 0, st>>>(a);
                    else prefix_attention_kernel<Wide, Wide><<<grid, 256, 0, st>>>(a);
                    return;
                }
            }
            if (f.rest.ring) prefix_attention_kernel<Ring, Ring><<<grid, 256, 0, st>>>(a);
            else if (f.prefix.ring) prefix_attention_kernel<Ring, Few><<<grid, 256, 0, st>>>(a);
            else prefix_attention_kernel<Few, Few><<<grid, 256, 0, st>>>(a);
        } else {
            if constexpr (DP <= 128) {
                using Two = FewRows<T, DP, 2, QT>;
                if (f.prefix.tile == 32) {
                    if (f.rest.tile == 16) prefix_attention_kernel<Two, Few><<<grid, 256, 0, st>>>(a);
                    else prefix_attention_kernel<Two, Two><<<grid, 256, 0, st>>>(a);
                    return;
                }
            }
            prefix_attention_kernel<Few, Few><<<grid, 256, 0, st>>>(a);
        }
    });
    if (e != hipSuccess) return e;
    const int rows = a.t.kv.tokens * a.t.heads;
    prefix_join_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a, FastDiv(a.t.heads), rows);
    return hipGetLastError();
}

}  // namespace ingot
