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
// read it for 4.
//
// Launches: one workgroup works out the spans (a group and its prefix, a sequence
// and its rest) and cuts them into pieces by their lengths, which only the device
// knows; the attention over the prefixes; the attention over the rests; the join.

#include "tree_attention.hpp"

namespace ingot {

namespace {

constexpr int PLAN = 1024;  // threads of the planning workgroup

// Exclusive sum over the workgroup's threads, and the whole in *all.
__device__ __forceinline__ int block_scan(int v, int* part, int* all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(upto, off);
        if (lane >= off) upto += u;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < PLAN / 64; ++w) {
        if (w < wave) before += part[w];
        sum += part[w];
    }
    __syncthreads();
    *all = sum;
    return before + upto - v;
}

// Cuts a list of spans into pieces of one length (but for rounding), as short as
// the workgroups that the card holds at once allow, and numbers them. Spans that
// do not fit the room for parts (starts that do not rise) get none.
__device__ __forceinline__ void cut_spans(const PrefixArgs& a, const PrefixList& l, float2* held, float (*sums)[64], int* part) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // lengths and weights (workgroups to a piece) of the spans
    float work = 0.f, weights = 0.f;
    for (int s = tid; s < l.count; s += PLAN) {
        const AttnSpan& sp = l.spans[s];
        const int len = max(sp.end - sp.begin, 0), w = len ? sp.tiles * a.kv.kv_heads : 0;
        work += (float)w * (float)len;
        weights += (float)w;
        if (s < PLAN) held[s] = make_float2((float)(len - 1), (float)w);
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) work += xor_partner(work, off, lane), weights += xor_partner(weights, off, lane);
    if (lane == 0) sums[0][wave] = work, sums[1][wave] = weights;
    __syncthreads();
    work = weights = 0.f;
#pragma unroll
    for (int w = 0; w < PLAN / 64; ++w) work += sums[0][w], weights += sums[1][w];
    __syncthreads();
    // each lane tries a length, from the shortest there could be to one at which the
    // pieces, at most work / length + weights, are few enough in any case
    const float slots = (float)a.slots;
    float per = 0.f;  // pieces to a position
    if (weights < slots && l.count <= PLAN) {
        const float low = fmaxf((float)l.least, work / slots), high = fmaxf(low, 1.001f * work / (slots - weights));
        const float mine = 1.f / (low + (high - low) * (float)lane * (1.f / 63.f));
        float sum = 0.f;
        for (int s = wave; s < l.count; s += PLAN / 64) sum += held[s].y * (float)((int)(fmaxf(held[s].x, 0.f) * mine) + 1);
        sums[wave][lane] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < PLAN / 64; ++w) sum += sums[w][lane];
        const uint64_t fits = __ballot(sum <= slots);
        if (fits) per = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), __builtin_ctzll(fits)));
        __syncthreads();
    }
    int base = 0;
    for (int s0 = 0; s0 < l.count; s0 += PLAN) {
        const int s = s0 + tid;
        int items = 0, len = 0, pieces = 0, chunk = 0, tiles = 0;
        if (s < l.count) {
            const AttnSpan& sp = l.spans[s];
            len = max(sp.end - sp.begin, 0);
            tiles = sp.tiles;
            if (len && tiles) {
                pieces = (int)((float)(len - 1) * per) + 1;
                chunk = ((len + pieces - 1) / pieces + l.step - 1) / l.step * l.step;
                pieces = (len + chunk - 1) / chunk;
                items = tiles * a.kv.kv_heads * pieces;
            }
        }
        int all;
        const int at = base + block_scan(items, part, &all);
        if (s < l.count) {
            AttnSpan& sp = l.spans[s];
            if (at + items > l.room) pieces = 0, sp.rows = 0;
            sp.pieces = pieces;
            sp.chunk = chunk;
            sp.item0 = at;
            l.item0[s] = at;
        }
        base += all;
    }
    if (tid == 0) *l.total = min(base, l.room);
}

__global__ void __launch_bounds__(PLAN) prefix_plan_kernel(PrefixArgs a) {
    __shared__ float2 held[PLAN];
    __shared__ float sums[PLAN / 64][64];
    __shared__ int part[PLAN / 64];
    const int tid = threadIdx.x, seqs = a.kv.batch;
    const auto tokens_of = [&](int from, int to, int most, int* start) {
        *start = a.kv.starts[from];
        const int last = min(a.kv.starts[to], a.kv.tokens);
        return *start < 0 ? 0 : min(max(last - *start, 0), most);
    };
    for (int g = tid; g < a.groups; g += PLAN) {
        const int s0 = min(max(a.first[g], 0), seqs), s1 = min(max(a.first[g + 1], 0), seqs);
        AttnSpan sp = {};
        if (s0 < s1) {
            const int n = tokens_of(s0, s1, a.kv.tokens, &sp.start);
            sp.row = a.kv.row_of(s0);
            sp.rows = n * a.group;
            sp.tiles = (sp.rows + a.prefix.rows - 1) / a.prefix.rows;
            sp.end = sp.len = sp.row < 0 ? 0 : min(max(a.shared[g], 0), a.max_shared);
        }
        a.prefix.spans[g] = sp;
    }
    for (int b = tid; b < seqs; b += PLAN) {
        AttnSpan sp = {};
        const int n = tokens_of(b, b + 1, a.max_nodes, &sp.start);
        sp.row = a.kv.row_of(b);
        sp.rows = n * a.group;
        sp.tiles = (sp.rows + a.rest.rows - 1) / a.rest.rows;
        sp.len = sp.row < 0 ? 0 : max(0, a.kv.len[sp.row]);
        sp.end = sp.row < 0 ? 0 : (int)min((int64_t)sp.len + n, (int64_t)a.max_tokens);
        // the group: the last g with first[g] <= b, if b is in it
        int lo = 0, hi = a.groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.first[mid] <= b) lo = mid; else hi = mid;
        }
        const bool in = a.groups && a.first[lo] >= 0 && a.first[lo] <= b && b < a.first[lo + 1];
        sp.begin = in ? min(max(a.shared[lo], 0), a.max_shared) : 0;
        if (sp.begin > min(sp.len, sp.end)) sp.begin = sp.end;  // the row holds less: nothing of its own
        a.group_of[b] = in ? lo : -1;
        a.rest.spans[b] = sp;
    }
    __syncthreads();
    cut_spans(a, a.prefix, held, sums, part);
    __syncthreads();
    cut_spans(a, a.rest, held, sums, part);
}

// Joins the pieces of a row's prefix and rest, a wave to a row (a token's head):
// lanes hold 4 dimensions each, and where that leaves lanes over, groups of lanes
// take the pieces in turn; the pieces' maxima and sums come at once, a lane each.
__global__ void __launch_bounds__(256) prefix_join_kernel(PrefixArgs a, TreeAttnArgs y, FastDiv by_heads, int rows) {
    const int lane = threadIdx.x & 63, at = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = by_heads.div(min(at, rows - 1)), head = min(at, rows - 1) - t * by_heads.d;
    int b = 0;
    for (int s = 0; s < a.kv.batch; s += 64)
        b += __builtin_popcountll(__ballot(s + lane < a.kv.batch && a.kv.starts[s + lane + 1] <= t));
    if (at >= rows || b >= a.kv.batch) return;
    b = __builtin_amdgcn_readfirstlane(b);
    const AttnSpan rest = a.rest.spans[b];
    const int g = a.group_of[b];
    const int h = y.by_group.div(head), in_group = head - h * a.group;
    const int64_t r = (int64_t)(t - rest.start) * a.group + in_group;
    if (t < rest.start || r >= rest.rows) return;
    AttnSpan prefix = {};
    int64_t rp = 0;
    if (g >= 0) {
        prefix = a.prefix.spans[g];
        rp = (int64_t)(t - prefix.start) * a.group + in_group;
        if (t < prefix.start || rp >= prefix.rows) prefix.pieces = 0;
    }
    // piece p of the row: the prefix' first
    const int pieces = prefix.pieces + rest.pieces;
    const int tp = (int)rp / a.prefix.rows, tr = (int)r / a.rest.rows;
    const auto part = [&](int p, const float** o) {
        const bool first = p < prefix.pieces;
        const AttnSpan& s = first ? prefix : rest;
        const PrefixList& l = first ? a.prefix : a.rest;
        const int64_t item = s.item0 + ((int64_t)(first ? p : p - prefix.pieces) * a.kv.kv_heads + h) * s.tiles + (first ? tp : tr);
        const int64_t row = item * l.rows + (first ? (int)rp - tp * l.rows : (int)r - tr * l.rows);
        *o = l.part_o + row * y.dim;
        return l.part_ml + row;
    };
    const int lanes = y.dim <= 64 ? 16 : y.dim <= 128 ? 32 : 64, turns = 64 / lanes;
    const int d = (lane % lanes) * 4, mine = lane / lanes, dd = d < y.dim ? d : 0;
    float top = -__builtin_inff();
    for (int p = lane; p < pieces; p += 64) {
        const float* o;
        top = fmaxf(top, part(p, &o)->x);
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, xor_partner(top, off, lane));
    const float tu = top == -__builtin_inff() ? 0.f : top;
    float sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < pieces; p0 += 64) {
        float2 own = make_float2(-__builtin_inff(), 0.f);
        const float* o = nullptr;
        if (p0 + lane < pieces) own = *part(p0 + lane, &o);
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
                const float* from;
                part(p0 + min(p, n - 1), &from);
                v[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (take) v[k] = *(const f32x4_t*)(from + dd);
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

size_t list_bytes(const PrefixList& l, int dim) {
    return align16((size_t)l.count * sizeof(AttnSpan)) + align16((size_t)l.count * sizeof(int32_t)) +
           align16((size_t)l.room * l.rows * (dim + 2) * sizeof(float));
}
char* place_list(PrefixList& l, int dim, int32_t* total, char* p) {
    l.total = total;
    l.spans = (AttnSpan*)p;
    p += align16((size_t)l.count * sizeof(AttnSpan));
    l.item0 = (int32_t*)p;
    p += align16((size_t)l.count * sizeof(int32_t));
    l.part_o = (float*)p;
    l.part_ml = (float2*)(l.part_o + (size_t)l.room * l.rows * dim);
    return p + align16((size_t)l.room * l.rows * (dim + 2) * sizeof(float));
}

// The attention over a list of spans.
hipError_t attend_list(TreeAttnArgs t, const PrefixList& l, const Form& f, int cache_dtype, hipStream_t st) {
    t.part_o = l.part_o;
    t.part_ml = l.part_ml;
    t.spans = l.spans;
    t.item0 = l.item0;
    t.total = l.total;
    t.num_spans = l.count;
    return attend<true>(t, f, cache_dtype, (unsigned)((l.room + 7) / 8 * 8), st);
}

Form rest_form(const TreeAttnArgs& t, int cache_dtype) { return form_of(t, cache_dtype); }
// Rows of a group: its share of the tokens.
Form prefix_form(TreeAttnArgs t, int groups, int cache_dtype) {
    t.max_nodes = (t.kv.tokens + groups - 1) / groups;
    return form_of(t, cache_dtype);
}

}  // namespace

size_t plan_prefix_attention(PrefixArgs& a, const TreeAttnArgs& t, int cache_dtype, int num_cus) {
    a.kv = t.kv;
    a.group = t.group;
    a.max_nodes = t.max_nodes;
    a.max_tokens = t.max_tokens;
    a.slots = 2 * num_cus;
    const int64_t rows = (int64_t)t.kv.tokens * t.group;
    const auto fill = [&](PrefixList& l, const Form& f, int count) {
        l.count = count;
        l.rows = f.rows();
        l.step = f.ring ? 64 : STEP;
        l.least = f.ring ? 256 : STEP;
        const int64_t room = std::max<int64_t>(a.slots, (rows / l.rows + count) * t.kv.kv_heads);
        l.room = room > kLaunchWorkgroups - 8 ? 0 : (int32_t)room;
    };
    fill(a.prefix, prefix_form(t, a.groups, cache_dtype), a.groups);
    fill(a.rest, rest_form(t, cache_dtype), t.kv.batch);
    if (!a.prefix.room || !a.rest.room || rows > 0x7FFFFFFF || (int64_t)t.kv.tokens * t.heads > 4 * kLaunchWorkgroups) return 0;
    return 16 + align16((size_t)t.kv.batch * sizeof(int32_t)) + list_bytes(a.prefix, t.dim) + list_bytes(a.rest, t.dim);
}

hipError_t launch_prefix_attention(PrefixArgs& a, const TreeAttnArgs& t, int cache_dtype, void* ws, hipStream_t st) {
    int32_t* totals = (int32_t*)ws;
    char* p = (char*)ws + 16;
    a.group_of = (int32_t*)p;
    p += align16((size_t)t.kv.batch * sizeof(int32_t));
    p = place_list(a.prefix, t.dim, totals, p);
    place_list(a.rest, t.dim, totals + 1, p);
    prefix_plan_kernel<<<1, PLAN, 0, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    TreeAttnArgs whole = t;
    whole.mask = nullptr;  // every row sees all of its prefix
    if ((e = attend_list(whole, a.prefix, prefix_form(t, a.groups, cache_dtype), cache_dtype, st)) != hipSuccess) return e;
    if ((e = attend_list(t, a.rest, rest_form(t, cache_dtype), cache_dtype, st)) != hipSuccess) return e;
    const int rows = t.kv.tokens * t.heads;
    prefix_join_kernel<<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a, t, FastDiv(t.heads), rows);
    return hipGetLastError();
}

}  // namespace ingot
