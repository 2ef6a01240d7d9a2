// Attention of new (drafted) tokens over a paged key/value cache: the plan of a
// call, the join of its pieces and the launches.

#include "tree_attention.hpp"

namespace ingot {

namespace {

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

template <int BR>
hipError_t join(const TreeAttnArgs& a, hipStream_t st) {
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
    const unsigned grid = (unsigned)grid_of(a);
    const hipError_t e = by_types(a, cache_dtype, [&](auto type, auto dim, auto qt) {
        using T = decltype(type);
        constexpr int DP = decltype(dim)::value, QT = decltype(qt)::value;
        if constexpr (sizeof(T) == 2) {
            if (f.ring) {
                if constexpr (DP <= 128 && QT == 1)
                    if (f.tile == 32) {
                        tree_attention_ring_kernel<DP, 32, QT, 2><<<grid, 256, 0, st>>>(a);
                        return;
                    }
                tree_attention_ring_kernel<DP, 16, QT, DP <= 128 ? 2 : 1><<<grid, 256, 0, st>>>(a);
                return;
            }
        } else if constexpr (DP <= 128) {
            if (f.tile == 32) {
                tree_attention_kernel<T, DP, 2, QT><<<grid, 256, 0, st>>>(a);
                return;
            }
        }
        tree_attention_kernel<T, DP, 1, QT><<<grid, 256, 0, st>>>(a);
    });
    if (e != hipSuccess || a.splits == 1) return e;
    switch (f.rows()) {
        case 16: return join<16>(a, st);
        case 32: return join<32>(a, st);
        case 64: return join<64>(a, st);
        default: return join<128>(a, st);
    }
}

}  // namespace ingot
