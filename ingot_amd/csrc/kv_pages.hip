// Operations on the pages of a key/value cache: copying, handing out, sharing
// (fork), freeing, and moving accepted tokens together.
//
// The state is a count of references per page; a free page is one with none, so
// there is no list to keep consistent. Handing out scans the counts for the
// lowest free pages in one workgroup, which makes the outcome independent of
// any order of execution. Counts change by atomics, whose order does not
// matter: nothing reads them in the same kernel.

#include <algorithm>

#include "decoder.hpp"
#include "launch_bound.hpp"

namespace ingot {

namespace {

constexpr int COPY = 4;  // 16-byte chunks a thread moves: all loaded before any is stored

// Position of chunk `i` of one page's slots 0 .. slots − 1 in every layer, keys
// and values: (((layer · 2 + value) · segs + seg) · slots + slot) · row_chunks + c.
struct ChunkOrder {
    FastDiv by_row, by_slots, by_seg;
    ChunkOrder(const PagesView& p, int slots) : by_row(p.row_chunks), by_slots(slots), by_seg(p.segs) {}
};
__device__ __forceinline__ char* chunk_at(const PagesView& p, const ChunkOrder& o, int i, int* slot, int64_t* off) {
    int q = o.by_row.div(i);
    const int c = i - q * o.by_row.d;
    i = q;
    q = o.by_slots.div(i);
    *slot = i - q * o.by_slots.d;
    i = q;
    q = o.by_seg.div(i);
    const int seg = i - q * o.by_seg.d;
    *off = (int64_t)(q >> 1) * p.stride_layer + seg * p.stride_seg + *slot * p.stride_slot + c * 16;
    return q & 1 ? p.v : p.k;
}

// Pages d_src[i] → d_dst[i]: bound by the bytes. A workgroup moves 16 KB of one
// page, its chunks in the order (layer, key or value, head, slot), so that
// neighbouring lanes read neighbouring bytes whatever the strides. 200 pages of
// 16 layers (839 MB read and written): 151 to 164 µs, 5.1 to 5.6 TB/s.
__global__ void __launch_bounds__(256) kv_copy_kernel(PagesView p, ChunkOrder o, const int32_t* src, const int32_t* dst,
                                                      int chunks, FastDiv by_blocks) {
    const int i = by_blocks.div((int)blockIdx.x), part = (int)blockIdx.x - i * by_blocks.d;
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= p.num_pages || d < 0 || d >= p.num_pages || s == d) return;
    const int base = part * 256 * COPY + threadIdx.x;
    i32x4_t v[COPY];
    char* to[COPY];
#pragma unroll
    for (int j = 0; j < COPY; ++j) {
        const int c = base + j * 256;
        to[j] = nullptr;
        if (c < chunks) {
            int slot;
            int64_t off;
            char* pool = chunk_at(p, o, c, &slot, &off);
            v[j] = *(const i32x4_t*)(pool + s * p.stride_page + off);
            to[j] = pool + d * p.stride_page + off;
        }
    }
#pragma unroll
    for (int j = 0; j < COPY; ++j)
        if (to[j]) *(i32x4_t*)to[j] = v[j];
}

__device__ __forceinline__ bool row_ok(const PagesView& p, int r) { return r >= 0 && r < p.rows; }
__device__ __forceinline__ bool page_ok(const PagesView& p, int id) { return id >= 0 && id < p.num_pages; }

// Sum over the workgroup's lower threads of v, and the whole in *total
// (1024 threads; `part` holds 17 values).
__device__ __forceinline__ int64_t scan_1024(int64_t v, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t run = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t o = __shfl_up(run, off);
        if (lane >= off) run += o;
    }
    __syncthreads();  // part's last readers are done
    if (lane == 63) part[wave] = run;
    __syncthreads();
    int64_t below = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
        const int64_t x = part[w];
        below += w < wave ? x : 0;
        all += x;
    }
    *total = all;
    return below + run - v;
}

// The workgroup's list of the lowest free pages, at most `want`; how many.
__device__ int collect_free(const PagesView& p, int64_t want, int32_t* list, int64_t* part) {
    constexpr int PER = 16;
    int64_t found = 0;
    for (int64_t at = 0; at < p.num_pages && found < want; at += 1024 * PER) {
        const int64_t mine = at + threadIdx.x * PER;
        uint32_t free_bits = 0;
        int32_t refs[PER];  // all asked for at once
#pragma unroll
        for (int j = 0; j < PER; ++j) refs[j] = p.refs[min(mine + j, (int64_t)p.num_pages - 1)];
#pragma unroll
        for (int j = 0; j < PER; ++j) free_bits |= (mine + j < p.num_pages && refs[j] <= 0 ? 1u : 0u) << j;
        int64_t total;
        int64_t place = found + scan_1024(__popc(free_bits), part, &total);
        while (free_bits && place < want) {
            const int j = __ffs((int)free_bits) - 1;
            free_bits &= free_bits - 1;
            list[place++] = (int32_t)(mine + j);
        }
        found += total;
    }
    __syncthreads();  // the list is written
    return (int)min(found, want);
}

struct AllocWs {
    int64_t* offset;  // [n] pages asked for before entry i
    int32_t* need;    // [n] pages entry i asks for (-1: none can serve it)
    int32_t* fresh;   // [n] fork: the page given, -1: none left, -2: none needed; reserve: pages held
    int32_t* list;    // [pages]
};
__host__ __device__ inline AllocWs alloc_ws(void* ws, int64_t n) {
    AllocWs w;
    w.offset = (int64_t*)ws;
    w.need = (int32_t*)(w.offset + n);
    w.fresh = w.need + n;
    w.list = w.fresh + n;
    return w;
}

// How many pages a row has: they come first in it. Seven places are tried at a
// time (one read's latency for three bits of the answer).
__device__ __forceinline__ int held_pages(const PagesView& p, int row) {
    const int32_t* pages = p.pages + (int64_t)row * p.max_pages;
    int lo = 0, hi = p.max_pages;  // entries before lo hold a page, from hi on none
    while (lo < hi) {
        const int step = (hi - lo + 7) >> 3;
        int have = 0;
        bool there[7];
#pragma unroll
        for (int i = 0; i < 7; ++i) there[i] = pages[min(lo + (i + 1) * step, hi) - 1] >= 0;
#pragma unroll
        for (int i = 0; i < 7; ++i) have += there[i] && have == i;
        const int from = min(lo + have * step, hi);
        if (have < 7) hi = min(lo + (have + 1) * step, hi) - 1;
        lo = from;
    }
    return lo;
}

// One workgroup: the needs, the free pages, the hand-out. The order of the list
// decides who is served, so the sums over it are a scan; with a workgroup there
// is no second launch between it and the hand-out. A chain of dependent reads
// bounds it: rows, lengths, page counts, references, list. 8 rows 8.9 µs, 122 rows
// of up to 44 pages 13.5 (with two bisections in place of held_pages 17.6).
__global__ void __launch_bounds__(1024) kv_reserve_kernel(PagesView p, const int32_t* row, const int32_t* tokens, int n,
                                                          AllocWs w) {
    __shared__ int64_t part[17];
    __shared__ unsigned long long lacking;  // up to 2^31 pages for each of 2^20 rows
    if (threadIdx.x == 0) lacking = 0;
    int64_t asked = 0;
    for (int at = 0; at < n; at += 1024) {
        const int i = at + threadIdx.x;
        int need = 0, held = 0;
        int64_t lack = 0;
        if (i < n && row_ok(p, row[i])) {
            const int64_t want = (int64_t)max(0, p.len[row[i]]) + max(0, tokens[i]);
            const bool past = want > 0x7FFFFFFF;  // more tokens than a length can count
            const int64_t pages_want = past ? (want + p.page_size - 1) / p.page_size
                                            : p.by_page.div((int)want) + (want % p.page_size != 0);
            held = held_pages(p, row[i]);
            if (past || pages_want > p.max_pages) lack = pages_want - held, need = -1;
            else need = (int)max((int64_t)0, pages_want - held);
        }
        int64_t total;
        const int64_t before = scan_1024(max(need, 0), part, &total);
        if (i < n) {
            w.offset[i] = asked + before;
            w.need[i] = need;
            w.fresh[i] = held;
        }
        asked += total;
        if (lack > 0) atomicAdd(&lacking, (unsigned long long)lack);
    }
    const int found = asked ? collect_free(p, min(asked, (int64_t)p.num_pages), w.list, part) : 0;
    __syncthreads();
    const int lane = threadIdx.x & 63;
    for (int i = threadIdx.x >> 6; i < n; i += 16) {
        const int need = w.need[i];
        if (need <= 0) continue;
        const int64_t off = w.offset[i];
        if (off + need > found) {
            if (lane == 0) atomicAdd(&lacking, (unsigned long long)need);
            continue;
        }
        int32_t* pages = p.pages + (int64_t)row[i] * p.max_pages + w.fresh[i];
        for (int j = lane; j < need; j += 64) {
            const int id = w.list[off + j];
            pages[j] = id;
            p.refs[id] = 1;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.missing = (int32_t)min(lacking, 0x7FFFFFFFull);
}

// Tokens of a row that fork shares: what its pages can hold.
struct ForkLen {
    int len, full, rest;
};
__device__ __forceinline__ ForkLen fork_len(const PagesView& p, int src) {
    ForkLen f;
    f.len = max(0, p.len[src]);
    f.full = p.by_page.div(f.len);
    f.rest = f.len - f.full * p.page_size;
    if (f.full >= p.max_pages) f.full = p.max_pages, f.rest = 0;
    return f;
}

// Entry j of row d: the old page loses its reference and the shared one gains
// it. Entries are exchanged, so each reference is released once whatever the
// lists hold.
__device__ __forceinline__ void share_entry(const PagesView& p, int s, int d, int j) {
    int id = p.pages[(int64_t)s * p.max_pages + j];
    const ForkLen f = fork_len(p, s);
    if (j >= f.full || !page_ok(p, id)) id = -1;
    if (id >= 0) atomicAdd(&p.refs[id], 1);
    const int old = atomicExch(&p.pages[(int64_t)d * p.max_pages + j], id);
    if (page_ok(p, old)) atomicSub(&p.refs[old], 1);
    if (j == 0) p.len[d] = f.len;
}
__device__ __forceinline__ bool fork_ok(const PagesView& p, int s, int d) {
    return row_ok(p, s) && row_ok(p, d) && s != d;
}
__global__ void __launch_bounds__(256) kv_fork_share_kernel(PagesView p, const int32_t* src, const int32_t* dst) {
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    if (!fork_ok(p, s, d)) return;
    for (int j = threadIdx.x; j < p.max_pages; j += 256) share_entry(p, s, d, j);
}

// One workgroup (see kv_reserve_kernel; 7 µs for 48 rows): the sharing where an
// entry a thread is enough for it (by_row of max_pages, else of 0), then a page
// for each part-filled one.
__global__ void __launch_bounds__(1024) kv_fork_alloc_kernel(PagesView p, const int32_t* src, const int32_t* dst, int n,
                                                             FastDiv by_row, AllocWs w) {
    __shared__ int64_t part[17];
    __shared__ int lacking;
    if (threadIdx.x == 0) lacking = 0;
    if ((int)threadIdx.x < n * by_row.d) {
        const int i = by_row.div((int)threadIdx.x), s = src[i], d = dst[i];
        if (fork_ok(p, s, d)) share_entry(p, s, d, (int)threadIdx.x - i * by_row.d);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the counts have changed before any wave reads them
    int64_t asked = 0;
    for (int at = 0; at < n; at += 1024) {
        const int i = at + threadIdx.x;
        int need = 0;
        if (i < n) {
            const int s = src[i], d = dst[i];
            if (fork_ok(p, s, d)) {
                // a source without its part-filled page has nothing to copy: a page
                // handed out for it would show what its last owner left
                const ForkLen f = fork_len(p, s);
                need = f.rest > 0 && page_ok(p, p.pages[(int64_t)s * p.max_pages + f.full]);
            }
        }
        int64_t total;
        const int64_t before = scan_1024(need, part, &total);
        if (i < n) {
            w.offset[i] = asked + before;
            w.need[i] = need;
        }
        asked += total;
    }
    __syncthreads();  // the counts are as the sharing left them
    const int found = asked ? collect_free(p, min(asked, (int64_t)p.num_pages), w.list, part) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 1024) {
        int fresh = -2;
        if (w.need[i]) {
            fresh = w.offset[i] < found ? w.list[w.offset[i]] : -1;
            if (fresh >= 0) {
                p.refs[fresh] = 1;
                p.pages[(int64_t)dst[i] * p.max_pages + fork_len(p, src[i]).full] = fresh;
            } else {
                atomicAdd(&lacking, 1);
            }
        }
        w.fresh[i] = fresh;
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.missing = lacking;
}

// The filled slots of the part-filled pages; rows that got no page are emptied.
// Bound by the bytes, in the chunk order of kv_copy_kernel: 48 rows of 16 layers
// (about 100 MB) 16 µs of the call's 25.
__global__ void __launch_bounds__(256) kv_fork_copy_kernel(PagesView p, ChunkOrder o, const int32_t* src,
                                                           const int32_t* dst, int chunks, FastDiv by_blocks, AllocWs w) {
    const int i = by_blocks.div((int)blockIdx.x), part = (int)blockIdx.x - i * by_blocks.d;
    const int fresh = w.fresh[i];
    if (fresh == -2) return;
    const int s = src[i], d = dst[i];
    if (fresh < 0) {
        if (part) return;
        for (int j = threadIdx.x; j < p.max_pages; j += 256) {
            const int old = atomicExch(&p.pages[(int64_t)d * p.max_pages + j], -1);
            if (page_ok(p, old)) atomicSub(&p.refs[old], 1);
        }
        if (threadIdx.x == 0) p.len[d] = 0;
        return;
    }
    const ForkLen f = fork_len(p, s);
    const int old = p.pages[(int64_t)s * p.max_pages + f.full];
    if (!page_ok(p, old)) return;
    i32x4_t v[COPY];
    char* to[COPY];
#pragma unroll
    for (int j = 0; j < COPY; ++j) {
        const int c = part * 256 * COPY + j * 256 + threadIdx.x;
        to[j] = nullptr;
        if (c < chunks) {
            int slot;
            int64_t off;
            char* pool = chunk_at(p, o, c, &slot, &off);
            if (slot < f.rest) {
                v[j] = *(const i32x4_t*)(pool + old * p.stride_page + off);
                to[j] = pool + fresh * p.stride_page + off;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < COPY; ++j)
        if (to[j]) *(i32x4_t*)to[j] = v[j];
}

__global__ void __launch_bounds__(256) kv_free_kernel(PagesView p, const int32_t* row) {
    const int r = row[blockIdx.x];
    if (!row_ok(p, r)) return;
    for (int j = threadIdx.x; j < p.max_pages; j += 256) {
        const int old = atomicExch(&p.pages[(int64_t)r * p.max_pages + j], -1);
        if (page_ok(p, old)) atomicSub(&p.refs[old], 1);
    }
    if (threadIdx.x == 0) p.len[r] = 0;
}

// A thread owns a 16-byte column (layer, key or value, head, part of the head)
// of one row's slots and moves its accepted tokens up in order, BATCH at a time:
// nodes rise, so node j is at or after slot j, and the slots written lie before
// every source still to be read. The places of 64 tokens are looked up once for
// the workgroup. Bound by the bytes, or one launch's latency and three dependent
// reads: 16 rows of up to 6 accepted tokens in 16 layers (6.3 MB) 4.3 µs.
__global__ void __launch_bounds__(256) kv_compact_kernel(PagesView p, FastDiv by_row, FastDiv by_seg, FastDiv by_blocks,
                                                         int columns, const int32_t* row, const int32_t* accept,
                                                         const int32_t* count, int max_accept, int32_t* new_len) {
    constexpr int STEP = 64, BATCH = 8;
    __shared__ int64_t from[STEP], to[STEP];
    const int i = by_blocks.div((int)blockIdx.x), part = (int)blockIdx.x - i * by_blocks.d;
    const int r = row[i];
    if (!row_ok(p, r)) return;
    const int n = min(max(count[i], 0), max_accept), len = p.len[r];
    const int32_t* pages = p.pages + (int64_t)r * p.max_pages;
    const int col = part * 256 + threadIdx.x;
    const int q = by_row.div(col), c = col - q * by_row.d;
    const int lv = by_seg.div(q), seg = q - lv * by_seg.d;
    char* base = (lv & 1 ? p.v : p.k) + (int64_t)(lv >> 1) * p.stride_layer + seg * p.stride_seg + c * 16;
    const auto place = [&](int64_t pos) -> int64_t {
        if (pos < 0 || pos > 0x7FFFFFFF) return -1;
        const int pg = p.by_page.div((int)pos);
        if (pg >= p.max_pages) return -1;
        const int id = pages[pg];
        return page_ok(p, id) ? id * p.stride_page + (pos - (int64_t)pg * p.page_size) * p.stride_slot : -1;
    };
    for (int at = 0; at < n; at += STEP) {
        __syncthreads();
        const int j = at + threadIdx.x;
        if (threadIdx.x < STEP) {
            int64_t f = -1, t = -1;
            if (j < n) {
                const int node = accept[(int64_t)i * max_accept + j];
                if (node >= 0 && node != j) {
                    f = place((int64_t)len + node);
                    t = place((int64_t)len + j);
                }
            }
            from[threadIdx.x] = t < 0 ? -1 : f;
            to[threadIdx.x] = t;
        }
        __syncthreads();
        if (col < columns) {
            const int m = min(STEP, n - at);
            for (int b = 0; b < m; b += BATCH) {
                i32x4_t v[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (b + k < m && from[b + k] >= 0) v[k] = *(const i32x4_t*)(base + from[b + k]);
#pragma unroll
                for (int k = 0; k < BATCH; ++k)
                    if (b + k < m && from[b + k] >= 0) *(i32x4_t*)(base + to[b + k]) = v[k];
            }
        }
    }
    if (part == 0 && threadIdx.x == 0) new_len[r] = (int32_t)min((int64_t)0x7FFFFFFF, (int64_t)len + n);
}

}  // namespace

hipError_t launch_kv_copy(const PagesView& p, const int32_t* src, const int32_t* dst, int64_t n, hipStream_t st) {
    const int chunks = p.layers * 2 * p.segs * p.page_size * p.row_chunks;
    const int blocks = (chunks + 256 * COPY - 1) / (256 * COPY);
    const int64_t step = entries_of_launch(blocks);  // at most 2^22 workgroups an entry
    for (int64_t first = 0; first < n; first += step) {
        const int64_t m = std::min(step, n - first);
        kv_copy_kernel<<<(unsigned)(m * blocks), 256, 0, st>>>(p, ChunkOrder(p, p.page_size), src + first, dst + first,
                                                               chunks, FastDiv(blocks));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

size_t kv_alloc_ws(int64_t n, int64_t pages) { return (size_t)(16 * n + 4 * pages + 256); }

hipError_t launch_kv_reserve(const PagesView& p, const int32_t* row, const int32_t* tokens, int n, void* ws,
                             hipStream_t st) {
    kv_reserve_kernel<<<1, 1024, 0, st>>>(p, row, tokens, n, alloc_ws(ws, n));
    return hipGetLastError();
}

hipError_t launch_kv_fork(const PagesView& p, const int32_t* src, const int32_t* dst, int n, void* ws, hipStream_t st) {
    const AllocWs w = alloc_ws(ws, n);
    // Up to an entry a thread the one workgroup does the sharing too: 39 rows of 5
    // pages take 11.6 µs so and 13.3 with a launch of its own; 48 rows of 33
    // (two entries a thread) 24.4 and 24.1 (all 0.3 more since the hand-out looks
    // whether the source's page is there).
    const bool few = (int64_t)n * p.max_pages <= 1024;
    if (n && !few) {
        kv_fork_share_kernel<<<n, 256, 0, st>>>(p, src, dst);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    kv_fork_alloc_kernel<<<1, 1024, 0, st>>>(p, src, dst, n, few ? FastDiv(p.max_pages) : FastDiv(), w);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !n) return e;
    const int chunks = p.layers * 2 * p.segs * p.page_size * p.row_chunks;
    const int blocks = (chunks + 256 * COPY - 1) / (256 * COPY);
    const int64_t step = entries_of_launch(blocks);  // at most 2^22 workgroups an entry
    for (int64_t first = 0; first < n; first += step) {
        const int64_t m = std::min<int64_t>(step, n - first);
        AllocWs part = w;
        part.fresh += first;
        kv_fork_copy_kernel<<<(unsigned)(m * blocks), 256, 0, st>>>(p, ChunkOrder(p, p.page_size), src + first,
                                                                    dst + first, chunks, FastDiv(blocks), part);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv_free(const PagesView& p, const int32_t* row, int n, hipStream_t st) {
    kv_free_kernel<<<n, 256, 0, st>>>(p, row);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const PagesView& p, const int32_t* row, const int32_t* accept, const int32_t* count, int n,
                             int max_accept, int32_t* new_len, hipStream_t st) {
    const int columns = p.layers * 2 * p.segs * p.row_chunks;
    const int blocks = (columns + 255) / 256;
    const int64_t step = entries_of_launch(blocks);  // at most 2^22 workgroups an entry
    for (int64_t first = 0; first < n; first += step) {
        const int64_t m = std::min<int64_t>(step, n - first);
        kv_compact_kernel<<<(unsigned)(m * blocks), 256, 0, st>>>(
            p, FastDiv(p.row_chunks), FastDiv(p.segs), FastDiv(blocks), columns, row + first,
            accept + first * max_accept, count + first, max_accept, new_len);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ingot
