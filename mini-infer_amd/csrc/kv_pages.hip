// kv_pages.hip -- the pages of a paged KV cache, managed on the device: copied, shared
// between sequences, reserved, freed, moved together.
//
// State: block_table [B, mb] (int32 page of each block of a row, -1 for none), seq_len [B]
// and ref_count [num_blocks], the number of table entries that hold a page; 0: free.  There
// is no list of free pages: those are found where they are needed, lowest first, so what a
// call leaves is a function of the state and of the call alone.  Copies are bound by HBM (two
// bytes moved per byte of page): 190 pages, 174 MB, 38 us, 4.6 TB/s; a cache of 8192 pages, half of them
// live, moved together, 1.07 GB, 215 us, 5.0 TB/s, of which 13 are the one workgroup that plans it.  The
// rest is bound by the latency of its launches: a step of 32 beams, freed, forked and given room, with
// 24 pages copied, 21 us.
#include <algorithm>

#include "mi_device.h"
#include "mi_host.h"

namespace mi {

constexpr int kPageCaches = 8;
constexpr int kRowsMax = 1024;  // rows of a call that are looked at together

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct PageCaches {
    int n;
    uint8_t* data[kPageCaches];
    int64_t layers[kPageCaches];
    int64_t bytes[kPageCaches];  // of a page in one layer
    int unit[kPageCaches];       // bytes of one access: 16, 4 or 1
    int64_t units[kPageCaches];  // of a page
    int64_t pieces[kPageCaches];  // of a page of 16-byte units
    int64_t num_blocks;
};
constexpr int kLarge = 8, kSmall = 2;  // KB that a wave moves at a time
constexpr int kInline = 64;            // pairs up to which every wave checks its own: one load each

// Pairs that copy: those whose pages are in the cache and whose destination is in no other
// pair as a source and in no earlier one as a destination; so the copies can run in any order.
__device__ __forceinline__ bool clashes(const int* src, const int* dst, int n, int i, int d, int from, int by) {
    bool b = false;
    for (int j = from; j < n; j += by) b |= (j != i && src[j] == d) || (j < i && dst[j] == d);
    return b;
}

__global__ __launch_bounds__(256) void pages_check_kernel(const int* src, const int* dst, int n,
                                                          int64_t num_blocks, int* status) {
    __shared__ int bad;
    const int i = blockIdx.x;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    const int s = src[i], d = dst[i];
    if (s < 0 || s >= num_blocks || d < 0 || d >= num_blocks || clashes(src, dst, n, i, d, threadIdx.x, 256)) bad = 1;
    __syncthreads();
    if (threadIdx.x == 0) status[i] = bad ? MI_KV_REFUSED : MI_KV_DONE;
}

// The pairs of a launch: `pairs` of them, copied where status says so; with `check`, each wave
// looks its own up and the first to handle a pair says what became of it.
struct Pairs {
    const int *src, *dst;
    int* status;
    int n, check;
};
__device__ __forceinline__ bool wanted(const Pairs& p, const PageCaches& c, uint32_t pair, int& s, int& d, bool say) {
    s = p.src[pair];
    d = p.dst[pair];
    bool ok = s >= 0 && s < c.num_blocks && d >= 0 && d < c.num_blocks;
    if (p.check) {
        if (ok) ok = !__any(clashes(p.src, p.dst, p.n, static_cast<int>(pair), d, threadIdx.x & 63, 64));
        if (say && (threadIdx.x & 63) == 0) p.status[pair] = ok ? MI_KV_DONE : MI_KV_REFUSED;
    } else if (p.status) {
        ok = ok && p.status[pair] == MI_KV_DONE;
    }
    return ok && s != d;
}

// One wave moves a piece of a page: R 16-byte accesses per lane, all loads before the stores.
// What names the page is the same for the wave and sits in scalar registers.
template <int R>
__device__ __forceinline__ void copy_piece(const PageCaches& c, int k, int64_t task, const Pairs& p) {
    constexpr int kPiece = R * 1024;
    const uint32_t pieces = static_cast<uint32_t>(c.pieces[k]), layers = static_cast<uint32_t>(c.layers[k]);
    const uint32_t page = static_cast<uint32_t>(task) / pieces, piece = static_cast<uint32_t>(task) - page * pieces;
    const uint32_t pair = page / layers;
    const int64_t layer = page - pair * layers;
    int s, d;
    if (!wanted(p, c, pair, s, d, k == 0 && layer == 0 && piece == 0)) return;
    const int lane = threadIdx.x & 63;
    const int64_t at = static_cast<int64_t>(piece) * kPiece + lane * 16;
    const uint8_t* const from = c.data[k] + (layer * c.num_blocks + s) * c.bytes[k] + at;
    uint8_t* const to = c.data[k] + (layer * c.num_blocks + d) * c.bytes[k] + at;
    const int left = static_cast<int>(min<int64_t>(c.bytes[k] - static_cast<int64_t>(piece) * kPiece, kPiece)) - lane * 16;
    u4 v[R];
    if (left + lane * 16 == kPiece) {
#pragma unroll
        for (int r = 0; r < R; ++r) v[r] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(from + r * 1024));
#pragma unroll
        for (int r = 0; r < R; ++r) __builtin_nontemporal_store(v[r], reinterpret_cast<u4*>(to + r * 1024));
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * 1024 < left) v[r] = *reinterpret_cast<const u4*>(from + r * 1024);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * 1024 < left) *reinterpret_cast<u4*>(to + r * 1024) = v[r];
    }
}

// Pages that no 16-byte access fits, scales for the most part: one pair and layer per group
// of lanes, or per wave where the pairs are checked here.
template <typename U>
__device__ __forceinline__ void copy_small(const PageCaches& c, int k, int64_t page, int64_t u0, int64_t by, const Pairs& p) {
    const uint32_t pair = static_cast<uint32_t>(page) / static_cast<uint32_t>(c.layers[k]);
    const int64_t layer = page - static_cast<int64_t>(pair) * c.layers[k];
    int s, d;
    if (!wanted(p, c, pair, s, d, k == 0 && layer == 0)) return;
    U* const to = reinterpret_cast<U*>(c.data[k] + (layer * c.num_blocks + d) * c.bytes[k]);
    const U* const from = reinterpret_cast<const U*>(c.data[k] + (layer * c.num_blocks + s) * c.bytes[k]);
    for (int64_t u = u0; u < c.units[k]; u += by) to[u] = from[u];
}

// pages src[i] -> dst[i] of every cache and layer; `count`: pairs known on the device
// alone, at most `most`.  The grid's waves walk the pieces.
template <int R>
__global__ __launch_bounds__(256) void pages_copy_kernel(PageCaches c, Pairs p, const int* count) {
    const int64_t pairs = count ? min(*count, p.n) : p.n;
    const int64_t waves = static_cast<int64_t>(gridDim.x) * 4;
    const int lane = threadIdx.x & 63;
    int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int k = 0; k < c.n; ++k) {  // the caches' tasks one behind the other
        const int64_t pages = pairs * c.layers[k];  // < 2^31, pieces too
        const int64_t tasks = pages * c.pieces[k];
        if (c.unit[k] == 16) {
            for (; t < tasks; t += waves) copy_piece<R>(c, k, t, p);
        } else if (p.check) {
            for (; t < tasks; t += waves) {
                if (c.unit[k] == 4) copy_small<uint32_t>(c, k, t, lane, 64, p);
                else copy_small<uint8_t>(c, k, t, lane, 64, p);
            }
        } else {  // eight lanes a page
            for (; t * 8 < tasks; t += waves) {
                const int64_t page = t * 8 + (lane >> 3);
                if (page >= tasks) continue;
                if (c.unit[k] == 4) copy_small<uint32_t>(c, k, page, lane & 7, 8, p);
                else copy_small<uint8_t>(c, k, page, lane & 7, 8, p);
            }
            t -= (tasks + 7) / 8;
            continue;
        }
        t -= tasks;
    }
}

struct PageState {
    int *table, *seq, *ref;
    int64_t B, mb, num_blocks;
};

// One workgroup per listed row.  A row listed twice acts at its first place.
__global__ __launch_bounds__(256) void pages_free_kernel(PageState p, const int* rows, int n) {
    __shared__ int skip;
    const int i = blockIdx.x, row = rows[i];
    if (row < 0 || row >= p.B) return;
    if (threadIdx.x == 0) skip = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < i; j += 256)
        if (rows[j] == row) skip = 1;
    __syncthreads();
    if (skip) return;
    int* const t = p.table + row * p.mb;
    for (int64_t j = threadIdx.x; j < p.mb; j += 256) {
        const int pg = t[j];
        if (pg >= 0 && pg < p.num_blocks && atomicSub(p.ref + pg, 1) <= 0) atomicAdd(p.ref + pg, 1);
        t[j] = -1;
    }
    if (threadIdx.x == 0) p.seq[row] = 0;
}

// One workgroup per (parent, child).
__global__ __launch_bounds__(256) void pages_fork_kernel(PageState p, const int* parents, const int* kids,
                                                         int n, int* status) {
    __shared__ int bad;
    const int i = blockIdx.x, from = parents[i], to = kids[i];
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    bool b = from < 0 || from >= p.B || to < 0 || to >= p.B;
    for (int j = threadIdx.x; j < n; j += 256) b |= kids[j] == from || (j < i && kids[j] == to);
    if (b) bad = 1;
    __syncthreads();
    b = bad;
    __syncthreads();
    if (!b) {  // the child's row is this workgroup's own from here on; it has to be empty
        const int* const t = p.table + to * p.mb;
        bool held = p.seq[to] != 0;
        for (int64_t j = threadIdx.x; j < p.mb; j += 256) held |= t[j] >= 0;
        if (held) bad = 1;
    }
    __syncthreads();
    if (threadIdx.x == 0) status[i] = bad ? MI_KV_REFUSED : MI_KV_DONE;
    if (bad) return;
    const int* const s = p.table + from * p.mb;
    int* const t = p.table + to * p.mb;
    for (int64_t j = threadIdx.x; j < p.mb; j += 256) {
        const int pg = s[j];
        t[j] = pg;
        if (pg >= 0 && pg < p.num_blocks) atomicAdd(p.ref + pg, 1);
    }
    if (threadIdx.x == 0) p.seq[to] = p.seq[from];
}

// Exclusive prefix sum over a workgroup of 1024 lanes, and the total.
template <typename T>
__device__ __forceinline__ T scan1024(T v, T& total, T* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T y = __shfl_up(x, d, kWave);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    T before = 0;
    total = 0;
    for (int w = 0; w < 16; ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    return before + x - v;
}

struct Reserve {
    PageState p;
    const int *rows, *lengths;
    int* status;
    int *fresh, *cp_src, *cp_dst;  // workspace: free pages found; the copies, -1 for none
    int64_t bs;
    int n;
};

// One workgroup: lane i is row rows[i].  Rows take pages in their order; where the free ones
// do not reach for a row, it and all behind it are left as they were.
__global__ __launch_bounds__(1024) void pages_reserve_kernel(Reserve a) {
    __shared__ int s_row[kRowsMax], s_last[kRowsMax];
    __shared__ int64_t s_first[kRowsMax + 1], waves[16];
    const int i = threadIdx.x;
    const PageState& p = a.p;
    int row = -1, last = -1, status = MI_KV_DONE;
    int64_t have = 0, want = 0, len = 0;
    bool part = false;
    s_row[i] = i < a.n ? a.rows[i] : -1;
    __syncthreads();
    if (i < a.n) {
        row = s_row[i];
        len = a.lengths[i];
        bool bad = row < 0 || row >= p.B || len < 0 || len > p.mb * a.bs;
        for (int j = 0; j < i; ++j) bad |= s_row[j] == row;
        if (!bad) {
            const int64_t now = p.seq[row];
            bad = now < 0 || now > p.mb * a.bs;
            if (!bad) {
                have = (now + a.bs - 1) / a.bs;
                want = max((len + a.bs - 1) / a.bs, have);
                if (len > now && now % a.bs != 0) {
                    last = p.table[row * p.mb + have - 1];
                    bad = last < 0 || last >= p.num_blocks;
                    part = !bad;
                }
                if (len <= now) len = now;
            }
        }
        if (bad) {
            status = MI_KV_REFUSED;
            want = have;
            last = -1;
        }
    }
    s_last[i] = last;
    __syncthreads();
    int rank = 0;
    if (part)
        for (int j = 0; j < i; ++j) rank += s_last[j] == last;
    const bool cow = part && rank < p.ref[last] - 1;
    const int64_t need = (cow ? 1 : 0) + want - have;
    int64_t total;
    const int64_t first = scan1024<int64_t>(need, total, waves);
    s_first[i] = first;
    if (i == 0) s_first[kRowsMax] = total;
    // free pages, lowest first, until there are enough
    int64_t found = 0;
    for (int64_t base = 0; base < p.num_blocks && found < total; base += 4096) {
        int r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t pg = base + 4 * i + k;
            r[k] = pg < p.num_blocks ? p.ref[pg] : 1;
        }
        int all;
        const int mine = (r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0);
        int64_t at = found + scan1024<int>(mine, all, reinterpret_cast<int*>(waves));
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r[k] == 0) {
                if (at < total) a.fresh[at] = static_cast<int>(base + 4 * i + k);
                ++at;
            }
        found += all;
        __syncthreads();
    }
    found = min(found, total);
    __syncthreads();  // the list, and every read of ref, before what follows
    if (i < a.n) {
        if (status == MI_KV_DONE && first + need > found) status = MI_KV_FULL;
        const bool go = status == MI_KV_DONE;
        a.cp_src[i] = go && cow ? last : -1;
        a.cp_dst[i] = go && cow ? a.fresh[first] : -1;
        if (go) {
            if (cow) {
                p.table[row * p.mb + have - 1] = a.fresh[first];
                atomicSub(p.ref + last, 1);
            }
            p.seq[row] = static_cast<int>(len);
        }
        a.status[i] = status;
        // where the row's new blocks begin, less their place in the list (for the loop below)
        s_last[i] = go ? static_cast<int>(have) : -1;
        s_row[i] = (row << 1) | (cow ? 1 : 0);
    }
    __syncthreads();
    for (int64_t k = i; k < found; k += 1024) {
        int lo = 0, hi = a.n - 1;  // the last row whose first page is at or before k
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_first[mid] <= k) lo = mid;
            else hi = mid - 1;
        }
        if (s_last[lo] < 0) continue;
        const int pg = a.fresh[k];
        p.ref[pg] = 1;
        const int64_t j = k - s_first[lo] - (s_row[lo] & 1);
        if (j >= 0) p.table[static_cast<int64_t>(s_row[lo] >> 1) * p.mb + s_last[lo] + j] = pg;
    }
}

// One workgroup: live pages at or behind the number of live pages take the free places
// before it, in order.  moved: each page's place afterwards, -1 for a free one.
__global__ __launch_bounds__(1024) void pages_plan_kernel(int* ref, int64_t num_blocks, int* moved,
                                                          int* src, int* dst, int* count) {
    __shared__ int waves[16];
    const int i = threadIdx.x;
    int64_t live = 0;
    for (int64_t base = 0; base < num_blocks; base += 4096) {
        int mine = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t pg = base + 4 * i + k;
            mine += pg < num_blocks && ref[pg] > 0;
        }
        int all;
        scan1024<int>(mine, all, waves);
        live += all;
        __syncthreads();
    }
    int holes = 0, movers = 0;
    for (int64_t base = 0; base < num_blocks; base += 4096) {
        int h[4], m[4], nh = 0, nm = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t pg = base + 4 * i + k;
            const bool in = pg < num_blocks, on = in && ref[pg] > 0;
            h[k] = in && !on && pg < live;
            m[k] = on && pg >= live;
            nh += h[k];
            nm += m[k];
            if (in) moved[pg] = on ? static_cast<int>(pg) : -1;
        }
        int th, tm;
        int ah = holes + scan1024<int>(nh, th, waves);
        __syncthreads();
        int am = movers + scan1024<int>(nm, tm, waves);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int pg = static_cast<int>(base + 4 * i + k);
            if (h[k]) dst[ah++] = pg;
            if (m[k]) src[am++] = pg;
        }
        holes += th;
        movers += tm;
        __syncthreads();
    }
    __syncthreads();
    for (int k = i; k < movers; k += 1024) {
        const int s = src[k], d = dst[k];
        moved[s] = d;
        ref[d] = ref[s];
        ref[s] = 0;
    }
    if (i == 0) *count = movers;
}

__global__ __launch_bounds__(256) void pages_remap_kernel(int* table, int64_t n, const int* moved, int64_t num_blocks) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int pg = table[i];
        table[i] = pg >= 0 && pg < num_blocks ? moved[pg] : -1;
    }
}

static int page_caches(const mi_kv_pages* caches, int num_caches, int64_t num_blocks, int64_t pairs, PageCaches& c) {
    if (num_caches < 0 || (num_caches > 0 && !caches) || num_blocks < 0) return MI_ERR_INVALID_ARGUMENT;
    if (num_caches > kPageCaches || num_blocks > INT32_MAX - 4096) return MI_ERR_UNSUPPORTED;
    c = PageCaches{};
    c.num_blocks = num_blocks;
    for (int i = 0; i < num_caches; ++i) {
        const mi_kv_pages& g = caches[i];
        if (g.layers < 0 || g.page_bytes < 0 || !product_fits({g.layers, std::max<int64_t>(num_blocks, 1), g.page_bytes}))
            return MI_ERR_INVALID_ARGUMENT;
        if (g.layers == 0 || g.page_bytes == 0 || num_blocks == 0) continue;
        if (!g.data) return MI_ERR_INVALID_ARGUMENT;
        if (!product_fits({pairs, g.layers, g.page_bytes}) || g.layers > INT32_MAX / std::max<int64_t>(pairs, 1))
            return MI_ERR_UNSUPPORTED;
        for (int j = 0; j < c.n; ++j)
            if (overlaps(g.data, g.layers * num_blocks * g.page_bytes, c.data[j], c.layers[j] * num_blocks * c.bytes[j]))
                return MI_ERR_ALIASING;
        const int k = c.n++;
        const uintptr_t place = reinterpret_cast<uintptr_t>(g.data) | static_cast<uintptr_t>(g.page_bytes);
        c.data[k] = static_cast<uint8_t*>(g.data);
        c.layers[k] = g.layers;
        c.bytes[k] = g.page_bytes;
        c.unit[k] = place % 16 == 0 ? 16 : place % 4 == 0 ? 4 : 1;
        c.units[k] = g.page_bytes / c.unit[k];
        if (!product_fits({pairs, g.layers, ceil_div(g.page_bytes, kSmall * 1024)}) ||
            pairs * g.layers * ceil_div(g.page_bytes, kSmall * 1024) > INT32_MAX)
            return MI_ERR_UNSUPPORTED;
    }
    return MI_OK;
}

// Copies n pairs, or the first *count of them.
static void copy_launch(PageCaches c, const int* src, const int* dst, int64_t n, const int* count,
                        int* status, bool check, hipStream_t s) {
    const auto waves_of = [&](int kb) {
        int64_t w = 0;
        for (int k = 0; k < c.n; ++k) {
            c.pieces[k] = c.unit[k] == 16 ? ceil_div(c.bytes[k], kb * 1024) : 1;
            const int64_t tasks = n * c.layers[k] * c.pieces[k];
            w += c.unit[k] == 16 || check ? tasks : ceil_div(tasks, 8);
        }
        return w;
    };
    // 8 KB a wave, in a grid that fills the GPU once, where that leaves each wave several
    // (1.07 GB moved: 190 us, 268 with 2 KB); 2 KB a wave for fewer (174 MB: 34 us, 38 with 8 KB)
    const bool large = count || waves_of(kLarge) > 32768;
    const int64_t waves = waves_of(large ? kLarge : kSmall);
    if (waves == 0) return;
    const Pairs p{src, dst, status, static_cast<int>(n), check};
    const dim3 grid(static_cast<unsigned>(std::min(ceil_div(waves, 4), large ? int64_t{2048} : int64_t{1} << 20)));
    if (large) pages_copy_kernel<kLarge><<<grid, dim3(256), 0, s>>>(c, p, count);
    else pages_copy_kernel<kSmall><<<grid, dim3(256), 0, s>>>(c, p, count);
}

static int page_state(int* table, int* seq, int* ref, int64_t B, int64_t mb, int64_t num_blocks, PageState& p) {
    if (B < 0 || mb < 0 || num_blocks < 0) return MI_ERR_INVALID_ARGUMENT;
    if (B > INT32_MAX / 4 || mb > INT32_MAX / 4 || num_blocks > INT32_MAX - 4096) return MI_ERR_UNSUPPORTED;
    if ((B > 0 && mb > 0 && !table) || (num_blocks > 0 && !ref) || !product_fits({B, mb, 4}))
        return MI_ERR_INVALID_ARGUMENT;
    p = PageState{table, seq, ref, B, mb, num_blocks};
    return MI_OK;
}

}  // namespace mi

extern "C" int mi_kv_pages_copy(const mi_kv_pages* caches, int num_caches, int64_t num_blocks,
                                const int* src, const int* dst, int64_t n, int* status, void* stream) {
    using namespace mi;
    if (n < 0) return MI_ERR_INVALID_ARGUMENT;
    PageCaches c;
    const int st = page_caches(caches, num_caches, num_blocks, n, c);
    if (st != MI_OK) return st;
    if (n == 0) return MI_OK;
    if (!src || !dst || !status) return MI_ERR_INVALID_ARGUMENT;
    if (n > (1 << 20)) return MI_ERR_UNSUPPORTED;
    const hipStream_t s = as_stream(stream);
    const bool check = n <= kInline && c.n > 0;
    if (!check)
        pages_check_kernel<<<dim3(static_cast<unsigned>(n)), dim3(256), 0, s>>>(src, dst, static_cast<int>(n), num_blocks, status);
    copy_launch(c, src, dst, n, nullptr, status, check, s);
    return launch_status();
}

extern "C" int mi_kv_pages_free(int* block_table, int* seq_len, int* ref_count, int64_t B,
                                int64_t max_blocks_per_seq, int64_t num_blocks, const int* rows,
                                int64_t n, void* stream) {
    using namespace mi;
    PageState p;
    const int st = page_state(block_table, seq_len, ref_count, B, max_blocks_per_seq, num_blocks, p);
    if (st != MI_OK) return st;
    if (n < 0) return MI_ERR_INVALID_ARGUMENT;
    if (n == 0) return MI_OK;
    if (!rows || (B > 0 && !seq_len)) return MI_ERR_INVALID_ARGUMENT;
    if (n > (1 << 20)) return MI_ERR_UNSUPPORTED;
    pages_free_kernel<<<dim3(static_cast<unsigned>(n)), dim3(256), 0, as_stream(stream)>>>(p, rows, static_cast<int>(n));
    return launch_status();
}

extern "C" int mi_kv_pages_fork(int* block_table, int* seq_len, int* ref_count, int64_t B,
                                int64_t max_blocks_per_seq, int64_t num_blocks, const int* parents,
                                const int* children, int64_t n, int* status, void* stream) {
    using namespace mi;
    PageState p;
    const int st = page_state(block_table, seq_len, ref_count, B, max_blocks_per_seq, num_blocks, p);
    if (st != MI_OK) return st;
    if (n < 0) return MI_ERR_INVALID_ARGUMENT;
    if (n == 0) return MI_OK;
    if (!parents || !children || !status || (B > 0 && !seq_len)) return MI_ERR_INVALID_ARGUMENT;
    if (n > (1 << 20)) return MI_ERR_UNSUPPORTED;
    pages_fork_kernel<<<dim3(static_cast<unsigned>(n)), dim3(256), 0, as_stream(stream)>>>(
        p, parents, children, static_cast<int>(n), status);
    return launch_status();
}

extern "C" int64_t mi_kv_pages_workspace_bytes(int64_t num_blocks, int64_t n) {
    if (num_blocks < 0 || n < 0 || num_blocks > INT32_MAX || n > INT32_MAX) return MI_ERR_INVALID_ARGUMENT;
    return 4 * (2 * num_blocks + 2 * n + 4);
}

extern "C" int mi_kv_pages_reserve(const mi_kv_pages* caches, int num_caches, int* block_table,
                                   int* seq_len, int* ref_count, int64_t B,
                                   int64_t max_blocks_per_seq, int64_t num_blocks,
                                   int64_t block_size, const int* rows, const int* lengths,
                                   int64_t n, int* status, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    using namespace mi;
    if (n < 0 || block_size <= 0) return MI_ERR_INVALID_ARGUMENT;
    PageState p;
    int st = page_state(block_table, seq_len, ref_count, B, max_blocks_per_seq, num_blocks, p);
    if (st != MI_OK) return st;
    if (n > kRowsMax || block_size > INT32_MAX || !product_fits({max_blocks_per_seq, block_size}) ||
        max_blocks_per_seq * block_size > INT32_MAX)
        return MI_ERR_UNSUPPORTED;
    PageCaches c;
    st = page_caches(caches, num_caches, num_blocks, n, c);
    if (st != MI_OK) return st;
    if (n == 0) return MI_OK;
    if (!rows || !lengths || !status || (B > 0 && !seq_len) || !workspace ||
        (reinterpret_cast<uintptr_t>(workspace) & 3) ||
        workspace_bytes < mi_kv_pages_workspace_bytes(num_blocks, n))
        return MI_ERR_INVALID_ARGUMENT;
    Reserve a{};
    a.p = p;
    a.rows = rows;
    a.lengths = lengths;
    a.status = status;
    a.fresh = static_cast<int*>(workspace);
    a.cp_src = a.fresh + num_blocks;
    a.cp_dst = a.cp_src + n;
    a.bs = block_size;
    a.n = static_cast<int>(n);
    const hipStream_t s = as_stream(stream);
    pages_reserve_kernel<<<dim3(1), dim3(1024), 0, s>>>(a);
    copy_launch(c, a.cp_src, a.cp_dst, n, nullptr, nullptr, false, s);
    return launch_status();
}

extern "C" int mi_kv_pages_compact(const mi_kv_pages* caches, int num_caches, int* block_table,
                                   int* ref_count, int64_t B, int64_t max_blocks_per_seq,
                                   int64_t num_blocks, int* moved, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
    using namespace mi;
    PageState p;
    int st = page_state(block_table, nullptr, ref_count, B, max_blocks_per_seq, num_blocks, p);
    if (st != MI_OK) return st;
    PageCaches c;
    const int64_t most = num_blocks / 2;  // movers and their holes are different pages
    st = page_caches(caches, num_caches, num_blocks, most, c);
    if (st != MI_OK) return st;
    if (num_blocks == 0) return MI_OK;
    if (!moved || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
        workspace_bytes < mi_kv_pages_workspace_bytes(num_blocks, 0))
        return MI_ERR_INVALID_ARGUMENT;
    int* const src = static_cast<int*>(workspace);
    int* const dst = src + num_blocks;
    int* const count = dst + num_blocks;
    const hipStream_t s = as_stream(stream);
    pages_plan_kernel<<<dim3(1), dim3(1024), 0, s>>>(ref_count, num_blocks, moved, src, dst, count);
    copy_launch(c, src, dst, most, count, nullptr, false, s);
    if (B * max_blocks_per_seq > 0)
        pages_remap_kernel<<<dim3(static_cast<unsigned>(std::min<int64_t>(ceil_div(B * max_blocks_per_seq, 256), 4096))),
                             dim3(256), 0, s>>>(block_table, B * max_blocks_per_seq, moved, num_blocks);
    return launch_status();
}
