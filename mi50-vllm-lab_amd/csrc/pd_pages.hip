// Block tables and reference counts of a paged cache, on the device: the tables of a serving step from those before it
// (fork) and the used pages moved into the lowest numbers (compact). refs[p] says how many table entries name page p; a page
// of count 0 is free, and free pages are handed out lowest first, so every result is fixed by the inputs.
//
// Fork. New row i goes on from row p = parents[i] of n = seq_lens[p] keys, f = n / block_size full pages. The old rows' references
// are dropped and the new rows' counted. Of the columns below ceil((n + grow) / block_size):
//   column c < f keeps p's entry, and so shares the page, unless every key of it lies behind the window: at or past `sinks` and
//     before n + 1 - window, what the next token at position n and all later ones do not see; then -1;
//   column c >= f has to be the row's own: the first child of p keeps p's entry if nothing else names that page (count 1);
//     else the row takes a free page, and column f's keys [f block_size, n) are copied into it.
// The r-th page that is taken, in the order of (row, column), is the r-th lowest free page of the counts before the call.
//
// Compact. Of n used pages, those numbered n or above move into the free ones below n, in order: the page with r used ones
// of [n, itself) before it goes to the r-th free page.
//
// Both need ranks in the free pages. A first launch turns the counts into bit masks (free, count 1) and counts per 1,024 pages;
// then any thread of the second finds the r-th free page, or a page's rank, from the prefix of those counts (in LDS), 16 mask
// words and population counts: no list of free pages is built, and tables, counts and copies run in one launch.
// The masks also hold the counts as they were, so refs may be updated in place.
//
// What bounds it: small calls their two launches. A step of 48 rows of 1,876 columns takes 3.1 us for masks and plan and 4.9 for the
// tables, each a few trips to memory that wait for one another. Large calls move pages: 64 rows that each copy a part-filled page in 16
// layers 2.9 + 7.8 us for 25 MB; a pool of 6,144 pages of 33,280 bytes, 55 % used, in 8 layers 4.7 + 170 us for 807 MB, 4.7 TB/s, the
// rate of a 4 GiB copy. Room for many new keys costs the plan: a row's thread walks the columns from the last full page on one after
// the other, a table entry each and, where one is named, its count. 48 rows in pages of 16 take 9.1 us with grow 1, 10.0 with 100, 29 with 2,048
// and 95 with 8,192, and 42 and 152 if their tables already have that room; one row 22 and 74 (30 and 103).
#include "pd_tile.hpp"
#include "pth_dec.h"

namespace pd {

constexpr int kPgThreads = 256;
constexpr int kPgChunk = 1024;                             // pages of a count
constexpr int kPgWords = kPgChunk / 64;                    // mask words of a chunk
constexpr int kPgMaxChunks = (int)(kMaxPages / kPgChunk);  // prefix of the counts in LDS

typedef unsigned long long word_t;
typedef word_t word2_t __attribute__((ext_vector_type(2)));

// Exclusive sum over the workgroup's threads and the total. `part` holds a value per wave.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* part, unsigned& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned incl = wave_scan(v);
    __syncthreads();  // the last use of `part` is over
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    unsigned before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPgThreads / 64; ++i) {
        const unsigned x = part[i];
        before += i < wave ? x : 0u;
        total += x;
    }
    return before + incl - v;
}

// The counts' prefix of a launch: before[c] = free pages below chunk c. Returns the free pages.
__device__ __forceinline__ unsigned load_prefix(const PageWork& w, unsigned* before, unsigned* part) {
    unsigned run = 0;
    for (int c0 = 0; c0 < w.chunks; c0 += kPgThreads) {
        const int c = c0 + (int)threadIdx.x;
        unsigned total;
        const unsigned ex = block_scan(c < w.chunks ? (unsigned)w.counts[c] : 0u, part, total);
        if (c < w.chunks) before[c] = run + ex;
        run += total;
    }
    __syncthreads();
    return run;
}

// Page of the r-th set bit (kFree) or clear bit of the free mask, r below their number.
template <bool kFree>
__device__ __forceinline__ int select_page(const PageWork& w, const unsigned* before, unsigned r) {
    int lo = 0, hi = w.chunks - 1;  // the last chunk that begins at or below rank r
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const unsigned at = kFree ? before[mid] : (unsigned)mid * kPgChunk - before[mid];
        if (at <= r)
            lo = mid;
        else
            hi = mid - 1;
    }
    unsigned left = r - (kFree ? before[lo] : (unsigned)lo * kPgChunk - before[lo]);
    word_t m[kPgWords];
    const word2_t* src = reinterpret_cast<const word2_t*>(w.free_mask + (int64_t)lo * kPgWords);
#pragma unroll
    for (int i = 0; i < kPgWords / 2; ++i) {
        const word2_t x = src[i];
        m[2 * i] = kFree ? x.x : ~x.x;
        m[2 * i + 1] = kFree ? x.y : ~x.y;
    }
    word_t word = 0;
    int at = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kPgWords; ++i) {
        const unsigned k = (unsigned)__popcll(m[i]);
        if (!found && left < k) {
            found = true;
            word = m[i];
            at = i;
        }
        if (!found) left -= k;
    }
    // bit number `left` of the word, by halves
    int bit = 0;
#pragma unroll
    for (int h = 32; h >= 1; h >>= 1) {
        const unsigned k = (unsigned)__popcll(word & ((word_t(1) << h) - 1));
        if (left >= k) {
            left -= k;
            word >>= h;
            bit += h;
        }
    }
    return lo * kPgChunk + at * 64 + bit;
}

// Free pages below page x < pages.
__device__ __forceinline__ unsigned rank_free(const PageWork& w, const unsigned* before, int x) {
    const int c = x / kPgChunk, last = (x % kPgChunk) / 64;
    const word2_t* src = reinterpret_cast<const word2_t*>(w.free_mask + (int64_t)c * kPgWords);
    unsigned r = before[c];
#pragma unroll
    for (int i = 0; i < kPgWords / 2; ++i) {
        const word2_t m = src[i];
        const word_t below = (word_t(1) << (x & 63)) - 1;
        r += 2 * i < last ? (unsigned)__popcll(m.x) : 2 * i == last ? (unsigned)__popcll(m.x & below) : 0u;
        r += 2 * i + 1 < last ? (unsigned)__popcll(m.y) : 2 * i + 1 == last ? (unsigned)__popcll(m.y & below) : 0u;
    }
    return r;
}
__device__ __forceinline__ bool mask_bit(const word_t* mask, int page) { return (mask[page >> 6] >> (page & 63)) & 1; }

// One chunk's masks and count; a fork's counts also go to new_refs, where that is another array or they are below 0 (as 0: the page
// may be taken, and is counted from there).
__device__ __forceinline__ void count_chunk(const PageWork& w, const int* refs, int* new_refs, int chunk, unsigned* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned n = 0;
#pragma unroll
    for (int j = 0; j < kPgChunk / kPgThreads; ++j) {
        const int word = wave * (kPgChunk / kPgThreads) + j, page = chunk * kPgChunk + word * 64 + lane;
        const int r = page < w.pages ? refs[page] : 2;  // (past the last page neither free nor alone)
        if (page < w.pages && new_refs && (new_refs != refs || r < 0)) new_refs[page] = max(r, 0);
        const word_t free = __ballot(r <= 0), alone = __ballot(r == 1);
        if (lane == 0) {
            w.free_mask[(int64_t)chunk * kPgWords + word] = free;
            w.alone_mask[(int64_t)chunk * kPgWords + word] = alone;
        }
        n += (unsigned)__popcll(free);
    }
    if (lane == 0) part[wave] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned total = 0;
        for (int i = 0; i < kPgThreads / 64; ++i) total += part[i];
        w.counts[chunk] = (int)total;
    }
}

// First launch of a compaction: a chunk of the counts per workgroup, 64 pages a wave and step: a launch and one trip to memory,
// 2.6 to 4.8 us.
__global__ void __launch_bounds__(kPgThreads) pd_pages_count_kernel(const PageWork w, const int* refs) {
    __shared__ unsigned part[kPgThreads / 64];
    count_chunk(w, refs, nullptr, (int)blockIdx.x, part);
}

// What a new row takes over: its parent's keys n, full pages, and the columns that it holds.
struct RowPlan {
    int parent;  // -1: an empty row
    int64_t n;
    int full, end;
};
__device__ __forceinline__ RowPlan row_plan(const ForkParams& a, int i) {
    RowPlan r;
    r.parent = a.parents ? a.parents[i] : i;
    if (r.parent < 0 || r.parent >= a.rows) r.parent = -1;
    r.n = r.parent >= 0 ? max(0, a.seq_lens[r.parent]) : 0;
    const int64_t end = (r.n + a.grow + a.block_size - 1) / a.block_size;
    r.end = r.parent >= 0 ? (int)min(end, (int64_t)a.cols) : 0;
    r.full = (int)min(r.n / a.block_size, (int64_t)a.cols);
    return r;
}
__device__ __forceinline__ bool names_page(const ForkParams& a, int e) { return e >= 0 && e < a.w.pages; }

// First launch of a fork: workgroup 0 plans the new rows (the first child of each old row, how many pages the rows before
// each new row take, and the list of the pages whose keys are copied), the others take one chunk of the counts each.
__global__ void __launch_bounds__(kPgThreads) pd_fork_plan_kernel(const ForkParams a) {
    __shared__ int eldest[kMaxForkRows];
    __shared__ unsigned part[kPgThreads / 64];
    if (blockIdx.x > 0) {
        count_chunk(a.w, a.refs, a.new_refs, (int)blockIdx.x - 1, part);
        return;
    }
    const int tid = threadIdx.x;
    if (a.parents) {
        for (int b = tid; b < a.rows; b += kPgThreads) eldest[b] = INT32_MAX;
        __syncthreads();
        for (int i = tid; i < a.new_rows; i += kPgThreads) {
            const int p = a.parents[i];
            if (p >= 0 && p < a.rows) atomicMin(&eldest[p], i);
        }
        __syncthreads();
        for (int b = tid; b < a.rows; b += kPgThreads) a.eldest[b] = eldest[b];
    }
    unsigned run = 0, ncopies = 0;
    for (int i0 = 0; i0 < a.new_rows; i0 += kPgThreads) {
        const int i = i0 + tid;
        unsigned takes = 0;
        int src = -1, keys = 0;
        if (i < a.new_rows) {
            const RowPlan r = row_plan(a, i);
            if (r.parent >= 0) {
                const int* row = a.table + (int64_t)r.parent * a.t_st;
                const bool heir = !a.parents || eldest[r.parent] == i;
                takes = (unsigned)max(0, r.end - r.full);
                bool first_kept = false;
                if (heir)
                    for (int c = r.full; c < r.end; ++c) {
                        const int e = row[c];
                        const bool kept = names_page(a, e) && a.refs[e] == 1;
                        takes -= kept ? 1u : 0u;
                        if (c == r.full) first_kept = kept;
                    }
                // (the part-filled page is the row's first column of its own, so its copy takes the row's first page)
                if (r.full < r.end && (int64_t)r.full * a.block_size < r.n && !first_kept) {
                    const int e = row[r.full];
                    src = names_page(a, e) ? e : -1;
                    keys = (int)(r.n - (int64_t)r.full * a.block_size);
                }
            }
        }
        unsigned total;
        const unsigned ex = block_scan(takes, part, total), run_before = run;
        if (i < a.new_rows) a.first_taken[i] = (int)(run + ex);
        run += total;
        const unsigned at = ncopies + block_scan(src >= 0 ? 1u : 0u, part, total);
        if (src >= 0) a.copy_list[at] = PageCopy{src, (int)(run_before + ex), keys};
        ncopies += total;
    }
    if (tid == 0) {
        a.needed[0] = (int)run;
        a.copies[0] = (int)ncopies;
    }
}

// `len` bytes, 8-byte aligned, by a wave, 8 KiB of them in flight.
__device__ __forceinline__ void copy_bytes(int8_t* dst, const int8_t* src, int64_t len) {
    const int lane = threadIdx.x & 63;
    const uintptr_t d = reinterpret_cast<uintptr_t>(dst);
    if (((d ^ reinterpret_cast<uintptr_t>(src)) & 15) == 0) {
        const int64_t head = (d & 15) && len ? 8 : 0, body = (len - head) / 16, tail = len - head - 16 * body;
        const uint4_t* s = reinterpret_cast<const uint4_t*>(src + head);
        uint4_t* o = reinterpret_cast<uint4_t*>(dst + head);
        if (lane == 0 && head) *reinterpret_cast<uint64_t*>(dst) = *reinterpret_cast<const uint64_t*>(src);
        if (lane == 1 && tail) *reinterpret_cast<uint64_t*>(dst + len - 8) = *reinterpret_cast<const uint64_t*>(src + len - 8);
        constexpr int kAhead = 8;
        for (int64_t i0 = lane; i0 < body; i0 += kAhead * 64) {
            uint4_t x[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i0 + k * 64 < body) x[k] = s[i0 + k * 64];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (i0 + k * 64 < body) o[i0 + k * 64] = x[k];
        }
    } else {
        for (int64_t i = lane; i < len / 8; i += 64)
            reinterpret_cast<uint64_t*>(dst)[i] = reinterpret_cast<const uint64_t*>(src)[i];
    }
}

// Piece `t` of the first `keys` keys of a page: the page's rows in runs of adjacent bytes, each run in `cuts` pieces.
__device__ __forceinline__ void copy_piece(const PageCaches& k, int layer, int from, int to, int t, int64_t keys) {
    const int run = t / k.cuts, cut = t - run * k.cuts;
    int64_t at, len;
    if (k.form == kPageWhole) {  // all rows adjacent, keys first: whole pages, or tokens-major ones
        at = 0;
        len = keys * k.key_bytes;
    } else if (k.form == kPageHeads) {  // a head's keys adjacent
        at = run * k.sh;
        len = keys * kRowBytes;
    } else {  // rows apart
        const int h = run / k.block_size, s = run - h * k.block_size;
        at = h * k.sh + s * k.ss;
        len = s < keys ? kRowBytes : 0;
    }
    const int64_t per = (len / k.cuts + 15) / 16 * 16, b0 = min(len, cut * per), b1 = cut + 1 == k.cuts ? len : min(len, b0 + per);
    int8_t* kv = k.kv[layer];
    copy_bytes(kv + (int64_t)to * k.sb + at + b0, kv + (int64_t)from * k.sb + at + b0, b1 - b0);
}

// Second launch of a fork: workgroups [0, new_rows) write a table row each, the next `rows` (with parents) drop the
// references of old rows without children, the others copy pieces of pages.
__global__ void __launch_bounds__(kPgThreads) pd_fork_kernel(const ForkParams a, const PageCaches k) {
    __shared__ unsigned before[kPgMaxChunks];
    __shared__ unsigned part[kPgThreads / 64];
    const int tid = threadIdx.x;
    int wg = (int)blockIdx.x;
    if (wg < a.new_rows) {
        const int i = wg;
        const RowPlan r = row_plan(a, i);
        const bool heir = r.parent >= 0 && (!a.parents || a.eldest[r.parent] == i);
        const int* row = a.table + (int64_t)max(0, r.parent) * a.t_st;
        int* out = a.new_table + (int64_t)i * a.n_st;
        // Full pages, and the columns behind the row's: each entry stands for itself, so four of a thread's are in flight.
        auto plain = [&](int c0, int c1, bool full) __attribute__((always_inline)) {
            constexpr int kAhead = 4;
            for (int b = c0 + tid; b < c1; b += kAhead * kPgThreads) {
                int e[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) e[k] = b + k * kPgThreads < c1 && r.parent >= 0 ? row[b + k * kPgThreads] : -1;
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int c = b + k * kPgThreads;
                    if (c >= c1) break;
                    const int64_t k0 = (int64_t)c * a.block_size;
                    const bool named = names_page(a, e[k]);
                    const bool stays = full && named && !(a.window > 0 && k0 >= a.sinks && k0 + a.block_size <= r.n + 1 - a.window);
                    if (heir && named && !stays) atomicAdd(a.new_refs + e[k], -1);
                    if (!heir && stays) atomicAdd(a.new_refs + e[k], 1);
                    out[c] = stays ? e[k] : -1;
                }
            }
        };
        const int full = min(r.full, r.end);
        plain(0, full, true);
        plain(r.end, a.cols, false);
        // the row's own columns
        unsigned run = (unsigned)a.first_taken[i], nfree = 0;
        bool have_prefix = false;
        for (int c0 = full; c0 < r.end; c0 += kPgThreads) {
            const int c = c0 + tid;
            int e = -1, v = -1;
            bool takes = false;
            if (c < r.end) {
                e = row[c];
                if (!names_page(a, e)) e = -1;
                takes = !(heir && e >= 0 && mask_bit(a.w.alone_mask, e));
                v = takes ? -1 : e;
            }
            unsigned total;
            const unsigned rank = run + block_scan(takes ? 1u : 0u, part, total);
            if (total > 0 && !have_prefix) {
                nfree = load_prefix(a.w, before, part);
                have_prefix = true;
            }
            if (takes && rank < nfree) v = select_page<true>(a.w, before, rank);
            run += total;
            if (c < r.end) {
                if (heir && e >= 0 && takes) atomicAdd(a.new_refs + e, -1);
                if (v >= 0 && takes) atomicAdd(a.new_refs + v, 1);
                out[c] = v;
            }
        }
        if (tid == 0) a.new_lens[i] = (int)r.n;
        return;
    }
    wg -= a.new_rows;
    if (a.parents) {
        if (wg < a.rows) {
            if (a.eldest[wg] != INT32_MAX) return;
            const int* row = a.table + (int64_t)wg * a.t_st;
            for (int c = tid; c < a.cols; c += kPgThreads) {
                const int e = row[c];
                if (names_page(a, e)) atomicAdd(a.new_refs + e, -1);
            }
            return;
        }
        wg -= a.rows;
    }
    // (a run of pieces per wave: they are mostly of one page, which is then looked up once)
    const int64_t nwave = (int64_t)((int)gridDim.x - a.new_rows - (a.parents ? a.rows : 0)) * (kPgThreads / 64);
    const int pieces = k.runs * k.cuts, each = k.layers * pieces;
    const int64_t tasks = (int64_t)a.copies[0] * each, per = (tasks + nwave - 1) / nwave;
    if ((int64_t)wg * (kPgThreads / 64) * per >= tasks) return;
    const unsigned nfree = load_prefix(a.w, before, part);
    const int64_t t0 = ((int64_t)wg * (kPgThreads / 64) + __builtin_amdgcn_readfirstlane(tid >> 6)) * per;
    int known = -1, to = -1;
    PageCopy copy = {};
    for (int64_t t = t0; t < min(tasks, t0 + per); ++t) {
        const int j = (int)(t / each), x = (int)(t - (int64_t)j * each), layer = x / pieces;
        if (j != known) {
            known = j;
            copy = a.copy_list[j];
            to = (unsigned)copy.rank < nfree ? select_page<true>(a.w, before, (unsigned)copy.rank) : -1;
        }
        if (to >= 0) copy_piece(k, layer, copy.from, to, x - layer * pieces, copy.keys);
    }
}

// Second launch of a compaction: workgroups [0, chunks) write places and counts, the next `rows` a table row each, the
// others copy pieces of pages.
__global__ void __launch_bounds__(kPgThreads) pd_compact_kernel(const CompactParams a, const PageCaches k) {
    __shared__ unsigned before[kPgMaxChunks];
    __shared__ unsigned part[kPgThreads / 64];
    const int tid = threadIdx.x;
    int wg = (int)blockIdx.x;
    const int used = a.w.pages - (int)load_prefix(a.w, before, part);
    const unsigned moves = used < a.w.pages ? rank_free(a.w, before, used) : 0u;  // free pages below `used`
    const unsigned r0 = (unsigned)used - moves;                                    // used pages below `used`
    auto place_of = [&](int page) {
        if (mask_bit(a.w.free_mask, page)) return -1;
        if (page < used) return page;
        return select_page<true>(a.w, before, (unsigned)page - rank_free(a.w, before, page) - r0);
    };
    if (wg < a.w.chunks) {
        if (wg == 0 && tid == 0) a.used[0] = used;
#pragma unroll 1
        for (int j = 0; j < kPgChunk / kPgThreads; ++j) {
            const int page = wg * kPgChunk + j * kPgThreads + tid;
            if (page >= a.w.pages) break;
            const int to = place_of(page);
            a.places[page] = to;
            // (a free page below `used` gets its count from the page that moves into it)
            if (to >= 0) {
                const int r = a.refs[page];
                a.new_refs[to] = r;
                if (to != page) a.new_refs[page] = 0;
            } else if (page >= used) {
                a.new_refs[page] = 0;
            }
        }
        return;
    }
    wg -= a.w.chunks;
    if (wg < a.rows) {
        for (int c = tid; c < a.cols; c += kPgThreads) {
            const int e = a.table[(int64_t)wg * a.t_st + c];
            a.new_table[(int64_t)wg * a.n_st + c] = e >= 0 && e < a.w.pages ? place_of(e) : -1;
        }
        return;
    }
    wg -= a.rows;
    const int64_t nwave = (int64_t)((int)gridDim.x - a.w.chunks - a.rows) * (kPgThreads / 64);
    const int pieces = k.runs * k.cuts, each = k.layers * pieces;
    const int64_t tasks = (int64_t)moves * each, per = (tasks + nwave - 1) / nwave;
    const int64_t t0 = ((int64_t)wg * (kPgThreads / 64) + __builtin_amdgcn_readfirstlane(tid >> 6)) * per;
    unsigned known = 0xffffffffu;
    int from = 0, to = 0;
    for (int64_t t = t0; t < min(tasks, t0 + per); ++t) {
        const unsigned m = (unsigned)(t / each);
        const int x = (int)(t - (int64_t)m * each), layer = x / pieces;
        if (m != known) {
            known = m;
            from = select_page<false>(a.w, before, r0 + m);
            to = select_page<true>(a.w, before, m);
        }
        copy_piece(k, layer, from, to, x - layer * pieces, a.block_size);
    }
}

// ---------------------------------------------------------------------------------------
// host side

// How a page's bytes are copied, whole pages or some of their first keys.
static void plan_copies(PageCaches& k, bool whole) {
    const int64_t head = k.block_size * kRowBytes;
    if (k.sh == kRowBytes && k.ss == k.Hkv * kRowBytes)  // tokens-major
        k.form = kPageWhole, k.runs = 1, k.key_bytes = k.Hkv * kRowBytes;
    else if (whole && k.ss == kRowBytes && k.sh == head)
        k.form = kPageWhole, k.runs = 1, k.key_bytes = k.Hkv * kRowBytes;
    else if (k.ss == kRowBytes)
        k.form = kPageHeads, k.runs = k.Hkv, k.key_bytes = kRowBytes;
    else
        k.form = kPageRows, k.runs = k.Hkv * k.block_size, k.key_bytes = kRowBytes;
    const int64_t longest = k.form == kPageRows ? kRowBytes : k.key_bytes * k.block_size;
    k.cuts = (int)((longest + kPagePiece - 1) / kPagePiece);
}

static int64_t copy_groups(int64_t tasks) {
    const int64_t wanted = (tasks + kPgThreads / 64 - 1) / (kPgThreads / 64);
    return wanted < kPageCopyGroups ? wanted : kPageCopyGroups;
}

hipError_t launch_fork(ForkParams p, PageCaches k, hipStream_t stream) {
    plan_copies(k, false);
    hipLaunchKernelGGL(pd_fork_plan_kernel, dim3(1 + p.w.chunks), dim3(kPgThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t tasks = (int64_t)p.new_rows * k.layers * k.runs * k.cuts;
    const int64_t wgs = p.new_rows + (p.parents ? p.rows : 0) + copy_groups(tasks);
    if (wgs == 0) return hipSuccess;
    hipLaunchKernelGGL(pd_fork_kernel, dim3((unsigned)wgs), dim3(kPgThreads), 0, stream, p, k);
    return hipGetLastError();
}

hipError_t launch_compact(const CompactParams& p, PageCaches k, hipStream_t stream) {
    plan_copies(k, true);
    hipLaunchKernelGGL(pd_pages_count_kernel, dim3(p.w.chunks), dim3(kPgThreads), 0, stream, p.w, p.refs);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t tasks = (int64_t)(p.w.pages / 2) * k.layers * k.runs * k.cuts;  // at most half of the pages move
    const int64_t wgs = p.w.chunks + p.rows + copy_groups(tasks);
    hipLaunchKernelGGL(pd_compact_kernel, dim3((unsigned)wgs), dim3(kPgThreads), 0, stream, p, k);
    return hipGetLastError();
}

}  // namespace pd
