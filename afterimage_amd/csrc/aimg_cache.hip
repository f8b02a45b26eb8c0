// Pages of a key/value cache: appending rows, forking, reserving, releasing,
// committing accepted drafts and compacting (gfx950).
//
// The page table, lengths, pages held and reference counts live on the GPU and
// every step runs there, so that a verification step (append, attend, commit)
// never waits for the host. Free pages are those without references; they are
// given out lowest first, in the order of the call's sequences, so that a
// call's result follows from its arguments alone (counts change by atomics,
// whose order a sum does not show).
//
// A step that scans the pages is one workgroup, 4096 reference counts a round:
// for pools of some hundred pages 5 us of dependent reads (slot, length, pages
// held, counts), for larger ones about 1 us more a round (compacting: 3). What
// moves rows is a grid of its own, bound by HBM: 16 bytes a lane, whole rows
// of a head at a time.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "afterimage_decode.h"
#include "aimg_internal.h"

namespace aimg {
namespace {

constexpr int kScan = 1024;                // threads of a scanning workgroup
constexpr int kEach = 4;                   // pages of a thread and round
constexpr int kMaxSeqs = 8192;             // sequences of one call (its counts are held in LDS)
constexpr int kWaves = kScan / 64;
constexpr int32_t kMaxPoolPages = (1 << 20) - 1;
constexpr int32_t kManyPages = 1 << 30;

constexpr int32_t kNoPages = 1, kRowFull = 2, kBadIndex = 4;  // bits of the status word

struct Cache {
    char* pool;
    int32_t *table, *lengths, *held, *refs, *status;
    int64_t plane_bytes, page_bytes, head_bytes;
    int32_t planes, n_pages, kv_heads, page_size, row_bytes, max_seqs, max_pages, table_stride;
};

__device__ __forceinline__ void tell(const Cache& C, int32_t what) { atomicOr(C.status, what); }

__device__ __forceinline__ bool known(const Cache& C, int32_t slot) { return slot >= 0 && slot < C.max_seqs; }

__device__ __forceinline__ int32_t length_of(const Cache& C, int32_t slot) {
    const int32_t n = C.lengths[slot], most = C.max_pages * C.page_size;
    return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ int32_t held_of(const Cache& C, int32_t slot) {
    const int32_t n = C.held[slot];
    return n < 0 ? 0 : n > C.max_pages ? C.max_pages : n;
}

// Sum of v over the threads before this one; all threads of the workgroup call it.
__device__ int32_t sum_before(int32_t v, int32_t* wave_sums, int32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t s = v;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const int32_t o = __shfl_up(s, x);
        if (lane >= x) s += o;
    }
    __syncthreads();
    if (lane == 63) wave_sums[wave] = s;
    __syncthreads();
    int32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += wave_sums[w];
        all += wave_sums[w];
    }
    total = all;
    return before + s - v;
}

// The counts[i] of n sequences into sums before each, in place; returns their
// sum, or kManyPages where it is more. (A count is below 2^20, so a round's sum fits.)
__device__ int32_t sums_of(int32_t* counts, int n, int32_t* wave_sums) {
    int32_t done = 0;
    for (int i0 = 0; i0 < n; i0 += kScan) {
        const int i = i0 + threadIdx.x;
        int32_t total;
        const int32_t v = i < n ? counts[i] : 0;
        const int32_t at = sum_before(v, wave_sums, total);
        if (i < n) counts[i] = done + at;
        done = done + total < kManyPages ? done + total : kManyPages;
    }
    __syncthreads();
    return done;
}

// The reference counts of a round's pages, four neighbours a thread (of page 0
// past the pool: whoever uses them looks at the page's number too).
__device__ __forceinline__ void read_round(const Cache& C, int32_t p0, int32_t (&refs)[kEach]) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int32_t p = p0 + threadIdx.x * kEach + j;
        refs[j] = C.refs[p < C.n_pages ? p : 0];
    }
}

// Calls give(rank, page) for the free pages of lowest index, ranks 0..want-1.
// Returns how many of `want` there were. from: a round before which no page is
// free; becomes the first one with a free page. (A round's counts are read
// while the one before is summed: with that and without the used rounds in
// the second pass, a reservation and a release in a pool of 100,000 used
// pages take 34 us, 81 without.)
template <typename Give>
__device__ int32_t each_free(const Cache& C, int32_t want, int32_t* wave_sums, int32_t& from, Give give) {
    int32_t done = 0, next[kEach];
    read_round(C, from, next);
    for (int32_t p0 = from; p0 < C.n_pages && done < want; p0 += kScan * kEach) {
        const int32_t p = p0 + threadIdx.x * kEach;
        int32_t free = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) free |= (p + j < C.n_pages && next[j] == 0 ? 1 : 0) << j;
        if (p0 + kScan * kEach < C.n_pages) read_round(C, p0 + kScan * kEach, next);
        int32_t total;
        int32_t rank = done + sum_before(__popc(free), wave_sums, total);
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (free >> j & 1) {
                if (rank < want) give(rank, p + j);
                ++rank;
            }
        if (done == 0 && total == 0) from = p0 + kScan * kEach;
        done += total;
    }
    return done < want ? done : want;
}

__device__ __forceinline__ uint4 get16(const char* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void put16(char* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }

// --------------------------------------------------------------------------
// Rows into pages.
// --------------------------------------------------------------------------

struct AppendArgs {
    Cache c;
    const char *k, *v;
    int64_t k_row, k_head, v_row, v_head;  // bytes
    const int32_t *seqs, *offsets;
    int64_t layer_at;  // of the layer's keys in the pool; its values follow a plane later
    int32_t n_seqs, n_rows;
};

// 16 bytes a thread, keys and values: a few rows a call (64 sequences of 12
// rows, 8 heads of 128: 3 MB), bound by the launch; many rows by HBM.
__global__ __launch_bounds__(256) void append_kernel(const AppendArgs A) {
    const Cache& C = A.c;
    const uint32_t pieces = C.row_bytes / 16, i = blockIdx.x * 256u + threadIdx.x;  // fewer than 2^31 in all
    const int32_t x = static_cast<int32_t>(i % pieces);
    const int32_t head = static_cast<int32_t>(i / pieces % C.kv_heads), row = static_cast<int32_t>(i / pieces / C.kv_heads);
    if (row >= A.n_rows) return;
    int lo = 0, hi = A.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (A.offsets[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int32_t first = A.offsets[lo];
    if (row < first || row >= A.offsets[lo + 1]) return;  // a row of no sequence
    const int32_t slot = A.seqs[lo];
    if (!known(C, slot)) return tell(C, kBadIndex);
    const int64_t at = static_cast<int64_t>(length_of(C, slot)) + row - first;  // first may be any int32
    const int64_t page = at / C.page_size;
    if (page >= held_of(C, slot)) return tell(C, kRowFull);
    const int32_t id = C.table[static_cast<int64_t>(slot) * C.table_stride + page];
    if (id < 0 || id >= C.n_pages) return tell(C, kBadIndex);
    char* const to = C.pool + A.layer_at + id * C.page_bytes + head * C.head_bytes + at % C.page_size * C.row_bytes + x * 16;
    put16(to, get16(A.k + row * A.k_row + head * A.k_head + x * 16));
    put16(to + C.plane_bytes, get16(A.v + row * A.v_row + head * A.v_head + x * 16));
}

__global__ __launch_bounds__(256) void advance_kernel(const Cache C, const int32_t* seqs, const int32_t* offsets, int n_seqs) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= n_seqs) return;
    const int32_t slot = seqs[b];
    if (!known(C, slot)) return tell(C, kBadIndex);
    // A length never falls: it could come to lie inside a page that another slot shares.
    const int64_t more = static_cast<int64_t>(offsets[b + 1]) - offsets[b], to = length_of(C, slot) + more;
    if (more < 0) return tell(C, kBadIndex);
    if (to > static_cast<int64_t>(held_of(C, slot)) * C.page_size) return tell(C, kRowFull);
    C.lengths[slot] = static_cast<int32_t>(to);
}

// --------------------------------------------------------------------------
// Pages taken and given back.
// --------------------------------------------------------------------------

// Pages for tokens[b] further positions of each sequence, all or none.
__global__ __launch_bounds__(kScan) void reserve_kernel(const Cache C, const int32_t* seqs, const int32_t* tokens, int n) {
    __shared__ int32_t start[kMaxSeqs];
    __shared__ int32_t wave_sums[kWaves];
    __shared__ int32_t bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    auto need = [&](int i) {
        const int32_t slot = seqs[i];
        if (!known(C, slot) || tokens[i] < 0) {
            atomicOr(&bad, kBadIndex);
            return 0;
        }
        const int64_t to = (static_cast<int64_t>(length_of(C, slot)) + tokens[i] + C.page_size - 1) / C.page_size;
        if (to > C.max_pages) atomicOr(&bad, kRowFull);
        const int64_t more = to - held_of(C, slot);
        if (more > C.n_pages) atomicOr(&bad, kNoPages);
        return more < 0 || more > C.n_pages || to > C.max_pages ? 0 : static_cast<int32_t>(more);
    };
    for (int i = threadIdx.x; i < n; i += kScan) start[i] = need(i);
    __syncthreads();
    const int32_t want = sums_of(start, n, wave_sums);
    int32_t wrong = bad, from = 0;
    if (wrong == 0 && each_free(C, want, wave_sums, from, [](int32_t, int32_t) {}) < want) wrong = kNoPages;
    if (wrong != 0) {
        if (threadIdx.x == 0) tell(C, wrong);
        return;
    }
    // The pass that counted left the counts of references as they were.
    each_free(C, want, wave_sums, from, [&](int32_t rank, int32_t page) {
        int lo = 0, hi = n - 1;  // the last sequence that starts at or before the rank
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (start[mid] <= rank) lo = mid; else hi = mid - 1;
        }
        const int32_t slot = seqs[lo];
        C.table[static_cast<int64_t>(slot) * C.table_stride + held_of(C, slot) + rank - start[lo]] = page;
        C.refs[page] = 1;
    });
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kScan) {
        const int32_t end = i + 1 < n ? start[i + 1] : want;
        if (end > start[i]) C.held[seqs[i]] += end - start[i];
    }
}

// A workgroup a sequence: its references go, its row is emptied. A slot named
// twice is released once: one workgroup takes its count of pages.
__global__ __launch_bounds__(256) void release_kernel(const Cache C, const int32_t* seqs) {
    __shared__ int32_t mine;
    const int32_t slot = seqs[blockIdx.x];
    if (!known(C, slot)) {
        if (threadIdx.x == 0) tell(C, kBadIndex);
        return;
    }
    if (threadIdx.x == 0) {
        const int32_t n = atomicExch(C.held + slot, 0);
        mine = n < 0 ? 0 : n > C.max_pages ? C.max_pages : n;
        C.lengths[slot] = 0;
    }
    __syncthreads();
    int32_t* const row = C.table + static_cast<int64_t>(slot) * C.table_stride;
    for (int32_t i = threadIdx.x; i < mine; i += 256) {
        const int32_t id = row[i];
        row[i] = -1;
        if (id >= 0 && id < C.n_pages) atomicSub(C.refs + id, 1);
    }
}

// --------------------------------------------------------------------------
// Forking: sequence dst[i] becomes a branch of src[i].
// --------------------------------------------------------------------------

struct ForkArgs {
    Cache c;
    const int32_t *src, *dst;
    int32_t* fresh;  // [n]: the pair's new last page, -1 none, -2 the pair stays as it is
    int32_t* lens;   // [n]: the branches' lengths
    int32_t* rows;   // [n][max_pages]: the branches' new rows
    int32_t n;
};

// The new last pages, from those free before the call.
__global__ __launch_bounds__(kScan) void fork_plan_kernel(const ForkArgs A) {
    const Cache& C = A.c;
    __shared__ int32_t start[kMaxSeqs];
    __shared__ int32_t fresh[kMaxSeqs];
    __shared__ int32_t wave_sums[kWaves];
    __shared__ int32_t bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    auto copies = [&](int i) {
        const int32_t s = A.src[i], d = A.dst[i];
        if (!known(C, s) || !known(C, d)) {
            atomicOr(&bad, kBadIndex);
            return 0;
        }
        const int32_t len = length_of(C, s);
        if ((len + C.page_size - 1) / C.page_size > held_of(C, s)) atomicOr(&bad, kBadIndex);
        return s != d && len % C.page_size != 0 ? 1 : 0;
    };
    for (int i = threadIdx.x; i < A.n; i += kScan) start[i] = copies(i);
    __syncthreads();
    const int32_t want = sums_of(start, A.n, wave_sums);
    int32_t wrong = bad, from = 0;
    if (wrong == 0 && each_free(C, want, wave_sums, from, [&](int32_t rank, int32_t page) { fresh[rank] = page; }) < want) wrong = kNoPages;
    __syncthreads();
    if (wrong != 0 && threadIdx.x == 0) tell(C, wrong);
    for (int i = threadIdx.x; i < A.n; i += kScan) {
        const int32_t end = i + 1 < A.n ? start[i + 1] : want;
        A.lens[i] = wrong != 0 ? 0 : length_of(C, A.src[i]);
        A.fresh[i] = wrong != 0 || A.src[i] == A.dst[i] ? -2 : end > start[i] ? fresh[start[i]] : -1;
    }
}

// Workgroup (pair, share of its rows to copy). The first share of a pair also
// counts its references and writes its new row beside the table: a pair's
// source may be another pair's branch, so no row changes before all were read.
// 96 branches, 16 planes of 8 heads of 128: 95 MB written in 39.5 us, and 8 MB
// read, for the sources' tails stay in the caches. That is half of what a copy
// of as many bytes reaches (21 us), and what bounds it is not known. Two, four
// and eight times the rows a thread, or twice as many in flight, took 0.2 to
// 2 us more.
__global__ __launch_bounds__(256) void fork_copy_kernel(const ForkArgs A) {
    const Cache& C = A.c;
    const int i = blockIdx.x;
    const int32_t page = A.fresh[i];
    if (page == -2) return;
    const int32_t s = A.src[i], d = A.dst[i];
    const int32_t len = A.lens[i], full = len / C.page_size, tail = len % C.page_size;
    const int32_t* const from = C.table + static_cast<int64_t>(s) * C.table_stride;
    if (blockIdx.y == 0) {
        const int32_t* const old = C.table + static_cast<int64_t>(d) * C.table_stride;
        const int32_t gone = held_of(C, d);
        for (int32_t x = threadIdx.x; x < C.max_pages; x += 256) {
            int32_t id = -1;
            if (x < full) {
                id = from[x];
                if (id >= 0 && id < C.n_pages) atomicAdd(C.refs + id, 1);
                else tell(C, kBadIndex);
            } else if (x == full && tail > 0) {
                id = page;
                atomicAdd(C.refs + id, 1);
            }
            A.rows[static_cast<int64_t>(i) * C.max_pages + x] = id;
            if (x < gone) {
                const int32_t o = old[x];
                if (o >= 0 && o < C.n_pages) atomicSub(C.refs + o, 1);
            }
        }
    }
    if (tail == 0) return;
    const int32_t last = from[full];
    if (last < 0 || last >= C.n_pages) {
        if (threadIdx.x == 0) tell(C, kBadIndex);
        return;
    }
    // The tail's rows of every head and plane, 16 bytes a thread and step: a
    // thread keeps its place in a head's rows and steps over heads and planes,
    // so it divides once (a division a step took longer than the bytes).
    const uint32_t pieces = static_cast<uint32_t>(tail) * (C.row_bytes / 16);
    const uint32_t heads = static_cast<uint32_t>(C.planes) * C.kv_heads, threads = gridDim.y * 256u;
    const uint32_t t = blockIdx.y * 256u + threadIdx.x;
    const int64_t away = (static_cast<int64_t>(page) - last) * C.page_bytes;
    char* const base = C.pool + last * C.page_bytes;
    const uint32_t step = pieces < threads ? threads / pieces : 1;
    uint32_t x = pieces < threads ? t % pieces : t;
    const uint32_t first = pieces < threads ? t / pieces : 0;
    if (first >= step) return;
    for (; x < pieces; x += threads) {
        for (uint32_t h = first; h < heads; h += 4 * step) {
            uint4 v[4];
            char* at[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t ph = h + i * step < heads ? h + i * step : h;
                at[i] = base + ph / C.kv_heads * C.plane_bytes + ph % C.kv_heads * C.head_bytes + x * 16u;
                v[i] = get16(at[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (h + i * step < heads) put16(at[i] + away, v[i]);
        }
    }
}

__global__ __launch_bounds__(256) void fork_rows_kernel(const ForkArgs A) {
    const Cache& C = A.c;
    const int i = blockIdx.x;
    if (A.fresh[i] == -2) return;
    const int32_t d = A.dst[i];
    const int32_t* const row = A.rows + static_cast<int64_t>(i) * C.max_pages;
    for (int32_t x = threadIdx.x; x < C.max_pages; x += 256) C.table[static_cast<int64_t>(d) * C.table_stride + x] = row[x];
    if (threadIdx.x == 0) {
        C.lengths[d] = A.lens[i];
        C.held[d] = (A.lens[i] + C.page_size - 1) / C.page_size;
    }
}

// --------------------------------------------------------------------------
// The accepted path of a verified tree to the front of the drafted rows.
// --------------------------------------------------------------------------

struct CommitArgs {
    Cache c;
    const int32_t *seqs, *accepted, *counts;
    int32_t* new_lengths;
    int32_t n_seqs, most;  // most: entries of a row of accepted
};

// Accepted tokens of sequence b, 0 where there cannot be as many or they are not in its pages.
__device__ __forceinline__ int32_t accepted_of(const CommitArgs& A, int b, int32_t slot) {
    const int32_t n = A.counts[b];
    if (n <= 0 || n > A.most) return 0;
    const int32_t last = A.accepted[static_cast<int64_t>(b) * A.most + n - 1];
    const int64_t end = static_cast<int64_t>(length_of(A.c, slot)) + last;
    return last >= n - 1 && end < static_cast<int64_t>(held_of(A.c, slot)) * A.c.page_size ? n : 0;
}

constexpr int kPath = 128;  // rows of a path whose places are held at a time

// A thread owns 16 bytes of one head in one plane and moves them for row after
// row of its sequence's path. Accepted indices rise, so row i goes to a place
// at or before its own and before every later source: four rows are read, then
// written, and no other thread touches these bytes. Bound by HBM: 64 sequences
// of up to 12 accepted rows, 6 on average, in 80 planes of 8 heads of 128 read
// 58 MB and write 58 in 25 us.
__global__ __launch_bounds__(256) void commit_kernel(const CommitArgs A) {
    const Cache& C = A.c;
    __shared__ int64_t from[kPath], to[kPath];
    const int b = blockIdx.y;
    const int32_t slot = A.seqs[b];
    if (!known(C, slot)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) tell(C, kBadIndex);
        return;
    }
    const int32_t len = length_of(C, slot), n = accepted_of(A, b, slot);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const int32_t asked = A.counts[b];
        if (n != asked) tell(C, asked < 0 || asked > A.most ? kBadIndex : kRowFull);
        if (A.new_lengths != C.lengths) A.new_lengths[slot] = len + n;
    }
    const uint32_t pieces = C.row_bytes / 16, all = static_cast<uint32_t>(C.planes) * C.kv_heads * pieces;  // below 2^31
    const uint32_t j = blockIdx.x * 256u + threadIdx.x, ph = j / pieces;
    char* const mine = C.pool + ph / C.kv_heads * C.plane_bytes + ph % C.kv_heads * C.head_bytes + j % pieces * 16;
    const int32_t* const row = C.table + static_cast<int64_t>(slot) * C.table_stride;
    const int64_t most = static_cast<int64_t>(held_of(C, slot)) * C.page_size;
    auto place = [&](int64_t at) -> int64_t {
        if (at < 0 || at >= most) return -1;
        const int32_t id = row[at / C.page_size];
        if (id < 0 || id >= C.n_pages) {
            tell(C, kBadIndex);
            return -1;
        }
        return id * C.page_bytes + at % C.page_size * C.row_bytes;
    };
    for (int32_t i0 = 0; i0 < n; i0 += kPath) {
        const int32_t here = n - i0 < kPath ? n - i0 : kPath;
        __syncthreads();
        for (int32_t i = threadIdx.x; i < here; i += 256) {
            const int32_t x = A.accepted[static_cast<int64_t>(b) * A.most + i0 + i];
            to[i] = x == i0 + i ? -1 : place(static_cast<int64_t>(len) + i0 + i);
            from[i] = place(static_cast<int64_t>(len) + x);
        }
        __syncthreads();
        if (j >= all) continue;
        for (int32_t i = 0; i < here; i += 4) {
            uint4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (i + x < here && to[i + x] >= 0 && from[i + x] >= 0) v[x] = get16(mine + from[i + x]);
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (i + x < here && to[i + x] >= 0 && from[i + x] >= 0) put16(mine + to[i + x], v[x]);
        }
    }
}

// Lengths in place, once every row has moved.
__global__ __launch_bounds__(256) void commit_lengths_kernel(const CommitArgs A) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= A.n_seqs || !known(A.c, A.seqs[b])) return;
    const int32_t slot = A.seqs[b];
    A.c.lengths[slot] = length_of(A.c, slot) + accepted_of(A, b, slot);
}

// --------------------------------------------------------------------------
// Used pages to the front of the pool.
// --------------------------------------------------------------------------

struct CompactArgs {
    Cache c;
    int32_t *new_table, *new_refs, *used;
    int32_t *moves, *high, *low, *remap;  // scratch: [1], [n_pages] each
};

// With n pages in use, the i-th used page at or past n goes to the i-th free
// one before it: the fewest moves there are, and no page written is read.
__global__ __launch_bounds__(kScan) void compact_plan_kernel(const CompactArgs A) {
    const Cache& C = A.c;
    __shared__ int32_t wave_sums[kWaves];
    int32_t mine = 0;
    for (int32_t p = threadIdx.x; p < C.n_pages; p += kScan) mine += C.refs[p] > 0 ? 1 : 0;
    int32_t n;
    sum_before(mine, wave_sums, n);
    int32_t highs = 0, lows = 0;
    for (int32_t p0 = 0; p0 < C.n_pages; p0 += kScan * kEach) {
        const int32_t p = p0 + threadIdx.x * kEach;
        int32_t high = 0, low = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (p + j >= C.n_pages) continue;
            const bool in_use = C.refs[p + j] > 0;
            high |= (in_use && p + j >= n ? 1 : 0) << j;
            low |= (!in_use && p + j < n ? 1 : 0) << j;
            A.remap[p + j] = p + j;
        }
        // Two counts of at most 4096 a round in one sum.
        int32_t total;
        const int32_t before = sum_before(__popc(high) << 16 | __popc(low), wave_sums, total);
        int32_t h = highs + (before >> 16), l = lows + (before & 0xFFFF);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (high >> j & 1) A.high[h++] = p + j;
            if (low >> j & 1) A.low[l++] = p + j;
        }
        highs += total >> 16, lows += total & 0xFFFF;
    }
    if (A.new_refs != C.refs)
        for (int32_t p = threadIdx.x; p < C.n_pages; p += kScan) A.new_refs[p] = C.refs[p];
    __syncthreads();
    for (int32_t i = threadIdx.x; i < highs; i += kScan) {
        const int32_t h = A.high[i], l = A.low[i];
        A.remap[h] = l;
        A.new_refs[l] = A.new_refs[h];
        A.new_refs[h] = 0;
    }
    if (threadIdx.x == 0) {
        *A.moves = highs;
        *A.used = n;
    }
}

constexpr int kSlice = 16384;  // bytes of a page that a workgroup moves at a time

// A grid that strides over (move, plane, slice), the table's entries among its
// threads first. Bound by HBM: 1.26 GB in 255 us, 4.9 TB/s, what a plain copy reaches.
__global__ __launch_bounds__(256) void compact_move_kernel(const CompactArgs A) {
    const Cache& C = A.c;
    const int64_t entries = static_cast<int64_t>(C.max_seqs) * C.max_pages;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < entries; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t at = i / C.max_pages * C.table_stride + i % C.max_pages;
        const int32_t id = C.table[at];
        A.new_table[at] = id >= 0 && id < C.n_pages ? A.remap[id] : id;
    }
    const int32_t slices = static_cast<int32_t>((C.page_bytes + kSlice - 1) / kSlice);
    const int64_t items = static_cast<int64_t>(*A.moves) * C.planes * slices;
    for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const int32_t slice = static_cast<int32_t>(i % slices), plane = static_cast<int32_t>(i / slices % C.planes);
        const int32_t move = static_cast<int32_t>(i / slices / C.planes);
        char* const base = C.pool + plane * C.plane_bytes;
        const char* const from = base + A.high[move] * C.page_bytes;
        char* const to = base + A.low[move] * C.page_bytes;
        uint4 v[kSlice / 4096];
#pragma unroll
        for (int j = 0; j < kSlice / 4096; ++j) {
            const int64_t x = static_cast<int64_t>(slice) * kSlice + j * 4096 + threadIdx.x * 16;
            if (x < C.page_bytes) v[j] = get16(from + x);
        }
#pragma unroll
        for (int j = 0; j < kSlice / 4096; ++j) {
            const int64_t x = static_cast<int64_t>(slice) * kSlice + j * 4096 + threadIdx.x * 16;
            if (x < C.page_bytes) put16(to + x, v[j]);
        }
    }
}

int launched() {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? AIMG_OK : fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
}

// The descriptor, checked.
int take(const aimg_cache* c, Cache& C, bool pool) {
    if (c == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "cache is null");
    if (c->n_layers < 1 || c->n_pages < 1 || c->kv_heads < 1 || c->page_size < 1 || c->dim < 1 || c->max_seqs < 1 || c->max_pages < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "cache: every size must be at least 1");
    if (c->n_pages > kMaxPoolPages) return fail(AIMG_ERR_UNSUPPORTED, "cache: a pool must have fewer than 2^20 pages");
    if (c->dim % 8 != 0) return fail(AIMG_ERR_UNSUPPORTED, "cache: dim must be a multiple of 8");
    if (static_cast<int64_t>(c->max_pages) * c->page_size > INT32_MAX / 2)
        return fail(AIMG_ERR_UNSUPPORTED, "cache: a sequence must hold fewer than 2^30 positions");
    // By division: the product of the three can pass 64 bits.
    if (static_cast<int64_t>(c->kv_heads) * c->dim > INT32_MAX / 2 / c->page_size)
        return fail(AIMG_ERR_UNSUPPORTED, "cache: a page must be below 2^31 bytes");
    const int64_t page = 2 * static_cast<int64_t>(c->kv_heads) * c->page_size * c->dim;
    if (c->page_table == nullptr || c->lengths == nullptr || c->held == nullptr || c->refs == nullptr || c->status == nullptr ||
        (pool && c->pool == nullptr))
        return fail(AIMG_ERR_INVALID_ARGUMENT, "cache: null pointer");
    if (2 * static_cast<int64_t>(c->n_layers) * c->kv_heads * (c->dim / 8) > INT32_MAX - 256)
        return fail(AIMG_ERR_UNSUPPORTED, "cache: a position must be below 2^34 bytes in all layers");
    if (reinterpret_cast<uintptr_t>(c->pool) % 16 != 0) return fail(AIMG_ERR_UNSUPPORTED, "cache: the pool must be 16-byte aligned");
    C = Cache{static_cast<char*>(c->pool), c->page_table, c->lengths, c->held, c->refs, c->status,
              page * c->n_pages, page, 2 * static_cast<int64_t>(c->page_size) * c->dim,
              2 * c->n_layers, c->n_pages, c->kv_heads, c->page_size, 2 * c->dim, c->max_seqs, c->max_pages, c->max_pages};
    return AIMG_OK;
}

int check_seqs(int n, const void* a, const void* b) {
    if (n < 0) return fail(AIMG_ERR_INVALID_ARGUMENT, "n_seqs must be >= 0");
    if (n > kMaxSeqs) return fail(AIMG_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxSeqs) + " sequences a call");
    if (n > 0 && (a == nullptr || b == nullptr)) return fail(AIMG_ERR_INVALID_ARGUMENT, "null sequence arrays");
    return AIMG_OK;
}

uint32_t blocks(int64_t work, int64_t each, int64_t most = INT32_MAX) {
    const int64_t n = (work + each - 1) / each;
    return static_cast<uint32_t>(n < 1 ? 1 : n < most ? n : most);
}

}  // namespace
}  // namespace aimg

using aimg::fail;

extern "C" int aimg_cache_append(const aimg_cache* cache, int layer, const aimg_heads* k, const aimg_heads* v, const int32_t* seqs,
                                 const int32_t* offsets, int n_seqs, void* stream) {
    aimg::AppendArgs a{};
    int rc = aimg::take(cache, a.c, true);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, offsets);
    if (rc != AIMG_OK) return rc;
    if (layer < 0 || layer >= cache->n_layers) return fail(AIMG_ERR_INVALID_ARGUMENT, "layer must be in 0.." + std::to_string(cache->n_layers - 1));
    if (k == nullptr || v == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "k or v is null");
    if (k->n_rows != v->n_rows || k->heads != cache->kv_heads || v->heads != cache->kv_heads || k->dim != cache->dim || v->dim != cache->dim)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "k and v must have the same rows and the cache's heads and dim");
    if (k->n_rows < 0 || k->n_rows > INT32_MAX) return fail(AIMG_ERR_INVALID_ARGUMENT, "n_rows must be in 0..2^31-1");
    if (n_seqs == 0 || k->n_rows == 0) return AIMG_OK;
    if (k->data == nullptr || v->data == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "k or v: null data");
    if ((reinterpret_cast<uintptr_t>(k->data) | reinterpret_cast<uintptr_t>(v->data)) % 16 != 0 ||
        (k->row_stride | k->head_stride | v->row_stride | v->head_stride) % 8 != 0)
        return fail(AIMG_ERR_UNSUPPORTED, "k and v: need 16-byte aligned data and strides of whole 16 bytes");
    a.k = static_cast<const char*>(k->data), a.v = static_cast<const char*>(v->data);
    a.k_row = 2 * k->row_stride, a.k_head = 2 * k->head_stride, a.v_row = 2 * v->row_stride, a.v_head = 2 * v->head_stride;
    a.seqs = seqs, a.offsets = offsets, a.n_seqs = n_seqs, a.n_rows = static_cast<int32_t>(k->n_rows);
    a.layer_at = 2 * layer * a.c.plane_bytes;
    const int64_t work = k->n_rows * cache->kv_heads * (cache->dim / 8);
    if (work > INT32_MAX - 256) return fail(AIMG_ERR_UNSUPPORTED, "too many rows");
    hipLaunchKernelGGL(aimg::append_kernel, dim3(aimg::blocks(work, 256)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return aimg::launched();
}

extern "C" int aimg_cache_advance(const aimg_cache* cache, const int32_t* seqs, const int32_t* offsets, int n_seqs, void* stream) {
    aimg::Cache c;
    int rc = aimg::take(cache, c, false);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, offsets);
    if (rc != AIMG_OK || n_seqs == 0) return rc;
    hipLaunchKernelGGL(aimg::advance_kernel, dim3(aimg::blocks(n_seqs, 256)), dim3(256), 0, static_cast<hipStream_t>(stream), c, seqs, offsets, n_seqs);
    return aimg::launched();
}

extern "C" int aimg_cache_reserve(const aimg_cache* cache, const int32_t* seqs, const int32_t* tokens, int n_seqs, void* stream) {
    aimg::Cache c;
    int rc = aimg::take(cache, c, false);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, tokens);
    if (rc != AIMG_OK || n_seqs == 0) return rc;
    hipLaunchKernelGGL(aimg::reserve_kernel, dim3(1), dim3(aimg::kScan), 0, static_cast<hipStream_t>(stream), c, seqs, tokens, n_seqs);
    return aimg::launched();
}

extern "C" int aimg_cache_release(const aimg_cache* cache, const int32_t* seqs, int n_seqs, void* stream) {
    aimg::Cache c;
    int rc = aimg::take(cache, c, false);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, seqs);
    if (rc != AIMG_OK || n_seqs == 0) return rc;
    hipLaunchKernelGGL(aimg::release_kernel, dim3(static_cast<uint32_t>(n_seqs)), dim3(256), 0, static_cast<hipStream_t>(stream), c, seqs);
    return aimg::launched();
}

extern "C" int aimg_cache_fork_workspace_nbytes(const aimg_cache* cache, int n_seqs, size_t* nbytes) {
    if (cache == nullptr || nbytes == nullptr || n_seqs < 0 || cache->max_pages < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "null pointer or negative size");
    *nbytes = 4 * static_cast<size_t>(n_seqs) * (2 + cache->max_pages);
    return AIMG_OK;
}

extern "C" int aimg_cache_fork(const aimg_cache* cache, const int32_t* src, const int32_t* dst, int n_seqs, void* workspace,
                               size_t workspace_nbytes, void* stream) {
    aimg::ForkArgs a{};
    int rc = aimg::take(cache, a.c, true);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, src, dst);
    if (rc != AIMG_OK || n_seqs == 0) return rc;
    size_t need = 0;
    aimg_cache_fork_workspace_nbytes(cache, n_seqs, &need);
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 || workspace_nbytes < need)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "the workspace is null, misaligned or below aimg_cache_fork_workspace_nbytes");
    a.src = src, a.dst = dst, a.n = n_seqs;
    a.fresh = static_cast<int32_t*>(workspace), a.lens = a.fresh + n_seqs, a.rows = a.lens + n_seqs;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(aimg::fork_plan_kernel, dim3(1), dim3(aimg::kScan), 0, s, a);
    // Shares of a pair: a thread moves up to four pieces of 16 bytes, in as many workgroups as a full tail takes.
    const int64_t pieces = static_cast<int64_t>(a.c.planes) * a.c.kv_heads * a.c.page_size * (a.c.row_bytes / 16);
    hipLaunchKernelGGL(aimg::fork_copy_kernel, dim3(static_cast<uint32_t>(n_seqs), aimg::blocks(pieces, 1024, 1024)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(aimg::fork_rows_kernel, dim3(static_cast<uint32_t>(n_seqs)), dim3(256), 0, s, a);
    return aimg::launched();
}

extern "C" int aimg_cache_commit(const aimg_cache* cache, const int32_t* seqs, const int32_t* accepted, int max_accepted,
                                 const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream) {
    aimg::CommitArgs a{};
    int rc = aimg::take(cache, a.c, true);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, counts);
    if (rc != AIMG_OK) return rc;
    if (max_accepted < 0) return fail(AIMG_ERR_INVALID_ARGUMENT, "max_accepted must be >= 0");
    if (n_seqs == 0) return AIMG_OK;
    if ((accepted == nullptr && max_accepted > 0) || new_lengths == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "null accepted or new_lengths");
    a.seqs = seqs, a.accepted = accepted, a.counts = counts, a.new_lengths = new_lengths, a.n_seqs = n_seqs, a.most = max_accepted;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t columns = static_cast<int64_t>(a.c.planes) * a.c.kv_heads * (a.c.row_bytes / 16);
    hipLaunchKernelGGL(aimg::commit_kernel, dim3(aimg::blocks(columns, 256), static_cast<uint32_t>(n_seqs)), dim3(256), 0, s, a);
    if (new_lengths == cache->lengths)
        hipLaunchKernelGGL(aimg::commit_lengths_kernel, dim3(aimg::blocks(n_seqs, 256)), dim3(256), 0, s, a);
    return aimg::launched();
}

extern "C" int aimg_cache_compact_workspace_nbytes(const aimg_cache* cache, size_t* nbytes) {
    if (cache == nullptr || nbytes == nullptr || cache->n_pages < 1) return fail(AIMG_ERR_INVALID_ARGUMENT, "null pointer or no pages");
    *nbytes = 4 * (1 + 3 * static_cast<size_t>(cache->n_pages));
    return AIMG_OK;
}

extern "C" int aimg_cache_compact(const aimg_cache* cache, int32_t* new_table, int32_t* new_refs, int32_t* used, void* workspace,
                                  size_t workspace_nbytes, void* stream) {
    aimg::CompactArgs a{};
    const int rc = aimg::take(cache, a.c, true);
    if (rc != AIMG_OK) return rc;
    size_t need = 0;
    aimg_cache_compact_workspace_nbytes(cache, &need);
    if (new_table == nullptr || new_refs == nullptr || used == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "null new_table, new_refs or used");
    if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 4 != 0 || workspace_nbytes < need)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "the workspace is null, misaligned or below aimg_cache_compact_workspace_nbytes");
    a.new_table = new_table, a.new_refs = new_refs, a.used = used;
    a.moves = static_cast<int32_t*>(workspace);
    a.high = a.moves + 1, a.low = a.high + a.c.n_pages, a.remap = a.low + a.c.n_pages;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(aimg::compact_plan_kernel, dim3(1), dim3(aimg::kScan), 0, s, a);
    const int64_t slices = (a.c.page_bytes + aimg::kSlice - 1) / aimg::kSlice;
    hipLaunchKernelGGL(aimg::compact_move_kernel, dim3(aimg::blocks(slices * a.c.planes * (a.c.n_pages / 2 + 1), 1, 2048)), dim3(256), 0, s, a);
    return aimg::launched();
}
