// Pages of a key/value cache: appending rows (turned by their positions on the
// way, where asked), reading them back, forking, reserving, releasing,
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
//
// A cache in 8 bits holds e4m3 values (4 bits of exponent, 3 of mantissa, no
// infinity, up to 448) and a scale for each 16 positions of a page and head,
// keys and values apart: element x stands for code * scale. A scale is the
// smallest power of two, 2^-100 to 2^119, that brings the block's largest
// element to at most 448, so the product is exact in bf16, and a block that
// takes further rows is formed anew from what it stands for: where its scale
// rises, only elements that fall below 2^-6 scales are rounded again (and stay
// so where the rows that raised it were drafts, and rejected).
#include <hip/hip_runtime.h>

#include <cmath>
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
    float* scales;        // of a cache in 8 bits: [planes][n_pages][kv_heads][blocks]; null in 16
    int32_t blocks;       // of a page, kBlock positions each
};

constexpr int kBlock = 16;
constexpr int kMaxDim8 = 256;
constexpr float kMost8 = 448.0f;                 // 0.875 * 2^9
constexpr int kLowExp = -100, kHighExp = 119;    // of scales

// Where the scales of a page's head begin (of page 0, plane 0: C.scales).
__device__ __forceinline__ int64_t scales_at(const Cache& C, int32_t plane, int32_t page, int32_t head) {
    return ((static_cast<int64_t>(plane) * C.n_pages + page) * C.kv_heads + head) * C.blocks;
}

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
// Rows turned by their positions on the way, and rows into blocks of 8 bits.
// --------------------------------------------------------------------------

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct AsBf16 {
    static __device__ f32x2 unpack(uint32_t w) { return f32x2{__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)}; }
    static __device__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2)); }
    // Two codes times a power of two, exact.
    template <bool kUpper>
    static __device__ uint32_t from8(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, kUpper));
    }
};

struct AsFp16 {
    static __device__ f32x2 unpack(uint32_t w) { return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2); }
    static __device__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2)); }
    template <bool kUpper>
    static __device__ uint32_t from8(uint32_t codes, float scale) {
        const f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), kUpper);
        return pack(x[0] * scale, x[1] * scale);
    }
};

template <typename T>
__device__ __forceinline__ void unpack8(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 p = T::unpack(u[i]);
        x[2 * i] = p[0], x[2 * i + 1] = p[1];
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
}

__device__ __forceinline__ void read8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// (a, b) by the angle of (c, s): three roundings each, the products' and the
// sum's, so that a row's values do not depend on what the compiler fuses where.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
#pragma clang fp contract(off)
    const float x = a * c - b * s, y = b * c + a * s;
    a = x, b = y;
}

struct TurnArgs {
    Cache c;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // elements
    const float *cos, *sin;   // [n_positions][half]
    const int32_t *positions, *seqs, *offsets;
    int32_t n_seqs, n_rows, heads, dim, half, n_positions;
    int32_t plane;            // of the layer's keys; its values are in the next
    uint32_t n_items;         // (block, head, keys or values) of a cache in 8 bits, a wave each
    bool paired;
};

// How a row's pairs lie in its 16-byte pieces.
constexpr int kHalves = 0;  // element i goes with i + half, 8 elements with 8 elements: half % 8 == 0
constexpr int kPairs = 1;   // 2 i goes with 2 i + 1, in one piece: half % 4 == 0
constexpr int kAny = 2;     // either, for every half: element by element (8192 rows of 40 and 2 * 8 heads of 128, half 50, 164-207 us; pieces, half 64, 37-41)

// Rows of a call in place of offsets that may be any numbers.
__device__ __forceinline__ int32_t row_bound(const int32_t* offsets, int b, int32_t n_rows) {
    const int32_t x = offsets[b];
    return x < 0 ? 0 : x > n_rows ? n_rows : x;
}

// The last sequence whose place is at most `at`, by the whole wave: its lanes
// look at 64 sequences at once (steps one after the other cost a memory latency
// each: 64 single tokens' append took 9.2 us, not 8.9).
template <typename Place>
__device__ __forceinline__ int last_before(int n_seqs, int64_t at, Place place) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = n_seqs;  // it is one of lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) / 64, b = lane * step;
        const int count = __popcll(__ballot(b < n && place(lo + (b < n ? b : 0)) <= at));
        const int from = count > 0 ? (count - 1) * step : 0;  // places rise, so those at or before are the first ones
        lo += from;
        n = n - from < step ? n - from : step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Eight elements of a turned row from element x on, one by one.
template <typename T>
__device__ __forceinline__ void turn_any(const TurnArgs& A, const uint16_t* row, int x, int32_t position, float (&out)[8]) {
    auto at = [&](int i) { return T::unpack(row[i])[0]; };
    const int64_t angle = static_cast<int64_t>(position) * A.half;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
        const int i = x + e;
        float a = at(i);
        if (i < 2 * A.half) {
            const bool second = A.paired ? i & 1 : i >= A.half;
            const int j = A.paired ? i / 2 : second ? i - A.half : i;
            float b = at(A.paired ? i ^ 1 : second ? i - A.half : i + A.half);
            const float c = A.cos[angle + j], s = A.sin[angle + j];
            if (second) {
                turn(b, a, c, s);
            } else {
                turn(a, b, c, s);
            }
        }
        out[e] = a;
    }
}

// Eight elements of a turned row from element x on, a multiple of 8.
template <typename T, int kMode>
__device__ __forceinline__ void turned8(const TurnArgs& A, const uint16_t* row, int x, int32_t position, float (&out)[8]) {
    if (kMode == kAny) return turn_any<T>(A, row, x, position, out);
    unpack8<T>(get16(reinterpret_cast<const char*>(row + x)), out);
    if (x >= 2 * A.half) return;
    const int64_t angle = static_cast<int64_t>(position) * A.half;
    float c[8], s[8];
    if (kMode == kHalves) {
        const bool second = x >= A.half;
        const int first = second ? x - A.half : x;
        float other[8];
        unpack8<T>(get16(reinterpret_cast<const char*>(row + (second ? first : x + A.half))), other);
        read8(A.cos + angle + first, c);
        read8(A.sin + angle + first, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (second) {
                turn(other[e], out[e], c[e], s[e]);
            } else {
                turn(out[e], other[e], c[e], s[e]);
            }
        }
    } else {
        const float4 c4 = *reinterpret_cast<const float4*>(A.cos + angle + x / 2), s4 = *reinterpret_cast<const float4*>(A.sin + angle + x / 2);
        turn(out[0], out[1], c4.x, s4.x);
        turn(out[2], out[3], c4.y, s4.y);
        turn(out[4], out[5], c4.z, s4.z);
        turn(out[6], out[7], c4.w, s4.w);
    }
}

// One row's queries, and its keys and values where the cache is in 16 bits, by
// a workgroup: a thread owns a pair of pieces (or a piece) of a head, keeps
// their angles and steps over the heads. It reads its pieces before it writes
// them, so the result may be q's own memory (kAny: the workgroup does).
template <typename T, int kMode>
__device__ __forceinline__ void turn_row(const TurnArgs& A, int32_t row) {
    const Cache& C = A.c;
    const int b = last_before(A.n_seqs, row, [&](int i) { return A.offsets[i]; });
    const int32_t first = A.offsets[b];
    if (row < first || row >= A.offsets[b + 1]) return;  // a row of no sequence
    const int32_t slot = A.seqs[b];
    auto wrong = [&](int32_t what) {
        if (threadIdx.x == 0) tell(C, what);
    };
    if (!known(C, slot)) return wrong(kBadIndex);
    const int64_t at = static_cast<int64_t>(length_of(C, slot)) + row - first;
    const int64_t position = A.positions != nullptr ? A.positions[row] : at;
    if (A.half > 0 && (position < 0 || position >= A.n_positions)) return wrong(kBadIndex);
    char* to = nullptr;  // the row's place in head 0 of the layer's keys
    if (C.scales == nullptr) {
        const int64_t page = at / C.page_size;
        if (page >= held_of(C, slot)) {
            wrong(kRowFull);
        } else {
            const int32_t id = C.table[static_cast<int64_t>(slot) * C.table_stride + page];
            if (id < 0 || id >= C.n_pages) wrong(kBadIndex);
            else to = C.pool + A.plane * C.plane_bytes + id * C.page_bytes + at % C.page_size * C.row_bytes;
        }
    }
    const int pairs = kMode == kHalves ? A.half / 8 : 0;
    const int units = A.dim / 8 - pairs, step = 256 / units;
    const int unit = static_cast<int>(threadIdx.x) % units, lane_head = static_cast<int>(threadIdx.x) / units;
    const bool two = unit < pairs;
    const int x = two ? 8 * unit : 8 * (unit + pairs), y = x + A.half;
    const int all = A.heads + (to != nullptr ? 2 * C.kv_heads : 0);
    auto from = [&](int h) {
        return h < A.heads ? A.q + row * A.q_row + h * A.q_head
               : h < A.heads + C.kv_heads ? A.k + row * A.k_row + (h - A.heads) * A.k_head : A.v + row * A.v_row + (h - A.heads - C.kv_heads) * A.v_head;
    };
    auto into = [&](int h) -> char* {
        if (h < A.heads) return reinterpret_cast<char*>(A.q_out + row * A.out_row + h * A.out_head);
        const bool value = h >= A.heads + C.kv_heads;
        return to + (value ? C.plane_bytes : 0) + (h - A.heads - (value ? C.kv_heads : 0)) * C.head_bytes;
    };
    if constexpr (kMode == kAny) {
        for (int h0 = 0; h0 < all; h0 += step) {
            const int h = h0 + lane_head;
            const bool mine = lane_head < step && h < all;
            float out[8];
            if (mine) {
                if (h < A.heads + C.kv_heads) turn_any<T>(A, from(h), x, static_cast<int32_t>(position), out);
                else unpack8<T>(get16(reinterpret_cast<const char*>(from(h) + x)), out);
            }
            __syncthreads();
            if (mine) put16(into(h) + 2 * x, pack8<T>(out));
        }
    } else {
        if (lane_head >= step) return;
        const bool turns = kMode == kHalves ? two : x < 2 * A.half;
        float c[8] = {}, s[8] = {};
        if (turns) {
            const int64_t angle = position * A.half + (kMode == kHalves ? x : x / 2);
            if (kMode == kHalves) {
                read8(A.cos + angle, c);
                read8(A.sin + angle, s);
            } else {
                const float4 c4 = *reinterpret_cast<const float4*>(A.cos + angle), s4 = *reinterpret_cast<const float4*>(A.sin + angle);
                c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w, s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
            }
        }
        constexpr int kAhead = 2;  // heads whose pieces are on their way together
        for (int h0 = lane_head; h0 < all; h0 += kAhead * step) {
            uint4 a[kAhead], o[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const uint16_t* const p = from(h0 + i * step < all ? h0 + i * step : h0);
                a[i] = get16(reinterpret_cast<const char*>(p + x));
                if (kMode == kHalves && two) o[i] = get16(reinterpret_cast<const char*>(p + y));
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int h = h0 + i * step;
                if (h >= all) continue;
                if (turns && h < A.heads + C.kv_heads) {
                    float u[8], w[8];
                    unpack8<T>(a[i], u);
                    if (kMode == kHalves) {
                        unpack8<T>(o[i], w);
#pragma unroll
                        for (int e = 0; e < 8; ++e) turn(u[e], w[e], c[e], s[e]);
                        o[i] = pack8<T>(w);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) turn(u[2 * e], u[2 * e + 1], c[e], s[e]);
                    }
                    a[i] = pack8<T>(u);
                }
                char* const d = into(h);
                put16(d + 2 * x, a[i]);
                if (kMode == kHalves && two) put16(d + 2 * y, o[i]);
            }
        }
    }
}

// A block's pieces as a wave holds them: NP pieces of 8 elements a lane, piece
// j * 64 + lane of the 16 rows' 2 * dim.
template <int NP>
struct Formed {
    float x[NP][8];

    // The exponent of the scale for these elements, by the whole wave.
    __device__ __forceinline__ int exponent() const {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = fabsf(x[j][e]);
                top = a < INFINITY && a > top ? a : top;  // infinities and NaNs have no say
            }
#pragma unroll
        for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
        const uint32_t bits = __float_as_uint(top);
        // top = m 2^e with m in [1, 2): 448 = 1.75 * 2^8. (What is not normal lies below the lowest scale.)
        const int e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7);
        return e < kLowExp ? kLowExp : e > kHighExp ? kHighExp : e;
    }

    // Piece j's codes for 1 / scale. Past 448 (at the highest scale alone) they stay there; infinities become NaN.
    __device__ __forceinline__ uint2 codes(int j, float by) const {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = x[j][e] * by;
            y[e] = fabsf(x[j][e]) < INFINITY ? fminf(fmaxf(v, -kMost8), kMost8) : NAN;
        }
        uint2 w;
        w.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
        w.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false), true);
        return w;
    }

    __device__ __forceinline__ void hold(int j, uint2 w, float scale) {
        const f32x2 p[4] = {__builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true),
                            __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true)};
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = p[e / 2][e % 2] * scale;
    }

    __device__ __forceinline__ void nothing(int j) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[j][e] = 0.0f;
    }
};

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }  // e in -126..127

// One block of 16 positions of a head's keys or values that takes rows of the
// call, by a wave: the rows it holds already (below the length) and the new
// ones, their largest element, their codes. Sequence b's blocks are counted
// from slot first_row / 16 + 2 b on: n rows lie in at most n / 16 + 2 blocks, so
// no sums over the sequences are needed; the slots that are left over return.
template <typename T, int kMode, int NP>
__device__ __forceinline__ void form_block(const TurnArgs& A, uint32_t item, int lane) {
    const Cache& C = A.c;
    const int32_t which = item & 1, head = static_cast<int32_t>((item >> 1) % C.kv_heads), unit = static_cast<int32_t>((item >> 1) / C.kv_heads);
    const int b = last_before(A.n_seqs, unit, [&](int i) { return row_bound(A.offsets, i, A.n_rows) / kBlock + 2 * static_cast<int64_t>(i); });
    const int32_t first = row_bound(A.offsets, b, A.n_rows), n = row_bound(A.offsets, b + 1, A.n_rows) - first;
    const int32_t i = unit - (first / kBlock + 2 * b);
    if (n <= 0 || i < 0) return;
    const int32_t slot = A.seqs[b];
    auto wrong = [&](int32_t what) {
        if (lane == 0) tell(C, what);
    };
    if (!known(C, slot)) return wrong(kBadIndex);
    const int64_t length = length_of(C, slot), end = length + n, at = (length / kBlock + i) * kBlock;
    if (at >= end) return;
    const int64_t page = at / C.page_size;
    if (page >= held_of(C, slot)) return wrong(kRowFull);
    const int32_t id = C.table[static_cast<int64_t>(slot) * C.table_stride + page];
    if (id < 0 || id >= C.n_pages) return wrong(kBadIndex);
    const int32_t row0 = static_cast<int32_t>(at % C.page_size);
    char* const codes = C.pool + (A.plane + which) * C.plane_bytes + id * C.page_bytes + head * C.head_bytes + row0 * C.row_bytes;
    float* const scale = C.scales + scales_at(C, A.plane + which, id, head) + row0 / kBlock;
    const int old = length > at ? static_cast<int>(length - at) : 0, rows = end - at < kBlock ? static_cast<int>(end - at) : kBlock;
    const float held = old > 0 ? *scale : 0.0f;
    const uint16_t* const from = which == 0 ? A.k + head * A.k_head : A.v + head * A.v_head;
    const int64_t from_row = which == 0 ? A.k_row : A.v_row;
    const int pieces = A.dim / 8;
    Formed<NP> f;
    uint32_t keep = 0;  // pieces that are written
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int r = (j * 64 + lane) / pieces, x = (j * 64 + lane) % pieces * 8;
        if (r < old) {
            f.hold(j, *reinterpret_cast<const uint2*>(codes + r * C.row_bytes + x), held);
            keep |= 1u << j;
        } else if (r < rows) {
            const int32_t row = first + static_cast<int32_t>(at - length) + r;
            const uint16_t* const p = from + row * from_row;
            const int64_t position = A.half == 0 ? 0 : A.positions != nullptr ? A.positions[row] : at + r;
            if (A.half > 0 && (position < 0 || position >= A.n_positions)) {
                f.nothing(j);
                bad = true;
            } else {
                if (which != 0 || A.half == 0) unpack8<T>(get16(reinterpret_cast<const char*>(p + x)), f.x[j]);
                else turned8<T, kMode>(A, p, x, static_cast<int32_t>(position), f.x[j]);
                keep |= 1u << j;
            }
        } else {
            f.nothing(j);
        }
    }
    if (bad) tell(C, kBadIndex);
    const int e = f.exponent();
    const float now = power_of_two(e), by = power_of_two(-e);
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int r = (j * 64 + lane) / pieces, x = (j * 64 + lane) % pieces * 8;
        if ((keep >> j & 1) == 0 || (r < old && now == held)) continue;
        *reinterpret_cast<uint2*>(codes + r * C.row_bytes + x) = f.codes(j, by);
    }
    if (lane == 0) *scale = now;
}

// Blocks first, four a workgroup, then a workgroup a row. NP: 0 for a cache in
// 16 bits. Many rows are bound by HBM: 16384 rows of 40 heads and 2 * 8 of 128,
// 478 MB read and written in 88 us, 5.4 TB/s; 8192 rows into 8 bits, 223 MB in 45
// to 53 us. A token is bound by its reads that wait for each other (its sequence,
// slot, length, page, block): one 5 us, 64 in sequences of their own 9.
template <typename T, int kMode, int NP>
__global__ __launch_bounds__(256) void turn_kernel(const TurnArgs A) {
    uint32_t group = blockIdx.x;
    if constexpr (NP > 0) {
        const uint32_t groups = (A.n_items + 3) / 4;
        if (group < groups) {
            const uint32_t item = __builtin_amdgcn_readfirstlane(group * 4 + (threadIdx.x >> 6));
            if (item < A.n_items) form_block<T, kMode, NP>(A, item, threadIdx.x & 63);
            return;
        }
        group -= groups;
    }
    turn_row<T, kMode>(A, static_cast<int32_t>(group));
}

// --------------------------------------------------------------------------
// Rows out of pages.
// --------------------------------------------------------------------------

struct ReadArgs {
    Cache c;
    uint16_t *k, *v;
    int64_t k_row, k_head, v_row, v_head;  // elements
    const int32_t *seqs, *offsets, *starts;
    int32_t n_seqs, n_rows, plane;
};

constexpr int kReadRows = 8;  // of a workgroup
constexpr int64_t kMostGroups = (1 << 24) - 1;  // of 256 threads, which a launch counts in 32 bits

// Eight threads find where a workgroup's rows lie, then all move pieces of 8
// elements: a thread keeps its place in a head and takes it from row after row,
// eight pieces on their way at once. Bound by HBM: 23912 rows of 2 * 8 heads of
// 128 from 8 bits, 147 MB read and written in 36 us, 4.1 TB/s; 16384 rows of 16
// bits that were just written, 134 MB in 23 us.
template <typename T, bool k8>
__global__ __launch_bounds__(256) void read_kernel(const ReadArgs A) {
    const Cache& C = A.c;
    __shared__ int64_t place[kReadRows];   // bytes from a head's start in the pool; -1: not read
    __shared__ int64_t scale[kReadRows];   // its block's scale of head 0, from the plane's first
    const int32_t row0 = static_cast<int32_t>(blockIdx.x) * kReadRows;  // fewer than 2^31 rows
    if (threadIdx.x < 64) {
        // The first row's sequence, then the row's own: one of the next, or the same.
        int b = last_before(A.n_seqs, row0, [&](int i) { return A.offsets[i]; });
        const int64_t row = static_cast<int64_t>(row0) + threadIdx.x;
        int64_t found = -1, its_scale = 0;
        if (threadIdx.x < kReadRows && row < A.n_rows) {
            while (b + 1 < A.n_seqs && A.offsets[b + 1] <= row) ++b;
            const int64_t i = row - A.offsets[b];
            if (i >= 0 && row < A.offsets[b + 1]) {
                const int32_t slot = A.seqs[b];
                const int64_t at = (A.starts != nullptr ? A.starts[b] : 0) + i;
                if (!known(C, slot) || at < 0) {
                    tell(C, kBadIndex);
                } else if (at / C.page_size >= held_of(C, slot)) {
                    tell(C, kRowFull);
                } else {
                    const int32_t id = C.table[static_cast<int64_t>(slot) * C.table_stride + at / C.page_size];
                    if (id < 0 || id >= C.n_pages) {
                        tell(C, kBadIndex);
                    } else {
                        found = id * C.page_bytes + at % C.page_size * C.row_bytes;
                        if (k8) its_scale = scales_at(C, 0, id, 0) + at % C.page_size / kBlock;
                    }
                }
            }
        }
        if (threadIdx.x < kReadRows) place[threadIdx.x] = found, scale[threadIdx.x] = its_scale;
    }
    __syncthreads();
    constexpr int kBytes = k8 ? 8 : 16;  // of a piece in the cache
    const int pieces = C.row_bytes / kBytes, all = 2 * C.kv_heads * pieces;
    for (int t = threadIdx.x; t < all; t += 256) {
        const int piece = t % pieces, h = t / pieces, which = h >= C.kv_heads ? 1 : 0, head = h - which * C.kv_heads;
        const char* const from = C.pool + (A.plane + which) * C.plane_bytes + head * C.head_bytes + piece * kBytes;
        const float* const scales = k8 ? C.scales + scales_at(C, A.plane + which, 0, head) : nullptr;
        uint16_t* const to = which == 0 ? A.k + head * A.k_head + piece * 8 : A.v + head * A.v_head + piece * 8;
        const int64_t to_row = which == 0 ? A.k_row : A.v_row;
        uint4 v[kReadRows];
        float f[kReadRows];
#pragma unroll
        for (int r = 0; r < kReadRows; ++r) {
            if (place[r] < 0) continue;
            if constexpr (k8) {
                const uint2 w = *reinterpret_cast<const uint2*>(from + place[r]);
                v[r].x = w.x, v[r].y = w.y;
                f[r] = scales[scale[r]];
            } else {
                v[r] = get16(from + place[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < kReadRows; ++r) {
            if (place[r] < 0) continue;
            uint4 w = v[r];
            if constexpr (k8)
                w = make_uint4(T::template from8<false>(v[r].x, f[r]), T::template from8<true>(v[r].x, f[r]),
                               T::template from8<false>(v[r].y, f[r]), T::template from8<true>(v[r].y, f[r]));
            put16(reinterpret_cast<char*>(to + (row0 + r) * to_row), w);
        }
    }
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

// The scales of the tails' blocks: a thread a scale and step. (A launch of its
// own, for caches in 8 bits alone, before the rows change: 5 us for 96 branches
// in 80 planes, beside the rows' 111.)
__global__ __launch_bounds__(256) void fork_scales_kernel(const ForkArgs A) {
    const Cache& C = A.c;
    const int i = blockIdx.x;
    const int32_t page = A.fresh[i], len = A.lens[i], full = len / C.page_size, tail = len % C.page_size;
    if (page < 0 || tail == 0) return;
    const int32_t last = C.table[static_cast<int64_t>(A.src[i]) * C.table_stride + full];
    if (last < 0 || last >= C.n_pages) return;
    const uint32_t used = (tail + kBlock - 1) / kBlock, all = static_cast<uint32_t>(C.planes) * C.kv_heads * used;
    for (uint32_t x = blockIdx.y * 256u + threadIdx.x; x < all; x += gridDim.y * 256u) {
        const int32_t ph = static_cast<int32_t>(x / used), block = static_cast<int32_t>(x % used);
        const int32_t plane = ph / C.kv_heads, head = ph % C.kv_heads;
        C.scales[scales_at(C, plane, page, head) + block] = C.scales[scales_at(C, plane, last, head) + block];
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

// The same for a cache in 8 bits, a wave a (plane, head): it takes the blocks
// of the path in turn. A block into which a row moves is formed anew: its rows
// below the length and those of the path, from wherever they lie, are held in
// registers before any is written. Sources lie at or behind their own places,
// so what one block writes no later block reads. A block with a place that is
// no page's stays as it is. 64 sequences of up to 12 accepted rows, 6 on average,
// in 80 planes of 8 heads of 128: 53 us; in 16 bits, where rows move without a
// look at their elements, 14. (Eight heads a wave, which finds the places once:
// 66; rows not written that stay as they are: 57.)
template <int NP>
__global__ __launch_bounds__(256) void commit8_kernel(const CommitArgs A) {
    const Cache& C = A.c;
    const int b = blockIdx.y, lane = threadIdx.x & 63;
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
    const int32_t ph = static_cast<int32_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (ph >= C.planes * C.kv_heads) return;
    const int32_t plane = ph / C.kv_heads, head = ph % C.kv_heads;
    char* const mine = C.pool + plane * C.plane_bytes + head * C.head_bytes;
    float* const scales = C.scales + scales_at(C, plane, 0, head);
    const int64_t page_scales = static_cast<int64_t>(C.kv_heads) * C.blocks;
    const int32_t* const row = C.table + static_cast<int64_t>(slot) * C.table_stride;
    const int64_t most = static_cast<int64_t>(held_of(C, slot)) * C.page_size;
    const int pieces = C.row_bytes / 8;
    // Where a position lies: its row's bytes and its block's scale; false where it is no page's.
    auto place = [&](int64_t at, int64_t& bytes, int64_t& scale) {
        bytes = 0, scale = 0;
        if (at < 0 || at >= most) return false;
        const int32_t id = row[at / C.page_size], r = static_cast<int32_t>(at % C.page_size);
        if (id < 0 || id >= C.n_pages) {
            tell(C, kBadIndex);
            return false;
        }
        bytes = id * C.page_bytes + r * C.row_bytes, scale = id * page_scales + r / kBlock;
        return true;
    };
    for (int64_t at = len / kBlock * kBlock; at < static_cast<int64_t>(len) + n; at += kBlock) {
        // Lane r < 16: row r of the block.
        const int64_t i = at + (lane & 15) - len;  // index in the path; negative: held already
        const int32_t x = i >= 0 && i < n ? A.accepted[static_cast<int64_t>(b) * A.most + i] : static_cast<int32_t>(i);
        const bool used = i < n;
        if (__ballot(used && x != i) == 0) continue;
        int64_t from, from_scale, to, to_scale;
        from = from_scale = 0;
        const bool there = used && place(static_cast<int64_t>(len) + x, from, from_scale);
        if (!place(at, to, to_scale) || __ballot(used && !there) != 0) continue;
        const float its = there ? scales[from_scale] : 0.0f;
        Formed<NP> f;
        int rows = static_cast<int>(static_cast<int64_t>(len) + n - at);
        rows = rows < kBlock ? rows : kBlock;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = (j * 64 + lane) / pieces, p = (j * 64 + lane) % pieces * 8;
            const int64_t here = __shfl(from, r & 15);
            const float scale = __shfl(its, r & 15);
            if (r < rows) f.hold(j, *reinterpret_cast<const uint2*>(mine + here + p), scale);
            else f.nothing(j);
        }
        const int e = f.exponent();
        const float by = power_of_two(-e);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = (j * 64 + lane) / pieces, p = (j * 64 + lane) % pieces * 8;
            if (r < rows) *reinterpret_cast<uint2*>(mine + to + r * C.row_bytes + p) = f.codes(j, by);
        }
        if (lane == 0) scales[to_scale] = power_of_two(e);
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
        if (C.scales != nullptr && slice == 0) {
            const float* const f = C.scales + scales_at(C, plane, A.high[move], 0);
            float* const t = C.scales + scales_at(C, plane, A.low[move], 0);
            for (int32_t x = threadIdx.x; x < C.kv_heads * C.blocks; x += 256) t[x] = f[x];
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
              2 * c->n_layers, c->n_pages, c->kv_heads, c->page_size, 2 * c->dim, c->max_seqs, c->max_pages, c->max_pages, nullptr, 0};
    return AIMG_OK;
}

// The same for a cache in 8 bits, which has scales; in 16 where they are null.
int take_as(const aimg_cache* c, float* scales, Cache& C) {
    const int rc = take(c, C, true);
    if (rc != AIMG_OK || scales == nullptr) return rc;
    if (c->dim % 16 != 0 || c->dim > kMaxDim8)
        return fail(AIMG_ERR_UNSUPPORTED, "cache: dim must be a multiple of 16 up to " + std::to_string(kMaxDim8) + " for 8 bits");
    if (c->page_size % kBlock != 0) return fail(AIMG_ERR_UNSUPPORTED, "cache: page_size must be a multiple of 16 for 8 bits");
    if (reinterpret_cast<uintptr_t>(scales) % 4 != 0) return fail(AIMG_ERR_UNSUPPORTED, "cache: the scales must be 4-byte aligned");
    C.page_bytes /= 2, C.plane_bytes /= 2, C.head_bytes /= 2, C.row_bytes /= 2;
    C.scales = scales, C.blocks = c->page_size / kBlock;
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

namespace {

// Rows of heads that a call reads or writes whole pieces of.
int check_rows(const aimg_heads* x, const char* name, int heads, int dim) {
    const std::string n(name);
    if (x == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, n + " is null");
    if (x->n_rows < 0 || x->n_rows > INT32_MAX - 8) return fail(AIMG_ERR_INVALID_ARGUMENT, n + ": n_rows must be in 0..2^31-9");
    if (x->heads != heads || x->dim != dim || heads < 1)
        return fail(AIMG_ERR_INVALID_ARGUMENT, n + " must have " + std::to_string(heads) + " heads of dim " + std::to_string(dim));
    if (x->n_rows == 0) return AIMG_OK;
    if (x->data == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, n + ": null data");
    if (x->row_stride < 0 || x->head_stride < 0) return fail(AIMG_ERR_UNSUPPORTED, n + ": strides must not be negative");
    if (reinterpret_cast<uintptr_t>(x->data) % 16 != 0 || (x->row_stride | x->head_stride) % 8 != 0)
        return fail(AIMG_ERR_UNSUPPORTED, n + ": needs 16-byte aligned data and strides of whole 16 bytes");
    return AIMG_OK;
}

int check_layer(const aimg_cache* cache, int layer) {
    if (layer < 0 || layer >= cache->n_layers) return fail(AIMG_ERR_INVALID_ARGUMENT, "layer must be in 0.." + std::to_string(cache->n_layers - 1));
    if (cache->dim > aimg::kMaxDim8) return fail(AIMG_ERR_UNSUPPORTED, "cache: dim must be at most " + std::to_string(aimg::kMaxDim8));
    return AIMG_OK;
}

int check_type(int type) {
    if (type != AIMG_BF16 && type != AIMG_FP16) return fail(AIMG_ERR_UNSUPPORTED, "type must be AIMG_BF16 or AIMG_FP16, got " + std::to_string(type));
    return AIMG_OK;
}

template <typename T, int kMode>
void launch_turn(const aimg::TurnArgs& a, hipStream_t s) {
    const dim3 grid((a.n_items + 3) / 4 + static_cast<uint32_t>(a.c.scales == nullptr || a.q != nullptr ? a.n_rows : 0)), block(256);
    if (a.c.scales == nullptr) hipLaunchKernelGGL((aimg::turn_kernel<T, kMode, 0>), grid, block, 0, s, a);
    else if (a.dim <= 64) hipLaunchKernelGGL((aimg::turn_kernel<T, kMode, 2>), grid, block, 0, s, a);
    else if (a.dim <= 128) hipLaunchKernelGGL((aimg::turn_kernel<T, kMode, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((aimg::turn_kernel<T, kMode, 8>), grid, block, 0, s, a);
}

template <typename T>
void launch_turn(const aimg::TurnArgs& a, hipStream_t s) {
    const bool whole = (reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) % 16 == 0;
    if (a.half == 0 || (whole && a.paired && a.half % 4 == 0)) launch_turn<T, aimg::kPairs>(a, s);
    else if (whole && !a.paired && a.half % 8 == 0) launch_turn<T, aimg::kHalves>(a, s);
    else launch_turn<T, aimg::kAny>(a, s);
}

}  // namespace

extern "C" int aimg_cache_append_rotated(const aimg_cache* cache, float* scales, int layer, const aimg_heads* q, const aimg_heads* k,
                                         const aimg_heads* v, const aimg_heads* q_out, const int32_t* seqs, const int32_t* offsets,
                                         int n_seqs, const aimg_rotary* rotary, const int32_t* positions, int type, void* stream) {
    aimg::TurnArgs a{};
    int rc = aimg::take_as(cache, scales, a.c);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, offsets);
    if (rc == AIMG_OK) rc = check_layer(cache, layer);
    if (rc == AIMG_OK) rc = check_type(type);
    if (rc == AIMG_OK) rc = check_rows(k, "k", cache->kv_heads, cache->dim);
    if (rc == AIMG_OK) rc = check_rows(v, "v", cache->kv_heads, cache->dim);
    if (rc == AIMG_OK && q != nullptr) rc = check_rows(q, "q", q->heads, cache->dim);
    if (rc == AIMG_OK && q != nullptr) rc = check_rows(q_out, "q_out", q->heads, cache->dim);
    if (rc != AIMG_OK) return rc;
    if (v->n_rows != k->n_rows || (q != nullptr && (q->n_rows != k->n_rows || q_out->n_rows != k->n_rows)))
        return fail(AIMG_ERR_INVALID_ARGUMENT, "q, k, v and q_out must have the same rows");
    if (rotary != nullptr) {
        if (rotary->cos == nullptr || rotary->sin == nullptr || rotary->n_positions < 1)
            return fail(AIMG_ERR_INVALID_ARGUMENT, "rotary: null tables or no positions");
        if (rotary->half < 1 || 2 * static_cast<int64_t>(rotary->half) > cache->dim)
            return fail(AIMG_ERR_INVALID_ARGUMENT, "rotary: half must be in 1..dim / 2, got " + std::to_string(rotary->half));
        if ((reinterpret_cast<uintptr_t>(rotary->cos) | reinterpret_cast<uintptr_t>(rotary->sin)) % 4 != 0)
            return fail(AIMG_ERR_UNSUPPORTED, "rotary: the tables must be 4-byte aligned");
        a.cos = rotary->cos, a.sin = rotary->sin, a.n_positions = rotary->n_positions, a.half = rotary->half, a.paired = rotary->interleaved != 0;
    }
    const int64_t rows = k->n_rows;
    if (n_seqs == 0 || rows == 0) return AIMG_OK;
    const int64_t items = scales != nullptr ? (rows / aimg::kBlock + 2 * static_cast<int64_t>(n_seqs)) * cache->kv_heads * 2 : 0;
    if (items > INT32_MAX || (items + 3) / 4 + rows > aimg::kMostGroups) return fail(AIMG_ERR_UNSUPPORTED, "too many rows");
    a.n_items = static_cast<uint32_t>(items);
    if (q != nullptr) {
        a.q = static_cast<const uint16_t*>(q->data), a.q_out = static_cast<uint16_t*>(q_out->data), a.heads = q->heads;
        a.q_row = q->row_stride, a.q_head = q->head_stride, a.out_row = q_out->row_stride, a.out_head = q_out->head_stride;
    }
    a.k = static_cast<const uint16_t*>(k->data), a.v = static_cast<const uint16_t*>(v->data);
    a.k_row = k->row_stride, a.k_head = k->head_stride, a.v_row = v->row_stride, a.v_head = v->head_stride;
    a.positions = positions, a.seqs = seqs, a.offsets = offsets, a.n_seqs = n_seqs, a.n_rows = static_cast<int32_t>(rows);
    a.dim = cache->dim, a.plane = 2 * layer;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == AIMG_BF16) launch_turn<aimg::AsBf16>(a, s);
    else launch_turn<aimg::AsFp16>(a, s);
    return aimg::launched();
}

extern "C" int aimg_cache_read(const aimg_cache* cache, float* scales, int layer, const int32_t* seqs, const int32_t* offsets,
                               const int32_t* starts, int n_seqs, const aimg_heads* k, const aimg_heads* v, int type, void* stream) {
    aimg::ReadArgs a{};
    int rc = aimg::take_as(cache, scales, a.c);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, offsets);
    if (rc == AIMG_OK) rc = check_layer(cache, layer);
    if (rc == AIMG_OK) rc = check_type(type);
    if (rc == AIMG_OK) rc = check_rows(k, "k", cache->kv_heads, cache->dim);
    if (rc == AIMG_OK) rc = check_rows(v, "v", cache->kv_heads, cache->dim);
    if (rc != AIMG_OK) return rc;
    if (v->n_rows != k->n_rows) return fail(AIMG_ERR_INVALID_ARGUMENT, "k and v must have the same rows");
    if (n_seqs == 0 || k->n_rows == 0) return AIMG_OK;
    if ((k->n_rows + aimg::kReadRows - 1) / aimg::kReadRows > aimg::kMostGroups) return fail(AIMG_ERR_UNSUPPORTED, "too many rows");
    a.k = static_cast<uint16_t*>(k->data), a.v = static_cast<uint16_t*>(v->data);
    a.k_row = k->row_stride, a.k_head = k->head_stride, a.v_row = v->row_stride, a.v_head = v->head_stride;
    a.seqs = seqs, a.offsets = offsets, a.starts = starts, a.n_seqs = n_seqs, a.n_rows = static_cast<int32_t>(k->n_rows), a.plane = 2 * layer;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid(aimg::blocks(k->n_rows, aimg::kReadRows)), block(256);
    if (scales == nullptr) hipLaunchKernelGGL((aimg::read_kernel<aimg::AsBf16, false>), grid, block, 0, s, a);
    else if (type == AIMG_BF16) hipLaunchKernelGGL((aimg::read_kernel<aimg::AsBf16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((aimg::read_kernel<aimg::AsFp16, true>), grid, block, 0, s, a);
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

namespace {

int fork(const aimg_cache* cache, float* scales, const int32_t* src, const int32_t* dst, int n_seqs, void* workspace,
         size_t workspace_nbytes, void* stream) {
    aimg::ForkArgs a{};
    int rc = aimg::take_as(cache, scales, a.c);
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
    if (scales != nullptr) {
        const int64_t most = static_cast<int64_t>(a.c.planes) * a.c.kv_heads * a.c.blocks;
        hipLaunchKernelGGL(aimg::fork_scales_kernel, dim3(static_cast<uint32_t>(n_seqs), aimg::blocks(most, 256, 64)), dim3(256), 0, s, a);
    }
    hipLaunchKernelGGL(aimg::fork_rows_kernel, dim3(static_cast<uint32_t>(n_seqs)), dim3(256), 0, s, a);
    return aimg::launched();
}

}  // namespace

extern "C" int aimg_cache_fork(const aimg_cache* cache, const int32_t* src, const int32_t* dst, int n_seqs, void* workspace,
                               size_t workspace_nbytes, void* stream) {
    return fork(cache, nullptr, src, dst, n_seqs, workspace, workspace_nbytes, stream);
}

extern "C" int aimg_cache8_fork(const aimg_cache* cache, float* scales, const int32_t* src, const int32_t* dst, int n_seqs,
                                void* workspace, size_t workspace_nbytes, void* stream) {
    if (scales == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "scales is null");
    return fork(cache, scales, src, dst, n_seqs, workspace, workspace_nbytes, stream);
}

namespace {

// Of a cache in 16 bits (scales null) or 8.
int commit(const aimg_cache* cache, float* scales, const int32_t* seqs, const int32_t* accepted, int max_accepted,
           const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream) {
    aimg::CommitArgs a{};
    int rc = aimg::take_as(cache, scales, a.c);
    if (rc == AIMG_OK) rc = aimg::check_seqs(n_seqs, seqs, counts);
    if (rc != AIMG_OK) return rc;
    if (max_accepted < 0) return fail(AIMG_ERR_INVALID_ARGUMENT, "max_accepted must be >= 0");
    if (n_seqs == 0) return AIMG_OK;
    if ((accepted == nullptr && max_accepted > 0) || new_lengths == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "null accepted or new_lengths");
    a.seqs = seqs, a.accepted = accepted, a.counts = counts, a.new_lengths = new_lengths, a.n_seqs = n_seqs, a.most = max_accepted;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t heads = static_cast<int64_t>(a.c.planes) * a.c.kv_heads;
    if (scales == nullptr) {
        hipLaunchKernelGGL(aimg::commit_kernel, dim3(aimg::blocks(heads * (a.c.row_bytes / 16), 256), static_cast<uint32_t>(n_seqs)), dim3(256), 0, s, a);
    } else {
        const dim3 grid(aimg::blocks(heads, 4), static_cast<uint32_t>(n_seqs));
        if (cache->dim <= 64) hipLaunchKernelGGL((aimg::commit8_kernel<2>), grid, dim3(256), 0, s, a);
        else if (cache->dim <= 128) hipLaunchKernelGGL((aimg::commit8_kernel<4>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((aimg::commit8_kernel<8>), grid, dim3(256), 0, s, a);
    }
    if (new_lengths == cache->lengths)
        hipLaunchKernelGGL(aimg::commit_lengths_kernel, dim3(aimg::blocks(n_seqs, 256)), dim3(256), 0, s, a);
    return aimg::launched();
}

}  // namespace

extern "C" int aimg_cache_commit(const aimg_cache* cache, const int32_t* seqs, const int32_t* accepted, int max_accepted,
                                 const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream) {
    return commit(cache, nullptr, seqs, accepted, max_accepted, counts, n_seqs, new_lengths, stream);
}

extern "C" int aimg_cache8_commit(const aimg_cache* cache, float* scales, const int32_t* seqs, const int32_t* accepted, int max_accepted,
                                  const int32_t* counts, int n_seqs, int32_t* new_lengths, void* stream) {
    if (scales == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "scales is null");
    return commit(cache, scales, seqs, accepted, max_accepted, counts, n_seqs, new_lengths, stream);
}

extern "C" int aimg_cache_compact_workspace_nbytes(const aimg_cache* cache, size_t* nbytes) {
    if (cache == nullptr || nbytes == nullptr || cache->n_pages < 1) return fail(AIMG_ERR_INVALID_ARGUMENT, "null pointer or no pages");
    *nbytes = 4 * (1 + 3 * static_cast<size_t>(cache->n_pages));
    return AIMG_OK;
}

namespace {

int compact(const aimg_cache* cache, float* scales, int32_t* new_table, int32_t* new_refs, int32_t* used, void* workspace,
            size_t workspace_nbytes, void* stream) {
    aimg::CompactArgs a{};
    const int rc = aimg::take_as(cache, scales, a.c);
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

}  // namespace

extern "C" int aimg_cache_compact(const aimg_cache* cache, int32_t* new_table, int32_t* new_refs, int32_t* used, void* workspace,
                                  size_t workspace_nbytes, void* stream) {
    return compact(cache, nullptr, new_table, new_refs, used, workspace, workspace_nbytes, stream);
}

extern "C" int aimg_cache8_compact(const aimg_cache* cache, float* scales, int32_t* new_table, int32_t* new_refs, int32_t* used,
                                   void* workspace, size_t workspace_nbytes, void* stream) {
    if (scales == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "scales is null");
    return compact(cache, scales, new_table, new_refs, used, workspace, workspace_nbytes, stream);
}
