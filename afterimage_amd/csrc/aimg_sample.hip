// Tokens from logits: temperature, top-k, top-p and min-p, with given random
// numbers (gfx950).
//
// A row's tokens stand in the order of falling logits, equal ones by rising
// index. With w_i = exp((x_i - max x) / T), each of the three rules keeps a
// prefix of that order: the first k; the shortest whose weights reach p times
// those of the first k; those with w_i >= min_p. The token drawn is the first
// whose weights, summed along the order, pass u times the sum of all that are
// kept. No row is sorted for it: sums over a few thousand bins of neighbouring
// weights say in which bins the prefixes end and the draw falls, and only these
// bins' tokens (a few hundred, mostly) are gathered and sorted.
//
// Sums. A token's place t = 64 log2(1 / w) is computed as a pair of floats
// (doubles run at half the rate); the first's whole part is its bin, and its
// weight against the bin's top, by both, is rounded to 2^-26. A bin's count and sum are integers
// in one 64-bit word, so a row's result does not depend on the order of the
// atomics that add them; sums of bins are doubles, in a fixed order. Tokens
// below 2^-64 of the largest weigh nothing.
//
// A row is read three times. 256 rows of 151936 logits of 16 bits (78 MB a time,
// 15 us at a copy's rate): 57 us, in which 234 MB come past the L2, 4.1 TB/s, four
// fifths of a copy's rate. The bins' some twenty instructions and an atomic in LDS
// a token go beside that (42% of a SIMD's cycles, LDS 25%), and as a CU's LDS
// holds one workgroup, no other row's loads go beside a row's barriers. 64 rows
// with settings of their own, by several workgroups each: 46 to 57 us, by how many
// tokens the settings ask for; one row 24; temperature 0 15 for 256 rows.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "afterimage_decode.h"
#include "aimg_internal.h"

namespace aimg {
namespace {

constexpr int kPerOctave = 64;             // bins of a factor of 2
constexpr int kBins = 4096;
constexpr int kList = 4096;                // tokens that are gathered and sorted
constexpr double kStray = 0x1p-10;         // a token's place lies less than this outside its bin (see Place)
constexpr int kCountShift = 45;            // of a bin's word: count above; below, what its tokens lack to kMostUnits, in 2^-26 of the weight of its top
constexpr uint64_t kLackMask = (uint64_t{1} << kCountShift) - 1;
constexpr int kMaxVocab = 1 << 18;         // so that neither overflows
constexpr uint32_t kUnits = 1u << 26;
constexpr uint32_t kMostUnits = kUnits + 1024;  // a token that lies kStray above its bin weighs 710 units more than the bin's top
constexpr int64_t kMaxRows = 1 << 21;      // a launch's threads are counted in 32 bits

struct SampleArgs {
    const void* logits;
    int64_t row_stride;  // elements
    const float* uniforms;
    const float *temperatures, *top_ps, *min_ps;  // null: the numbers below for every row
    const int32_t* top_ks;
    double temperature, top_p, min_p;
    int32_t top_k, vocab;
    int64_t* tokens;
    float* logprobs;
};

struct LogitBf16 {
    typedef uint16_t Element;
    static __device__ float value(uint16_t x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
};

struct LogitFp16 {
    typedef uint16_t Element;
    static __device__ float value(uint16_t x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
};

struct LogitFp32 {
    typedef uint32_t Element;
    static __device__ float value(uint32_t x) { return __uint_as_float(x); }
};

// A piece's logits.
template <typename L, int kPiece>
__device__ __forceinline__ void values_of(const uint4& w, float (&x)[kPiece]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < kPiece; ++e) x[e] = L::value(static_cast<typename L::Element>(kPiece == 8 ? u[e / 2] >> 16 * (e % 2) : u[e]));
}

// Calls f(index of the first, logits) for 16-byte pieces thread, thread +
// threads, .. of a row, each thread's by rising index, those that test(logits)
// holds for. A row may begin and end anywhere: what lies outside whole pieces
// comes one by one, untested. kOnce: f where few pieces pass, one after the
// other, so that its code is there once (256 rows of 151936 55.5 us, not 59.6).
template <typename L, bool kOnce, typename Test, typename F>
__device__ __forceinline__ void each_piece(const typename L::Element* row, int n, int thread, int threads, Test test, F f) {
    typedef typename L::Element E;
    constexpr int kPiece = 16 / sizeof(E), kAhead = 4;
    int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(E));
    if (head > n) head = n;
    if (thread < head) {
        const float one[1] = {L::value(row[thread])};
        f(thread, one);
    }
    const int pieces = (n - head) / kPiece;
    for (int c0 = thread; c0 < pieces; c0 += kAhead * threads) {
        uint4 w[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int c = c0 + j * threads;
            w[j] = *reinterpret_cast<const uint4*>(row + head + static_cast<int64_t>(c < pieces ? c : c0) * kPiece);
        }
        uint32_t passed = 0;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int c = c0 + j * threads;
            if (c >= pieces) break;
            float x[kPiece];
            values_of<L>(w[j], x);
            if (!test(x)) continue;
            if constexpr (kOnce) passed |= 1u << j;
            else f(head + c * kPiece, x);
        }
        while (kOnce && passed != 0) {
            const int j = __builtin_ctz(passed);
            passed &= passed - 1;
            uint4 v = w[0];
#pragma unroll
            for (int i = 1; i < kAhead; ++i) {
                v.x = i == j ? w[i].x : v.x, v.y = i == j ? w[i].y : v.y;
                v.z = i == j ? w[i].z : v.z, v.w = i == j ? w[i].w : v.w;
            }
            float x[kPiece];
            values_of<L>(v, x);
            f(head + (c0 + j * threads) * kPiece, x);
        }
    }
    const int done = head + pieces * kPiece;
    if (done + thread < n) {  // fewer than a piece
        const float one[1] = {L::value(row[done + thread])};
        f(done + thread, one);
    }
}

// The same with f(index, logit). (No comparison with a NaN holds, so a NaN is never taken.)
template <typename L, typename F>
__device__ __forceinline__ void each_logit(const typename L::Element* row, int n, int thread, int threads, F f) {
    each_piece<L, false>(row, n, thread, threads, [](const auto&) { return true; }, [&](int i, const auto& x) {
#pragma unroll
        for (int e = 0; e < static_cast<int>(sizeof(x) / sizeof(float)); ++e) f(i + e, x[e]);
    });
}

// Unsigned numbers in the order of logits; equal ones for both zeros.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// A token's place: how far below the largest, 64 to a factor of 2, as the whole
// part `bin` of t, its value in 32 bits, and the rest f. What the product loses
// in 32 bits goes into the rest, and so does what max - x loses, for fp32
// logits: half a step of t (2^-13 below 4096) and 2^-24 of t for the difference's
// rounding and the factor's each, less than kStray together, by which f may lie
// outside [0, 1). (max - x loses nothing of bf16 logits unless their sizes are
// 2^16 apart, nor of fp16 ones unless 2^13, and then 2^-24 of itself at most,
// which weighs as much of (max - x) / T and is left: what takes it up would cost
// five instructions a token, 256 rows of 151936 60.1 us, not 57.6.) Bins rise
// as the logits fall, for both roundings keep the order; on which side of a
// border between two bins a place this near to it lies, they do not say. An
// infinite maximum leaves its equals alone at 0.
struct Place {
    float t;  // the bin's number and more; from kBins on, or NaN: no weight
    float f;
    __device__ __forceinline__ int bin() const { return static_cast<int>(t); }
    __device__ __forceinline__ double exact() const { return static_cast<double>(bin()) + f; }
};

template <typename L>
struct Places {
    float top, per, rest;  // per + rest: 64 log2(e) / temperature
    bool endless;          // the top is infinite

    __device__ __forceinline__ Place of(float x) const { return endless ? Place{x == top ? 0.0f : INFINITY, 0.0f} : of_finite(x); }

    __device__ __forceinline__ Place of_finite(float x) const {
#pragma clang fp contract(off)
        const float d = top - x, t = d * per;
        float f = fmaf(d, rest, fmaf(d, per, -t));
        if constexpr (sizeof(typename L::Element) == 4) {
            const float v = d - top;
            f = fmaf((top - (d - v)) - (x + v), per, f);
        }
        return Place{t, __builtin_amdgcn_fractf(t) + f};
    }

    // Logits whose places may lie in bins first .. last (all that do, and some more).
    __device__ __forceinline__ void span(int first, int last, float& low, float& high) const {
        if (endless) {
            low = high = top;
            return;
        }
        const double by = per, room = 1e-6 * fabs(static_cast<double>(top)), far = (last + 1) / by * (1.0 + 1e-6), near = first / by * (1.0 - 1e-6);
        low = static_cast<float>(top - far - room - 1e-6 * far);
        high = static_cast<float>(top - near + room + 1e-6 * near);
        if (first == 0 || !(high > low)) high = top;  // (nothing is above it; near is 0 / 0 where the temperature is infinite)
    }
};

// Spans of logits, of which a piece's nearest to any says whether it holds one:
// two instructions a logit and span, no masks.
struct Spans {
    float low[4], high[4], by[4], off[4];  // |x * by + off| <= 1 inside
    float room = 1.0f;                     // 1 and the roundings of that
    int n = 0;
    bool exact = true;

    __device__ __forceinline__ void add(float l, float h) {
        const double mid = 0.5 * (static_cast<double>(l) + h), half = 0.5 * (static_cast<double>(h) - l);
        const double to = half > 0.0 ? 1.0 / half : INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i == n) low[i] = l, high[i] = h, by[i] = static_cast<float>(to), off[i] = static_cast<float>(-mid * to);
        ++n;
        // x * by is off by 2^-24 of itself from by's rounding, and the sum by 2^-24 of off.
        const float far = static_cast<float>(fabs(mid * to));
        if (far < 1e5f) room = fmaxf(room, 1.0f + far * 1e-6f + 1e-6f);
        else exact = false;  // NaN too: infinite ends, spans of nearly no width
    }

    template <int kSpans, int kPiece>
    __device__ __forceinline__ bool any(const float (&x)[kPiece]) const {
        if (!exact) {
            bool in = false;
#pragma unroll
            for (int e = 0; e < kPiece; ++e) in |= holds<kSpans>(x[e]);
            return in;
        }
        float least = INFINITY;
#pragma unroll
        for (int i = 0; i < kSpans; ++i) {
            if (i > 1 && i >= n) break;
#pragma unroll
            for (int e = 0; e < kPiece; ++e) least = fminf(least, fabsf(fmaf(x[e], by[i], off[i])));
        }
        return least <= room;
    }

    template <int kSpans>
    __device__ __forceinline__ bool holds(float x) const {
        bool in = false;
#pragma unroll
        for (int i = 0; i < kSpans; ++i) in |= (i < 2 || i < n) && x >= low[i] && x <= high[i];
        return in;
    }
};

// What 2^(-f / 64) lacks to kMostUnits, in 2^-26 and rounded, for f in [-kStray,
// 1 + kStray], where it is above 0: the series of 1 - 2^(-f / 64) in g = f ln 2 / 64 < 0.011,
// whose fourth term is below 2^-30. The sum with 2^23 is the rounded number in
// its last 23 bits (of an f that is anywhere else or NaN, some number).
__device__ __forceinline__ uint32_t lack_in_bin(float f) {
    constexpr float g = 0.6931471805599453f / kPerOctave;
    const float x = fmaf(f, fmaf(f, fmaf(f, g * g * g / 6.0f * kUnits, -g * g / 2.0f * kUnits), g * kUnits), 0x1p23f + (kMostUnits - kUnits));
    return __float_as_uint(x) & 0x7FFFFFu;
}

__device__ __forceinline__ uint64_t word_of(float f) { return uint64_t{1} << kCountShift | lack_in_bin(f); }
__device__ __forceinline__ int32_t count_of(uint64_t word) { return static_cast<int32_t>(word >> kCountShift); }
__device__ __forceinline__ uint64_t units_of(uint64_t word) { return (word >> kCountShift) * kMostUnits - (word & kLackMask); }

// 2^(-i / 64), i < 64: a table that a workgroup makes once (exp2 for every bin took longer than their sums).
struct Octave {
    double part[kPerOctave];
    __device__ __forceinline__ void make() {
        if (threadIdx.x < kPerOctave) part[threadIdx.x] = exp2(-static_cast<double>(threadIdx.x) / kPerOctave);
    }
    // What a unit of a bin's sum weighs.
    __device__ __forceinline__ double unit(int bin) const { return ldexp(part[bin % kPerOctave], -26 - bin / kPerOctave); }
};

template <typename V>
__device__ __forceinline__ V before_in_wave(V v, V& all) {
    const int lane = threadIdx.x & 63;
    V s = v;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const V o = __shfl_up(s, x);
        if (lane >= x) s += o;
    }
    all = __shfl(s, 63);
    const V e = __shfl_up(s, 1);
    return lane == 0 ? V(0) : e;
}

// A row's settings. Numbers out of range mean the nearest in it: no rule, or the first token.
struct Rules {
    bool greedy;
    double per, p, min_t, u;
    int32_t k;
};

__device__ __forceinline__ bool greedy(const SampleArgs& A, int row) {
    return !((A.temperatures != nullptr ? A.temperatures[row] : A.temperature) > 0.0);
}

__device__ __forceinline__ Rules rules_of(const SampleArgs& A, int row) {
    Rules r;
    const double t = A.temperatures != nullptr ? A.temperatures[row] : A.temperature;
    const double p = A.top_ps != nullptr ? A.top_ps[row] : A.top_p, m = A.min_ps != nullptr ? A.min_ps[row] : A.min_p;
    const int32_t k = A.top_ks != nullptr ? A.top_ks[row] : A.top_k;
    const double u = A.uniforms[row];
    r.greedy = greedy(A, row);
    r.per = r.greedy ? 0.0 : kPerOctave * 1.4426950408889634 / t;
    if (r.per > 1e30) r.per = 1e30;
    r.k = k > 0 ? k : INT32_MAX;
    r.p = p < 1.0 ? (p > 0.0 ? p : 0.0) : 1.0;
    r.min_t = m > 0.0 ? (m < 1.0 ? -kPerOctave * log2(m) : 0.0) : INFINITY;
    r.u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-53) : 0.0;
    return r;
}

// What a row's workgroup keeps in LDS. The words are the bins, later the
// gathered tokens: ~key above, index below.
template <int kThreads>
struct Shared {
    static constexpr int kWaves = kThreads / 64;
    uint64_t words[kBins + 64];
    Octave octave;
    double wave_weight[kWaves], start[kThreads + 1];
    uint64_t wave_best[kWaves];
    int32_t wave_count[kWaves], wave_first[kWaves];
    double found_low[7], found_high[7], end_weight[3], found_weight;
    int32_t found[7], end_count[3], n, drawn, before_count, inside_count;
    uint64_t inside;
    int32_t at;
};

// Tokens and weights before each bin, and of all: [kBins + 1].
struct Sums {
    double* weight;
    int32_t* count;
};

// The bins where a row's prefixes may end (what the first k weigh is known to a
// bin, so what p of it is lies in some range; tokens next to min_p's border may
// lie in either of two bins) and where its draw may fall; -1: none.
struct Found {
    int32_t bin_k, low_p, high_p, low_m, high_m, low_u, high_u, last;
    __device__ __forceinline__ bool wanted(int b) const {
        return b == bin_k || (b >= low_p && b <= high_p) || (b >= low_m && b <= high_m) || (b >= low_u && b <= high_u);
    }
};

__device__ __forceinline__ double reached(double x, double all) { return x < 1e-300 ? 1e-300 : x > all ? all : x; }

// The words' sums and those bins, by a workgroup. `to` (where not null) takes the
// sums: of all bins, or of those wanted alone.
template <bool kAll, int kThreads>
__device__ __forceinline__ Found find_bins(Shared<kThreads>& S, const Rules& R, const Sums& to) {
    constexpr int kEach = kBins / kThreads, kWaves = kThreads / 64;
    const int t = threadIdx.x, wave = t >> 6;
    int32_t count[kEach + 1], all_c, my_c = 0;
    double weight[kEach + 1], all_w, my_w = 0.0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const uint64_t x = S.words[t * kEach + j];
        count[j + 1] = count_of(x);
        weight[j + 1] = static_cast<double>(units_of(x)) * S.octave.unit(t * kEach + j);
        my_c += count[j + 1], my_w += weight[j + 1];
    }
    count[0] = before_in_wave(my_c, all_c);
    weight[0] = before_in_wave(my_w, all_w);
    if ((t & 63) == 0) S.wave_count[wave] = all_c, S.wave_weight[wave] = all_w;
    if (t < 7) S.found[t] = -1, S.found_low[t] = S.found_high[t] = 0.0;
    __syncthreads();
    int32_t total_c = 0;
    double base = 0.0, total = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i == wave) count[0] += total_c, base = total;
        total_c += S.wave_count[i], total += S.wave_weight[i];
    }
    weight[0] += base;
    S.start[t] = weight[0];
    if (t == 0) S.start[kThreads] = total;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (kAll) to.count[t * kEach + j] = count[j], to.weight[t * kEach + j] = weight[j];
        count[j + 1] += count[j];
        weight[j + 1] = j + 1 < kEach ? weight[j] + weight[j + 1] : S.start[t + 1];  // where the next thread begins
    }
    if (kAll && t == 0) to.count[kBins] = total_c, to.weight[kBins] = total;
    auto mark = [&](int i, int j) { S.found[i] = t * kEach + j, S.found_low[i] = weight[j], S.found_high[i] = weight[j + 1]; };
    Found f;
    f.low_m = 0, f.high_m = -1;
    if (R.min_t < kBins) {
        f.low_m = R.min_t > kStray ? static_cast<int>(R.min_t - kStray) : 0;
        f.high_m = R.min_t + kStray < kBins ? static_cast<int>(R.min_t + kStray) : kBins - 1;
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (R.k < total_c && count[j] < R.k && R.k <= count[j + 1]) mark(0, j);
        if (t * kEach + j == f.low_m) mark(3, j);
        if (t * kEach + j == f.high_m) mark(6, j);
    }
    __syncthreads();
    f.bin_k = S.found[0];
    double low = total, high = total;  // that the kept tokens weigh
    if (f.bin_k >= 0) low = S.found_low[0], high = S.found_high[0];
    if (R.p < 1.0) {
        const double x = reached(R.p * low, total), y = reached(R.p * high, total);
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            if (weight[j] < x && x <= weight[j + 1]) mark(1, j);
            if (weight[j] < y && y <= weight[j + 1]) mark(2, j);
        }
    }
    __syncthreads();
    f.low_p = S.found[1], f.high_p = S.found[2];
    int end = f.bin_k >= 0 ? f.bin_k : kBins - 1;
    if (f.high_p >= 0) {
        low = fmin(low, f.low_p >= 0 ? S.found_low[1] : 0.0), high = fmin(high, S.found_high[2]);
        end = f.high_p < end ? f.high_p : end;
    }
    if (f.high_m >= 0) {
        low = fmin(low, S.found_low[3]), high = fmin(high, S.found_high[6]);
        if (f.low_m > end) f.high_m = -1;  // min_p ends no prefix
        else end = f.high_m < end ? f.high_m : end;
    }
    const double x = R.u * low, y = R.u * high;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        if (weight[j] <= x && x < weight[j + 1]) mark(4, j);
        if (weight[j] <= y && y < weight[j + 1]) mark(5, j);
    }
    __syncthreads();
    f.low_u = S.found[4] < 0 ? 0 : S.found[4];
    f.high_u = S.found[5] < 0 ? end : S.found[5];
    f.last = f.bin_k > f.high_p ? f.bin_k : f.high_p;
    f.last = f.high_u > f.last ? f.high_u : f.last;
    f.last = f.high_m > f.last ? f.high_m : f.last;
    if (!kAll && to.count != nullptr) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int b = t * kEach + j;
            if (!f.wanted(b)) continue;
            to.count[b] = count[j], to.weight[b] = weight[j];
            to.count[b + 1] = count[j + 1], to.weight[b + 1] = weight[j + 1];
        }
        __syncthreads();  // the total's place follows the last bin's
        if (t == 0) to.count[kBins] = total_c, to.weight[kBins] = total;
    }
    return f;
}

// The tokens of those bins among logits thread, thread + threads, .. into the
// words, which hold kList of them; S.n counts all. Their logits lie in four spans at most, which
// are tested a piece at a time and first: a place takes ten times as long.
template <typename L, int kThreads>
__device__ __forceinline__ void gather(Shared<kThreads>& S, const typename L::Element* row, int n, int thread, int threads, const Places<L>& P, const Found& f) {
    Spans spans{};
    auto add = [&](int first, int to) {
        float low, high;
        P.span(first, to, low, high);
        spans.add(low, high);
    };
    add(f.low_u, f.high_u);
    if (f.high_p >= 0) add(f.low_p < 0 ? 0 : f.low_p, f.high_p);
    if (f.bin_k >= 0) add(f.bin_k, f.bin_k);
    if (f.high_m >= 0) add(f.low_m, f.high_m);
    auto take = [&](auto number) {
        constexpr int kSpans = decltype(number)::value;
        auto test = [&](const auto& x) { return spans.template any<kSpans>(x); };
        each_piece<L, true>(row, n, thread, threads, test, [&](int i, const auto& x) {
            constexpr int kPiece = static_cast<int>(sizeof(x) / sizeof(float));
            uint32_t hits = 0;
#pragma unroll
            for (int e = 0; e < kPiece; ++e) hits |= spans.template holds<kSpans>(x[e]) ? 1u << e : 0u;
            while (hits != 0) {
                const int e = __builtin_ctz(hits);
                hits &= hits - 1;
                float v = x[0];
#pragma unroll
                for (int j = 1; j < kPiece; ++j) v = e == j ? x[j] : v;
                const Place place = P.of(v);
                if (!(place.t < f.last + 1 && f.wanted(place.bin()))) continue;
                const int at = atomicAdd(&S.n, 1);
                if (at < kList) S.words[at] = static_cast<uint64_t>(~key_of(v)) << 32 | static_cast<uint32_t>(i + e);
            }
        });
    };
    if (spans.n == 1) take(std::integral_constant<int, 1>{});
    else if (spans.n == 2) take(std::integral_constant<int, 2>{});
    else take(std::integral_constant<int, 4>{});
}

// How a prefix ends, or which token is drawn, where a bin holds more tokens
// than are gathered (equal logits by the thousand, very high temperatures): the
// bin's keys are binned again, 4096 at a time, until one key is left. It ends
// after at most three passes over the row, for each border and the draw, by one
// workgroup. bf16 logits around 20 with a deviation of 1 do that, since some 7500
// of 151936 are equal: 256 rows with all kept 306 us (around 0: 66), with top_p
// 0.9 520 (103), 64 rows 266 (64), one 170-240 (29-43); with top-k 50 65 (53).
struct Equals {
    uint32_t key;
    int32_t count, n;      // tokens before the equals, and the equals
    double weight, each;   // of those before, and of one of them
};

enum Goal { kCounted, kReached, kPassed };

template <typename L, Goal kGoal, int kThreads>
__device__ __forceinline__ Equals narrow(const SampleArgs& A, Shared<kThreads>& S, const Sums& B, const typename L::Element* row, const Places<L>& P, int bin, int32_t k, double x) {
    constexpr int kEach = kBins / kThreads, kWaves = kThreads / 64;
    uint32_t low = 0, high = 0xFFFFFFFFu;
    int32_t count = B.count[bin];
    double weight = B.weight[bin];
    const double unit = S.octave.unit(bin);
    for (;;) {
        int shift = 0;
        while (((high - low) >> shift) >= kBins) ++shift;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) S.words[i] = 0;
        if (threadIdx.x == 0) S.found[0] = -1;
        __syncthreads();
        each_logit<L>(row, A.vocab, threadIdx.x, kThreads, [&](int, float v) {
            const Place t = P.of(v);
            const uint32_t key = key_of(v);
            if (t.t < kBins && t.bin() == bin && key >= low && key <= high)
                atomicAdd(reinterpret_cast<unsigned long long*>(&S.words[(high - key) >> shift]), word_of(t.f));
        });
        __syncthreads();
        // The parts' sums before each, by one thread after the other: a part's
        // numbers are exact integers, so sums of this bin's are too.
        uint64_t mine = 0, all;
        for (int j = 0; j < kEach; ++j) mine += S.words[threadIdx.x * kEach + j];
        uint64_t sum = before_in_wave(mine, all);
        if ((threadIdx.x & 63) == 0) S.wave_best[threadIdx.x >> 6] = all;
        __syncthreads();
        uint64_t total = 0;
        for (int i = 0; i < kWaves; ++i) {
            if (i < (threadIdx.x >> 6)) sum += S.wave_best[i];
            total += S.wave_best[i];
        }
        for (int j = 0; j < kEach; ++j) {
            const uint64_t one = S.words[threadIdx.x * kEach + j], next = sum + one;
            if (one != 0) {
                const int32_t c0 = count + count_of(sum), c1 = count + count_of(next);
                const double w0 = weight + static_cast<double>(units_of(sum)) * unit;
                // The last part takes what rounding leaves over.
                const double w1 = next == total ? INFINITY : weight + static_cast<double>(units_of(next)) * unit;
                const bool first = sum == 0;
                const bool here = kGoal == kCounted ? c0 < k && (k <= c1 || next == total)
                                  : kGoal == kReached ? (first || w0 < x) && x <= w1 : (first || w0 <= x) && x < w1;
                if (here) S.found[0] = threadIdx.x * kEach + j, S.before_count = c0, S.found_weight = w0, S.inside = one, S.inside_count = c1 - c0;
            }
            sum = next;
        }
        __syncthreads();
        const int32_t at = S.found[0];
        if (at < 0) {  // no token of the bin, which no caller asks for
            Equals none{0, count, 0, weight, 0.0};
            return none;
        }
        count = S.before_count, weight = S.found_weight;
        const uint32_t part = static_cast<uint32_t>(at);
        const uint32_t top = high - (part << shift), size = shift == 0 ? 1u : 1u << shift;
        const uint32_t bottom = top - low < size ? low : top - size + 1;
        if (shift == 0) {
            Equals e{top, count, S.inside_count, weight, static_cast<double>(units_of(S.inside)) / S.inside_count * unit};
            __syncthreads();
            return e;
        }
        high = top, low = bottom;
        __syncthreads();
    }
}

// The index of the j-th token with this key.
template <typename L, int kThreads>
__device__ __forceinline__ int32_t index_of(const SampleArgs& A, Shared<kThreads>& S, const typename L::Element* row, uint32_t key, int32_t j) {
    const int each = (A.vocab + kThreads - 1) / kThreads, from = threadIdx.x * each < A.vocab ? threadIdx.x * each : A.vocab;
    const int to = from + each < A.vocab ? from + each : A.vocab;
    int32_t n = 0, all;
    for (int i = from; i < to; ++i) {
        const float x = L::value(row[i]);
        n += x == x && key_of(x) == key ? 1 : 0;
    }
    int32_t at = before_in_wave(n, all);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) S.wave_count[threadIdx.x >> 6] = all;
    __syncthreads();
    for (int i = 0; i < static_cast<int>(threadIdx.x >> 6); ++i) at += S.wave_count[i];
    if (at <= j && j < at + n)
        for (int i = from; i < to; ++i) {
            const float x = L::value(row[i]);
            if (x == x && key_of(x) == key && at++ == j) S.drawn = i;
        }
    __syncthreads();
    return S.drawn;
}

// Where a row's prefixes end and its draw falls, one after the other.
template <typename L, int kThreads>
__device__ __forceinline__ void resolve_large(const SampleArgs& A, Shared<kThreads>& S, const Sums& B, const typename L::Element* row, const Places<L>& P, const Rules& R,
                              const Found& f, int32_t& token, double& weight, double& kept) {
    const int bin_k = f.bin_k;
    int32_t most = B.count[kBins];
    kept = B.weight[kBins];
    // The bin where a weight is reached (weight before < x <= with it) or passed (<=, <).
    auto find = [&](double x, bool passed) {
        __syncthreads();
        if (threadIdx.x == 0) S.found[1] = -1;
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            const double low = B.weight[b], high = B.weight[b + 1];
            if (passed ? low <= x && x < high : low < x && x <= high) S.found[1] = b;
        }
        __syncthreads();
        return S.found[1];
    };
    if (bin_k >= 0) {
        const Equals e = narrow<L, kCounted>(A, S, B, row, P, bin_k, R.k, 0.0);
        most = R.k;
        kept = e.weight + (R.k - e.count) * e.each;
    }
    if (R.p < 1.0) {
        const double x = reached(R.p * kept, B.weight[kBins]);
        const int b = find(x, false);
        if (b >= 0) {
            const Equals e = narrow<L, kReached>(A, S, B, row, P, b, 0, x);
            double n = ceil((x - e.weight) / e.each);
            n = n < 1.0 ? 1.0 : n > e.n ? e.n : n;
            if (e.count + static_cast<int32_t>(n) < most) most = e.count + static_cast<int32_t>(n), kept = e.weight + n * e.each;
        }
    }
    if (f.high_m >= 0 && B.count[f.low_m] < most) {
        // The tokens of its bins that weigh enough.
        int32_t n = B.count[f.low_m];
        double with = B.weight[f.low_m];
        for (int bin = f.low_m; bin <= f.high_m; ++bin) {
            __syncthreads();
            if (threadIdx.x == 0) S.inside = 0;
            __syncthreads();
            uint64_t mine = 0;
            each_logit<L>(row, A.vocab, threadIdx.x, kThreads, [&](int, float v) {
                const Place t = P.of(v);
                if (t.t < kBins && t.bin() == bin && t.exact() <= R.min_t) mine += word_of(t.f);
            });
            if (mine != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&S.inside), mine);
            __syncthreads();
            n += count_of(S.inside), with += static_cast<double>(units_of(S.inside)) * S.octave.unit(bin);
        }
        if (n < most) most = n, kept = with;
    }
    const double x = R.u * kept;
    int b = find(x, true);
    if (b < 0) b = find(B.weight[kBins], false);
    const Equals e = narrow<L, kPassed>(A, S, B, row, P, b < 0 ? 0 : b, 0, x);
    double j = floor((x - e.weight) / e.each);
    j = j < 0.0 ? 0.0 : j > e.n - 1 ? e.n - 1 : j;
    if (e.count + j > most - 1) j = most - 1 > e.count ? most - 1 - e.count : 0;
    token = index_of<L>(A, S, row, e.key, static_cast<int32_t>(j));
    weight = e.each;
}

// The largest logit's key, and of its tokens the first where asked, in one word; 0 where there is none.
template <typename L>
__device__ __forceinline__ uint64_t largest(const typename L::Element* row, int n, int thread, int threads, bool first) {
    float best = -INFINITY;
    int32_t best_at = 0;
    if (first) {
        each_logit<L>(row, n, thread, threads, [&](int i, float x) {
            if (x > best) best = x, best_at = i;
        });
    } else {
        each_logit<L>(row, n, thread, threads, [&](int, float x) { best = fmaxf(best, x); });  // of a number and a NaN: the number
    }
    uint64_t top = best == -INFINITY ? 0 : static_cast<uint64_t>(key_of(best)) << 32 | ~static_cast<uint32_t>(best_at);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const uint64_t o = __shfl_xor(top, x);
        top = o > top ? o : top;
    }
    return top;
}

template <typename L>
__device__ __forceinline__ Places<L> places_of(uint64_t top, const Rules& R) {
    // (The same in every lane, which the compiler cannot tell.)
    const float per = static_cast<float>(R.per);
    const float x = of_key(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(top >> 32)))));
    return Places<L>{x, per, static_cast<float>(R.per - per), x == INFINITY};
}

// Tokens into their bins: kBins words, and one more for each lane, which takes
// what has no place (a branch around the atomic for each token took twice as
// long). Without top-p nothing asks for tokens that weigh less than min_p.
template <typename L>
__device__ __forceinline__ void fill_bins(const typename L::Element* row, int n, int thread, int threads, const Places<L>& P, const Rules& R, uint64_t* bins) {
    const float end = R.p < 1.0 || !(R.min_t < kBins - 1) ? kBins : static_cast<float>(static_cast<int>(R.min_t + kStray) + 1);
    const int nowhere = kBins + (threadIdx.x & 63);
    auto fill = [&](auto place_of) {
        each_logit<L>(row, n, thread, threads, [&](int, float x) {
            const Place p = place_of(x);
            atomicAdd(reinterpret_cast<unsigned long long*>(&bins[p.t < end ? p.bin() : nowhere]), word_of(p.f));
        });
    };
    if (P.endless) fill([&](float x) { return P.of(x); });
    else fill([&](float x) { return P.of_finite(x); });
}

// The sorted tokens' places in the row's order, where its prefixes end, and the
// draw, by the first wave alone or the workgroup.
template <bool kWave>
__device__ __forceinline__ void sync_as() {
    if constexpr (kWave) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    } else {
        __syncthreads();
    }
}

template <bool kWave, int kMine, typename L, int kThreads>
__device__ __forceinline__ void finish_as(Shared<kThreads>& S, const Sums& B, uint64_t* sums, const Places<L>& P, const Rules& R, int n, const Found& f, double& kept) {
    const int t = threadIdx.x, wave = t >> 6;
    const int32_t all = B.count[kBins];
    const int bin_k = f.bin_k;
    auto sync = [] { sync_as<kWave>(); };
    // Each token's bin, weight and sums before it in its bin.
    int bin_of[kMine];
    uint32_t w[kMine];
    bool weighs[kMine];  // at least min_p
    int first[kMine];  // of its bin, in the list
    uint64_t mine = 0, all_sum;
    int start = -1, previous = -1;
    if (t * kMine > 0 && t * kMine - 1 < n) previous = P.of(of_key(~static_cast<uint32_t>(S.words[t * kMine - 1] >> 32))).bin();
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const int i = t * kMine + j;
        w[j] = 0, bin_of[j] = 0, first[j] = -1, weighs[j] = false;
        if (i >= n) continue;
        const Place place = P.of(of_key(~static_cast<uint32_t>(S.words[i] >> 32)));
        bin_of[j] = place.bin(), weighs[j] = place.exact() <= R.min_t;
        w[j] = kMostUnits - lack_in_bin(place.f);
        if (bin_of[j] != previous) start = i;
        first[j] = start, previous = bin_of[j];
        mine += w[j];
    }
    uint64_t sum = before_in_wave(mine, all_sum);
    // The last start at or before a thread's tokens: starts rise along the list.
    int starts = start;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const int o = __shfl_up(starts, x);
        if ((t & 63) >= x && o > starts) starts = o;
    }
    const int in_wave = __shfl_up(starts, 1);
    int carried = (t & 63) == 0 ? -1 : in_wave;
    if ((t & 63) == 63) S.wave_best[wave] = all_sum, S.wave_first[wave] = starts;
    sync();
    for (int i = 0; i < wave; ++i) {
        sum += S.wave_best[i];
        carried = S.wave_first[i] > carried ? S.wave_first[i] : carried;
    }
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const int i = t * kMine + j;
        if (i >= n) break;
        sums[i] = sum;
        sum += w[j];
        if (first[j] < 0) first[j] = carried;
    }
    sync();
    // In the row's order: tokens before it, weights before and with it (the last
    // of a bin ends where the next begins). Read once: the sums may lie in
    // global memory.
    int32_t rank[kMine];
    double before[kMine], with[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
        const int i = t * kMine + j, bin = bin_of[j];
        rank[j] = INT32_MAX - 1, before[j] = with[j] = INFINITY;
        if (i >= n) continue;
        const int32_t count = B.count[bin], next = B.count[bin + 1];
        const double base = B.weight[bin], end = B.weight[bin + 1], unit = S.octave.unit(bin);
        const uint64_t from = sums[i] - sums[first[j]];
        rank[j] = count + i - first[j];
        before[j] = base + static_cast<double>(from) * unit;
        with[j] = rank[j] + 1 == next ? end : base + static_cast<double>(from + w[j]) * unit;
    }
    if (bin_k >= 0)
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (rank[j] == R.k - 1) S.end_count[0] = R.k, S.end_weight[0] = with[j];
    sync();
    if (R.p < 1.0) {
        const double x = reached(R.p * (bin_k >= 0 ? S.end_weight[0] : B.weight[kBins]), B.weight[kBins]);
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (before[j] < x && x <= with[j]) S.end_count[1] = rank[j] + 1, S.end_weight[1] = with[j];
    }
    if (f.high_m >= 0) {
        if (t == 0) S.found[2] = B.count[f.low_m];
        sync();
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (bin_of[j] >= f.low_m && bin_of[j] <= f.high_m && weighs[j]) atomicMax(&S.found[2], rank[j] + 1);
        sync();
        if (t == 0 && S.found[2] == B.count[f.low_m]) S.end_count[2] = S.found[2], S.end_weight[2] = B.weight[f.low_m];
#pragma unroll
        for (int j = 0; j < kMine; ++j)
            if (bin_of[j] >= f.low_m && bin_of[j] <= f.high_m && rank[j] + 1 == S.found[2]) S.end_count[2] = S.found[2], S.end_weight[2] = with[j];
    }
    if (t == 0) S.found[3] = 0;
    sync();
    int32_t most = all;
    kept = B.weight[kBins];
    for (int i = 0; i < 3; ++i)
        if (S.end_count[i] < most) most = S.end_count[i], kept = S.end_weight[i];
    const double x = R.u * kept;
#pragma unroll
    for (int j = 0; j < kMine; ++j)
        if (rank[j] < most && before[j] <= x) atomicMax(&S.found[3], rank[j] + 1);
    sync();
#pragma unroll
    for (int j = 0; j < kMine; ++j)
        if (rank[j] + 1 == S.found[3]) {
            S.drawn = static_cast<int32_t>(static_cast<uint32_t>(S.words[t * kMine + j]));
            S.found_weight = static_cast<double>(w[j]) * S.octave.unit(bin_of[j]);
        }
    sync();
}

// Up to kThreads words, in order: each wave sorts 64 in registers, and a word's
// place is its own there plus the numbers of smaller ones in the other waves',
// by bisection. (Counting all smaller words took 12 us for 352, not 2.)
template <int kThreads>
__device__ __forceinline__ void sort_few(Shared<kThreads>& S, int n) {
    const int t = threadIdx.x, lane = t & 63, runs = (n + 63) / 64, mine = t >> 6;
    uint64_t x = t < n ? S.words[t] : ~uint64_t{0};
    if (mine < runs) {
#pragma unroll 1
        for (int span = 2; span <= 64; span *= 2)
#pragma unroll 1
            for (int gap = span / 2; gap > 0; gap /= 2) {
                const uint64_t o = __shfl_xor(x, gap);
                const bool low = ((lane & gap) == 0) == ((lane & span) == 0);
                x = (x < o) == low ? x : o;
            }
        S.words[t] = x;
    }
    if (runs == 1) {
        __syncthreads();
        return;
    }
    __syncthreads();
    int at = lane;
    if (mine < runs)
        for (int r = 0; r < runs; ++r) {
            const uint64_t* const run = S.words + 64 * r;
            int below = 0;
#pragma unroll
            for (int step = 32; step > 0; step /= 2) below += run[below + step - 1] < x ? step : 0;
            below += run[below] < x ? 1 : 0;
            at += r == mine ? 0 : below;
        }
    __syncthreads();
    if (t < n || x != ~uint64_t{0}) S.words[at] = x;
    __syncthreads();
}

// The token, from the S.n gathered ones in the words. sums: room for kList numbers in LDS.
template <typename L, int kThreads>
__device__ __forceinline__ void finish(const SampleArgs& A, Shared<kThreads>& S, const Sums& B, uint64_t* sums, const typename L::Element* row, int row_at,
                                       const Places<L>& P, const Rules& R, const Found& f, int n) {
    constexpr int kEach = kList / kThreads;  // tokens of a thread
    const int t = threadIdx.x;
    if (t < 3) S.end_count[t] = INT32_MAX;
    int32_t token = -1;
    double weight = 0.0, kept = 0.0;
    if (n > kList || n < 1) {
        resolve_large<L>(A, S, B, row, P, R, f, token, weight, kept);
    } else {
        if (n <= kThreads) {
            sort_few(S, n);
        } else {
            int size = 2 * kThreads;
            while (size < n) size *= 2;
            for (int i = n + t; i < size; i += kThreads) S.words[i] = ~uint64_t{0};
            __syncthreads();
            for (int span = 2; span <= size; span *= 2)
                for (int gap = span / 2; gap > 0; gap /= 2) {
                    for (int i = t; i < size / 2; i += kThreads) {
                        const int a = 2 * i - (i & (gap - 1)), b = a + gap;
                        const uint64_t x = S.words[a], y = S.words[b];
                        if ((x > y) == ((a & span) == 0)) S.words[a] = y, S.words[b] = x;
                    }
                    __syncthreads();
                }
        }
        // A wave alone needs no barriers.
        if (n <= 64 * kEach && t >= 64) return;
        if (n <= 64) finish_as<true, 1, L>(S, B, sums, P, R, n, f, kept);
        else if (n <= 64 * kEach) finish_as<true, kEach, L>(S, B, sums, P, R, n, f, kept);
        else finish_as<false, kEach, L>(S, B, sums, P, R, n, f, kept);
        token = S.drawn, weight = S.found_weight;
    }
    if (t == 0) {
        A.tokens[row_at] = token;
        if (A.logprobs != nullptr) A.logprobs[row_at] = static_cast<float>(log(weight / kept));
    }
}

// A row without tokens, or whose largest logit decides.
__device__ __forceinline__ bool decided(const SampleArgs& A, int row_at, uint64_t top, const Rules& R, bool writes) {
    if (top != 0 && !R.greedy) return false;
    if (writes) {
        A.tokens[row_at] = top == 0 ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(top));
        if (A.logprobs != nullptr) A.logprobs[row_at] = top == 0 ? -INFINITY : 0.0f;
    }
    return true;
}

template <int kThreads>
__device__ __forceinline__ void clear(Shared<kThreads>& S) {
    S.octave.make();
    for (int i = threadIdx.x; i < kBins; i += kThreads) S.words[i] = 0;
    if (threadIdx.x == 0) S.n = 0, S.drawn = 0;
}

template <int kThreads>
__device__ __forceinline__ uint64_t largest_of_waves(Shared<kThreads>& S, uint64_t top) {
    constexpr int kWaves = kThreads / 64;
    if ((threadIdx.x & 63) == 0) S.wave_best[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = S.wave_best[i] > top ? S.wave_best[i] : top;
    return top;
}

// Many rows, or few logits: a workgroup a row. 256 rows of 151936 57 us, 37 of
// 50001 in fp32 24.5, one of 4096 13.
template <typename L, int kThreads>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs A) {
    __shared__ Shared<kThreads> S;
    __shared__ double weight[kBins + 1];
    __shared__ int32_t count[kBins + 1];
    __shared__ uint64_t sums[kList];
    Sums B;
    B.weight = weight, B.count = count;
    const int row_at = blockIdx.x;
    const typename L::Element* const row = static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride;
    const Rules R = rules_of(A, row_at);
    clear(S);
    const uint64_t top = largest_of_waves(S, largest<L>(row, A.vocab, threadIdx.x, kThreads, R.greedy));
    if (decided(A, row_at, top, R, threadIdx.x == 0)) return;
    const Places<L> P = places_of<L>(top, R);
    fill_bins<L>(row, A.vocab, threadIdx.x, kThreads, P, R, S.words);
    __syncthreads();
    const Found f = find_bins<true>(S, R, B);
    gather<L>(S, row, A.vocab, threadIdx.x, kThreads, P, f);
    __syncthreads();
    finish<L>(A, S, B, sums, row, row_at, P, R, f, S.n);
}

// Fewer rows: `n` workgroups a row, in four launches: the largest logit; the
// bins; their tokens; by one workgroup, the draw. One row of 151936 in 19 slices
// 3.4, 4.3, 11.6 and 5.8 us, 64 rows in 4 slices 8.6, 10.4, 17.8 and 11.3: from
// the gather on, sums over the bins and steps of a sort that wait for each
// other, not HBM (0.06 and 4 us). (Fewer launches, where the last
// workgroup of a row to come goes on with what the others wrote, need fences
// over all L2s: 64 rows 290 us.)
constexpr int kSliceThreads = 512;

struct Slices {
    uint64_t* tops;      // [rows][n]
    uint64_t* bins;      // [rows][kBins]
    double* weight;      // [rows][kBins + 1]
    uint64_t* list;      // [rows][kList]
    Rules* rules;        // [rows]
    Found* found;        // [rows]
    int32_t* count;      // [rows][kBins + 1]
    int32_t* gathered;   // [rows]
    int32_t n;

    __device__ __forceinline__ Sums sums(int row) const {
        return Sums{weight + static_cast<int64_t>(row) * (kBins + 1), count + static_cast<int64_t>(row) * (kBins + 1)};
    }
};

// (A row has at most 64 slices.)
__device__ __forceinline__ uint64_t top_of(const Slices& W, int row) {
    const int lane = threadIdx.x & 63;
    uint64_t top = W.tops[static_cast<int64_t>(row) * W.n + (lane < W.n ? lane : 0)];
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const uint64_t o = __shfl_xor(top, x);
        top = o > top ? o : top;
    }
    return top;
}

template <typename L>
__global__ __launch_bounds__(kSliceThreads) void sample_top_kernel(const SampleArgs A, const Slices W) {
    __shared__ uint64_t best[kSliceThreads / 64];
    const int row_at = blockIdx.y, t = threadIdx.x;
    for (int i = blockIdx.x * kSliceThreads + t; i < kBins; i += W.n * kSliceThreads) W.bins[static_cast<int64_t>(row_at) * kBins + i] = 0;
    if (blockIdx.x == 0 && t == 0) W.gathered[row_at] = 0, W.rules[row_at] = rules_of(A, row_at);
    uint64_t top = largest<L>(static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride, A.vocab, blockIdx.x * kSliceThreads + t,
                              W.n * kSliceThreads, greedy(A, row_at));
    if ((t & 63) == 0) best[t >> 6] = top;
    __syncthreads();
    for (int i = 0; i < kSliceThreads / 64; ++i) top = best[i] > top ? best[i] : top;
    if (t == 0) W.tops[static_cast<int64_t>(row_at) * W.n + blockIdx.x] = top;
}

template <typename L>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(const SampleArgs A, const Slices W) {
    __shared__ uint64_t words[kBins + 64];
    const int row_at = blockIdx.y, t = threadIdx.x;
    const typename L::Element* const row = static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride;
    const Rules R = W.rules[row_at];
    const uint64_t top = top_of(W, row_at);
    if (decided(A, row_at, top, R, blockIdx.x == 0 && t == 0)) return;
    for (int i = t; i < kBins; i += kSliceThreads) words[i] = 0;
    __syncthreads();
    fill_bins<L>(row, A.vocab, blockIdx.x * kSliceThreads + t, W.n * kSliceThreads, places_of<L>(top, R), R, words);
    __syncthreads();
    uint64_t* const bins = W.bins + static_cast<int64_t>(row_at) * kBins;
    for (int i = t; i < kBins; i += kSliceThreads)
        if (words[i] != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&bins[i]), words[i]);
}

// (Each workgroup looks at the bins for itself: a launch for that took 4 us more.)
template <typename L>
__global__ __launch_bounds__(kSliceThreads) void sample_gather_kernel(const SampleArgs A, const Slices W) {
    __shared__ Shared<kSliceThreads> S;
    const int row_at = blockIdx.y, t = threadIdx.x;
    const typename L::Element* const row = static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride;
    const Rules R = W.rules[row_at];
    const uint64_t top = top_of(W, row_at);
    if (decided(A, row_at, top, R, false)) return;
    S.octave.make();
    for (int i = t; i < kBins; i += kSliceThreads) S.words[i] = W.bins[static_cast<int64_t>(row_at) * kBins + i];
    if (t == 0) S.n = 0;
    __syncthreads();
    const Found f = find_bins<false>(S, R, blockIdx.x == 0 ? W.sums(row_at) : Sums{nullptr, nullptr});
    if (blockIdx.x == 0 && t == 0) W.found[row_at] = f;
    gather<L>(S, row, A.vocab, blockIdx.x * kSliceThreads + t, W.n * kSliceThreads, places_of<L>(top, R), f);
    __syncthreads();
    // Its tokens to the row's.
    uint64_t* const list = W.list + static_cast<int64_t>(row_at) * kList;
    const int32_t n = S.n;
    if (n == 0) return;
    if (t == 0) S.at = atomicAdd(&W.gathered[row_at], n);
    __syncthreads();
    const int32_t at = S.at;
    for (int i = t; i < n && i < kList && at + i < kList; i += kSliceThreads) list[at + i] = S.words[i];
}

template <typename L>
__global__ __launch_bounds__(kSliceThreads) void sample_draw_kernel(const SampleArgs A, const Slices W) {
    __shared__ Shared<kSliceThreads> S;
    __shared__ uint64_t sums[kList];
    const int row_at = blockIdx.x, t = threadIdx.x;
    const typename L::Element* const row = static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride;
    const Rules R = W.rules[row_at];
    const uint64_t top = top_of(W, row_at);
    if (decided(A, row_at, top, R, false)) return;
    const int32_t n = W.gathered[row_at];
    S.octave.make();
    if (n <= kList) {
        for (int i = t; i < n; i += kSliceThreads) S.words[i] = W.list[static_cast<int64_t>(row_at) * kList + i];
    } else {  // too many tokens to sort: every bin's sums are needed
        for (int i = t; i < kBins; i += kSliceThreads) S.words[i] = W.bins[static_cast<int64_t>(row_at) * kBins + i];
        __syncthreads();
        find_bins<true>(S, R, W.sums(row_at));
    }
    __syncthreads();
    finish<L>(A, S, W.sums(row_at), sums, row, row_at, places_of<L>(top, R), R, W.found[row_at], n);
}

}  // namespace
}  // namespace aimg

namespace aimg {
namespace {

// Threads of a row's only workgroup: 1024 where its logits are many, which are
// read and put into bins faster by more waves; else 512, since barriers cost
// more the more waves there are. (256 rows with top_p 0.9, by 512 and by 1024:
// of 4096 logits of 16 bits 13.8 us and 15.2, 16384 20.4 and 20.2, 32000 25.7
// and 23.8, 151936 85.7 and 63.9; of 16384 in fp32 18.3 and 18.2, 32000 31.3 and
// 25.7.)
constexpr int64_t kWideBytes = 48 << 10;

// Workgroups a row; 0: one, in one launch. Four launches, and bins that each
// workgroup looks at for itself, pay where rows are long and do not fill the
// chip. What a row costs goes by its tokens and an eighth of its bytes; that is
// compared with a number that rises with the rows, and faster where four
// workgroups a row are more than the 256 CUs.
// Several workgroups' time by one's, for rows with all kept, top_p 0.9, top-k 50
// and top_p 0.95, and settings of their own (us by one, with all kept):
//   bf16, 65536 logits: 1 row 0.91 - 0.99 (23), 12 rows 1.02 - 1.08 (28), 64 1.12 - 1.21 (30)
//   bf16, 90112: 8 rows 0.87 - 0.94 (31), 32 0.95 - 1.03 (34), 64 1.03 - 1.10 (36)
//   bf16, 151936: 1 row 0.61 - 0.65 (38), 64 0.87 - 1.04 (49), 72 1.00 - 1.18 (49)
//   bf16, 262144: 64 rows 0.76 - 0.89 (74), 96 0.87 - 1.03 (77), 192 1.16 - 1.24 (86)
//   fp32, 50001: 1 row 0.95 - 1.01 (22), 8 1.02 - 1.06 (24)
//   fp32, 65536: 8 rows 0.94 - 0.98 (29), 40 1.07 - 1.14 (31)
//   fp32, 151936: 64 rows 0.83 - 0.93 (61), 80 0.92 - 0.95 (62), 128 1.04 - 1.13 (63)
//   fp32, 262144: 128 rows 0.93 - 1.01 (113), 192 1.08 - 1.11 (128)
// Of 994 such measurements, of 50001 to 262144 logits and 1 to 256 rows, it chooses
// what takes over 5% longer in 12, 11% at most.
constexpr int64_t kDealtLeast = 90000, kDealtRow = 640, kDealtManyRow = 2700, kOneEachRows = 64;

int slices_of(int64_t n_rows, int vocab, int element_bytes) {
    const int64_t cost = static_cast<int64_t>(vocab) * (8 + element_bytes) / 8;
    if (n_rows < 1 || cost < (n_rows <= kOneEachRows ? kDealtLeast + kDealtRow * n_rows : kDealtManyRow * n_rows)) return 0;
    const int64_t most = (vocab + 8191) / 8192, n = 256 / n_rows;
    return static_cast<int>(n < 4 ? 4 : n < most ? n : most);
}

// Where a call's arrays lie in its workspace, those of 8 bytes first; returns its size.
size_t slices_at(Slices& w, char* at, int64_t rows) {
    const size_t tops = 8 * static_cast<size_t>(rows) * w.n, bins = 8 * static_cast<size_t>(rows) * kBins, weight = 8 * static_cast<size_t>(rows) * (kBins + 1);
    const size_t list = 8 * static_cast<size_t>(rows) * kList, rules = sizeof(Rules) * rows, found = sizeof(Found) * rows, count = 4 * static_cast<size_t>(rows) * (kBins + 1);
    w.tops = reinterpret_cast<uint64_t*>(at), w.bins = reinterpret_cast<uint64_t*>(at + tops), w.weight = reinterpret_cast<double*>(at + tops + bins);
    w.list = reinterpret_cast<uint64_t*>(at + tops + bins + weight), w.rules = reinterpret_cast<Rules*>(at + tops + bins + weight + list);
    at += tops + bins + weight + list + rules;
    w.found = reinterpret_cast<Found*>(at), w.gathered = reinterpret_cast<int32_t*>(at + found);
    w.count = reinterpret_cast<int32_t*>(at + found + 4 * rows);
    return tops + bins + weight + list + rules + found + 4 * rows + count;
}

template <typename L>
void launch_sample(const SampleArgs& a, int64_t n_rows, const Slices& w, hipStream_t s) {
    const dim3 rows(static_cast<uint32_t>(n_rows)), slices(static_cast<uint32_t>(w.n), static_cast<uint32_t>(n_rows)), block(kSliceThreads);
    if (w.n == 0) {
        if (static_cast<int64_t>(a.vocab) * sizeof(typename L::Element) < kWideBytes) hipLaunchKernelGGL((sample_kernel<L, 512>), rows, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((sample_kernel<L, 1024>), rows, dim3(1024), 0, s, a);
        return;
    }
    hipLaunchKernelGGL((sample_top_kernel<L>), slices, block, 0, s, a, w);
    hipLaunchKernelGGL((sample_bins_kernel<L>), slices, block, 0, s, a, w);
    hipLaunchKernelGGL((sample_gather_kernel<L>), slices, block, 0, s, a, w);
    hipLaunchKernelGGL((sample_draw_kernel<L>), rows, block, 0, s, a, w);
}

int check_sample(int64_t n_rows, int vocab) {
    if (n_rows < 0 || vocab < 1) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: n_rows must not be negative and vocab at least 1");
    if (vocab > kMaxVocab || n_rows > kMaxRows) return fail(AIMG_ERR_UNSUPPORTED, "sample: vocab must be at most 2^18 and n_rows 2^21");
    return AIMG_OK;
}

}  // namespace
}  // namespace aimg

extern "C" int aimg_sample_workspace_nbytes(int64_t n_rows, int vocab, size_t* nbytes) {
    if (nbytes == nullptr) return aimg::fail(AIMG_ERR_INVALID_ARGUMENT, "nbytes is null");
    const int rc = aimg::check_sample(n_rows, vocab);
    if (rc != AIMG_OK) return rc;
    aimg::Slices w{};
    w.n = aimg::slices_of(n_rows, vocab, 4);  // whatever the logits' type: more are dealt out in 32 bits, to as many workgroups
    *nbytes = w.n == 0 ? 0 : aimg::slices_at(w, nullptr, n_rows);
    return AIMG_OK;
}

extern "C" int aimg_sample(const void* logits, int64_t n_rows, int64_t row_stride, int vocab, int type, const float* uniforms,
                           const aimg_sampling* settings, int64_t* tokens, float* logprobs, void* workspace, size_t workspace_nbytes,
                           void* stream) {
    using aimg::fail;
    const int rc = aimg::check_sample(n_rows, vocab);
    if (rc != AIMG_OK) return rc;
    if (row_stride < 0) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: row_stride must not be negative");
    if (type != AIMG_BF16 && type != AIMG_FP16 && type != AIMG_FP32)
        return fail(AIMG_ERR_UNSUPPORTED, "sample: type must be AIMG_BF16, AIMG_FP16 or AIMG_FP32, got " + std::to_string(type));
    if (settings == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: settings is null");
    if (n_rows == 0) return AIMG_OK;
    if (logits == nullptr || uniforms == nullptr || tokens == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: null pointer");
    if (reinterpret_cast<uintptr_t>(logits) % (type == AIMG_FP32 ? 4 : 2) != 0 || reinterpret_cast<uintptr_t>(tokens) % 8 != 0)
        return fail(AIMG_ERR_UNSUPPORTED, "sample: logits and tokens must be aligned to their elements");
    aimg::Slices w{};
    w.n = aimg::slices_of(n_rows, vocab, type == AIMG_FP32 ? 4 : 2);
    if (w.n > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 8 != 0 ||
                    workspace_nbytes < aimg::slices_at(w, static_cast<char*>(workspace), n_rows)))
        return fail(AIMG_ERR_INVALID_ARGUMENT, "the workspace is null, misaligned or below aimg_sample_workspace_nbytes");
    aimg::SampleArgs a{};
    a.logits = logits, a.row_stride = row_stride, a.uniforms = uniforms, a.vocab = vocab;
    a.temperatures = settings->temperatures, a.top_ks = settings->top_ks, a.top_ps = settings->top_ps, a.min_ps = settings->min_ps;
    a.temperature = settings->temperature, a.top_k = settings->top_k, a.top_p = settings->top_p, a.min_p = settings->min_p;
    a.tokens = tokens, a.logprobs = logprobs;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == AIMG_BF16) aimg::launch_sample<aimg::LogitBf16>(a, n_rows, w, s);
    else if (type == AIMG_FP16) aimg::launch_sample<aimg::LogitFp16>(a, n_rows, w, s);
    else aimg::launch_sample<aimg::LogitFp32>(a, n_rows, w, s);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
    return AIMG_OK;
}
