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
// Sums. A token's place t = 64 log2(1 / w) is computed in 64 bits; its whole
// part is its bin, and its weight against the bin's top is rounded to 2^-26. A
// bin's count and sum are integers in one 64-bit word, so a row's result does
// not depend on the order of the atomics that add them; sums of bins are
// doubles, in a fixed order. Tokens below 2^-64 of the largest weigh nothing.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "afterimage_decode.h"
#include "aimg_internal.h"

namespace aimg {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kPerOctave = 64;             // bins of a factor of 2
constexpr int kBins = 4096;
constexpr int kEach = kBins / kThreads;    // bins, and sorted tokens, of a thread
constexpr int kList = 4096;                // tokens that are gathered and sorted
constexpr int kCountShift = 45;            // of a bin's word: count above, sum of weights (in 2^-26) below
constexpr uint64_t kSumMask = (uint64_t{1} << kCountShift) - 1;
constexpr int kMaxVocab = 1 << 18;         // so that neither overflows
constexpr float kUnit = 67108864.0f;       // 2^26

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

// Calls f(index, logit) for logits thread, thread + step, .. of 16-byte pieces
// (a row may begin and end anywhere; what lies outside whole pieces comes one by
// one), each thread's by rising index. A NaN is -inf, which no token has.
template <typename L, typename F>
__device__ __forceinline__ void each_logit(const typename L::Element* row, int n, int thread, int threads, F f) {
    typedef typename L::Element E;
    constexpr int kPiece = 16 / sizeof(E), kAhead = 4;
    auto give = [&](int i, float x) { f(i, x != x ? -INFINITY : x); };
    int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(E));
    if (head > n) head = n;
    if (thread < head) give(thread, L::value(row[thread]));
    const int pieces = (n - head) / kPiece;
    for (int c0 = thread; c0 < pieces; c0 += kAhead * threads) {
        uint4 w[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int c = c0 + j * threads;
            w[j] = *reinterpret_cast<const uint4*>(row + head + static_cast<int64_t>(c < pieces ? c : c0) * kPiece);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int c = c0 + j * threads;
            if (c >= pieces) break;
            const uint32_t u[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
            for (int e = 0; e < kPiece; ++e)
                give(head + c * kPiece + e, L::value(static_cast<E>(sizeof(E) == 2 ? u[e / 2] >> 16 * (e % 2) : u[e])));
        }
    }
    const int done = head + pieces * kPiece;
    if (done + thread < n) give(done + thread, L::value(row[done + thread]));  // fewer than a piece
}

// Unsigned numbers in the order of logits; equal ones for both zeros.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// A token's place: how far below the largest, 64 to a factor of 2. (max - x is
// exact in 64 bits or rounds without changing the order; an infinite maximum
// leaves its equals alone at 0.)
struct Places {
    double top, per;
    __device__ __forceinline__ double of(float x) const { return static_cast<double>(x) == top ? 0.0 : (top - static_cast<double>(x)) * per; }
};

// 2^(-f / 64) in 2^-26, f in [0, 1): one minus its series in g = f ln 2 / 64 < 0.011, whose fourth term is below 2^-30.
__device__ __forceinline__ uint32_t weight_in_bin(float f) {
    const float g = f * (0.693147180559945f / kPerOctave);
    const float less = g * (1.0f - g * (0.5f - g * (1.0f / 6.0f)));
    return static_cast<uint32_t>(kUnit) - static_cast<uint32_t>(__float2int_rn(less * kUnit));
}

__device__ __forceinline__ uint64_t word_of(double t) {
    const int bin = static_cast<int>(t);
    return uint64_t{1} << kCountShift | weight_in_bin(static_cast<float>(t - bin));
}

// What a unit of a bin's sum weighs.
__device__ __forceinline__ double unit_of(int bin) { return exp2(-static_cast<double>(bin) / kPerOctave - 26.0); }

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

struct Shared {
    uint64_t words[kBins];      // bins, then the gathered tokens: ~key above, index below
    double weight[kBins + 1];   // of the bins before
    int32_t count[kBins + 1];
    uint64_t sums[kList];       // of the tokens before, in their bins' units
    double wave_weight[kWaves];
    uint64_t wave_best[kWaves];
    int32_t wave_count[kWaves], wave_first[kWaves];
    double end_weight[3], found_weight;
    int32_t end_count[3], found[4], n, drawn;
};

// Sums over the bins before each, and of all.
__device__ __forceinline__ void sum_bins(Shared& S) {
    const int t = threadIdx.x, wave = t >> 6;
    int32_t c[kEach], all_c;
    double w[kEach], all_w;
    int32_t my_c = 0;
    double my_w = 0.0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const uint64_t x = S.words[t * kEach + j];
        c[j] = static_cast<int32_t>(x >> kCountShift);
        w[j] = x == 0 ? 0.0 : static_cast<double>(x & kSumMask) * unit_of(t * kEach + j);
        my_c += c[j], my_w += w[j];
    }
    int32_t at_c = before_in_wave(my_c, all_c);
    double at_w = before_in_wave(my_w, all_w);
    if ((t & 63) == 0) S.wave_count[wave] = all_c, S.wave_weight[wave] = all_w;
    __syncthreads();
    double base = 0.0;
    for (int i = 0; i < wave; ++i) at_c += S.wave_count[i], base += S.wave_weight[i];
    at_w += base;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        S.count[t * kEach + j] = at_c, S.weight[t * kEach + j] = at_w;
        at_c += c[j], at_w += w[j];
    }
    if (t == kThreads - 1) S.count[kBins] = at_c, S.weight[kBins] = at_w;
    __syncthreads();
}

// The bin where a weight is reached (weight before < x <= with it) or passed (<=, <): one thread finds it.
template <bool kPassed>
__device__ __forceinline__ void find_weight(Shared& S, double x, int32_t* to) {
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int b = threadIdx.x * kEach + j;
        const double low = S.weight[b], high = S.weight[b + 1];
        if (kPassed ? low <= x && x < high : low < x && x <= high) *to = b;
    }
}

// A row's settings. Numbers out of range mean the nearest in it: no rule, or the first token.
struct Rules {
    bool greedy;
    double per, p, min_t, u;
    int32_t k;
};

__device__ __forceinline__ Rules rules_of(const SampleArgs& A, int row) {
    Rules r;
    const double t = A.temperatures != nullptr ? A.temperatures[row] : A.temperature;
    const double p = A.top_ps != nullptr ? A.top_ps[row] : A.top_p, m = A.min_ps != nullptr ? A.min_ps[row] : A.min_p;
    const int32_t k = A.top_ks != nullptr ? A.top_ks[row] : A.top_k;
    const double u = A.uniforms[row];
    r.greedy = !(t > 0.0);
    r.per = r.greedy ? 0.0 : kPerOctave * 1.4426950408889634 / t;
    if (r.per > 1e300) r.per = 1e300;
    r.k = k > 0 ? k : INT32_MAX;
    r.p = p < 1.0 ? (p > 0.0 ? p : 0.0) : 1.0;
    r.min_t = m > 0.0 ? (m < 1.0 ? -kPerOctave * log2(m) : 0.0) : INFINITY;
    r.u = u > 0.0 ? (u < 1.0 ? u : 1.0 - 0x1p-53) : 0.0;
    return r;
}

// How a prefix ends, or which token is drawn, where a bin holds more tokens
// than are gathered (equal logits by the thousand, very high temperatures): the
// bin's keys are binned again, 4096 at a time, until one key is left. It ends
// after at most three passes over the row.
struct Equals {
    uint32_t key;
    int32_t count, n;      // tokens before the equals, and the equals
    double weight, each;   // of those before, and of one of them
};

enum Goal { kCounted, kReached, kPassed };

template <typename L, Goal kGoal>
__device__ Equals narrow(const SampleArgs& A, Shared& S, const typename L::Element* row, const Places& P, int bin, int32_t k, double x) {
    uint32_t low = 0, high = 0xFFFFFFFFu;
    int32_t count = S.count[bin];
    double weight = S.weight[bin];
    const double unit = unit_of(bin);
    __shared__ int32_t at;
    __shared__ int32_t before_count, inside_count;
    __shared__ double before_weight;
    __shared__ uint64_t inside;
    for (;;) {
        int shift = 0;
        while (((high - low) >> shift) >= kBins) ++shift;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) S.words[i] = 0;
        if (threadIdx.x == 0) at = -1;
        __syncthreads();
        each_logit<L>(row, A.vocab, threadIdx.x, kThreads, [&](int, float v) {
            const double t = P.of(v);
            const uint32_t key = key_of(v);
            if (t < kBins && static_cast<int>(t) == bin && key >= low && key <= high)
                atomicAdd(reinterpret_cast<unsigned long long*>(&S.words[(high - key) >> shift]), word_of(t));
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
                const int32_t c0 = count + static_cast<int32_t>(sum >> kCountShift), c1 = count + static_cast<int32_t>(next >> kCountShift);
                const double w0 = weight + static_cast<double>(sum & kSumMask) * unit;
                // The last part takes what rounding leaves over.
                const double w1 = next == total ? INFINITY : weight + static_cast<double>(next & kSumMask) * unit;
                const bool first = sum == 0;
                const bool here = kGoal == kCounted ? c0 < k && (k <= c1 || next == total)
                                  : kGoal == kReached ? (first || w0 < x) && x <= w1 : (first || w0 <= x) && x < w1;
                if (here) at = threadIdx.x * kEach + j, before_count = c0, before_weight = w0, inside = one, inside_count = c1 - c0;
            }
            sum = next;
        }
        __syncthreads();
        if (at < 0) {  // no token of the bin, which no caller asks for
            Equals none{0, count, 0, weight, 0.0};
            return none;
        }
        count = before_count, weight = before_weight;
        const uint32_t part = static_cast<uint32_t>(at);
        const uint32_t top = high - (part << shift), size = shift == 0 ? 1u : 1u << shift;
        const uint32_t bottom = top - low < size ? low : top - size + 1;
        if (shift == 0) {
            Equals e{top, count, inside_count, weight, static_cast<double>(inside & kSumMask) / inside_count * unit};
            __syncthreads();
            return e;
        }
        high = top, low = bottom;
        __syncthreads();
    }
}

// The index of the j-th token with this key.
template <typename L>
__device__ int32_t index_of(const SampleArgs& A, Shared& S, const typename L::Element* row, uint32_t key, int32_t j) {
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
template <typename L>
__device__ void resolve_large(const SampleArgs& A, Shared& S, const typename L::Element* row, const Places& P, const Rules& R, int bin_k, int bin_m,
                              int32_t& token, double& weight, double& kept) {
    int32_t most = S.count[kBins];
    kept = S.weight[kBins];
    auto find = [&](double x, bool passed) {
        __syncthreads();
        if (threadIdx.x == 0) S.found[0] = -1;
        __syncthreads();
        if (passed) find_weight<true>(S, x, &S.found[0]);
        else find_weight<false>(S, x, &S.found[0]);
        __syncthreads();
        return S.found[0];
    };
    if (bin_k >= 0) {
        const Equals e = narrow<L, kCounted>(A, S, row, P, bin_k, R.k, 0.0);
        most = R.k;
        kept = e.weight + (R.k - e.count) * e.each;
    }
    if (R.p < 1.0) {
        double x = R.p * kept;
        x = x < 1e-300 ? 1e-300 : x > S.weight[kBins] ? S.weight[kBins] : x;
        const int b = find(x, false);
        if (b >= 0) {
            const Equals e = narrow<L, kReached>(A, S, row, P, b, 0, x);
            double n = ceil((x - e.weight) / e.each);
            n = n < 1.0 ? 1.0 : n > e.n ? e.n : n;
            if (e.count + static_cast<int32_t>(n) < most) most = e.count + static_cast<int32_t>(n), kept = e.weight + n * e.each;
        }
    }
    if (bin_m >= 0 && S.count[bin_m] < most) {
        // The tokens of the bin that weigh enough.
        __syncthreads();
        if (threadIdx.x == 0) S.sums[0] = 0;
        __syncthreads();
        uint64_t mine = 0;
        each_logit<L>(row, A.vocab, threadIdx.x, kThreads, [&](int, float v) {
            const double t = P.of(v);
            if (t < kBins && static_cast<int>(t) == bin_m && t <= R.min_t) mine += word_of(t);
        });
        if (mine != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&S.sums[0]), mine);
        __syncthreads();
        const int32_t n = S.count[bin_m] + static_cast<int32_t>(S.sums[0] >> kCountShift);
        if (n < most) most = n, kept = S.weight[bin_m] + static_cast<double>(S.sums[0] & kSumMask) * unit_of(bin_m);
    }
    const double x = R.u * kept;
    int b = find(x, true);
    if (b < 0) b = find(S.weight[kBins], false);
    const Equals e = narrow<L, kPassed>(A, S, row, P, b < 0 ? 0 : b, 0, x);
    double j = floor((x - e.weight) / e.each);
    j = j < 0.0 ? 0.0 : j > e.n - 1 ? e.n - 1 : j;
    if (e.count + j > most - 1) j = most - 1 > e.count ? most - 1 - e.count : 0;
    token = index_of<L>(A, S, row, e.key, static_cast<int32_t>(j));
    weight = e.each;
}

// A workgroup a row. Bound by the arithmetic on its tokens (64-bit places).
template <typename L>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs A) {
    __shared__ Shared S;
    const int row_at = blockIdx.x, t = threadIdx.x, wave = t >> 6;
    const typename L::Element* const row = static_cast<const typename L::Element*>(A.logits) + row_at * A.row_stride;
    const Rules R = rules_of(A, row_at);

    // The largest logit and its first token; the bins are empty meanwhile.
    for (int i = t; i < kBins; i += kThreads) S.words[i] = 0;
    float best = -INFINITY;
    int32_t best_at = -1;
    each_logit<L>(row, A.vocab, t, kThreads, [&](int i, float x) {
        if (x > best || (x == best && i < best_at)) best = x, best_at = i;
    });
    uint64_t top = static_cast<uint64_t>(key_of(best)) << 32 | ~static_cast<uint32_t>(best_at);
    if (best_at < 0) top = 0;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
        const uint64_t o = __shfl_xor(top, x);
        top = o > top ? o : top;
    }
    if ((t & 63) == 0) S.wave_best[wave] = top;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) top = S.wave_best[i] > top ? S.wave_best[i] : top;
    if (top == 0 || R.greedy) {
        if (t == 0) {
            A.tokens[row_at] = top == 0 ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(top));
            if (A.logprobs != nullptr) A.logprobs[row_at] = top == 0 ? -INFINITY : 0.0f;
        }
        return;
    }
    const Places P{static_cast<double>(of_key(static_cast<uint32_t>(top >> 32))), R.per};

    each_logit<L>(row, A.vocab, t, kThreads, [&](int, float x) {
        const double place = P.of(x);
        if (place < kBins) atomicAdd(reinterpret_cast<unsigned long long*>(&S.words[static_cast<int>(place)]), word_of(place));
    });
    __syncthreads();
    sum_bins(S);

    // The bins where the prefixes may end (what the first k weigh is known to a
    // bin, so what p of it is lies in some range) and the draw may fall.
    const int32_t all = S.count[kBins];
    if (t < 4) S.found[t] = -1;
    if (t < 3) S.end_count[t] = INT32_MAX;
    if (t == 0) S.n = 0, S.drawn = 0;
    __syncthreads();
    if (R.k < all) {
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (S.count[t * kEach + j] < R.k && R.k <= S.count[t * kEach + j + 1]) S.found[0] = t * kEach + j;
    }
    __syncthreads();
    const int bin_k = S.found[0];
    const double low_k = bin_k >= 0 ? S.weight[bin_k] : S.weight[kBins], high_k = bin_k >= 0 ? S.weight[bin_k + 1] : S.weight[kBins];
    auto reached = [&](double x) { return x < 1e-300 ? 1e-300 : x > S.weight[kBins] ? S.weight[kBins] : x; };
    if (R.p < 1.0) {
        find_weight<false>(S, reached(R.p * low_k), &S.found[1]);
        find_weight<false>(S, reached(R.p * high_k), &S.found[2]);
    }
    __syncthreads();
    const int low_p = S.found[1], high_p = S.found[2];
    const int bin_m = R.min_t < kBins ? static_cast<int>(R.min_t) : -1;
    int low_end = kBins - 1, high_end = kBins - 1;
    auto ends = [&](int low, int high) {
        if (high < 0) return;
        low_end = low < low_end ? low : low_end, high_end = high < high_end ? high : high_end;
    };
    ends(bin_k, bin_k), ends(low_p, high_p), ends(bin_m, bin_m);
    __syncthreads();
    if (t < 2) S.found[t] = -1;
    __syncthreads();
    find_weight<true>(S, R.u * S.weight[low_end], &S.found[0]);
    find_weight<true>(S, R.u * S.weight[high_end + 1], &S.found[1]);
    __syncthreads();
    const int low_u = S.found[0], high_u = S.found[1];

    // Their tokens.
    auto wanted = [&](int b) {
        return b == bin_k || (b >= low_p && b <= high_p) || (b == bin_m && bin_m <= high_end) || (b >= low_u && b <= high_u);
    };
    int last = bin_k > high_p ? bin_k : high_p;
    last = high_u > last ? high_u : last;
    last = bin_m <= high_end && bin_m > last ? bin_m : last;
    __syncthreads();
    each_logit<L>(row, A.vocab, t, kThreads, [&](int i, float x) {
        const double place = P.of(x);
        if (place < last + 1 && wanted(static_cast<int>(place))) {
            const int at = atomicAdd(&S.n, 1);
            if (at < kList) S.words[at] = static_cast<uint64_t>(~key_of(x)) << 32 | static_cast<uint32_t>(i);
        }
    });
    __syncthreads();
    const int n = S.n;
    int32_t token = -1;
    double weight = 0.0, kept = 0.0;
    if (n > kList || n == 0) {
        resolve_large<L>(A, S, row, P, R, bin_k, bin_m, token, weight, kept);
    } else {
        int size = 64;
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
        // Each token's bin, weight and sums before it in its bin.
        double place[kEach];
        uint32_t w[kEach];
        int first[kEach];  // of its bin, in the list
        uint64_t mine = 0, all_sum;
        int start = -1, previous = -1;
        if (t * kEach > 0 && t * kEach - 1 < n) previous = static_cast<int>(P.of(of_key(~static_cast<uint32_t>(S.words[t * kEach - 1] >> 32))));
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = t * kEach + j;
            w[j] = 0, place[j] = 0.0, first[j] = -1;
            if (i >= n) continue;
            place[j] = P.of(of_key(~static_cast<uint32_t>(S.words[i] >> 32)));
            const int bin = static_cast<int>(place[j]);
            w[j] = weight_in_bin(static_cast<float>(place[j] - bin));
            if (bin != previous) start = i;
            first[j] = start, previous = bin;
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
        __syncthreads();
        for (int i = 0; i < wave; ++i) {
            sum += S.wave_best[i];
            carried = S.wave_first[i] > carried ? S.wave_first[i] : carried;
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = t * kEach + j;
            if (i >= n) break;
            S.sums[i] = sum;
            sum += w[j];
            if (first[j] < 0) first[j] = carried;
        }
        __syncthreads();
        // In the row's order: tokens before it, weights before and with it (the last of a bin ends where the next begins).
        auto before = [&](int j) {
            const int bin = static_cast<int>(place[j]);
            return S.weight[bin] + static_cast<double>(S.sums[t * kEach + j] - S.sums[first[j]]) * unit_of(bin);
        };
        auto with = [&](int j) {
            const int i = t * kEach + j, bin = static_cast<int>(place[j]);
            if (S.count[bin] + i - first[j] + 1 == S.count[bin + 1]) return S.weight[bin + 1];
            return S.weight[bin] + static_cast<double>(S.sums[i] - S.sums[first[j]] + w[j]) * unit_of(bin);
        };
        auto rank = [&](int j) { return S.count[static_cast<int>(place[j])] + t * kEach + j - first[j]; };
        const int mine_n = n - t * kEach < kEach ? n - t * kEach : kEach;
        if (bin_k >= 0)
            for (int j = 0; j < mine_n; ++j)
                if (rank(j) == R.k - 1) S.end_count[0] = R.k, S.end_weight[0] = with(j);
        __syncthreads();
        if (R.p < 1.0) {
            const double x = reached(R.p * (bin_k >= 0 ? S.end_weight[0] : S.weight[kBins]));
            for (int j = 0; j < mine_n; ++j)
                if (before(j) < x && x <= with(j)) S.end_count[1] = rank(j) + 1, S.end_weight[1] = with(j);
        }
        if (bin_m >= 0 && bin_m <= high_end) {
            if (t == 0) S.found[2] = S.count[bin_m];
            __syncthreads();
            for (int j = 0; j < mine_n; ++j)
                if (static_cast<int>(place[j]) == bin_m && place[j] <= R.min_t) atomicMax(&S.found[2], rank(j) + 1);
            __syncthreads();
            if (t == 0 && S.found[2] == S.count[bin_m]) S.end_count[2] = S.found[2], S.end_weight[2] = S.weight[bin_m];
            for (int j = 0; j < mine_n; ++j)
                if (static_cast<int>(place[j]) == bin_m && rank(j) + 1 == S.found[2]) S.end_count[2] = S.found[2], S.end_weight[2] = with(j);
        }
        if (t == 0) S.found[3] = 0;
        __syncthreads();
        int32_t most = all;
        kept = S.weight[kBins];
        for (int i = 0; i < 3; ++i)
            if (S.end_count[i] < most) most = S.end_count[i], kept = S.end_weight[i];
        const double x = R.u * kept;
        for (int j = 0; j < mine_n; ++j)
            if (rank(j) < most && before(j) <= x) atomicMax(&S.found[3], rank(j) + 1);
        __syncthreads();
        for (int j = 0; j < mine_n; ++j)
            if (rank(j) + 1 == S.found[3]) {
                S.drawn = static_cast<int32_t>(static_cast<uint32_t>(S.words[t * kEach + j]));
                S.found_weight = static_cast<double>(w[j]) * unit_of(static_cast<int>(place[j]));
            }
        __syncthreads();
        token = S.drawn, weight = S.found_weight;
    }
    if (t == 0) {
        A.tokens[row_at] = token;
        if (A.logprobs != nullptr) A.logprobs[row_at] = static_cast<float>(log(weight / kept));
    }
}

}  // namespace
}  // namespace aimg

extern "C" int aimg_sample(const void* logits, int64_t n_rows, int64_t row_stride, int vocab, int type, const float* uniforms,
                           const aimg_sampling* settings, int64_t* tokens, float* logprobs, void* stream) {
    using aimg::fail;
    if (n_rows < 0 || n_rows > INT32_MAX || vocab < 1 || row_stride < 0)
        return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: n_rows must be in 0..2^31-1, vocab at least 1 and row_stride not negative");
    if (vocab > aimg::kMaxVocab) return fail(AIMG_ERR_UNSUPPORTED, "sample: vocab must be at most 2^18");
    if (type != AIMG_BF16 && type != AIMG_FP16 && type != AIMG_FP32)
        return fail(AIMG_ERR_UNSUPPORTED, "sample: type must be AIMG_BF16, AIMG_FP16 or AIMG_FP32, got " + std::to_string(type));
    if (settings == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: settings is null");
    if (n_rows == 0) return AIMG_OK;
    if (logits == nullptr || uniforms == nullptr || tokens == nullptr) return fail(AIMG_ERR_INVALID_ARGUMENT, "sample: null pointer");
    if (reinterpret_cast<uintptr_t>(logits) % (type == AIMG_FP32 ? 4 : 2) != 0 || reinterpret_cast<uintptr_t>(tokens) % 8 != 0)
        return fail(AIMG_ERR_UNSUPPORTED, "sample: logits and tokens must be aligned to their elements");
    aimg::SampleArgs a{};
    a.logits = logits, a.row_stride = row_stride, a.uniforms = uniforms, a.vocab = vocab;
    a.temperatures = settings->temperatures, a.top_ks = settings->top_ks, a.top_ps = settings->top_ps, a.min_ps = settings->min_ps;
    a.temperature = settings->temperature, a.top_k = settings->top_k, a.top_p = settings->top_p, a.min_p = settings->min_p;
    a.tokens = tokens, a.logprobs = logprobs;
    const dim3 grid(static_cast<uint32_t>(n_rows)), block(aimg::kThreads);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == AIMG_BF16) hipLaunchKernelGGL((aimg::sample_kernel<aimg::LogitBf16>), grid, block, 0, s, a);
    else if (type == AIMG_FP16) hipLaunchKernelGGL((aimg::sample_kernel<aimg::LogitFp16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((aimg::sample_kernel<aimg::LogitFp32>), grid, block, 0, s, a);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return fail(AIMG_ERR_HIP, std::string("kernel launch failed: ") + hipGetErrorString(err));
    return AIMG_OK;
}
